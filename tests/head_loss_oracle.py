"""64-bit definitions of the vocabulary-head losses, with the error bounds their kernels are held to.

Bounds are elementwise.  ``logit``: an fp32 sum of H products is off by about sqrt(H) half
steps of the sum of magnitudes; twice that is allowed.  A gradient adds half a step of
bf16 (2^-8 relative) for the output and half a step for every term of the logits' gradient,
which is rounded to bf16 once, besides what the logits' own error does to a probability
(relative error of p: twice the logit's).  Steps of many rows keep their exponentials in fp16
between the passes: half a step of fp16 (2^-11 relative, or 2^-40 of the largest of 128 columns,
which is at most 1) on every probability.
"""

import math

import torch

BF16_HALF = 2.0 ** -8
FP16_HALF = 2.0 ** -11
FP32_HALF = 2.0 ** -24


def make_inputs(rows, hidden, vocab, seed, device, scale=2.0):
    g = torch.Generator().manual_seed(seed)
    h = torch.randn(rows, hidden, generator=g)
    w = torch.randn(vocab, hidden, generator=g) * (scale / math.sqrt(hidden))
    lean = torch.randint(0, vocab, (rows,), generator=g)
    h = h + torch.rand(rows, 1, generator=g) * w[lean]
    return h.bfloat16().to(device), w.bfloat16().to(device), lean.to(device), g


def _logit_error(h, w):
    mag = (h.abs() @ w.abs().t()).amax(1)
    return 2 * math.sqrt(h.shape[1]) * FP32_HALF * mag


def _products(dl, dl_err, h, w, rows, count):
    """dh, dW with their bounds, rows scattered back to ``count``."""
    dh = torch.zeros(count, h.shape[1], dtype=torch.float64, device=h.device)
    dh_tol = torch.zeros_like(dh)
    step = dl.abs() * BF16_HALF + dl_err
    part = dl @ w
    dh[rows] = part
    # 2^-133: the last place of a bf16 denormal; sums in fp32 add sqrt(terms) of its half steps
    tiny = 2.0 ** -133
    dh_tol[rows] = part.abs() * BF16_HALF + step @ w.abs() + tiny
    dw = dl.t() @ h
    dw_tol = dw.abs() * BF16_HALF + step.t() @ h.abs() + tiny
    return dh, dh_tol, dw, dw_tol


def cross_entropy(h, weight, targets, g, ignore_index=-100, smoothing=0.0, z_loss=0.0):
    """(loss, tol, dh, tol, dW, tol) in 64 bits."""
    rows = torch.nonzero(targets != ignore_index)[:, 0]
    hd, w, t, gd = h.detach().double()[rows], weight.detach().double(), targets[rows].long(), g.double()[rows]
    l = hd @ w.t()
    err = _logit_error(hd, w) if len(rows) else l.new_zeros(0)
    lse = l.logsumexp(1)
    at = torch.arange(len(rows), device=h.device)
    part = lse - (1 - smoothing) * l[at, t] - smoothing * l.mean(1) + z_loss * lse ** 2
    tol = (2 + 2 * z_loss * lse.abs()) * err + 8 * FP32_HALF * (part.abs() + 1)
    p = (l - lse[:, None]).exp()
    a = 1 + 2 * z_loss * lse
    dl = a[:, None] * p - smoothing / weight.shape[0]
    dl[at, t] -= 1 - smoothing
    dl_err = (a[:, None] * p) * (2 * err + 2.0 ** -19 + FP16_HALF)[:, None] + 4 * FP32_HALF * smoothing
    dl_err = dl_err + a[:, None] * 2.0 ** -40 * p.amax(1, keepdim=True) if p.numel() else dl_err
    dl, dl_err = dl * gd[:, None], dl_err * gd.abs()[:, None]
    loss = torch.zeros(h.shape[0], dtype=torch.float64, device=h.device)
    loss_tol = torch.zeros_like(loss)
    loss[rows], loss_tol[rows] = part, tol
    return (loss, loss_tol, *_products(dl, dl_err, hd, w, rows, h.shape[0]))


def topk_divergence(h, weight, ids, teacher, g, inv_temp=None, teacher_lse=None):
    """(loss, tol, dh, tol, dW, tol) in 64 bits; a dense teacher over all columns, one row at a time."""
    vocab = weight.shape[0]
    w = weight.detach().double()
    loss = torch.zeros(h.shape[0], dtype=torch.float64, device=h.device)
    loss_tol = torch.zeros_like(loss)
    rows, dls, errs = [], [], []
    ids_host, teacher_host = ids.cpu(), teacher.double().cpu()
    for r in range(h.shape[0]):
        z = {}
        it = 1.0 if inv_temp is None else float(inv_temp[r])
        for c, x in zip(ids_host[r].tolist(), teacher_host[r].tolist()):
            if 0 <= c < vocab and x != -math.inf:
                z.setdefault(c, []).append(x * it)
        if not z:
            continue
        flat = [x for v in z.values() for x in v]
        top = max(flat)
        norm = top + math.log(sum(math.exp(x - top) for x in flat)) if teacher_lse is None else float(teacher_lse[r])
        p = torch.zeros(vocab, dtype=torch.float64, device=h.device)
        cols = torch.tensor(list(z), device=h.device)
        p[cols] = torch.tensor([sum(math.exp(x - norm) for x in v) for v in z.values()], dtype=torch.float64,
                               device=h.device)
        hr = h[r:r + 1].detach().double()
        l = (hr @ w.t())[0]
        err = float(_logit_error(hr, w)[0]) * it
        log_q = (l * it).log_softmax(0)
        q = log_q.exp()
        on = p > 0
        value = float((p[on] * (p[on].log() - log_q[on])).sum())
        d = q - p
        listed = torch.zeros(vocab, dtype=torch.bool, device=h.device)
        listed[cols] = True
        size = float((p[on] * (p[on].log().abs() + log_q[on].abs())).sum())
        ratio = 0.0
        if teacher_lse is not None and not bool(listed.all()):
            rest_p = max(0.0, 1.0 - float(p.sum()))
            rest_q = float(q[~listed].sum())
            if rest_p > 0:
                value += rest_p * math.log(rest_p / rest_q)
                size += rest_p * (abs(math.log(rest_p)) + abs(math.log(rest_q)))
                ratio = rest_p / rest_q
                d = torch.where(listed, d, q * (1 - ratio))
        loss[r] = value
        loss_tol[r] = 2 * err + 16 * FP32_HALF * (size + 1)
        rows.append(r)
        dls.append(d * it * float(g[r]))
        off = (1 + ratio) * (q * (4 * err + 2.0 ** -18 + FP16_HALF) + 2.0 ** -40 * q.max())
        errs.append((off + p * 4 * FP32_HALF) * it * abs(float(g[r])))
    if not rows:
        zero = torch.zeros(h.shape, dtype=torch.float64, device=h.device)
        return loss, loss_tol, zero, zero, torch.zeros_like(w), torch.zeros_like(w)
    at = torch.tensor(rows, device=h.device)
    return (loss, loss_tol, *_products(torch.stack(dls), torch.stack(errs), h.detach().double()[at], w, at, h.shape[0]))


def within(got, want, tol, what):
    assert got.shape == want.shape, what
    off = (got.double() - want).abs()
    bad = ~(off <= tol)
    assert not bool(bad.any()), (what, int(bad.sum()), float((off - tol).nan_to_num(1e30).max()),
                                 float(off.nan_to_num(1e30).max()))
