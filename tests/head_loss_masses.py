"""64-bit definition of the divergence from listed teacher logits whose masses need not sum to one.

With p the listed masses, S their sum, q = softmax(it l) and, where a column is left out of the list,
rest = max(0, 1 - S) and r = softmax of it l over the unlisted columns::

    loss = sum p (log p - log q) + rest (log rest - log q_rest)
    d loss / d l = it ((S + rest) q - p)          on the listed columns
                   it ((S + rest) q - rest r)     on the others

S is above one where the teacher's logits were rounded (bf16) and its normaliser was not.

Bounds: as in ``head_loss_oracle``, with ``err`` the error of a scaled logit.  q and r are off by twice that relative
(a logit and a normaliser) and by 2^-18 for the exponential; kept in fp16 by half its step, or 2^-40 of the
largest.  On the unlisted columns the two terms are formed as r (q_rest (S + rest) - rest).
"""

import math

import torch

import head_loss_oracle as oracle


def losses(h, w, ids, teacher, inv_temp=None, teacher_lse=None):
    """(loss, what the gradient needs) in the type of ``h`` and ``w``, differentiable."""
    return losses_of_logits(h @ w.t(), ids, teacher, inv_temp, teacher_lse)


def losses_of_logits(logits, ids, teacher, inv_temp=None, teacher_lse=None):
    vocab = logits.shape[1]
    slot = (ids >= 0) & (teacher != -math.inf)
    it = logits.new_ones(logits.shape[0]) if inv_temp is None else inv_temp.to(logits.dtype)
    z = (teacher.to(logits.dtype) * it[:, None]).masked_fill(~slot, -math.inf)
    spot = torch.where(slot, ids.long(), vocab)
    some = slot.any(1)
    norm = torch.where(some, z.logsumexp(1), 0.0) if teacher_lse is None else teacher_lse.to(logits.dtype)
    p = logits.new_zeros(logits.shape[0], vocab + 1).scatter_add_(1, spot, (z - norm[:, None]).exp())[:, :-1]
    on = torch.zeros(p.shape[0], vocab + 1, dtype=torch.bool, device=logits.device).scatter_(1, spot, True)[:, :-1]
    total, whole = p.sum(1), on.all(1)
    rest = torch.where(whole | ~some, 0.0, (1 - total).clamp_min(0)) if teacher_lse is not None else torch.zeros_like(total)
    log_q = (logits * it[:, None]).log_softmax(1)
    log_rest = log_q.masked_fill(on & ~whole[:, None], -math.inf).logsumexp(1)
    part = torch.where(p > 0, p * (torch.where(p > 0, p, 1.0).log() - log_q), 0.0).sum(1)
    part = part + torch.where(rest > 0, rest * (torch.where(rest > 0, rest, 1.0).log() - log_rest), 0.0)
    return torch.where(some, part, 0.0), (p, on, rest, log_q, log_rest, it, some)


def divergence(h, weight, ids, teacher, g, inv_temp=None, teacher_lse=None):
    """(loss, tol, dh, tol, dW, tol) in 64 bits."""
    hd, w = h.detach().double(), weight.detach().double()
    loss, (p, on, rest, log_q, log_rest, it, some) = losses(hd, w, ids, teacher, inv_temp, teacher_lse)
    q, mass = log_q.exp(), p.sum(1) + rest
    r = (log_q - log_rest[:, None]).exp().masked_fill(on, 0.0)
    d = mass[:, None] * q - torch.where(on, p, rest[:, None] * r)
    err = oracle._logit_error(hd, w) * it
    size = torch.where(p > 0, p * (torch.where(p > 0, p, 1.0).log().abs() + log_q.abs()), 0.0).sum(1)
    size = size + torch.where(rest > 0, rest * (torch.where(rest > 0, rest, 1.0).log().abs() + log_rest.abs()), 0.0)
    loss_tol = 2 * mass * err + 16 * oracle.FP32_HALF * (size + 1)
    rel = (4 * err + 2.0 ** -18 + oracle.FP16_HALF)[:, None]
    q_rest = log_rest.exp()
    lift = (mass * q_rest - rest).abs()
    off = torch.where(on, mass[:, None] * q * rel + p * 4 * oracle.FP32_HALF,
                      r * ((lift + mass * q_rest)[:, None] * rel) + (2.0 ** -40 * lift * r.amax(1))[:, None])
    scale = torch.where(some, it * g.double(), 0.0)[:, None]
    rows = torch.nonzero(some)[:, 0]
    dl, dl_err = (d * scale)[rows], (off * scale.abs())[rows]
    return (loss, torch.where(some, loss_tol, 0.0), *oracle._products(dl, dl_err, hd[rows], w, rows, h.shape[0]))


def sure_inputs(rows, hidden, vocab, k, seed, device):
    """A teacher with its mass in three columns near 20, listed and rounded to bf16 with the normaliser of the logits as
    they were, and a student that leans towards the same columns."""
    h, w, _, gen = oracle.make_inputs(rows, hidden, vocab, seed, "cpu")
    big = torch.randn(rows, vocab, generator=gen)
    best = torch.stack([torch.randperm(vocab, generator=gen)[:min(3, vocab)] for _ in range(rows)])
    big.scatter_(1, best, 20 + torch.rand(rows, best.shape[1], generator=gen))
    lse = big.double().logsumexp(1).float()
    values, ids = big.topk(k, 1)
    h = (0.2 * h.float() + 5 * w[best].float().mean(1) * torch.rand(rows, 1, generator=gen)).bfloat16()
    g = torch.randn(rows, generator=gen)
    return [x.to(device) for x in (h, w, ids, values.bfloat16(), lse, g)]
