"""Cases of the vocabulary-head training operators: cross entropy, distillation from a
teacher's top logits, and the top logits themselves, with their plain forms.

Sizes: 512 / 2048 wide heads over 2048 columns are the small decoders of the tests; the
large ones are the head shapes of the package's presets (hidden 896 / 1536 / 2048 / 3584,
vocabularies of 151936 / 152064 / 157184 columns).
"""

import math

import torch

own = False

DEV = "cuda"


def listed():
    return [
        # one step of a small head on a handful of tokens: launch latency
        {"name": "ce_small_step", "op": "ce", "rows": 33, "hidden": 512, "vocab": 2048, "ignored": 5, "smooth": 0.0,
         "z": 0.0, "grad": "both"},
        # scoring the next token of a decode batch, no gradient: the head is read once
        {"name": "ce_score_batch", "op": "ce", "rows": 64, "hidden": 3584, "vocab": 152064, "ignored": 0,
         "smooth": 0.0, "z": 0.0, "grad": "none"},
        # a policy step over padded completions of a mid-size model, tied head trained
        {"name": "ce_train_padded", "op": "ce", "rows": 2048, "hidden": 1536, "vocab": 151936, "ignored": 700,
         "smooth": 0.0, "z": 0.0, "grad": "both"},
        # adapters below a frozen diffusion head, odd row count, smoothed targets
        {"name": "ce_frozen_head_odd", "op": "ce", "rows": 1021, "hidden": 2048, "vocab": 157184, "ignored": 0,
         "smooth": 0.1, "z": 0.0, "grad": "h"},
        # full training step of the largest head, with the log-normaliser penalty
        {"name": "ce_train_large", "op": "ce", "rows": 4096, "hidden": 3584, "vocab": 152064, "ignored": 512,
         "smooth": 0.0, "z": 1e-4, "grad": "both"},
        # a small draft head against eight teacher logits a row
        {"name": "topk_small_step", "op": "topk", "rows": 48, "hidden": 512, "vocab": 2048, "k": 8, "rest": False,
         "temp": False, "empty": 3, "grad": "both"},
        # the online learner's rows (64 chains, three draft positions) on a frozen head, with the rest bucket
        {"name": "topk_draft_learner", "op": "topk", "rows": 192, "hidden": 3584, "vocab": 152064, "k": 64,
         "rest": True, "temp": True, "empty": 17, "grad": "h"},
        # offline distillation of a trained head from a cached teacher
        {"name": "topk_train", "op": "topk", "rows": 4096, "hidden": 1536, "vocab": 151936, "k": 128, "rest": True,
         "temp": False, "empty": 300, "grad": "both"},
        # top logits of one speculative block
        {"name": "top_block", "op": "top", "rows": 4, "vocab": 152064, "k": 16, "dtype": "float32", "temp": True,
         "pad": 0},
        # top logits of a decode batch of a small model
        {"name": "top_small", "op": "top", "rows": 48, "vocab": 2048, "k": 8, "dtype": "float32", "temp": False,
         "pad": 0},
        # filling a teacher cache
        {"name": "top_cache_fill", "op": "top", "rows": 2048, "vocab": 152064, "k": 64, "dtype": "float32",
         "temp": True, "pad": 0},
        # bf16 logits, odd columns, rows that start at any address; bf16 logits have many ties
        {"name": "top_bf16_odd", "op": "top", "rows": 1021, "vocab": 151937, "k": 256, "dtype": "bfloat16",
         "temp": False, "pad": 6},
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["ce", "ce", "topk", "topk", "top"])
    rows = _log_uniform(rng, 1, 4096)
    vocab = _log_uniform(rng, 500, 152064)
    if op == "top":
        return {"op": op, "rows": rows, "vocab": vocab, "k": _log_uniform(rng, 1, 256),
                "dtype": rng.choice(["float32", "bfloat16"]), "temp": rng.random() < 0.5,
                "pad": rng.choice([0, 0, 1, 5, 8])}
    case = {"op": op, "rows": rows, "hidden": 8 * _log_uniform(rng, 8, 448), "vocab": vocab,
            "grad": rng.choice(["both", "both", "h", "none"])}
    if op == "ce":
        case.update(ignored=int(rows * rng.choice([0.0, 0.0, 0.2, 0.6])), smooth=rng.choice([0.0, 0.0, 0.1]),
                    z=rng.choice([0.0, 1e-4]))
    else:
        case.update(k=_log_uniform(rng, 1, 256), rest=rng.random() < 0.5, temp=rng.random() < 0.5,
                    empty=int(rows * rng.choice([0.0, 0.0, 0.2])))
    return case


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed) * 7919 + 11)
    randn = lambda *s: torch.randn(*s, device=DEV, generator=g)  # noqa: E731
    rows, vocab = case["rows"], case["vocab"]
    state = {"op": case["op"], "case": dict(case)}
    if case["op"] == "top":
        dtype = getattr(torch, case["dtype"])
        wide = vocab + case["pad"]
        logits = (3.0 * randn(rows, wide)).to(dtype)
        state["logits"] = logits[:, case["pad"] // 2:case["pad"] // 2 + vocab]
        state["inv_temp"] = 0.5 + torch.rand(rows, device=DEV, generator=g) if case["temp"] else None
        return state
    hidden = case["hidden"]
    # a normalised hidden row leans towards the head's row of the token that follows it
    weight = (randn(vocab, hidden) * (2.0 / math.sqrt(hidden))).bfloat16()
    token = torch.randint(0, vocab, (rows,), device=DEV, generator=g)
    h = randn(rows, hidden) + 1.5 * torch.rand(rows, 1, device=DEV, generator=g) * weight[token].float()
    order = torch.randperm(rows, device=DEV, generator=g)
    if case["op"] == "ce":
        token[order[: case["ignored"]]] = -100
        state["targets"] = token
    else:
        k = min(case["k"], vocab)
        # a teacher that a young student is still far from; only its best k logits were kept, fewer in sure rows
        seen = (h + 0.75 * randn(rows, hidden)).bfloat16()
        full = (seen @ weight.t()).float()
        inv_temp = 0.5 + torch.rand(rows, device=DEV, generator=g) if case["temp"] else None
        z = full if inv_temp is None else full * inv_temp[:, None]
        state["teacher_lse"] = z.logsumexp(1) if case["rest"] else None
        del z
        state["teacher"], ids = full.topk(k, dim=1)
        del full
        kept = torch.randint((k + 1) // 2, k + 1, (rows,), device=DEV, generator=g)
        kept[order[: case["empty"]]] = 0
        state["ids"] = torch.where(torch.arange(k, device=DEV)[None] < kept[:, None], ids, -1).to(torch.int32)
        state["inv_temp"] = inv_temp
    grad = case["grad"]
    state["h"] = h.bfloat16().requires_grad_(grad != "none")
    state["weight"] = weight.requires_grad_(grad == "both")
    # what the mean over the rows that count and a per-row weight hand back
    state["g"] = (0.5 + torch.rand(rows, device=DEV, generator=g)) / rows
    return state


def _plain_lse(z):
    m = z.amax(1)
    return m + (z - m[:, None]).exp().sum(1).log()


def _plain_products(state, logits_grad):
    """Gradients of the two factors of logits = h @ weight.T, rounded once."""
    out = []
    if state["h"].requires_grad:
        out.append((logits_grad @ state["weight"].detach().float()).to(state["h"].dtype))
    if state["weight"].requires_grad:
        out.append((logits_grad.t() @ state["h"].detach().float()).to(state["weight"].dtype))
    return out


def _plain_ce(state):
    smooth, z = state["case"]["smooth"], state["case"]["z"]
    targets = state["targets"]
    logits = state["h"].detach().float() @ state["weight"].detach().float().t()
    vocab = logits.shape[1]
    counts = targets != -100
    at = torch.where(counts, targets, 0)[:, None]
    lse = _plain_lse(logits)
    loss = lse - (1 - smooth) * logits.gather(1, at)[:, 0] + z * lse * lse
    if smooth:
        loss = loss - smooth * logits.mean(1)
    loss = torch.where(counts, loss, 0.0)
    if not state["h"].requires_grad:
        return [loss]
    dl = (logits - lse[:, None]).exp() * (1 + 2 * z * lse)[:, None] - smooth / vocab
    del logits
    dl.scatter_add_(1, at, torch.full_like(dl[:, :1], smooth - 1))
    dl = torch.where(counts[:, None], dl * state["g"][:, None], 0.0)
    return [loss] + _plain_products(state, dl)


def _plain_topk(state):
    logits = state["h"].detach().float() @ state["weight"].detach().float().t()
    it = state["inv_temp"]
    it = torch.ones_like(logits[:, 0]) if it is None else it
    valid = state["ids"] >= 0
    at = torch.where(valid, state["ids"], 0).long()
    some = valid.any(1)
    logits = logits * it[:, None]
    # a divergence is a small difference of log-probabilities: normalisers and listed terms in 64 bits
    lse = _plain_lse(logits.double())
    t = torch.where(valid, state["teacher"].double() * it[:, None].double(), -math.inf)
    if state["teacher_lse"] is None:
        top = torch.where(some, t.amax(1), 0.0)
        norm = top + (t - top[:, None]).exp().sum(1).log()
        p_rest = torch.zeros_like(norm)
    else:
        norm = state["teacher_lse"].double()
        p_rest = torch.where(some, (1 - (t - norm[:, None]).exp().sum(1)).clamp_min(0), 0.0)
    log_p = t - torch.where(some, norm, 0.0)[:, None]
    p = log_p.exp()
    log_q = logits.gather(1, at).double() - lse[:, None]
    loss = torch.where(valid, p * (log_p - log_q), 0.0).sum(1)
    listed_logit = torch.where(valid, logits.gather(1, at), -math.inf)
    rest = logits.clone()
    rest.scatter_(1, torch.where(valid, at, at[:, :1]), -math.inf)
    log_q_rest = _plain_lse(rest.double()) - lse
    del rest
    tail = p_rest > 0
    loss = loss + torch.where(tail, p_rest * (torch.where(tail, p_rest, 1.0).log() - log_q_rest), 0.0)
    loss = torch.where(some, loss, 0.0).float()
    if not state["h"].requires_grad:
        return [loss]
    scale = torch.where(some, state["g"] * it, 0.0)
    rest_factor = torch.where(tail, 1 - p_rest * (-log_q_rest).exp(), 1.0).float()
    q = (logits - lse.float()[:, None]).exp()
    del logits
    on = torch.where(valid, ((listed_logit - lse[:, None]).exp() - p).float(), 0.0)
    q = q * rest_factor[:, None]
    # listed columns are replaced (they are distinct); an empty slot names the row's first column, added as it stands
    q.scatter_(1, torch.where(valid, at, at[:, :1]), 0.0)
    q.scatter_add_(1, at, on)
    return [loss] + _plain_products(state, torch.where(some[:, None], q * scale[:, None], 0.0))


def _plain_top(state):
    x = state["logits"].float()
    values, ids = torch.sort(x, dim=1, descending=True, stable=True)
    k = min(state["case"]["k"], x.shape[1])
    z = x if state["inv_temp"] is None else x * state["inv_temp"][:, None]
    return [values[:, :k].clone(), ids[:, :k].to(torch.int32), _plain_lse(z)]


def run(state):
    case = state["case"]
    if not own:
        return {"ce": _plain_ce, "topk": _plain_topk, "top": _plain_top}[state["op"]](state)
    from online_speculation_b200.ops import kernels as K

    if state["op"] == "top":
        return list(K.top_logits(state["logits"], min(case["k"], case["vocab"]), inv_temp=state["inv_temp"]))
    if state["op"] == "ce":
        loss = K.head_cross_entropy(state["h"], state["weight"], state["targets"], ignore_index=-100,
                                    label_smoothing=case["smooth"], z_loss=case["z"])
    else:
        loss = K.head_topk_divergence(state["h"], state["weight"], state["ids"], state["teacher"],
                                      inv_temp=state["inv_temp"], teacher_lse=state["teacher_lse"])
    leaves = [t for t in (state["h"], state["weight"]) if t.requires_grad]
    if not leaves:
        return [loss]
    return [loss.detach(), *torch.autograd.grad(loss, leaves, state["g"])]


def work(case):
    rows, vocab = case["rows"], case["vocab"]
    if case["op"] == "top":
        size = 4 if case["dtype"] == "float32" else 2
        return {"bytes": rows * (vocab * size + 8 * min(case["k"], vocab) + 4 + 4 * case["temp"]),
                "flops": 4 * rows * vocab}
    hidden, grad = case["hidden"], case["grad"]
    live = rows - case.get("ignored", 0) - case.get("empty", 0)
    products = {"none": 1, "h": 2, "both": 3}[grad]
    size = 2 * hidden * (live + vocab) + 4 * rows
    if grad != "none":
        size += 2 * hidden * rows + 4 * rows
    if grad == "both":
        size += 2 * hidden * vocab
    size += 8 * rows if case["op"] == "ce" else 8 * rows * min(case["k"], vocab)
    return {"bytes": size, "flops": 2 * products * live * hidden * vocab}


def exact(case, seed):
    """The definitions in 64 bits."""
    s = prepare(case, seed)
    if case["op"] == "top":
        x = s["logits"].double()
        z = x if s["inv_temp"] is None else x * s["inv_temp"].double()[:, None]
        k = min(case["k"], case["vocab"])
        return [x.float().sort(1, descending=True).values[:, :k].double(), None, z.logsumexp(1)]
    h, w = s["h"].detach().double(), s["weight"].detach().double()
    logits = h @ w.t()
    g = s["g"].double()
    if case["op"] == "ce":
        live = s["targets"] >= 0
        rows = torch.nonzero(live)[:, 0]
        logits, t, g = logits[rows], s["targets"][rows], g[rows]
        log_p = logits.log_softmax(1)
        lse = logits[:, 0] - log_p[:, 0]
        hot = -log_p[torch.arange(len(rows), device=DEV), t]
        part = (1 - case["smooth"]) * hot - case["smooth"] * log_p.mean(1) + case["z"] * lse.square()
        want = (1 - case["smooth"]) * torch.nn.functional.one_hot(t, case["vocab"]) if len(rows) else log_p
        dl = log_p.exp().mul_((1 + 2 * case["z"] * lse)[:, None]).sub_(want).sub_(case["smooth"] / case["vocab"])
        del want, log_p
    else:
        live = (s["ids"] >= 0).any(1)
        rows = torch.nonzero(live)[:, 0]
        logits, ids, g = logits[rows], s["ids"][rows].long(), g[rows]
        it = torch.ones_like(g) if s["inv_temp"] is None else s["inv_temp"].double()[rows]
        log_q = (logits * it[:, None]).log_softmax(1)
        slot = ids >= 0
        t = (s["teacher"].double()[rows] * it[:, None]).masked_fill(~slot, -math.inf)
        log_p = t - (t.logsumexp(1) if s["teacher_lse"] is None else s["teacher_lse"].double()[rows])[:, None]
        # the teacher over all columns, empty slots in a spare one behind the last
        spot = ids.masked_fill(~slot, case["vocab"])
        p = torch.zeros(len(rows), case["vocab"] + 1, dtype=torch.float64, device=DEV)
        p.scatter_(1, spot, log_p.exp())
        on = torch.zeros(len(rows), case["vocab"] + 1, dtype=torch.bool, device=DEV)
        on.scatter_(1, spot, True)
        p, on = p[:, :-1], on[:, :-1]
        part = torch.where(p > 0, p * (p.log() - log_q), 0.0).sum(1)
        q = log_q.exp()
        dl = q - p
        if s["teacher_lse"] is not None:
            rest_p = (1 - p.sum(1)).clamp_min(0)
            rest_q = q.masked_fill(on, 0.0).sum(1)
            has = rest_p > 0
            part = part + torch.where(has, rest_p * (torch.where(has, rest_p, 1.0) / rest_q).log(), 0.0)
            ratio = torch.where(has, rest_p / rest_q, 0.0)
            dl = dl - (~on) * q * ratio[:, None]
        dl.mul_(it[:, None])
        del p, on, q, log_q
    loss = torch.zeros(case["rows"], dtype=torch.float64, device=DEV)
    loss[rows] = part
    out = [loss]
    if case["grad"] != "none":
        dl.mul_(g[:, None])
        dh = torch.zeros_like(h)
        dh[rows] = dl @ w
        out.append(dh)
    if case["grad"] == "both":
        out.append(dl.t() @ h[rows])
    return out
