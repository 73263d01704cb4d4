"""Losses on a vocabulary head without a matrix of its logits, and a teacher's top logits.

* :func:`head_cross_entropy`: softmax cross entropy of ``h @ weight.T``, with label
  smoothing and a penalty on the log-normaliser;
* :func:`head_topk_divergence`: KL divergence of the head's distribution from a teacher of
  which only the best logits were kept;
* :func:`top_logits`: those best logits, their columns and the log-normaliser.

CUDA tensors run the kernels of ``csrc/head_loss.cu`` and ``csrc/top_logits.cu``; CPU tensors
run the fp32 oracles below, which the kernel tests compare against.  Both losses return one
value per row, so the caller weighs rows as it likes; both are differentiable in ``h`` and
``weight`` (once), never in the teacher.
"""

from __future__ import annotations

import math

import torch

from . import _ext, workspace

MAX_LISTED = 512          # csrc/head_loss.h kHeadMaxListed, csrc/top_logits.h kTopLogitsMax
PIECE_COLUMNS = 256       # granularity of the backward pass's vocabulary pieces


def _check_head(h, weight, piece):
    for name, t in (("h", h), ("weight", weight)):
        if t.dim() != 2:
            raise ValueError(f"{name} must be 2-D")
        if t.dtype != torch.bfloat16:
            raise TypeError(f"{name} must be bfloat16, got {t.dtype}")
    if h.shape[1] != weight.shape[1]:
        raise ValueError(f"h rows are {h.shape[1]} wide, the head's {weight.shape[1]}")
    if h.shape[1] == 0 or h.shape[1] % 8:
        raise ValueError("the hidden width must be a positive multiple of 8")
    if weight.shape[0] == 0:
        raise ValueError("the vocabulary is empty")
    if h.device != weight.device:
        raise ValueError(f"h is on {h.device}, weight on {weight.device}")
    if piece is not None and (piece <= 0 or piece % PIECE_COLUMNS):
        raise ValueError(f"piece must be a positive multiple of {PIECE_COLUMNS} columns")


def _check_rows(name, t, shape, dtypes, device):
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} must be one of {[str(d) for d in dtypes]}, got {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")


_INDEX = (torch.int32, torch.int64)


def _head_loss(h, weight, ids, teacher, teacher_lse, inv_temp, ignore_index, smoothing, z_loss, piece):
    """The extension's autograd node.  Forward: row lists, compaction, the statistics GEMM, the row losses.
    Backward: per vocabulary piece the gradient of its logits and the two products with it."""
    return _ext.require().head_loss(h, weight, ids, teacher, teacher_lse, inv_temp, ignore_index, smoothing, z_loss,
                                    piece or 0, workspace.status(h.device))


def head_cross_entropy(h: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, *, ignore_index: int = -100,
                       label_smoothing: float = 0.0, z_loss: float = 0.0, piece: int | None = None) -> torch.Tensor:
    """Cross entropy of ``softmax(h @ weight.T)`` per row (fp32 [R]).

    With l = h W^T, e = ``label_smoothing`` and z = ``z_loss``::

        loss = lse(l) - (1 - e) l[target] - e mean(l) + z lse(l)^2

    ``h`` [R, H] and ``weight`` [V, H] are bf16 with H a multiple of 8; ``targets`` [R] int32 or
    int64.  A row whose target is ``ignore_index`` gives 0 and takes no part in any product: its
    hidden row may hold anything.  A target outside the vocabulary raises on the CPU; on the GPU
    its row is ignored and ``workspace.check_status`` reports it.  Gradients are bf16, summed in
    fp32.

    Between the passes a step keeps its hidden rows and 2 bytes a logit (up to 2 GB; rows in whole 256; H at least
    384) or, of at most 128 (and H) rows on 32768 columns or more, 4 bytes (up to 256 MB); larger ones, and
    all others, keep no logits and compute them twice.  ``piece`` (a multiple of 256) bounds the memory: no logits
    are kept, and the backward pass works on that many vocabulary columns at a time with ``2 R piece`` bytes
    of scratch (twice that up to 128 rows; 256 MB without it), next to 4 bytes an entry of ``h`` for each part
    of its gradient.

    A training step that is captured into a CUDA graph takes its gradients with
    ``torch.autograd.grad``; no eager graph of the same leaves may be alive meanwhile.
    """
    _check_head(h, weight, piece)
    _check_rows("targets", targets, h.shape[:1], _INDEX, h.device)
    if not 0.0 <= label_smoothing <= 1.0:
        raise ValueError("label_smoothing must be between 0 and 1")
    if not (z_loss >= 0.0 and math.isfinite(z_loss)):
        raise ValueError("z_loss must be finite and not negative")
    if h.shape[0] == 0:
        return _empty_loss(h, weight)
    if h.is_cuda:
        return _head_loss(h, weight, targets.contiguous(), None, None, None, int(ignore_index),
                          float(label_smoothing), float(z_loss), piece)
    return _cross_entropy_reference(h, weight, targets, ignore_index, label_smoothing, z_loss)


def head_topk_divergence(h: torch.Tensor, weight: torch.Tensor, ids: torch.Tensor, teacher: torch.Tensor, *,
                         inv_temp: torch.Tensor | None = None, teacher_lse: torch.Tensor | None = None,
                         piece: int | None = None) -> torch.Tensor:
    """KL(teacher || softmax(inv_temp * h @ weight.T)) per row (fp32 [R]).

    ``ids`` [R, K] (int32 or int64) and ``teacher`` [R, K] (fp32 or bf16 logits) list the teacher's
    best columns of every row, in any order, K at most 512; a slot with a negative id or a logit
    of -inf is empty, a column listed twice counts once with its masses added.  ``inv_temp`` [R]
    fp32 (positive) scales the logits of both sides.

    Without ``teacher_lse`` the teacher is the softmax of its listed logits.  With it (fp32 [R], the
    logsumexp of all of the teacher's scaled logits, as :func:`top_logits` returns it) the listed
    columns keep their true masses and all others together are one more outcome on both sides
    (where the list holds every column there is none).  Masses are taken as they are: those of a teacher
    whose logits were rounded sum to a little more or less than 1, and the gradient is that of the loss
    with them.

    A row without a listed column gives 0 and takes no part in any product.  A column beyond the
    vocabulary raises on the CPU; on the GPU its slot is empty and ``workspace.check_status``
    reports it.  ``h``, ``weight``, ``piece`` and the gradients are as in :func:`head_cross_entropy`.
    """
    _check_head(h, weight, piece)
    if ids.dim() != 2 or not 1 <= ids.shape[1] <= MAX_LISTED:
        raise ValueError(f"ids must be [rows, K] with K between 1 and {MAX_LISTED}")
    _check_rows("ids", ids, (h.shape[0], ids.shape[1]), _INDEX, h.device)
    _check_rows("teacher", teacher, ids.shape, (torch.float32, torch.bfloat16), h.device)
    for name, t in (("inv_temp", inv_temp), ("teacher_lse", teacher_lse)):
        if t is not None:
            _check_rows(name, t, h.shape[:1], (torch.float32,), h.device)
    if h.shape[0] == 0:
        return _empty_loss(h, weight)
    teacher = teacher.detach()
    if h.is_cuda:
        return _head_loss(h, weight, ids.contiguous(), teacher.contiguous(),
                          None if teacher_lse is None else teacher_lse.detach().contiguous(),
                          None if inv_temp is None else inv_temp.detach().contiguous(), 0, 0.0, 0.0, piece)
    return _topk_divergence_reference(h, weight, ids, teacher, inv_temp, teacher_lse)


def top_logits(logits: torch.Tensor, k: int, *, inv_temp: torch.Tensor | None = None):
    """The ``k`` largest logits of every row: (values fp32 [R, k], columns int32 [R, k], lse fp32 [R]).

    Descending; equal logits in the order of their columns, NaN above everything.  ``lse`` is the
    logsumexp of ``inv_temp * logits`` over the whole row (``inv_temp`` [R] fp32, positive; None: 1).
    ``logits`` [R, V] fp32 or bf16 with any row stride; k at most 512.  What
    :func:`head_topk_divergence` needs of a teacher.
    """
    if logits.dim() != 2:
        raise ValueError("logits must be 2-D")
    if logits.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"logits must be float32 or bfloat16, got {logits.dtype}")
    rows, vocab = logits.shape
    if not 1 <= k <= min(vocab, MAX_LISTED):
        raise ValueError(f"k must be between 1 and min(columns, {MAX_LISTED}), got {k} of {vocab}")
    if inv_temp is not None:
        _check_rows("inv_temp", inv_temp, (rows,), (torch.float32,), logits.device)
    logits = logits.detach()
    if rows == 0:
        return (logits.new_empty(0, k, dtype=torch.float32), logits.new_empty(0, k, dtype=torch.int32),
                logits.new_empty(0, dtype=torch.float32))
    if logits.is_cuda:
        return _ext.require().top_logits(logits if logits.stride(1) == 1 else logits.contiguous(), int(k),
                                         None if inv_temp is None else inv_temp.detach().contiguous())
    x = logits.float()
    # NaN first, then descending, equal ones by column (-0 equals 0)
    order = torch.sort(torch.where(x.isnan(), math.inf, x), dim=1, descending=True, stable=True).indices
    order = order.gather(1, torch.sort((~x.isnan()).int().gather(1, order), dim=1, stable=True).indices)[:, :k]
    z = x if inv_temp is None else x * inv_temp[:, None]
    return x.gather(1, order), order.to(torch.int32), z.logsumexp(1)


# ----------------------------------------------------------------- oracles --
def _empty_loss(h, weight):
    """No rows: an empty loss that still reaches its inputs, and reads none of the head."""
    return h.float().sum(1) + weight[:0].float().sum()


def _scatter_rows(rows, values, count):
    return torch.zeros(count, dtype=torch.float32, device=values.device).index_copy(0, rows, values)


def _cross_entropy_reference(h, weight, targets, ignore_index, smoothing, z_loss):
    rows = torch.nonzero(targets != ignore_index)[:, 0]
    t = targets[rows].long()
    if bool(((t < 0) | (t >= weight.shape[0])).any()):
        raise IndexError("a target is outside the vocabulary")
    logits = h[rows].float() @ weight.float().t()
    lse = logits.logsumexp(1)
    loss = lse - (1 - smoothing) * logits.gather(1, t[:, None])[:, 0] + z_loss * lse.square()
    if smoothing:
        loss = loss - smoothing * logits.mean(1)
    return _scatter_rows(rows, loss, h.shape[0])


def _topk_divergence_reference(h, weight, ids, teacher, inv_temp, teacher_lse):
    vocab = weight.shape[0]
    if bool((ids >= vocab).any()):
        raise IndexError("a listed column is outside the vocabulary")
    slot = (ids >= 0) & (teacher != -math.inf)
    rows = torch.nonzero(slot.any(1))[:, 0]
    slot, at = slot[rows], ids[rows].long()
    it = torch.ones(len(rows)) if inv_temp is None else inv_temp.detach()[rows]
    z = (teacher[rows].double() * it.double()[:, None]).masked_fill(~slot, -math.inf)
    norm = z.logsumexp(1) if teacher_lse is None else teacher_lse.detach()[rows].double()
    # dense masses; empty slots go to a spare column
    spot = at.masked_fill(~slot, vocab)
    p = torch.zeros(len(rows), vocab + 1, dtype=torch.float64).scatter_add_(1, spot, (z - norm[:, None]).exp())[:, :-1]
    listed = torch.zeros(len(rows), vocab + 1, dtype=torch.bool).scatter_(1, spot, True)[:, :-1]
    log_q = ((h[rows].float() @ weight.float().t()) * it[:, None]).double().log_softmax(1)
    loss = torch.where(p != 0, p * (torch.where(p != 0, p, 1.0).log() - log_q), 0.0).sum(1)
    if teacher_lse is not None:
        rest = torch.where(p.sum(1).isnan(), math.nan, (1 - p.sum(1)).clamp_min(0))
        rest = torch.where(listed.all(1), 0.0, rest)
        log_rest = log_q.masked_fill(listed, -math.inf)
        log_rest = torch.where(listed.all(1)[:, None], log_q, log_rest).logsumexp(1)
        loss = loss + torch.where(rest != 0, rest * (torch.where(rest != 0, rest, 1.0).log() - log_rest), 0.0)
    return _scatter_rows(rows, loss.float(), h.shape[0])
