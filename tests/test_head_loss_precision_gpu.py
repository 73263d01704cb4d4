"""How far the vocabulary-head losses' gradients and losses are from 64 bits, as a norm: what the kernels add to lose no more
than the rounding of their outputs.

Rounding to bf16 is off by at most half a step; its error is spread evenly over a step of 2^-7 of the binade, so the relative
norm of the error is 2^-7 / sqrt(12 mean(m^2)) with m in [1, 2) the significands: 0.00148 where they are spread evenly
(mean 7/3), 0.00166 where low ones are as frequent as in a density 1/m^3 (mean 1.85).  One rounding is therefore below
0.0017, and two independent ones (of the logits' gradient, then of the output) are above 0.0021.  The bound is between.
"""

import pytest
import torch

import head_loss_oracle as oracle
from online_speculation_b200.ops import kernels as K

pytestmark = pytest.mark.gpu

ONE_ROUNDING = 0.0019


def _off(got, want):
    return float((got.double() - want).norm() / want.norm())


# logits computed again and kept; up to 128 rows (two bf16 halves), 256, more
@pytest.mark.parametrize("rows,hidden,vocab", [(100, 512, 3000), (100, 512, 33000), (200, 512, 3000), (200, 512, 33000),
                                               (300, 256, 3000), (600, 512, 3000)])
def test_gradients_of_one_target_a_row(cuda, rows, hidden, vocab):
    """dh, which is mostly the target's entry of the logits' gradient; dW too up to 128 rows."""
    h, w, _, gen = oracle.make_inputs(rows, hidden, vocab, rows, cuda, scale=1.0)
    t = torch.randint(0, vocab, (rows,), generator=gen).to(cuda)
    g = torch.randn(rows, generator=gen).to(cuda)
    want = oracle.cross_entropy(h, w, t, g)
    h.requires_grad_()
    w.requires_grad_()
    dh, dw = torch.autograd.grad(K.head_cross_entropy(h, w, t), [h, w], g)
    assert _off(dh, want[2]) <= ONE_ROUNDING
    if rows <= 128:
        assert _off(dw, want[4]) <= ONE_ROUNDING


@pytest.mark.parametrize("rows,hidden,vocab,k", [(100, 512, 3000, 40), (200, 512, 33000, 30), (300, 512, 20000, 4)])
def test_gradients_of_short_lists(cuda, rows, hidden, vocab, k):
    h, w, _, gen = oracle.make_inputs(rows, hidden, vocab, rows, cuda, scale=1.0)
    ids = torch.stack([torch.randperm(vocab, generator=gen)[:k] for _ in range(rows)]).to(cuda)
    teacher = torch.randn(rows, k, generator=gen).to(cuda)
    g = torch.randn(rows, generator=gen).to(cuda)
    want = oracle.topk_divergence(h, w, ids, teacher, g)
    h.requires_grad_()
    w.requires_grad_()
    dh, dw = torch.autograd.grad(K.head_topk_divergence(h, w, ids, teacher), [h, w], g)
    assert _off(dh, want[2]) <= ONE_ROUNDING
    if rows <= 128:
        assert _off(dw, want[4]) <= ONE_ROUNDING


def test_losses_of_few_rows_sum_in_chains(cuda):
    """The tensor core truncates at every addition, so a sum in four chains loses about a quarter of what one chain does.
    The same rows, alone (four chains) and among others (one)."""
    rows, hidden, vocab = 64, 3584, 20000
    h, w, t, _ = oracle.make_inputs(192, hidden, vocab, 5, cuda)
    want = oracle.cross_entropy(h[:rows], w, t[:rows], torch.ones(rows, device=cuda))[0]
    with torch.no_grad():
        four = _off(K.head_cross_entropy(h[:rows].contiguous(), w, t[:rows]), want)
        one = _off(K.head_cross_entropy(h, w, t)[:rows], want)
    assert four <= 0.6 * one, (four, one)
