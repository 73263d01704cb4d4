"""How far the vocabulary-head losses' gradients and losses are from 64 bits, as a norm: what the kernels add to lose no more
than the rounding of their outputs.

Rounding to bf16 is off by at most half a step; its error is spread evenly over a step of 2^-7 of the binade, so the relative
norm of the error is 2^-7 / sqrt(12 mean(m^2)) with m in [1, 2) the significands: 0.00148 where they are spread evenly
(mean 7/3), 0.00166 where low ones are as frequent as in a density 1/m^3 (mean 1.85).  One rounding is therefore below
0.0017, and two independent ones (of the logits' gradient, then of the output) are above 0.0021.  The bound is between.
"""

import pytest
import torch

import head_loss_masses as masses
import head_loss_oracle as oracle
from online_speculation_b200.ops import kernels as K

pytestmark = pytest.mark.gpu

ONE_ROUNDING = 0.0019


def _off(got, want):
    return float((got.double() - want).norm() / want.norm())


# logits computed again and kept; up to 128 rows (two bf16 halves), more
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


@pytest.mark.parametrize("rows,hidden", [(64, 3584), (64, 8192), (70, 2048), (128, 3584), (129, 3584), (192, 1536),
                                         (256, 3584), (300, 3584), (300, 1536), (300, 896), (300, 2048), (513, 4096)])
@pytest.mark.parametrize("listed", [0, 8])
@pytest.mark.parametrize("kept", [False, True])
def test_losses_are_summed_in_parts(cuda, rows, hidden, listed, kept):
    """No more than twice as far from 64 bits as losses of fp32 products.  The tensor core truncates at every addition, so a
    sum loses in proportion to its length: in one sum the losses of these widths were three to six times as far, in parts
    of at most 14 blocks of 64 they are a quarter to a half of that."""
    vocab = 20000
    h, w, t, gen = oracle.make_inputs(rows, hidden, vocab, 5, cuda)
    seen = (h + 0.75 * torch.randn(rows, hidden, generator=gen).to(cuda)).bfloat16()
    teacher, ids, lse = K.top_logits((seen @ w.t()).float(), max(listed, 1))
    fp32 = (h.float() @ w.float().t()).double()
    one = torch.ones(rows, device=cuda)
    h.requires_grad_(kept)
    if listed:
        want = masses.divergence(h, w, ids, teacher, one, None, lse)[0]
        plain = masses.losses_of_logits(fp32, ids, teacher, None, lse)[0]
        got = K.head_topk_divergence(h, w, ids, teacher, teacher_lse=lse)
    else:
        want = oracle.cross_entropy(h, w, t, one)[0]
        plain = fp32.logsumexp(1) - fp32.gather(1, t[:, None])[:, 0]
        got = K.head_cross_entropy(h, w, t)
    assert _off(got.detach(), want) <= 2 * _off(plain, want)
