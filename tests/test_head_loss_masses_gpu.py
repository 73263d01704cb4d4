"""The divergence from listed teacher logits whose masses sum to more, or less, than one, on the kernels."""

import pytest
import torch

import head_loss_masses as masses
import head_loss_oracle as oracle
from online_speculation_b200.ops import kernels as K
from online_speculation_b200.ops import workspace

pytestmark = pytest.mark.gpu

# logits computed again and kept, of few rows and of many; lists of one column, of several, of every one
SHAPES = [(40, 64, 3000, 1), (40, 64, 3000, 8), (150, 72, 700, 40), (30, 512, 33000, 8), (200, 512, 33000, 1),
          (300, 64, 3000, 8), (300, 512, 3000, 8), (300, 512, 3000, 1), (9, 72, 40, 40), (300, 64, 40, 40), (300, 400, 40, 40),
          (5, 8, 1, 1)]


@pytest.mark.parametrize("rows,hidden,vocab,k", SHAPES)
@pytest.mark.parametrize("temp", [False, True])
def test_rounded_teachers(cuda, rows, hidden, vocab, k, temp):
    h, w, ids, teacher, lse, g = masses.sure_inputs(rows, hidden, vocab, k, rows + k, cuda)
    it = 0.97 + 0.06 * torch.rand(rows, generator=torch.Generator().manual_seed(1)) if temp else None
    it = it if it is None else it.to(cuda)
    total = (teacher.double() - lse.double()[:, None]).exp().sum(1)
    assert k == 1 or (bool((total > 1.003).any()) and bool((total < 0.997).any()))
    want = masses.divergence(h, w, ids, teacher, g, it, lse)
    h.requires_grad_()
    w.requires_grad_()
    loss = K.head_topk_divergence(h, w, ids, teacher, inv_temp=it, teacher_lse=lse)
    got = (loss.detach(), *torch.autograd.grad(loss, [h, w], g))
    workspace.check_status(cuda)
    hc, wc = (x.detach().cpu().requires_grad_() for x in (h, w))
    there = K.head_topk_divergence(hc, wc, ids.cpu(), teacher.cpu(), inv_temp=None if it is None else it.cpu(),
                                   teacher_lse=lse.cpu())
    there = (there.detach(), *torch.autograd.grad(there, [hc, wc], g.cpu()))
    for a, b, i in zip(got, there, (0, 2, 4)):
        oracle.within(a, want[i], want[i + 1], i)
        oracle.within(a.cpu(), b.double(), 2 * want[i + 1].cpu(), ("cpu", i))


@pytest.mark.parametrize("rows,hidden,vocab,k", [(1, 8, 1, 1), (3, 72, 40, 40), (256, 64, 600, 512), (257, 64, 512, 512),
                                                 (130, 136, 777, 64), (40, 64, 3001, 512)])
def test_lifted_normalisers(cuda, rows, hidden, vocab, k):
    """bf16 teachers in no order, listed from random logits, whose normaliser was lifted by 0.01."""
    h, w, _, gen = oracle.make_inputs(rows, hidden, vocab, rows + k, cuda)
    logits = 3 * torch.randn(rows, vocab, generator=gen)
    ids = torch.stack([torch.randperm(vocab, generator=gen)[:k] for _ in range(rows)])
    teacher = logits.gather(1, ids).bfloat16().to(cuda)
    ids, lse, g = ids.to(cuda), (logits.logsumexp(1) + 0.01).to(cuda), torch.randn(rows, generator=gen).to(cuda)
    want = masses.divergence(h, w, ids, teacher, g, None, lse)
    h.requires_grad_()
    w.requires_grad_()
    loss = K.head_topk_divergence(h, w, ids, teacher, teacher_lse=lse, piece=512)
    for got, i in zip((loss.detach(), *torch.autograd.grad(loss, [h, w], g)), (0, 2, 4)):
        oracle.within(got, want[i], want[i + 1], i)
