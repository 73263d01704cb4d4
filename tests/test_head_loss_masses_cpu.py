"""The divergence from listed teacher logits whose masses sum to more, or less, than one: the 64-bit definition against
differences, the CPU oracle against it."""

import pytest
import torch

import head_loss_masses as masses
import head_loss_oracle as oracle
from online_speculation_b200.ops import kernels as K


def _sums(case):
    h, w, ids, teacher, lse, g = case
    return (teacher.double() - lse.double()[:, None]).exp().sum(1)


@pytest.mark.parametrize("vocab,k", [(12, 4), (12, 12), (1, 1)])
def test_definition_against_differences(vocab, k):
    """Central differences of smooth functions: error O(step^2), 1e-6 at step 1e-4 for logits of order one."""
    case = masses.sure_inputs(7, 8, vocab, k, 5, "cpu")
    h, w, ids, teacher, lse, g = case
    h, w, g = 0.2 * h.double(), w.double(), g.double()
    total = _sums(case)
    assert k == 1 or (bool((total > 1.003).any()) and bool((total < 0.997).any()))
    out = masses.divergence(h, w, ids, teacher, g, None, lse)
    step = 1e-4
    for x, grad in ((h, out[2]), (w, out[4])):
        for i in range(x.numel()):
            keep = float(x.view(-1)[i])
            ends = []
            for s in (step, -step):
                x.view(-1)[i] = keep + s
                ends.append(float((masses.losses(h, w, ids, teacher, None, lse)[0] * g).sum()))
            x.view(-1)[i] = keep
            assert abs((ends[0] - ends[1]) / (2 * step) - float(grad.view(-1)[i])) < 1e-6


@pytest.mark.parametrize("rows,hidden,vocab,k", [(40, 64, 300, 8), (9, 72, 40, 40), (5, 8, 1, 1)])
@pytest.mark.parametrize("temp", [False, True])
def test_cpu_oracle_matches_definition(rows, hidden, vocab, k, temp):
    h, w, ids, teacher, lse, g = masses.sure_inputs(rows, hidden, vocab, k, 6, "cpu")
    it = 0.9 + 0.2 * torch.rand(rows, generator=torch.Generator().manual_seed(1)) if temp else None
    want = masses.divergence(h, w, ids, teacher, g, it, lse)
    h.requires_grad_()
    w.requires_grad_()
    loss = K.head_topk_divergence(h, w, ids, teacher, inv_temp=it, teacher_lse=lse)
    for got, i in zip((loss.detach(), *torch.autograd.grad(loss, [h, w], g)), (0, 2, 4)):
        oracle.within(got, want[i], want[i + 1], i)
