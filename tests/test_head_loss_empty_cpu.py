"""Empty batches of the vocabulary-head losses."""

import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

from online_speculation_b200.ops import kernels as K


class _Largest(TorchDispatchMode):
    """The most elements that any operation returned."""

    elements = 0

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        out = func(*args, **(kwargs or {}))
        for t in out if isinstance(out, (tuple, list)) else (out,):
            if isinstance(t, torch.Tensor):
                self.elements = max(self.elements, t.numel())
        return out


@pytest.mark.parametrize("kind", ["ce", "topk"])
def test_empty_batch_copies_no_head(kind):
    h = torch.zeros(0, 16, dtype=torch.bfloat16, requires_grad=True)
    w = torch.full((50, 16), float("nan"), dtype=torch.bfloat16, requires_grad=True)
    with _Largest() as seen:
        if kind == "ce":
            loss = K.head_cross_entropy(h, w, torch.zeros(0, dtype=torch.long))
        else:
            loss = K.head_topk_divergence(h, w, torch.zeros(0, 3, dtype=torch.long), torch.zeros(0, 3))
    assert loss.shape == (0,) and loss.dtype == torch.float32 and seen.elements < 50
    dh, dw = torch.autograd.grad(loss, [h, w], torch.zeros(0))
    assert dh.shape == h.shape and dw.dtype == torch.bfloat16 and bool((dw == 0).all())
