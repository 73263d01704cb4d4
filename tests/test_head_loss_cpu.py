"""Vocabulary-head losses and top logits without a GPU: the fp32 oracles against 64-bit definitions, those
against differences, and what the entry points refuse."""

import math

import pytest
import torch

import head_loss_oracle as oracle
from online_speculation_b200.ops import kernels as K

CPU = torch.device("cpu")


@pytest.mark.parametrize("smoothing,z_loss", [(0.0, 0.0), (0.1, 1e-3)])
def test_cross_entropy_matches_definition(smoothing, z_loss):
    h, w, t, gen = oracle.make_inputs(19, 64, 300, 1, CPU)
    t[[2, 18]] = -100
    g = torch.randn(19, generator=gen)
    want = oracle.cross_entropy(h, w, t, g, smoothing=smoothing, z_loss=z_loss)
    h[2] = math.nan
    h.requires_grad_()
    w.requires_grad_()
    loss = K.head_cross_entropy(h, w, t, label_smoothing=smoothing, z_loss=z_loss)
    dh, dw = torch.autograd.grad(loss, [h, w], g)
    oracle.within(loss.detach(), want[0], want[1], "loss")
    oracle.within(dh, want[2], want[3], "dh")
    oracle.within(dw, want[4], want[5], "dW")


@pytest.mark.parametrize("rest,k", [(False, 7), (True, 7), (True, 60)])
def test_topk_divergence_matches_definition(rest, k):
    h, w, _, gen = oracle.make_inputs(9, 64, 60, 2, CPU)
    logits = 2 * torch.randn(9, 60, generator=gen)
    it = 0.5 + torch.rand(9, generator=gen)
    values, ids, lse = K.top_logits(logits, k, inv_temp=it)
    ids[4] = -1
    ids[5, 1] = ids[5, 0]
    g = torch.randn(9, generator=gen)
    want = oracle.topk_divergence(h, w, ids, values, g, it, lse if rest else None)
    h.requires_grad_()
    w.requires_grad_()
    loss = K.head_topk_divergence(h, w, ids, values, inv_temp=it, teacher_lse=lse if rest else None)
    dh, dw = torch.autograd.grad(loss, [h, w], g)
    oracle.within(loss.detach(), want[0], want[1], "loss")
    oracle.within(dh, want[2], want[3], "dh")
    oracle.within(dw, want[4], want[5], "dW")


@pytest.mark.parametrize("kind", ["ce", "topk", "rest"])
def test_definitions_against_differences(kind):
    """Central differences of the 64-bit losses: error O(step^2) of smooth functions, 1e-6 at step 1e-4."""
    h, w, t, gen = oracle.make_inputs(5, 8, 12, 3, CPU)
    h, w = h.double(), w.double()
    t[1] = -100
    ids = torch.stack([torch.randperm(12, generator=gen)[:4] for _ in range(5)])
    ids[2, 3] = -1
    teacher = torch.randn(5, 4, generator=gen)
    it = 0.5 + torch.rand(5, generator=gen)
    lse = (teacher * it[:, None]).logsumexp(1) + 0.3
    g = torch.randn(5, generator=gen).double()

    def evaluate(h, w):
        if kind == "ce":
            return oracle.cross_entropy(h, w, t, g, smoothing=0.1, z_loss=0.01)
        return oracle.topk_divergence(h, w, ids, teacher, g, it, lse if kind == "rest" else None)

    out = evaluate(h, w)
    step = 1e-4
    for x, grad in ((h, out[2]), (w, out[4])):
        for i in range(0, x.numel(), 3):
            keep = float(x.view(-1)[i])
            ends = []
            for s in (step, -step):
                x.view(-1)[i] = keep + s
                ends.append(float((evaluate(h, w)[0] * g).sum()))
            x.view(-1)[i] = keep
            assert abs((ends[0] - ends[1]) / (2 * step) - float(grad.view(-1)[i])) < 1e-6


def test_full_list_with_rest_is_the_plain_divergence():
    """A list of every column leaves no rest: rounding of the teacher's normaliser must not invent one."""
    h, w, _, gen = oracle.make_inputs(6, 32, 20, 4, CPU)
    logits = torch.randn(6, 20, generator=gen)
    values, ids, lse = K.top_logits(logits, 20)
    p = logits.double().softmax(1)
    log_q = (h.double() @ w.double().t()).log_softmax(1)
    want = (p * (p.log() - log_q)).sum(1)
    got = K.head_topk_divergence(h, w, ids, values, teacher_lse=lse)
    torch.testing.assert_close(got.double(), want, rtol=1e-5, atol=1e-5)


def test_top_logits_order():
    x = torch.tensor([[1.0, math.nan, 3.0, 3.0, -0.0, 0.0, math.inf, -math.inf]])
    values, ids, lse = K.top_logits(x, 8)
    assert ids[0].tolist() == [1, 6, 2, 3, 0, 4, 5, 7] and ids.dtype == torch.int32
    values, ids, lse = K.top_logits(x[:, 2:6].bfloat16(), 2, inv_temp=torch.tensor([0.5]))
    assert ids[0].tolist() == [0, 1] and values.dtype == torch.float32
    torch.testing.assert_close(lse, (x[:, 2:6] * 0.5).logsumexp(1))


def test_empty_batches():
    h = torch.zeros(0, 16, dtype=torch.bfloat16, requires_grad=True)
    w = torch.zeros(5, 16, dtype=torch.bfloat16, requires_grad=True)
    for loss in (K.head_cross_entropy(h, w, torch.zeros(0, dtype=torch.long)),
                 K.head_topk_divergence(h, w, torch.zeros(0, 3, dtype=torch.long), torch.zeros(0, 3))):
        assert loss.shape == (0,) and loss.dtype == torch.float32
        dh, dw = torch.autograd.grad(loss, [h, w], torch.zeros(0))
        assert dh.shape == h.shape and bool((dw == 0).all())
    values, ids, lse = K.top_logits(torch.zeros(0, 9), 4)
    assert values.shape == (0, 4) and ids.shape == (0, 4) and lse.shape == (0,)
    # rows, but none that counts
    h = torch.zeros(3, 16, dtype=torch.bfloat16, requires_grad=True)
    loss = K.head_cross_entropy(h, w, torch.full((3,), -100))
    dh, dw = torch.autograd.grad(loss, [h, w], torch.ones(3))
    assert bool((loss == 0).all() and (dh == 0).all() and (dw == 0).all())


def _head(rows=3, hidden=16, vocab=9, dtype=torch.bfloat16):
    return torch.zeros(rows, hidden, dtype=dtype), torch.zeros(vocab, hidden, dtype=dtype)


@pytest.mark.parametrize("change,error", [
    (dict(h=torch.zeros(3, 16)), TypeError), (dict(weight=torch.zeros(9, 16, dtype=torch.float16)), TypeError),
    (dict(h=torch.zeros(3, 2, 16, dtype=torch.bfloat16)), ValueError),
    (dict(h=torch.zeros(3, 24, dtype=torch.bfloat16)), ValueError),
    (dict(weight=torch.zeros(0, 16, dtype=torch.bfloat16)), ValueError),
    (dict(targets=torch.zeros(4, dtype=torch.long)), ValueError), (dict(targets=torch.zeros(3)), TypeError),
    (dict(targets=torch.zeros(3, 1, dtype=torch.long)), ValueError),
    (dict(label_smoothing=-0.1), ValueError), (dict(label_smoothing=1.5), ValueError),
    (dict(z_loss=-1.0), ValueError), (dict(z_loss=math.nan), ValueError), (dict(piece=100), ValueError),
    (dict(piece=0), ValueError), (dict(targets=torch.tensor([0, 9, 1])), IndexError),
    (dict(targets=torch.tensor([0, -5, 1])), IndexError)])
def test_cross_entropy_refusals(change, error):
    h, w = _head()
    args = dict(h=h, weight=w, targets=torch.zeros(3, dtype=torch.long))
    args.update(change)
    with pytest.raises(error):
        K.head_cross_entropy(args.pop("h"), args.pop("weight"), args.pop("targets"), **args)


@pytest.mark.parametrize("hidden", [0, 4, 20])
def test_widths_off_eight_are_refused(hidden):
    h, w = _head(hidden=hidden)
    with pytest.raises(ValueError, match="multiple of 8"):
        K.head_cross_entropy(h, w, torch.zeros(3, dtype=torch.long))


@pytest.mark.parametrize("change,error", [
    (dict(ids=torch.zeros(3, dtype=torch.long)), ValueError), (dict(ids=torch.zeros(3, 0, dtype=torch.long)), ValueError),
    (dict(ids=torch.zeros(3, 513, dtype=torch.long), teacher=torch.zeros(3, 513)), ValueError),
    (dict(ids=torch.zeros(2, 4, dtype=torch.long)), ValueError), (dict(ids=torch.zeros(3, 4)), TypeError),
    (dict(teacher=torch.zeros(3, 5)), ValueError), (dict(teacher=torch.zeros(3, 4, dtype=torch.float64)), TypeError),
    (dict(inv_temp=torch.ones(2)), ValueError), (dict(inv_temp=torch.ones(3, dtype=torch.float64)), TypeError),
    (dict(teacher_lse=torch.ones(3, 1)), ValueError), (dict(piece=17), ValueError),
    (dict(ids=torch.full((3, 4), 9)), IndexError)])
def test_topk_divergence_refusals(change, error):
    h, w = _head()
    args = dict(ids=torch.zeros(3, 4, dtype=torch.long), teacher=torch.zeros(3, 4))
    args.update(change)
    with pytest.raises(error):
        K.head_topk_divergence(h, w, args.pop("ids"), args.pop("teacher"), **args)


@pytest.mark.parametrize("args,error", [
    ((torch.zeros(3), 1), ValueError), ((torch.zeros(3, 4), 0), ValueError), ((torch.zeros(3, 4), 5), ValueError),
    ((torch.zeros(3, 600), 513), ValueError), ((torch.zeros(3, 4, dtype=torch.float64), 1), TypeError),
    ((torch.zeros(3, 4, dtype=torch.long), 1), TypeError)])
def test_top_logits_refusals(args, error):
    with pytest.raises(error):
        K.top_logits(*args)
    with pytest.raises(ValueError):
        K.top_logits(torch.zeros(3, 4), 1, inv_temp=torch.ones(4))
