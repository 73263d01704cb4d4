"""Edges of the vocabulary-head losses and top logits on the kernels."""

import pytest
import torch

import head_loss_masses as masses
import head_loss_oracle as oracle
from online_speculation_b200.ops import kernels as K
from online_speculation_b200.ops import workspace

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [65, 72, 80])
@pytest.mark.parametrize("listed", [0, 5])
def test_two_tiles_a_pair_of_65_to_80_rows(cuda, rows, listed):
    """Logits computed again with rows in columns, in three chains of 80 columns, both accumulators used."""
    hidden, vocab = 512, 24000
    h, w, t, gen = oracle.make_inputs(rows, hidden, vocab, rows, cuda)
    g = torch.randn(rows, generator=gen).to(cuda)
    if listed:
        ids = torch.randint(0, vocab, (rows, listed), generator=gen).to(cuda)
        teacher = torch.randn(rows, listed, generator=gen).to(cuda)
        lse = teacher.logsumexp(1) + 0.5
        want = oracle.topk_divergence(h, w, ids, teacher, g, None, lse)
    else:
        want = oracle.cross_entropy(h, w, t, g, smoothing=0.1)
    h.requires_grad_()
    w.requires_grad_()
    if listed:
        loss = K.head_topk_divergence(h, w, ids, teacher, teacher_lse=lse)
    else:
        loss = K.head_cross_entropy(h, w, t, label_smoothing=0.1)
    for got, i in zip((loss.detach(), *torch.autograd.grad(loss, [h, w], g)), (0, 2, 4)):
        oracle.within(got, want[i], want[i + 1], i)
    workspace.check_status(cuda)


def test_low_logits_of_many_rows(cuda):
    """Every logit near -120, so that exponentials about another row's normaliser, or about none, overflow: what stands
    behind the last row must not reach dW.  Several row tiles, two items a CTA pair, logits computed again."""
    rows, hidden, vocab = 701, 64, 10000
    h, w, t, gen = oracle.make_inputs(rows, hidden, vocab, 3, cuda)
    h[:, 0], w[:, 0] = -120.0, 1.0
    g = torch.randn(rows, generator=gen).to(cuda)
    want = oracle.cross_entropy(h, w, t, g)
    h.requires_grad_()
    w.requires_grad_()
    loss = K.head_cross_entropy(h, w, t)
    for got, i in zip((loss.detach(), *torch.autograd.grad(loss, [h, w], g)), (0, 2, 4)):
        oracle.within(got, want[i], want[i + 1], i)


def test_training_after_rollouts_in_inference_mode(cuda, monkeypatch):
    """The package's first kernel may run in inference mode: what it makes for the device serves training too."""
    monkeypatch.setattr(workspace, "_buffers", {})
    h, w, t, gen = oracle.make_inputs(20, 64, 300, 4, cuda)
    with torch.inference_mode():
        K.head_cross_entropy(h, w, t)
    g = torch.randn(20, generator=gen).to(cuda)
    want = oracle.cross_entropy(h, w, t, g)
    h.requires_grad_()
    w.requires_grad_()
    loss = K.head_cross_entropy(h, w, t)
    dh, dw = torch.autograd.grad(loss, [h, w], g)
    oracle.within(dh, want[2], want[3], "dh")
    oracle.within(dw, want[4], want[5], "dW")


def test_error_reported_between_the_passes(cuda):
    """A bad target is reported and its row left out; the step it was in, and others, still have their gradients."""
    h, w, t, gen = oracle.make_inputs(20, 64, 300, 4, cuda)
    bad = t.clone()
    bad[3] = 300
    g = torch.randn(20, generator=gen).to(cuda)
    without = torch.where(bad == 300, -100, t)
    want = oracle.cross_entropy(h, w, without, g)
    h.requires_grad_()
    w.requires_grad_()
    loss, other = K.head_cross_entropy(h, w, bad), K.head_cross_entropy(h, w, without)
    with pytest.raises(RuntimeError, match="out of range"):
        workspace.check_status(cuda)
    for x in (loss, other):
        dh, dw = torch.autograd.grad(x, [h, w], g)
        oracle.within(dh, want[2], want[3], "dh")
        oracle.within(dw, want[4], want[5], "dW")
    workspace.check_status(cuda)


def test_error_after_a_first_use_in_inference_mode(cuda, monkeypatch):
    monkeypatch.setattr(workspace, "_buffers", {})
    h, w, t, _ = oracle.make_inputs(20, 64, 300, 4, cuda)
    t[3] = 300
    with torch.inference_mode():
        K.head_cross_entropy(h, w, t)
    with pytest.raises(RuntimeError, match="out of range"):
        workspace.check_status(cuda)
    workspace.check_status(cuda)


def test_scratch_first_made_in_inference_mode(cuda, monkeypatch):
    monkeypatch.setattr(workspace, "_buffers", {})
    with torch.inference_mode():
        buffer = workspace.scratch(cuda, "test", 8, torch.float32)
    assert not buffer.is_inference() and not workspace.scratch(cuda, "test", 4, torch.float32).is_inference()


@pytest.mark.parametrize("rows,hidden,vocab", [(20, 512, 33000), (100, 512, 3000), (200, 512, 33000), (200, 512, 3000),
                                               (300, 512, 3000), (300, 256, 3000)])
@pytest.mark.parametrize("k", [1, 6])
@pytest.mark.parametrize("lead", [60.0, 100.0, 150.0, 900.0])
def test_rest_of_sure_students(cuda, rows, hidden, vocab, k, lead):
    """The best listed logit stands `lead` above the unlisted ones, whose mass is below what fp32 (88) or fp64 (745) holds: their
    gradient is that of their own softmax times what the teacher has there."""
    h, w, t, gen = oracle.make_inputs(rows, hidden, vocab, 7, cuda)
    ids = torch.stack([torch.randperm(vocab, generator=gen)[:k] for _ in range(rows)]).to(cuda)
    ids[:, 0] = torch.arange(rows, device=cuda)
    h = (h.float() + lead / 3 * w[:rows].float()).bfloat16()
    teacher = torch.randn(rows, k, generator=gen).to(cuda)
    lse = teacher.logsumexp(1) + 0.3
    g = torch.randn(rows, generator=gen).to(cuda)
    want = masses.divergence(h, w, ids, teacher, g, None, lse)
    h.requires_grad_()
    w.requires_grad_()
    loss = K.head_topk_divergence(h, w, ids, teacher, teacher_lse=lse)
    for got, i in zip((loss.detach(), *torch.autograd.grad(loss, [h, w], g)), (0, 2, 4)):
        oracle.within(got, want[i], want[i + 1], i)


@pytest.mark.parametrize("layout", ["transposed", "every_other"])
def test_one_column_of_any_stride(cuda, layout):
    """The inner stride of a single column means nothing."""
    x = torch.randn(5, generator=torch.Generator().manual_seed(1))
    wide = torch.zeros(5, 6)
    wide[:, 0] = x
    logits = x.to(cuda)[None].t() if layout == "transposed" else wide.to(cuda)[:, ::2][:, :1]
    assert logits.shape == (5, 1) and logits.stride(1) != 1
    values, ids, lse = K.top_logits(logits, 1)
    assert torch.equal(values.cpu()[:, 0], x) and not bool(ids.any()) and torch.equal(lse.cpu(), x)
