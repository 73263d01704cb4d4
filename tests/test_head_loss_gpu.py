"""The vocabulary-head losses and top logits on the sm_100a kernels against 64-bit definitions."""

import math

import pytest
import torch

import head_loss_oracle as oracle
from online_speculation_b200.ops import kernels as K
from online_speculation_b200.ops import workspace

pytestmark = pytest.mark.gpu


def _grads(loss, h, w, g):
    return torch.autograd.grad(loss, [h, w], g)


# rows, hidden, vocabulary: single rows and columns, one past a tile, odd, several tiles of each kind
SHAPES = [(1, 8, 1), (1, 64, 500), (2, 72, 257), (33, 512, 2048), (129, 136, 777), (300, 264, 1025), (257, 64, 20001),
          (64, 1536, 5000), (256, 520, 20011), (177, 1000, 40000), (512, 136, 513)]


@pytest.mark.parametrize("rows,hidden,vocab", SHAPES)
@pytest.mark.parametrize("smoothing,z_loss,piece,ignored", [(0.0, 0.0, None, 0.0), (0.1, 1e-3, 256, 0.4),
                                                            (0.0, 1e-3, 512, 0.2), (0.3, 0.0, None, 0.7)])
def test_cross_entropy(cuda, rows, hidden, vocab, smoothing, z_loss, piece, ignored):
    h, w, t, gen = oracle.make_inputs(rows, hidden, vocab, rows + vocab, cuda)
    t = torch.where(torch.rand(rows, generator=gen).to(cuda) < ignored, -100, t)
    if smoothing:
        t = t.int()
    g = torch.randn(rows, generator=gen).to(cuda)
    want = oracle.cross_entropy(h, w, t, g, smoothing=smoothing, z_loss=z_loss)
    h.requires_grad_()
    w.requires_grad_()
    loss = K.head_cross_entropy(h, w, t, label_smoothing=smoothing, z_loss=z_loss, piece=piece)
    dh, dw = _grads(loss, h, w, g)
    workspace.check_status(cuda)
    assert loss.dtype == torch.float32 and dh.dtype == dw.dtype == torch.bfloat16
    oracle.within(loss.detach(), want[0], want[1], "loss")
    oracle.within(dh, want[2], want[3], "dh")
    oracle.within(dw, want[4], want[5], "dW")


@pytest.mark.parametrize("pattern", ["none", "all", "first", "last"])
def test_ignored_rows_may_hold_anything(cuda, pattern):
    """NaN and infinities in ignored hidden rows reach neither the losses nor dW; no rows at all give zeros."""
    rows, hidden, vocab = 200, 128, 600
    h, w, t, gen = oracle.make_inputs(rows, hidden, vocab, 5, cuda)
    keep = {"none": slice(0, 0), "all": slice(0, rows), "first": slice(0, 131), "last": slice(rows - 1, rows)}[pattern]
    drop = torch.ones(rows, dtype=torch.bool, device=cuda)
    drop[keep] = False
    t[drop] = 7777
    g = torch.randn(rows, generator=gen).to(cuda)
    want = oracle.cross_entropy(h, w, t, g, ignore_index=7777)
    h[drop] = math.nan
    h[drop, 0] = math.inf
    g[drop] = math.nan
    h.requires_grad_()
    w.requires_grad_()
    loss = K.head_cross_entropy(h, w, t, ignore_index=7777, piece=256)
    dh, dw = _grads(loss, h, w, g)
    workspace.check_status(cuda)
    for got, i, name in ((loss.detach(), 0, "loss"), (dh, 2, "dh"), (dw, 4, "dW")):
        oracle.within(got, want[i], want[i + 1], name)
    assert bool((dh[drop] == 0).all()) and bool((loss[drop] == 0).all())


@pytest.mark.parametrize("rows,hidden,vocab,piece", [(90, 256, 1500, 512), (290, 400, 1500, None), (90, 256, 33000, None)])
@pytest.mark.parametrize("need", ["h", "w"])
def test_one_gradient(cuda, need, rows, hidden, vocab, piece):
    h, w, t, gen = oracle.make_inputs(rows, hidden, vocab, 9, cuda)
    g = torch.randn(rows, generator=gen).to(cuda)
    want = oracle.cross_entropy(h, w, t, g)
    leaf = (h if need == "h" else w).requires_grad_()
    loss = K.head_cross_entropy(h, w, t, piece=piece)
    (got,) = torch.autograd.grad(loss, [leaf], g)
    i = 2 if need == "h" else 4
    oracle.within(got, want[i], want[i + 1], need)


@pytest.mark.parametrize("layout", ["wide_rows", "shifted", "transposed", "one_row_view"])
def test_strides_and_alignment(cuda, layout):
    h, w, t, gen = oracle.make_inputs(45, 64, 700, 11, cuda)
    g = torch.randn(45, generator=gen).to(cuda)
    want = oracle.cross_entropy(h, w, t, g)

    def lay(x):
        n, m = x.shape
        if layout == "wide_rows":
            y = torch.full((n, m + 24), math.nan, dtype=x.dtype, device=cuda)[:, 8:8 + m]
        elif layout == "shifted":
            y = torch.full((n * (m + 5) + 3,), math.nan, dtype=x.dtype, device=cuda)[3:].view(n, m + 5)[:, :m]
        elif layout == "transposed":
            y = torch.empty(m, n, dtype=x.dtype, device=cuda).t()
        else:
            y = torch.full((2 * n, m), math.nan, dtype=x.dtype, device=cuda)[::2]
        y.copy_(x)
        return y.requires_grad_()

    hs, ws = lay(h), lay(w)
    wide_t = torch.zeros(45, 3, dtype=t.dtype, device=cuda)
    wide_t[:, 1] = t
    loss = K.head_cross_entropy(hs, ws, wide_t[:, 1])
    dh, dw = torch.autograd.grad(loss, [hs, ws], g.expand(2, 45)[1])
    oracle.within(loss.detach(), want[0], want[1], "loss")
    oracle.within(dh, want[2], want[3], "dh")
    oracle.within(dw, want[4], want[5], "dW")


def test_sum_backward_and_sure_rows(cuda):
    """An expanded upstream gradient (loss.sum()), and rows whose target has nearly all the mass: the
    gradient there is minus the mass of the rest, not the rounding of p - 1."""
    h, w, t, _ = oracle.make_inputs(40, 64, 300, 3, cuda, scale=1.0)
    h = (h + 40 * w[t]).bfloat16().requires_grad_()
    w.requires_grad_()
    want = oracle.cross_entropy(h, w, t, torch.ones(40, device=cuda))
    K.head_cross_entropy(h, w, t).sum().backward()
    oracle.within(h.grad, want[2], want[3], "dh")
    oracle.within(w.grad, want[4], want[5], "dW")


def test_bad_target_is_reported_and_left_out(cuda):
    h, w, t, gen = oracle.make_inputs(20, 64, 300, 4, cuda)
    bad = t.clone()
    bad[3], bad[7] = 300, -1
    with torch.no_grad():
        loss = K.head_cross_entropy(h, w, bad)
    with pytest.raises(RuntimeError, match="out of range"):
        workspace.check_status(cuda)
    assert float(loss[3]) == 0.0 and float(loss[7]) == 0.0
    want = oracle.cross_entropy(h, w, t, torch.ones(20, device=cuda))
    keep = torch.tensor([i for i in range(20) if i not in (3, 7)], device=cuda)
    oracle.within(loss[keep], want[0][keep], want[1][keep], "loss")


def _teacher(rows, vocab, k, gen, cuda, dtype, ragged):
    logits = 3 * torch.randn(rows, vocab, generator=gen)
    order = torch.stack([torch.randperm(vocab, generator=gen)[:k] for _ in range(rows)])
    teacher = logits.gather(1, order).to(dtype)
    if ragged:
        kept = torch.randint(0, k + 1, (rows,), generator=gen)
        kept[rows // 2] = 0
        order = torch.where(torch.arange(k)[None] < kept[:, None], order, -1)
    return logits.to(cuda), order.to(cuda), teacher.to(cuda)


@pytest.mark.parametrize("rows,hidden,vocab,k", [(1, 8, 1, 1), (1, 64, 500, 1), (3, 72, 40, 40), (50, 512, 2048, 8),
                                                 (130, 136, 777, 64), (40, 64, 3001, 512), (260, 200, 1030, 17),
                                                 (256, 64, 600, 512), (100, 72, 9000, 100), (257, 64, 512, 512), (400, 64, 5000, 33),
                                                 (20, 64, 140000, 200)])
@pytest.mark.parametrize("rest,temp,ragged,dtype,piece", [(False, False, False, torch.float32, None),
                                                          (True, True, True, torch.float32, 256),
                                                          (True, False, False, torch.bfloat16, 512),
                                                          (False, True, True, torch.bfloat16, None)])
def test_topk_divergence(cuda, rows, hidden, vocab, k, rest, temp, ragged, dtype, piece):
    h, w, _, gen = oracle.make_inputs(rows, hidden, vocab, rows + k, cuda)
    logits, ids, teacher = _teacher(rows, vocab, k, gen, cuda, dtype, ragged)
    it = (0.5 + torch.rand(rows, generator=gen)).to(cuda) if temp else None
    scaled = logits if it is None else logits * it[:, None]
    # a little above the listed mass where rounding the teacher to bf16 could have lifted it past the whole
    lse = scaled.logsumexp(1) + 0.01 if rest else None
    if temp:
        ids = ids.int()
    g = torch.randn(rows, generator=gen).to(cuda)
    want = oracle.topk_divergence(h, w, ids, teacher, g, it, lse)
    h.requires_grad_()
    w.requires_grad_()
    loss = K.head_topk_divergence(h, w, ids, teacher, inv_temp=it, teacher_lse=lse, piece=piece)
    dh, dw = _grads(loss, h, w, g)
    workspace.check_status(cuda)
    oracle.within(loss.detach(), want[0], want[1], "loss")
    oracle.within(dh, want[2], want[3], "dh")
    oracle.within(dw, want[4], want[5], "dW")


def test_topk_slots(cuda):
    """Columns listed twice, empty slots among full ones, -inf logits, a list without order, rows without a
    column, NaN in rows that do not count."""
    rows, vocab = 6, 900
    h, w, _, gen = oracle.make_inputs(rows, 64, vocab, 21, cuda)
    ids = torch.tensor([[5, 5, 5, 5], [899, -1, 0, 256], [-1, -1, -1, -1], [300, 300, 2, -7], [10, 11, 12, 13],
                        [255, 256, 511, 512]], device=cuda)
    teacher = torch.randn(rows, 4, generator=gen).to(cuda)
    teacher[4] = -math.inf
    teacher[5, 1] = -math.inf
    teacher[2] = math.nan
    g = torch.randn(rows, generator=gen).to(cuda)
    for lse in (None, torch.full((rows,), 4.0, device=cuda)):
        want = oracle.topk_divergence(h, w, ids, teacher, g, None, lse)
        hn = h.clone()
        hn[2], hn[4] = math.nan, math.inf
        hn.requires_grad_()
        wn = w.clone().requires_grad_()
        loss = K.head_topk_divergence(hn, wn, ids, teacher, teacher_lse=lse, piece=256)
        dh, dw = _grads(loss, hn, wn, g)
        oracle.within(loss.detach(), want[0], want[1], "loss")
        oracle.within(dh, want[2], want[3], "dh")
        oracle.within(dw, want[4], want[5], "dW")


def test_nan_stays_in_its_row(cuda):
    h, w, t, _ = oracle.make_inputs(30, 64, 300, 2, cuda)
    h[4, 3] = math.nan
    h.requires_grad_()
    loss = K.head_cross_entropy(h, w, t)
    (dh,) = torch.autograd.grad(loss.sum(), [h])
    for x in (loss.detach()[:, None], dh):
        bad = x.isnan().any(1)
        assert bool(bad[4]) and int(bad.sum()) == 1


def test_bad_column_is_reported_and_empty(cuda):
    h, w, _, gen = oracle.make_inputs(4, 64, 300, 6, cuda)
    ids = torch.tensor([[1, 300], [2, 3], [1 << 20, 4], [5, 6]], device=cuda)
    teacher = torch.randn(4, 2, generator=gen).to(cuda)
    with torch.no_grad():
        loss = K.head_topk_divergence(h, w, ids, teacher)
    with pytest.raises(RuntimeError, match="out of range"):
        workspace.check_status(cuda)
    want = oracle.topk_divergence(h, w, ids, teacher, torch.ones(4, device=cuda))
    oracle.within(loss, want[0], want[1], "loss")


def _top_reference(logits, k, it=None):
    x = logits.float().cpu()
    order = sorted_columns(x)[:, :k]
    z = x.double() if it is None else x.double() * it.double().cpu()[:, None]
    return x.gather(1, order), order, z.logsumexp(1)


def sorted_columns(x):
    """Columns by (NaN first, value descending, column)."""
    key = torch.where(x.isnan(), math.inf, x + 0.0)
    order = torch.sort(key, dim=1, descending=True, stable=True).indices
    nan = x.isnan().gather(1, order)
    return order.gather(1, torch.sort((~nan).int(), dim=1, stable=True).indices)


@pytest.mark.parametrize("rows,vocab,k", [(1, 1, 1), (1, 7, 7), (3, 4095, 5), (48, 2048, 8), (4, 40000, 16), (2, 152064, 512),
                                          (5, 151937, 1), (700, 9001, 64), (3, 513, 512), (1, 70001, 300)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("order", ["random", "rising", "falling", "few", "minus_inf"])
def test_top_logits(cuda, rows, vocab, k, dtype, order):
    g = torch.Generator().manual_seed(rows + vocab)
    x = 3 * torch.randn(rows, vocab, generator=g)
    if order in ("rising", "falling"):
        x = x.sort(1, descending=order == "falling").values
    elif order == "few":
        x = torch.randint(-1, 2, (rows, vocab), generator=g).float() * torch.rand(rows, 1, generator=g)
    elif order == "minus_inf":
        x[torch.rand(rows, vocab, generator=g) < 0.999] = -math.inf
        x[:, vocab // 2] = 0.5
    pad = vocab % 3
    wide = torch.zeros(rows, vocab + pad, dtype=dtype, device=cuda)
    wide[:, pad:] = x.to(dtype)
    logits = wide[:, pad:]
    it = (0.5 + torch.rand(rows, generator=g)).to(cuda) if k % 2 else None
    values, ids, lse = K.top_logits(logits, k, inv_temp=it)
    v, i, s = _top_reference(logits, k, it)
    assert values.dtype == torch.float32 and ids.dtype == torch.int32
    assert torch.equal(ids.cpu().long(), i) and torch.equal(values.cpu(), v)
    # exponentials within 2^-21, arguments rounded once at magnitudes below 64, sums of a few hundred terms a thread
    torch.testing.assert_close(lse.cpu().double(), s, rtol=2.0 ** -22, atol=2.0 ** -17)


def test_top_logits_nan_and_signed_zero(cuda):
    x = torch.full((2, 10000), -1.0)
    x[0, [17, 9000]] = math.nan
    x[0, 5] = math.inf
    x[1, [100, 200, 300]] = torch.tensor([-0.0, 0.0, -0.0])
    values, ids, lse = K.top_logits(x.to(cuda), 4)
    assert ids[0].tolist()[:3] == [17, 9000, 5] and bool(values[0, :2].isnan().all())
    assert ids[1].tolist() == [100, 200, 300, 0]
    assert math.copysign(1, float(values[1, 0])) == -1 and bool(lse[0].isnan())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [300, 10007, 200001])
def test_top_logits_extremes(cuda, dtype, vocab):
    """Infinities and the type's lowest value: columns and logsumexp as in 64 bits."""
    lowest = torch.finfo(dtype).min
    x = torch.randn(6, vocab, generator=torch.Generator().manual_seed(vocab)).to(dtype)
    x[0, vocab // 3] = math.inf
    x[1, [5, vocab - 1]] = math.inf
    x[2] = -math.inf
    x[3] = lowest
    x[4, 100:] = lowest
    x[5, : vocab - 1] = -math.inf
    values, ids, lse = K.top_logits(x.to(cuda), 7)
    v, i, s = _top_reference(x, 7)
    assert torch.equal(ids.cpu().long(), i) and torch.equal(values.cpu(), v)
    torch.testing.assert_close(lse.cpu().double(), s, rtol=2.0 ** -22, atol=2.0 ** -17)


def test_teacher_to_student(cuda):
    """Teacher logits are listed and kept; the student's head trains on them and on hard labels."""
    rows, hidden, vocab, k = 70, 256, 3000, 32
    h, w, t, gen = oracle.make_inputs(rows, hidden, vocab, 31, cuda)
    big = 2 * torch.randn(rows, vocab, generator=gen).to(cuda)
    it = (0.7 + torch.rand(rows, generator=gen)).to(cuda)
    values, ids, lse = K.top_logits(big, k, inv_temp=it)
    g = torch.ones(rows, device=cuda)
    a = oracle.topk_divergence(h, w, ids, values, g, it, lse)
    b = oracle.cross_entropy(h, w, t, 0.5 * g)
    h.requires_grad_()
    w.requires_grad_()
    loss = K.head_topk_divergence(h, w, ids, values, inv_temp=it, teacher_lse=lse)
    (loss.sum() + 0.5 * K.head_cross_entropy(h, w, t).sum()).backward()
    oracle.within(loss.detach(), a[0], a[1], "loss")
    # the two gradients are added in bf16: one more half step of each and of the sum
    for got, i in ((h.grad, 2), (w.grad, 4)):
        want = a[i] + b[i]
        oracle.within(got, want, a[i + 1] + b[i + 1] + oracle.BF16_HALF * (want.abs() + a[i].abs() + b[i].abs()), i)


def test_many_rows_and_pieces(cuda):
    """More rows than one block numbers at a time, an odd number of them counting, several pieces."""
    rows, hidden, vocab = 2500, 64, 1800
    h, w, t, gen = oracle.make_inputs(rows, hidden, vocab, 13, cuda)
    t[torch.rand(rows, generator=gen).to(cuda) < 0.45] = -100
    g = torch.randn(rows, generator=gen).to(cuda)
    want = oracle.cross_entropy(h, w, t, g)
    h.requires_grad_()
    w.requires_grad_()
    for piece in (None, 768):
        loss = K.head_cross_entropy(h, w, t, piece=piece)
        dh, dw = _grads(loss, h, w, g)
        for got, i, name in ((loss.detach(), 0, "loss"), (dh, 2, "dh"), (dw, 4, "dW")):
            oracle.within(got, want[i], want[i + 1], name)


# few rows on many columns: the backward pass reads the logits that the forward pass left
KEPT = [(3, 8, 32768), (200, 256, 40000), (255, 264, 32769), (1, 1024, 65537), (30, 1000, 70001), (70, 1024, 65700),
        (128, 1024, 65800), (130, 1048, 64501), (256, 2048, 33001)]


@pytest.mark.parametrize("rows,hidden,vocab", KEPT)
@pytest.mark.parametrize("listed", [0, 1, 40])
def test_kept_logits(cuda, rows, hidden, vocab, listed):
    h, w, t, gen = oracle.make_inputs(rows, hidden, vocab, rows + listed, cuda)
    drop = (torch.rand(rows, generator=gen) < 0.3).to(cuda)
    drop[rows // 2] = False
    g = torch.randn(rows, generator=gen).to(cuda)
    if listed:
        it = (0.5 + torch.rand(rows, generator=gen)).to(cuda)
        ids = torch.randint(0, vocab, (rows, listed), generator=gen).to(cuda)
        ids[0, 0] = vocab - 1
        ids[-1, -1] = 0
        ids[drop] = -1
        teacher = torch.randn(rows, listed, generator=gen).to(cuda)
        lse = teacher.logsumexp(1) + 1.0 + math.log(2.0)
        want = oracle.topk_divergence(h, w, ids, teacher, g, it, lse)
        call = lambda piece: K.head_topk_divergence(h, w, ids, teacher, inv_temp=it, teacher_lse=lse, piece=piece)
    else:
        t[drop] = -100
        t[rows // 2] = vocab - 1
        want = oracle.cross_entropy(h, w, t, g, smoothing=0.1, z_loss=1e-3)
        call = lambda piece: K.head_cross_entropy(h, w, t, label_smoothing=0.1, z_loss=1e-3, piece=piece)
    h[drop] = math.nan
    h.requires_grad_()
    w.requires_grad_()
    for piece in (None, 16384):
        loss = call(piece)
        first = torch.autograd.grad(loss, [h, w], g, retain_graph=True)
        only = torch.autograd.grad(loss, [h], g)[0]
        workspace.check_status(cuda)
        oracle.within(loss.detach(), want[0], want[1], "loss")
        oracle.within(first[0], want[2], want[3], "dh")
        oracle.within(first[1], want[4], want[5], "dW")
        oracle.within(only, want[2], want[3], "dh alone")


def test_kept_exponentials_in_pieces(cuda):
    """Many rows, several pieces whose length is no multiple of a block's columns, targets around the seams."""
    rows, hidden, vocab = 2560, 392, 60000
    h, w, t, gen = oracle.make_inputs(rows, hidden, vocab, 17, cuda)
    t[::2] = torch.randint(52100, 57400, (rows // 2,), generator=gen).to(cuda)
    t[5::40] = -100
    g = torch.randn(rows, generator=gen).to(cuda)
    want = oracle.cross_entropy(h, w, t, g, smoothing=0.1)
    h.requires_grad_()
    w.requires_grad_()
    loss = K.head_cross_entropy(h, w, t, label_smoothing=0.1)
    for got, i in zip((loss.detach(), *_grads(loss, h, w, g)), (0, 2, 4)):
        oracle.within(got, want[i], want[i + 1], i)


@pytest.mark.parametrize("k", [1, 100])
def test_kept_exponentials_of_lists(cuda, k):
    """Rows sure of one unlisted column, listed columns at the ends, a list in one block of columns."""
    rows, hidden, vocab = 300, 400, 20001
    h, w, t, gen = oracle.make_inputs(rows, hidden, vocab, 18, cuda)
    h = (h + 12 * w[t] * (torch.arange(rows, device=cuda) % 3 == 0)[:, None]).bfloat16()
    ids = torch.randint(0, vocab, (rows, k), generator=gen).to(cuda)
    ids[::4] = 9000 + torch.arange(k, device=cuda)
    ids[1, 0], ids[2, 0] = 0, vocab - 1
    ids[7] = -1
    teacher = torch.randn(rows, k, generator=gen).to(cuda)
    lse = teacher.logsumexp(1) + math.log(3.0)
    g = torch.randn(rows, generator=gen).to(cuda)
    want = oracle.topk_divergence(h, w, ids, teacher, g, None, lse)
    h.requires_grad_()
    w.requires_grad_()
    loss = K.head_topk_divergence(h, w, ids, teacher, teacher_lse=lse)
    first = torch.autograd.grad(loss, [h, w], g, retain_graph=True)
    again = torch.autograd.grad(loss, [h, w], g)
    for got, i in zip((loss.detach(), *first), (0, 2, 4)):
        oracle.within(got, want[i], want[i + 1], i)
    assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_what_is_kept(cuda):
    """A step keeps the logits of few rows until its graph goes; without gradients, or with a piece, nothing."""
    rows, hidden, vocab = 16, 1024, 65792
    h, w, t, _ = oracle.make_inputs(rows, hidden, vocab, 3, cuda)
    logits = 4 * 32 * vocab

    def held(piece=None):
        before = torch.cuda.memory_allocated()
        loss = K.head_cross_entropy(h, w, t, piece=piece)
        return torch.cuda.memory_allocated() - before, loss

    assert held()[0] < logits
    h.requires_grad_()
    with torch.no_grad():
        assert held()[0] < logits
    assert held(256)[0] < logits
    size, loss = held()
    assert size >= logits
    whole = torch.cuda.memory_allocated()
    loss.sum().backward()
    h.grad = None
    del loss
    assert torch.cuda.memory_allocated() <= whole - logits
    # two steps at a time have their own
    t2 = t.flip(0)
    a, b = K.head_cross_entropy(h, w, t), K.head_cross_entropy(h, w, t2)
    ga, gb = torch.autograd.grad(a.sum(), [h])[0], torch.autograd.grad(b.sum(), [h])[0]
    ones = torch.ones(rows, device=cuda)
    for got, target in ((ga, t), (gb, t2)):
        want = oracle.cross_entropy(h, w, target, ones)
        oracle.within(got, want[2], want[3], "dh")


def test_two_streams_at_once(cuda):
    """Eager calls in flight on two streams share no scratch."""
    cases = []
    for i, rows in enumerate((220, 700)):
        h, w, t, gen = oracle.make_inputs(rows, 128, 5000, 50 + i, cuda)
        g = torch.randn(rows, generator=gen).to(cuda)
        want = oracle.cross_entropy(h, w, t, g)
        logits = torch.randn(rows, 30000, generator=gen).to(cuda)
        cases.append((h.requires_grad_(), w.requires_grad_(), t, g, want, logits, torch.cuda.Stream()))
    torch.cuda.synchronize()
    results = [[], []]
    for _ in range(4):
        for i, (h, w, t, g, _, logits, stream) in enumerate(cases):
            with torch.cuda.stream(stream):
                loss = K.head_cross_entropy(h, w, t, piece=512)
                results[i].append((loss.detach(), *_grads(loss, h, w, g), K.top_logits(logits, 20)))
    torch.cuda.synchronize()
    for (h, w, t, g, want, logits, _), runs in zip(cases, results):
        values, ids, _ = _top_reference(logits, 20)
        for loss, dh, dw, top in runs:
            for got, j in ((loss, 0), (dh, 2), (dw, 4)):
                oracle.within(got, want[j], want[j + 1], j)
            assert torch.equal(top[1].cpu().long(), ids) and torch.equal(top[0].cpu(), values)


def test_gradient_rules(cuda):
    """Once differentiable; a head changed between the passes is noticed; the graph can be kept."""
    h, w, t, gen = oracle.make_inputs(20, 64, 300, 14, cuda)
    h.requires_grad_()
    w.requires_grad_()
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(K.head_cross_entropy(h, w, t).sum(), [h], create_graph=True)
    loss = K.head_cross_entropy(h, w, t)
    a = torch.autograd.grad(loss.sum(), [h, w], retain_graph=True)
    b = torch.autograd.grad(loss.sum(), [h, w], retain_graph=True)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    with torch.no_grad():
        w.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(loss.sum(), [h])
    assert not K.head_cross_entropy(h.detach(), w.detach(), t).requires_grad


def test_empty_batch(cuda):
    h = torch.zeros(0, 64, dtype=torch.bfloat16, device=cuda, requires_grad=True)
    w = torch.zeros(9, 64, dtype=torch.bfloat16, device=cuda, requires_grad=True)
    loss = K.head_cross_entropy(h, w, torch.zeros(0, dtype=torch.long, device=cuda))
    dh, dw = torch.autograd.grad(loss, [h, w], torch.zeros(0, device=cuda))
    assert loss.shape == (0,) and dh.shape == (0, 64) and bool((dw == 0).all())
    assert K.top_logits(torch.zeros(0, 9, device=cuda), 3)[0].shape == (0, 3)


def test_repeats_are_bitwise_equal(cuda):
    h, w, t, gen = oracle.make_inputs(500, 256, 9000, 8, cuda)
    h.requires_grad_()
    w.requires_grad_()
    g = torch.randn(500, generator=gen).to(cuda)
    runs = []
    for _ in range(3):
        loss = K.head_cross_entropy(h, w, t, piece=2048)
        runs.append((loss.detach(), *_grads(loss, h, w, g)))
    for other in runs[1:]:
        assert all(torch.equal(x, y) for x, y in zip(runs[0], other))


def test_side_stream_and_graph_replay(cuda):
    """The whole step captured once, replayed on new inputs, two graphs at the same time."""
    shapes = [(100, 128, 1500), (60, 256, 700)]
    graphs = []
    for i, (rows, hidden, vocab) in enumerate(shapes):
        h, w, t, gen = oracle.make_inputs(rows, hidden, vocab, 40 + i, cuda)
        h.requires_grad_()
        w.requires_grad_()
        g = torch.randn(rows, generator=gen).to(cuda)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())

        def step(h=h, w=w, t=t, g=g):
            loss = K.head_cross_entropy(h, w, t, piece=512)
            return (loss.detach(), *torch.autograd.grad(loss, [h, w], g))

        with torch.cuda.stream(stream):
            step()
        torch.cuda.current_stream().wait_stream(stream)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = step()
        graphs.append((graph, stream, h, w, t, g, out))
    for seed in (70, 71):
        for i, (_, _, h, w, t, g, _) in enumerate(graphs):
            nh, nw, nt, gen = oracle.make_inputs(*shapes[i], seed + 2 * i, cuda)
            nt[:: 3 + i] = -100
            with torch.no_grad():
                h.copy_(nh)
                w.copy_(nw)
                t.copy_(nt)
        torch.cuda.synchronize()
        for graph, stream, *_ in graphs:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for _, _, h, w, t, g, out in graphs:
            want = oracle.cross_entropy(h, w, t, g)
            for got, j in zip(out, (0, 2, 4)):
                oracle.within(got, want[j], want[j + 1], (seed, j))
    workspace.check_status(cuda)


def test_distillation_step_in_a_graph(cuda):
    """Teacher logits listed, student trained on them (kept logits), in one captured step next to an eager one."""
    rows, hidden, vocab, k = 48, 256, 33000, 20
    h, w, _, gen = oracle.make_inputs(rows, hidden, vocab, 90, cuda)
    big = torch.randn(rows, vocab, generator=gen).to(cuda)
    it = (0.7 + torch.rand(rows, generator=gen)).to(cuda)
    g = torch.randn(rows, generator=gen).to(cuda)
    h.requires_grad_()
    w.requires_grad_()

    def step():
        values, ids, lse = K.top_logits(big, k, inv_temp=it)
        loss = K.head_topk_divergence(h, w, ids, values, inv_temp=it, teacher_lse=lse)
        return (loss.detach(), *torch.autograd.grad(loss, [h, w], g), ids, values, lse)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = step()
    for seed in (91, 92):
        nh, nw, _, gen = oracle.make_inputs(rows, hidden, vocab, seed, cuda)
        with torch.no_grad():
            h.copy_(nh)
            w.copy_(nw)
            big.copy_(3 * torch.randn(rows, vocab, generator=gen).to(cuda))
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        eager = step()
        torch.cuda.synchronize()
        want = oracle.topk_divergence(h, w, eager[3], eager[4], g, it, eager[5])
        for run in (out, eager):
            for i in range(3):
                oracle.within(run[i], want[2 * i], want[2 * i + 1], (seed, i))
        assert all(torch.equal(a, b) for a, b in zip(out, eager))
    workspace.check_status(cuda)


@pytest.mark.parametrize("rows", [40, 300])
def test_edges_of_the_arguments(cuda, rows):
    """Targets smoothed away, an ignored index inside the vocabulary, a piece beyond it, inference mode."""
    h, w, t, gen = oracle.make_inputs(rows, 64, 500, 15, cuda)
    t[::3] = 7
    g = torch.randn(rows, generator=gen).to(cuda)
    want = oracle.cross_entropy(h, w, t, g, ignore_index=7, smoothing=1.0, z_loss=0.5)
    h.requires_grad_()
    w.requires_grad_()
    loss = K.head_cross_entropy(h, w, t, ignore_index=7, label_smoothing=1.0, z_loss=0.5, piece=1 << 30)
    for got, i in zip((loss.detach(), *_grads(loss, h, w, g)), (0, 2, 4)):
        oracle.within(got, want[i], want[i + 1], i)
    with torch.inference_mode():
        again = K.head_cross_entropy(h, w, t, ignore_index=7, label_smoothing=1.0, z_loss=0.5)
    assert not again.requires_grad
    oracle.within(again, want[0], want[1], "loss")


def test_offsets_past_32_bits(cuda):
    """Rows more than 2^31 elements apart, and a head whose rows reach past 2^31 elements."""
    gen = torch.Generator().manual_seed(1)
    far = (1 << 31) + 24
    logits = torch.empty(far + 6000, dtype=torch.bfloat16, device=cuda).as_strided((2, 5000), (far, 1), 3)
    logits.copy_(torch.randn(2, 5000, generator=gen))
    values, ids, lse = K.top_logits(logits, 9)
    v, i, s = _top_reference(logits, 9)
    assert torch.equal(ids.cpu().long(), i) and torch.equal(values.cpu(), v)
    torch.testing.assert_close(lse.cpu().double(), s, rtol=2.0 ** -22, atol=2.0 ** -17)
    del logits
    vocab, hidden = 140000, 64
    pitch = 16 * 1025
    wide = torch.empty(vocab * pitch, dtype=torch.bfloat16, device=cuda).as_strided((vocab, hidden), (pitch, 1))
    for rows in (20, 300):
        h, w, t, gen = oracle.make_inputs(rows, hidden, vocab, rows, cuda)
        wide.copy_(w)
        t[0] = vocab - 1
        g = torch.randn(rows, generator=gen).to(cuda)
        want = oracle.cross_entropy(h, w, t, g)
        h.requires_grad_()
        head = wide.detach().requires_grad_()
        loss = K.head_cross_entropy(h, head, t)
        for got, i in zip((loss.detach(), *_grads(loss, h, head, g)), (0, 2, 4)):
            oracle.within(got, want[i], want[i + 1], (rows, i))


def test_head_of_more_than_32_bits(cuda):
    """A contiguous head, and its gradient, of more than 2^31 elements; a few rows of it are looked at."""
    rows, hidden, vocab = 5, 16384, 133000
    h = torch.randn(rows, hidden, device=cuda).bfloat16()
    w = torch.empty(vocab, hidden, dtype=torch.bfloat16, device=cuda).normal_(0, 1 / 128)
    t = torch.tensor([0, vocab - 1, 70001, 132000, vocab - 1], device=cuda)
    logits = torch.cat([(h.double() @ w[i:i + 7000].double().t()) for i in range(0, vocab, 7000)], 1)
    lse = logits.logsumexp(1)
    dl = (logits - lse[:, None]).exp()
    dl[torch.arange(rows, device=cuda), t] -= 1
    dh_want = sum(dl[:, i:i + 7000] @ w[i:i + 7000].double() for i in range(0, vocab, 7000))
    h.requires_grad_()
    w.requires_grad_()
    loss = K.head_cross_entropy(h, w, t)
    dh, dw = _grads(loss, h, w, torch.ones(rows, device=cuda))
    hd = h.detach().double()
    err = 2 * math.sqrt(hidden) * oracle.FP32_HALF * float((hd.abs() @ w[:7000].detach().double().abs().t()).max())
    want = lse - logits.gather(1, t[:, None])[:, 0]
    assert float((loss.detach() - want).abs().max()) <= 2 * err + 8 * oracle.FP32_HALF * (float(want.max()) + 1)
    # half a step of the output, and what the logits' error (relative to p: twice it) does
    off = oracle.BF16_HALF + 4 * err
    assert float((dh - dh_want).norm()) <= off * float(dh_want.norm())
    for part in (slice(0, 300), slice(69900, 70100), slice(vocab - 300, vocab)):
        dw_want = dl[:, part].t() @ hd
        assert float((dw[part] - dw_want).norm()) <= off * float(dw_want.norm())
