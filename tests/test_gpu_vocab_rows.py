"""Kernels of the operators on vocabulary rows against plain 64-bit statements: types, odd sizes, strides, empty and unusual
rows, streams, graphs, repeated backward passes."""
import math

import pytest
import torch

import vocab_rows_oracle as oracle

pytestmark = pytest.mark.gpu
INF, NAN = math.inf, math.nan
BF16, F32 = torch.bfloat16, torch.float32


def _ops():
    from multimodal_training_b200.ops import functional as F
    return F


@pytest.fixture(autouse=True)
def _no_device_error():
    yield
    from multimodal_training_b200.ops import native as nv
    assert nv.get_error()[0] == 0


def _laid_out(x, layout):
    """The same values as `x` [.., V] behind other strides."""
    if layout == "dense":
        return x
    V = x.shape[-1]
    pad = {"padded": (0, 8 - V % 8 + 8), "shifted": (3, 2)}[layout]
    return torch.nn.functional.pad(x, pad, value=1e4)[..., pad[0]:pad[0] + V]


# ---------------------------------------------------------------- top logits
def _rows_of(kind, T, V, dtype):
    g = torch.Generator().manual_seed(V)
    x = 3 * torch.randn(T, V, generator=g)
    if kind == "equal":
        x = torch.zeros(T, V)
        x[:, ::3] = -0.0
    elif kind == "few":
        x = torch.randint(-2, 3, (T, V), generator=g).float()
    elif kind == "rising":
        x = torch.arange(V).float().expand(T, V) / V + torch.arange(T)[:, None]
    elif kind == "falling":
        x = -torch.arange(V).float().expand(T, V) / V
    elif kind == "special":
        x[0, V // 2] = NAN
        x[-1] = -INF
        x[-1, V // 3] = INF
        x[0, -1] = -NAN
    return x.to(dtype).cuda()


@pytest.mark.parametrize("V", [1, 2, 9, 255, 256, 1000, 4097, 16385, 50001, 152064])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("kind", ["normal", "equal", "few", "rising", "falling", "special"])
def test_top_logits(V, dtype, kind):
    F = _ops()
    x = _rows_of(kind, 3, V, dtype)
    for k in sorted({1, min(V, 7), min(V, 64), min(V, 256)}):
        for layout in ("dense", "shifted"):
            values, ids = F.top_logits(_laid_out(x, layout), k)
            want_v, want_i = oracle.top(x, k)
            assert torch.equal(ids.cpu(), want_i), (k, layout)
            assert torch.equal(values.cpu().view(torch.int16 if dtype == BF16 else torch.int32),
                               want_v.view(torch.int16 if dtype == BF16 else torch.int32))


@pytest.mark.parametrize("T", [1, 2, 37, 147, 148, 149, 600])
def test_top_logits_of_many_rows(T):
    F = _ops()
    x = _rows_of("normal", T, 5003, BF16)
    values, ids = F.top_logits(x, 40)
    want_v, want_i = oracle.top(x, 40)
    assert torch.equal(ids.cpu(), want_i) and torch.equal(values.cpu(), want_v)


@pytest.mark.parametrize("V", [700, 3001, 30001, 70001])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("kind", ["normal", "equal", "few", "rising", "special"])
def test_top_logits_of_a_block_a_row(V, dtype, kind):
    """So many rows that none is cut over blocks: the blocks of all sizes, also with ties and lists that overflow."""
    F = _ops()
    x = _rows_of(kind, 3, V, dtype)
    for k in (8, 64, 65, 256):
        values, ids = F.top_logits(x.repeat(100, 1), k)
        want_v, want_i = oracle.top(x, k)
        assert torch.equal(ids.cpu(), want_i.repeat(100, 1)), k
        assert torch.equal(values.cpu().view(torch.int16 if dtype == BF16 else torch.int32),
                           want_v.repeat(100, 1).view(torch.int16 if dtype == BF16 else torch.int32))


def _tied_rows(V, dtype):
    """Rows of which many logits share the k-th place, far below the largest one or as the largest one."""
    g = torch.Generator().manual_seed(V)
    x = torch.full((8, V), -1.0)
    x[1] = -0.5
    for r, some in ((2, 20), (3, 40), (4, 100)):    # log-probabilities of a masked vocabulary
        some = min(some, V)
        x[r] = -INF
        x[r, torch.randperm(V, generator=g)[:some]] = -0.3 - 5.7 * torch.rand(some, generator=g)
    x[5] = 0.0                                      # few late positive logits
    x[5, -min(100, V):] = 2.0 + 30 * torch.rand(min(100, V), generator=g)
    x[6, ::2] = -2.0
    x[7] = -1e4
    x[7, V // 2] = 3.0
    return x.to(dtype).cuda()


@pytest.mark.parametrize("V", [130, 300, 1000, 2048, 5003, 30001, 152064])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("copies", [1, 80])
def test_top_logits_of_rows_with_many_equal_ones(V, dtype, copies):
    """With 8 rows they are cut over blocks, with 640 a block has a row, in the sizes that k and V ask for."""
    F = _ops()
    x = _tied_rows(V, dtype)
    wide = x.repeat(copies, 1)
    want_v, want_i = oracle.top(x, min(V, 256))
    for k in sorted({min(V, k) for k in (40, 64, 65, 100, 129, 130, 150, 191, 200, 230, 255, 256)}):
        values, ids = F.top_logits(wide, k)
        assert torch.equal(ids.cpu(), want_i[:, :k].repeat(copies, 1)), k
        assert torch.equal(values.cpu(), want_v[:, :k].repeat(copies, 1)), k


def test_rows_behind_two_to_the_31_elements():
    F = _ops()
    ld, V = 1_100_000_003, 1001
    big = torch.empty(2 * ld + V, device="cuda", dtype=BF16)
    x = big.as_strided((3, V), (ld, 1))
    x.copy_(_rows_of("normal", 3, V, BF16))
    values, ids = F.top_logits(x, 9)
    want_v, want_i = oracle.top(x, 9)
    assert torch.equal(ids.cpu(), want_i) and torch.equal(values.cpu(), want_v)
    ids, teacher = ids.roll(1, 0), values.roll(1, 0).float()
    loss, grad = _loss_and_grad(x, ids, teacher)
    want, dx, size = oracle.distill(x, ids, teacher)
    _near(loss, grad, want, dx, size, 1.0, BF16)
    target = big.as_strided((1, 3, V), (0, ld, 1))
    u = torch.rand(1, 3, device="cuda")
    _same(F.verify_drafts(target, ids[:2, :1].T, None, u), oracle.verify(target, ids[:2, :1].T, None, u))


# ---------------------------------------------------------------- distillation
def _batch(T, V, K, dtype, seed=0, scale=2.5):
    g = torch.Generator().manual_seed(seed)
    x = scale * torch.randn(T, V, generator=g)
    teacher, ids = (x + 0.7 * torch.randn(T, V, generator=g)).topk(K, dim=1)
    ids[1::4] = -1                                  # rows without a teacher
    if K > 2:
        ids[2::4, 1] = -1                           # fewer logits
        ids[3::4, 2] = ids[3::4, 0]                 # an id twice
        teacher[0, 1] = -INF
    labels = torch.randint(0, V, (T,), generator=g)
    labels[::3] = -100
    labels[4::9] = ids[4::9, 0]
    return x.to(dtype).cuda(), ids.cuda(), teacher.cuda(), labels.cuda()


def _loss_and_grad(x, ids, teacher, **kw):
    x = x.detach().requires_grad_()
    loss = _ops().distillation_loss(x, ids, teacher, **kw)
    return loss.detach(), torch.autograd.grad(loss, x)[0]


def _near(loss, grad, want, dx, size, temperature, dtype):
    """A sum over up to 2^18 logits in fp32 is at most 300 additions of one thread and a few of the block: 2^-15.7 of it;
    an exponent of up to 60 is off by 2^-18.6, both at most 2^-15 together.  The gradient's two parts are off by that
    before they cancel, and the result is rounded once.  A row's loss is off by as much of tau^2."""
    assert loss.dtype == F32 and grad.dtype == dtype
    half = torch.finfo(dtype).eps / 2
    off = (grad.cpu().double() - dx).abs()
    assert (off <= half * dx.abs() + 2.0 ** -15 * size + 1e-37).all(), float((off - half * dx.abs() - 2.0 ** -15 * size).max())
    assert abs(float(loss) - want) <= 2.0 ** -15 * max(1.0, temperature ** 2) + 2.0 ** -23 * abs(want)


@pytest.mark.parametrize("T,V,K", [(1, 1, 1), (1, 8, 8), (5, 9, 3), (3, 1000, 256), (70, 1023, 5), (33, 4096, 17), (6, 50001, 64),
                                   (9, 152064, 64), (2, 262145, 9)])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("temperature,share", [(1.0, 0.0), (2.0, 0.3), (1.0, 0.5), (0.5, 1.0)])
def test_distillation(T, V, K, dtype, temperature, share):
    x, ids, teacher, labels = _batch(T, V, K, dtype)
    want = oracle.distill(x, ids, teacher, temperature, labels, share)
    for layout in ("dense", "padded", "shifted"):
        got = _loss_and_grad(_laid_out(x, layout), ids, teacher, temperature=temperature, labels=labels, label_weight=share)
        _near(*got, *want, temperature, dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_distillation_takes_other_types_and_strides(dtype):
    x, ids, teacher, labels = _batch(24, 501, 6, dtype)
    want = oracle.distill(x, ids, teacher.bfloat16(), 1.0, labels, 0.5)
    wide_i, wide_t = torch.stack([ids, ids - 1], -1)[..., 0], _laid_out(teacher.bfloat16(), "shifted")
    kw = dict(labels=labels.int(), label_weight=0.5)
    got = _loss_and_grad(x.view(2, 12, -1), wide_i.int().view(2, 12, -1), wide_t.reshape(2, 12, -1),
                         labels=labels.int().view(2, 12), label_weight=0.5)
    _near(got[0], got[1].view(24, -1), *want, 1.0, dtype)
    _near(*_loss_and_grad(x.T.contiguous().T, wide_i, wide_t, **kw), *want, 1.0, dtype)
    _near(*_loss_and_grad(x, ids, teacher.bfloat16().double(), **kw), *want, 1.0, dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_distillation_of_unusual_rows(dtype):
    T, V, K = 40, 1234, 5
    x, ids, teacher, labels = _batch(T, V, K, dtype)
    ids[8:20] = -1
    teacher[20] = -INF
    labels[8:21] = -100
    x[8:21] = NAN                                   # what a row without teacher and label holds does not matter
    x[21, 3:700] = -INF                             # columns without mass
    ids[21] = torch.arange(700, 700 + K, device="cuda")
    labels[21] = 900
    x[22] = 77.0                                    # all equal
    x[23] *= 1e3                                    # all mass on one
    teacher[23] = teacher[23] * 1e3
    ids[23, 1:] = -1
    ids[23, 0] = x[23].argmax()
    labels[23] = ids[23, 0]
    for share in (0.0, 0.4):
        want = oracle.distill(x, ids, teacher, 1.5, labels, share)
        got = _loss_and_grad(x, ids, teacher, temperature=1.5, labels=labels, label_weight=share)
        assert not got[1][8:21].any()
        _near(*got, *want, 1.5, dtype)
    x[22, ids[22][ids[22] >= 0][0]] = -INF          # the teacher has mass where the student has none
    assert math.isinf(float(_loss_and_grad(x, ids, teacher)[0]))
    nothing = _loss_and_grad(x, torch.full_like(ids, -1), teacher)
    assert float(nothing[0]) == 0.0 and not nothing[1].any()
    loss, grad = _loss_and_grad(x[:0], ids[:0], teacher[:0])
    assert float(loss) == 0.0 and grad.shape == (0, V)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("temperature,share", [(1.0, 0.5), (2.0, 0.5), (3.0, 0.5)])
def test_distillation_of_rows_masked_with_the_lowest_value(dtype, temperature, share):
    T, V, K = 8, 1003, 4
    low = torch.finfo(dtype).min
    x, ids, teacher, labels = _batch(T, V, K, dtype)
    ids[:], labels[:] = torch.arange(K, device="cuda"), 2
    teacher[:] = torch.arange(K, device="cuda").float()
    x[0, 10:] = low                                 # part of a row
    x[1] = low                                      # all of it: every id is as likely
    x[2] = -low
    x[3] = 1e30
    x[4, :] = 2e4
    x[4, ::2] += 100
    # what is masked has no part in the divergence here, so fp64 has an answer for all of them; its quotients by the
    # temperature do not overflow
    want = oracle.distill(x, ids, teacher, temperature, labels, share)
    _near(*_loss_and_grad(x, ids, teacher, temperature=temperature, labels=labels, label_weight=share), *want, temperature, dtype)


@pytest.mark.parametrize("dtype,V", [(BF16, 820_001), (F32, 410_003)])
@pytest.mark.parametrize("temperature,share", [(2.0, 0.3), (1.0, 0.5)])
def test_distillation_of_a_vocabulary_that_no_cluster_holds(dtype, V, temperature, share):
    x, ids, teacher, labels = _batch(6, V, 5, dtype)
    labels[2] = 7
    x[4] = torch.finfo(dtype).min
    want = oracle.distill(x, ids, teacher, temperature, labels, share)
    _near(*_loss_and_grad(x, ids, teacher, temperature=temperature, labels=labels, label_weight=share), *want, temperature, dtype)


@pytest.mark.parametrize("temperature,share", [(1.0, 0.0), (2.0, 0.3), (0.5, 1.0)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_distillation_of_vocabulary_shards(monkeypatch, dtype, temperature, share):
    """The ranks are threads that meet on the host where they would reduce."""
    import threading
    from multimodal_training_b200.ops import vocab_rows
    F = _ops()
    T, V, K, world = 12, 1000, 6, 2
    x, ids, teacher, labels = _batch(T, V, K, dtype)
    x[4, :V // 2] = -INF                            # one shard has nothing
    ids[4], labels[4] = torch.arange(V // 2, V // 2 + K, device="cuda"), V - 1
    x[5, V // 2:], x[8] = torch.finfo(dtype).min, torch.finfo(dtype).min
    ids[5], ids[8], labels[8] = torch.arange(K, device="cuda"), torch.arange(497, 497 + K, device="cuda"), 500
    meet, given, rank_of = threading.Barrier(world, timeout=60), [None] * world, threading.local()

    def all_reduce(t, op, group):
        given[rank_of.rank] = t.clone()
        meet.wait()
        both = torch.stack(given)
        meet.wait()
        t.copy_(both.amax(0) if op == torch.distributed.ReduceOp.MAX else both.sum(0))

    monkeypatch.setattr(F, "_all_reduce", all_reduce)
    labels_or_none = None if share == 0 else labels
    out = [None] * world

    def rank(r):
        rank_of.rank = r
        lo = r * (V // world)
        mine = x[:, lo:lo + V // world]
        d = vocab_rows._Distill(ids, teacher, labels_or_none, temperature, share, lo, V, dtype == F32, V // world)
        d.row_stats(mine)
        d.reduce(0, T, None)
        grad = torch.empty(T, V // world, device="cuda", dtype=dtype)
        d.grad(mine, grad)
        out[r] = d.loss(), grad

    threads = [threading.Thread(target=rank, args=(r,)) for r in range(world)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert torch.equal(out[0][0], out[1][0])
    _near(out[0][0], torch.cat([g for _, g in out], 1), *oracle.distill(x, ids, teacher, temperature, labels, share), temperature,
          dtype)


def _group_of(monkeypatch, world, all_reduce):
    """A process group of `world` ranks of which this process is one."""
    from multimodal_training_b200.ops import vocab_rows
    monkeypatch.setattr(vocab_rows, "_multi", lambda group: group is not None)
    monkeypatch.setattr(torch.distributed, "get_world_size", lambda group=None: world)
    monkeypatch.setattr(_ops(), "_all_reduce", all_reduce)
    return object()


@pytest.mark.parametrize("temperature,share", [(1.0, 0.0), (2.0, 0.3), (0.5, 1.0)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_repeated_backward_passes_of_vocabulary_shards(monkeypatch, dtype, temperature, share):
    """The loss is there before the gradient is formed again."""
    import threading
    T, V, K, world = 12, 1000, 6, 2
    x, ids, teacher, labels = _batch(T, V, K, dtype)
    meet, given, rank_of = threading.Barrier(world, timeout=60), [None] * world, threading.local()

    def all_reduce(t, op, group):
        given[rank_of.rank] = t.clone()
        meet.wait()
        both = torch.stack(given)
        meet.wait()
        t.copy_(both.amax(0) if op == torch.distributed.ReduceOp.MAX else both.sum(0))

    group, out = _group_of(monkeypatch, world, all_reduce), [None] * world
    factors = (1.0, 0.25, 3.0)

    def rank(r):
        rank_of.rank = r
        lo = r * (V // world)
        mine = x[:, lo:lo + V // world].detach().requires_grad_()
        loss = _ops().distillation_loss(mine, ids, teacher, temperature=temperature, labels=labels, label_weight=share,
                                        vocab_lo=lo, group=group)
        out[r] = loss.detach(), [torch.autograd.grad(loss, mine, torch.tensor(f, device="cuda"), retain_graph=True)[0]
                                 for f in factors]

    threads = [threading.Thread(target=rank, args=(r,)) for r in range(world)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    want, dx, size = oracle.distill(x, ids, teacher, temperature, labels, share)
    for i, f in enumerate(factors):
        _near(out[0][0], torch.cat([g[i] for _, g in out], 1), want, f * dx, f * size, temperature, dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_captured_backward_pass_of_a_vocabulary_shard(monkeypatch, dtype):
    """The other rank's half of the vocabulary has no mass, so that this one's answer is the whole one."""
    T, V, K = 12, 1000, 6
    group = _group_of(monkeypatch, 2, lambda t, op, group: None)
    x, ids, teacher, labels = _batch(T, V, K, dtype)
    x.requires_grad_()

    def step():
        loss = _ops().distillation_loss(x, ids, teacher, temperature=2.0, labels=labels, label_weight=0.3, group=group)
        return loss.detach(), torch.autograd.grad(loss * 0.5, x)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, grad = step()
    for seed in (1, 2):
        y = _batch(T, V, K, dtype, seed=seed)[0]
        with torch.no_grad():
            x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        want, dx, size = oracle.distill(y, ids, teacher, 2.0, labels, 0.3)
        _near(loss, grad, want, 0.5 * dx, 0.5 * size, 2.0, dtype)


def test_rows_that_all_weight_leaves_are_not_read():
    x, ids, teacher, labels = _batch(8, 500, 4, BF16)
    labels[:] = torch.tensor([3, -100] * 4)
    want = _loss_and_grad(x, ids, teacher, labels=labels, label_weight=1.0)
    x[1::2] = NAN                                   # a teacher without weight, no label
    got = _loss_and_grad(x, ids, teacher, labels=labels, label_weight=1.0)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and not got[1][1::2].any()


def test_rows_of_a_broadcast_batch():
    x, ids, teacher, _ = _batch(1, 3001, 5, BF16)
    wide = x.detach().requires_grad_()
    loss = _ops().distillation_loss(wide.expand(40, 3001).unflatten(0, (4, 10)), ids.expand(4, 10, 5), teacher.expand(4, 10, 5))
    want, dx, size = oracle.distill(x, ids, teacher)
    # a fortieth each, rounded, whose sum rounds to bf16 once more (or on the way: 40 terms at half a step each)
    (grad,) = torch.autograd.grad(loss, wide)
    assert ((grad.cpu().double() - dx).abs() <= 2.0 ** -8 * 41 * dx.abs() + 2.0 ** -15 * size + 1e-37).all()
    assert abs(loss.item() - want) <= 2.0 ** -15
    values, top = _ops().top_logits(x.expand(3, 3001), 4)
    assert torch.equal(top, top[:1].expand(3, 4)) and torch.equal(top[:1].cpu(), oracle.top(x, 4)[1])


def test_a_captured_backward_pass_has_a_captured_forward_pass(monkeypatch):
    F = _ops()
    x, ids, teacher, _ = _batch(4, 64, 4, BF16)
    w = torch.ones(64, 64, device="cuda", dtype=BF16)
    losses = F.distillation_loss(x.requires_grad_(), ids, teacher), F.lm_head_distillation(x, w, ids, teacher)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    for loss in losses:
        with pytest.raises(RuntimeError, match="capture both"):
            loss.backward()


def test_ids_outside_the_vocabulary_are_left_out_and_reported():
    from multimodal_training_b200.ops import native as nv
    x, ids, teacher, labels = _batch(8, 300, 6, BF16)
    ids[0, 2] = 300
    loss, grad = _loss_and_grad(x, ids, teacher)
    with pytest.raises(RuntimeError, match="out-of-range"):
        nv.raise_on_device_error()
    ids[0, 2] = -1
    want = oracle.distill(x, ids, teacher)
    _near(loss, grad, *want, 1.0, BF16)


def test_repeated_and_scaled_backward_passes():
    F = _ops()
    x, ids, teacher, labels = _batch(30, 2049, 6, F32)
    want, dx, size = oracle.distill(x, ids, teacher)
    x.requires_grad_()
    loss = F.distillation_loss(x, ids, teacher)
    for factor in (1.0, 0.25, 3.0, 0.0):
        (got,) = torch.autograd.grad(loss, x, torch.tensor(factor, device="cuda"), retain_graph=True)
        _near(loss.detach(), got, want, factor * dx, factor * size, 1.0, F32)
    (2.0 * F.distillation_loss(x, ids, teacher)).backward()
    _near(loss.detach(), x.grad, want, 2 * dx, 2 * size, 1.0, F32)
    with torch.no_grad():
        assert F.distillation_loss(x, ids, teacher).item() == loss.item()


def test_same_bits_every_time():
    F = _ops()
    x, ids, teacher, labels = _batch(300, 8191, 20, BF16)
    first = _loss_and_grad(x, ids, teacher, labels=labels, label_weight=0.2)
    for _ in range(5):
        again = _loss_and_grad(x, ids, teacher, labels=labels, label_weight=0.2)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
    assert torch.equal(F.distillation_loss(x, ids, teacher, labels=labels, label_weight=0.2), first[0])


@pytest.mark.parametrize("T,H,V,K,chunk", [(1, 64, 1024, 4, 4096), (70, 128, 1544, 9, 4096), (300, 256, 1032, 256, 128),
                                           (1025, 192, 2056, 33, 512)])
@pytest.mark.parametrize("temperature,share", [(1.0, 0.0), (2.0, 0.3)])
def test_head(T, H, V, K, chunk, temperature, share):
    F = _ops()
    g = torch.Generator().manual_seed(T)
    h = torch.randn(T, H, generator=g).cuda().bfloat16()
    w = (torch.randn(V, H, generator=g) / H ** 0.5).cuda().bfloat16()
    _, ids, teacher, labels = _batch(T, V, K, BF16)
    ids[T // 8:T // 2] = -1                         # image tokens
    labels[T // 8:T // 2] = -100
    if T > 1:
        h[T // 8:T // 2] *= 1e4
    kw = dict(temperature=temperature, labels=labels, label_weight=share)
    hd, wd = h.double().cpu().requires_grad_(), w.double().cpu().requires_grad_()
    z = hd @ wd.T
    want, dz, _ = oracle.distill(z, ids, teacher, temperature, labels, share)
    dh, dw = torch.autograd.grad(z, (hd, wd), dz)
    h.requires_grad_(), w.requires_grad_()
    loss = F.lm_head_distillation(h, w, ids, teacher, chunk_rows=chunk, **kw)
    # logits, their gradient and the results are rounded to bf16: logits of up to 5 are off by up to 2^-7 (3 rms of them 2^-9
    # of their size), which moves a row's loss by less than 2^-7 tau^2 and the gradients by about 2^-8 of the whole
    assert abs(loss.item() - want) < 2.0 ** -7 * max(1.0, temperature)
    for factor in (1.0, 0.5):
        got = torch.autograd.grad(loss, (h, w), torch.tensor(factor, device="cuda"), retain_graph=True)
        for a, b in zip(got, (dh, dw)):
            assert ((a.cpu().double() - factor * b).norm() <= 8e-3 * factor * b.norm() + 1e-30)
    assert not got[0][T // 8:T // 2].any()
    (only,) = torch.autograd.grad(F.lm_head_distillation(h.detach(), w, ids, teacher, chunk_rows=chunk, **kw), w)
    assert torch.equal(only, got[1] * 2)


def test_head_of_chunks_that_differ_in_size():
    """A last chunk of 6 rows has more blocks for a row than the ones before, and the vocabulary of its gradient is cut."""
    F = _ops()
    T, H, V, K = 70, 64, 20000, 5
    g = torch.Generator().manual_seed(1)
    h = torch.randn(T, H, generator=g).cuda().bfloat16().requires_grad_()
    w = (torch.randn(V, H, generator=g) / 8).cuda().bfloat16().requires_grad_()
    _, ids, teacher, labels = _batch(T, V, K, BF16)
    hd, wd = h.detach().double().cpu().requires_grad_(), w.detach().double().cpu().requires_grad_()
    z = hd @ wd.T
    want, dz, _ = oracle.distill(z, ids, teacher, 2.0, labels, 0.3)
    dh, dw = torch.autograd.grad(z, (hd, wd), dz)
    junk = [torch.full((n,), NAN, device="cuda", dtype=torch.float64) for n in (70, 140, 560) for _ in range(40)]
    del junk                                        # what the workspaces hold before
    loss = F.lm_head_distillation(h, w, ids, teacher, temperature=2.0, labels=labels, label_weight=0.3, chunk_rows=64)
    # fp32 logits: sums of 64 products in fp32, 2^-18 of numbers of up to 5, times tau^2
    assert abs(loss.item() - want) < 2.0 ** -12
    for a, b in zip(torch.autograd.grad(loss, (h, w)), (dh, dw)):
        assert (a.cpu().double() - b).norm() <= 8e-3 * b.norm()


def test_head_of_hidden_states_that_are_not_numbers_where_nothing_is_taught():
    F = _ops()
    T, H, V, K = 80, 64, 520, 4
    h = torch.randn(T, H, device="cuda").bfloat16()
    w = torch.randn(V, H, device="cuda").bfloat16().requires_grad_()
    _, ids, teacher, _ = _batch(T, V, K, BF16)      # every fourth row is without a teacher
    want = torch.autograd.grad(F.lm_head_distillation(h.requires_grad_(), w, ids, teacher), (h, w))
    h = h.detach().clone()
    h[1::4] = NAN
    h[5::8] = INF
    got = torch.autograd.grad(F.lm_head_distillation(h.requires_grad_(), w, ids, teacher), (h, w))
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_head_of_hidden_states_at_any_address():
    F = _ops()
    T, H, V, K = 40, 64, 520, 4
    g = torch.Generator().manual_seed(2)
    h = torch.randn(T, H, generator=g).cuda().bfloat16()
    w = torch.randn(V, H, generator=g).cuda().bfloat16()
    _, ids, teacher, _ = _batch(T, V, K, BF16)
    want = torch.autograd.grad(F.lm_head_distillation(h.requires_grad_(), w.requires_grad_(), ids, teacher), (h, w))
    for off in (1, 3, 4):
        there = torch.empty(T * H + off, device="cuda", dtype=BF16)[off:].view(T, H).copy_(h.detach()).requires_grad_()
        assert there.data_ptr() % 16 and there.is_contiguous()
        got = torch.autograd.grad(F.lm_head_distillation(there, w, ids, teacher), (there, w))
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    wide = torch.empty(V * H + 4, device="cuda", dtype=BF16)[4:].view(V, H).copy_(w.detach())
    with pytest.raises(ValueError, match="16 bytes"):
        F.lm_head_distillation(h, wide, ids, teacher)


@pytest.mark.parametrize("temperature,share", [(1.0, 0.0), (4.0, 0.5), (0.5, 1.0)])
def test_losses_without_gradients(temperature, share):
    F = _ops()
    T, H, V, K = 37, 64, 1032, 6
    x, ids, teacher, labels = _batch(T, V, K, F32)
    kw = dict(temperature=temperature, labels=labels, label_weight=share)
    want, _ = _loss_and_grad(x, ids, teacher, **kw)
    with torch.no_grad():
        assert torch.equal(F.distillation_loss(x.requires_grad_(), ids, teacher, **kw), want)
    h = torch.randn(T, H, device="cuda").bfloat16().requires_grad_()
    w = (torch.randn(V, H, device="cuda") / 8).bfloat16().requires_grad_()
    want = F.lm_head_distillation(h, w, ids, teacher, **kw)
    with torch.no_grad():
        got = F.lm_head_distillation(h, w, ids, teacher, **kw)
    assert torch.equal(got, want.detach()) and not got.requires_grad
    # weight or hidden states alone
    both = torch.autograd.grad(want, (h, w))
    assert torch.equal(torch.autograd.grad(F.lm_head_distillation(h, w.detach(), ids, teacher, **kw), h)[0], both[0])
    assert torch.equal(torch.autograd.grad(F.lm_head_distillation(h.detach(), w, ids, teacher, **kw), w)[0], both[1])


def test_head_writes_into_the_flat_gradient():
    F = _ops()
    T, H, V, K = 90, 128, 520, 7
    w = torch.nn.Parameter((torch.randn(V, H, device="cuda") * 0.1).bfloat16())
    w.main_grad = torch.full((V, H), 7.0, device="cuda").bfloat16()        # stale values of an earlier step
    w.grad_written = False
    total = torch.zeros(V, H, dtype=torch.float64)
    for step, n in enumerate((0, 90, 50)):
        h = torch.randn(T, H, device="cuda").bfloat16()
        _, ids, teacher, _ = _batch(T, V, K, BF16, seed=step)
        ids[n:] = -1
        F.lm_head_distillation(h, w, ids, teacher, chunk_rows=64).backward()
        assert w.grad is None and w.grad_written
        z = h.double().cpu() @ w.detach().double().cpu().T
        total += oracle.distill(z, ids, teacher)[1].T @ h.double().cpu()
    # every accumulation rounds to bf16
    assert ((w.main_grad.cpu().double() - total).norm() / total.norm()).item() < 1.5e-2
    w.grad_written = False
    F.lm_head_distillation(h[:0], w, ids[:0], teacher[:0])
    assert not w.main_grad.any()


# ---------------------------------------------------------------- verification
def _drafts(B, n, V, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    target = 4 * torch.randn(B, n + 1, V, generator=g)
    draft = target[:, :n] + 0.8 * torch.randn(B, n, V, generator=g)
    ids = torch.randint(0, V, (B, n), generator=g)
    likely = torch.rand(B, n, generator=g) < 0.85
    ids = torch.where(likely, draft.argmax(-1), ids) if n else ids
    return target.to(dtype).cuda(), ids.cuda(), draft.to(dtype).cuda(), torch.rand(B, n + 1, generator=g).cuda()


def _same(got, want):
    assert torch.equal(got.accepted.cpu(), want[0])
    assert torch.equal(got.tokens.cpu(), want[1])
    prob = got.accept_prob.cpu()
    assert torch.equal(prob.isnan(), want[2].isnan())
    # the normalisers may be sums of fp32 terms: 2^-15 as above, for both models
    # (and the chance is returned in fp32, with what is below its smallest normal number, 2^-126, flushed to zero)
    assert ((prob.double() - want[2]).nan_to_num(0.0).abs() <= 2.0 ** -14 * want[2].nan_to_num(1.0) + 2.0 ** -126).all()


@pytest.mark.parametrize("B,n,V", [(1, 0, 1), (1, 4, 7), (3, 1, 1000), (40, 3, 1025), (2, 8, 50001), (2, 2, 152064), (70, 0, 4096)])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("temperature,drafter", [(0.0, False), (1.0, False), (1.0, True), (0.6, True), (2.0, False)])
def test_verification(B, n, V, dtype, temperature, drafter):
    F = _ops()
    target, ids, draft, u = _drafts(B, n, V, dtype)
    lens = torch.arange(B, device="cuda") % (n + 2)
    draft = draft if drafter else None
    u = u if temperature else None
    for lay in ("dense", "shifted"):
        for ln in (None, lens):
            got = F.verify_drafts(_laid_out(target, lay), ids, None if draft is None else _laid_out(draft, lay), u,
                                  temperature=temperature, draft_lens=ln)
            _same(got, oracle.verify(target, ids, draft, u, temperature, ln))


@pytest.mark.parametrize("B", [1, 20, 48, 200])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("temperature", [0.0, 1.0])
def test_more_drafts_than_a_warp_has_lanes(B, dtype, temperature):
    F = _ops()
    n, V = 70, 300
    target, ids, draft, u = _drafts(B, n, V, dtype, seed=B)
    draft[::2] = target[::2, :n]                    # such drafts stand, whatever the uniforms
    if temperature == 0:
        ids[::2] = target[::2, :n].float().argmax(-1)
    ids[::2] = torch.where(torch.arange(n, device="cuda") < 20 + torch.arange(B, device="cuda")[::2, None] * 7 % 53, ids[::2], -1)
    got = (F.verify_drafts(target, ids, draft, u, temperature=temperature) if temperature else
           F.verify_drafts(target, ids, temperature=0.0))
    _same(got, oracle.verify(target, ids, draft, u, temperature) if temperature else
          oracle.verify(target, ids, None, None, 0.0))
    assert got.accepted.max() >= 20


@pytest.mark.parametrize("drafter", [False, True])
def test_a_large_batch_of_short_rows(drafter):
    F = _ops()
    target, ids, draft, u = _drafts(3000, 2, 37, F32)
    draft = draft if drafter else None
    _same(F.verify_drafts(target, ids, draft, u.double(), temperature=1.4),
          oracle.verify(target, ids, draft, u, 1.4))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_the_drawn_token_over_the_whole_range(dtype):
    """Random numbers from both ends and all over, ids in every part of the vocabulary."""
    F = _ops()
    B, V = 200, 30011
    g = torch.Generator().manual_seed(5)
    target = (1.5 * torch.randn(1, 1, V, generator=g)).to(dtype).cuda().expand(B, 1, V)
    ids = torch.empty(B, 0, dtype=torch.int64, device="cuda")
    u = torch.linspace(0, 1, B + 1, dtype=torch.float64)[:B, None]
    u[-1] = 1 - 2.0 ** -50
    u = u.cuda()
    got = F.verify_drafts(target, ids, None, u)
    p = (target[0, 0].double().cpu()).softmax(0).cumsum(0)
    want = torch.searchsorted(p / p[-1], u.cpu()[:, 0], right=True).clamp(max=V - 1)
    assert torch.equal(got.tokens[:, 0].cpu(), want)
    target, ids, draft, u = _drafts(B, 1, 3001, dtype)
    ids = torch.randint(0, 3001, (B, 1), generator=g).cuda()               # mostly rejected
    _same(F.verify_drafts(target, ids, draft, u), oracle.verify(target, ids, draft, u))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_verification_of_unusual_rows(dtype):
    F = _ops()
    V = 700
    target = torch.zeros(8, 2, V)
    target[0, 0, 300:] = -INF                       # ids without mass
    target[1, 0] = NAN
    target[2, 0] = -INF
    target[3, 1, :650] = -INF                       # few ids left
    draft = torch.zeros(8, 1, V)
    target[6, 0, 400] = 30.0                        # nearly all mass on one id
    draft[7, 0, :] = -INF
    draft[7, 0, 5] = 0.0
    ids = torch.tensor([[400], [1], [1], [2], [5], [-7], [3], [V]]).cuda()
    u = torch.tensor([[0.5, 0.999]] * 8).cuda()
    target, draft = target.to(dtype).cuda(), draft.to(dtype).cuda()
    got = F.verify_drafts(target, ids, draft, u)
    _same(got, oracle.verify(target, ids, draft, u))
    assert got.tokens[1].tolist() == [-1, -1] and got.tokens[2].tolist() == [-1, -1]
    _same(F.verify_drafts(target, ids, None, u), oracle.verify(target, ids, None, u))
    greedy = torch.zeros(4, 1, V)
    greedy[1, 0, 444] = NAN
    greedy[2, 0, 699] = INF
    greedy[3] = -INF
    none = torch.empty(4, 0, dtype=torch.int64, device="cuda")
    got = F.verify_drafts(greedy.to(dtype).cuda(), none, temperature=0.0)
    assert got.tokens[:, 0].tolist() == [0, 444, 699, 0]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("temperature", [0.0, 0.7, 1.0])
def test_verification_of_rows_far_from_zero(dtype, temperature):
    F = _ops()
    V = 3001
    low = torch.finfo(dtype).min
    g = torch.Generator().manual_seed(4)
    target = torch.randn(6, 2, V, generator=g)
    draft = target[:, :1] + torch.randn(6, 1, V, generator=g)
    target[0], draft[0, :, 5:] = low, low
    target[1, :, ::2], draft[1] = low, low
    target[2:4], draft[2:4] = 1e30 * target[2:4].round(), 1e30
    target[4:], draft[4:] = 30000.0 + 64 * target[4:].round(), 30000.0
    ids = torch.tensor([[3], [7], [9], [11], [12], [0]]).cuda()
    u = torch.tensor([[0.9, 0.3]] * 6).cuda() if temperature else None
    target, draft = target.to(dtype).cuda(), draft.to(dtype).cuda() if temperature else None
    got = F.verify_drafts(target, ids, draft, u, temperature=temperature)
    _same(got, oracle.verify(target, ids, draft, u, temperature))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("temperature", [1.0, 2.0 ** -20])
@pytest.mark.parametrize("drafter", [False, True])
def test_verification_at_every_distance_from_zero(dtype, sign, temperature, drafter):
    """Largest logits of 2^20 to 2^60 temperatures; logits a few steps of their type below, at half or twice the distance from
    zero, at zero, without mass."""
    F = _ops()
    V, exponents = 1501, range(20, 61)
    g = torch.Generator().manual_seed(8)
    n = len(exponents)
    top = torch.tensor([sign * 2.0 ** e * temperature for e in exponents]).to(dtype)
    below = [top]
    for _ in range(3):
        bits = below[-1].view(torch.int16 if dtype == BF16 else torch.int32)
        below.append((bits - int(sign)).view(dtype))
    assert all((b < a).all() for a, b in zip(below, below[1:]))
    far = torch.full_like(top, -INF)
    choice = torch.stack([*below, top * (0.5 if sign > 0 else 2), -0.25 * top if sign > 0 else 3 * top, far])   # [7, n]
    pick = torch.randint(1, 7, (n, 3, V), generator=g)
    pick[torch.rand(n, 3, V, generator=g) < 0.01] = 0
    pick[:, :, 700] = 0
    rows = choice.T[:, None].expand(n, 3, 7).gather(2, pick).cuda()
    target, draft = rows[:, :2], rows[:, 2:] if drafter else None
    ids = torch.randint(0, V, (n, 1), generator=g)
    ids[::2] = 700
    ids, u = ids.cuda(), torch.rand(n, 2, generator=g).cuda()
    got = F.verify_drafts(target, ids, draft, u, temperature=temperature)
    _same(got, oracle.verify(target, ids, draft, u, temperature))


def test_acceptance_where_sums_of_fp32_are_long():
    """So many rows that none is cut: a thread adds its part of 2^25 columns in 8192 steps, each of them lost beside a one."""
    F = _ops()
    B, V = 600, 2 ** 25
    row = torch.full((V,), -27.01 * math.log(2.0), device="cuda")
    row[:1024:4] = 0.0                              # one for each of 256 threads
    total = 256.0 + (V - 256) * 2.0 ** -27.01       # a fp32 sum may be off by half of the second term, 2^-11 of all
    u = torch.zeros(B, 2, dtype=torch.float64)
    u[:, 1] = 0.5
    u[0, 0] = (1.0 + 1e-4) / total                  # not accepted, by less than the sum's error
    got = F.verify_drafts(row.expand(B, 2, V), torch.zeros(B, 1, dtype=torch.int64, device="cuda"), None, u.cuda())
    assert got.accepted.tolist() == [0] + [1] * (B - 1)
    # half of the mass, with and without the first id, ends behind the ones at 0, 4, ... 508
    assert got.tokens[0].tolist() == [512, -1] and (got.tokens[1:].cpu() == torch.tensor([0, 512])).all()


def test_rows_behind_a_shorter_draft_are_not_read():
    F = _ops()
    target, ids, draft, u = _drafts(3, 4, 2000, BF16)
    lens = torch.tensor([0, 2, 4], device="cuda")
    want = F.verify_drafts(target, ids, draft, u, draft_lens=lens)
    for b in range(3):
        target[b, lens[b] + 1:] = NAN
        draft[b, lens[b]:] = NAN
        ids[b, lens[b]:] = 99
    got = F.verify_drafts(target, ids, draft, u, draft_lens=lens)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


# ---------------------------------------------------------------- streams, graphs, empty batches
def test_another_stream():
    F = _ops()
    side = torch.cuda.Stream()
    x, ids, teacher, _ = _batch(64, 9001, 8, BF16)
    target, dids, draft, u = _drafts(4, 3, 9001, BF16)
    want = (F.top_logits(x, 5), _loss_and_grad(x, ids, teacher), F.verify_drafts(target, dids, draft, u))
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        x2 = x + 0
        got = (F.top_logits(x2, 5), _loss_and_grad(x2, ids, teacher), F.verify_drafts(target + 0, dids, draft, u))
    side.synchronize()
    for a, b in zip(want, got):
        for p, q in zip(a, b):
            assert torch.equal(p, q)


def test_two_streams_at_once():
    F = _ops()
    batches = [(_batch(40, 50001, 8, BF16, seed=s), _drafts(3, 3, 20001, BF16, seed=s)) for s in (0, 1)]

    def work(b):
        (x, ids, teacher, _), (target, dids, draft, u) = b
        return (*F.top_logits(x, 5), *_loss_and_grad(x, ids, teacher), *F.verify_drafts(target, dids, draft, u))

    want = [work(b) for b in batches]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in batches]
    got = [[], []]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(work(batches[i]))
    torch.cuda.synchronize()
    for i in (0, 1):
        for run in got[i]:
            for a, b in zip(run, want[i]):
                assert torch.equal(a, b)


def test_teacher_student_and_draft_model_as_they_are_used():
    """The same weights on both devices: top logits, the student's step and an answer with a draft model."""
    from multimodal_training_b200.models.vlm import Qwen2_5_VLForConditionalGeneration as Model
    from test_vlm_wrapper import _batch as sample
    cpu = [Model("smoke", seed=s) for s in (3, 4)]
    gpu = [Model("smoke", seed=s).cuda().bfloat16() for s in (3, 4)]
    ids, pix, labels = sample(cpu[0].config, [(1, 16, 16)], text_len=24)
    grid = [(1, 16, 16)]
    losses = []
    for teacher, student in (cpu, gpu):
        dtype = student.model.language_model.embed_tokens.dtype
        dev = student.model.language_model.embed_tokens.device
        pix = pix.to(dtype)
        values, top = teacher.top_logits(9, ids, pix, grid)
        out = student(ids, pix, grid, labels=labels, teacher_ids=top, teacher_logits=values, temperature=2.0, label_weight=0.25)
        out["loss"].backward()
        losses.append(out["loss"].item())
        assert all(p.grad.isfinite().all() for p in student.parameters() if p.grad is not None)
        # what the operators say on this device of this device's logits
        logits = teacher(ids, pix, grid)["logits"].detach()
        assert torch.equal(logits.gather(1, top.clamp(min=0))[top[:, 0] >= 0], values[top[:, 0] >= 0])
        plain = teacher.generate(ids[0], pix, grid, max_new_tokens=6)
        with_draft = teacher.generate(ids[0], pix, grid, 6, draft_model=student, draft_tokens=3)
        drawn = teacher.generate(ids[0], pix, grid, 6, temperature=0.8, draft_model=student, draft_tokens=3,
                                 generator=torch.Generator(dev).manual_seed(0))
        assert plain.shape == with_draft.shape == drawn.shape == (ids.numel() + 6,)
        assert (drawn >= 0).all() and (drawn < teacher.config.text.vocab_size).all()
        assert dtype == (F32 if dev.type == "cpu" else BF16)
    # bf16 hidden states through a few layers: 2^-8 a rounding, a few tens of them, of logits of about one
    assert abs(losses[0] - losses[1]) < 0.1 * abs(losses[0])


def test_two_graphs_of_all_operators_replayed_in_turn():
    F = _ops()

    def work(s):
        values, ids = F.top_logits(s["teacher"], 6)
        loss = F.distillation_loss(s["x"], ids, values, temperature=2.0)
        (grad,) = torch.autograd.grad(loss * 0.5, s["x"])
        hloss = F.lm_head_distillation(s["h"], s["w"], ids, values)
        dh, dw = torch.autograd.grad(hloss * 0.5, (s["h"], s["w"]))
        r = F.verify_drafts(s["teacher"].view(10, 4, -1), s["dids"], s["x"].detach().view(10, 4, -1)[:, :3], s["u"])
        return (values, ids, loss.detach(), grad, hloss.detach(), dh, dw, *r)

    def inputs(seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        r = dict(x=torch.randn(40, 1000, generator=g, device="cuda").bfloat16().requires_grad_(),
                 teacher=torch.randn(40, 1000, generator=g, device="cuda").bfloat16(),
                 h=torch.randn(40, 64, generator=g, device="cuda").bfloat16().requires_grad_(),
                 w=torch.randn(1000, 64, generator=g, device="cuda").bfloat16().requires_grad_(),
                 dids=torch.randint(0, 1000, (10, 3), generator=g, device="cuda"),
                 u=torch.rand(10, 4, generator=g, device="cuda"))
        return r

    graphs = []
    for seed in (0, 1):
        s = inputs(seed)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            work(s)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = work(s)
        graphs.append((graph, s, out))
    for turn in range(2):
        for i, (graph, s, _) in enumerate(graphs):
            with torch.no_grad():
                for k, v in inputs(10 * turn + i + 2).items():
                    s[k].copy_(v)
            graph.replay()
        graphs[0][0].replay()                       # once more on the same inputs
        torch.cuda.synchronize()
        for graph, s, out in graphs:
            for a, b in zip(out, work(s)):
                assert torch.equal(a, b)


def test_empty_batches_and_refusals():
    F = _ops()
    x = torch.empty(0, 64, device="cuda", dtype=BF16)
    assert F.top_logits(x, 3)[1].shape == (0, 3)
    none = torch.empty(0, 2, device="cuda", dtype=torch.int64)
    r = F.verify_drafts(torch.empty(0, 3, 64, device="cuda"), none, None, torch.empty(0, 3, device="cuda"))
    assert r.accepted.shape == (0,) and r.tokens.shape == (0, 3)
    with pytest.raises(TypeError):
        F.top_logits(torch.ones(2, 9, device="cuda", dtype=torch.float16), 1)
    with pytest.raises(TypeError):
        F.distillation_loss(torch.ones(2, 9, device="cuda", dtype=torch.float64), none[:0].new_zeros(2, 1),
                            torch.zeros(2, 1, device="cuda"))
    ids = torch.zeros(2, 1, device="cuda", dtype=torch.int64)
    with pytest.raises(ValueError):
        F.distillation_loss(torch.ones(2, 9, device="cuda"), ids.cpu(), torch.zeros(2, 1, device="cuda"))
    h, w = torch.ones(2, 64, device="cuda", dtype=BF16), torch.ones(16, 64, device="cuda", dtype=BF16)
    for a, b in ((h[:, :9], w[:, :9].contiguous()), (h, w[:9]), (h[:, ::2], w[:, ::2])):
        with pytest.raises(ValueError):
            F.lm_head_distillation(a, b, ids, torch.zeros(2, 1, device="cuda"))
    with pytest.raises(TypeError):
        F.lm_head_distillation(h.float(), w.float(), ids, torch.zeros(2, 1, device="cuda"))
