"""Top logits, distillation and draft verification on CPU: explicit formulas, differences, refusals, shards of the
vocabulary on gloo ranks."""
import math

import pytest
import torch

import vocab_rows_oracle as oracle
from dist_utils import run_ranks
from multimodal_training_b200.ops import functional as F

INF, NAN = math.inf, math.nan


# ---------------------------------------------------------------- top logits
@pytest.mark.parametrize("V,k", [(1, 1), (7, 7), (50, 3), (300, 256)])
def test_top_logits_orders_ties_by_id(V, k):
    g = torch.Generator().manual_seed(V)
    x = torch.randint(-3, 4, (5, V), generator=g).float()
    x[1] = 0.0
    x[2, ::2] = -0.0
    x[3, V // 2] = NAN
    x[4, V // 3] = INF
    x[4, 0] = -INF
    values, ids = F.top_logits(x, k)
    want_v, want_i = oracle.top(x, k)
    assert torch.equal(ids, want_i) and torch.equal(values.isnan(), want_v.isnan())
    assert torch.equal(values.nan_to_num(9.0), want_v.nan_to_num(9.0))


def test_top_logits_keeps_leading_dimensions_and_dtype():
    x = torch.randn(2, 3, 40, dtype=torch.bfloat16, requires_grad=True)
    values, ids = F.top_logits(x, 4)
    assert values.shape == ids.shape == (2, 3, 4) and values.dtype == torch.bfloat16 and not values.requires_grad
    assert torch.equal(x.gather(2, ids), values)
    values, ids = F.top_logits(torch.empty(0, 9), 2)
    assert values.shape == (0, 2)
    values, ids = F.top_logits(torch.tensor([1.0, 3.0, 2.0]), 2)
    assert ids.tolist() == [1, 2]


def test_top_logits_refusals():
    x = torch.randn(2, 9)
    for k in (0, -1, 10):
        with pytest.raises(ValueError):
            F.top_logits(x, k)
    with pytest.raises(ValueError):
        F.top_logits(torch.randn(1, 500), 257)
    with pytest.raises(ValueError):
        F.top_logits(torch.empty(2, 0), 1)
    with pytest.raises(TypeError):
        F.top_logits(torch.ones(2, 9, dtype=torch.int64), 1)


def _top_worker(rank, world, k):
    import torch.distributed as dist
    x = torch.randint(-4, 5, (6, 40), generator=torch.Generator().manual_seed(3)).float()
    per = 40 // world
    return F.top_logits(x[:, rank * per:(rank + 1) * per], k, vocab_lo=rank * per, group=dist.group.WORLD)


@pytest.mark.parametrize("k", [5, 33])
def test_top_logits_of_vocabulary_shards(tmp_path, k):
    x = torch.randint(-4, 5, (6, 40), generator=torch.Generator().manual_seed(3)).float()
    want_v, want_i = oracle.top(x, k)
    for values, ids in run_ranks(_top_worker, 2, tmp_path, k):
        assert torch.equal(values, want_v) and torch.equal(ids, want_i)


# ---------------------------------------------------------------- distillation
def _batch(T, V, K, seed=0, dtype=torch.float64):
    g = torch.Generator().manual_seed(seed)
    x = 2 * torch.randn(T, V, generator=g, dtype=torch.float64)
    teacher, ids = (x + torch.randn(T, V, generator=g)).topk(K, dim=1)
    ids[1::4] = -1                                  # rows without a teacher
    if K > 2:
        ids[2::4, 1] = -1                           # fewer logits
        ids[3::4, 2] = ids[3::4, 0]                 # an id twice
        teacher[0, 1] = -INF
    labels = torch.randint(0, V, (T,), generator=g)
    labels[::3] = -100
    return x.to(dtype), ids, teacher, labels


@pytest.mark.parametrize("T,V,K", [(1, 1, 1), (1, 30, 3), (9, 50, 7), (14, 33, 33)])
@pytest.mark.parametrize("temperature", [1.0, 0.5, 3.0])
@pytest.mark.parametrize("share", [0.0, 0.3, 1.0])
def test_distillation_follows_the_formula(T, V, K, temperature, share):
    x, ids, teacher, labels = _batch(T, V, K)
    x.requires_grad_()
    loss = F.distillation_loss(x, ids, teacher, temperature=temperature, labels=labels, label_weight=share)
    want, grad, _ = oracle.distill(x, ids, teacher, temperature, labels, share)
    assert abs(float(loss.detach()) - want) < 1e-12 * max(1.0, abs(want))
    (got,) = torch.autograd.grad(loss, x)
    assert (got - grad).abs().max() < 1e-13


def test_distillation_gradient_against_differences():
    x, ids, teacher, labels = _batch(6, 11, 4)
    x.requires_grad_()
    assert torch.autograd.gradcheck(lambda t: F.distillation_loss(t, ids, teacher, temperature=1.7, labels=labels,
                                                                  label_weight=0.4), x, eps=1e-6, atol=1e-8)


def test_distillation_of_rows_without_a_teacher():
    x, ids, teacher, labels = _batch(6, 11, 4)
    ids[2:4] = -1
    teacher[5] = -INF                               # ids, but no logit
    labels[2:4] = -100
    x[2:4] = NAN                                    # what such a row holds does not matter
    x.requires_grad_()
    loss = F.distillation_loss(x, ids, teacher, labels=labels, label_weight=0.5)
    (got,) = torch.autograd.grad(loss, x)
    assert math.isfinite(float(loss)) and not got[2:4].any() and got.isfinite().all()
    empty = F.distillation_loss(x, torch.full_like(ids, -1), teacher)
    assert float(empty) == 0.0
    (got,) = torch.autograd.grad(empty, x)
    assert not got.any()
    none = torch.empty(0, 11, requires_grad=True)
    loss = F.distillation_loss(none, ids[:0], teacher[:0])
    assert float(loss) == 0.0 and torch.autograd.grad(loss, none)[0].shape == (0, 11)


def test_distillation_of_itself_is_zero_and_infinite_where_the_student_has_no_mass():
    x = torch.randn(3, 8, dtype=torch.float64)
    values, ids = F.top_logits(x, 8)
    assert abs(float(F.distillation_loss(x, ids, values))) < 1e-14
    x[1, 2] = -INF
    assert float(F.distillation_loss(x, ids, values)) == INF
    values[1][ids[1] == 2] = -INF                   # nor has the teacher
    assert math.isfinite(float(F.distillation_loss(x, ids, values)))


def test_distillation_refusals():
    x, ids, teacher, labels = _batch(4, 11, 3)
    ok = dict(temperature=1.0, labels=labels, label_weight=0.5)
    F.distillation_loss(x, ids, teacher, **ok)
    for bad in (dict(ok, temperature=0.0), dict(ok, temperature=1e-7), dict(ok, temperature=2e6), dict(ok, temperature=-1.0), dict(ok, temperature=NAN), dict(ok, temperature=INF),
                dict(ok, label_weight=1.5), dict(ok, label_weight=-0.1), dict(ok, labels=None), dict(ok, labels=labels[:2])):
        with pytest.raises(ValueError):
            F.distillation_loss(x, ids, teacher, **bad)
    for i, t in ((ids[:3], teacher), (ids, teacher[:, :2]), (ids[:, :0], teacher[:, :0]),
                 (ids, teacher.clone().requires_grad_()), (ids + 11, teacher),
                 (torch.zeros(4, 257, dtype=torch.int64), torch.zeros(4, 257))):
        with pytest.raises(ValueError):
            F.distillation_loss(x, i, t)
    for i, t, lab in ((ids.float(), teacher, labels), (ids, ids, labels), (ids, teacher, labels.float())):
        with pytest.raises(TypeError):
            F.distillation_loss(x, i, t, labels=lab, label_weight=0.5)
    with pytest.raises(TypeError):
        F.distillation_loss(x.long(), ids, teacher)
    h, w = torch.randn(4, 6), torch.randn(11, 6)
    for a, b in ((h, w[:, :5]), (h[0], w), (h, w[:0])):
        with pytest.raises(ValueError):
            F.lm_head_distillation(a, b, ids, teacher)
    with pytest.raises(ValueError):
        F.lm_head_distillation(h, w, ids, teacher, chunk_rows=0)
    with pytest.raises(TypeError):
        F.lm_head_distillation(h, w.double(), ids, teacher)


def test_a_shard_of_the_vocabulary_needs_its_group():
    """Ids are those of the whole vocabulary: without the other ranks there is none that starts behind its first id."""
    x, ids, teacher, _ = _batch(4, 24, 3)
    h, w = torch.randn(4, 6), torch.randn(24, 6)
    for lo in (1, 24, -1):
        with pytest.raises(ValueError, match="vocab_lo"):
            F.distillation_loss(x, ids, teacher, vocab_lo=lo)
        with pytest.raises(ValueError, match="vocab_lo"):
            F.lm_head_distillation(h, w, ids, teacher, vocab_lo=lo)


def _shard_worker(rank, world, lo):
    import torch.distributed as dist
    x, ids, teacher, _ = _batch(4, 24, 3)
    with pytest.raises(ValueError, match="vocab_lo"):
        F.distillation_loss(x, ids, teacher, vocab_lo=lo, group=dist.group.WORLD)
    return True


@pytest.mark.parametrize("lo", [-1, 25])
def test_a_shard_lies_in_the_vocabulary(tmp_path, lo):
    assert run_ranks(_shard_worker, 2, tmp_path, lo) == [True, True]


@pytest.mark.parametrize("src,dst", [(0x1008, 0x2000), (0x1002, 0x2000), (0x1000, 0x2004)])
def test_rows_at_any_other_address_than_16_bytes_are_not_gathered(src, dst):
    """The kernel reads and writes 16 bytes at a time; nothing is launched here."""
    from multimodal_training_b200.ops import native as nv
    if not nv.available():
        pytest.skip("the kernel library is not built")
    assert nv.lib().mmt_gather_rows(src, 0x3000, dst, 1, 8, 0, 1, 8, 8, None) == -3


def test_head_and_logits_agree():
    x, ids, teacher, labels = _batch(9, 24, 5)
    h = torch.randn(9, 8, dtype=torch.float64, requires_grad=True)
    w = torch.randn(24, 8, dtype=torch.float64, requires_grad=True)
    more = dict(temperature=2.0, labels=labels, label_weight=0.25)
    a = torch.autograd.grad(F.lm_head_distillation(h, w, ids, teacher, **more), (h, w))
    b = torch.autograd.grad(F.distillation_loss(h @ w.T, ids, teacher, **more), (h, w))
    for p, q in zip(a, b):
        assert (p - q).abs().max() < 1e-14


def _distill_worker(rank, world):
    import torch.distributed as dist

    from multimodal_training_b200.parallel.comm import copy_to_group
    x, ids, teacher, labels = _batch(9, 24, 5)
    g = torch.Generator().manual_seed(1)
    h = torch.randn(9, 8, generator=g, dtype=torch.float64).requires_grad_()
    w = torch.randn(24, 8, generator=g, dtype=torch.float64)
    per = 24 // world
    w = w[rank * per:(rank + 1) * per].clone().requires_grad_()
    loss = F.lm_head_distillation(copy_to_group(h, dist.group.WORLD), w, ids, teacher, temperature=2.0, labels=labels,
                                  label_weight=0.25, vocab_lo=rank * per, group=dist.group.WORLD)
    loss.backward()
    return float(loss), h.grad, w.grad


def test_distillation_of_vocabulary_shards(tmp_path):
    res = run_ranks(_distill_worker, 2, tmp_path)
    x, ids, teacher, labels = _batch(9, 24, 5)
    g = torch.Generator().manual_seed(1)
    h = torch.randn(9, 8, generator=g, dtype=torch.float64).requires_grad_()
    w = torch.randn(24, 8, generator=g, dtype=torch.float64).requires_grad_()
    loss = F.lm_head_distillation(h, w, ids, teacher, temperature=2.0, labels=labels, label_weight=0.25)
    loss.backward()
    for r, (got, dh, dw) in enumerate(res):
        assert abs(got - float(loss)) < 1e-13
        assert (dh - h.grad).abs().max() < 1e-13 and (dw - w.grad[12 * r:12 * r + 12]).abs().max() < 1e-13


# ---------------------------------------------------------------- verification
def _drafts(B, n, V, seed=0, noise=0.7):
    g = torch.Generator().manual_seed(seed)
    target = 2 * torch.randn(B, n + 1, V, generator=g)
    draft = target[:, :n] + noise * torch.randn(B, n, V, generator=g)
    ids = torch.randint(0, V, (B, n), generator=g)
    likely = torch.rand(B, n, generator=g) < 0.8
    ids = torch.where(likely, draft.argmax(-1), ids) if n else ids
    return target, ids, draft, torch.rand(B, n + 1, generator=g)


def _same(got, want):
    assert torch.equal(got.accepted.cpu(), want[0])
    assert torch.equal(got.tokens.cpu(), want[1])
    assert torch.equal(got.accept_prob.cpu().isnan(), want[2].isnan())
    # fp64 rounded to fp32
    assert ((got.accept_prob.cpu().double() - want[2]).nan_to_num(0.0).abs() <= 2.0 ** -24 * 1.01 * want[2].nan_to_num(1.0)).all()


@pytest.mark.parametrize("B,n,V", [(1, 0, 5), (7, 1, 3), (40, 4, 50), (5, 3, 1)])
@pytest.mark.parametrize("temperature", [0.0, 0.7, 1.0])
@pytest.mark.parametrize("drafter", [False, True])
def test_verification_follows_the_loops(B, n, V, temperature, drafter):
    target, ids, draft, u = _drafts(B, n, V)
    lens = torch.arange(B) % (n + 2)
    if temperature == 0:
        _same(F.verify_drafts(target, ids, temperature=0.0, draft_lens=lens), oracle.verify(target, ids, None, None, 0.0, lens))
        return
    draft = draft if drafter else None
    _same(F.verify_drafts(target, ids, draft, u, temperature=temperature, draft_lens=lens),
          oracle.verify(target, ids, draft, u, temperature, lens))


def test_verified_tokens_have_the_targets_distribution():
    """Sum over the draft's own distribution and a grid of random numbers: the first token is distributed as the target."""
    V, N = 4, 60
    target, draft = torch.randn(1, 2, V, dtype=torch.float64), torch.randn(1, 1, V, dtype=torch.float64)
    q = draft[0, 0].softmax(0)
    grid = (torch.arange(N) + 0.5) / N
    u = torch.stack(torch.meshgrid(grid, grid, indexing="ij"), -1).reshape(-1, 2)
    mass = torch.zeros(V, dtype=torch.float64)
    for x in range(V):
        B = u.shape[0]
        r = F.verify_drafts(target.expand(B, -1, -1), torch.full((B, 1), x), draft.expand(B, -1, -1), u)
        mass += q[x] * torch.bincount(r.tokens[:, 0], minlength=V) / B
    # each border of the grid is off by at most half a step: one for the acceptance and V for the draw of each x
    assert (mass - target[0, 0].softmax(0)).abs().max() < (V + 1) * 0.5 / N


def test_verification_of_unusual_rows():
    V = 6
    target = torch.zeros(6, 2, V)
    target[0, 0, 3:] = -INF                         # ids without mass
    target[1, 0] = NAN
    target[2, 0] = -INF
    target[3, 1, :5] = -INF                         # one id left
    draft = torch.zeros(6, 1, V)
    draft[4, 0] = target[4, 0]                      # the same distribution: always accepted
    ids = torch.tensor([[4], [1], [1], [2], [5], [-7]])
    u = torch.tensor([[0.5, 0.999]] * 6)
    got = F.verify_drafts(target, ids, draft, u)
    _same(got, oracle.verify(target, ids, draft, u))
    assert got.accepted.tolist() == [0, 0, 0, 1, 1, 0]
    assert got.tokens[0].tolist() == [2, -1] and got.tokens[1].tolist() == [-1, -1] and got.tokens[3].tolist() == [2, 5]
    greedy = torch.zeros(3, 1, V)
    greedy[1, 0, 4] = NAN
    greedy[2, 0, 5] = INF
    none = torch.empty(3, 0, dtype=torch.int64)
    assert F.verify_drafts(greedy, none, temperature=0.0).tokens[:, 0].tolist() == [0, 4, 5]


def test_rows_behind_a_shorter_draft_are_not_read():
    target, ids, draft, u = _drafts(3, 4, 20)
    lens = torch.tensor([0, 2, 4])
    want = F.verify_drafts(target, ids, draft, u, draft_lens=lens)
    for b in range(3):
        target[b, lens[b] + 1:] = NAN
        draft[b, lens[b]:] = NAN
        ids[b, lens[b]:] = 99
    got = F.verify_drafts(target, ids, draft, u, draft_lens=lens)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_verification_refusals():
    target, ids, draft, u = _drafts(3, 2, 9)
    F.verify_drafts(target, ids, draft, u)
    bad = [(target[:, :2], ids, draft, u), (target[0], ids, draft, u), (target, ids[0], draft, u), (target, ids, draft[:2], u),
           (target, ids, draft, u[:, :2]), (target, ids, draft, None)]
    for args in bad:
        with pytest.raises(ValueError):
            F.verify_drafts(*args)
    for kw in (dict(temperature=-1.0), dict(temperature=1e-7), dict(temperature=2e6), dict(temperature=NAN), dict(temperature=0.0), dict(draft_lens=torch.zeros(2, dtype=torch.int64))):
        with pytest.raises(ValueError):
            F.verify_drafts(target, ids, draft, u, **kw)
    for args in ((target.long(), ids, None, u), (target, ids.float(), draft, u), (target, ids, draft.double(), u),
                 (target, ids, draft, u.half())):
        with pytest.raises(TypeError):
            F.verify_drafts(*args)
    with pytest.raises(TypeError):
        F.verify_drafts(target, ids, draft, u, draft_lens=torch.ones(3))
