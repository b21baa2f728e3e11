"""Operators on rows of vocabulary logits with a second model beside the first.

* :func:`top_logits`: the k largest logits of every row with their ids, what a teacher hands to a student;
* :func:`distillation_loss` and :func:`lm_head_distillation`: a student's loss against them, with its gradient;
* :func:`verify_drafts`: what a target model accepts of the tokens that a draft model proposes.

They are reached through :mod:`.functional`, next to the cross-entropy, and follow its rules: CUDA tensors run the kernels
of ``csrc/top_logits.cu``, ``csrc/distill.cu`` and ``csrc/verify.cu`` (logits in bf16 or fp32) on the current stream, CPU
tensors of any float dtype run plain PyTorch, which is the oracle of the tests.
"""
from __future__ import annotations

import ctypes
import functools
import math
import struct
from typing import NamedTuple

import torch

from . import native as nv

MAX_TOP = 256          # most logits of a row that a teacher keeps

_KERNEL_TYPES = (torch.bfloat16, torch.float32)


# --------------------------------------------------------------------------------------
# What the operators check alike
# --------------------------------------------------------------------------------------
def _on_gpu(logits: torch.Tensor, *others: torch.Tensor | None) -> bool:
    """Whether the kernels run; refuses tensors that they cannot take."""
    for t in others:
        if t is not None and t.device != logits.device:
            raise ValueError(f"tensors on {logits.device} and {t.device}")
    if not logits.is_cuda:
        return False
    if logits.dtype not in _KERNEL_TYPES:
        raise TypeError(f"the sm_100a path takes bf16 or fp32 logits, got {logits.dtype}")
    here = torch.cuda.current_device()
    if logits.device.index != here:
        raise ValueError(f"tensors on {logits.device}, but this process drives cuda:{here}")
    return True


def _floating(t: torch.Tensor, name: str) -> None:
    if not t.is_floating_point():
        raise TypeError(f"{name} must be floating point, got {t.dtype}")


def _integral(t: torch.Tensor, name: str) -> None:
    if t.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"{name} must be int64 or int32, got {t.dtype}")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """[..., V] as [rows, V] with dense columns (a view where the strides allow it)."""
    t = t.reshape(-1, t.shape[-1]) if t.dim() != 2 else t
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _ld(t: torch.Tensor) -> int:
    """Elements between two rows."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _ids64(t: torch.Tensor) -> torch.Tensor:
    return t if t.dtype == torch.int64 else t.to(torch.int64)


def _vocab(logits: torch.Tensor, name: str = "logits") -> int:
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"{name} need a vocabulary, got shape {tuple(logits.shape)}")
    if logits.shape[-1] >= 2 ** 30:
        raise ValueError(f"a vocabulary of {logits.shape[-1]} is too large")
    return logits.shape[-1]


def _multi(group) -> bool:
    return group is not None and torch.distributed.get_world_size(group) > 1


@functools.lru_cache(maxsize=None)
def _same_layout(entry: str, size: int) -> None:
    """The library takes the layout of a call's words on trust, so it has to agree on their size before the first call."""
    n = getattr(nv.lib(), entry)()
    if n != size:
        raise RuntimeError(f"{entry}: the kernel library has {n} bytes, this module {size}: rebuild it with "
                           "`python -m multimodal_training_b200.csrc.build`")


# --------------------------------------------------------------------------------------
# Top logits
# --------------------------------------------------------------------------------------
nv.declare("mmt_top_logits", nv.c_int, [nv._P, nv.c_int, nv._P, nv._P, nv.c_long, nv.c_int, nv.c_long, nv.c_int, nv.c_long,
                                        nv._P])


@torch.no_grad()
def _top_reference(logits: torch.Tensor, k: int) -> tuple[torch.Tensor, torch.Tensor]:
    values, ids = torch.sort(logits, dim=1, descending=True, stable=True)
    return values[:, :k].contiguous(), ids[:, :k].contiguous()


def _top_rows(logits: torch.Tensor, k: int, vocab_lo: int) -> tuple[torch.Tensor, torch.Tensor]:
    if not _on_gpu(logits):
        values, ids = _top_reference(logits, k)
        return values, ids + vocab_lo
    rows, V = logits.shape
    values = torch.empty(rows, k, device=logits.device, dtype=logits.dtype)
    ids = torch.empty(rows, k, device=logits.device, dtype=torch.int64)
    if rows:
        nv.call("mmt_top_logits", logits.data_ptr(), int(logits.dtype == torch.float32), values.data_ptr(), ids.data_ptr(),
                rows, V, _ld(logits), k, vocab_lo, nv.stream())
    return values, ids


def top_logits(logits: torch.Tensor, k: int, *, vocab_lo: int = 0, group=None) -> tuple[torch.Tensor, torch.Tensor]:
    """The ``k`` largest logits of every row of [..., V], largest first, and their ids: ``(values, ids)``, both [..., k].

    Equal logits go by the lower id, NaN counts as larger than everything.  ``values`` have the logits' dtype, ``ids`` are
    int64; neither takes part in autograd.  1 <= k <= 256.  With a group, ``logits`` are this rank's shard of the
    vocabulary, which starts at ``vocab_lo`` (ascending with the rank), and every rank gets the whole vocabulary's answer.
    """
    V = _vocab(logits)
    _floating(logits, "logits")
    world = torch.distributed.get_world_size(group) if _multi(group) else 1
    if not 1 <= k <= min(MAX_TOP, V * world):
        raise ValueError(f"k = {k} is not between 1 and {min(MAX_TOP, V * world)}")
    lead = logits.shape[:-1]
    values, ids = _top_rows(_rows(logits), min(k, V), vocab_lo)
    if world > 1:
        # every rank's largest, in the order of the ranks and so of the ids among equals
        parts_v = [torch.empty_like(values) for _ in range(world)]
        parts_i = [torch.empty_like(ids) for _ in range(world)]
        torch.distributed.all_gather(parts_v, values, group=group)
        torch.distributed.all_gather(parts_i, ids, group=group)
        values, at = _top_rows(torch.cat(parts_v, 1), k, 0)
        ids = torch.cat(parts_i, 1).gather(1, at)
    return (values, ids) if logits.dim() == 2 else (values.view(*lead, k), ids.view(*lead, k))


# --------------------------------------------------------------------------------------
# Distillation
# --------------------------------------------------------------------------------------
class _DistillWords(ctypes.Structure):
    _fields_ = [("logits", ctypes.c_void_p), ("out", ctypes.c_void_p), ("ld", ctypes.c_long), ("out_ld", ctypes.c_long),
                ("vocab_lo", ctypes.c_long), ("rows", ctypes.c_long), ("places", ctypes.c_long), ("src", ctypes.c_void_p),
                ("cnt", ctypes.c_void_p), ("slot_id", ctypes.c_void_p), ("slot_p", ctypes.c_void_p),
                ("info", ctypes.c_void_p), ("mark", ctypes.c_void_p), ("counts", ctypes.c_void_p),
                ("stats", ctypes.c_void_p), ("ticket", ctypes.c_void_p), ("dloss", ctypes.c_void_p),
                ("temperature", ctypes.c_double), ("share", ctypes.c_double), ("V", ctypes.c_int), ("K", ctypes.c_int),
                ("is_f32", ctypes.c_int), ("out_f32", ctypes.c_int), ("parts", ctypes.c_int)]


nv.declare("mmt_distill_bytes", nv.c_int, [])
nv.declare("mmt_distill_count_rows", nv.c_int, [])
nv.declare("mmt_distill_stats_count", nv.c_int, [])
nv.declare("mmt_distill_prepare", nv.c_int, [nv._P, nv._P, nv.c_long, nv._P, nv.c_long, nv.c_int, nv._P, nv.c_long, nv._P,
                                             nv._P])
nv.declare("mmt_distill_stats", nv.c_int, [nv._P, nv._P])
nv.declare("mmt_distill_grad", nv.c_int, [nv._P, nv._P])
nv.declare("mmt_distill_fused", nv.c_int, [nv._P, nv._P])
nv.declare("mmt_distill_fused_columns", nv.c_long, [nv.c_int])
nv.declare("mmt_distill_loss", nv.c_int, [nv._P, nv._P, nv._P])
nv.declare("mmt_gemm_split", nv.c_int, [nv.c_int, nv.c_int, nv.c_int])
nv.declare("mmt_gemm_bf16_split", nv.c_int, [nv._P, nv._P, nv._P, nv.c_int, nv.c_int, nv.c_int, nv.c_int, nv.c_int, nv._P,
                                             nv.c_int, nv._P])
nv.declare("mmt_sum_runs", nv.c_int, [nv._P, nv.c_int, nv._P, nv.c_int, nv.c_int, nv._P, nv._P])
nv.declare("mmt_distill_scale", nv.c_int, [nv._P, nv.c_int, nv.c_long, nv._P, nv._P])


class _Distill:
    """The native side of one batch: the teacher's slots, the statistics of the rows and the words of the calls."""

    def __init__(self, teacher_ids, teacher_logits, labels, temperature, share, vocab_lo, vocab_total, is_f32, V,
                 need: torch.Tensor | None = None):
        _same_layout("mmt_distill_bytes", ctypes.sizeof(_DistillWords))
        rows, K = teacher_ids.shape
        lib = nv.lib()
        per, n_stats = lib.mmt_distill_count_rows(), lib.mmt_distill_stats_count()
        n_counts = (rows + per - 1) // per
        # one workspace, 16-byte words first: info, statistics, pairs of counts, tickets, ids and probabilities, marks
        n_slots = rows * (K + 1)
        self.n_stats = n_stats * rows
        at_counts = self.n_stats + 2 * rows
        words = at_counts + n_counts + 1
        self.work = torch.empty(words + n_slots + (rows + 1) // 2, device=teacher_ids.device, dtype=torch.float64)
        at = self.work.data_ptr()
        w = self.words = _DistillWords(rows=rows, vocab_lo=vocab_lo, temperature=temperature, share=share, V=V, K=K,
                                       is_f32=int(is_f32), info=at, stats=at + 16 * rows, counts=at + 8 * at_counts,
                                       ticket=at + 8 * (words - 1), slot_id=at + 8 * words,
                                       slot_p=at + 8 * words + 4 * n_slots, mark=at + 8 * (words + n_slots))
        if rows:
            nv.call("mmt_distill_prepare", ctypes.addressof(w), teacher_ids.data_ptr(), _ld(teacher_ids),
                    teacher_logits.data_ptr(), _ld(teacher_logits), int(teacher_logits.dtype == torch.float32),
                    nv.ptr(labels), vocab_total, nv.ptr(need), nv.stream())

    @property
    def stats(self) -> torch.Tensor:
        rows = self.words.rows
        return self.work[2 * rows:2 * rows + self.n_stats].view(nv.lib().mmt_distill_stats_count(), rows)

    def _rows(self, logits, src, cnt):
        w = self.words
        w.logits, w.ld, w.places = logits.data_ptr(), _ld(logits), logits.shape[0]
        w.src, w.cnt = nv.ptr(src), nv.ptr(cnt)

    def row_stats(self, logits, src=None, cnt=None) -> None:
        self._rows(logits, src, cnt)
        if logits.shape[0]:
            nv.call("mmt_distill_stats", ctypes.addressof(self.words), nv.stream())

    def reduce(self, lo: int, hi: int, group) -> None:
        """Statistics of rows [lo, hi) over the shards of the vocabulary."""
        from . import functional as F
        stats = self.stats
        top = stats[:2, lo:hi].contiguous()
        mine = top.clone()
        F._all_reduce(top, torch.distributed.ReduceOp.MAX, group)
        rest = stats[2:8, lo:hi].contiguous()
        sums, label, dot, mass, has_label = rest[:2], rest[2], rest[3], rest[4], rest[5]
        # from below this shard's largest logit to below the whole vocabulary's; a shard of nothing but -inf has a sum of
        # zero, which stays
        down = mine - top
        sums.copy_(torch.where(sums > 0, sums * torch.exp2(down), sums))
        label.add_(torch.where(has_label > 0, down[1], 0.0))
        dot.add_(torch.where(mass > 0, mass * down[0], 0.0))
        F._all_reduce(rest, torch.distributed.ReduceOp.SUM, group)
        stats[:2, lo:hi] = top
        stats[2:8, lo:hi] = rest

    def _out(self, out, dloss=None) -> None:
        w = self.words
        w.out, w.out_ld, w.dloss = nv.ptr(out), 0 if out is None else _ld(out), nv.ptr(dloss)
        w.out_f32 = int(out is not None and out.dtype == torch.float32)

    def both(self, logits, out, src=None, cnt=None, dloss=None) -> None:
        """Statistics of a whole vocabulary and (unless ``out`` is None) the gradient."""
        w = self.words
        if w.V > nv.lib().mmt_distill_fused_columns(w.is_f32):
            self.row_stats(logits, src, cnt)
            if out is not None:
                self.grad(logits, out, src, cnt, dloss)
            return
        self._rows(logits, src, cnt)
        self._out(out, dloss)
        if logits.shape[0]:
            nv.call("mmt_distill_fused", ctypes.addressof(w), nv.stream())

    def grad(self, logits, out, src=None, cnt=None, dloss=None) -> None:
        self._rows(logits, src, cnt)
        self._out(out, dloss)
        w = self.words
        if logits.shape[0]:
            nv.call("mmt_distill_grad", ctypes.addressof(w), nv.stream())

    def loss(self) -> torch.Tensor:
        out = torch.empty((), device=self.work.device, dtype=torch.float32)
        nv.call("mmt_distill_loss", ctypes.addressof(self.words), out.data_ptr(), nv.stream())
        return out


def _captured_with_forward(ctx) -> None:
    """What an eager forward pass keeps is freed behind its backward pass, so that a replay would read anything."""
    if torch.cuda.is_current_stream_capturing() and not ctx.captured:
        raise RuntimeError("this backward pass is being captured into a graph, its forward pass was not: capture both")


class _DistillFn(torch.autograd.Function):
    """The gradient is written in forward, while the row's statistics are at hand, and handed over by the first backward
    pass (times its ``dloss``, where that is not one: a bf16 gradient is then rounded a second time, unless the factor is a
    power of two).  Another backward pass, and one that is captured into a graph (a replay would scale once more), form it
    again from the logits, with the factor in front of the one rounding.

    2048 x 152064 bf16, two softmaxes: 202 us, 454 with a factor of 1/3."""

    @staticmethod
    def forward(ctx, logits, teacher_ids, teacher_logits, labels, temperature, share, vocab_lo, group):
        rows, V = logits.shape
        world = torch.distributed.get_world_size(group) if _multi(group) else 1
        d = _Distill(teacher_ids, teacher_logits, labels, temperature, share, vocab_lo, V * world,
                     logits.dtype == torch.float32, V)
        ctx.early = None
        if ctx.needs_input_grad[0]:
            if not torch.cuda.is_current_stream_capturing():
                ctx.early = torch.empty(rows, V, device=logits.device, dtype=logits.dtype)
            ctx.save_for_backward(logits, d.work)
            ctx.d, ctx.world, ctx.captured = d, world, torch.cuda.is_current_stream_capturing()
        if world > 1:
            d.row_stats(logits)
            d.reduce(0, rows, group)
            if ctx.early is not None:
                d.grad(logits, ctx.early)
        else:
            d.both(logits, ctx.early)
        return d.loss()

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dloss):
        _captured_with_forward(ctx)
        dloss = dloss.to(torch.float32)
        early, ctx.early = ctx.early, None
        if early is not None and not torch.cuda.is_current_stream_capturing():
            nv.call("mmt_distill_scale", early.data_ptr(), int(early.dtype == torch.float32), early.numel(),
                    dloss.data_ptr(), nv.stream())
            grad = early
        else:
            logits = ctx.saved_tensors[0]
            grad = torch.empty(logits.shape, device=logits.device, dtype=logits.dtype)
            (ctx.d.grad if ctx.world > 1 else ctx.d.both)(logits, grad, dloss=dloss)
        return (grad,) + (None,) * 7


# Temperatures beyond these are mistakes (of units, or a zero that was to mean greedy), and keep log2(e) / temperature and the
# squares of both far from the ends of fp32.
_COLDEST, _HOTTEST = 2.0 ** -20, 2.0 ** 20


def _check_distill(shape, device, teacher_ids, teacher_logits, temperature, labels, label_weight):
    """Teacher and labels as the kernels take them: [rows, K] twice, [rows] or None."""
    if teacher_ids.shape != teacher_logits.shape or teacher_ids.dim() < 1 or teacher_ids.shape[:-1] != shape:
        raise ValueError(f"teacher_ids {tuple(teacher_ids.shape)} and teacher_logits {tuple(teacher_logits.shape)} must both "
                         f"be [*{tuple(shape)}, k]")
    K = teacher_ids.shape[-1]
    if not 1 <= K <= MAX_TOP:
        raise ValueError(f"a teacher keeps between 1 and {MAX_TOP} logits of a row, got {K}")
    _integral(teacher_ids, "teacher_ids")
    _floating(teacher_logits, "teacher_logits")
    if teacher_logits.requires_grad:
        raise ValueError("teacher_logits are data of the loss: detach them")
    if not _COLDEST <= temperature <= _HOTTEST:
        raise ValueError(f"temperature must be positive, from 2^-20 to 2^20, got {temperature}")
    if not 0.0 <= label_weight <= 1.0:
        raise ValueError(f"label_weight must be in [0, 1], got {label_weight}")
    if label_weight > 0.0 and labels is None:
        raise ValueError("label_weight > 0 needs labels")
    if labels is not None:
        if labels.shape != shape:
            raise ValueError(f"labels {tuple(labels.shape)} must be {tuple(shape)}")
        _integral(labels, "labels")
        if labels.device != device:
            raise ValueError(f"tensors on {device} and {labels.device}")
    ids = _rows(_ids64(teacher_ids))
    if teacher_logits.dtype not in _KERNEL_TYPES and teacher_logits.is_cuda:
        teacher_logits = teacher_logits.float()
    labels = None if label_weight == 0.0 else _ids64(labels.reshape(-1)).contiguous()
    return ids, _rows(teacher_logits), labels


def _check_shard(V, vocab_lo, group):
    """The shard's place in a vocabulary of as many equal ones as the group has ranks."""
    world = torch.distributed.get_world_size(group) if _multi(group) else 1
    if not 0 <= vocab_lo <= V * (world - 1):
        raise ValueError(f"vocab_lo = {vocab_lo}: {world} shard(s) of {V} ids start between 0 and {V * (world - 1)}")


def _distill_reference(logits, ids, teacher, labels, temperature, share, vocab_lo, group):
    """Plain PyTorch, differentiable; fp32 or the logits' wider type."""
    from ..parallel.comm import all_reduce_sum_autograd
    from . import functional as F
    V = logits.shape[1]
    vocab = V * (torch.distributed.get_world_size(group) if _multi(group) else 1)
    for t, name in ((ids, "teacher_ids"), (labels, "labels")):
        if t is not None and t.numel() and int(t.max()) >= vocab:
            raise ValueError(f"{name} hold {int(t.max())}, the vocabulary ends at {vocab}")
    wide = torch.float64 if logits.dtype == torch.float64 else torch.float32

    def total(t):
        return all_reduce_sum_autograd(t, group) if _multi(group) else t

    def picked(x, at):
        local = at - vocab_lo
        mine = (local >= 0) & (local < V) & (at >= 0)
        return total(torch.where(mine, x.gather(1, local.clamp(0, V - 1)), torch.zeros((), dtype=x.dtype)))

    def log_q(x, at):
        top = x.detach().amax(1)
        if _multi(group):
            F._all_reduce(top, torch.distributed.ReduceOp.MAX, group)
        x = x - top[:, None]
        return picked(x, at) - total(x.exp().sum(1)).log()[:, None]

    loss = logits.sum() * 0.0 if logits.shape[0] == 0 else torch.zeros((), dtype=wide)
    here = (ids >= 0) & (teacher != -math.inf)
    rows = here.any(1).nonzero()[:, 0]
    if rows.numel() and share < 1.0:
        z = (teacher[rows].to(wide) / temperature).masked_fill(~here[rows], -math.inf)
        log_p = z.log_softmax(1)
        p = log_p.exp()
        lq = log_q(logits[rows].to(wide) / temperature, ids[rows])
        terms = torch.where(p == 0, torch.zeros((), dtype=wide), p * (log_p - lq))
        loss = loss + (1.0 - share) * temperature ** 2 * terms.sum() / rows.numel()
    if share > 0.0:
        rows = (labels >= 0).nonzero()[:, 0]
        if rows.numel():
            loss = loss - share * log_q(logits[rows].to(wide), labels[rows][:, None]).sum() / rows.numel()
    if not loss.requires_grad and logits.requires_grad:
        loss = loss + (logits.narrow(0, 0, 0).sum() if logits.shape[0] else logits.sum())
    return loss


def distillation_loss(logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_logits: torch.Tensor, *,
                      temperature: float = 1.0, labels: torch.Tensor | None = None, label_weight: float = 0.0,
                      vocab_lo: int = 0, group=None) -> torch.Tensor:
    """Loss of a student's ``logits`` [..., V] against the top logits of a teacher (:func:`top_logits`).

    With p = softmax over the kept entries of ``teacher_logits / temperature`` and q = softmax over the vocabulary of
    ``logits / temperature``: the divergence sum_j p_j (log p_j - log q_{id_j}) times ``temperature ** 2``, mean over the
    rows that have a teacher.  ``teacher_ids`` and ``teacher_logits`` are [..., k], k <= 256; an entry is absent if its id
    is negative or its logit -inf, and a row whose entries are all absent (image tokens, padding) has no loss and a zero
    gradient, whatever its logits hold.  An id that is given more than once counts with each of its entries.

    ``label_weight`` = a in [0, 1]: (1 - a) times the above plus a times the cross-entropy with ``labels`` [...] (at
    temperature one, mean over the rows whose label is not negative).

    The result is an fp32 scalar, differentiable with respect to ``logits`` only.  On the GPU an id outside the vocabulary
    is left out and reported through the device error word, sums over the vocabulary and the teacher's probabilities are
    fp32, ``teacher_logits`` of other types than bf16 and fp32 are rounded to fp32, and a gradient in bf16 is rounded once
    when it is formed and once more by a factor of the loss that is no power of two.  With a group, ``logits`` are this rank's shard of the
    vocabulary, one of as many equal ones as there are ranks, starting at ``vocab_lo``, as in
    :func:`.functional.lm_head_cross_entropy`; without one, ``vocab_lo`` is 0.
    """
    V = _vocab(logits)
    _floating(logits, "logits")
    _check_shard(V, vocab_lo, group)
    gpu = _on_gpu(logits, teacher_ids, teacher_logits, labels)
    ids, teacher, labels = _check_distill(logits.shape[:-1], logits.device, teacher_ids, teacher_logits, temperature, labels,
                                          label_weight)
    rows = logits if logits.dim() == 2 else logits.reshape(-1, V)
    if not gpu:
        return _distill_reference(rows, ids, teacher, labels, temperature, label_weight, vocab_lo, group)
    return _DistillFn.apply(_rows(rows), ids, teacher, labels, float(temperature), float(label_weight), vocab_lo, group)


def _gemm_over_vocab(grad, weight, out, count) -> None:
    """``out[r] = grad[r] @ weight`` for as many rows as ``count[0]``.  A few rows have few tiles, each with the whole
    vocabulary as its K: then the vocabulary is cut into runs, whose fp32 results are added up."""
    from . import functional as F
    rows, V = grad.shape
    H = weight.shape[1]
    runs = nv.lib().mmt_gemm_split(rows, H, V)
    if runs < 2:
        F._gemm_counted(grad, weight, out, count, b_mn=True)
        return
    parts = torch.empty(runs, rows, H, device=grad.device, dtype=torch.float32)
    nv.call("mmt_gemm_bf16_split", grad.data_ptr(), weight.data_ptr(), parts.data_ptr(), rows, H, V, grad.stride(0),
            weight.stride(0), count.data_ptr(), runs, nv.stream())
    nv.call("mmt_sum_runs", parts.data_ptr(), runs, count.data_ptr(), rows, H, out.data_ptr(), nv.stream())


def _head_pass(hidden, weight, teacher, temperature, share, vocab_lo, group, chunk_rows, need_h, dw, add):
    """Loss, and the gradient of ``hidden`` (if ``need_h``) and of ``weight`` (into ``dw``, on top of it if ``add``).

    As in the head's cross-entropy, the logits of a chunk of rows and their gradient live in workspaces only, and rows
    without a teacher or label are left out of the products in groups of 16.  The logits stay fp32: rounded to bf16 they
    would move a row's loss by 2^-9 of their size, where the divergence is what is left of numbers of that size.  (They are
    sums of the tensor cores, which round towards zero: 1e-6 of their size too small for each 1000 of H, and the loss off by
    2e-7 to 4e-6 of itself, where fp32 sums that round to nearest leave about 1e-7.)

    Their gradient is rounded to bf16 once, for the tensor cores, as in the head's cross-entropy.  The gradients of hidden
    states and weight are then off by 0.0020 to 0.0033 of their norm, most where one teacher's logit or label is nearly all of
    a row; of fp32 products 0.0017 is left by the rounding of the result.  The part that is lost could only be had by the two
    products over again with what the rounding leaves."""
    from . import functional as F
    T, V = hidden.shape[0], weight.shape[0]
    dev = hidden.device
    world = torch.distributed.get_world_size(group) if _multi(group) else 1
    need = torch.empty(T, device=dev, dtype=torch.int64)
    d = _Distill(*teacher, temperature, share, vocab_lo, V * world, True, V, need)
    if T == 0:
        if dw is not None and not add:
            dw.zero_()
        return d.loss(), torch.empty_like(hidden) if need_h else None
    chunk_rows = min(chunk_rows, T)
    src, lab, pos = torch.empty(3, T, device=dev, dtype=torch.int64)
    count = torch.empty((T + chunk_rows - 1) // chunk_rows, device=dev, dtype=torch.int32)
    nv.call("mmt_compact_labels", need.data_ptr(), T, chunk_rows, src.data_ptr(), lab.data_ptr(), pos.data_ptr(),
            count.data_ptr(), nv.stream())
    # `lab` is `src` less the rows without either inside a group that is kept: what they hold stays out of the products
    x = F.gather_rows_raw(hidden, lab)
    dx = torch.empty_like(hidden) if need_h else None
    ws = torch.empty(chunk_rows, V, device=dev, dtype=torch.float32)
    gs = torch.empty(chunk_rows, V, device=dev, dtype=torch.bfloat16) if need_h or dw is not None else None
    for i, c0 in enumerate(range(0, T, chunk_rows)):
        c1 = min(T, c0 + chunk_rows)
        h, logits, n = x[c0:c1], ws[:c1 - c0], count[i:]
        grad = None if gs is None else gs[:c1 - c0]
        F._gemm_counted(h, weight, logits, n)
        if world > 1:
            d.row_stats(logits, src[c0:], n)
            d.reduce(c0, c1, group)
            if grad is not None:
                d.grad(logits, grad, src[c0:], n)
        else:
            d.both(logits, grad, src[c0:], n)
        if need_h:
            _gemm_over_vocab(grad, weight, dx[c0:c1], n)
        if dw is not None:
            F._gemm_counted(grad, h, dw, n, of_k=True, a_mn=True, b_mn=True, accumulate=add or c0 > 0)
    return d.loss(), F.gather_rows_raw(dx, pos) if need_h else None


class _LMHeadDistillFn(torch.autograd.Function):
    """Both gradients are produced in forward and handed over by the first backward pass, times its ``dloss`` (which rounds
    them once more, unless it is a power of two); another one runs the products again.  In a captured graph they stay as
    forward left them, for the next replay."""

    @staticmethod
    def forward(ctx, hidden, weight, teacher_ids, teacher_logits, labels, *call):
        need_h, need_w = ctx.needs_input_grad[:2]
        mg = getattr(weight, "main_grad", None) if need_w else None
        dw, add = None, False
        if mg is not None:
            dw, add = mg, bool(getattr(weight, "grad_written", False))
        elif need_w:
            dw = torch.empty_like(weight)
        teacher = (teacher_ids, teacher_logits, labels)
        loss, dh = _head_pass(hidden, weight, teacher, *call, need_h, dw, add)
        if mg is not None:
            weight.grad_written = True
        ctx.grads = (dh, dw if mg is None else None)
        ctx.need = (need_h, need_w and mg is None)
        ctx.call, ctx.captured = call, torch.cuda.is_current_stream_capturing()
        ctx.save_for_backward(hidden, weight, *teacher)
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dloss):
        _captured_with_forward(ctx)
        grads = ctx.grads
        if ctx.captured:
            grads = [None if g is None else g.clone() for g in grads]
        elif grads is None:
            hidden, weight, *teacher = ctx.saved_tensors
            need_h, need_w = ctx.need
            dw = torch.empty_like(weight) if need_w else None
            grads = (_head_pass(hidden, weight, teacher, *ctx.call, need_h, dw, False)[1], dw)
        if not ctx.captured:
            ctx.grads = None
        dloss = dloss.to(torch.float32)
        for g in grads:
            if g is not None:
                nv.call("mmt_distill_scale", g.data_ptr(), 0, g.numel(), dloss.data_ptr(), nv.stream())
        return (*grads,) + (None,) * (3 + len(ctx.call))


def lm_head_distillation(hidden: torch.Tensor, weight: torch.Tensor, teacher_ids: torch.Tensor,
                         teacher_logits: torch.Tensor, *, temperature: float = 1.0, labels: torch.Tensor | None = None,
                         label_weight: float = 0.0, vocab_lo: int = 0, group=None, chunk_rows: int = 4096) -> torch.Tensor:
    """:func:`distillation_loss` of ``hidden @ weight^T`` without keeping the logits: ``hidden`` is [T, H], ``weight`` this
    rank's [V_local, H] shard of the head, teacher and labels are those of the T rows.

    On the GPU path hidden states and weight are bf16, H and V_local multiples of 8, the weight starts at a multiple of 16
    bytes, and its gradient assumes ``dloss == 1`` when it is written into ``main_grad``, as in
    :func:`.functional.lm_head_cross_entropy`.  The workspaces hold ``chunk_rows`` rows of fp32 logits and of their gradient in
    bf16: 6 bytes a logit, 3.7 GB for 4096 rows of 152064, three times what the cross-entropy takes.
    """
    if hidden.dim() != 2 or weight.dim() != 2 or hidden.shape[1] != weight.shape[1]:
        raise ValueError(f"hidden {tuple(hidden.shape)} and weight {tuple(weight.shape)} must be [T, H] and [V, H]")
    if weight.shape[0] < 1 or chunk_rows < 1:
        raise ValueError("the head needs a vocabulary and chunks of at least one row")
    if hidden.dtype != weight.dtype:
        raise TypeError(f"hidden is {hidden.dtype}, weight {weight.dtype}")
    _floating(hidden, "hidden")
    _check_shard(weight.shape[0], vocab_lo, group)
    from . import functional as F
    gpu = _on_gpu(hidden, weight, teacher_ids, teacher_logits, labels)
    ids, teacher, labels = _check_distill(hidden.shape[:1], hidden.device, teacher_ids, teacher_logits, temperature, labels,
                                          label_weight)
    if not gpu:
        logits = torch.nn.functional.linear(hidden, weight)
        return _distill_reference(logits, ids, teacher, labels, temperature, label_weight, vocab_lo, group)
    F._native(hidden)
    if hidden.shape[1] % 8 or weight.shape[0] % 8 or not weight.is_contiguous() or weight.data_ptr() % 16:
        raise ValueError(f"the sm_100a path needs a contiguous weight of multiples of 8 that starts at a multiple of 16 bytes, "
                         f"got {tuple(weight.shape)}")
    hidden = F._c(hidden)
    if hidden.data_ptr() % 16:                     # rows are read in 16-byte vectors
        hidden = hidden.clone()
    return _LMHeadDistillFn.apply(hidden, weight, ids, teacher, labels, float(temperature), float(label_weight),
                                  vocab_lo, group, chunk_rows)


# --------------------------------------------------------------------------------------
# Verification of drafted tokens
# --------------------------------------------------------------------------------------
class Verified(NamedTuple):
    """What the target makes of a batch of drafts."""

    accepted: torch.Tensor       # [B] int64: drafted tokens that stand
    tokens: torch.Tensor         # [B, n + 1] int64: those, the token that follows them, then -1
    accept_prob: torch.Tensor    # [B, n] fp32: min(1, p / q) of every drafted token, 0 behind a sequence's last; on the
    #                              GPU of fp32 sums over the vocabulary


_VERIFY_WORDS = struct.Struct("@2P4l7Pd8i")


nv.declare("mmt_verify_bytes", nv.c_int, [])
nv.declare("mmt_verify_splits", nv.c_int, [nv.c_long, nv.c_int, nv.c_int])
nv.declare("mmt_verify_drafts", nv.c_int, [nv._P, nv._P])


@torch.no_grad()
def _verify_reference(target, draft_ids, draft, uniforms, temperature, lens) -> Verified:
    """Plain PyTorch, in fp64."""
    B, m, V = target.shape
    n, dev = m - 1, target.device
    rows = torch.arange(B, device=dev)
    inside = torch.arange(n, device=dev) < lens[:, None]
    known = (draft_ids >= 0) & (draft_ids < V)
    at = draft_ids.clamp(0, V - 1)

    def finish(ok, prob, draw):
        accepted = (ok & inside).long().cumprod(1).sum(1)
        place = torch.arange(m, device=dev)
        ids = torch.nn.functional.pad(draft_ids, (0, 1))
        tokens = torch.where(place < accepted[:, None], ids, torch.full_like(ids, -1))
        tokens[rows, accepted] = draw(accepted)
        return Verified(accepted, tokens, torch.where(inside, prob, torch.zeros_like(prob)).float())

    if temperature == 0.0:
        order = target.double().masked_fill(target.isnan(), math.inf)
        # NaN above +inf: a row with NaN is decided among its NaN alone
        has = target.isnan().any(-1, keepdim=True)
        best = torch.where(has, target.isnan(), order == order.amax(-1, keepdim=True))
        choice = torch.where(best, torch.arange(V, device=dev), V).amin(-1)
        ok = draft_ids == choice[:, :n]
        return finish(ok, ok.double(), lambda a: choice[rows, a])

    def prob(t):
        z = t.double()
        e = ((z - z.amax(-1, keepdim=True)) / temperature).exp()
        return e / e.sum(-1, keepdim=True)

    p = prob(target)
    q = None if draft is None else prob(draft)
    px = torch.where(known, p[:, :n].gather(2, at[..., None])[..., 0], torch.zeros((), dtype=p.dtype, device=dev))
    qx = torch.ones_like(px)
    if q is not None:
        qx = torch.where(known, q.gather(2, at[..., None])[..., 0], torch.zeros_like(px))
    u = uniforms.double()
    ratio = torch.where(px > 0, torch.where(px >= qx, torch.ones_like(px), px / qx), px * 0.0)

    def draw(a):
        w = p[rows, a]
        if n:
            spot = a.clamp(max=n - 1)
            if q is not None:
                qa = q[rows, spot]
            else:
                qa = torch.zeros_like(w).scatter_(1, at[rows, spot][:, None], known[rows, spot].double()[:, None])
            rest = (w - qa).clamp(min=0.0)
            least = 0.0 if q is None else 2.0 ** -46      # of p that is q but for its rounding
            w = torch.where((a < lens)[:, None] & (rest.sum(1, keepdim=True) > least), rest, w)
        sums = w.cumsum(1)
        goal = u[:, n:] * sums[:, -1:]
        first = (sums <= goal).sum(1)
        last = torch.where(w > 0, torch.arange(V, device=dev), -1).amax(1)
        return torch.where(sums[:, -1] > 0, torch.minimum(first, last), torch.full_like(last, -1))

    return finish(u[:, :n] * qx < px, ratio, draw)


def verify_drafts(target_logits: torch.Tensor, draft_ids: torch.Tensor, draft_logits: torch.Tensor | None = None,
                  uniforms: torch.Tensor | None = None, *, temperature: float = 1.0,
                  draft_lens: torch.Tensor | None = None) -> Verified:
    """What a target model accepts of drafted tokens, and the token that follows them.

    ``draft_ids`` [B, n] are the drafts of B sequences (n may be 0: the next token is drawn from the target), of which
    sequence b has the first ``draft_lens[b]`` (default n).  ``target_logits`` [B, n + 1, V]: row i holds the logits behind
    which draft i was proposed, row ``draft_lens[b]`` those behind the last draft; later rows are not read.
    ``draft_logits`` [B, n, V] are what the drafts were drawn from; None: tokens that were looked up or chosen, all of
    whose probability counts as theirs.  ``uniforms`` [B, n + 1] (fp32 or fp64, in [0, 1)) are the random numbers: column i
    accepts draft i if ``u q(x) < p(x)`` with p, q = softmax(logits / temperature), the last column draws the next token
    from ``max(p - q, 0)`` at the first rejected place (from p if that has no mass beyond rounding), or from the target's
    row behind the last draft.  The tokens then have the target's own distribution.

    ``temperature == 0``: greedy, without ``draft_logits`` and ``uniforms``: a draft stands while it is the id of the
    largest logit (lowest id among equals, NaN above everything), which is also the next token.

    A drafted id outside the vocabulary is rejected.  A target row that is no distribution (NaN, all -inf) accepts nothing
    and draws -1.  Acceptance and the drawn token are those of fp64 probabilities and sums, so they do not depend on how the
    vocabulary is cut.
    """
    if target_logits.dim() != 3 or draft_ids.dim() != 2:
        raise ValueError(f"target_logits {tuple(target_logits.shape)} and draft_ids {tuple(draft_ids.shape)} must be "
                         "[B, n + 1, V] and [B, n]")
    V = _vocab(target_logits, "target_logits")
    B, n = draft_ids.shape
    if target_logits.shape[:2] != (B, n + 1):
        raise ValueError(f"target_logits {tuple(target_logits.shape)} do not have a row more than draft_ids ({B}, {n})")
    _floating(target_logits, "target_logits")
    _integral(draft_ids, "draft_ids")
    if not (temperature == 0.0 or _COLDEST <= temperature <= _HOTTEST):
        raise ValueError(f"temperature must be 0 (greedy) or from 2^-20 to 2^20, got {temperature}")
    if temperature == 0.0:
        if draft_logits is not None or uniforms is not None:
            raise ValueError("temperature 0 takes neither draft_logits nor uniforms")
    else:
        if uniforms is None or uniforms.shape != (B, n + 1):
            raise ValueError(f"uniforms must be [{B}, {n + 1}]")
        if uniforms.dtype not in (torch.float32, torch.float64):
            raise TypeError(f"uniforms must be fp32 or fp64, got {uniforms.dtype}")
        if draft_logits is not None:
            if draft_logits.shape != (B, n, V):
                raise ValueError(f"draft_logits {tuple(draft_logits.shape)} must be {(B, n, V)}")
            if draft_logits.dtype != target_logits.dtype:
                raise TypeError(f"draft_logits are {draft_logits.dtype}, target_logits {target_logits.dtype}")
    if draft_lens is not None:
        _integral(draft_lens, "draft_lens")
        if draft_lens.shape != (B,):
            raise ValueError(f"draft_lens {tuple(draft_lens.shape)} must be ({B},)")
    if B > 65535 or n > 32767:
        raise ValueError(f"at most 65535 sequences and 32767 drafts, got {B} and {n}")
    gpu = _on_gpu(target_logits, draft_ids, draft_logits, uniforms, draft_lens)
    draft_ids = _ids64(draft_ids).contiguous()
    lens = None if draft_lens is None else _ids64(draft_lens).contiguous()
    if not gpu:
        lens = torch.full((B,), n, dtype=torch.int64) if lens is None else lens.clamp(0, n)
        return _verify_reference(target_logits, draft_ids, draft_logits, uniforms, temperature, lens)
    _same_layout("mmt_verify_bytes", _VERIFY_WORDS.size)
    dev = target_logits.device
    target = target_logits if target_logits.stride(2) == 1 or V == 1 else target_logits.contiguous()
    draft = draft_logits
    if draft is not None and draft.stride(2) != 1 and V > 1:
        draft = draft.contiguous()
    if draft is not None and n == 0:
        draft = None
    uniforms = None if uniforms is None else uniforms.contiguous()
    accepted = torch.empty(B, device=dev, dtype=torch.int64)
    tokens = torch.empty(B, n + 1, device=dev, dtype=torch.int64)
    prob = torch.empty(B, n, device=dev, dtype=torch.float32)
    if B:
        rows, is_f32 = n + 1 + (n if draft is not None else 0), int(target.dtype == torch.float32)
        splits = nv.lib().mmt_verify_splits(B * rows, V, is_f32)
        parts = torch.empty(B * rows * splits, device=dev, dtype=torch.int64)
        # the words of the call in the order of Verify in csrc/verify.cu; a packed string costs a fifth of a ctypes structure
        words = _VERIFY_WORDS.pack(
            target.data_ptr(), 0 if draft is None else draft.data_ptr(), target.stride(0), target.stride(1),
            0 if draft is None else draft.stride(0), 0 if draft is None else draft.stride(1), draft_ids.data_ptr(),
            0 if uniforms is None else uniforms.data_ptr(), 0 if lens is None else lens.data_ptr(), accepted.data_ptr(),
            tokens.data_ptr(), prob.data_ptr(), parts.data_ptr(), 1.0 / temperature if temperature else 0.0, B, n, V, is_f32,
            int(uniforms is not None and uniforms.dtype == torch.float64), int(temperature > 0.0), rows, splits)
        nv.call("mmt_verify_drafts", words, nv.stream())
        nv.launch_count += 1                       # rows, then sequences
    return Verified(accepted, tokens, prob)
