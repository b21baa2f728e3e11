"""Performance cases of the operators that work on rows of vocabulary logits with a second model beside the first: a
teacher whose top logits a student is trained on, and a target that checks what a draft model proposes.

kind        one pass
``top``     ``top_logits``: the k largest logits of every row with their ids, what a teacher hands to a student
``distill`` ``distillation_loss``: loss and gradient of the student's logits against a teacher's top logits
``head``    ``lm_head_distillation``: the same from hidden states and the head's weight, gradients of both
``verify``  ``verify_drafts``: drafted tokens accepted or replaced from given random numbers, or greedily

A case is a dict of plain values.  ``own`` chooses between elementary torch operations and the package's operators.
"""
from __future__ import annotations

import math

import torch

own = False
DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def listed() -> list[dict]:
    return [
        # a teacher answers one prompt and keeps a handful of logits of its last row: latency
        dict(name="top_one_row", kind="top", rows=1, vocab=152064, k=8, type="bf16"),
        # the teacher's pass over the benchmark's sample (1024 text and 1024 vision tokens, vocabulary of the 7B model)
        dict(name="top_sample", kind="top", rows=2048, vocab=152064, k=64, type="bf16"),
        # a teacher whose logits are kept in 32 bits, odd sizes, as many logits as the operator takes
        dict(name="top_wide_fp32", kind="top", rows=333, vocab=49999, k=256, type="fp32"),
        # the small model of the smoke runs on a short answer: launches count
        dict(name="distill_short", kind="distill", rows=37, vocab=4096, k=8, type="bf16", temperature=1.0, share=0.0),
        # a student's training step on the benchmark's sample: rows of image tokens have neither teacher nor label
        dict(name="distill_sample", kind="distill", rows=2048, vocab=152064, k=64, type="bf16", temperature=2.0, share=0.3),
        # logits in 32 bits, odd sizes, a temperature below one
        dict(name="distill_odd_fp32", kind="distill", rows=777, vocab=50001, k=17, type="fp32", temperature=0.7, share=0.0),
        # one short sample through the head of the 3B model
        dict(name="head_256", kind="head", rows=256, hidden=2048, vocab=151936, k=32, temperature=1.0, share=0.0),
        # the benchmark's sample through the head of the 7B model, a tenth of the loss from the labels
        dict(name="head_sample", kind="head", rows=2048, hidden=3584, vocab=152064, k=64, temperature=2.0, share=0.1),
        # one sequence, four drafted tokens: what an interactive answer waits for between two passes of the target
        dict(name="verify_one", kind="verify", batch=1, drafts=4, vocab=151936, type="bf16", temperature=1.0, drafter=True),
        # the same without sampling
        dict(name="verify_greedy", kind="verify", batch=1, drafts=7, vocab=152064, type="bf16", temperature=0.0,
             drafter=False),
        # a batch of an evaluation, drafts of different lengths
        dict(name="verify_batch", kind="verify", batch=48, drafts=5, vocab=152064, type="bf16", temperature=0.8,
             drafter=True),
        # drafts looked up in the prompt (no draft model), logits in 32 bits, odd sizes
        dict(name="verify_lookup_fp32", kind="verify", batch=61, drafts=3, vocab=32003, type="fp32", temperature=1.3,
             drafter=False),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    kind = rng.choice(["top", "distill", "head", "verify"])
    most = 2048 * 152064                          # elements of the largest listed case
    vocab = _log_int(rng, 1000, 152064)
    if kind == "top":
        return dict(kind=kind, rows=_log_int(rng, 1, min(4096, most // vocab)), vocab=vocab, k=_log_int(rng, 1, 256),
                    type=rng.choice(["bf16", "bf16", "fp32"]))
    if kind == "verify":
        drafts = rng.randint(0, 8)
        return dict(kind=kind, batch=_log_int(rng, 1, 64), drafts=drafts, vocab=vocab,
                    type=rng.choice(["bf16", "bf16", "fp32"]), temperature=rng.choice([0.0, 0.6, 1.0, 1.4]),
                    drafter=rng.random() < 0.6)
    more = dict(k=_log_int(rng, 1, 256), temperature=rng.choice([0.5, 1.0, 1.0, 2.0, 4.0]), share=rng.choice([0.0, 0.0, 0.5]))
    if kind == "head":
        # the framework's products want multiples of 8
        return dict(kind=kind, rows=_log_int(rng, 1, 2048), hidden=64 * rng.randint(4, 56), vocab=vocab // 8 * 8, **more)
    rows = _log_int(rng, 1, min(4096, most // vocab))
    return dict(kind=kind, rows=rows, vocab=vocab, type=rng.choice(["bf16", "bf16", "fp32"]), **more)


# --------------------------------------------------------------------------------------
# Inputs
# --------------------------------------------------------------------------------------
def _image_rows(rows: int) -> tuple[int, int]:
    """The run of rows that stand for image tokens: half of a sample, behind its first eighth."""
    return rows // 8, rows // 8 + rows // 2


def _teacher(base, case, gen):
    """Ids and logits of a teacher that agrees with `base` up to noise, labels that mostly follow it."""
    rows, vocab, k = case["rows"], case["vocab"], case["k"]
    full = base + 0.7 * torch.randn(base.shape, generator=gen, device=DEV)
    values, ids = full.topk(k, dim=1)
    short = torch.rand(rows, generator=gen, device=DEV) < 0.1          # rows of which fewer logits were kept
    ids[short, k // 2 + 1:] = -1
    labels = torch.randint(0, vocab, (rows,), generator=gen, device=DEV)
    agree = torch.rand(rows, generator=gen, device=DEV) < 0.7
    labels[agree] = ids[agree, 0]
    lo, hi = _image_rows(rows)
    ids[lo:hi] = -1
    labels[lo:hi] = -100
    return ids.contiguous(), values.contiguous(), labels


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device=DEV).manual_seed(seed)
    s = dict(case)
    if case["kind"] == "top":
        logits = 3.0 * torch.randn(case["rows"], case["vocab"], generator=gen, device=DEV)
        s["logits"] = logits.to(TYPES[case["type"]])
    elif case["kind"] == "distill":
        base = 2.5 * torch.randn(case["rows"], case["vocab"], generator=gen, device=DEV)
        s["ids"], s["teacher"], s["labels"] = _teacher(base, case, gen)
        s["logits"] = base.to(TYPES[case["type"]]).requires_grad_()
    elif case["kind"] == "head":
        hidden = torch.randn(case["rows"], case["hidden"], generator=gen, device=DEV).bfloat16()
        weight = (0.02 * torch.randn(case["vocab"], case["hidden"], generator=gen, device=DEV)).bfloat16()
        s["ids"], s["teacher"], s["labels"] = _teacher(1.5 * (hidden @ weight.T).float(), case, gen)
        s["hidden"], s["weight"] = hidden.requires_grad_(), weight.requires_grad_()
    else:
        B, n, V = case["batch"], case["drafts"], case["vocab"]
        target = 5.0 * torch.randn(B, n + 1, V, generator=gen, device=DEV)
        draft = target[:, :n] + 1.0 * torch.randn(B, n, V, generator=gen, device=DEV)
        # tokens drawn from the draft model, or the most likely ones where there is none
        race = torch.empty(B, n, V, device=DEV).exponential_(generator=gen)
        heat = case["temperature"] if case["drafter"] and case["temperature"] > 0 else 1e-3
        s["draft_ids"] = ((draft / heat).softmax(-1) / race).argmax(-1) if n else torch.zeros(B, 0, dtype=torch.int64, device=DEV)
        s["target"] = target.to(TYPES[case["type"]])
        s["draft"] = draft.to(TYPES[case["type"]]) if case["drafter"] else None
        s["uniforms"] = torch.rand(B, n + 1, generator=gen, device=DEV)
        s["lens"] = torch.tensor(_lens(case), device=DEV)
    return s


def _lens(case) -> list[int]:
    """Every third sequence of a batch has a shorter draft."""
    n = case["drafts"]
    return [n - (b // 3) % (n + 1) if b % 3 == 2 else n for b in range(case["batch"])]


# --------------------------------------------------------------------------------------
# One pass
# --------------------------------------------------------------------------------------
def run(s: dict):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    from multimodal_training_b200.ops import functional as F
    if s["kind"] == "top":
        values, ids = F.top_logits(s["logits"], s["k"])
        return dict(values=values, ids=ids)
    if s["kind"] == "verify":
        sampled = s["temperature"] > 0
        r = F.verify_drafts(s["target"], s["draft_ids"], s["draft"] if sampled else None,
                            s["uniforms"] if sampled else None, temperature=s["temperature"], draft_lens=s["lens"])
        return dict(accepted=r.accepted, tokens=r.tokens, accept_prob=r.accept_prob)
    more = dict(temperature=s["temperature"], labels=s["labels"] if s["share"] > 0 else None, label_weight=s["share"])
    if s["kind"] == "distill":
        loss = F.distillation_loss(s["logits"], s["ids"], s["teacher"], **more)
        (grad,) = torch.autograd.grad(loss, s["logits"])
        return dict(loss=loss.detach(), grad=grad)
    loss = F.lm_head_distillation(s["hidden"], s["weight"], s["ids"], s["teacher"], **more)
    dhidden, dweight = torch.autograd.grad(loss, (s["hidden"], s["weight"]))
    return dict(loss=loss.detach(), dhidden=dhidden, dweight=dweight)


def _run_plain(s):
    if s["kind"] == "top":
        return _plain_top(s["logits"], s["k"])
    if s["kind"] == "verify":
        return _plain_greedy(s) if s["temperature"] == 0 else _plain_verify(s)
    if s["kind"] == "distill":
        logits = s["logits"].detach()
        loss, grad = _plain_distill(logits.float(), s)
        return dict(loss=loss, grad=grad.to(logits.dtype))
    hidden, weight = s["hidden"].detach().float(), s["weight"].detach().float()
    loss, grad = _plain_distill(hidden @ weight.T, s)
    return dict(loss=loss, dhidden=(grad @ weight).bfloat16(), dweight=(grad.T @ hidden).bfloat16())


def _plain_top(logits, k):
    """One integer for each logit, in the logits' order and with the lower id first among equals."""
    bits = (logits.float() + 0.0).view(torch.int32).to(torch.int64)
    order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
    ids = torch.arange(logits.shape[1], device=logits.device)
    keys = (order << 32) - ids
    ids = (-keys.topk(k, dim=1).values) & 0xFFFFFFFF
    return dict(values=logits.gather(1, ids), ids=ids)


def _plain_distill(logits, s):
    """Loss and its gradient with respect to `logits` (32 bits), which may be written over."""
    heat, share = s["temperature"], s["share"]
    ids, rows = s["ids"], torch.arange(logits.shape[0], device=logits.device)
    there = ids >= 0
    z = torch.where(there, s["teacher"].double() / heat, -math.inf)
    taught = there.any(1)
    z = z - torch.where(taught, z.amax(1), 0.0)[:, None]
    e = z.exp()
    p = e / torch.where(taught, e.sum(1), 1.0)[:, None]

    def log_q(heat, at):
        """Log-probabilities of the ids `at`, and those of all ids as exp(logits / heat - offset)."""
        top = logits.amax(1)
        total = ((logits - top[:, None]) / heat).exp().sum(1, dtype=torch.float64)
        z = (logits.gather(1, at).double() - top.double()[:, None]) / heat
        return z - total.log()[:, None], top.double() / heat + total.log()

    at = ids.clamp(min=0)
    lq, norm = log_q(heat, at)
    each = torch.where(p > 0, p * (p.clamp(min=1e-300).log() - lq), 0.0).sum(1)
    n = taught.sum().clamp(min=1)
    loss = (1 - share) * heat ** 2 * each.sum() / n
    scale = (1 - share) * heat * taught.float() / n
    grad = (logits / heat - norm.float()[:, None]).exp() * scale[:, None]
    grad.scatter_add_(1, at, -(p * scale[:, None]).float())
    if share > 0:
        labelled = s["labels"] >= 0
        at = s["labels"].clamp(min=0)[:, None]
        lq, norm = log_q(1.0, at)
        n = labelled.sum().clamp(min=1)
        loss = loss - share * torch.where(labelled, lq[:, 0], 0.0).sum() / n
        scale = share * labelled.float() / n
        grad += (logits - norm.float()[:, None]).exp() * scale[:, None]
        grad[rows, at[:, 0]] -= scale
    return loss.float(), grad


def _plain_greedy(s):
    target, n = s["target"], s["drafts"]
    V = target.shape[-1]
    ids = torch.arange(V, device=target.device)
    best = target.amax(-1, keepdim=True)
    choice = torch.where(target == best, ids, V).amin(-1)              # [B, n + 1], the lowest id among equals
    spot = torch.arange(n, device=target.device)
    match = (s["draft_ids"] == choice[:, :n]) & (spot < s["lens"][:, None])
    return _plain_tokens(s, match, match.float(), lambda a: choice.gather(1, a[:, None])[:, 0])


def _plain_tokens(s, match, prob, draw):
    B, n = match.shape
    accepted = match.long().cumprod(1).sum(1)
    place = torch.arange(n + 1, device=match.device)
    tokens = torch.where(place < accepted[:, None], torch.nn.functional.pad(s["draft_ids"], (0, 1)), -1)
    tokens = torch.where(place == accepted[:, None], draw(accepted)[:, None], tokens)
    return dict(accepted=accepted, tokens=tokens, accept_prob=prob)


def _plain_verify(s):
    """In 64 bits: a drawn token depends on a sum over the vocabulary that ends next to a border."""
    heat, n = s["temperature"], s["drafts"]
    target, lens, u = s["target"], s["lens"], s["uniforms"].double()
    B, _, V = target.shape
    rows = torch.arange(B, device=target.device)

    def prob(logits):
        z = logits.double() / heat
        e = (z - z.amax(-1, keepdim=True)).exp()
        return e / e.sum(-1, keepdim=True)

    p = prob(target)
    q = prob(s["draft"]) if s["drafter"] else None
    at = s["draft_ids"][..., None]
    px = p[:, :n].gather(2, at)[..., 0]
    qx = q.gather(2, at)[..., 0] if s["drafter"] else torch.ones_like(px)
    inside = torch.arange(n, device=target.device) < lens[:, None]
    match = (u[:, :n] * qx < px) & inside
    ratio = torch.where(inside, (px / qx).clamp(max=1.0), 0.0).float()

    def draw(a):
        pa = p[rows, a]
        rejected = (a < lens)[:, None]
        spot = a.clamp(max=max(n - 1, 0))
        if n == 0:
            qa = torch.zeros_like(pa)
        elif s["drafter"]:
            qa = q[rows, spot]
        else:
            qa = torch.zeros_like(pa).scatter_(1, s["draft_ids"][rows, spot][:, None], 1.0)
        rest = torch.where(rejected, (pa - qa).clamp(min=0.0), pa)
        rest = torch.where(rest.sum(1, keepdim=True) > 0, rest, pa)
        up_to = rest.cumsum(1)
        first = (up_to <= u[:, n:] * up_to[:, -1:]).sum(1)
        last = torch.where(rest > 0, torch.arange(V, device=rest.device), 0).amax(1)
        return torch.minimum(first, last)

    return _plain_tokens(s, match, ratio, draw)


# --------------------------------------------------------------------------------------
# What a pass cannot do without, and its outputs in 64 bits
# --------------------------------------------------------------------------------------
def work(case: dict) -> dict:
    V, size = case["vocab"], 4 if case.get("type") == "fp32" else 2
    if case["kind"] == "top":
        rows, k = case["rows"], case["k"]
        return dict(bytes=rows * V * size + rows * k * (size + 8), flops=rows * V)
    if case["kind"] == "verify":
        B, n, sampled = case["batch"], case["drafts"], case["temperature"] > 0
        drafted = sum(_lens(case))
        rows = drafted + B + (drafted if sampled and case["drafter"] else 0)
        return dict(bytes=rows * V * size + B * (n * 24 + 32), flops=rows * V * (3 if sampled else 1))
    lo, hi = _image_rows(case["rows"])
    rows, taught = case["rows"], case["rows"] - (hi - lo)
    small = taught * case["k"] * 12 + rows * 8
    if case["kind"] == "distill":
        return dict(bytes=(taught + rows) * V * size + small, flops=taught * V * 8)
    H = case["hidden"]
    return dict(bytes=2 * (2 * V * H + (taught + rows) * H) + small, flops=6 * taught * V * H)


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if case["kind"] == "top":
        x = s["logits"].double()
        values, ids = x.sort(dim=1, descending=True, stable=True)
        return dict(values=values[:, :case["k"]], ids=None)
    if case["kind"] == "verify":
        return dict(accepted=None, tokens=None, accept_prob=_exact_accept(s))
    if case["kind"] == "distill":
        x = s["logits"].detach().double().requires_grad_()
        loss = _exact_loss(x, s)
        return dict(loss=loss.detach(), grad=torch.autograd.grad(loss, x)[0])
    h, w = (s[k].detach().double().requires_grad_() for k in ("hidden", "weight"))
    loss = _exact_loss(h @ w.T, s)
    dh, dw = torch.autograd.grad(loss, (h, w))
    return dict(loss=loss.detach(), dhidden=dh, dweight=dw)


def _exact_loss(x, s):
    """Kullback-Leibler divergence over the kept logits of the teacher times the temperature squared, mean over the rows
    with a teacher, and the labels' cross-entropy, mean over the rows with a label."""
    heat, share = s["temperature"], s["share"]
    rows = (s["ids"] >= 0).any(1).nonzero()[:, 0]
    total = x.sum() * 0.0
    if len(rows):
        ids = s["ids"][rows]
        log_p = (s["teacher"][rows].double() / heat).masked_fill(ids < 0, -math.inf).log_softmax(1)
        log_q = (x[rows] / heat).log_softmax(1).gather(1, ids.clamp(min=0))
        terms = (log_p.exp() * (log_p - log_q)).masked_fill(ids < 0, 0.0)
        total = total + (1 - share) * heat ** 2 * terms.sum() / len(rows)
    if share > 0:
        rows = (s["labels"] >= 0).nonzero()[:, 0]
        if len(rows):
            total = total - share * x[rows].log_softmax(1)[torch.arange(len(rows), device=x.device), s["labels"][rows]].mean()
    return total


def _exact_accept(s):
    n = s["drafts"]
    prob = torch.zeros(s["batch"], n, dtype=torch.float64, device=DEV)
    for b, length in enumerate(s["lens"].tolist()):
        for i in range(length):
            x = int(s["draft_ids"][b, i])
            row = s["target"][b, i].double()
            if s["temperature"] == 0:
                prob[b, i] = float(int(row.argmax()) == x and bool((row[:x] < row[x]).all()))
                continue
            gain = (row / s["temperature"]).log_softmax(0)[x]
            if s["drafter"]:
                gain = gain - (s["draft"][b, i].double() / s["temperature"]).log_softmax(0)[x]
            prob[b, i] = gain.clamp(max=0.0).exp()
    return prob
