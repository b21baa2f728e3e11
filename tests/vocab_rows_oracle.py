"""Plain 64-bit statements of the operators on vocabulary rows, row by row, for the tests."""
import math

import numpy as np
import torch


def top(logits, k):
    """Descending, equal values by the lower id, NaN first."""
    x = logits.detach().double().cpu().numpy()
    x = x.reshape(-1, x.shape[-1])
    ids = np.empty((x.shape[0], k), np.int64)
    for r, row in enumerate(x):
        key = np.where(np.isnan(row), np.inf, row)
        ids[r] = np.lexsort((np.arange(row.size), -key, ~np.isnan(row)))[:k]
    ids = torch.from_numpy(ids).reshape(*logits.shape[:-1], k)
    return logits.detach().cpu().gather(-1, ids), ids


def distill(logits, ids, teacher, temperature=1.0, labels=None, share=0.0):
    """(loss, gradient, size of the gradient's two parts before they cancel), all fp64."""
    x = logits.detach().double().cpu()
    x = x.reshape(-1, x.shape[-1])
    ids = ids.cpu().reshape(x.shape[0], -1)
    t = teacher.detach().double().cpu().reshape(ids.shape) / temperature
    here = (ids >= 0) & (t != -math.inf)
    taught = here.any(1)
    labels = torch.full((x.shape[0],), -1) if labels is None else labels.cpu().reshape(-1)
    labelled = (labels >= 0) & (share > 0)
    loss, grad, size = 0.0, torch.zeros_like(x), torch.zeros_like(x)
    wt, wl = (1 - share) / max(int(taught.sum()), 1), share / max(int(labelled.sum()), 1)
    for r in range(x.shape[0]):
        if taught[r]:
            at = ids[r][here[r]]
            log_p = t[r][here[r]].log_softmax(0)
            log_q = (x[r] / temperature).log_softmax(0)
            p = log_p.exp()
            terms = torch.where(p > 0, p * (log_p - log_q[at]), torch.zeros_like(p))
            if not p.isnan().any():
                loss = loss + wt * temperature ** 2 * float(terms.sum()) if share < 1 else loss
            else:
                loss = math.nan
            grad[r] += wt * temperature * log_q.exp()
            size[r] += wt * temperature * log_q.exp()
            grad[r].index_add_(0, at, -wt * temperature * p)
            size[r].index_add_(0, at, wt * temperature * p)
        if labelled[r]:
            log_q = x[r].log_softmax(0)
            loss = loss - wl * float(log_q[labels[r]])
            grad[r] += wl * log_q.exp()
            size[r] += wl * log_q.exp()
            grad[r, labels[r]] -= wl
            size[r, labels[r]] += wl
    return loss, grad.reshape(logits.shape), size.reshape(logits.shape)


def verify(target, draft_ids, draft=None, uniforms=None, temperature=1.0, lens=None):
    """(accepted, tokens, accept_prob) from loops over sequences and places."""
    target = target.detach().double().cpu().numpy()
    draft = None if draft is None else draft.detach().double().cpu().numpy()
    draft_ids = draft_ids.cpu().numpy()
    u = None if uniforms is None else uniforms.double().cpu().numpy()
    B, m, V = target.shape
    n = m - 1
    accepted = np.zeros(B, np.int64)
    tokens = np.full((B, m), -1, np.int64)
    prob = np.zeros((B, n), np.float64)

    def softmax(row):
        with np.errstate(invalid="ignore", over="ignore"):
            e = np.exp((row - row.max()) / temperature)
            return e / e.sum()

    def largest(row):
        return int(np.flatnonzero(np.isnan(row))[0]) if np.isnan(row).any() else int(np.flatnonzero(row == row.max())[0])

    for b in range(B):
        length = n if lens is None else min(max(int(lens[b]), 0), n)
        stop = length
        for i in range(length):
            x = int(draft_ids[b, i])
            if temperature == 0:
                ok = largest(target[b, i]) == x
                prob[b, i] = float(ok)
            else:
                known = 0 <= x < V
                p = softmax(target[b, i])[x] if known else 0.0
                q = 1.0 if draft is None else softmax(draft[b, i])[x] if known else 0.0
                ok = u[b, i] * q < p
                prob[b, i] = np.nan if np.isnan(p) else 0.0 if p == 0 else 1.0 if p >= q else p / q
            if not ok:
                stop = min(stop, i)
        accepted[b] = stop
        tokens[b, :stop] = draft_ids[b, :stop]
        if temperature == 0:
            tokens[b, stop] = largest(target[b, stop])
            continue
        p = softmax(target[b, stop])
        w = p
        if stop < length:
            x = int(draft_ids[b, stop])
            q = np.zeros(V)
            if draft is not None:
                q = softmax(draft[b, stop])
            elif 0 <= x < V:
                q[x] = 1.0
            rest = np.maximum(p - q, 0.0)
            w = rest if rest.sum() > 0 else p
        sums = np.cumsum(w)
        if sums[-1] > 0:
            above = np.flatnonzero(sums > u[b, n] * sums[-1])
            tokens[b, stop] = above[0] if above.size else np.flatnonzero(w > 0)[-1]
    return torch.from_numpy(accepted), torch.from_numpy(tokens), torch.from_numpy(prob)
