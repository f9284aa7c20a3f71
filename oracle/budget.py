"""CPU restatement of eviction by accumulated attention weight, in numpy.

TEST INFRASTRUCTURE ONLY: only `tests/` may import it; the
product package never does.

attention_weights: what each row of the keys collects from a pass of queries,
the softmax weights of the rows each query reads (max(0, p - window + 1,
floor) .. min(p, N - 1)) summed over queries and heads, in float64.
evict: the rows a budget leaves, in their order.
"""

import numpy as np


def visible(positions, N, window=0, floor=None):
    """(B, T, N): whether query (b, t) at positions[b, t] reads row n."""
    p = np.asarray(positions, np.int64)[..., None]
    n = np.arange(N)
    seen = n <= p
    if window > 0:
        seen &= n > p - window
    if floor is not None:
        seen &= n >= np.asarray(floor, np.int64)[..., None]
    return seen


def attention_weights(q, k, positions, lse, scale, weights, window=0, floor=None):
    q, k, lse = (np.asarray(x, np.float64) for x in (q, k, lse))
    out = np.asarray(weights, np.float64).copy()
    seen = visible(positions, k.shape[1], window, floor)
    for b in range(q.shape[0]):
        with np.errstate(all="ignore"):
            s = np.einsum("thc,nc->thn", q[b], k[b]) * scale - lse[b][..., None]
            p = np.exp(s)
        out[b] += np.where(seen[b][:, None], p, 0.0).sum((0, 1))
    return out


def log_sums(q, k, positions, scale, window=0, floor=None, sink=None):
    """(B, T, H) float64: the forward pass's log-sum-exp (-inf for no rows)."""
    q, k = np.asarray(q, np.float64), np.asarray(k, np.float64)
    seen = visible(positions, k.shape[1], window, floor)
    out = np.full(q.shape[:3], -np.inf)
    for b in range(q.shape[0]):
        with np.errstate(all="ignore"):
            s = np.where(seen[b][:, None], np.einsum("thc,nc->thn", q[b], k[b]) * scale, -np.inf)
            m = s.max(-1)
            out[b] = np.where(np.isneginf(m), -np.inf, m + np.log(np.exp(s - m[..., None]).sum(-1)))
        if sink is not None:
            out[b] = np.logaddexp(out[b], np.asarray(sink, np.float64))
    return out


def evict(held, weights, lengths, keep, recent=0, first=0, capacity=None):
    held, weights = np.asarray(held), np.asarray(weights, np.float32)
    B, N = weights.shape
    capacity = keep if capacity is None else capacity
    out = np.zeros((B, capacity) + held.shape[2:], held.dtype)
    out_weights = np.zeros((B, capacity), np.float32)
    rows = np.full((B, keep), -1, np.int64)
    counts = np.zeros(B, np.int64)
    for b in range(B):
        n = int(np.clip(lengths[b], 0, N))
        at = np.arange(n)
        if n > keep:
            middle = np.where(np.isnan(weights[b, first:n - recent]), -np.inf, weights[b, first:n - recent])
            best = np.argsort(-middle, kind="stable")[:keep - first - recent] + first
            at = np.concatenate([at[:first], np.sort(best), at[n - recent:]])
        counts[b] = len(at)
        rows[b, :len(at)] = at
        out[b, :len(at)] = held[b, at]
        out_weights[b, :len(at)] = weights[b, at]
    return out, out_weights, rows, counts
