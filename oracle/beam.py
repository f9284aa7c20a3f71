"""CPU restatement of beam search's step, in numpy (float64).

TEST INFRASTRUCTURE ONLY: only `tests/` may import it; the
product package never does.
"""

import numpy as np


def values(scores, totals, done=None, end=None):
    """(R, W * V): totals + log_softmax(scores), an ended beam's only value its
    total at `end`; -inf where there is no candidate."""
    x, totals = np.asarray(scores, np.float64), np.asarray(totals, np.float64)
    with np.errstate(all="ignore"):
        d = x - x.max(-1, keepdims=True)
        v = totals[..., None] + d - np.log(np.exp(d).sum(-1, keepdims=True))
    if done is not None:
        alone = np.full_like(v, -np.inf)
        alone[..., end] = totals
        v = np.where(np.asarray(done)[..., None], alone, v)
    v = np.where(np.isnan(v), -np.inf, v)
    return v.reshape(v.shape[0], -1)


def select(scores, totals, beams, done=None, end=None):
    """(totals, parents, tokens), (R, beams) each: the largest values, equal
    ones by the lowest index; -inf, -1, -1 where there are too few."""
    V = np.asarray(scores).shape[-1]
    v = values(scores, totals, done, end)
    at = np.argsort(-v, axis=1, kind="stable")[:, :beams]
    best = np.full((v.shape[0], beams), -np.inf)
    best[:, :at.shape[1]] = np.take_along_axis(v, at, 1)
    index = np.full(best.shape, -1)
    index[:, :at.shape[1]] = at
    some = best > -np.inf
    return best, np.where(some, index // V, -1), np.where(some, index % V, -1)


def reorder(table, parents, lengths, first=None):
    """A table (R * W, N, ...) with each beam's rows first .. lengths[parent] - 1
    taken from its parent."""
    old = np.asarray(table)
    new = old.copy()
    R, W = np.asarray(parents).shape
    for r in range(R):
        a = 0 if first is None else max(0, int(first[r]))
        for w in range(W):
            p = int(parents[r, w])
            if 0 <= p < W:
                n = int(lengths[r * W + p])
                new[r * W + w, a:max(a, n)] = old[r * W + p, a:max(a, n)]
    return new
