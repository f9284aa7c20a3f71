"""The cache operators' boundary without a GPU: the C entry points check their
arguments on the host before any device call, the Python functions refuse CPU
tensors, and the float64 restatements that the GPU tests compare with agree
with the definitions worked out by loops."""

import math

import numpy as np
import pytest
import torch

from oracle import beam as obeam
from oracle import budget as obudget


@pytest.fixture(scope="module")
def lib():
    from wpt_b200 import _lib, build
    build.build()
    return _lib


def _weights(lib, B=1, T=1, H=1, C=128, N=1, window=0, ld=1, scratch=None):
    return lib.lib().wpt_attn_weights(None, None, 0, 128, None, None, None, None, ld, scratch, B, T, H, C, N, window, 1.0,
                                      None)


def test_attn_weights_arguments(lib):
    assert _weights(lib, C=96) == lib.ERR_UNSUPPORTED
    assert _weights(lib, T=1 << 20, H=1 << 12) == lib.ERR_UNSUPPORTED
    assert _weights(lib, window=-1) == lib.ERR_INVALID
    assert _weights(lib, H=0) == lib.ERR_INVALID
    assert _weights(lib) == lib.ERR_INVALID  # NULL pointers
    for empty in (dict(B=0), dict(T=0), dict(N=0)):
        assert _weights(lib, **empty) == lib.OK
    size = lib.lib().wpt_attn_weights_scratch_bytes
    assert size(4, 16, 16, 1000) == 0 and size(4, 17, 16, 1000) > 0 and size(0, 1, 1, 1) == 0


def _evict(lib, B=1, N=8, row_bytes=16, keep=4, recent=0, first=0, capacity=4):
    return lib.lib().wpt_cache_evict(None, 0, 0, None, N, None, None, None, None, None, B, N, row_bytes, keep, recent,
                                     first, capacity, None)


def test_cache_evict_arguments(lib):
    for bad in (dict(keep=-1), dict(capacity=3), dict(recent=3, first=2), dict(N=-1), dict(first=-1)):
        assert _evict(lib, **bad) == lib.ERR_INVALID
    assert _evict(lib, row_bytes=6) == lib.ERR_UNSUPPORTED
    assert _evict(lib) == lib.ERR_INVALID  # NULL pointers
    assert _evict(lib, B=0) == lib.OK


def _select(lib, R=1, W=1, V=8, K=1, end=0):
    return lib.lib().wpt_beam_select(None, 0, 8, 8, None, None, end, None, None, None, None, R, W, V, K, None)


def test_beam_select_arguments(lib):
    assert _select(lib, W=65) == lib.ERR_UNSUPPORTED and _select(lib, K=65) == lib.ERR_UNSUPPORTED
    assert _select(lib, W=64, V=1 << 27) == lib.ERR_UNSUPPORTED
    for bad in (dict(W=0), dict(V=0), dict(K=0), dict(R=-1)):
        assert _select(lib, **bad) == lib.ERR_INVALID
    assert _select(lib) == lib.ERR_INVALID  # NULL pointers
    assert _select(lib, R=0) == lib.OK


def test_cache_reorder_arguments(lib):
    call = lib.lib().wpt_cache_reorder
    assert call(None, 1, None, None, None, 1, 65, None) == lib.ERR_UNSUPPORTED
    assert call(None, 33, None, None, None, 1, 2, None) == lib.ERR_UNSUPPORTED
    assert call(None, -1, None, None, None, 1, 2, None) == lib.ERR_INVALID
    assert call(None, 1, None, None, None, 1, 2, None) == lib.ERR_INVALID  # NULL pointers
    assert call(None, 0, None, None, None, 1, 2, None) == lib.OK


def test_cpu_tensors_are_refused():
    import wpt_b200
    f, i = torch.zeros, torch.int64
    with pytest.raises(ValueError, match="CUDA"):
        wpt_b200.attention_weights(f(1, 1, 2, 128).bfloat16(), f(1, 4, 128).bfloat16(), f(1, 1, dtype=i), f(1, 1, 2), 1.0)
    with pytest.raises(ValueError, match="CUDA"):
        wpt_b200.cache_evict(f(1, 4, 8), f(1, 4), f(1, dtype=i), 2)
    with pytest.raises(ValueError, match="CUDA"):
        wpt_b200.beam_select(f(1, 2, 8), f(1, 2), 2)
    with pytest.raises(ValueError, match="CUDA"):
        wpt_b200.cache_reorder(f(2, 4, 8), f(1, 2, dtype=i), f(2, dtype=i))


def test_weights_restatement():
    rng = np.random.default_rng(0)
    B, T, H, C, N, window = 2, 3, 2, 4, 7, 3
    q, k = rng.normal(size=(B, T, H, C)), rng.normal(size=(B, N, C))
    positions, floor = rng.integers(-1, N + 2, (B, T)), rng.integers(-2, 4, (B, T))
    lse = obudget.log_sums(q, k, positions, 0.5, window, floor)
    got = obudget.attention_weights(q, k, positions, lse, 0.5, np.zeros((B, N)), window, floor)
    want = np.zeros((B, N))
    for b in range(B):
        for t in range(T):
            p = int(positions[b, t])
            rows = range(max(0, p - window + 1, int(floor[b, t])), min(p, N - 1) + 1)
            for h in range(H):
                s = [math.exp(0.5 * q[b, t, h] @ k[b, n]) for n in rows]
                for n, x in zip(rows, s):
                    want[b, n] += x / sum(s)
    assert np.abs(got - want).max() < 1e-12


def test_evict_restatement():
    weights = np.array([[5, 1, np.nan, 1, -0.0, 0.0, 7, 1, 2, 0]], np.float32)
    held = np.arange(10).reshape(1, 10, 1)
    out, w, rows, counts = obudget.evict(held, weights, [9], 6, recent=1, first=1, capacity=7)
    assert rows.tolist() == [[0, 1, 3, 6, 7, 8]] and counts.tolist() == [6]
    assert out[0, :, 0].tolist() == [0, 1, 3, 6, 7, 8, 0] and w[0, 6] == 0
    assert obudget.evict(held, weights, [9], 7, recent=1, first=1)[2].tolist() == [[0, 1, 3, 4, 6, 7, 8]]  # -0 ties 0
    assert obudget.evict(held, weights, [3], 6)[2].tolist() == [[0, 1, 2, -1, -1, -1]]


def test_select_and_reorder_restatements():
    x = np.zeros((1, 2, 3))
    best, parents, tokens = obeam.select(x, [[0.0, 0.0]], 4)
    assert np.allclose(best, -math.log(3)) and parents.tolist() == [[0, 0, 0, 1]] and tokens.tolist() == [[0, 1, 2, 0]]
    best, parents, tokens = obeam.select(x, [[-9.0, -0.5]], 5, done=[[False, True]], end=2)
    assert parents.tolist() == [[1, 0, 0, 0, -1]] and tokens.tolist() == [[2, 0, 1, 2, -1]] and best[0, 0] == -0.5
    t = np.arange(2 * 4).reshape(2, 4)
    assert obeam.reorder(t, np.array([[1, 0]]), [4, 3], [1]).tolist() == [[0, 5, 6, 3], [4, 1, 2, 3]]
