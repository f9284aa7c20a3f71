"""Rotary positions and the paged cache without a GPU: the C entry points check
their arguments on the host, the Python functions refuse CPU tensors, plans
cover every shape, and the float64 restatements agree with the definitions."""

import ctypes
import math

import numpy as np
import pytest
import torch

from oracle import paged as op


@pytest.fixture(scope="module")
def lib():
    from wpt_b200 import _lib, build
    build.build()
    return _lib


def _rotate(lib, B=1, T=1, H=1, C=8, dims=4, start=0, x=None, f=None):
    return lib.lib().wpt_rotate(x, 8, 8, 8, None, 0, f, 1, None, 0, B, T, H, C, dims, start, 0, 1.0, 0, None)


def test_rotate_arguments(lib):
    one = ctypes.c_void_p(16)
    for bad in (dict(dims=3), dict(dims=-2), dict(start=-1), dict(start=5), dict(dims=10), dict(C=0), dict(B=-1),
                dict(start=2 ** 31 - 2)):
        assert _rotate(lib, f=one, **bad) == lib.ERR_INVALID
    assert _rotate(lib) == lib.ERR_INVALID and _rotate(lib, f=one) == lib.ERR_INVALID  # NULL pointers
    for empty in (dict(B=0), dict(T=0), dict(H=0)):
        assert _rotate(lib, f=one, **empty) == lib.OK


def _append(lib, at=None, B=1, n=1, C=128, M=1, P=1, S=16, dims=0, start=0, stride=256, f=None):
    return lib.lib().wpt_paged_append(at, 0, 256, 256, at, 4096, stride, at, 2, at, 0, 1, at, at, None, f, 1, B, n, C, M, P,
                                      S, dims, start, 0, 1.0, None)


def test_paged_append_arguments(lib):
    one = ctypes.c_void_p(16)
    for bad in (dict(C=24), dict(C=1024), dict(S=48), dict(S=0), dict(S=192), dict(S=-16)):
        assert _append(lib, one, **bad) == lib.ERR_UNSUPPORTED
    for bad in (dict(n=-1), dict(P=-1), dict(C=0), dict(dims=2), dict(dims=130, f=one), dict(stride=240), dict(stride=264),
                dict(dims=64, start=65, f=one)):
        assert _append(lib, one, **bad) == lib.ERR_INVALID
    assert _append(lib) == lib.ERR_INVALID  # NULL pointers
    assert _append(lib, ctypes.c_void_p(24)) == lib.ERR_INVALID  # pages at 8 bytes
    for empty in (dict(B=0), dict(n=0), dict(M=0), dict(P=0)):
        assert _append(lib, **empty) == lib.OK


def _attend(lib, at=None, splits=1, ctas=1, scratch=None, B=1, T=1, H=1, C=128, M=1, P=1, S=16, window=0, stride=256):
    return lib.lib().wpt_paged_attention(at, at, 4096, stride, at, 2, at, 0, 1, at, None, at, at, scratch, splits, ctas, B,
                                         T, H, C, M, P, S, window, 1.0, None)


def test_paged_attention_arguments(lib):
    one = ctypes.c_void_p(16)
    for bad in (dict(C=64), dict(H=65), dict(H=0), dict(S=48), dict(M=1 << 27), dict(B=1 << 26, T=1 << 4, H=64),
                dict(splits=0, scratch=one, B=257), dict(splits=0, scratch=one, ctas=1 << 24)):
        assert _attend(lib, one, **bad) == lib.ERR_UNSUPPORTED, bad
    for bad in (dict(splits=9), dict(splits=-1), dict(splits=0), dict(splits=0, scratch=one, ctas=0), dict(window=-1),
                dict(stride=240), dict(stride=248), dict(B=-1)):
        assert _attend(lib, one, **bad) == lib.ERR_INVALID, bad
    assert _attend(lib) == lib.ERR_INVALID  # NULL pointers
    assert _attend(lib, ctypes.c_void_p(8)) == lib.ERR_INVALID
    for empty in (dict(B=0), dict(T=0)):
        assert _attend(lib, **empty) == lib.OK
    size = lib.lib().wpt_paged_scratch_bytes
    assert size(2, 1, 32, 0, 10) == (2 + 10) * 32 * 520 + 16 and size(1, 5, 12, 0, 3) == 6 * 32 * 520 + 24
    assert size(3, 2, 33, 0, 1) == (12 + 1) * 32 * 520 + 96  # two groups for a query's heads
    assert size(1, 1, 1, 1, 1) == 0 and size(1, 1, 65, 0, 1) == 0 and size(0, 1, 1, 0, 1) == 0


def test_cpu_tensors_are_refused():
    import wpt_b200
    z, i = torch.zeros, torch.int64
    pages, scales, table = z(1, 16, 256, dtype=torch.float8_e4m3fn), z(1, 1, 2), z(1, 1, dtype=i)
    with pytest.raises(ValueError, match="CUDA"):
        wpt_b200.rotate(z(1, 1, 8), z(1, dtype=i), z(2))
    with pytest.raises(ValueError, match="CUDA"):
        wpt_b200.paged_append(pages, scales, table, z(1, 1, 256), z(1, dtype=i), z(1, dtype=i))
    with pytest.raises(ValueError, match="CUDA"):
        wpt_b200.paged_attention(z(1, 1, 2, 128).bfloat16(), pages, scales, table, z(1, 1, dtype=i), 1.0)


def test_plans():
    """Every shape has a plan that the library takes: clusters of one wave, balanced calls of up to 256 groups, else
    whole rows."""
    from wpt_b200 import ops
    for sms in (148, 132):
        for B in (1, 2, 7, 64, 255, 256, 257, 5000):
            for T, H in ((1, 1), (1, 16), (1, 32), (1, 64), (5, 12), (64, 1), (65, 1), (300, 16)):
                for N in (16, 128, 129, 1024, 4096, 8192, 32768, 262144, 2 ** 30):
                    for window in (0, 1, 128, 1024):
                        splits, ctas = ops._paged_plan_for(B, T, H, N, window, sms)
                        ncol = 16 if T * H <= 16 else 32
                        groups, slots = B * (math.ceil(T / (ncol // H)) if H <= 32 else 2 * T), 2 * sms
                        assert 0 <= splits <= 8
                        if splits > 1:
                            assert groups * splits <= slots
                        if splits == 0:
                            assert groups <= 256 and 1 <= ctas <= slots and groups * (math.ceil(N / 128) + 4) < 2 ** 31


def test_frequencies():
    import wpt_b200
    f = wpt_b200.rotary_frequencies(8)
    assert f.dtype == torch.float64 and torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64))
    assert torch.allclose(wpt_b200.rotary_frequencies(8, scaling="linear", factor=4.0), f / 4)
    base = wpt_b200.rotary_frequencies(8, scaling="base", factor=4.0)
    assert abs(base[0] - 1) < 1e-15 and abs(base[-1] - f[-1] / 4) < 1e-12
    parts = wpt_b200.rotary_frequencies(8, scaling="parts", factor=4.0, original=4096)
    turns = 4096 * f / (2 * math.pi)  # 652, 65, 6.5, 0.65
    assert parts[0] == f[0] and parts[1] == f[1] and abs(parts[3] - f[3] / 4) < 1e-18
    keep = (turns[2] - 1) / 31
    assert abs(parts[2] - (f[2] * keep + f[2] / 4 * (1 - keep))) < 1e-18
    assert wpt_b200.rotary_frequencies(0).shape == (0,)
    for bad in (dict(dims=3), dict(dims=-2), dict(dims=4, scaling="ntk"), dict(dims=4, base=0), dict(dims=4, scaling="parts"),
                dict(dims=4, factor=0.0), dict(dims=4, scaling="parts", original=10, low=3.0, high=3.0)):
        with pytest.raises(ValueError):
            wpt_b200.rotary_frequencies(**bad)


def test_e4m3_restatement():
    every = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    finite = np.unique(np.abs(every[np.isfinite(every)]))
    assert np.array_equal(finite, op.e4m3_values())
    x = np.concatenate([np.random.default_rng(0).normal(size=4000) * 2.0 ** e for e in range(-12, 7)] +
                       [finite, (finite[1:] + finite[:-1]) / 2])
    x = x[np.abs(x) <= 448]
    assert np.array_equal(op.to_e4m3(x), torch.from_numpy(x).float().to(torch.float8_e4m3fn).double().numpy())
    assert np.isnan(op.to_e4m3(np.nan)) and op.least_scale(448.0) == 1 and op.least_scale(448.001) == 2
    assert op.least_scale(0.0) == 2.0 ** -60


def test_rotate_restatement():
    rng = np.random.default_rng(1)
    x, f = rng.normal(size=(2, 10)), np.array([1.0, 0.3])
    for interleaved in (False, True):
        y = op.rotate(x, np.array([0, 7]), f, 3, interleaved, 2.0)
        assert np.array_equal(y[:, :3], x[:, :3]) and np.array_equal(y[:, 7:], x[:, 7:])
        for i in range(2):
            a, b = (3 + 2 * i, 4 + 2 * i) if interleaved else (3 + i, 5 + i)
            t = 7 * f[i]
            assert abs(y[1, a] - 2 * (x[1, a] * math.cos(t) - x[1, b] * math.sin(t))) < 1e-12
            assert abs(y[1, b] - 2 * (x[1, b] * math.cos(t) + x[1, a] * math.sin(t))) < 1e-12
        back = op.rotate(y / 4, np.array([0, 7]), f, 3, interleaved, 2.0, inverse=True)
        assert np.abs(back[:, 3:7] - x[:, 3:7]).max() < 1e-12


def test_cache_restatements():
    rng = np.random.default_rng(2)
    cache = dict(values=np.zeros((3, 32, 8)), scales=np.zeros((3, 2, 2)))
    table = np.array([[2, 0]])
    new = rng.normal(size=(1, 20, 8)) * 4.0 ** np.arange(20)[None, :, None] / 2.0 ** 10
    for i in range(20):
        cache, _ = op.append(cache, table, new[:, i:i + 1], [25 + i], [1])
    got = cache["values"][2, 25:] * np.repeat(cache["scales"][2, 1], 4)
    big = np.repeat(cache["scales"][2, 1], 4)
    # rounded once for each growth of the scale: within a step in all
    assert (np.abs(got - new[0, :7]) <= 2.0 ** -3 * np.abs(new[0, :7]) + 2.0 ** -9 * big).all()
    assert cache["scales"][0, 0, 0] >= np.abs(new[0, 7:, :4]).max() / 448 > cache["scales"][0, 0, 0] / 2
    q = rng.normal(size=(1, 2, 3, 4))
    out, lse = op.attention(q, cache, table, np.array([[40, -1]]), 0.5, 20, np.zeros(3))
    e = np.concatenate([cache["values"][2, 21:] * np.repeat(cache["scales"][2, 1], 4),
                        cache["values"][0, :9] * np.repeat(cache["scales"][0, 0], 4)])
    z = 0.5 * q[0, 0] @ e[:, :4].T
    top = np.maximum(z.max(1, keepdims=True), 0)  # the sink's logit is 0
    w, s = np.exp(z - top), np.exp(-top)
    total = w.sum(1, keepdims=True) + s
    assert np.allclose(out[0, 0], w @ e[:, 4:] / total) and np.allclose(lse[0, 0], (top + np.log(total))[:, 0])
    assert (out[0, 1] == 0).all() and (lse[0, 1] == 0).all()
