"""Rotary positions where test_gpu_rotate.py's tolerance is wide or its sizes
end, against angles of extended precision.

Tolerance. An angle is off by 2^-52 |p f| (1 / (2 pi) and its product with f, each
rounded to double), 2 pi 2^-65 |p| (the fraction of a turn, rounded to 2^-64) and
2 pi 2^-32 (the phase, cut off); its distance to the nearest quarter turn is
rounded to fp32 as a whole number and as radians, 2^-23 of pi / 4 at most; sine and
cosine are cut after terms of 1.8e-9 and less, and their last steps, on values up
to 1, round by 2^-24 with what the steps before left (under a quarter of
that each): 4 * 2^-24 in all with the phase. Two products and their sum round by
2^-24 each of |x_a| + |x_b| at most, the magnitude once more."""

import numpy as np
import pytest
import torch

from test_gpu_rotate import _np, _sizes, wb  # noqa: F401

pytestmark = pytest.mark.gpu

PI = np.longdouble("3.14159265358979323846264338327950288")


def _turned(x, angle):
    """Pairs in halves, x (..., C) by angle (..., C / 2)."""
    half = x.shape[-1] // 2
    c, s = np.cos(angle).astype(np.float64), np.sin(angle).astype(np.float64)
    a, b = x[..., :half], x[..., half:]
    return np.concatenate((a * c - b * s, b * c + a * s), -1)


@pytest.mark.parametrize("first", [0, -7, 2 ** 20 - 3, -2 ** 31, 2 ** 40, 2 ** 48, -2 ** 48])
@pytest.mark.parametrize("dtype64", [True, False])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_each_pairs_angle(wb, first, dtype64, sign):  # noqa: F811
    """Slow pairs at far positions, and turns the other way: each pair within the bound of its own frequency."""
    f = sign * torch.tensor([1.0, 0.7310585, 3.1, 40.0, 1e-3, 1e-6, 1e-9, 1e-12, 0.0], dtype=torch.float64).cuda()
    f = f if dtype64 else f.float()
    x = torch.randn(1, 9, 3, 18, generator=torch.Generator().manual_seed(40)).cuda()
    positions = first + torch.arange(9).cuda()
    got, p = _np(wb.rotate(x, positions, f)), positions.cpu().numpy().astype(np.longdouble)
    angle = p[:, None] * _np(f).astype(np.longdouble)
    want = _turned(_np(x), np.mod(angle, 2 * PI)[None, :, None])
    off = 2.0 ** -52 * np.abs(angle) + 2 * PI * (2.0 ** -65 * np.abs(p)[:, None] + 2.0 ** -32)
    off = np.tile((off + 8 * 2.0 ** -24).astype(np.float64), 2)[None, :, None]
    assert (np.abs(got - want) <= off * _sizes(_np(x), 18, 0, False)).all()


def test_more_threads_than_32_bits(wb):  # noqa: F811
    """2^31 and more items of work, one element each: both ends and the middle are as in calls of their own."""
    T, C = 2 ** 24 + 5, 129
    x = torch.empty(1, T, C, dtype=torch.bfloat16, device="cuda")
    parts = [slice(0, 700), slice(T // 2 - 300, T // 2 + 300), slice(T - 700, T)]
    assert T * (C - 1) > 2 ** 31
    for part in parts:
        x[:, part] = torch.randn(x[:, part].shape, generator=torch.Generator().manual_seed(41)).cuda()
    positions, f = torch.arange(T, device="cuda") + 11, torch.tensor([0.37], dtype=torch.float64, device="cuda")
    y = wb.rotate(x, positions, f)
    for part in parts:
        assert torch.equal(y[:, part], wb.rotate(x[:, part], positions[part], f))
        assert torch.equal(y[:, part, :127], x[:, part, :127]) and not torch.equal(y[:, part], x[:, part])
