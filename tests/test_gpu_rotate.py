"""Rotary positions on the GPU against oracle/paged.py in float64, forward and
backward.

Tolerance. An angle in half turns is rounded to fp32 once (2^-25, times pi:
1.6 roundings of 2^-24) after a turn's fraction that is off by 2^-52 p f
(nothing at these positions); sin and cos are within 2 units in the last place
(4 roundings of at most 1), the two products and their sum round 3 times, the
magnitude once: under 12 * 2^-24 of |x_a| + |x_b|. Then comes the output's own
rounding, half a step of its type."""

import numpy as np
import pytest
import torch

from oracle import paged as op

pytestmark = pytest.mark.gpu

TURN = 12 * 2.0 ** -24


@pytest.fixture(scope="module")
def wb():
    import wpt_b200
    from wpt_b200 import build
    build.build()
    return wpt_b200


def _np(t):
    return t.detach().double().cpu().numpy()


def _sizes(x, dims, start, interleaved):
    """|x_a| + |x_b| of each turned channel's pair, 0 of the others."""
    a = np.abs(x)
    out = np.zeros_like(a)
    part = a[..., start:start + dims]
    if interleaved:
        both = np.repeat(part[..., 0::2] + part[..., 1::2], 2, -1)
    else:
        both = np.tile(part[..., :dims // 2] + part[..., dims // 2:], 2)
    out[..., start:start + dims] = both
    return out


def _check(got, x, positions, f, start, interleaved, magnitude=1.0, inverse=False):
    x, f = _np(x), _np(f)
    start = x.shape[-1] - 2 * len(f) if start is None else start
    p = positions.cpu().numpy()
    p = np.broadcast_to(p, x.shape[:2]).reshape(x.shape[:2] + (1,) * (x.ndim - 3))  # (B, T) or (B, T, 1)
    p = np.broadcast_to(p, x.shape[:-1])
    ref = op.rotate(x, p, f, start, interleaved, magnitude, inverse)
    half_step = torch.finfo(got.dtype).eps / 2
    off = np.abs(_np(got) - ref)
    sizes = magnitude * _sizes(x, 2 * len(f), start, interleaved)
    assert (off <= TURN * sizes * (1 + half_step) + half_step * np.abs(ref)).all()
    kept = sizes == 0
    kept[..., start:start + 2 * len(f)] = False
    assert (_np(got)[kept] == x[kept]).all()  # channels that do not turn are copied


CASES = [
    # B, T, H, C, dims, start, interleaved, dtype
    (1, 1, 16, 128, 64, None, False, torch.bfloat16),
    (1, 1, 1, 128, 128, None, True, torch.bfloat16),
    (2, 33, 5, 128, 64, 0, False, torch.float32),
    (2, 17, 3, 64, 64, None, True, torch.float32),
    (3, 7, 12, 96, 40, 8, True, torch.bfloat16),
    (3, 7, 12, 96, 48, 16, False, torch.bfloat16),
    (2, 9, 4, 62, 34, 3, False, torch.bfloat16),   # nothing aligned
    (2, 9, 4, 62, 34, 3, True, torch.float32),
    (1, 5, 64, 130, 2, 127, False, torch.float32),
    (2, 19, 5, 132, 52, None, False, torch.bfloat16),  # vectors of 2
    (2, 19, 5, 102, 52, 6, True, torch.bfloat16),
    (3, 5, 2, 22, 12, 2, False, torch.float32),
    (3, 5, 2, 22, 14, 6, True, torch.float32),
    (4, 300, 16, 128, 64, None, False, torch.bfloat16),
    (1, 1200, 2, 256, 256, None, True, torch.bfloat16),
    (2, 3, 0, 128, 64, None, False, torch.bfloat16),
    (2, 0, 4, 128, 64, None, False, torch.float32),
]


@pytest.mark.parametrize("case", CASES)
def test_forward(wb, case):
    B, T, H, C, dims, start, interleaved, dtype = case
    g = torch.Generator().manual_seed(1)
    x = torch.randn(B, T, H, C, generator=g).to(dtype).cuda()
    positions = (torch.randint(0, 100000, (B, 1), generator=g) + torch.arange(T)).cuda()
    f = wb.rotary_frequencies(dims, device="cuda")
    _check(wb.rotate(x, positions, f, start, interleaved), x, positions, f, start, interleaved)
    if H:  # keys: no head axis, one position row for all
        _check(wb.rotate(x[:, :, 0], positions[0], f, start, interleaved, 1.25), x[:, :, 0], positions[:1], f, start,
               interleaved, 1.25)


@pytest.mark.parametrize("first", [0, 2 ** 20 - 3, 2 ** 31 - 2, 2 ** 40, -5])
@pytest.mark.parametrize("dtype64", [True, False])
def test_far_positions_are_exact(wb, first, dtype64):
    f = torch.tensor([1.0, 0.7310585, 3.1, 1e-3, 1e-9, 0.0], dtype=torch.float64).cuda()
    if not dtype64:
        f = f.float()
    x = torch.randn(1, 9, 2, 12, generator=torch.Generator().manual_seed(2)).cuda()
    positions = first + torch.arange(9).cuda()
    # a frequency's own rounding, 2^-53 of p f radians, is all that grows with the position
    got, want = _np(wb.rotate(x, positions, f)), op.rotate(_np(x), positions.cpu().numpy()[None, :, None].repeat(2, 2), _np(f))
    grown = 2.0 ** -52 * abs(first + 9) * 3.1
    assert (np.abs(got - want) <= (TURN + grown + 2.0 ** -24) * _sizes(_np(x), 12, 0, False)).all()


def test_strides(wb):
    g = torch.Generator().manual_seed(3)
    f = wb.rotary_frequencies(64, device="cuda")
    positions = torch.arange(7).cuda()
    packed = torch.randn(2, 7, 6, 3 * 128, generator=g).bfloat16().cuda()
    views = [packed[..., 128:256], packed[..., 1:129], packed[..., 2:130], packed[:, :, ::2, :128], packed[:, :, :, ::3],
             packed.transpose(0, 1)[:, :1].transpose(0, 1)[..., :128].expand(2, 7, 6, 128),
             packed[:, :, :1, :128].expand(2, 7, 6, 128), packed[..., :128].permute(0, 2, 1, 3).contiguous().transpose(1, 2)]
    for x in views:
        y = wb.rotate(x, positions, f)
        assert y.is_contiguous()
        _check(y, x, positions[None], f, None, False)
    _check(wb.rotate(views[0], positions.int().expand(2, 7), f), views[0], positions[None], f, None, False)
    wide = torch.arange(14).view(7, 2).cuda().t()  # positions of strides (1, 2)
    _check(wb.rotate(views[0], wide, f), views[0], wide, f, None, False)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
def test_gradient(wb, interleaved, dtype):
    g = torch.Generator().manual_seed(4)
    x = torch.randn(2, 11, 3, 96, generator=g).to(dtype).cuda().requires_grad_()
    d = torch.randn(2, 11, 3, 96, generator=g).to(dtype).cuda()
    positions = torch.randint(0, 5000, (2, 11), generator=g).cuda()
    f = wb.rotary_frequencies(48, scaling="parts", factor=4.0, original=1000, device="cuda")
    y = wb.rotate(x, positions, f, 16, interleaved, 0.75)
    dx, = torch.autograd.grad(y, x, d)
    assert dx.dtype == dtype
    _check(dx, d, positions, f, 16, interleaved, 0.75, inverse=True)
    if dtype == torch.float32:  # against differences: the map is linear, so any step will do
        v = torch.randn(x.shape, generator=g).cuda()
        with torch.no_grad():
            diff = (wb.rotate(x + v, positions, f, 16, interleaved, 0.75) - wb.rotate(x - v, positions, f, 16, interleaved, 0.75)) / 2
        left, right = (diff.double() * d.double()).sum().item(), (dx.double() * v.double()).sum().item()
        terms = (diff.abs().double() * d.abs().double()).sum().item()
        assert abs(left - right) <= 16 * 2.0 ** -24 * 3 * terms + 1e-9


def test_gradient_of_shared_heads_and_sums(wb):
    """An input broadcast over heads, and gradients that come expanded (of a sum) or in another type."""
    f = wb.rotary_frequencies(64, device="cuda")
    positions = torch.arange(40, 45).cuda()
    x = torch.randn(2, 5, 1, 64, generator=torch.Generator().manual_seed(5)).cuda().requires_grad_()
    wb.rotate(x.expand(2, 5, 7, 64), positions, f).sum().backward()
    one = op.rotate(np.ones((2, 5, 1, 64)), positions.cpu().numpy()[None, :, None].repeat(2, 0), _np(f), inverse=True)
    # 7 equal terms, each within TURN * 2, added in fp32
    assert (np.abs(_np(x.grad) - 7 * one) <= 7 * (2 * TURN + 8 * 2.0 ** -24 * 2)).all()
    with torch.no_grad():
        assert not wb.rotate(x, positions, f).requires_grad


def test_second_derivative(wb):
    """The gradient is a rotation too, of d_out: it can be differentiated again."""
    g = torch.Generator().manual_seed(6)
    f = wb.rotary_frequencies(16, device="cuda")
    positions = torch.arange(3, 8).cuda()
    x, d, v = (torch.randn(1, 5, 2, 24, generator=g).cuda().requires_grad_() for _ in range(3))
    dx, = torch.autograd.grad(wb.rotate(x, positions, f, 4, True), x, d, create_graph=True)
    dd, = torch.autograd.grad(dx, d, v)
    _check(dd, v, positions[None], f, 4, True)


def test_more_than_32_bits_of_elements(wb):
    """2.2e9 elements: the ends are as in calls of their own."""
    B, T, H, C = 33, 8192, 64, 128
    x = torch.empty(B, T, H, C, dtype=torch.bfloat16, device="cuda")
    assert x.numel() > 2 ** 31
    x[0], x[-1] = torch.randn(2, T, H, C, device="cuda")
    f = wb.rotary_frequencies(40, device="cuda")
    positions = torch.arange(T, device="cuda") + 5
    y = wb.rotate(x, positions, f, 20)
    for b in (0, B - 1):
        assert torch.equal(y[b:b + 1], wb.rotate(x[b:b + 1], positions, f, 20))
    _check(y[-1:, -3:], x[-1:, -3:], positions[None, -3:], f, 20, False)


def test_graph_and_streams(wb):
    f = wb.rotary_frequencies(64, device="cuda")
    x = torch.randn(2, 9, 4, 128).bfloat16().cuda()
    leaf = x.clone().requires_grad_()
    d = torch.randn_like(x)
    positions = torch.arange(9).cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(wb.rotate(leaf, positions, f), leaf, d)  # warm-up
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        y = wb.rotate(leaf, positions, f)
        dx, = torch.autograd.grad(y, leaf, d)
    for n in (3, 77):
        positions.copy_(torch.arange(n, n + 9))
        graph.replay()
        torch.cuda.synchronize()
        _check(y, x, positions[None], f, None, False)
        want = wb.ops.rotate(d, positions, f, inverse=True)
        assert torch.equal(dx, want)
    # a leaf with an eager graph alive keeps it
    kept = wb.rotate(leaf, positions, f)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(torch.autograd.grad(kept, leaf, d)[0], dx)


def test_refusals(wb):
    f = wb.rotary_frequencies(64, device="cuda")
    x, p = torch.zeros(1, 2, 3, 128, device="cuda"), torch.arange(2, device="cuda")
    with pytest.raises(NotImplementedError, match="bfloat16 or float32"):
        wb.rotate(x.half(), p, f)
    for bad in (dict(positions=torch.arange(3, device="cuda")), dict(positions=torch.zeros(2, 2, dtype=torch.int64, device="cuda")),
                dict(x=x[0, 0]), dict(start=65), dict(start=-1), dict(frequencies=f[None]), dict(frequencies=f.long()),
                dict(x=x[..., :32])):
        with pytest.raises(ValueError):
            wb.rotate(**(dict(x=x, positions=p, frequencies=f) | bad))
    with pytest.raises(ValueError, match="CUDA"):
        wb.rotate(x.cpu(), p, f)
    with pytest.raises(ValueError):
        wb.rotate(x, p.cpu(), f)
