"""The paged cache held in 8 bits on the GPU, its append and the attention that
reads it, against oracle/paged.py in float64.

Tolerances.
Append: an entry's value in units of its block's scale is within half a step of
e4m3 (2^-4 of it, 2^-10 at least) of the exact one, plus what fp32 leaves of a
turned key (TURN of |x_a| + |x_b| <= 2 * 448); scales, and the entries that are
rounded again, are exact.
Attention: a score is a sum of 128 products that fp32 holds, off by at most 128
truncations (2^-23 each) of a running sum under A = scale sum |q||k| (A < 32 in
these tests), plus what q's two parts leave, 2^-22.8 of the largest |q| times
scale sum |k| (under 2^-22.8 * 6 * 64), plus roundings of its exponent (2^-23 of
64, twice): SCORE = 6e-4 in all. The log-sum is off by as much and its own
rounding. A weight's parts are within 2^-8.6 of it and 2^-21 of the largest
weight of a run of keys (n of them); so an output is within (2^-8.6 + 2 SCORE)
sum w|v| + n 2^-21 max|v| of the exact one, and half a step of bf16 (2^-8)."""

import math

import numpy as np
import pytest
import torch

from oracle import paged as op

pytestmark = pytest.mark.gpu

TURN = 12 * 2.0 ** -24
SCORE = 6e-4


@pytest.fixture(scope="module")
def wb():
    import wpt_b200
    from wpt_b200 import build
    build.build()
    return wpt_b200


def _np(t):
    return t.detach().double().cpu().numpy()


def _cache(pages, scales):
    return dict(values=_np(pages), scales=_np(scales))


def _table(B, M, P, g, dtype=torch.int32):
    """Pages of the B rows, each one's own, from anywhere."""
    return torch.randperm(P, generator=g)[:B * M].view(B, M).to(dtype)


def _filled(B, M, S, C, g, spread=2.0, spare=2):
    """A full cache: values whose size changes from block to block by up to 2^spread."""
    P = B * M + spare
    x = torch.randn(P, S // 16, 16, 2, C, generator=g)
    x *= torch.exp2((torch.rand(P, S // 16, 1, 2, 1, generator=g) - 0.5) * spread)
    scales = torch.tensor([[[op.least_scale(v) for v in k] for k in p] for p in x.abs().amax((2, 4)).tolist()])
    pages = (x / scales[:, :, None, :, None]).reshape(P, S, 2 * C).to(torch.float8_e4m3fn)
    return pages, scales, _table(B, M, P, g)


# ----------------------------------------------------------------- append

def _check_append(got, cache, table, new, first, counts, f=None, positions=None, start=None, interleaved=False,
                  magnitude=1.0, slack=0.0):
    want, exact = op.append(cache, table.cpu().numpy(), _np(new), first.tolist(), counts.tolist(),
                            None if f is None else _np(f), None if positions is None else positions.cpu().numpy(),
                            start, interleaved, magnitude)
    values, scales = _np(got[0]), _np(got[1])
    assert np.array_equal(scales, want["scales"])
    written = np.zeros(values.shape[:2], bool)
    for (page, place), x in exact.items():
        written[page, place] = True
        v = values[page, place]
        assert np.array_equal(np.isnan(v), np.isnan(x))
        fine = ~np.isnan(x)
        off = np.abs(v - x)[fine]
        assert (off <= np.maximum(2.0 ** -4 * np.abs(x[fine]), 2.0 ** -10) + 2 * 448 * TURN + slack).all()
    assert np.array_equal(values[~written], want["values"][~written], equal_nan=True)


APPENDS = [
    # B, n, S, M, C, dims, interleaved, dtype
    (1, 1, 16, 2, 128, 0, False, torch.bfloat16),
    (1, 1, 16, 4, 128, 64, False, torch.bfloat16),
    (3, 5, 32, 3, 128, 128, False, torch.bfloat16),
    (2, 70, 64, 2, 64, 64, True, torch.bfloat16),
    (2, 70, 128, 1, 80, 36, True, torch.float32),
    (4, 33, 16, 5, 16, 6, False, torch.float32),
    (2, 40, 32, 2, 144, 18, False, torch.bfloat16),  # nothing aligned
    (1, 300, 256, 2, 32, 30, True, torch.bfloat16),
    (1, 17, 128, 1, 512, 512, False, torch.float32),
    (2, 20, 32, 2, 112, 28, False, torch.bfloat16),  # vectors of 2
    (2, 20, 32, 2, 224, 46, True, torch.bfloat16),
    (2, 20, 32, 2, 48, 36, False, torch.float32),
    (2, 40, 32, 2, 144, 64, False, torch.bfloat16),  # more than 16 vectors a key
    (2, 40, 32, 2, 256, 256, True, torch.bfloat16),
    (3, 21, 16, 3, 128, 64, False, torch.float32),
    (1, 40, 32, 2, 304, 64, False, torch.bfloat16),  # more than 32
    (5, 19, 64, 1, 16, 16, False, torch.bfloat16),   # 2: all entries of a warp at a time
    (2, 19, 64, 1, 80, 0, False, torch.bfloat16),    # 10: three, then one
    (5, 0, 16, 2, 128, 64, False, torch.bfloat16),
]


@pytest.mark.parametrize("case", APPENDS)
def test_append(wb, case):
    B, n, S, M, C, dims, interleaved, dtype = case
    g = torch.Generator().manual_seed(7)
    pages, scales, table = _filled(B, M, S, C, g)
    room = M * S - n
    first = torch.randint(0, room + 1, (B,), generator=g)
    counts = torch.randint(0, n + 1, (B,), generator=g)
    counts[0] = n
    new = (torch.randn(B, n, 2 * C, generator=g) * torch.exp2(torch.randint(-3, 4, (B, n, 1), generator=g).float())).to(dtype)
    f = wb.rotary_frequencies(dims) if dims else None
    cache = _cache(pages, scales)
    dev = [t.cuda() for t in (pages, scales, table, new, first, counts)]
    got = wb.paged_append(*dev, frequencies=None if f is None else f.cuda(), interleaved=interleaved)
    assert got[0] is dev[0] and got[1] is dev[1]
    _check_append(got, cache, table, new, first, counts, f, None, None, interleaved)
    assert wb.device_status() == 0


def test_append_token_by_token(wb):
    """A text written entry by entry, sizes rising and falling: scales only grow within a block, and a rolled-back
    text (drafts refused) is written over."""
    g = torch.Generator().manual_seed(8)
    pages, scales = (t.cuda() for t in wb.paged_cache(4, 32, 64, "cuda"))
    table = torch.tensor([[2, 0], [3, 1]])
    size = torch.exp2(torch.cat((torch.arange(-10.0, 10), torch.arange(10.0, -10, -1))))
    new = (torch.randn(2, 40, 128, generator=g) * size[:, None]).bfloat16()
    steps = list(range(37)) + list(range(29, 40))
    for i in steps:
        cache = _cache(pages, scales)
        first, counts = torch.tensor([i, max(0, i - 3)]), torch.tensor([1, 1])
        part = torch.stack((new[0, i], new[1, max(0, i - 3)]))[:, None]
        got = wb.paged_append(pages, scales, table.cuda(), part.cuda(), first.cuda(), counts.cuda())
        _check_append(got, cache, table, part, first, counts)


def test_append_places(wb):
    """Entries before the table, past it, on no page, and padding: dropped, with the status word's bit."""
    g = torch.Generator().manual_seed(9)
    pages, scales, _ = _filled(4, 2, 32, 32, g)
    table = torch.tensor([[0, -1], [1, 99], [2, 3], [4, 5], [-7, 6]], dtype=torch.int64)
    first = torch.tensor([20, 25, 50, -10, 3])
    counts = torch.tensor([40, 40, 40, 40, 40])
    new = torch.randn(5, 40, 64, generator=g)
    cache = _cache(pages, scales)
    got = wb.paged_append(*(t.cuda() for t in (pages, scales, table, new, first, counts)))
    _check_append(got, cache, table, new, first, counts)
    assert wb.device_status() == 2
    for at, count in ((2 ** 62, 3), (-2 ** 62, 3), (64, 1), (0, -5), (-3, 3), (-3, 2 ** 62)):
        before = pages.cuda(), scales.cuda()
        n = torch.full((5,), count)
        got = wb.paged_append(before[0].clone(), before[1].clone(), table.cuda(), new[:, :3].cuda(),
                              torch.full((5,), at).cuda(), n.cuda())
        assert torch.equal(got[0].view(torch.uint8), before[0].view(torch.uint8)) and torch.equal(got[1], before[1])
        wb.device_status()


def test_append_values_that_are_not_finite(wb):
    g = torch.Generator().manual_seed(10)
    pages, scales, table = _filled(1, 2, 16, 16, g)
    new = torch.randn(1, 20, 32, generator=g)
    new[0, 2, 3], new[0, 5, 20], new[0, 7, 0] = math.inf, math.nan, -math.inf
    new[0, 17, 1], new[0, 18, 17], new[0, 19, 18] = 3e38, 448 * 2.0 ** 60, 1e-30
    new[0, 16, 16:] = 0
    first, counts = torch.tensor([0]), torch.tensor([20])
    cache = _cache(pages, scales)
    got = wb.paged_append(*(t.cuda() for t in (pages, scales, table, new, first, counts)))
    _check_append(got, cache, table, new, first, counts)
    zeros = wb.paged_append(*(t.cuda() for t in (pages, scales, table, torch.zeros(1, 20, 32), first, counts)))
    assert (_np(zeros[1])[table[0].numpy()] == 2.0 ** -60).all()


def test_append_strides_positions_and_layers(wb):
    g = torch.Generator().manual_seed(11)
    f = wb.rotary_frequencies(32)
    wide = torch.zeros(6, 3, 32, 160, dtype=torch.float8_e4m3fn, device="cuda")  # layers of a page, wider entries
    pages = wide[:, 1, :, 16:144]
    scales = torch.zeros(6, 3, 2, 2, device="cuda")[:, 2]
    table = torch.stack((_table(2, 2, 6, g), _table(2, 2, 6, g)), -1).cuda()[..., 0]  # strided
    new = torch.randn(2, 3, 21, 140, generator=g).bfloat16().cuda()[:, 1, :, 5:133]
    first, counts = torch.tensor([11, 40]), torch.tensor([21, 20])
    positions = torch.randint(0, 10 ** 6, (2, 21), generator=g)
    cache = _cache(pages, scales)
    got = wb.paged_append(pages, scales, table, new, first.cuda(), counts.cuda(), frequencies=f.cuda(),
                          positions=positions.cuda(), start=8, magnitude=1.5)
    _check_append(got, cache, table, new.cpu(), first, counts, f, positions, 8, False, 1.5)
    untouched = wide.view(torch.uint8).clone()
    untouched[:, 1, :, 16:144] = 0
    assert not untouched.any()


# -------------------------------------------------------------- attention

def _check_attention(got, q, cache, table, positions, scale, window=0, sink=None):
    table, positions, sink = table.cpu().numpy(), positions.cpu().numpy(), None if sink is None else _np(sink)
    q = _np(q)
    ref, lse = op.attention(q, cache, table, positions, scale, window, sink)
    C = q.shape[-1]
    sizes = dict(cache, values=np.concatenate((cache["values"][..., :C], np.abs(cache["values"][..., C:])), -1))
    around, _ = op.attention(q, sizes, table, positions, scale, window, sink)
    out, got_lse = _np(got[0]), _np(got[1])
    assert np.array_equal(np.isnan(out), np.isnan(ref)) and np.array_equal(np.isnan(got_lse), np.isnan(lse))
    n = table.shape[1] * cache["values"].shape[1]
    big = np.nanmax(np.abs(cache["values"][..., C:]) * np.repeat(cache["scales"][..., 1], 16, 1)[..., None], initial=0)
    tol = 2.0 ** -8 * np.abs(ref) + (2.0 ** -8.6 + 2 * SCORE) * around + n * 2.0 ** -21 * min(big, np.nanmax(around, initial=0) * 64)
    fine = ~np.isnan(ref)
    assert (np.abs(out - ref)[fine] <= tol[fine]).all(), np.nanmax((np.abs(out - ref) / (tol + 1e-30)))
    empty = np.isneginf(lse)
    assert (out[empty] == 0).all() and np.isneginf(got_lse[empty]).all()
    some = ~empty & ~np.isnan(lse)
    assert (np.abs(got_lse - lse)[some] <= SCORE + 2.0 ** -22 * np.abs(lse[some])).all()


def _queries(B, T, H, g, size=1.0):
    return (torch.randn(B, T, H, 128, generator=g) * size).bfloat16()


ATTENDS = [
    # B, T, H, S, M, window, sink
    (1, 1, 1, 16, 1, 0, False),        # one key
    (1, 1, 16, 16, 8, 0, False),
    (2, 1, 16, 32, 5, 0, True),
    (3, 1, 32, 64, 9, 0, False),
    (5, 1, 12, 128, 3, 100, True),
    (2, 1, 64, 256, 2, 0, False),      # two groups a query
    (3, 4, 8, 16, 21, 0, True),        # 32 columns
    (2, 5, 12, 32, 17, 0, True),       # three groups a row
    (2, 9, 12, 64, 5, 37, False),      # five
    (1, 70, 1, 16, 12, 50, True),      # 70 queries of one head
    (4, 3, 21, 128, 7, 300, True),
    (40, 1, 32, 64, 11, 0, False),     # balanced over the CTAs
    (7, 3, 5, 16, 90, 0, True),        # 1,440 entries
    (150, 2, 33, 16, 5, 0, False),     # more groups than a balanced call takes
    (1, 1, 32, 128, 60, 0, False),     # one row over many CTAs
]


@pytest.mark.parametrize("case", ATTENDS)
def test_attention(wb, case):
    B, T, H, S, M, window, sink = case
    g = torch.Generator().manual_seed(12)
    pages, scales, table = _filled(B, M, S, 128, g)
    q = _queries(B, T, H, g)
    lengths = torch.randint(0, M * S + 1, (B,), generator=g)
    lengths[0] = M * S
    positions = lengths[:, None] - T + torch.arange(T)
    positions = torch.where(positions < 0, -1, positions)
    s = torch.randn(H, generator=g) if sink else None
    cache = _cache(pages, scales)
    got = wb.paged_attention(*(t.cuda() for t in (q, pages, scales, table, positions)), 128 ** -0.5, window=window,
                             sink=None if s is None else s.cuda())
    _check_attention(got, q, cache, table, positions, 128 ** -0.5, window, s)
    again = wb.paged_attention(*(t.cuda() for t in (q, pages, scales, table.long(), positions)), 128 ** -0.5,
                               window=window, sink=None if s is None else s.cuda())
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])  # bit for bit
    assert wb.device_status() == 0


@pytest.mark.parametrize("splits,ctas", [(1, 1), (2, 1), (3, 1), (8, 1), (0, 1), (0, 2), (0, 7), (0, 40), (0, 500)])
def test_every_way_of_splitting(wb, splits, ctas, monkeypatch):
    """The same rows by each plan that the library takes, windows and odd lengths among them."""
    monkeypatch.setattr(wb.ops, "_paged_plan", lambda *a: (splits, ctas))
    g = torch.Generator().manual_seed(13)
    for B, T, H, S, M, window in ((3, 2, 8, 16, 37, 0), (2, 3, 11, 32, 11, 70), (4, 2, 32, 64, 6, 0)):
        pages, scales, table = _filled(B, M, S, 128, g)
        q = _queries(B, T, H, g)
        lengths = torch.randint(T, M * S + 1, (B,), generator=g)
        lengths[-1] = 0
        positions = torch.clamp(lengths[:, None] - T + torch.arange(T), min=-1)
        sink = torch.randn(H, generator=g)
        got = wb.paged_attention(*(t.cuda() for t in (q, pages, scales, table, positions)), 128 ** -0.5, window=window,
                                 sink=sink.cuda())
        _check_attention(got, q, _cache(pages, scales), table, positions, 128 ** -0.5, window, sink)
    assert wb.device_status() == 0


def test_unread_entries_reach_nothing(wb):
    """NaN in keys, values and scales of entries past the position, before the window and on pages of no row, pages
    that are missing in the middle, and positions past the table."""
    g = torch.Generator().manual_seed(14)
    B, T, H, S, M, window = 3, 3, 16, 32, 12, 150
    pages, scales, table = _filled(B, M, S, 128, g)
    positions = torch.tensor([[200, 201, 202], [90, 17, 383], [380, 383, 5000]])
    table[1, 3] = -1
    table[2, 9] = 10 ** 6
    clean = _cache(pages, scales)
    read = torch.zeros(B, M * S, dtype=torch.bool)
    n = torch.arange(M * S)
    for b in range(B):
        for t in range(T):
            read[b] |= (n <= positions[b, t]) & (n > positions[b, t] - window)
    dirty = pages.clone()
    raw = dirty.view(torch.uint8)
    mine = torch.zeros(pages.shape[0], S, dtype=torch.bool)
    for b in range(B):
        for i in range(M):
            if 0 <= table[b, i] < pages.shape[0]:
                mine[table[b, i]] |= read[b, i * S:(i + 1) * S]
    raw[~mine] = 0x7F
    bad = scales.clone()
    bad[~mine.view(-1, S // 16, 16).any(-1)] = math.nan
    q = _queries(B, T, H, g)
    got = wb.paged_attention(*(t.cuda() for t in (q, dirty, bad, table, positions)), 128 ** -0.5, window=window)
    _check_attention(got, q, clean, table, positions, 128 ** -0.5, window)
    # without a window too
    read = n <= positions.max(1).values[:, None]
    got = wb.paged_attention(*(t.cuda() for t in (q, pages, scales, table, positions)), 128 ** -0.5)
    _check_attention(got, q, clean, table, positions, 128 ** -0.5)


@pytest.mark.parametrize("T,H", [(1, 32), (4, 8), (6, 10)])
def test_nan_shows_where_it_is_read_and_nowhere_else(wb, T, H):
    """A NaN in a value reaches its channel of the queries that read it (drafts that come before it do not); a NaN
    in a key, all channels of them."""
    g = torch.Generator().manual_seed(15)
    S, M = 16, 10
    pages, scales, table = _filled(4, M, S, 128, g)
    positions = torch.full((4, 1), 150) + torch.arange(T)
    raw = pages.view(torch.uint8)

    def put(b, n, channel):
        raw[table[b, n // S], n % S, channel] = 0xFF

    put(0, 150 + T - 1, 128 + 5)   # the last draft's value
    put(1, 77, 128 + 99)           # every query's
    put(2, 150 + T - 1, 3)         # the last draft's key
    put(3, 150 + T // 2, 128)
    put(3, 150 + T // 2, 255)
    q = _queries(4, T, H, g)
    cache = _cache(pages, scales)
    got = wb.paged_attention(*(t.cuda() for t in (q, pages, scales, table, positions)), 128 ** -0.5)
    _check_attention(got, q, cache, table, positions, 128 ** -0.5)
    q[0, 0, 1, 7], q[1, T - 1, 0, 100] = math.inf, math.nan
    got = wb.paged_attention(*(t.cuda() for t in (q, pages, scales, table, positions)), 128 ** -0.5)
    out = got[0].float()
    assert out[0, 0, 1].isnan().all() and out[1, T - 1, 0].isnan().all()
    rest = torch.ones(4, T, H, dtype=torch.bool)
    rest[0, 0, 1] = rest[1, T - 1, 0] = False
    clean = q.clone()
    clean[0, 0, 1, 7] = clean[1, T - 1, 0, 100] = 0
    want = wb.paged_attention(*(t.cuda() for t in (clean, pages, scales, table, positions)), 128 ** -0.5)
    a, b = out.cpu()[rest], want[0].float().cpu()[rest]
    assert torch.equal(a.isnan(), b.isnan())


def test_scores_that_jump(wb):
    """A score far past those before it (the running maximum moves by 100 and by 1,000), early and late in a run of
    keys, for some heads only; and one that leaves all others nothing."""
    g = torch.Generator().manual_seed(16)
    S, M, H = 64, 30, 32
    for jump in (9.0, 30.0, 100.0, 1000.0):
        pages, scales, table = _filled(2, M, S, 128, g, spread=0.0)
        q = _queries(2, 1, H, g)
        raw = pages.view(torch.uint8)
        for b, at in ((0, 5), (0, 700), (0, 1900), (1, 1000)):
            h = int(torch.randint(0, H, (1,), generator=g))
            page, place = int(table[b, at // S]), at % S
            # a key along q, so that head h's score is about `jump`
            k = q[b, 0, h].float()
            k = k * (jump * 128 ** 0.5 / (k @ k))
            block = pages[page, place // 16 * 16:place // 16 * 16 + 16, :128].float() * scales[page, place // 16, 0]
            block[place % 16] = k
            s = op.least_scale(block.abs().max().item())
            scales[page, place // 16, 0] = s
            pages[page, place // 16 * 16:place // 16 * 16 + 16, :128] = (block / s).to(torch.float8_e4m3fn)
        positions = torch.tensor([[1915], [1200]])
        cache = _cache(pages, scales)
        got = wb.paged_attention(*(t.cuda() for t in (q, pages, scales, table, positions)), 128 ** -0.5)
        ref, lse = op.attention(_np(q), cache, table.numpy(), positions.numpy(), 128 ** -0.5)
        # scores of this size are held to 128 * 2^-23 of A = about 11 times the largest
        slack = 128 * 2.0 ** -23 * 11 * jump
        assert (np.abs(_np(got[1]) - lse) <= SCORE + slack).all()
        assert (np.abs(_np(got[0]) - ref) <= 2.0 ** -8 * np.abs(ref) + (2.0 ** -8.6 + 2 * SCORE + 2 * slack) * 8).all()


@pytest.mark.parametrize("T,H", [(1, 16), (4, 8), (3, 12), (1, 64)])
def test_heads_and_padding_of_other_sizes(wb, T, H):
    """Heads whose queries are 2^-20 to 1 of the others', and padding queries of up to 2^120 next to live ones: each
    column's result is as if it were alone. (Smaller queries' scores are off by less; the padding's own are not
    looked at, but for being there.)"""
    g = torch.Generator().manual_seed(23)
    B, S, M = 4, 32, 9
    pages, scales, table = _filled(B, M, S, 128, g)
    q = _queries(B, T, H, g) * torch.exp2(torch.randint(-20, 1, (B, 1, H, 1), generator=g).float()).bfloat16()
    q[2, :, H // 2] = 0
    positions = torch.full((B, 1), M * S - T) + torch.arange(T)
    cache = _cache(pages, scales)
    dev = [t.cuda() for t in (pages, scales, table, positions)]
    plain = wb.paged_attention(q.cuda(), *dev, 128 ** -0.5)
    _check_attention(plain, q, cache, table, positions, 128 ** -0.5)
    padded = q.clone()
    padded[0, T - 1, H - 1] *= 2.0 ** 120
    padded[1, 0, 0] = 2.0 ** 100
    padded[3, :, ::2] *= 2.0 ** 30
    got = wb.paged_attention(padded.cuda(), *dev, 128 ** -0.5)
    same = (padded == q).all(-1)
    assert same.sum() > 0
    ref = torch.where(same[..., None], padded, 0).bfloat16()  # the padding's columns as zeros, which the check passes over
    out, lse = got[0].clone(), got[1].clone()
    zero = wb.paged_attention(ref.cuda(), *dev, 128 ** -0.5)
    out[~same.cuda()], lse[~same.cuda()] = zero[0][~same.cuda()], zero[1][~same.cuda()]
    _check_attention((out, lse), ref, cache, table, positions, 128 ** -0.5)
    assert wb.device_status() == 0


def test_scales_of_all_sizes(wb):
    """Blocks of zeros (scale 0, or the least), and blocks whose values are far larger or smaller than the others'."""
    g = torch.Generator().manual_seed(17)
    S, M, H = 32, 20, 16
    pages, scales, table = _filled(3, M, S, 128, g)
    raw = pages.view(torch.uint8)
    raw[table[0, 4], :, 128:] = 0
    scales[table[0, 4], :, 1] = 0.0
    raw[table[0, 7], 16:, 128:] = 0
    scales[table[0, 7], 1, 1] = 2.0 ** -60
    scales[table[1, ::2].long(), :, 1] *= 2.0 ** 20
    scales[table[1, 5].long(), :, 1] *= 2.0 ** -30
    scales[table[2].long(), :, 1] *= 2.0 ** 50
    raw[table[1, 9], :16, :128] = 0
    scales[table[1, 9], 0, 0] = 0.0
    scales[table[2, 3].long(), 0, 0] *= 0.3  # not a power of two
    scales[table[0, 3].long(), 1, 1] *= 1.7
    q = _queries(3, 2, H, g)
    positions = torch.tensor([[500, 501], [639, 600], [300, 3]])
    got = wb.paged_attention(*(t.cuda() for t in (q, pages, scales, table, positions)), 128 ** -0.5)
    _check_attention(got, q, _cache(pages, scales), table, positions, 128 ** -0.5)


def test_sinks_of_all_sizes(wb):
    g = torch.Generator().manual_seed(18)
    for B, M in ((2, 6), (30, 20)):  # a cluster, and parts merged
        pages, scales, table = _filled(B, M, 64, 128, g)
        q = _queries(B, 1, 8, g)
        positions = torch.randint(0, M * 64, (B, 1), generator=g)
        positions[0] = -1
        sink = torch.tensor([-1e4, -300.0, -5.0, 0.0, 5.0, 300.0, 1e4, -math.inf])
        got = wb.paged_attention(*(t.cuda() for t in (q, pages, scales, table, positions)), 128 ** -0.5, sink=sink.cuda())
        _check_attention(got, q, _cache(pages, scales), table, positions, 128 ** -0.5, 0, sink)
        assert np.allclose(_np(got[1])[0, 0, :7], sink[:7].numpy(), atol=1e-3) and (_np(got[0])[0] == 0).all()


def test_small_weights_keep_their_sum(wb):
    """One key with half of the weight and 30,000 that share the rest."""
    g = torch.Generator().manual_seed(19)
    S, M, H = 128, 240, 4
    n = M * S
    pages = torch.zeros(M, S, 256).to(torch.float8_e4m3fn)
    pages[:, :, 128:] = (torch.rand(M, S, 128, generator=g) + 0.5).to(torch.float8_e4m3fn)
    scales = torch.ones(M, S // 16, 2)
    at = 17 * S + 3
    pages[17, 3, 0] = 8.0
    q = torch.zeros(1, 1, H, 128)
    q[..., 0] = math.log(n) / 8 * 128 ** 0.5
    q = q.bfloat16()
    table, positions = torch.arange(M)[None].int(), torch.tensor([[n - 1]])
    got = wb.paged_attention(*(t.cuda() for t in (q, pages, scales, table, positions)), 128 ** -0.5)
    ref, lse = op.attention(_np(q), _cache(pages, scales), table.numpy(), positions.numpy(), 128 ** -0.5)
    assert (np.abs(_np(got[1]) - lse) <= SCORE).all() and at < n
    # 130 tiles or fewer a run: a weight is off by 2^-8.6 of it, or 2^-21 of the run's largest
    assert (np.abs(_np(got[0]) - ref) <= 2.0 ** -8 * np.abs(ref) + (2.0 ** -8.6 + 2 * SCORE) * np.abs(ref) + n * 2.0 ** -21 * 0.5 * 1.5).all()
    assert (np.abs(_np(got[0]) - ref) <= 0.01 * np.abs(ref)).all()


def test_layers_strides_and_shared_pages(wb):
    g = torch.Generator().manual_seed(20)
    P, S = 14, 32
    wide = torch.randn(P, 2, S, 320, generator=g).to(torch.float8_e4m3fn).cuda()
    pages = wide[:, 1, :, 48:304]
    scales = torch.rand(P, 2, 2, 2, generator=g).cuda()[:, 0] + 0.1
    table = torch.randint(0, P, (5, 2, 8), generator=g).cuda()[:, 1]  # rows share pages
    q = torch.randn(5, 16, 2, 128, generator=g).bfloat16().cuda().transpose(1, 2)
    positions = torch.randint(0, 256, (5, 2), generator=g)
    got = wb.paged_attention(q, pages, scales, table, positions.cuda(), 0.05)
    _check_attention(got, q.cpu(), _cache(pages, scales), table, positions, 0.05)
    one = wb.paged_attention(q, pages, scales, table, positions[0].cuda(), 0.05)  # positions of one row for all
    _check_attention(one, q.cpu(), _cache(pages, scales), table, positions[:1].expand(5, 2), 0.05)


def test_empty_calls(wb):
    pages, scales = wb.paged_cache(3, 32, 128)
    table, p = torch.zeros(2, 4, dtype=torch.int32, device="cuda"), torch.full((2, 1), 9, device="cuda")
    q = torch.randn(2, 1, 4, 128, device="cuda").bfloat16()
    for args in ((q[:0], pages, scales, table[:0], p[:0]), (q[:, :0], pages, scales, table, p[:, :0]),
                 (q[:, :, :0], pages, scales, table, p), (q, pages, scales, table[:, :0], p), (q, pages[:0], scales[:0], table, p)):
        out, lse = wb.paged_attention(*args, 1.0)
        assert out.shape == args[0].shape and (out == 0).all() and (lse == -math.inf).all()
    new = torch.zeros(2, 3, 256, device="cuda")
    at, n = torch.zeros(2, dtype=torch.int64, device="cuda"), torch.full((2,), 3, device="cuda")
    wb.paged_append(pages[:0], scales[:0], table, new, at, n)
    wb.paged_append(pages, scales, table[:, :0], new, at, n)
    wb.paged_append(pages, scales, table, new[:, :0], at, n)
    assert not pages.view(torch.uint8).any() and wb.device_status() == 0


# --------------------------------------------------------------- together

def test_generation(wb):
    """Prompts and steps as a writer makes them: queries turned, entries appended with their keys turned, attention
    over all of them; against exact attention over entries turned in 64 bits."""
    g = torch.Generator().manual_seed(21)
    B, H, S, M, C = 3, 16, 16, 8, 128
    pages, scales = wb.paged_cache(B * M + 1, S, C)
    table = _table(B, M, B * M + 1, g).cuda()
    f = wb.rotary_frequencies(64, device="cuda")
    lengths = torch.zeros(B, dtype=torch.int64)
    entries = torch.randn(B, M * S, 2 * C, generator=g).bfloat16()
    for n, counts in ((41, [41, 7, 20]), (1, [1, 1, 1]), (4, [4, 2, 1]), (1, [1, 1, 1])):
        counts = torch.tensor(counts)
        new = torch.stack([entries[b, lengths[b]:lengths[b] + n] for b in range(B)])
        q = _queries(B, n, H, g)
        positions = lengths[:, None] + torch.arange(n)
        turned = wb.rotate(q.cuda(), positions.cuda(), f)
        wb.paged_append(pages, scales, table, new.cuda(), lengths.cuda(), counts.cuda(), frequencies=f)
        last = torch.minimum(torch.arange(n), counts[:, None] - 1)
        out, _ = wb.paged_attention(turned, pages, scales, table, (lengths[:, None] + last).cuda(), C ** -0.5)
        for b in range(B):
            for t in range(int(counts[b])):
                p = int(lengths[b]) + t
                e = _np(entries[b, :p + 1])
                k = op.rotate(e[:, :C], np.arange(p + 1), _np(f))
                qt = op.rotate(_np(q[b, t]), np.full(H, p), _np(f))
                z = qt @ k.T * C ** -0.5
                w = np.exp(z - z.max(1, keepdims=True))
                want = w / w.sum(1, keepdims=True) @ e[:, C:]
                # e4m3 entries (a step is 2^-3): scores off by some 2^-4.6 |q||k| / sqrt(128), values by 2^-4
                assert np.linalg.norm(_np(out[b, t]) - want) <= 0.12 * np.linalg.norm(want) + 1e-3
        lengths += counts
    assert wb.device_status() == 0


def test_graphs_and_streams(wb):
    """A step captured once and replayed as the text grows, two graphs in turn, another stream than the tensors'."""
    g = torch.Generator().manual_seed(22)
    B, H, S, M = 6, 16, 32, 40
    f = wb.rotary_frequencies(128, device="cuda")
    pages, scales, table = _filled(B, M, S, 128, g)
    dev = [t.cuda() for t in (pages, scales, table)]
    q, new = _queries(B, 1, H, g).cuda(), torch.randn(B, 1, 256, generator=g).bfloat16().cuda()
    first, counts = torch.randint(0, M * S - 8, (B,), generator=g).cuda(), torch.ones(B, dtype=torch.int64).cuda()

    def step():
        turned = wb.rotate(q, first[:, None], f)
        wb.paged_append(*dev, new, first, counts, frequencies=f)
        return wb.paged_attention(turned, *dev, first[:, None], 128 ** -0.5)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = step()
        graphs.append((graph, out))
    for i in range(4):
        q.copy_(_queries(B, 1, H, g))
        new.copy_(torch.randn(B, 1, 256, generator=g))
        first.add_(1)
        kept = [t.clone() for t in dev]
        graph, out = graphs[i % 2]
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        after = [t.clone() for t in dev]
        for t, k in zip(dev, kept):
            t.copy_(k)
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(after, dev))


def test_two_streams_at_once(wb):
    """Balanced calls (with scratch) and appends to different pools on two streams, over and over: what one alone gives."""
    g = torch.Generator().manual_seed(24)
    sides, runs = [torch.cuda.Stream() for _ in range(2)], []
    for B, H, S, M in ((5, 16, 16, 200), (3, 24, 32, 150)):
        pages, scales, table = _filled(B, M, S, 128, g)
        dev = [t.cuda() for t in (pages, scales, table)]
        q, new = _queries(B, 2, H, g).cuda(), torch.randn(B, 2, 256, generator=g).bfloat16().cuda()
        first, counts = torch.randint(0, M * S - 2, (B,), generator=g).cuda(), torch.full((B,), 2).cuda()
        wb.paged_append(*dev, new, first, counts)
        positions = first[:, None] + torch.arange(2).cuda()
        runs.append((dev, q, new, first, counts, positions, wb.paged_attention(q, *dev, positions, 128 ** -0.5)))
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for k, (side, (dev, q, new, first, counts, positions, _)) in enumerate(zip(sides, runs)):
            with torch.cuda.stream(side):
                wb.paged_append(*dev, new, first, counts)  # the same entries again
                got[k].append(wb.paged_attention(q, *dev, positions, 128 ** -0.5))
    torch.cuda.synchronize()
    for outs, run in zip(got, runs):
        for out in outs:
            assert torch.equal(out[0], run[-1][0]) and torch.equal(out[1], run[-1][1])
    assert wb.device_status() == 0


def test_offsets_past_32_bits(wb):
    """A pool of 5 GB: rows on its last pages, on its first, and on both."""
    g = torch.Generator().manual_seed(25)
    B, n, S, M, P = 3, 50, 64, 2, 327_680
    pages, scales = wb.paged_cache(P, S, 128)
    assert pages.numel() > 2 ** 32
    table = torch.tensor([[P - 1, P - 2], [0, 1], [2, P - 3]])
    new = torch.randn(B, n, 256, generator=g).bfloat16()
    first, counts = torch.tensor([70, 0, 40]), torch.tensor([50, 50, 50])
    wb.paged_append(pages, scales, table.cuda(), new.cuda(), first.cuda(), counts.cuda())
    used = torch.tensor([P - 1, P - 2, 0, 1, 2, P - 3])
    near = torch.tensor([[0, 1], [2, 3], [4, 5]])
    few = pages.view(torch.uint8)[used.cuda()].view(torch.float8_e4m3fn), scales[used.cuda()]
    empty = dict(values=np.zeros((6, S, 256)), scales=np.zeros((6, S // 16, 2)))
    _check_append(few, empty, near, new, first, counts)
    q, positions = _queries(B, 1, 8, g), (first + n - 1)[:, None]
    got = wb.paged_attention(q.cuda(), pages, scales, table.cuda(), positions.cuda(), 128 ** -0.5)
    _check_attention(got, q, _cache(*few), near, positions, 128 ** -0.5)
    assert wb.device_status() == 0


def test_refusals(wb):
    pages, scales = wb.paged_cache(4, 32, 128)
    table, p = torch.zeros(2, 3, dtype=torch.int32, device="cuda"), torch.zeros(2, 1, dtype=torch.int64, device="cuda")
    q = torch.zeros(2, 1, 4, 128, device="cuda").bfloat16()
    attend = dict(q=q, pages=pages, scales=scales, table=table, positions=p, scale=1.0)
    for bad in (dict(q=q.float()), dict(pages=pages.view(torch.uint8)), dict(scales=scales.double()),
                dict(q=torch.zeros(2, 1, 65, 128, device="cuda").bfloat16())):
        with pytest.raises(NotImplementedError):
            wb.paged_attention(**(attend | bad))
    for bad in (dict(scales=scales[:, :1]), dict(table=table[:1]), dict(table=table.float()), dict(table=table[0]),
                dict(q=q[..., :64]), dict(positions=p[:1, :0]), dict(window=-1), dict(sink=torch.zeros(3, device="cuda")),
                dict(pages=pages[..., :128]), dict(positions=p.cpu()), dict(scales=scales.cpu()),
                dict(pages=pages[:, :, 8:136])):
        with pytest.raises(ValueError):
            wb.paged_attention(**(attend | bad))
    new = torch.zeros(2, 3, 256, device="cuda")
    append = dict(pages=pages, scales=scales, table=table, new=new, first=p[:, 0], counts=p[:, 0])
    f = wb.rotary_frequencies(64, device="cuda")
    with pytest.raises(NotImplementedError):
        wb.paged_append(**(append | dict(new=new.half())))
    for bad in (dict(new=new[..., :128]), dict(new=new[:1]), dict(first=p), dict(counts=p[:1, 0]), dict(new=new.cpu()),
                dict(frequencies=f, start=65), dict(frequencies=f.cpu()), dict(frequencies=f, positions=p)):
        with pytest.raises(ValueError):
            wb.paged_append(**(append | bad))
    for args in ((2, 48, 128), (2, 192, 128), (2, 0, 128), (2, 32, 24), (2, 32, 1024)):
        with pytest.raises(NotImplementedError):
            wb.paged_cache(*args)
    assert not pages.view(torch.uint8).any()
