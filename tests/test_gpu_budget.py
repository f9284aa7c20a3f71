"""Eviction by accumulated attention weight on the GPU against the float64
restatement (oracle/budget.py): the weights that cached rows collect, in both
kernel forms (up to 256 (query, head) columns the keys stream past the
queries, above that the queries past the keys), and the rows a budget keeps.

Tolerance of a weight, relative to its float64 value. A term is exp(x) with
x = scale q.k - lse computed in fp32: bf16 products are exact; their sum of C
<= 128 terms is off by at most C roundings (or truncations, 2^-23 each) of a
running sum that stays under A = scale sum |q||k| <= 2 C scale max|q||k|'s
observed bound, here A < 32; lse in base 2 and the final sum round to 2^-24
of at most 64 each. So |dx| <= 128 * 2^-23 * 32 + 2 * 64 * 2^-24 = 5e-4 in
the worst case and a hundredth of that at random signs. WORST is that bound
on every weight; TYPICAL, a twentieth of it, on the error's 2-norm over the
weights' (roundings of independent signs). Terms are positive, so the sum
over columns cannot lose more."""

import numpy as np
import pytest
import torch

from oracle import budget as ob

pytestmark = pytest.mark.gpu

WORST, TYPICAL = 5e-4, 2.5e-5


@pytest.fixture(scope="module")
def wb():
    import wpt_b200
    from wpt_b200 import build
    build.build()
    return wpt_b200


def _np(t):
    return t.float().cpu().numpy().astype(np.float64)


def _weights_case(B, T, H, C, N, window, ragged, floored, seed=0):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(B, T, H, C, generator=g).bfloat16()
    entries = torch.randn(B, N, 2 * C, generator=g).bfloat16()
    lengths = torch.randint(0, N + 1, (B,), generator=g) if ragged else torch.full((B,), N)
    positions = lengths[:, None] - T + torch.arange(T)  # negative: a query before the text reads nothing
    floor = None
    if floored:
        floor = torch.randint(-3, N + 3, (B, T), generator=g)  # above the position: nothing is read
    start = torch.rand(B, N, generator=g)
    scale = C ** -0.5
    lse = torch.from_numpy(ob.log_sums(_np(q), _np(entries[..., :C]), positions.numpy(), scale, window,
                                       None if floor is None else floor.numpy())).float()
    return q, entries, positions, floor, start, lse, scale


def _check_weights(wb, got, ref, start):
    got, ref, start = got.double().cpu().numpy(), ref, start.double().numpy()
    add = ref - start
    # adding to a start under 1 rounds to 2^-24 of the sum, once
    off = np.abs(got - ref) - 2.0 ** -23 * np.abs(ref)
    assert (off <= WORST * add + 1e-30).all(), (off / np.maximum(add, 1e-30)).max()
    # a weight's own roundings: of the running sum and of the last addition
    assert np.linalg.norm(np.maximum(off, 0)) <= TYPICAL * np.linalg.norm(add) + 1e-30
    assert wb.device_status() == 0


SHAPES = [
    # B, T, H, C, N, window, ragged, floored
    (1, 1, 1, 128, 1, 0, False, False),        # one key, one column
    (1, 1, 16, 128, 127, 0, False, False),
    (2, 1, 16, 64, 128, 0, False, False),
    (3, 1, 32, 128, 129, 0, True, False),
    (64, 1, 32, 128, 1300, 0, True, False),    # tiles of rows laid end to end over the CTAs
    (5, 1, 12, 128, 700, 100, True, False),    # window
    (3, 1, 64, 128, 515, 0, True, True),
    (4, 3, 16, 128, 600, 0, True, False),      # 48 columns, several queries
    (4, 5, 5, 64, 333, 50, True, True),        # odd heads, window and floor
    (2, 8, 16, 128, 1000, 0, True, False),     # 128 columns
    (3, 7, 31, 128, 401, 64, True, False),     # 217 columns
    (2, 256, 1, 64, 300, 0, False, False),     # 256 columns of one head
    (1100, 1, 4, 64, 130, 0, True, False),     # more batch rows than are laid end to end
    (1, 257, 1, 128, 257, 0, False, False),    # the first above 256 columns
    (2, 37, 12, 64, 700, 0, True, False),
    (2, 40, 16, 128, 256, 0, False, False),
    (3, 65, 24, 128, 511, 130, True, True),
    (1, 300, 16, 128, 300, 0, False, False),   # a key's columns in several runs
    (2, 700, 8, 64, 900, 200, True, True),
    (1, 33, 130, 128, 140, 0, False, False),   # more heads than a column tile
]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s[:6])) + "rf"[:s[6] + s[7]])
def test_attention_weights(wb, shape):
    B, T, H, C, N, window, ragged, floored = shape
    q, entries, positions, floor, start, lse, scale = _weights_case(*shape)
    ref = ob.attention_weights(_np(q), _np(entries[..., :C]), positions.numpy(), lse.numpy(), scale, start.numpy(),
                               window, None if floor is None else floor.numpy())
    e = entries.cuda()
    args = (q.cuda(), e[..., :C], positions.cuda(), lse.cuda(), scale)
    more = dict(window=window, floor=None if floor is None else floor.cuda())
    got = wb.attention_weights(*args, start.cuda(), **more)
    _check_weights(wb, got, ref, start)
    again = wb.attention_weights(*args, start.cuda(), **more)
    assert torch.equal(got, again)  # a fixed order of sums


@pytest.mark.parametrize("T, H", [(1, 32), (5, 16), (40, 16), (300, 16)])
def test_attention_weights_of_the_forward_pass(wb, T, H):
    """With the library's own lse, each query and head hands out weights that sum to 1 (less the sink's share)."""
    B, C, N = 2, 128, 900
    g = torch.Generator().manual_seed(5)
    q = torch.randn(B, T, H, C, generator=g).bfloat16().cuda()
    e = torch.randn(B, N, 2 * C, generator=g).bfloat16().cuda()
    positions = torch.arange(N - T, N).expand(B, T).contiguous().cuda()
    scale = C ** -0.5
    _, lse = wb.forward_with_lse(q, e[..., :C], e[..., C:], positions, scale)
    w = wb.attention_weights(q, e[..., :C], positions, lse, scale)
    assert w.shape == (B, N) and w.dtype == torch.float32
    # lse is held to 1e-3 by the library's own tests, a factor of the weights
    assert (w.double().sum(1) / (T * H) - 1).abs().max() < 1.5e-3
    sink = torch.full((H,), 2.0, device="cuda")
    _, lse2 = wb.forward_with_lse(q, e[..., :C], e[..., C:], positions, scale, sink=sink)
    w2 = wb.attention_weights(q, e[..., :C], positions, lse2, scale)
    share = torch.exp(lse.double() - lse2.double()).sum((1, 2))
    assert (w2.double().sum(1) / share - 1).abs().max() < 3e-3


@pytest.mark.parametrize("T, H", [(1, 16), (3, 16), (40, 16)])
def test_stale_and_masked_rows_reach_no_other_row(wb, T, H):
    """NaN, infinities and the type's lowest value in rows that no query reads, and in a query without rows."""
    B, C, N, live = 3, 128, 400, 219
    q, entries, _, _, start, _, scale = _weights_case(B, T, H, C, N, 0, False, False)
    positions = (torch.arange(live - T, live)).expand(B, T).clone()
    if T > 1:
        positions[:, 0] = -1
    positions[2] = -1  # no query of this batch row reads anything
    lse = torch.from_numpy(ob.log_sums(_np(q), _np(entries[..., :C]), positions.numpy(), scale)).float()
    ref = ob.attention_weights(_np(q), _np(entries[..., :C]), positions.numpy(), lse.numpy(), scale, start.numpy())
    for poison in (float("nan"), float("inf"), -float("inf"), torch.finfo(torch.bfloat16).min):
        bad, bad_q, bad_start = entries.clone(), q.clone(), start.clone()
        bad[:, live:] = poison
        bad_start[:, live:] = float("nan")
        bad[2] = poison
        if T > 1:
            bad_q[:, 0] = poison
        bad_q[2] = poison
        got = wb.attention_weights(bad_q.cuda(), bad.cuda()[..., :C], positions.cuda(), lse.cuda(), scale,
                                   bad_start.cuda())
        _check_weights(wb, got[:2, :live], ref[:2, :live], start[:2, :live])
        assert got[:, live:].isnan().all()
        assert torch.equal(got[2, :live].cpu(), start[2, :live])


def test_weights_at_strides_on_another_stream(wb):
    B, T, H, C, N = 4, 1, 16, 128, 500
    q, entries, positions, _, start, lse, scale = _weights_case(B, T, H, C, N, 0, True, False)
    ref = ob.attention_weights(_np(q), _np(entries[..., :C]), positions.numpy(), lse.numpy(), scale, start.numpy())
    wide = torch.full((B, N + 37), -1.0, device="cuda")
    wide[:, :N] = start.cuda()
    table = torch.empty(N, B, 3 * C, dtype=torch.bfloat16, device="cuda")  # (N, B) order, a third of wider rows
    table[..., C:2 * C] = entries[..., :C].transpose(0, 1).cuda()
    k = table.transpose(0, 1)[..., C:2 * C]
    qg, pg, lg = q.cuda().transpose(1, 2).contiguous().transpose(1, 2), positions.cuda(), lse.cuda()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = wb.attention_weights(qg, k, pg.int(), lg, scale, wide[:, :N])
    stream.synchronize()
    assert got.data_ptr() == wide.data_ptr()
    _check_weights(wb, got, ref, start)
    assert (wide[:, N:] == -1).all()


def test_weights_replay_in_a_graph(wb):
    for T in (1, 300):
        q, entries, positions, _, start, lse, scale = _weights_case(2, T, 16, 128, 600, 0, False, False)
        args = (q.cuda(), entries.cuda()[..., :128], positions.cuda(), lse.cuda(), scale)
        once = wb.attention_weights(*args, torch.zeros(2, 600, device="cuda"))
        w = torch.zeros(2, 600, device="cuda")
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            wb.attention_weights(*args, w)
        w.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(w, once)


def test_weights_refusals(wb):
    q = torch.zeros(2, 1, 4, 128, dtype=torch.bfloat16, device="cuda")
    k = torch.zeros(2, 10, 128, dtype=torch.bfloat16, device="cuda")
    positions = torch.zeros(2, 1, dtype=torch.int64, device="cuda")
    lse = torch.zeros(2, 1, 4, device="cuda")
    w = torch.zeros(2, 10, device="cuda")
    with pytest.raises(NotImplementedError):
        wb.attention_weights(q.float(), k, positions, lse, 1.0, w)
    with pytest.raises(NotImplementedError):
        wb.attention_weights(q[..., :96].contiguous(), k[..., :96].contiguous(), positions, lse, 1.0, w)
    with pytest.raises(ValueError):
        wb.attention_weights(q, k, positions, lse[:, :, :3], 1.0, w)
    with pytest.raises(ValueError):
        wb.attention_weights(q, k, positions, lse, 1.0, w.double())
    with pytest.raises(ValueError):
        wb.attention_weights(q, k, positions, lse, 1.0, torch.zeros(10, 2, device="cuda").t())
    with pytest.raises(ValueError):
        wb.attention_weights(q, k, positions, lse.cpu(), 1.0, w)
    with pytest.raises(ValueError):
        wb.attention_weights(q, k, positions, lse, 1.0, w, window=-1)
    empty = wb.attention_weights(q[:, :0], k, positions[:, :0], lse[:, :0], 1.0, w)
    assert empty is w and not w.any()


# ------------------------------------------------------------------ eviction

def _evict_case(B, N, width, dtype, kind, seed=0):
    g = torch.Generator().manual_seed(seed)
    held = torch.randn(B, N, *width, generator=g).to(dtype)
    weights = torch.exp(2 * torch.randn(B, N, generator=g) - 4)
    if kind == "ties":
        weights = (weights * 20).round() / 4  # few values, most of them equal
    elif kind == "equal":
        weights = torch.full((B, N), 0.25)
    elif kind == "strange":
        pick = torch.randint(0, 8, (B, N), generator=g)
        for i, x in enumerate((float("nan"), float("inf"), -float("inf"), 0.0, -0.0, -3.5)):
            weights = torch.where(pick == i, x, weights)
    lengths = torch.randint(0, N + 1, (B,), generator=g)
    lengths[0] = N
    return held, weights, lengths


EVICT = [
    # B, N, entry, dtype, keep, recent, first, capacity, kind
    (1, 1, (8,), torch.bfloat16, 1, 0, 0, 1, "plain"),
    (1, 2, (8,), torch.bfloat16, 1, 0, 0, 1, "plain"),
    (3, 31, (16,), torch.bfloat16, 7, 2, 1, 9, "plain"),
    (4, 1000, (256,), torch.bfloat16, 300, 16, 4, 300, "plain"),
    (5, 1024, (3,), torch.float32, 1023, 0, 0, 1024, "ties"),       # 12-byte entries
    (2, 1025, (24,), torch.bfloat16, 512, 512, 0, 512, "plain"),    # nothing but the recent rows
    (2, 1025, (2, 12), torch.bfloat16, 512, 0, 512, 600, "plain"),  # nothing but the first rows
    (3, 5000, (8,), torch.float32, 700, 0, 0, 700, "equal"),
    (3, 5000, (8,), torch.float32, 700, 33, 5, 700, "strange"),
    (3, 300, (8,), torch.float32, 299, 3, 5, 299, "strange"),
    (1, 20001, (8,), torch.bfloat16, 5000, 64, 4, 5000, "ties"),    # a cluster of CTAs a row
    (2, 70001, (4,), torch.bfloat16, 35000, 0, 3, 35000, "ties"),
    (1, 262144, (2,), torch.float32, 100000, 1000, 4, 100000, "plain"),
    (1, 400003, (1,), torch.float32, 1, 0, 0, 1, "plain"),          # slices longer than shared memory holds
    (150, 60000, (1,), torch.float32, 999, 9, 1, 999, "ties"),      # the same, one CTA a row
    (3, 100, (8,), torch.bfloat16, 0, 0, 0, 5, "plain"),            # nothing is kept
    (3, 100, (8,), torch.bfloat16, 100, 0, 0, 100, "plain"),        # everything is
]


@pytest.mark.parametrize("case", EVICT, ids=lambda c: f"{c[0]}x{c[1]}-keep{c[4]}-{c[8]}")
def test_cache_evict(wb, case):
    B, N, width, dtype, keep, recent, first, capacity, kind = case
    held, weights, lengths = _evict_case(B, N, width, dtype, kind)
    as_int = torch.int16 if dtype == torch.bfloat16 else torch.int32
    ref = ob.evict(held.view(as_int).numpy(), weights.numpy(), lengths.numpy(), keep, recent, first, capacity)
    out, out_weights, rows, counts = wb.cache_evict(held.cuda(), weights.cuda(), lengths.cuda(), keep, recent, first,
                                                    capacity)
    assert np.array_equal(counts.cpu().numpy(), ref[3])
    assert np.array_equal(rows.cpu().numpy(), ref[2])
    assert out.shape == (B, capacity) + width and out.dtype == dtype
    assert np.array_equal(out.cpu().view(as_int).numpy(), ref[0])
    assert np.array_equal(out_weights.cpu().numpy(), ref[1], equal_nan=True)
    assert wb.device_status() == 0


def test_cache_evict_at_strides(wb):
    held, weights, lengths = _evict_case(3, 500, (24,), torch.bfloat16, "plain")
    lengths[1], lengths[2] = -4, 1 << 40  # clamped to the table
    ref = ob.evict(held.view(torch.int16).numpy(), weights.numpy(), lengths.numpy(), 100, 7, 3)
    big = torch.zeros(500, 3, 50, dtype=torch.bfloat16, device="cuda")
    big[..., 2:26] = held.transpose(0, 1).cuda()  # 4-byte aligned only
    wide = torch.zeros(3, 777, device="cuda")
    wide[:, 5:505] = weights.cuda()
    for table, w in ((big.transpose(0, 1)[..., 2:26], wide[:, 5:505]), (held.cuda(), weights.t().contiguous().cuda().t()),
                     (held.permute(2, 0, 1).contiguous().cuda().permute(1, 2, 0), weights.cuda())):
        out, out_weights, rows, counts = wb.cache_evict(table, w, lengths.cuda().int() if w is wide else lengths.cuda(),
                                                        100, 7, 3)
        assert np.array_equal(rows.cpu().numpy(), ref[2]) and np.array_equal(counts.cpu().numpy(), ref[3])
        assert np.array_equal(out.cpu().view(torch.int16).numpy(), ref[0])
        assert np.array_equal(out_weights.cpu().numpy(), ref[1])


def test_cache_evict_refusals(wb):
    held = torch.zeros(2, 10, 8, device="cuda")
    w, n = torch.zeros(2, 10, device="cuda"), torch.full((2,), 10, device="cuda")
    for bad in (dict(keep=-1), dict(keep=4, recent=3, first=2), dict(keep=4, recent=-1), dict(keep=4, capacity=3)):
        with pytest.raises(ValueError):
            wb.cache_evict(held, w, n, **bad)
    with pytest.raises(ValueError):
        wb.cache_evict(held, w[:, :9], n, 4)
    with pytest.raises(ValueError):
        wb.cache_evict(held, w.double(), n, 4)
    with pytest.raises(ValueError):
        wb.cache_evict(held.cpu(), w, n, 4)
    with pytest.raises(NotImplementedError):
        wb.cache_evict(held[..., :1].bfloat16(), w, n, 4)  # 2-byte entries
    out, out_weights, rows, counts = wb.cache_evict(held[:0], w[:0], n[:0], 4)
    assert out.shape == (0, 4, 8) and rows.shape == (0, 4)
    out, out_weights, rows, counts = wb.cache_evict(held[:, :0], w[:, :0], n, 4)
    assert not out.any() and not out_weights.any() and (rows == -1).all() and not counts.any()


def test_positions_of_one_pass_serve_every_row(wb):
    q, entries, positions, _, start, lse, scale = _weights_case(3, 2, 16, 128, 50, 0, False, False)
    args = (q.cuda(), entries.cuda()[..., :128])
    each = wb.attention_weights(*args, positions.cuda(), lse.cuda(), scale, start.cuda())
    one = wb.attention_weights(*args, positions[0].cuda(), lse.cuda(), scale, start.cuda())
    assert torch.equal(each, one)
    assert torch.equal(wb.attention_weights(*args, positions.cuda(), lse.cuda(), scale) > 0,
                       torch.ones(3, 50, dtype=torch.bool, device="cuda"))


def test_a_small_weight_comes_back_exactly(wb):
    """Weights under 2^-126 and zeros of both signs are kept as they are."""
    w = torch.tensor([[1e-42, -0.0, 0.0, -1e-42, 1.0, 2e-42, -2.0, 3.0]]).cuda()
    held = torch.arange(8.0).view(1, 8, 1).cuda()
    out, kept, rows, _ = wb.cache_evict(held, w, torch.tensor([8]).cuda(), 5)
    assert rows.tolist() == [[0, 1, 4, 5, 7]]
    assert torch.equal(kept.view(torch.int32), w[:, [0, 1, 4, 5, 7]].view(torch.int32))
