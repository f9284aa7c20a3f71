"""Eviction by accumulated attention weight on the GPU where it can go wrong:
NaN and infinities beside padding columns, broken queries, items that a CTA
takes one after the other, long runs of columns; the weights' accuracy at
ordinary inputs; eviction at odd offsets, in a graph and on another stream.

The float64 values of the larger cases are worked out on the GPU with torch."""

import math
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from oracle import budget as ob

pytestmark = pytest.mark.gpu

# A term exp(x), x = scale q.k - lse in fp32, for normalised inputs (scores of
# standard deviation 1, lse under 10): the product is summed in C / 16 <= 8
# steps, each of which may drop 2^-23 of a sum of size 1, all in one direction:
# 9.5e-7 of the term. The other roundings (of lse in base 2 and of the exponent,
# 2^-24 of at most 16; the exponential, 2^-22; the sums) have independent signs
# and partly cancel over the at least 12 columns of a key: 3e-7. So a norm of
# errors is under 1.3e-6 of the norm of what was added. One weight alone, and the
# largest of the terms that it adds up, may be off by their plain sum with scores
# up to 6: 6 * 9.5e-7 + 2 * 2^-24 * 16 + 2^-22 = 8e-6.
NORM, EACH = 1.3e-6, 8e-6

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def wb():
    import wpt_b200
    from wpt_b200 import build
    build.build()
    return wpt_b200


def _reference(q, k, positions, scale, start, window=0, floor=None):
    """(lse fp32, weights float64) of queries on the GPU, in float64."""
    B, T, H, C = q.shape
    N = k.shape[1]
    n = torch.arange(N, device=q.device)
    lse = torch.empty(B, T, H, device=q.device)
    out = start.double()
    step = max(1, 2 ** 25 // (H * N))
    for b in range(B):
        keys = k[b].double()
        for t in range(0, T, step):
            p = positions[b, t:t + step, None]
            seen = n <= p
            if window:
                seen = seen & (n > p - window)
            if floor is not None:
                seen = seen & (n >= floor[b, t:t + step, None])
            s = torch.matmul(q[b, t:t + step].double().reshape(-1, C), keys.t()).view(-1, H, N) * scale
            s = s.masked_fill(~seen[:, None], -math.inf)
            lse[b, t:t + step] = torch.logsumexp(s, -1).float()
            term = torch.exp(s - lse[b, t:t + step, :, None].double())
            out[b] += torch.where(seen[:, None], term, 0.0).sum((0, 1))
    return lse, out


def _inputs(B, T, H, C, N, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randn(B, T, H, C, generator=g, device="cuda").bfloat16()
    k = torch.randn(B, N, C, generator=g, device="cuda").bfloat16()
    return g, q, k


def _check(wb, got, ref, start, norm=NORM):
    add = ref - start.double()
    off = (got.double() - ref).abs() - 2.0 ** -23 * ref.abs()  # less the addition to the old weight
    assert (off <= EACH * add + 1e-30).all(), (off / add.clamp_min(1e-30)).max()
    assert off.clamp_min(0).norm() <= norm * add.norm() + 1e-30
    assert wb.device_status() == 0


@pytest.mark.parametrize("B, T, H, C, N", [(3, 1, 16, 128, 900), (3, 1, 12, 64, 700), (2, 5, 20, 128, 600),
                                           (2, 16, 16, 128, 500), (2, 40, 16, 128, 700), (5, 37, 12, 64, 1007)])
def test_weights_are_within_a_few_roundings(wb, B, T, H, C, N):
    _, q, k = _inputs(B, T, H, C, N)
    positions = (N - T + torch.arange(T, device="cuda")).expand(B, T).contiguous()
    start = torch.zeros(B, N, device="cuda")
    lse, ref = _reference(q, k, positions, C ** -0.5, start)
    _check(wb, wb.attention_weights(q, k, positions, lse, C ** -0.5), ref, start)


# ------------------------------------------------- NaN, infinities and padding

@pytest.mark.parametrize("T, H", [(2, 6), (2, 12), (2, 33), (3, 70), (2, 150)])
@pytest.mark.parametrize("floored", [False, True])
@pytest.mark.parametrize("poison", [math.nan, math.inf, -math.inf])
def test_rows_between_the_queries_rows_keep_their_weight(wb, T, H, floored, poison):
    """What rows that no query reads hold reaches no weight, padding columns (T * H is no tile's width) or not."""
    B, C, N = 2, 128, 400
    g, q, k = _inputs(B, T, H, C, N)
    positions = torch.tensor([10, 300, 305][:T], device="cuda").expand(B, T).contiguous()
    floor = (positions - 7).contiguous() if floored else None
    window = 0 if floored else 8
    start = torch.rand(B, N, generator=g, device="cuda")
    lse, ref = _reference(q, k, positions, C ** -0.5, start, window, floor)
    read = torch.zeros(N, dtype=torch.bool, device="cuda")
    for p in positions[0].tolist():
        read[p - 7:p + 1] = True
    k[:, ~read] = poison
    got = wb.attention_weights(q, k, positions, lse, C ** -0.5, start.clone(), window=window, floor=floor)
    assert torch.equal(got[:, ~read], start[:, ~read])
    _check(wb, got[:, read], ref[:, read], start[:, read], norm=EACH)


@pytest.mark.parametrize("T, H", [(1, 1), (1, 12), (1, 16), (1, 40), (1, 100), (3, 43), (1, 300), (1, 129), (1, 260)])
def test_a_key_of_minus_infinity_gets_no_weight(wb, T, H):
    """A row whose scores are all -inf adds exp(-inf) = 0, padding columns or not."""
    B, C, N = 2, 64, 300
    g, q, k = _inputs(B, T, H, C, N)
    q[..., 5] = q[..., 5].abs() + 0.5
    positions = (N - 1 + torch.arange(T, device="cuda")).expand(B, T).contiguous()  # every row is read by all
    start = torch.rand(B, N, generator=g, device="cuda")
    k[:, 7, 5] = k[:, 200, 5] = -math.inf
    lse, ref = _reference(q, k, positions, C ** -0.5, start)
    got = wb.attention_weights(q, k, positions, lse, C ** -0.5, start.clone())
    assert torch.equal(got[:, [7, 200]], start[:, [7, 200]])
    _check(wb, got, ref, start, norm=EACH)


@pytest.mark.parametrize("T, H", [(1, 16), (1, 24), (9, 8), (40, 16), (37, 12)])
@pytest.mark.parametrize("broken", ["query", "lse"])
def test_a_broken_column_shows_in_every_row_that_it_reads(wb, T, H, broken):
    """A NaN query or lse makes all the weights that it adds to NaN, in whichever column and form; the others stay."""
    B, C, N = 1, 128, 700
    _, q, k = _inputs(B, T, H, C, N)
    positions = torch.full((B, T), N - 1, device="cuda")
    positions[0, 0] = 300
    start = torch.zeros(B, N, device="cuda")
    lse, ref = _reference(q, k, positions, C ** -0.5, start)
    for h in range(min(H, 16)):
        bad_q, bad_lse = q.clone(), lse.clone()
        if broken == "query":
            bad_q[0, 0, h, 3] = math.nan
        else:
            bad_lse[0, 0, h] = math.nan
        got = wb.attention_weights(bad_q, k, positions, bad_lse, C ** -0.5)
        assert got[0, :301].isnan().all(), h
        _check(wb, got[:, 301:], ref[:, 301:], start[:, 301:], norm=EACH)


@pytest.mark.parametrize("T, H", [(1, 16), (40, 16)])
def test_extreme_log_sums(wb, T, H):
    """lse +inf adds nothing, -inf neither; one far under the scores gives +inf, in every column."""
    B, C, N = 1, 128, 300
    _, q, k = _inputs(B, T, H, C, N)
    positions = torch.full((B, T), N - 1, device="cuda")
    for value in (math.inf, -math.inf):
        got = wb.attention_weights(q, k, positions, torch.full((B, T, H), value, device="cuda"), C ** -0.5)
        assert (got == 0).all()
    lse, _ = _reference(q, k, positions, C ** -0.5, torch.zeros(B, N, device="cuda"))
    for h in range(H):
        low = lse.clone()
        low[0, 0, h] = -1000.0
        assert (wb.attention_weights(q, k, positions, low, C ** -0.5) == math.inf).all(), h


# ------------------------------------------- the query-stream form's machinery

def _runs(wb, B, T, H, N):
    """Runs that each key's column tiles are summed in: from the scratch's size, which holds a sum a run and key."""
    from wpt_b200 import _lib
    size = _lib.lib().wpt_attn_weights_scratch_bytes(B, T, H, N)
    tiles = -(-T * H // 128)
    sums = size - 16 - B * tiles * (16 + 128 * 12)
    return tiles, max(1, sums // (4 * B * N))


LONG = [
    # B, T, H, C, N, window, ragged, floored, column tiles a run
    (8, 1600, 32, 64, 1501, 0, False, False, 16),   # 400 column tiles: 600 items of 4 key tiles, several a CTA
    (8, 1600, 32, 128, 1501, 200, True, True, 16),  # items that no query reads among them
    (5, 1252, 32, 128, 1301, 0, True, False, 8),
    (3, 900, 24, 64, 2501, 300, True, False, 4),
    (150, 17, 16, 128, 333, 0, True, True, 3),      # an item a row and CTA, and some over; three column tiles
    (1, 2200, 64, 128, 17409, 0, False, False, 32),  # runs of more than 16 column tiles
]


@pytest.mark.parametrize("case", LONG, ids=lambda c: "x".join(map(str, c[:6])) + "rf"[:c[6] + c[7]])
def test_items_one_after_the_other(wb, case):
    B, T, H, C, N, window, ragged, floored, run = case
    tiles, runs = _runs(wb, B, T, H, N)
    assert runs == -(-tiles // run)
    assert B * -(-N // 512) * runs > 148  # even with four key tiles an item, some CTA takes a second one
    g, q, k = _inputs(B, T, H, C, N)
    lengths = torch.randint(0, N + 1, (B,), generator=g, device="cuda") if ragged else torch.full((B,), N, device="cuda")
    positions = lengths[:, None] - T + torch.arange(T, device="cuda")
    floor = torch.randint(-3, N + 3, (B, T), generator=g, device="cuda") if floored else None
    start = torch.rand(B, N, generator=g, device="cuda")
    lse, ref = _reference(q, k, positions, C ** -0.5, start, window, floor)
    args = (q, k, positions, lse, C ** -0.5)
    got = wb.attention_weights(*args, start.clone(), window=window, floor=floor)
    # the runs' sums and a run's own are of up to thousands of terms, each addition 2^-24 of the running sum, at
    # random signs: 64 roundings and more, 4e-6 of it
    assert wb.device_status() == 0
    add = ref - start.double()
    off = (got.double() - ref).abs() - 2.0 ** -23 * ref.abs()
    assert (off <= 2 * EACH * add + 1e-30).all(), (off / add.clamp_min(1e-30)).max()
    assert off.clamp_min(0).norm() <= 4 * NORM * add.norm()
    assert torch.equal(got, wb.attention_weights(*args, start.clone(), window=window, floor=floor))


# ------------------------------------------------------------------ arguments

def test_positions_of_one_row_serve_every_row(wb):
    _, q, k = _inputs(3, 2, 16, 128, 50)
    one = torch.tensor([[30, 31]], device="cuda")
    _, lse = wb.forward_with_lse(q, k, k, one, 0.1)
    assert torch.equal(wb.attention_weights(q, k, one, lse, 0.1),
                       wb.attention_weights(q, k, one.expand(3, 2).contiguous(), lse, 0.1))
    with pytest.raises(ValueError):
        wb.attention_weights(q, k, one.expand(2, 2), lse, 0.1)


def test_a_window_past_32_bits_is_no_window(wb):
    _, q, k = _inputs(2, 1, 16, 128, 300)
    positions = torch.full((2, 1), 299, device="cuda")
    _, lse = wb.forward_with_lse(q, k, k, positions, 0.1)
    every = wb.attention_weights(q, k, positions, lse, 0.1)
    assert torch.equal(wb.attention_weights(q, k, positions, lse, 0.1, window=2 ** 32 + 5), every)
    assert torch.equal(wb.attention_weights(q, k, positions, lse, 0.1, window=2 ** 31), every)
    with pytest.raises(ValueError):
        wb.attention_weights(q, k, positions, lse, 0.1, window=-2 ** 32 + 5)


# ------------------------------------------------------------------- eviction

def _evict_case(B, N, width, seed=0):
    g = torch.Generator().manual_seed(seed)
    held = torch.randn(B, N, width, generator=g).bfloat16()
    weights = torch.rand(B, N, generator=g)
    lengths = torch.randint(N // 2, N + 1, (B,), generator=g)
    return held, weights, lengths


def _same(got, ref):
    return np.array_equal(got[0].cpu().view(torch.int16).numpy(), ref[0]) and all(
        np.array_equal(a.cpu().numpy(), b) for a, b in zip(got[1:], ref[1:]))


def test_cache_evict_at_offsets_of_two_bytes(wb):
    held, weights, lengths = _evict_case(3, 200, 24)
    ref = ob.evict(held.view(torch.int16).numpy(), weights.numpy(), lengths.numpy(), 50, 7, 3)
    for width, at in ((25, 1), (26, 1), (25, 0)):  # odd strides, an odd offset
        big = torch.zeros(3, 200, width, dtype=torch.bfloat16, device="cuda")
        big[..., at:at + 24] = held.cuda()
        assert _same(wb.cache_evict(big[..., at:at + 24], weights.cuda(), lengths.cuda(), 50, 7, 3), ref)


@pytest.mark.parametrize("B, N, keep", [(3, 500, 100), (2, 30000, 9000)])
def test_cache_evict_replays_in_a_graph_and_on_another_stream(wb, B, N, keep):
    held, weights, lengths = _evict_case(B, N, 64)
    ref = ob.evict(held.view(torch.int16).numpy(), weights.numpy(), lengths.numpy(), keep, 7, 3)
    args = held.cuda(), weights.cuda(), lengths.cuda(), keep, 7, 3
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = wb.cache_evict(*args)
    stream.synchronize()
    assert _same(got, ref)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = wb.cache_evict(*args)
    for t in got:
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert _same(got, ref)


def test_cache_evict_of_tables_past_32_bits_is_refused(wb):
    n = torch.ones(1, dtype=torch.int64, device="cuda")
    long = torch.zeros(1, 1, device="cuda").expand(1, 2 ** 32 + 5)
    with pytest.raises(NotImplementedError):
        wb.cache_evict(long[..., None], long, n, 1)
    held, weights = torch.zeros(1, 4, 8, device="cuda"), torch.zeros(1, 4, device="cuda")
    with pytest.raises(NotImplementedError):
        wb.cache_evict(held, weights, n, 1, capacity=2 ** 32 + 5)
    with pytest.raises(NotImplementedError):
        wb.cache_evict(held, weights, n, 2 ** 32 + 5)
    with pytest.raises(NotImplementedError):
        wb.cache_evict(torch.zeros(1, device="cuda").expand(1, 4, 2 ** 30 + 4), weights, n, 1)


def test_threads_evict_tables_of_all_lengths(wb):
    """Each thread's calls ask for shared memory of their own size, from the process's first calls on."""
    code = """
import threading, torch, wpt_b200
start, failed = threading.Barrier(8), []
cases = []
for n in range(1, 13):
    cases.append((torch.arange(4096.0 * n).flip(0).view(1, -1).cuda(), torch.tensor([4096 * n]).cuda()))
def work(t):
    try:
        start.wait()
        with torch.cuda.stream(torch.cuda.Stream()):
            for i in range(120):
                w, n = cases[(i * (2 * t + 1) + t) % 12]
                rows = wpt_b200.cache_evict(w[..., None], w, n, 9)[2]
                torch.cuda.current_stream().synchronize()
                if rows.tolist() != [list(range(9))]:
                    failed.append((t, i, rows.tolist()))
    except BaseException as e:
        failed.append((t, repr(e)))
threads = [threading.Thread(target=work, args=(t,)) for t in range(8)]
torch.cuda.synchronize()
[t.start() for t in threads]
[t.join() for t in threads]
assert not failed, failed
print("done")
"""
    for _ in range(3):
        run = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
        assert run.returncode == 0 and run.stdout.strip() == "done", run.stderr[-2000:]
