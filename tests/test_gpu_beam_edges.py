"""Beam search's step on the GPU where it can go wrong: masks of large finite
values, values that tie only after rounding, refusals that change nothing,
replay in a graph and other streams. Values against oracle/beam.py."""

import math

import numpy as np
import pytest
import torch

from oracle import beam as ob

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def wb():
    import wpt_b200
    from wpt_b200 import build
    build.build()
    return wpt_b200


# ------------------------------------------------------- large finite scores

# An ordinary value is within 5e-5 of its float64 one (log s of a sum in fp32,
# three roundings under 64); a value of any size is rounded three more times,
# to 2^-24 of itself.
TOL = 5e-5


def _check_values(wb, got, scores, totals, beams):
    out, parents, tokens = (t.cpu().numpy() for t in got)
    x, t = scores.float().cpu().numpy(), totals.cpu().numpy()
    ref, ref_parents, ref_tokens = ob.select(x, t, beams)
    V = x.shape[-1]
    every = ob.values(x, t)
    for r in range(x.shape[0]):
        some = ref[r] > -np.inf
        # a float64 value past fp32's range is no candidate in fp32
        assert (out[r] > -np.inf).sum() == (ref[r] > -3.4e38).sum()
        some &= out[r] > -np.inf
        tol = TOL + 4 * 2.0 ** -24 * np.abs(ref[r][some])
        assert (np.abs(out[r][some] - ref[r][some]) <= tol).all(), (r, out[r], ref[r])
        flat = parents[r][some] * V + tokens[r][some]
        assert len(set(flat.tolist())) == some.sum()
        assert (np.abs(every[r, flat] - out[r][some]) <= tol).all()
        order = np.sort(every[r])[::-1]
        for i in np.flatnonzero(some):
            near = np.abs(order - ref[r, i]) <= 2 * (TOL + 4 * 2.0 ** -24 * abs(ref[r, i]))
            if near.sum() == 1:
                assert (parents[r, i], tokens[r, i]) == (ref_parents[r, i], ref_tokens[r, i])
    assert wb.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("mask", [-1e8, -5.3e8, -5.5e8, -1e9, -5e9, -1e10, -1e11, -1e12, -1e15, -1e20, -1e30, 3e9, 1e12])
def test_masks_of_large_finite_values(wb, mask, dtype):
    """Texts with some, all but one, the first half and all of a beam's tokens at the mask's value."""
    V = 30011
    g = torch.Generator().manual_seed(8)
    scores = torch.randn(5, 2, V, generator=g) * 2
    hidden = torch.zeros(5, 2, V, dtype=torch.bool)
    hidden[0] = torch.rand(2, V, generator=g) < 0.5
    hidden[1, :, :V // 2] = True              # whole runs, and all that some threads read
    hidden[2] = True
    hidden[2, 0, 20000] = hidden[2, 1, 5] = False
    hidden[3] = True
    hidden[4, 1] = True                       # one beam of two
    scores = scores.masked_fill(hidden, mask)
    totals = -3 * torch.rand(5, 2, generator=g)
    x = scores.to(dtype).cuda()
    for beams in (1, 4):
        _check_values(wb, wb.beam_select(x, totals.cuda(), beams), x, totals, beams)
    got = wb.beam_select(x[:, 1:], totals[:, 1:].cuda(), 3)  # one beam in: many runs
    _check_values(wb, got, x[:, 1:], totals[:, 1:], 3)


# --------------------------------------------- values that tie after rounding

def _live(step, spread):
    """A number of live tokens whose log sum is, with values within `spread` of
    the largest, under a fifth of `step` from a multiple of it: at totals that
    are multiples of `step`, in the range where fp32 numbers are that far
    apart, all values round to one, whatever the last digits of the sum."""
    for n in range(4000, 40000):
        low = math.log(n) / step
        if abs(low - round(low)) + spread / step < 0.2:
            return n
    raise AssertionError


# A value is off its float64 one by TOL before its last rounding: a fifth of a
# step and TOL are less than the half that would change the rounding.
@pytest.mark.parametrize("total, step, dtype, spread", [
    (-4096.0, 2.0 ** -11, torch.float32, 100 * 2.0 ** -21),
    (-2.0 ** 20, 0.125, torch.float32, None),             # scores that rise with the token
    (-2.0 ** 22, 0.5, torch.bfloat16, 3 * 2.0 ** -5),
])
@pytest.mark.parametrize("beams", [1, 4, 17, 64])
def test_values_that_tie_after_rounding(wb, total, step, dtype, spread, beams):
    """Equal values go to the lowest beam and token, also where their scores differ."""
    if spread is None:
        n = next(n for n in range(28300, 28200, -1) if abs(math.log(n) / step - round(math.log(n) / step)) < 0.05)
        x = 5 + torch.arange(n) * 2.0 ** -21
        assert TOL / step + 0.05 + n * 2.0 ** -21 / step < 0.45
    else:
        n = _live(step, spread)
        assert 0.2 + TOL / step < 0.45
        levels = round(spread * (2 ** 21 if dtype == torch.float32 else 32))
        g = torch.Generator().manual_seed(1)
        x = 5 + torch.randint(0, levels, (n,), generator=g) * (spread / levels)
    for W in (1, 3):
        V = n + 11
        scores = torch.full((2, W, V), -math.inf)
        scores[:, :, 3:3 + n] = x
        scores = scores.to(dtype).cuda()
        assert torch.equal(scores[0, 0, 3:3 + n].float().cpu(), x.float())
        totals = torch.full((2, W), total)
        totals[1, W - 1] += step  # the last beam of the second text is better
        out, parents, tokens = wb.beam_select(scores, totals.cuda(), beams)
        assert (parents[0] == 0).all() and (parents[1] == W - 1).all()
        want = torch.arange(3, 3 + beams)
        assert torch.equal(tokens[0].cpu(), want) and torch.equal(tokens[1].cpu(), want)
        assert (out == out[:, :1]).all()
        ref = ob.select(scores.float().cpu().numpy(), totals.numpy(), beams)[0]
        assert np.abs(out.cpu().numpy() - ref).max() <= step
    assert wb.device_status() == 0


def test_ties_join_other_candidates(wb):
    """A beam's larger values stay first, then the tie's lowest tokens, whichever run they are in; an ended beam among them."""
    step, total, V = 2.0 ** -11, -4096.0, 60000
    n = _live(step, 4 * 2.0 ** -21)
    scores = torch.full((1, 2, V), -math.inf)
    at = torch.arange(n)
    scores[0, 0, 1000 + at] = 5 + (at % 5) * 2.0 ** -21
    scores[0, 1, :2] = 0.0
    # beam 1 offers two values above the tie, ln 2 under its total
    totals = torch.tensor([[total, total - 2.0]])
    out, parents, tokens = wb.beam_select(scores.cuda(), totals.cuda(), 5)
    assert parents.tolist() == [[1, 1, 0, 0, 0]] and tokens.tolist() == [[0, 1, 1000, 1001, 1002]]
    done = torch.tensor([[False, True]])
    tie = round((total - math.log(n)) / step) * step
    out, parents, tokens = wb.beam_select(scores.cuda(), torch.tensor([[total, tie]]).cuda(), 4, done=done.cuda(), end=7)
    assert parents.tolist() == [[0, 0, 0, 0]] and tokens.tolist() == [[1000, 1001, 1002, 1003]] and (out == tie).all()
    out, parents, tokens = wb.beam_select(scores.flip(1).contiguous().cuda(), torch.tensor([[tie, total]]).cuda(), 4,
                                          done=done.flip(1).cuda(), end=7)
    assert parents.tolist() == [[0, 1, 1, 1]] and tokens.tolist() == [[7, 1000, 1001, 1002]] and (out == tie).all()


# ------------------------------------------------------------------- refusals

def test_numbers_past_32_bits_are_refused(wb):
    x, t = torch.zeros(2, 3, 10, device="cuda"), torch.zeros(2, 3, device="cuda")
    done = torch.ones(2, 3, dtype=torch.bool, device="cuda")
    for end in (2 ** 32 + 1, -2 ** 32 + 1, -1):
        with pytest.raises(ValueError):
            wb.beam_select(x, t, 2, done=done, end=end)
    with pytest.raises(NotImplementedError):
        wb.beam_select(x, t, 2 ** 32 + 2)
    wide = torch.zeros(1, 1, 1, device="cuda").expand(1, 1, 2 ** 32 + 10)
    with pytest.raises(NotImplementedError):
        wb.beam_select(wide, t[:1, :1], 2)


def test_tables_that_share_memory_are_refused(wb):
    parents, lengths = torch.tensor([[1, 0, 0]], device="cuda"), torch.full((3,), 10, device="cuda")
    t = torch.randn(3, 10, 8, device="cuda")
    flat = torch.randn(1000, device="cuda")
    was = t.clone()
    for bad in ([t, t], [t, torch.zeros_like(t), t[:, 5:]], [t, t.transpose(0, 1).contiguous().transpose(0, 1), t[..., 4:]],
                flat.as_strided((3, 10, 8), (8, 8, 1)), flat.as_strided((3, 10, 8), (40, 8, 1)),
                flat.as_strided((3, 10, 8), (12, 20, 1))):
        with pytest.raises(ValueError):
            wb.cache_reorder(bad, parents, lengths)
    empty = torch.zeros(3, 0, 8, device="cuda")
    with pytest.raises(ValueError):
        wb.cache_reorder([t, empty, t[..., 4:]], parents, lengths)
    assert torch.equal(t, was)
    # what shares a range of addresses and no byte is taken: the halves of entries, in either order of places
    for big in (torch.randn(3, 10, 16, device="cuda"), torch.randn(10, 3, 16, device="cuda").transpose(0, 1)):
        want = ob.reorder(big.cpu().numpy(), parents.cpu().numpy(), lengths.cpu().numpy())
        wb.cache_reorder([big[..., 8:], big[..., :8]], parents, lengths)
        assert np.array_equal(big.cpu().numpy(), want)
    odd = flat.as_strided((3, 10, 8), (8, 24, 1))
    want = ob.reorder(odd.cpu().numpy(), parents.cpu().numpy(), lengths.cpu().numpy())
    assert np.array_equal(wb.cache_reorder(odd, parents, lengths).cpu().numpy(), want)


def test_a_refused_reorder_moves_nothing(wb):
    tables = [torch.arange(2 * 3.0, device="cuda").view(2, 3, 1) for _ in range(40)]
    was = tables[0].clone()
    tables[35] = torch.zeros(2, 3, 1, dtype=torch.int16, device="cuda")  # 2-byte entries
    with pytest.raises(NotImplementedError):
        wb.cache_reorder(tables, torch.tensor([[1, 0]], device="cuda"), torch.tensor([3, 3], device="cuda"))
    assert all(torch.equal(t, was) for t in tables[:35])


# ----------------------------------------------------------- graphs, streams

def test_reorder_replays_in_a_graph_and_on_another_stream(wb):
    R, W, N = 3, 4, 50
    g = torch.Generator().manual_seed(2)
    start = [torch.randn(R * W, N, 16, generator=g), torch.randn(R * W, N, generator=g)]
    parents = torch.randint(0, W, (R, W), generator=g)
    lengths = torch.randint(1, N + 1, (R * W,), generator=g)
    want = [ob.reorder(t.numpy(), parents.numpy(), lengths.numpy()) for t in start]
    tables = [t.cuda() for t in start]
    on_gpu = parents.cuda(), lengths.cuda()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        wb.cache_reorder(tables, *on_gpu)
    stream.synchronize()
    assert all(np.array_equal(t.cpu().numpy(), w) for t, w in zip(tables, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        wb.cache_reorder(tables, *on_gpu)
    for t, s in zip(tables, start):
        t.copy_(s)
    graph.replay()
    torch.cuda.synchronize()
    assert all(np.array_equal(t.cpu().numpy(), w) for t, w in zip(tables, want))


def test_select_replays_in_a_graph(wb):
    x = torch.randn(3, 4, 5003, generator=torch.Generator().manual_seed(5)).cuda()
    totals = torch.zeros(3, 4, device="cuda")
    want = wb.beam_select(x, totals, 6)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = wb.beam_select(x, totals, 6)
    for t in got:
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("kind", ["masked", "equal"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_equal_scores_cost_no_more_than_a_few_passes(wb, kind, dtype):
    """Most tokens at a finite mask, or all scores equal: within ten times the time of scores that differ (a run's
    scores are then read a few times over, not ranked against each other), and the right choice."""
    R, W, V, beams = 16, 8, 50001, 8
    g = torch.Generator(device="cuda").manual_seed(9)
    plain = torch.randn(R, W, V, generator=g, device="cuda")
    hidden = torch.rand(R, W, V, generator=g, device="cuda") < 0.9999
    scores = dict(masked=plain.masked_fill(hidden, -1e9), equal=torch.zeros_like(plain))[kind].to(dtype)
    plain = plain.to(dtype)
    totals = -torch.rand(R, W, generator=g, device="cuda")

    def time(x):
        wb.beam_select(x, totals, beams)
        best = math.inf
        for _ in range(5):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            for _ in range(10):
                wb.beam_select(x, totals, beams)
            b.record()
            b.synchronize()
            best = min(best, a.elapsed_time(b))
        return best

    assert time(scores) < 10 * time(plain)
    _check_values(wb, wb.beam_select(scores, totals, beams), scores, totals, beams)
    if kind == "equal":
        _, parents, tokens = wb.beam_select(scores, totals, beams)
        assert (parents == totals.argmax(1, keepdim=True)).all() and (tokens == torch.arange(beams, device="cuda")).all()
