"""Beam search's step on the GPU against the float64 restatement
(oracle/beam.py): the selection over beams and vocabulary, and the reordering
of the beams' cached rows.

A value is totals + ((x - m) - log s) in fp32. x - m and the two sums round
to 2^-24 of at most LARGE = 64 each; s is a sum of at most 2^17 positive
terms, each off by 2^-21 (the exponential, its argument's rounding) and each
addition by 2^-24 of the running sum over a tree of depth at most 600 (a
thread's terms, then the block's and the runs'), so log s is off by at most
2^-21 + 600 * 2^-24 = 3.7e-5, and a value by TOL = 3.7e-5 + 3 * 64 * 2^-24 =
5e-5. Choices whose float64 values are further apart than twice that have to
be the oracle's own."""

import numpy as np
import pytest
import torch

from oracle import beam as ob

pytestmark = pytest.mark.gpu

TOL = 5e-5


@pytest.fixture(scope="module")
def wb():
    import wpt_b200
    from wpt_b200 import build
    build.build()
    return wpt_b200


def _check(wb, got, scores, totals, beams, done=None, end=None):
    out, parents, tokens = (t.cpu().numpy() for t in got)
    x = scores.float().cpu().numpy()
    t = totals.cpu().numpy()
    d = None if done is None else done.cpu().numpy()
    ref, ref_parents, ref_tokens = ob.select(x, t, beams, d, end)
    V = x.shape[-1]
    every = ob.values(x, t, d, end)
    assert np.array_equal(out > -np.inf, ref > -np.inf)
    some = ref > -np.inf
    assert np.abs(out[some] - ref[some]).max(initial=0) <= TOL
    assert (parents[~some] == -1).all() and (tokens[~some] == -1).all()
    for r in range(x.shape[0]):
        n = int(some[r].sum())
        flat = parents[r, :n] * V + tokens[r, :n]
        assert len(set(flat.tolist())) == n  # n different candidates, each worth what is said
        assert np.abs(every[r, flat] - out[r, :n]).max(initial=0) <= TOL
        order = np.sort(every[r])[::-1]
        for i in range(n):  # where no other value is near, the choice is the oracle's
            near = np.abs(order[:n + 1] - ref[r, i]) <= 2 * TOL
            if near.sum() == 1:
                assert (parents[r, i], tokens[r, i]) == (ref_parents[r, i], ref_tokens[r, i])
        assert (np.diff(out[r, :n]) <= 0).all()
    assert wb.device_status() == 0


CASES = [
    # R, W, V, beams, dtype
    (1, 1, 1, 1, torch.float32),
    (1, 1, 3, 5, torch.float32),       # fewer candidates than beams
    (2, 3, 17, 64, torch.float32),
    (3, 1, 1000, 4, torch.float32),    # the first step: one beam
    (2, 4, 4096, 4, torch.float32),
    (2, 4, 4097, 4, torch.bfloat16),
    (3, 5, 50021, 7, torch.bfloat16),  # rows that start off the 16-byte boundary
    (3, 5, 50021, 7, torch.float32),
    (1, 4, 65536, 4, torch.float32),
    (40, 16, 5003, 16, torch.float32),
    (2, 64, 9001, 64, torch.float32),
    (2, 64, 9001, 64, torch.bfloat16),
    (1, 2, 131071, 33, torch.float32),
]


@pytest.mark.parametrize("R, W, V, beams, dtype", CASES)
def test_beam_select(wb, R, W, V, beams, dtype):
    g = torch.Generator().manual_seed(R + V)
    scores = (torch.randn(R, W, V, generator=g) * 2).to(dtype).cuda()
    totals = (-20 * torch.rand(R, W, generator=g)).cuda()
    _check(wb, wb.beam_select(scores, totals, beams), scores, totals, beams)
    done = (torch.rand(R, W, generator=g) < 0.4).cuda()
    end = V // 2
    got = wb.beam_select(scores, totals, beams, done=done, end=end)
    _check(wb, got, scores, totals, beams, done, end)
    again = wb.beam_select(scores, totals, beams, done=done, end=end)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("order", ["rising", "falling", "equal", "few", "one"])
@pytest.mark.parametrize("beams", [1, 8, 64])
def test_beam_select_of_hard_orders(wb, order, beams):
    """Sorted scores (every tile beats the one before), equal ones (ties go to the lowest index), few values."""
    V = 30011
    g = torch.Generator().manual_seed(3)
    x = dict(rising=torch.arange(V) / 4096.0, falling=-torch.arange(V) / 4096.0, equal=torch.zeros(V),
             few=torch.randint(0, 3, (V,), generator=g).float(),
             one=torch.where(torch.arange(V) == 20000, 0.0, -float("inf")))[order]
    scores = x.expand(2, 3, V).contiguous().cuda()
    totals = torch.tensor([[0.0, 0.0, 0.0], [-1.0, 0.0, -1.0]]).cuda()
    got = wb.beam_select(scores, totals, beams)
    _check(wb, got, scores, totals, beams)
    if order in ("equal", "few", "one"):
        # equal rows have equal sums whatever their rounding: the choice is the oracle's, ties and all
        ref = ob.select(x.expand(2, 3, V).numpy(), totals.cpu().numpy(), beams)
        assert np.array_equal(got[1].cpu().numpy(), ref[1]) and np.array_equal(got[2].cpu().numpy(), ref[2])


def test_masked_and_broken_scores(wb):
    V = 5000
    g = torch.Generator().manual_seed(4)
    scores = torch.randn(4, 3, V, generator=g)
    totals = torch.zeros(4, 3)
    scores[0, 0] = -float("inf")            # a beam with no token left
    scores[0, 1, 10:] = -float("inf")       # ten tokens left
    scores[1, 0, 7] = float("nan")          # a broken beam
    scores[1, 1, 4999] = float("inf")       # and another
    scores[2, :, 100:] = torch.finfo(torch.float32).min
    totals[2, 0] = -float("inf")            # a dead beam
    scores[3] = -float("inf")               # a text with nothing to say
    for dtype in (torch.float32, torch.bfloat16):
        x = scores.to(dtype).cuda()
        got = wb.beam_select(x, totals.cuda(), 6)
        _check(wb, got, x, totals, 6)
        assert (got[1][1] == 2).all() and (got[1][3] == -1).all() and not (got[1][2] == 0).any()


def test_beam_select_at_strides(wb):
    g = torch.Generator().manual_seed(6)
    big = torch.randn(3, 9, 4, 1203, generator=g).cuda()
    totals = torch.randn(4, 3, generator=g).cuda().t()
    scores = big[:, 8, :, 3:1200]  # the last place of each beam's pass, not the whole vocabulary
    _check(wb, wb.beam_select(scores, totals, 5), scores, totals, 5)
    turned = big[:, 8].transpose(1, 2).contiguous().transpose(1, 2)  # tokens are not contiguous
    _check(wb, wb.beam_select(turned, totals, 5), turned, totals, 5)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = wb.beam_select(scores, totals, 5)
    stream.synchronize()
    _check(wb, got, scores, totals, 5)


def test_beam_select_refusals(wb):
    x, t = torch.zeros(2, 3, 10, device="cuda"), torch.zeros(2, 3, device="cuda")
    with pytest.raises(NotImplementedError):
        wb.beam_select(x.half(), t, 2)
    with pytest.raises(NotImplementedError):
        wb.beam_select(x, t, 65)
    with pytest.raises(NotImplementedError):
        wb.beam_select(torch.zeros(1, 65, 10, device="cuda"), torch.zeros(1, 65, device="cuda"), 2)
    with pytest.raises(ValueError):
        wb.beam_select(x, t, 0)
    with pytest.raises(ValueError):
        wb.beam_select(x, t[:, :2], 2)
    done = torch.zeros(2, 3, dtype=torch.bool, device="cuda")
    with pytest.raises(ValueError):
        wb.beam_select(x, t, 2, done=done)
    with pytest.raises(ValueError):
        wb.beam_select(x, t, 2, done=done, end=10)
    with pytest.raises(ValueError):
        wb.beam_select(x.cpu(), t.cpu(), 2)
    with pytest.raises(ValueError):
        wb.beam_select(x[..., :0], t, 2)
    out, parents, tokens = wb.beam_select(x[:0], t[:0], 2)
    assert out.shape == parents.shape == tokens.shape == (0, 2)


# --------------------------------------------------------------- reordering

REORDER = [
    # R, W, N, entry, dtype
    (1, 1, 5, (8,), torch.bfloat16),
    (1, 2, 1, (8,), torch.bfloat16),
    (3, 4, 100, (256,), torch.bfloat16),
    (2, 8, 333, (24,), torch.bfloat16),
    (5, 3, 77, (3,), torch.float32),       # 12-byte entries
    (2, 16, 50, (2, 40), torch.bfloat16),
    (2, 32, 41, (16,), torch.float32),
    (1, 64, 30, (16,), torch.float32),     # above 32 beams: 4-byte units
    (1, 33, 30, (1,), torch.int32),
    (40, 5, 64, (), torch.float32),        # accumulated weights
]


@pytest.mark.parametrize("R, W, N, entry, dtype", REORDER)
def test_cache_reorder(wb, R, W, N, entry, dtype):
    g = torch.Generator().manual_seed(W + N)
    tables = [torch.randint(-2 ** 15, 2 ** 15, (R * W, N) + entry, generator=g).to(dtype) for _ in range(2)]
    patterns = [torch.randint(-1, W, (R, W), generator=g), torch.arange(W).expand(R, W),
                torch.arange(W).flip(0).expand(R, W), torch.full((R, W), W - 1),
                (torch.arange(W) + 1).expand(R, W) % W]  # any, none, swaps, one for all, a cycle
    for parents in patterns:
        for ragged in (False, True):
            lengths = torch.randint(0, N + 1, (R * W,), generator=g) if ragged else torch.full((R * W,), N)
            first = torch.randint(0, N + 1, (R,), generator=g) if ragged else None
            on_gpu = [t.cuda() for t in tables]
            got = wb.cache_reorder(on_gpu, parents.cuda(), lengths.cuda(), None if first is None else first.cuda())
            assert got is on_gpu
            for t, out in zip(tables, got):
                ref = ob.reorder(t.float().numpy(), parents.numpy(), lengths.numpy(),
                                 None if first is None else first.numpy())
                assert np.array_equal(out.float().cpu().numpy(), ref)
    assert wb.device_status() == 0


def test_cache_reorder_many_tables_at_strides(wb):
    R, W = 2, 3
    g = torch.Generator().manual_seed(1)
    parents = torch.tensor([[1, 1, 0], [2, -1, 2]])
    tables = [torch.randint(0, 1000, (R * W, 5 + i, 8 + 4 * (i % 3)), generator=g).int() for i in range(40)]
    on_gpu = []
    for i, t in enumerate(tables):
        if i % 4 == 0:  # (N, R * W) order
            on_gpu.append(t.transpose(0, 1).contiguous().cuda().transpose(0, 1))
        elif i % 4 == 1:  # part of wider entries
            wide = torch.full(t.shape[:2] + (t.shape[2] + 9,), -7, dtype=torch.int32, device="cuda")
            wide[..., 1:1 + t.shape[2]] = t.cuda()
            on_gpu.append(wide[..., 1:1 + t.shape[2]])
        else:
            on_gpu.append(t.cuda())
    lengths = torch.full((R * W,), 1000)  # clamped to each table
    wb.cache_reorder(on_gpu, parents.cuda(), lengths.cuda())
    for t, out in zip(tables, on_gpu):
        clamp = np.full(R * W, t.shape[1])
        assert np.array_equal(out.cpu().numpy(), ob.reorder(t.numpy(), parents.numpy(), clamp))
    whole = on_gpu[1]._base
    assert (whole[..., 0] == -7).all() and (whole[..., 1 + tables[1].shape[2]:] == -7).all()


def test_a_parent_past_the_beams_is_skipped_and_reported(wb):
    t = torch.arange(3 * 4 * 4).float().view(3, 4, 4).cuda()
    was = t.clone()
    wb.cache_reorder(t, torch.tensor([[7, 0, -1]]).cuda(), torch.full((3,), 4).cuda())
    assert wb.device_status(reset=True) & 2
    assert torch.equal(t[0], was[0]) and torch.equal(t[1], was[0]) and torch.equal(t[2], was[2])


def test_cache_reorder_refusals(wb):
    t = torch.zeros(6, 10, 8, device="cuda")
    parents, lengths = torch.zeros(2, 3, dtype=torch.int64, device="cuda"), torch.full((6,), 10, device="cuda")
    with pytest.raises(ValueError):
        wb.cache_reorder(t[:5], parents, lengths)
    with pytest.raises(ValueError):
        wb.cache_reorder(t, parents, lengths[:5])
    with pytest.raises(ValueError):
        wb.cache_reorder(t, parents, lengths, first=lengths)
    with pytest.raises(ValueError):
        wb.cache_reorder(t[:1].expand(6, 10, 8), parents, lengths)  # one place for all beams
    with pytest.raises(ValueError):
        wb.cache_reorder(torch.zeros(6, 8, 10, device="cuda").transpose(1, 2), parents, lengths)
    with pytest.raises(ValueError):
        wb.cache_reorder(t.cpu(), parents, lengths)
    with pytest.raises(NotImplementedError):
        wb.cache_reorder(torch.zeros(6, 10, 1, dtype=torch.int16, device="cuda"), parents, lengths)
    with pytest.raises(NotImplementedError):
        wb.cache_reorder(torch.zeros(65, 10, 8, device="cuda"), torch.zeros(1, 65, dtype=torch.int64, device="cuda"),
                         torch.full((65,), 10, device="cuda"))
    assert wb.cache_reorder([], parents, lengths) == []


@pytest.mark.parametrize("value", [torch.finfo(torch.float32).min, torch.finfo(torch.float32).max, -2e30, 3e30])
def test_scores_of_one_far_value(wb, value):
    """A beam whose scores are all the type's lowest (or highest) value is uniform; one other score above it is all."""
    V = 9001
    scores = torch.full((2, 2, V), value)
    scores[0, 1, 40:] = -float("inf")
    scores[1, 0, 8500] = 0.0 if value < 0 else value
    scores[1, 1, 3] = -5.0
    totals = torch.tensor([[0.0, -9.0], [0.0, -1.0]])
    x = scores.cuda()
    _check(wb, wb.beam_select(x, totals.cuda(), 5), x, totals, 5)
