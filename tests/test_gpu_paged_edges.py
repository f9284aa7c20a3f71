"""The paged cache's operators at the edges that test_gpu_paged.py leaves out,
against oracle/paged.py in float64. Its tolerances and checks are used where a
test says nothing else."""

import math

import numpy as np
import pytest
import torch

from oracle import paged as op
from test_gpu_paged import (SCORE, _cache, _check_append, _check_attention, _filled, _np, _queries,  # noqa: F401
                             wb)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tiles", [1, 2, 3, 5])
def test_results_wait_for_a_segments_last_product(wb, tiles, monkeypatch):  # noqa: F811
    """Runs of so many tiles a CTA, over and over: the same bits, and right."""
    g = torch.Generator().manual_seed(30)
    B, H, S, M = 2, 32, 128, 60
    monkeypatch.setattr(wb.ops, "_paged_plan", lambda *a: (0, -(-B * (M + 4) // tiles)))
    pages, scales, table = _filled(B, M, S, 128, g)
    q, positions = _queries(B, 1, H, g), torch.tensor([[M * S - 1], [M * S - 300]])
    dev = [t.cuda() for t in (q, pages, scales, table, positions)]
    got = wb.paged_attention(*dev, 128 ** -0.5)
    _check_attention(got, q, _cache(pages, scales), table, positions, 128 ** -0.5)
    for _ in range(30):
        again = wb.paged_attention(*dev, 128 ** -0.5)
        assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])
    assert wb.device_status() == 0


def _dominated(N, at, share, deviation, g, H=8, S=64):
    """A row of N entries of which those at `at` take `share` of each head's weight while their values are 0, as a
    text's first tokens may: (q (1, 1, H, 128), pages, scales, out and log-sum in 64 bits, sum w|v|). Half of the
    channels' values are positive, so that a weight that is lost shows in full. All on the GPU."""
    k, v = (torch.randn(N, 128, generator=g).cuda() for _ in range(2))
    v[:, ::2] = v[:, ::2].abs()
    k[:, 0] = 0
    k[at] = 0
    k[at, 0], v[at] = 8.0, 0.0
    held, scales = [], []
    for x in (k, v):
        top = x.view(-1, 16 * 128).abs().amax(1)
        s = torch.exp2(torch.ceil(torch.log2(top.double() / 448))).float()
        held.append((x.view(-1, 16, 128) / s[:, None, None]).to(torch.float8_e4m3fn).view(N, 128))
        scales.append(s)
    keys, values = (h.double() * s.double().repeat_interleave(16)[:, None] for h, s in zip(held, scales))
    q = (torch.randn(1, 1, H, 128, generator=g) * deviation).cuda()
    q[..., 0] = 0
    q = q.bfloat16()
    rest = torch.logsumexp(q[0, 0].double() @ keys.t() * 128 ** -0.5, 1)
    q[0, 0, :, 0] = ((rest + math.log(share / (1 - share) / len(at))) * 128 ** 0.5 / 8).bfloat16()
    z = q[0, 0].double() @ keys.t() * 128 ** -0.5
    lse = torch.logsumexp(z, 1)
    w = torch.exp(z - lse[:, None])
    assert (w[:, at].sum(1) > share - 0.1 * (1 - share) ** 0.5).all()
    pages = torch.cat([h.view(torch.uint8) for h in held], 1).view(N // S, S, 256).view(torch.float8_e4m3fn)
    return q, pages, torch.stack(scales, 1).view(N // S, S // 16, 2), w @ values, lse, w @ values.abs()


def _check_dominated(got, ref, lse, around):
    """As near as weights and results in bf16 are: nothing here grows with the row."""
    out = got[0].double()
    assert ((out - ref).abs() <= 2.0 ** -8 * ref.abs() + (2.0 ** -8.6 + 2 * SCORE) * around).all()
    # a scale of the whole result is seen much finer: by the weights' mean error, here under 2^-10
    some = around[:, ::2] > 0
    kept = (out[:, ::2][some].sum() / ref[:, ::2][some].sum()).item()
    assert abs(kept - 1) <= 2.0 ** -10 + 2 * SCORE, kept
    assert ((got[1].double() - lse).abs() <= SCORE + 2.0 ** -22 * lse.abs()).all()


@pytest.mark.parametrize("at", [[0], [5], [0, 1, 2, 3], [77], [127, 128], [20000]])
@pytest.mark.parametrize("N,deviation,share", [(2048, 1.0, 0.98), (32768, 1.0, 0.98), (32768, 2.0, 0.98), (32768, 2.0, 0.999),
                                               (131072, 1.0, 0.98), (262144, 2.0, 0.98)])
def test_keys_that_take_nearly_all_of_the_weight(wb, N, deviation, share, at):  # noqa: F811
    """Their rows' other weights keep their precision, in runs of whole rows (more than 256 groups), of clusters and in
    balanced ones."""
    if at[0] >= N:
        pytest.skip("past the row")
    g = torch.Generator().manual_seed(31)
    q, pages, scales, ref, lse, around = _dominated(N, at, share, deviation, g)
    table = torch.randperm(N // 64, generator=g).cuda()
    pages, scales = pages[torch.argsort(table)], scales[torch.argsort(table)]
    for rows in (1, 6, 260):
        got = wb.paged_attention(q.expand(rows, -1, -1, -1), pages, scales, table.int().expand(rows, -1),
                                 torch.tensor([N - 1]).cuda(), 128 ** -0.5)
        assert (got[0] == got[0][:1]).all() and (got[1] == got[1][:1]).all() or rows == 6  # (balanced runs differ)
        for b in (0, rows - 1):
            _check_dominated((got[0][b, 0], got[1][b, 0]), ref, lse, around)
    assert wb.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.bfloat16, torch.bool])
def test_positions_that_are_not_whole_are_refused(wb, dtype):  # noqa: F811
    """Cut off, a fractional position would be another one."""
    pages, scales = wb.paged_cache(4, 32, 128)
    table, at = torch.zeros(2, 3, dtype=torch.int32, device="cuda"), torch.zeros(2, 1, dtype=torch.int64, device="cuda")
    q, new = torch.zeros(2, 1, 4, 128, device="cuda").bfloat16(), torch.ones(2, 1, 256, device="cuda")
    f, one = wb.rotary_frequencies(64, device="cuda"), torch.ones(2, dtype=torch.int64, device="cuda")
    for positions in (at, at[0], at[:, :0].expand(2, 0)):
        x = q[:, :positions.shape[-1]]
        assert wb.rotate(x, positions, f).shape == x.shape
        with pytest.raises(ValueError, match="whole"):
            wb.rotate(x, positions.to(dtype), f)
    with pytest.raises(ValueError, match="whole"):
        wb.paged_attention(q, pages, scales, table, at.to(dtype), 1.0)
    with pytest.raises(ValueError, match="whole"):
        wb.paged_attention(q, pages, scales, table, at[0].to(dtype), 1.0)
    for bad in (dict(first=at[:, 0].to(dtype)), dict(counts=one.to(dtype)), dict(positions=at.to(dtype), frequencies=f)):
        with pytest.raises(ValueError, match="whole"):
            wb.paged_append(**(dict(pages=pages, scales=scales, table=table, new=new, first=at[:, 0], counts=one) | bad))
    assert not pages.view(torch.uint8).any()
    for small in (torch.int32, torch.uint8):  # whole numbers of other types are taken
        assert torch.equal(wb.rotate(q, at.to(small), f), wb.rotate(q, at, f))
        wb.paged_append(pages.clone(), scales.clone(), table, new, at[:, 0].to(small), one.to(small), f, at.to(small))
    assert wb.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotation_in_forward_mode(wb, interleaved, dtype):  # noqa: F811
    """A dual tensor's tangent is turned as its value is, leaf or not, and the tangent's gradient back."""
    from torch.autograd import forward_ad

    g = torch.Generator().manual_seed(32)
    x, v, d = (torch.randn(2, 7, 3, 96, generator=g).to(dtype).cuda() for _ in range(3))
    positions, f = torch.randint(0, 5000, (2, 7), generator=g).cuda(), wb.rotary_frequencies(48, device="cuda")
    how = (positions, f, 16, interleaved, 0.75)
    value, turned = wb.rotate(x, *how), wb.rotate(v, *how)
    for leaf in (False, True):
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(x.clone().requires_grad_(leaf), v)
            y = forward_ad.unpack_dual(wb.rotate(dual, *how))
            assert torch.equal(y.primal, value) and torch.equal(y.tangent, turned)
            plain = wb.rotate(x, *how)  # no tangent: none comes out
            assert forward_ad.unpack_dual(plain).tangent is None and torch.equal(plain, value)
            if leaf:
                tangent = v.clone().requires_grad_()
                y = forward_ad.unpack_dual(wb.rotate(forward_ad.make_dual(x, tangent), *how))
                back, = torch.autograd.grad(y.tangent, tangent, d)
                assert torch.equal(back, wb.ops.rotate(d, *how, inverse=True))
    y = wb.rotate(x.requires_grad_(), *how)
    assert torch.equal(torch.autograd.grad(y, x, d)[0], wb.ops.rotate(d, *how, inverse=True))


@pytest.mark.parametrize("size", [2.0 ** 28, 2.0 ** 33, 2.0 ** 60, 2.0 ** 104, 2.0 ** 117, 2.0 ** 122])
@pytest.mark.parametrize("which", ["some", "all"])
def test_queries_of_any_size(wb, which, size):  # noqa: F811
    """Heads and drafts of very large queries, all of them or next to ordinary and to tiny ones: their scores are
    finite, so all weight is the largest one's, and the others are as if alone."""
    g = torch.Generator().manual_seed(33)
    B, T, H, S, M = 2, 2, 8, 32, 12
    pages, scales, table = _filled(B, M, S, 128, g)
    q = _queries(B, T, H, g)
    large = torch.full((B, T, H), which == "all")
    large[0, 0, 3] = large[1, :, 5] = True
    if which == "some":
        q[0, 1, 0] = (q[0, 1, 0].float() * 2.0 ** -100).bfloat16()
    q[large] = (q[large].float() * size).bfloat16()
    positions = torch.full((B, 1), M * S - T) + torch.arange(T)
    cache = _cache(pages, scales)
    for window in (0, 200):
        args = [t.cuda() for t in (pages, scales, table, positions)]
        got = wb.paged_attention(q.cuda(), *args, 128 ** -0.5, window=window)
        out, lse = got[0].float().cpu(), got[1].cpu()
        ref, top = (torch.from_numpy(t) for t in op.attention(_np(q), cache, table.numpy(), positions.numpy(),
                                                               128 ** -0.5, window))
        assert out.isfinite().all() and lse.isfinite().all()
        # one key's value, its weight held to 2^-8.6, and the result's rounding; its score to 128 truncations of 2^-23 of
        # a sum that is 32 times it at most
        assert ((out - ref)[large].abs() <= (2.0 ** -8.6 + 2.0 ** -8) * ref[large].abs()).all()
        assert ((lse - top)[large].abs() <= 128 * 2.0 ** -23 * 32 * top[large].abs()).all()
        plain = torch.where(large[..., None], 0, q).bfloat16()  # the others, with zeros in the large ones' place
        zero = wb.paged_attention(plain.cuda(), *args, 128 ** -0.5, window=window)
        out, lse = torch.where(large[..., None], zero[0].cpu().float(), out), torch.where(large, zero[1].cpu(), lse)
        _check_attention((out, lse), plain, cache, table, positions, 128 ** -0.5, window)
    assert wb.device_status() == 0


def test_what_an_append_reports(wb):  # noqa: F811
    """The status word's shape bit for each way to miss the table, and none for calls that miss nothing; without any
    page at all a call writes and reports nothing."""
    g = torch.Generator().manual_seed(35)
    pages, scales, _ = _filled(4, 2, 32, 32, g)
    pages, scales = pages.cuda(), scales.cuda()
    table = torch.tensor([[0, 1]], device="cuda")
    new = torch.randn(1, 3, 64, generator=g).cuda()
    for first, count, want in ((2 ** 62, 3, 2), (-2 ** 62, 3, 2), (64, 1, 2), (63, 2, 2), (61, 3, 0), (-3, 3, 2), (-3, 2 ** 62, 2),
                               (-1, 2, 2), (0, 0, 0), (70, 0, 0), (0, -5, 0), (-9, -5, 0), (61, 2 ** 62, 0), (62, 2 ** 62, 2)):
        wb.paged_append(pages.clone(), scales.clone(), table, new, torch.tensor([first]).cuda(), torch.tensor([count]).cuda())
        assert wb.device_status() == want, (first, count)
    one, at = torch.ones(1, dtype=torch.int64, device="cuda"), torch.zeros(1, dtype=torch.int64, device="cuda")
    for missing in (-1, 10, 2 ** 40):
        wb.paged_append(pages.clone(), scales.clone(), torch.tensor([[missing, 1]]).cuda(), new, at, one)
        assert wb.device_status() == 2
    wb.paged_append(pages[:0], scales[:0], table, new, at, one)
    wb.paged_append(pages, scales, table[:, :0], new, at, one)
    assert wb.device_status() == 0


def test_entries_after_an_append_keep_their_bytes(wb):  # noqa: F811
    """An append inside a text: what follows in its last block keeps its bytes, other blocks their scales too."""
    g = torch.Generator().manual_seed(36)
    pages, scales, table = _filled(1, 3, 32, 64, g)
    new, first, counts = 50 * torch.randn(1, 20, 128, generator=g), torch.tensor([21]), torch.tensor([20])
    cache = _cache(pages, scales)
    got = wb.paged_append(*(t.cuda() for t in (pages, scales, table, new, first, counts)))
    _check_append(got, cache, table, new, first, counts)
    before, after = (t.view(torch.uint8)[table[0].long()].view(96, 128) for t in (pages, got[0].cpu()))
    assert torch.equal(before[:16], after[:16]) and torch.equal(before[41:], after[41:])
    changed = (scales[table[0].long()] != got[1].cpu()[table[0].long()]).view(6, 2).all(1)
    assert changed.tolist() == [False, True, True, False, False, False]


def test_unread_entries_without_a_window(wb):  # noqa: F811
    """NaN in keys, values and scales of whatever no query reads, as recycled pages may hold: past the positions, in
    rows that read nothing, behind a missing page, and on pages of no row."""
    g = torch.Generator().manual_seed(34)
    B, H, S, M = 5, 16, 32, 12
    for T, at in ((1, [200, 0, -1, 383, 5000]), (3, [[200, 201, 202], [0, 1, 2], [-1, -1, 7], [90, 17, 383], [63, 64, -5]])):
        pages, scales, table = _filled(B, M, S, 128, g)
        positions = torch.tensor(at).view(B, T)
        table[3, 2] = -1
        clean = _cache(pages, scales)
        read = torch.arange(M * S) <= positions.max(1).values[:, None]
        mine = torch.zeros(pages.shape[0], S, dtype=torch.bool)
        for b in range(B):
            for i in range(M):
                if table[b, i] >= 0:
                    mine[table[b, i]] |= read[b, i * S:(i + 1) * S]
        dirty, bad = pages.clone(), scales.clone()
        dirty.view(torch.uint8)[~mine] = 0x7F
        bad[~mine.view(-1, S // 16, 16).any(-1)] = math.nan
        assert bad.isnan().any() and not bad.isnan().all()
        q = _queries(B, T, H, g)
        got = wb.paged_attention(*(t.cuda() for t in (q, dirty, bad, table, positions)), 128 ** -0.5)
        _check_attention(got, q, clean, table, positions, 128 ** -0.5)
    assert wb.device_status() == 0


@pytest.mark.parametrize("H", [1, 16, 32])
def test_each_weight(wb, H):  # noqa: F811
    """Key i's value is 1 in channel i and 0 elsewhere, so the result is the weights themselves, from the largest (some
    keys near it in each eight of the first 32, so that it sets the base) down to 2^-28 of it."""
    g = torch.Generator().manual_seed(37)
    S, M, C = 32, 4, 128
    pages = torch.zeros(M, S, 2 * C)
    pages[:, :, 0] = 14 * torch.rand(M, S, generator=g)  # scores, in units of q's: weights down to e^-14 q
    pages[0, 0, 0], pages[0, 4::8, 0] = 14.0, 13.0
    for i in range(C):
        pages[i // S, i % S, C + i] = 1.0
    pages = pages.to(torch.float8_e4m3fn)
    scales, table = torch.ones(M, S // 16, 2), torch.arange(M).int()[None]
    q = torch.zeros(1, 1, H, C)
    q[..., 0] = 128 ** 0.5 * torch.linspace(0.7, 1.4, H)
    q, positions = q.bfloat16(), torch.tensor([[C - 1]])
    out, _ = wb.paged_attention(*(t.cuda() for t in (q, pages, scales, table, positions)), 128 ** -0.5)
    z = (_np(q)[0, 0, :, :1] * _np(pages)[:, :, 0].reshape(1, C)) * 128 ** -0.5
    w = np.exp(z - z.max(1, keepdims=True))
    total = w.sum(1, keepdims=True)
    # a score is one product of up to 20 and its exponent's roundings: 1e-5; the result's own rounding is half a step of
    # bf16, which keeps 8 bits: torch.finfo(torch.bfloat16).eps / 2 = 2^-8
    tol = np.maximum(2.0 ** -8.6 * w, 2.0 ** -21.8) / total
    off = np.abs(_np(out)[0, 0] - w / total)
    assert (off <= tol + (2.0 ** -8 + 1e-5) * (w / total + tol)).all(), (off / tol).max()
    assert w.min() < 2.0 ** -14
