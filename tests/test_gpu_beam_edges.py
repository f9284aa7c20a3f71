"""Beam search's step on the GPU where it can go wrong: masks of large finite
values, values that tie only after rounding, refusals that change nothing,
replay in a graph and other streams. Values against oracle/beam.py."""

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
