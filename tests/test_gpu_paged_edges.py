"""The paged cache's operators at the edges that test_gpu_paged.py leaves out,
against oracle/paged.py in float64. Its tolerances and checks are used where a
test says nothing else."""

import pytest
import torch

from test_gpu_paged import _cache, _check_attention, _filled, _queries, wb  # noqa: F401

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
