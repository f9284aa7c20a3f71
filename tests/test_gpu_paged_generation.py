"""examples/paged_generation.py: ragged prompts in chunks, then tokens one by one,
over paged caches. Every call of the three operators that it makes is checked
against oracle/paged.py on what it was given, and the caches' contents are
carried along in float64 from call to call."""

import importlib.util
import os

import pytest
import torch

from test_gpu_paged import _cache, _check_append, _check_attention
from test_gpu_rotate import _check as _check_rotate

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example():
    from wpt_b200 import build
    build.build()
    spec = importlib.util.spec_from_file_location("paged_generation", os.path.join(ROOT, "examples", "paged_generation.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def _prompts(model, lengths, seed=3):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(0, model.embedding.shape[0], (len(lengths), max(lengths)), generator=g).cuda()


def test_every_call_of_a_run(example, monkeypatch):
    import wpt_b200
    rotate, append, attend = wpt_b200.rotate, wpt_b200.paged_append, wpt_b200.paged_attention
    seen = []

    def checked_rotate(x, positions, f):
        y = rotate(x, positions, f)
        _check_rotate(y, x, positions, f, None, False)
        seen.append("rotate")
        return y

    def checked_append(pages, scales, table, new, first, counts, f):
        before = _cache(pages, scales)
        got = append(pages, scales, table, new, first, counts, f)
        _check_append(got, before, table, new, first, counts, f)
        seen.append("append")
        return got

    def checked_attend(q, pages, scales, table, positions, scale):
        got = attend(q, pages, scales, table, positions, scale)
        _check_attention(got, q, _cache(pages, scales), table, positions, scale)
        seen.append("attend")
        return got

    monkeypatch.setattr(wpt_b200, "rotate", checked_rotate)
    monkeypatch.setattr(wpt_b200, "paged_append", checked_append)
    monkeypatch.setattr(wpt_b200, "paged_attention", checked_attend)
    model = example.Decoder(vocab=500, model=256, heads=4)
    lengths = [70, 1, 33]
    tokens, cache = example.generate(model, _prompts(model, lengths), lengths, 4, page=16, chunk=32)
    assert tokens.shape == (3, 4) and (tokens >= 0).all() and (tokens < 500).all()
    assert seen == ["rotate", "append", "attend"] * 2 * (3 + 3)  # 2 layers; 3 chunks, 3 steps
    held = sum(cache.held, [])
    assert len(set(held)) == len(held) and [len(h) for h in cache.held] == [5, 1, 3]
    cache.release(0)
    assert len(cache.free) == 5 and (cache.table[0] == -1).all()
    assert wpt_b200.device_status() == 0


@pytest.mark.parametrize("page", [16, 128])
def test_a_run_repeats_itself(example, page):
    model = example.Decoder(vocab=300, model=256, heads=8)
    lengths = [150, 40, 97]
    prompts = _prompts(model, lengths, 4)
    one, _ = example.generate(model, prompts, lengths, 8, page=page, chunk=64)
    again, _ = example.generate(model, prompts, lengths, 8, page=page, chunk=64)
    assert torch.equal(one, again)


def test_training_step():
    """Queries and keys turned, then window attention over them: the gradients that come back through the turn are the
    attention's own, turned back."""
    import wpt_b200
    g = torch.Generator().manual_seed(5)
    B, T, H, W = 2, 20, 4, 16
    f = wpt_b200.rotary_frequencies(64, device="cuda")
    positions = torch.arange(T).cuda()
    rows = torch.arange(1 - W, T).cuda()  # the positions of the table's rows
    q = torch.randn(B, T, H, 128, generator=g).bfloat16().cuda().requires_grad_()
    k, v = (torch.randn(B, W - 1 + T, 128, generator=g).bfloat16().cuda().requires_grad_() for _ in range(2))
    qt, kt = wpt_b200.rotate(q, positions, f), wpt_b200.rotate(k, rows, f)
    qt.retain_grad()
    kt.retain_grad()
    out = wpt_b200.window_attention(qt, kt, v, torch.zeros(H, device="cuda"), positions, 128 ** -0.5, window=W)
    out.backward(torch.randn(out.shape, generator=g).to(out.dtype).cuda())
    _check_rotate(q.grad, qt.grad, positions[None], f, None, False, inverse=True)
    _check_rotate(k.grad, kt.grad, rows[None], f, None, False, inverse=True)
    assert q.grad.abs().sum() > 0 and k.grad.abs().sum() > 0 and v.grad.abs().sum() > 0
