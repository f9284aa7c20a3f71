"""The cache operators together, as examples/beam_search.py runs them: beams
searched over a cache that is appended to, reordered and, with a budget, cut by
accumulated attention weight.

Without a budget the totals have to be the log-probabilities of the returned
tokens, read again in one pass without any cache. The two differ by the bf16
roundings of the hidden states: each (2^-9 of its size, a dozen a layer at
random signs) moves a score of standard deviation 3 by at most about 12^0.5 *
2 layers * 2^-9 * 3 = 0.04, so a step's log-probability by under 0.1."""

import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
STEP = 0.1


@pytest.fixture(scope="module")
def example():
    from wpt_b200 import build
    build.build()
    spec = importlib.util.spec_from_file_location("beam_search", os.path.join(ROOT, "examples", "beam_search.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def _prompts(model, texts, length):
    g = torch.Generator(device="cuda").manual_seed(2)
    return torch.randint(0, model.embedding.shape[0], (texts, length), generator=g, device="cuda")


def _read_again(example, model, prompts, tokens):
    """(R, W) log-probabilities of the continuations, one pass over each whole text."""
    R, W, S = tokens.shape
    P = prompts.shape[1]
    text = torch.cat([prompts[:, None].expand(R, W, P), tokens], 2).reshape(R * W, P + S)
    x = model.embedding[text]
    positions = torch.arange(P + S, device="cuda").expand(R * W, -1).contiguous()
    for layer in model.layers:
        x, _, _ = model.attend(layer, x, model.entries(layer, x), positions)
    scores = model.scores(x[:, P - 1:P + S - 1].reshape(R * W * S, -1)).view(R, W, S, -1).double()
    return torch.gather(torch.log_softmax(scores, -1), 3, tokens[..., None])[..., 0].sum(-1)


@pytest.mark.parametrize("beams, prompt", [(1, 40), (4, 130), (7, 33)])
def test_totals_are_the_tokens_log_probabilities(example, beams, prompt):
    import wpt_b200
    model = example.Decoder(vocab=1000, model=256)
    prompts = _prompts(model, 3, prompt)
    steps = 9
    tokens, totals = example.search(model, prompts, beams, steps)
    assert tokens.shape == (3, beams, steps) and (tokens >= 0).all()
    again = _read_again(example, model, prompts, tokens)
    assert (again - totals.double()).abs().max() < STEP * steps
    assert (totals[:, :-1] >= totals[:, 1:]).all()
    assert len({tuple(t) for t in tokens[0].tolist()}) == beams  # different continuations
    assert wpt_b200.device_status() == 0


def test_more_beams_find_no_worse_a_continuation(example):
    model = example.Decoder(vocab=1000, model=256)
    prompts = _prompts(model, 4, 50)
    one = example.search(model, prompts, 1, 1)[1][:, 0]
    assert torch.equal(example.search(model, prompts, 8, 1)[1][:, 0], one)


@pytest.mark.parametrize("budget", [16, 80])
def test_a_budget_holds_the_cache_and_cuts_it_again(example, budget):
    import wpt_b200
    model = example.Decoder(vocab=1000, model=256)
    prompts = _prompts(model, 2, 90)
    steps = 40  # a budget of 80 cuts the prompt alone, one of 16 the beams too, again and again
    cut = []
    evict = wpt_b200.cache_evict

    def watched(held, weights, lengths, keep, **more):
        result = evict(held, weights, lengths, keep, **more)
        cut.append((held.shape[0], int(lengths[0]), keep))
        assert (result[3] == keep).all()
        # the kept rows are the first, the last and the heaviest of the others
        first, recent = more["first"], more["recent"]
        n = int(lengths[0])
        for b in range(held.shape[0]):
            rows = result[2][b]
            assert rows[:first].tolist() == list(range(first))
            assert rows[keep - recent:].tolist() == list(range(n - recent, n))
            others = weights[b, first:n - recent].clone()
            inside = rows[first:keep - recent] - first
            least = others[inside].min()
            others[inside] = -1
            assert others.max() <= least
            assert torch.equal(result[0][b, :keep], held[b, rows])
        return result

    wpt_b200.cache_evict = watched
    try:
        tokens, totals = example.search(model, prompts, 3, steps, budget=budget)
    finally:
        wpt_b200.cache_evict = evict
    assert tokens.shape == (2, 3, steps) and torch.isfinite(totals).all()
    assert cut and all(c[2] == budget for c in cut)
    if budget == 16:
        assert cut[0] == (2, 90, 16) and cut[-1] == (6, 24, 16)
    assert wpt_b200.device_status() == 0


def test_an_ended_beam_keeps_its_total(example):
    model = example.Decoder(vocab=50, model=256)
    prompts = _prompts(model, 2, 20)
    free, _ = example.search(model, prompts, 4, 3)
    end = int(free[0, 0, 0])  # the first text's best beam ends at once
    tokens, totals = example.search(model, prompts, 4, 12, end=end)
    ended = (tokens == end).cumsum(-1) > 0
    assert ended[0].any()
    assert (tokens[ended] == end).all()  # nothing follows the end
