"""What belongs to a beam follows it: the accumulated weights and the totals
that examples/beam_search.py holds, against a replay of each beam's own
lineage, and ended beams' totals."""

import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


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


def test_weights_follow_their_beam(example, monkeypatch):
    """At every step the weights that a layer adds to are those that the beam and
    its parents have collected, over the prompt's rows too, which all beams share."""
    import wpt_b200
    R, W, P, steps = 2, 4, 40, 14
    model = example.Decoder(vocab=300, model=256)
    layers = len(model.layers)
    collected, calls, moved = [], [0], [0]
    weigh, select = wpt_b200.attention_weights, wpt_b200.beam_select

    def watched_weights(q, k, positions, lse, scale, weights=None, **more):
        if weights is None:  # the prompt: what all beams of a text start from
            first = weigh(q, k, positions, lse, scale, **more)
            collected.append(first.double().repeat_interleave(W, 0))
            return first
        layer = calls[0] % layers
        calls[0] += 1
        rows = weights.shape[1]
        mine = collected[layer]
        mine = torch.cat([mine, mine.new_zeros(R * W, rows - mine.shape[1])], 1)
        # each addition rounds once, to 2^-24 of at most the pass's 16 heads' sum
        assert (weights.double() - mine).abs().max() <= 1e-6 * mine.max() * steps, layer
        collected[layer] = mine + weigh(q, k, positions, lse, scale, torch.zeros_like(weights).contiguous(),
                                        **more).double()
        return weigh(q, k, positions, lse, scale, weights, **more)

    def watched_select(scores, totals, beams, **more):
        chosen = select(scores, totals, beams, **more)
        if scores.shape[1] == W:
            parents = chosen[1]
            moved[0] += int((parents != torch.arange(W, device="cuda")).sum())
            at = (torch.arange(R, device="cuda")[:, None] * W + parents).reshape(-1)
            for i in range(layers):
                collected[i] = collected[i][at]
        return chosen

    monkeypatch.setattr(wpt_b200, "attention_weights", watched_weights)
    monkeypatch.setattr(wpt_b200, "beam_select", watched_select)
    tokens, _ = example.search(model, _prompts(model, R, P), W, steps, budget=200)  # never cut
    assert tokens.shape == (R, W, steps) and calls[0] == layers * (steps - 1)
    assert moved[0] > W  # beams took others' places
    assert wpt_b200.device_status() == 0


def test_an_ended_beams_total_stays(example, monkeypatch):
    """Once a continuation has ended, every later step carries its total on to the bit."""
    import wpt_b200
    model = example.Decoder(vocab=50, model=256)
    prompts = _prompts(model, 3, 20)
    free, _ = example.search(model, prompts, 4, 3)
    end = int(free[0, 0, 0])
    seen, kept = [], [0]
    select = wpt_b200.beam_select

    def watched(scores, totals, beams, done=None, end=None):
        out, parents, tokens = select(scores, totals, beams, done=done, end=end)
        if done is not None:
            before = torch.gather(totals, 1, parents)
            ended = torch.gather(done, 1, parents)
            assert (tokens[ended] == end).all()
            assert torch.equal(out[ended], before[ended])
            assert (out[~ended] < before[~ended]).all()  # a live token's probability is under 1
            kept[0] += int(ended.sum())
        seen.append(out)
        return out, parents, tokens

    monkeypatch.setattr(wpt_b200, "beam_select", watched)
    tokens, totals = example.search(model, prompts, 4, 12, end=end)
    assert kept[0] > 0 and torch.equal(totals, seen[-1])
    ended = (tokens[..., -1] == end)
    assert ended.any()


def test_a_wider_search_holds_a_narrow_ones_choices(example):
    """As many beams as there are continuations of two tokens find the best one; a narrow search finds no better."""
    model = example.Decoder(vocab=7, model=256)
    prompts = _prompts(model, 3, 30)
    every, totals = example.search(model, prompts, 49, 2)
    # 49 different continuations of 7 x 7; the first step offers 7, the rest are empty
    assert (totals > -float("inf")).all() and (every >= 0).all()
    for r in range(3):
        assert len({tuple(t) for t in every[r].tolist()}) == 49
    # the probabilities of all continuations sum to one
    assert (totals.double().exp().sum(1) - 1).abs().max() < 1e-3
    for beams in (1, 2, 7):
        best = example.search(model, prompts, beams, 2)[1][:, 0]
        assert (best <= totals[:, 0] + 0.2).all()  # the same numbers but for the bf16 roundings of another batch
    assert torch.equal(example.search(model, prompts, 7, 2)[0][:, 0], every[:, 0])
