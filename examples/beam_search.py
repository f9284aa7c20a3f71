"""Beam search over a generation cache with a budget, on wpt_b200's kernels.

    python examples/beam_search.py [--texts 4] [--beams 4] [--prompt 600] [--steps 64] [--budget 256]

A small random decoder (one shared key/value head a layer, no position
encoding, as WPT's exact layers) reads a batch of prompts and searches their
continuations. With --budget, each layer's cache keeps that many rows of the
prompt, chosen by the attention weight that its last places gave them, and is
cut to the budget again whenever it has grown by half of it. Every step runs

    forward_with_lse    attention over the cache (and its log-sum-exp)
    attention_weights   what each cached row collected (with a budget)
    head_scores         the vocabulary's scores
    beam_select         the next beams over beams and vocabulary
    cache_reorder       each beam's cached rows become its parent's
    cache_append        and its new token's entry is written
    cache_evict         the cache is cut to its budget (when it is over)

and reads nothing back to the host.
"""

import argparse
import os
import sys
import time

import torch

if __name__ == "__main__":
    sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import wpt_b200
from wpt_b200 import ops

WIDTH = 128  # of a head


class Decoder:
    """Random weights from a seed: `layers` of attention over a shared
    key/value head, then the output head."""

    def __init__(self, vocab=4096, model=512, heads=16, layers=2, seed=0, device="cuda"):
        g = torch.Generator(device=device).manual_seed(seed)

        def matrix(rows, columns):
            return (torch.randn(rows, columns, generator=g, device=device) * rows ** -0.5).bfloat16()

        self.heads = heads
        self.embedding = torch.randn(vocab, model, generator=g, device=device).bfloat16()
        self.layers = [dict(q=2 * matrix(model, heads * WIDTH), kv=matrix(model, 2 * WIDTH),
                            out=matrix(heads * WIDTH, model)) for _ in range(layers)]
        self.head = (3 * matrix(model, vocab)).t().contiguous()

    @staticmethod
    def _norm(x):
        return torch.nn.functional.rms_norm(x, x.shape[-1:])

    def attend(self, layer, x, table, positions):
        """The layer's output for x (B, T, model) at `positions` (B, T) over the
        entries table (B, N, 2 * WIDTH), with the queries and the log-sum-exp."""
        B, T, _ = x.shape
        q = (self._norm(x) @ layer["q"]).view(B, T, self.heads, WIDTH)
        o, lse = wpt_b200.forward_with_lse(q, table[..., :WIDTH], table[..., WIDTH:], positions, WIDTH ** -0.5)
        return x + o.reshape(B, T, -1) @ layer["out"], q, lse

    def entries(self, layer, x):
        return self._norm(x) @ layer["kv"]

    def scores(self, x):
        """(rows, vocab) scores of hidden states (rows, model)."""
        return ops.head_scores(self._norm(x), self.head, round_bf16=False)


class Layer:
    """One layer's cache: entries (rows, capacity, 2 * WIDTH), and the weight that each has collected."""

    def __init__(self, table, weights):
        self.table, self.weights = table, weights


def _evict(layer, length, budget, room):
    """Cuts a layer's cache of `length` rows a text to `budget`, with room for more."""
    lengths = torch.full((layer.table.shape[0],), length, dtype=torch.int64, device=layer.table.device)
    layer.table, layer.weights, _, _ = wpt_b200.cache_evict(layer.table, layer.weights, lengths, budget,
                                                            recent=budget // 4, first=min(4, budget // 4),
                                                            capacity=budget + room)


def search(model, prompts, beams, steps, budget=None, end=None, observe=32):
    """The `beams` best continuations of prompts (R, P) that beam search finds
    in `steps` tokens: (tokens (R, beams, steps), totals (R, beams)). budget:
    cached rows a text and layer (None: all). end: the token that ends a
    continuation (it is repeated from there on)."""
    R, P = prompts.shape
    device = prompts.device
    limit = P + steps if budget is None else budget + max(1, budget // 2)  # rows before a cut
    scale = WIDTH ** -0.5

    # the prompt: every layer's entries and, for its budget, what the last places look at
    x = model.embedding[prompts]
    positions = torch.arange(P, device=device).expand(R, P).contiguous()
    layers = []
    for layer in model.layers:
        table = model.entries(layer, x)
        x, q, lse = model.attend(layer, x, table, positions)
        cache = Layer(table, None)
        if budget is not None:
            cache.weights = wpt_b200.attention_weights(q[:, -observe:], table[..., :WIDTH], positions[:, -observe:],
                                                       lse[:, -observe:], scale)
        layers.append(cache)
    rows = P
    if budget is not None and P > budget:
        for cache in layers:
            _evict(cache, P, budget, limit - budget)
        rows = budget
    shared = rows  # the first rows are the same in all beams of a text
    for cache in layers:  # a copy for each beam, with room
        grown = cache.table.new_zeros(R * beams, limit, 2 * WIDTH)
        grown[:, :rows] = cache.table[:, :rows].repeat_interleave(beams, 0)
        weights = torch.zeros(R * beams, limit, device=device)
        if budget is not None:
            weights[:, :rows] = cache.weights[:, :rows].repeat_interleave(beams, 0)
        cache.table, cache.weights = grown, weights

    totals, parents, tokens = wpt_b200.beam_select(model.scores(x[:, -1])[:, None], torch.zeros(R, 1, device=device),
                                                   beams)
    history = tokens[..., None]
    one = torch.ones(R * beams, dtype=torch.int64, device=device)
    for _ in range(steps - 1):
        if rows == limit:  # over the budget by half of it
            for cache in layers:
                _evict(cache, rows, budget, limit - budget)
            rows, shared = budget, 0
        x = model.embedding[tokens.reshape(-1, 1).clamp_min(0)]
        at = one * rows
        for layer, cache in zip(model.layers, layers):
            cache.table, table = wpt_b200.cache_append(cache.table, model.entries(layer, x), at, one, need=rows + 1)
            x, q, lse = model.attend(layer, x, table, at[:, None])
            if budget is not None:
                wpt_b200.attention_weights(q, table[..., :WIDTH], at[:, None], lse, scale, cache.weights[:, :rows + 1])
        rows += 1
        done = None if end is None else tokens == end
        totals, parents, tokens = wpt_b200.beam_select(model.scores(x[:, 0]).view(R, beams, -1), totals, beams,
                                                       done=done, end=end)
        wpt_b200.cache_reorder([c.table for c in layers], parents, one * rows, first=one[:R] * shared)
        if budget is not None:  # the shared rows too: their entries are the same in all beams, their weights are not
            wpt_b200.cache_reorder([c.weights for c in layers], parents, one * rows)
        history = torch.cat([torch.gather(history, 1, parents.clamp_min(0)[..., None].expand_as(history)),
                             tokens[..., None]], 2)
    return history, totals


def main():
    parser = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    parser.add_argument("--texts", type=int, default=4)
    parser.add_argument("--beams", type=int, default=4)
    parser.add_argument("--prompt", type=int, default=600)
    parser.add_argument("--steps", type=int, default=64)
    parser.add_argument("--budget", type=int, default=None)
    args = parser.parse_args()
    model = Decoder()
    g = torch.Generator(device="cuda").manual_seed(1)
    prompts = torch.randint(0, model.embedding.shape[0], (args.texts, args.prompt), generator=g, device="cuda")
    search(model, prompts, args.beams, min(args.steps, 4), args.budget)  # the library loads, its kernels too
    torch.cuda.synchronize()
    start = time.perf_counter()
    tokens, totals = search(model, prompts, args.beams, args.steps, args.budget)
    torch.cuda.synchronize()
    seconds = time.perf_counter() - start
    for r in range(args.texts):
        print(f"text {r}: best total {totals[r, 0].item():.3f}, tokens {tokens[r, 0, :12].tolist()} ...")
    kept = "all rows" if args.budget is None else f"a budget of {args.budget} rows"
    print(f"{args.steps} steps of {args.texts} x {args.beams} beams with {kept}: {seconds * 1e3:.1f} ms, "
          f"{args.texts * args.steps / seconds:.0f} tokens/s of the texts")
    if wpt_b200.device_status():
        raise RuntimeError("a kernel reported a status")


if __name__ == "__main__":
    main()
