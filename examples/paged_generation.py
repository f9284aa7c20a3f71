"""Generation for texts of different lengths over a paged cache in 8 bits, on wpt_b200's kernels.

    python examples/paged_generation.py [--texts 8] [--prompt 2000] [--steps 64] [--page 64] [--chunk 512]

A small random decoder (one shared key/value head a layer, the last 64 channels
of queries and keys turned by their positions) reads prompts of ragged lengths in
chunks and continues each. A text holds pages of its own, taken from one pool for
all texts as it grows; a layer's entries lie in its own pool at the same pages.
Every pass, of a chunk or of one token a text, runs in each layer

    rotate              the queries' positions
    paged_append        the new entries, their keys turned, rounded to 8 bits
    paged_attention     over all entries of each text

then head_scores for each text's last place. Pages are handed out on the host,
which knows all lengths; nothing is read back from the GPU.
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

WIDTH = 128   # of a head
TURNED = 64   # channels of it that turn


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

    def forward(self, tokens, cache, first, counts):
        """Scores (B, vocab) after the last of each text's counts new tokens
        (B, n), which become its entries first .. of the cache."""
        B, n = tokens.shape
        x = self.embedding[tokens]
        positions = first[:, None] + torch.arange(n, device=tokens.device)
        for layer, (pages, scales) in zip(self.layers, cache.pools):
            y = torch.nn.functional.rms_norm(x, x.shape[-1:])
            q = wpt_b200.rotate((y @ layer["q"]).view(B, n, self.heads, WIDTH), positions, cache.frequencies)
            wpt_b200.paged_append(pages, scales, cache.table, y @ layer["kv"], first, counts, cache.frequencies)
            o, _ = wpt_b200.paged_attention(q, pages, scales, cache.table, positions, WIDTH ** -0.5)
            x = x + o.reshape(B, n, -1) @ layer["out"]
        last = x[torch.arange(B, device=x.device), (counts - 1).clamp_min(0)]
        return ops.head_scores(torch.nn.functional.rms_norm(last, last.shape[-1:]), self.head, round_bf16=False)


class Cache:
    """A pool of `pages` pages for each layer, and each text's table of them."""

    def __init__(self, layers, texts, capacity, page, pages, device="cuda"):
        self.page, self.free, self.held = page, list(range(pages)), [[] for _ in range(texts)]
        self.pools = [wpt_b200.paged_cache(pages, page, WIDTH, device) for _ in range(layers)]
        self.table = torch.full((texts, -(-capacity // page)), -1, dtype=torch.int32, device=device)
        self.frequencies = wpt_b200.rotary_frequencies(TURNED, device=device)

    def grow(self, lengths):
        """Pages for each text to hold lengths[b] entries."""
        new = [(b, i) for b, n in enumerate(lengths) for i in range(len(self.held[b]), -(-n // self.page))]
        if len(new) > len(self.free):
            raise RuntimeError(f"{len(new)} pages asked for, {len(self.free)} left")
        taken = [self.free.pop() for _ in new]
        for (b, _), page in zip(new, taken):
            self.held[b].append(page)
        if new:
            at = torch.tensor(new, device=self.table.device)
            self.table[at[:, 0], at[:, 1]] = torch.tensor(taken, dtype=torch.int32, device=self.table.device)

    def release(self, b):
        """Text b has ended: its pages are free again."""
        self.free += self.held[b]
        self.held[b] = []
        self.table[b] = -1


def generate(model, prompts, lengths, steps, page=64, chunk=512):
    """The likeliest next `steps` tokens (B, steps) of prompts (B, P), of which
    text b has lengths[b] (a list), and the cache that holds them."""
    B, P = prompts.shape
    device = prompts.device
    pages = sum(-(-(n + steps) // page) for n in lengths)
    cache = Cache(len(model.layers), B, P + steps, page, pages, device)
    total = torch.tensor(lengths, device=device)
    token = torch.zeros(B, dtype=torch.int64, device=device)
    for at in range(0, P, chunk):  # the prompts, a chunk of all texts that go on at a time
        part = prompts[:, at:at + chunk]
        cache.grow([min(n, at + part.shape[1]) for n in lengths])
        counts = (total - at).clamp(0, part.shape[1])
        scores = model.forward(part, cache, torch.minimum(total, torch.full_like(total, at)), counts)
        token = torch.where((total > at) & (total <= at + part.shape[1]), scores.argmax(-1), token)
    out = [token]
    ones = torch.ones_like(total)
    for step in range(steps - 1):
        cache.grow([n + step + 1 for n in lengths])
        token = model.forward(token[:, None], cache, total + step, ones).argmax(-1)
        out.append(token)
    return torch.stack(out, 1), cache


def main():
    parser = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    parser.add_argument("--texts", type=int, default=8)
    parser.add_argument("--prompt", type=int, default=2000)
    parser.add_argument("--steps", type=int, default=64)
    parser.add_argument("--page", type=int, default=64)
    parser.add_argument("--chunk", type=int, default=512)
    args = parser.parse_args()
    model = Decoder()
    g = torch.Generator().manual_seed(1)
    prompts = torch.randint(0, model.embedding.shape[0], (args.texts, args.prompt), generator=g).cuda()
    lengths = torch.randint(max(1, args.prompt // 8), args.prompt + 1, (args.texts,), generator=g).tolist()
    generate(model, prompts, lengths, min(args.steps, 4), args.page, args.chunk)  # the library loads, its kernels too
    torch.cuda.synchronize()
    start = time.perf_counter()
    tokens, cache = generate(model, prompts, lengths, args.steps, args.page, args.chunk)
    torch.cuda.synchronize()
    seconds = time.perf_counter() - start
    for b in range(args.texts):
        print(f"text {b}: {lengths[b]} tokens, {len(cache.held[b])} pages, then {tokens[b, :10].tolist()} ...")
    print(f"{sum(lengths)} tokens read and {args.texts} x {args.steps} written in {seconds * 1e3:.1f} ms")
    if wpt_b200.device_status():
        raise RuntimeError("a kernel reported a status")


if __name__ == "__main__":
    main()
