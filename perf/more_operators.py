"""What a generation step does between a layer's projections and its attention's
output, measured: rotary positions (with their gradient), appending entries to a
paged cache held in 8 bits, and attention over that cache.

With `own` false, run() computes them from elementary torch operations in 32
bits (angles in 64); with `own` true, it makes the calls that a user of wpt_b200
makes.

The cache: pages (P, page, 2c) of float8_e4m3fn, an entry's key then its value;
scales (P, page / 16, 2) float32, one for the keys and one for the values of each
block of 16 entries; a table (rows, M) of page numbers, -1 for none.
"""

import math

import torch

own = False

_DEVICE = "cuda"
_BLOCK = 16   # entries that share a scale
_TOP = 448.0  # the largest e4m3 number


# ------------------------------------------------------------------ cases

def listed():
    return [
        # one writer's step, the queries of one token (64 of 128 channels turn): launch latency
        dict(name="rotate, one token", op="rotate", rows=1, tokens=1, heads=16, width=128, dims=64, far=4096,
             interleaved=False, scaling="none", dtype="bfloat16", train=False),
        # far positions, pairs of neighbours, odd sizes, float32, a context made eight times as long
        dict(name="rotate, odd", op="rotate", rows=3, tokens=1021, heads=12, width=96, dims=44, far=1048576,
             interleaved=True, scaling="parts", dtype="float32", train=False),
        # a training batch's queries, forward and backward: streams from HBM
        dict(name="rotate, training", op="rotate", rows=8, tokens=4096, heads=16, width=128, dims=64, far=4096,
             interleaved=False, scaling="none", dtype="bfloat16", train=True),
        # one writer's step: one entry after 1,000 others
        dict(name="append, one row", op="append", rows=1, tokens=1, keys=1024, page=16, width=128, dims=64,
             interleaved=False, dtype="bfloat16", ragged=False),
        # a batch's decode step: 64 texts get one entry each
        dict(name="append, 64 rows", op="append", rows=64, tokens=1, keys=8192, page=64, width=128, dims=64,
             interleaved=False, dtype="bfloat16", ragged=True),
        # drafts of unequal lengths, pairs of neighbours, float32 entries of an odd width
        dict(name="append, odd", op="append", rows=5, tokens=37, keys=1999, page=32, width=80, dims=36,
             interleaved=True, dtype="float32", ragged=True),
        # a batch's prompts: streams to HBM
        dict(name="append, prompts", op="append", rows=16, tokens=4096, keys=4096, page=128, width=128, dims=128,
             interleaved=False, dtype="bfloat16", ragged=False),
        # one writer's decode step on a short cache: launch latency
        dict(name="attend, one row", op="attend", rows=1, queries=1, heads=16, keys=1024, page=16, window=0,
             sink=False, ragged=False),
        # four to seven drafts' verification on an odd cache, with sinks
        dict(name="attend, drafts", op="attend", rows=7, queries=5, heads=12, keys=6007, page=32, window=0, sink=True,
             ragged=True),
        # a window layer's decode step
        dict(name="attend, window", op="attend", rows=64, queries=1, heads=32, keys=8192, page=64, window=1024,
             sink=True, ragged=True),
        # a batch's decode step, rows of 1,024 to 32,768 cached tokens: the cache streams from HBM
        dict(name="attend, 64 rows", op="attend", rows=64, queries=1, heads=32, keys=32768, page=64, window=0,
             sink=False, ragged=True),
        # one long text's decode step
        dict(name="attend, one long row", op="attend", rows=1, queries=1, heads=32, keys=262144, page=128, window=0,
             sink=False, ragged=False),
    ]


def _spread(rng, low, high):
    """A size whose logarithm is uniform; most are odd."""
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    return max(low, min(high, n if rng.random() < 0.25 else n | 1))


def draw(rng):
    op = rng.choice(["rotate", "append", "attend", "attend"])
    while True:
        if op == "rotate":
            width = 2 * rng.randint(8, 128)
            case = dict(op=op, rows=_spread(rng, 1, 64), tokens=_spread(rng, 1, 8192),
                        heads=rng.choice([1, 4, 8, 12, 16, 32, 64]), width=width,
                        dims=rng.choice([width, 2 * rng.randint(1, width // 2)]), far=_spread(rng, 128, 1048576),
                        interleaved=rng.random() < 0.5, scaling=rng.choice(["none", "linear", "base", "parts"]),
                        dtype=rng.choice(["bfloat16", "bfloat16", "float32"]), train=rng.random() < 0.5)
            if case["rows"] * case["tokens"] * case["heads"] * width <= 8 * 4096 * 16 * 64:
                return case
        elif op == "append":
            width = 16 * rng.randint(2, 16)
            keys = _spread(rng, 64, 32768)
            case = dict(op=op, rows=_spread(rng, 1, 64), tokens=min(keys, _spread(rng, 1, 4096)), keys=keys,
                        page=rng.choice([16, 32, 64, 128, 256]), width=width,
                        dims=rng.choice([0, width, 2 * rng.randint(1, width // 2)]), interleaved=rng.random() < 0.5,
                        dtype=rng.choice(["bfloat16", "bfloat16", "float32"]), ragged=rng.random() < 0.6)
            if case["rows"] * keys * width <= 64 * 8192 * 128 and \
                    case["rows"] * case["tokens"] * width <= 16 * 4096 * 128:
                return case
        else:
            step = rng.random() < 0.6
            case = dict(op=op, rows=_spread(rng, 1, 64), queries=1 if step else _spread(rng, 2, 64),
                        heads=rng.choice([1, 4, 8, 12, 16, 24, 32, 64]), keys=_spread(rng, 16, 262144),
                        page=rng.choice([16, 32, 64, 128, 256]), window=0 if rng.random() < 0.7 else _spread(rng, 16, 2048),
                        sink=rng.random() < 0.5, ragged=rng.random() < 0.6)
            if case["rows"] * case["keys"] <= 2 ** 20 and \
                    case["rows"] * case["keys"] * case["queries"] * case["heads"] <= 2 ** 26:
                return case


# ----------------------------------------------------------------- inputs

def _frequencies(dims, scaling, factor=8.0, base=10000.0, original=4096):
    """(dims / 2,) float64 angles a position, on the GPU; for a context `factor` times as long as the
    `original`: all slower ("linear"), a larger base ("base"), or only those that turn slowly ("parts")."""
    if scaling == "base":
        base = base * factor ** (dims / max(1, dims - 2))
    i = torch.arange(0, dims, 2, dtype=torch.float64, device=_DEVICE)
    f = base ** (-i / max(1, dims))
    if scaling == "linear":
        f = f / factor
    elif scaling == "parts":
        turns = original * f / (2 * math.pi)  # in the original context: 32 and more stay, one and less slow down
        keep = ((turns - 1) / 31).clamp(0, 1)
        f = f * keep + f / factor * (1 - keep)
    return f


def _power(amax):
    """The least power of two with amax <= 448 times it (2^-60 at least)."""
    m, e = torch.frexp(amax.float() / _TOP)
    e = torch.where(m == 0.5, e - 1, e)
    return torch.ldexp(torch.ones_like(amax, dtype=torch.float32), e.clamp(min=-60))


def _lengths(case, g):
    """Live entries of each row: all of the table's, or from a thirty-second of them up."""
    B, N = case["rows"], case["keys"]
    if not case["ragged"]:
        return torch.full((B,), N, dtype=torch.int64, device=_DEVICE)
    return torch.randint(max(1, N // 32), N + 1, (B,), generator=g, device=_DEVICE)


def _mean_length(case):
    N = case["keys"]
    return (max(1, N // 32) + N) / 2 if case["ragged"] else N


def _cache(case, g, lengths):
    """Pages, scales and table: each row's `lengths` entries in pages taken from anywhere, which hold
    entries to their ends (those of an earlier text)."""
    B, N, S, C = case["rows"], case["keys"], case["page"], case["width"]
    M = -(-N // S)
    used = -(-lengths // S)
    P = B * M + 3
    free = torch.randperm(P, generator=g, device=_DEVICE)[:B * M].view(B, M)
    table = torch.where(torch.arange(M, device=_DEVICE) < used[:, None], free, -1).int()
    pages = torch.zeros(P, S, 2 * C, dtype=torch.float8_e4m3fn, device=_DEVICE)
    scales = torch.zeros(P, S // _BLOCK, 2, device=_DEVICE)
    some = max(1, min(P, 2 ** 25 // (S * C)))
    for p in range(0, P, some):  # the entries' size changes from block to block
        n = min(some, P - p)
        x = torch.randn(n, S // _BLOCK, _BLOCK, 2, C, generator=g, device=_DEVICE)
        x *= torch.exp2(torch.rand(n, S // _BLOCK, 1, 2, 1, generator=g, device=_DEVICE) * 2 - 1)
        s = _power(x.abs().amax((2, 4)))
        scales[p:p + n] = s
        pages[p:p + n] = (x / s[:, :, None, :, None]).reshape(n, S, 2 * C).to(torch.float8_e4m3fn)
    return pages, scales, table


def prepare(case, seed):
    g = torch.Generator(device=_DEVICE).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=_DEVICE)

    if case["op"] == "rotate":
        B, T, H, C = (case[k] for k in ("rows", "tokens", "heads", "width"))
        dtype = getattr(torch, case["dtype"])
        x = normal(B, T, H, C).to(dtype)
        d_out = None
        if case["train"]:
            x.requires_grad_()
            d_out = normal(B, T, H, C).to(dtype)
        first = torch.randint(0, max(1, case["far"] - T) + 1, (B, 1), generator=g, device=_DEVICE)
        return dict(case=case, x=x, d_out=d_out, positions=first + torch.arange(T, device=_DEVICE),
                    frequencies=_frequencies(case["dims"], case["scaling"]))

    if case["op"] == "append":
        B, n, N, C = (case[k] for k in ("rows", "tokens", "keys", "width"))
        new = normal(B, n, 2 * C).to(getattr(torch, case["dtype"]))
        counts = torch.full((B,), n, dtype=torch.int64, device=_DEVICE)
        if case["ragged"] and n > 1:
            counts = torch.randint(1, n + 1, (B,), generator=g, device=_DEVICE)
        lengths = torch.maximum(_lengths(case, g), counts)
        if N > n and not case["ragged"]:
            lengths -= torch.randint(0, min(24, N - n) + 1, (B,), generator=g, device=_DEVICE)
        first = lengths - counts
        pages, scales, table = _cache(case, g, lengths)
        return dict(case=case, new=new, counts=counts, first=first, pages=pages, scales=scales, table=table,
                    frequencies=_frequencies(case["dims"], "none") if case["dims"] else None)

    B, T, H = (case[k] for k in ("rows", "queries", "heads"))
    lengths = torch.clamp(_lengths(case, g), min=min(T, case["keys"]))
    pages, scales, table = _cache(dict(case, width=128), g, lengths)
    # normalised queries, sharp enough to prefer some entries
    q = (normal(B, T, H, 128) * 1.5).bfloat16()
    positions = torch.clamp(lengths[:, None] - T + torch.arange(T, device=_DEVICE), min=-1)
    return dict(case=case, q=q, pages=pages, scales=scales, table=table, positions=positions, scale=128 ** -0.5,
                sink=normal(H) if case["sink"] else None)


# ------------------------------------------------------------- plain forms

def _turn(x, angle, interleaved, sign=1.0):
    """x (..., c), float32, its last channels turned by `angle` (..., dims / 2), float64."""
    cos, sin = torch.cos(angle).float(), (sign * torch.sin(angle)).float()
    dims = 2 * angle.shape[-1]
    held, turned = x[..., :x.shape[-1] - dims], x[..., x.shape[-1] - dims:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        both = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = turned[..., :dims // 2], turned[..., dims // 2:]
        both = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((held, both), -1)


def _rotate_plain(s):
    x, case = s["x"].detach(), s["case"]
    angle = (s["positions"].double()[..., None] * s["frequencies"])[:, :, None]
    y = _turn(x.float(), angle, case["interleaved"]).to(x.dtype)
    if s["d_out"] is None:
        return y
    return y, _turn(s["d_out"].float(), angle, case["interleaved"], -1.0).to(x.dtype)


def _touched(s):
    """The blocks that an append changes, of each row as many as the longest may need: (places in the
    flattened pages, which of them are new, which held an entry before, the new entries' numbers)."""
    case, first, counts, table = s["case"], s["first"], s["counts"], s["table"]
    n, S = case["tokens"], case["page"]
    at = (first // _BLOCK * _BLOCK)[:, None] + torch.arange((n + _BLOCK - 1) // _BLOCK * _BLOCK + _BLOCK, device=first.device)
    new = (at >= first[:, None]) & (at < (first + counts)[:, None])
    begun = (at < first[:, None]) & (counts > 0)[:, None]
    page = torch.gather(table.long(), 1, torch.clamp(at // S, max=table.shape[1] - 1))
    return page * S + at % S, new, begun, torch.clamp(at - first[:, None], 0, n - 1)


def _append_plain(s):
    case, pages, scales = s["case"], s["pages"], s["scales"]
    C = case["width"]
    places, new, begun, which = _touched(s)
    B, K = places.shape
    x = torch.gather(s["new"], 1, which[..., None].expand(-1, -1, 2 * C)).float()
    if s["frequencies"] is not None:
        angle = (s["first"][:, None] + which).double()[..., None] * s["frequencies"]
        x = torch.cat((_turn(x[..., :C], angle, case["interleaved"]), x[..., C:]), -1)
    live = (new | begun).view(B, -1, _BLOCK)
    use = live.any(-1)  # blocks that are there
    spot = torch.where(new | begun, places, 0)
    block = spot.view(B, -1, _BLOCK).amax(-1) // _BLOCK
    flat = scales.view(-1, 2)
    old = torch.where(begun.view(B, -1, _BLOCK).any(-1)[..., None], flat[block], 0.0)
    size = torch.where(new[..., None], x.abs().view(B, K, 2, C).amax(-1), 0.0).view(B, -1, _BLOCK, 2).amax(2)
    scale = torch.maximum(old, _power(size))
    held = pages.view(-1, 2, C)
    shrink = (old / scale).repeat_interleave(_BLOCK, 1)[..., None]
    before = held.view(torch.uint8)[spot].view(torch.float8_e4m3fn).float() * shrink
    after = x.view(B, K, 2, C) / scale.repeat_interleave(_BLOCK, 1)[..., None]
    value = torch.where(new[..., None, None], after, before).to(torch.float8_e4m3fn)
    chosen = new | begun
    held.view(torch.uint8)[places[chosen]] = value.view(torch.uint8)[chosen]
    flat[block[use]] = scale[use]
    return pages, scales


def _entries(s, rows, dtype):
    """(rows, N, 2, c): the cache as one table."""
    pages, scales, table = s["pages"], s["scales"], s["table"][rows].long().clamp(min=0)
    P, S, C2 = pages.shape
    x = pages.view(torch.uint8)[table].view(torch.float8_e4m3fn).to(dtype)
    x = x.view(*table.shape, S // _BLOCK, _BLOCK, 2, C2 // 2) * scales[table].to(dtype)[:, :, :, None, :, None]
    return x.view(table.shape[0], -1, 2, C2 // 2)


def _attend_plain(s, rows=slice(None), dtype=torch.float32):
    case, q, positions = s["case"], s["q"][rows].to(dtype), s["positions"][rows]
    B, T, H, C = q.shape
    x = _entries(s, rows, dtype)
    N = x.shape[1]
    scores = torch.matmul(q.reshape(B, T * H, C), x[:, :, 0].transpose(1, 2)).view(B, T, H, N) * s["scale"]
    n = torch.arange(N, device=q.device)
    seen = n <= positions[..., None]
    if case["window"]:
        seen = seen & (n > positions[..., None] - case["window"])
    scores = torch.where(seen[:, :, None], scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    if s["sink"] is not None:
        top = torch.maximum(top, s["sink"].to(dtype).view(H, 1))
    top = torch.where(top > -math.inf, top, 0.0)
    p = torch.exp(scores - top)
    total = p.sum(-1)
    if s["sink"] is not None:
        total = total + torch.exp(s["sink"].to(dtype).view(H, 1) - top)[..., 0]
    out = torch.matmul(p.view(B, T * H, N), x[:, :, 1]).view(B, T, H, C)
    out = torch.where(total[..., None] > 0, out / total[..., None], 0.0)
    return out, top[..., 0] + torch.log(total)


def run(state):
    op, case = state["case"]["op"], state["case"]
    if own:
        import wpt_b200
        if op == "rotate":
            y = wpt_b200.rotate(state["x"], state["positions"], state["frequencies"], interleaved=case["interleaved"])
            if state["d_out"] is None:
                return y
            return y.detach(), torch.autograd.grad(y, state["x"], state["d_out"])[0]
        if op == "append":
            return wpt_b200.paged_append(state["pages"], state["scales"], state["table"], state["new"],
                                         state["first"], state["counts"], frequencies=state["frequencies"],
                                         interleaved=case["interleaved"])
        return wpt_b200.paged_attention(state["q"], state["pages"], state["scales"], state["table"],
                                        state["positions"], state["scale"], window=case["window"],
                                        sink=state["sink"])
    if op == "rotate":
        return _rotate_plain(state)
    if op == "append":
        return _append_plain(state)
    out, lse = _attend_plain(state)
    return out.bfloat16(), lse


# -------------------------------------------------------- work and 64 bits

def _bytes(name):
    return 4 if name == "float32" else 2


def work(case):
    if case["op"] == "rotate":
        B, T, H, C = (case[k] for k in ("rows", "tokens", "heads", "width"))
        ways = 2 if case["train"] else 1
        return dict(bytes=ways * (2 * B * T * H * C * _bytes(case["dtype"]) + 8 * B * T),
                    flops=ways * 3 * B * T * H * case["dims"])
    if case["op"] == "append":
        B, n, C = (case[k] for k in ("rows", "tokens", "width"))
        n = (n + 1) / 2 if case["ragged"] and n > 1 else n
        # entries in, one byte a value and a scale for each block out
        return dict(bytes=B * (n * 2 * C * (_bytes(case["dtype"]) + 1) + (n + _BLOCK) / _BLOCK * 8 + 24),
                    flops=B * n * (3 * case["dims"] + 2 * C))
    B, T, H, C = case["rows"], case["queries"], case["heads"], 128
    live = max(_mean_length(case), min(T, case["keys"]))
    window = case["window"] or live
    # queries end at the row's last entry: query t from the end reads live - t entries, or its window
    short = min(T, max(0, int(live - window)))  # queries that have a whole window
    rest = min(T, int(live)) - short            # the others read all entries up to themselves
    pairs = short * window + sum(min(window, live - short - i) for i in range(rest))
    keys = min(live, window + T - 1)
    return dict(bytes=B * (keys * (2 * C + 8 / _BLOCK) + keys / case["page"] * 4 + T * H * (4 * C + 4) + 8 * T),
                flops=B * pairs * H * 4 * C)


def _turn64(x, positions, f, interleaved, sign=1):
    """The same turn from complex numbers in 64 bits."""
    dims = 2 * f.numel()
    y = x.double().clone()
    part = y[..., x.shape[-1] - dims:]
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=x.device),
                       sign * positions.double()[..., None] * f)
    if interleaved:
        z = torch.view_as_complex(part.reshape(*part.shape[:-1], dims // 2, 2).contiguous()) * turn
        part.copy_(torch.view_as_real(z).flatten(-2))
    else:
        z = torch.complex(part[..., :dims // 2].contiguous(), part[..., dims // 2:].contiguous()) * turn
        part.copy_(torch.cat((z.real, z.imag), -1))
    return y


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotate":
        p = s["positions"][:, :, None]
        y = _turn64(s["x"].detach(), p, s["frequencies"], case["interleaved"])
        if s["d_out"] is None:
            return y
        return y, _turn64(s["d_out"], p, s["frequencies"], case["interleaved"], -1)
    if case["op"] == "append":
        # the values before their rounding to 8 bits, in units of their block's scale
        S, C = case["page"], case["width"]
        pages, scales = s["pages"].double().view(-1, _BLOCK, 2, C), s["scales"].double().view(-1, 2)
        for b in range(case["rows"]):
            first, count = int(s["first"][b]), int(s["counts"][b])
            x = s["new"][b, :count].double().view(count, 2, C)
            if s["frequencies"] is not None:
                at = first + torch.arange(count, device=x.device)
                x[:, 0] = _turn64(x[:, 0], at, s["frequencies"], case["interleaved"])
            begun = first % _BLOCK
            blocks = -(-(begun + count) // _BLOCK)
            full = torch.zeros(blocks * _BLOCK, 2, C, dtype=torch.float64, device=x.device)
            full[begun:begun + count] = x
            full = full.view(blocks, _BLOCK, 2, C)
            where = torch.arange(first // _BLOCK, first // _BLOCK + blocks, device=x.device)
            where = s["table"][b].long()[where * _BLOCK // S] * (S // _BLOCK) + where % (S // _BLOCK)
            size = full.abs().amax((1, 3))
            scale = torch.exp2(torch.ceil(torch.log2(size / _TOP)).clamp(min=-60))
            if begun:
                scale[0] = torch.maximum(scale[0], scales[where[0]])
                full[0, :begun] = pages[where[0], :begun] * scales[where[0]][:, None]
            mine = torch.zeros(blocks * _BLOCK, dtype=torch.bool, device=x.device)
            mine[:begun + count] = True
            mine = mine.view(blocks, _BLOCK, 1, 1)
            pages[where] = torch.where(mine, full / scale[:, None, :, None], pages[where])
            scales[where] = scale
        return pages.view(s["pages"].shape), scales.view(s["scales"].shape)
    outs, sums = [], []
    for b in range(case["rows"]):
        x = _entries(s, slice(b, b + 1), torch.float64)[0]
        pos = s["positions"][b]
        z = torch.einsum("thc,nc->thn", s["q"][b].double(), x[:, 0]) * s["scale"]
        n = torch.arange(x.shape[0], device=x.device)
        hidden = (n > pos[:, None])[:, None]
        if case["window"]:
            hidden = hidden | (n <= pos[:, None] - case["window"])[:, None]
        z = z.masked_fill(hidden, -math.inf)
        if s["sink"] is not None:
            z = torch.cat((z, s["sink"].double().view(1, -1, 1).expand(z.shape[0], -1, 1)), -1)
        lse = torch.logsumexp(z, -1)
        p = torch.exp(z - lse[..., None]).masked_fill(lse[..., None] == -math.inf, 0)
        outs.append(torch.einsum("thn,nc->thc", p[..., :x.shape[0]], x[:, 1]))
        sums.append(lse)
    return torch.stack(outs), torch.stack(sums)
