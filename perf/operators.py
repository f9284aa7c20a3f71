"""The generation cache's bookkeeping between two decode steps, measured: the
attention weight that each cached row collects, the eviction of the rows that
collect least, beam search's selection over beams and vocabulary, and the
reordering of the beams' cached rows.

With `own` false, run() computes them from elementary torch operations in 32
bits; with `own` true, it makes the calls that a user of wpt_b200 makes.
"""

import math

import torch

own = False

_DEVICE = "cuda"


# ------------------------------------------------------------------ cases

def listed():
    return [
        # one writer's decode step on a short cache: launch latency
        dict(name="weights step, one row", op="weights", rows=1, queries=1, heads=16, keys=1024, width=128, window=0,
             ragged=False),
        # a batch's decode step, rows of 1,024 to 32,768 cached tokens: the keys stream from HBM
        dict(name="weights step, 64 rows", op="weights", rows=64, queries=1, heads=32, keys=32768, width=128,
             window=0, ragged=True),
        # the last places of ragged prompts observe all of their prompt: narrow heads, odd sizes
        dict(name="weights of the last places", op="weights", rows=5, queries=37, heads=12, keys=6007, width=64,
             window=0, ragged=True),
        # every place of a batch of prompts (causal): tensor cores and exponentials
        dict(name="weights of whole prompts", op="weights", rows=8, queries=4096, heads=16, keys=4096, width=128,
             window=0, ragged=False),
        # one row over its budget
        dict(name="evict, one row", op="evict", rows=1, keys=1024, keep=512, recent=64, first=4, width=256,
             dtype="bfloat16", ragged=False),
        # odd budget, ragged rows (some under it), a float32 table
        dict(name="evict, odd", op="evict", rows=7, keys=10007, keep=1501, recent=33, first=1, width=96,
             dtype="float32", ragged=True),
        # a batch of prompts cut to a quarter before decoding
        dict(name="evict, 64 rows", op="evict", rows=64, keys=8192, keep=2048, recent=128, first=4, width=256,
             dtype="bfloat16", ragged=False),
        # one text, four beams: launch latency
        dict(name="select, one text", op="select", rows=1, beams_in=4, beams=4, vocab=65536, dtype="float32",
             finished=False),
        # scores as a bfloat16 head leaves them (ties), an odd vocabulary, more beams out than in, ended beams
        dict(name="select, odd", op="select", rows=5, beams_in=3, beams=7, vocab=50021, dtype="bfloat16",
             finished=True),
        # a batch of 64 texts with eight beams: the scores stream from HBM
        dict(name="select, 64 texts", op="select", rows=64, beams_in=8, beams=8, vocab=65536, dtype="float32",
             finished=True),
        # one text's beams after a short prompt, in two layers' tables
        dict(name="reorder, one text", op="reorder", rows=1, beams=4, keys=600, prompt=500, width=256,
             tables=2, dtype="bfloat16"),
        # 16 texts with eight beams, four layers' tables, 512 shared prompt rows stay where they are
        dict(name="reorder, 16 texts", op="reorder", rows=16, beams=8, keys=2048, prompt=512, width=256,
             tables=4, dtype="bfloat16"),
    ]


def _spread(rng, low, high):
    """A size whose logarithm is uniform; most are odd."""
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    return max(low, min(high, n if rng.random() < 0.25 else n | 1))


def draw(rng):
    op = rng.choice(["weights", "evict", "select", "reorder"])
    while True:
        if op == "weights":
            step = rng.random() < 0.5
            case = dict(op=op, rows=_spread(rng, 1, 64), queries=1 if step else _spread(rng, 2, 4096),
                        heads=rng.choice([1, 4, 8, 12, 16, 24, 32, 64]), keys=_spread(rng, 128, 262144 if step else 8192),
                        width=rng.choice([64, 128, 128]), window=0 if rng.random() < 0.7 else _spread(rng, 64, 2048),
                        ragged=rng.random() < 0.6)
            size = case["rows"] * case["keys"] * (case["queries"] * case["heads"] + 8)
            if size <= 2 ** 31 and case["rows"] * case["keys"] <= 2 ** 21:
                return case
        elif op == "evict":
            keys = _spread(rng, 64, 262144)
            keep = _spread(rng, 16, keys)
            case = dict(op=op, rows=_spread(rng, 1, 64), keys=keys, keep=keep, recent=rng.randint(0, keep // 4),
                        first=rng.randint(0, min(8, keep // 4)), width=8 * rng.randint(2, 64),
                        dtype=rng.choice(["bfloat16", "bfloat16", "float32"]), ragged=rng.random() < 0.6)
            if case["rows"] * keys * case["width"] <= 64 * 8192 * 256:
                return case
        elif op == "select":
            case = dict(op=op, rows=_spread(rng, 1, 64), beams_in=rng.randint(1, 16), beams=rng.randint(1, 16),
                        vocab=_spread(rng, 1000, 131072), dtype=rng.choice(["float32", "bfloat16"]),
                        finished=rng.random() < 0.5)
            if case["rows"] * case["beams_in"] * case["vocab"] <= 2 ** 25:
                return case
        else:
            keys = _spread(rng, 32, 16384)
            case = dict(op=op, rows=_spread(rng, 1, 64), beams=rng.randint(2, 16), keys=keys,
                        prompt=rng.randint(0, keys - 1), width=8 * rng.randint(2, 64), tables=rng.randint(1, 6),
                        dtype=rng.choice(["bfloat16", "bfloat16", "float32"]))
            if case["rows"] * case["beams"] * keys * case["width"] * case["tables"] <= 16 * 8 * 2048 * 256 * 4:
                return case


# ----------------------------------------------------------------- inputs

def _lengths(case, g):
    """Live rows of each cache: the whole table, or from a thirty-second of it up."""
    B, N = case["rows"], case["keys"]
    if not case["ragged"]:
        return torch.full((B,), N, dtype=torch.int64, device=_DEVICE)
    return torch.randint(max(1, N // 32), N + 1, (B,), generator=g, device=_DEVICE)


def _mean_length(case):
    N = case["keys"]
    return (max(1, N // 32) + N) / 2 if case["ragged"] else N


def _visible(case, positions, n):
    """(..., n) whether each query at `positions` reads each row."""
    rows = torch.arange(n, device=positions.device)
    seen = rows <= positions[..., None]
    return seen & (rows > positions[..., None] - case["window"]) if case["window"] else seen


def prepare(case, seed):
    g = torch.Generator(device=_DEVICE).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=_DEVICE)

    if case["op"] == "weights":
        B, T, H, N, C = (case[k] for k in ("rows", "queries", "heads", "keys", "width"))
        # normalised queries and keys, the queries sharp enough to prefer some rows; the keys are one half of
        # the cache's entries; weights hold what earlier steps collected
        q = (normal(B, T, H, C) * 1.5).bfloat16()
        entries = torch.empty(B, N, 2 * C, dtype=torch.bfloat16, device=_DEVICE)
        for b in range(B):
            entries[b] = normal(N, 2 * C).bfloat16()
        lengths = _lengths(case, g)
        # a pass of T queries ends at each row's last token (before the text: no rows)
        positions = lengths[:, None] - T + torch.arange(T, device=_DEVICE)
        positions = torch.where(positions < 0, -1, positions)
        k = entries[..., :C]
        scale = C ** -0.5
        lse = torch.empty(B, T, H, device=_DEVICE)
        for b in range(B):  # what the forward pass returned
            s = torch.einsum("thc,nc->thn", q[b].float(), k[b].float()) * scale
            s = s.masked_fill(~_visible(case, positions[b], N)[:, None], -math.inf)
            lse[b] = torch.logsumexp(s, -1)
        weights = torch.rand(B, N, generator=g, device=_DEVICE)
        return dict(case=case, q=q, k=k, positions=positions, lse=lse, weights=weights, scale=scale)

    if case["op"] == "evict":
        B, N = case["rows"], case["keys"]
        held = normal(B, N, case["width"]).to(getattr(torch, case["dtype"]))
        weights = torch.exp(2 * normal(B, N) - 4)  # few rows hold most of the weight
        return dict(case=case, held=held, weights=weights, lengths=_lengths(case, g))

    if case["op"] == "select":
        R, W, V = case["rows"], case["beams_in"], case["vocab"]
        scores = (normal(R, W, V) * 2).to(getattr(torch, case["dtype"]))
        totals = -20 * torch.rand(R, W, generator=g, device=_DEVICE)
        done = torch.rand(R, W, generator=g, device=_DEVICE) < 0.2 if case["finished"] else None
        return dict(case=case, scores=scores, totals=totals, done=done, end=1 if case["finished"] else None)

    R, W, N = case["rows"], case["beams"], case["keys"]
    tables = [normal(R * W, N, case["width"]).to(getattr(torch, case["dtype"])) for _ in range(case["tables"])]
    parents = torch.randint(0, W, (R, W), generator=g, device=_DEVICE)
    lengths = torch.full((R * W,), N, dtype=torch.int64, device=_DEVICE)
    first = torch.full((R,), case["prompt"], dtype=torch.int64, device=_DEVICE)
    return dict(case=case, tables=tables, parents=parents, lengths=lengths, first=first)


# ------------------------------------------------------------- plain forms

def _weights_plain(s):
    q, k, positions = s["q"], s["k"], s["positions"]
    B, T, H, C = q.shape
    scores = torch.matmul(q.float().reshape(B, T * H, C), k.float().transpose(1, 2)).view(B, T, H, -1)
    p = torch.exp(scores * s["scale"] - s["lse"][..., None])
    seen = _visible(s["case"], positions, k.shape[1])[:, :, None]
    return s["weights"].add_(torch.where(seen, p, 0.0).sum((1, 2)))


def _evict_plain(s):
    case, held, weights, lengths = s["case"], s["held"], s["weights"], s["lengths"]
    N, keep = case["keys"], case["keep"]
    n = torch.arange(N, device=held.device)
    live = n < lengths[:, None]
    kept = (n < case["first"]) | (n >= lengths[:, None] - case["recent"])
    rank = torch.where(live, torch.where(kept, math.inf, weights), -math.inf)  # the weights are finite
    order = torch.sort(rank, dim=1, descending=True, stable=True).indices[:, :keep]
    counts = torch.clamp(lengths, max=keep)
    valid = torch.arange(keep, device=held.device) < counts[:, None]
    rows = torch.sort(torch.where(valid, order, N), dim=1).values
    at = torch.where(valid, rows, 0)
    out = torch.gather(held, 1, at[..., None].expand(-1, -1, held.shape[2]))
    out = torch.where(valid[..., None], out, 0.0)
    return out, torch.where(valid, torch.gather(weights, 1, at), 0.0), torch.where(valid, rows, -1), counts


def _select_plain(s):
    totals, done, end, K = s["totals"], s["done"], s["end"], s["case"]["beams"]
    x = s["scores"].float()
    R, W, V = x.shape
    d = x - x.amax(-1, keepdim=True)
    value = totals[..., None] + (d - torch.log(torch.exp(d).sum(-1, keepdim=True)))
    if done is not None:  # an ended beam has one candidate, itself
        ended = torch.where(torch.arange(V, device=x.device) == end, totals[..., None], -math.inf)
        value = torch.where(done[..., None], ended, value)
    # equal values go to the lowest index: the value's bits in an order of whole numbers, then the index
    value = value.reshape(R, W * V) + 0.0
    bits = value.view(torch.int32).long()
    bits = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
    key = bits * 2 ** 32 + (2 ** 32 - 1 - torch.arange(W * V, device=x.device))
    at = torch.topk(key, K, dim=1).indices
    best = torch.gather(value, 1, at)
    some = best > -math.inf
    parents = torch.where(some, torch.div(at, V, rounding_mode="floor"), -1)
    return torch.where(some, best, -math.inf), parents, torch.where(some, at % V, -1)


def _reorder_plain(s):
    parents, lengths, first, case = s["parents"], s["lengths"], s["first"], s["case"]
    R, W = parents.shape
    n = torch.arange(case["keys"], device=parents.device)
    source = (torch.arange(R, device=parents.device)[:, None] * W + parents).reshape(-1)
    moved = (n >= first.repeat_interleave(W)[:, None]) & (n < lengths[source][:, None])
    return [t.copy_(torch.where(moved[..., None], t[source], t)) for t in s["tables"]]


def run(state):
    op, case = state["case"]["op"], state["case"]
    if own:
        import wpt_b200
        if op == "weights":
            return wpt_b200.attention_weights(state["q"], state["k"], state["positions"], state["lse"],
                                              state["scale"], state["weights"], window=case["window"])
        if op == "evict":
            return wpt_b200.cache_evict(state["held"], state["weights"], state["lengths"], case["keep"],
                                        recent=case["recent"], first=case["first"])
        if op == "select":
            return wpt_b200.beam_select(state["scores"], state["totals"], case["beams"], done=state["done"],
                                        end=state["end"])
        return wpt_b200.cache_reorder(state["tables"], state["parents"], state["lengths"], first=state["first"])
    return dict(weights=_weights_plain, evict=_evict_plain, select=_select_plain, reorder=_reorder_plain)[op](state)


# -------------------------------------------------------- work and 64 bits

def _bytes(name):
    return 4 if name == "float32" else 2


def work(case):
    if case["op"] == "weights":
        B, T, H, C = (case[k] for k in ("rows", "queries", "heads", "width"))
        live = _mean_length(case)
        window = case["window"] or live
        # queries end at the row's last token: query t from the end reads live - t rows, or its window
        short = min(T, max(0, int(live - window)))  # queries that have a whole window
        rest = min(T, int(live)) - short            # the others read all rows up to themselves
        pairs = short * window + sum(min(window, live - short - i) for i in range(rest))
        keys = min(live, window + T)
        return dict(bytes=B * (keys * (2 * C + 8) + T * H * (2 * C + 4) + 8 * T), flops=B * pairs * H * 2 * C)
    if case["op"] == "evict":
        B, keep, row = case["rows"], case["keep"], case["width"] * _bytes(case["dtype"])
        live = _mean_length(case)
        kept = min(keep, live)
        return dict(bytes=B * (4 * live + kept * row + keep * (row + 4 + 8) + 16), flops=0)
    if case["op"] == "select":
        R, W, K = case["rows"], case["beams_in"], case["beams"]
        beams = W * (0.8 if case["finished"] else 1)  # an ended beam's scores are not read
        return dict(bytes=R * (beams * case["vocab"] * _bytes(case["dtype"]) + 5 * W + 20 * K), flops=0)
    R, W = case["rows"], case["beams"]
    span = (case["keys"] - case["prompt"]) * case["width"] * _bytes(case["dtype"]) * case["tables"]
    # random parents: W - 1 beams of W change, and a beam is read unless no other one takes it
    return dict(bytes=R * span * ((W - 1) + W * (1 - (1 - 1 / W) ** (W - 1))) + 16 * R * W, flops=0)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "weights":
        out = s["weights"].double()
        T = case["queries"]
        step = max(1, 2 ** 28 // (case["heads"] * case["keys"]))
        for b in range(case["rows"]):
            k = s["k"][b].double()
            for t in range(0, T, step):
                score = torch.einsum("thc,nc->thn", s["q"][b, t:t + step].double(), k) * s["scale"]
                score -= s["lse"][b, t:t + step].double()[..., None]
                p = s["positions"][b, t:t + step, None, None]
                n = torch.arange(case["keys"], device=_DEVICE)
                hidden = n > p
                if case["window"]:
                    hidden = hidden | (n <= p - case["window"])
                out[b] += score.exp_().masked_fill_(hidden, 0).sum((0, 1))
        return out
    if case["op"] == "evict":
        B, keep, first, recent = case["rows"], case["keep"], case["first"], case["recent"]
        out = torch.zeros(B, keep, case["width"], dtype=torch.float64, device=_DEVICE)
        held_weights = torch.zeros(B, keep, dtype=torch.float64, device=_DEVICE)
        for b in range(B):
            n = int(s["lengths"][b])
            at = torch.arange(n, device=_DEVICE)
            if n > keep:
                middle = s["weights"][b, first:n - recent].double()
                best = torch.sort(middle, descending=True, stable=True).indices[:keep - first - recent] + first
                at = torch.cat([at[:first], torch.sort(best).values, at[n - recent:]])
            out[b, :len(at)] = s["held"][b, at].double()
            held_weights[b, :len(at)] = s["weights"][b, at].double()
        return out, held_weights, None, None
    if case["op"] == "select":
        R, W, K = case["rows"], case["beams_in"], case["beams"]
        best = torch.full((R, K), -math.inf, dtype=torch.float64, device=_DEVICE)
        for r in range(R):
            value = s["totals"][r].double()[:, None] + torch.log_softmax(s["scores"][r].double(), -1)
            found = torch.topk(value, min(K, value.shape[1]), dim=1).values
            if s["done"] is not None:
                found = [s["totals"][r, w:w + 1].double() if s["done"][r, w] else found[w] for w in range(W)]
                found = torch.cat(found)
            top = torch.sort(found.reshape(-1), descending=True).values[:K]
            best[r, :len(top)] = top
        return best, None, None
    W, cut = case["beams"], case["prompt"]
    done = []
    for t in s["tables"]:
        moved = t.double().view(case["rows"], W, case["keys"], -1)
        old = moved.clone()
        for r in range(case["rows"]):
            for w, parent in enumerate(s["parents"][r].tolist()):
                moved[r, w, cut:] = old[r, parent, cut:]
        done.append(moved.view(t.shape))
    return done
