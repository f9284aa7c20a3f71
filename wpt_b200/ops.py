"""Forward operations over the C ABI (include/wpt_attn.h): tensor checks,
output and scratch allocation through torch's caching allocator, and the
choice of kernel and split count. Every function here launches CUDA
kernels of libwpt_b200.so on the current stream; none has a CPU path.

Kernel choice: queries x heads of one batch row fill the 128 rows of the
prefill kernel's tiles (tcgen05, M = 128 rows); with few queries per row
(decode, short extends) the key-stream kernel computes S^T = K Q^T with the
keys as M instead, and splits long rows over many CTAs.
"""

import ctypes
import math
import os

import torch

from . import _lib

LAUNCHES = [0]  # kernels this module has launched (read by bench.py around its timed region)
# key tiles per key-stream CTA when set (WPT_B200_CHUNK, read once): overrides the split heuristic
CHUNK_TILES = int(os.environ.get("WPT_B200_CHUNK", "0"))
# the prefill kernel's 2-split cluster combine (WPT_B200_PREFILL_CLUSTER=0 turns it off)
PREFILL_CLUSTER = os.environ.get("WPT_B200_PREFILL_CLUSTER", "1") != "0"


def _need_cuda(*tensors):
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise ValueError("wpt_b200 computes on a CUDA device only; got a tensor on " + str(t.device))


_SMS = {}


def sm_count(device):
    """The streaming multiprocessors of `device`, asked of the runtime once."""
    index = device.index if device.index is not None else torch.cuda.current_device()
    n = _SMS.get(index)
    if n is None:
        n = _SMS[index] = torch.cuda.get_device_properties(index).multi_processor_count
    return n


def _bf16(x):
    """The kernels compute in bf16 (WPT's compute dtype under autocast,
    packages/wpt-model/src/wpt_model/layers.py:13-17). Other dtypes are
    refused rather than rounded: the reference computes in the inputs'
    dtype, so silently rounding float32 inputs would return float32
    tensors of bf16 accuracy. NotImplementedError is what the reference's
    kernel tests skip on (tests/test_kernels.py:149-154)."""
    if x.dtype != torch.bfloat16:
        raise NotImplementedError(f"wpt_b200 computes attention in bfloat16; got {x.dtype} "
                                  "(cast q, k and v to bfloat16, as WPT's autocast does)")
    return x


def _table(x):
    """A (B, N, C) table whose last dimension is contiguous, strides in
    multiples of 8 elements (16 bytes), at a 16-byte aligned address."""
    x = _bf16(x)
    sb, sn, sc = x.stride()
    ok = sc == 1 and sn % 8 == 0 and (sb % 8 == 0 or x.shape[0] == 1) and x.data_ptr() % 16 == 0
    return x if ok else x.contiguous()


def _rows(x):
    if x.dtype == torch.int64 and x.is_contiguous():
        return x
    return x.to(torch.int64).contiguous()


def _splits_for(ctas, tiles, sms):
    """Split count for a grid of `ctas` work items over `tiles` key tiles
    each: the persistent kernel runs the ctas * splits items in waves of
    one per SM, so the estimate is waves x (tiles per item + about 2 tiles'
    worth of per-item cost), plus half a tile per split for the merge; the
    cheapest count up to 32 (never more than the tiles) wins."""
    if ctas >= sms or tiles <= 1:
        return 1
    best, best_cost = 1, None
    for s in range(1, min(tiles, 32) + 1):
        cost = math.ceil(ctas * s / sms) * (tiles / s + 2) + (0.5 * s if s > 1 else 0.0)
        if best_cost is None or cost < best_cost:
            best, best_cost = s, cost
    return best


def prefill_forward(q, k, v, positions, scale, window=0, floor=None, tree_bits=None, tree_base=None, sink=None,
                    splits=None):
    """(out (B, T, H, C) bf16, lse (B, T, H) fp32) from the tcgen05 prefill
    kernel: each query reads rows max(0, p - window + 1, floor) ..
    min(p, N - 1) of k and v, p its position; tree_bits/tree_base give the
    tree mask; sink (H,) joins each head's denominator."""
    _need_cuda(q, k, v, positions, floor, tree_bits, tree_base, sink)
    q = _bf16(q).contiguous()
    k, v = _table(k), _table(v)
    B, T, H, C = q.shape
    N = k.shape[1]
    positions = _rows(positions)
    floor = None if floor is None else _rows(floor)
    if tree_bits is not None:
        tree_bits = tree_bits.to(torch.int64).contiguous()
        tree_base = _rows(tree_base)
    if sink is not None:
        sink = sink.float().contiguous()
    out = torch.empty_like(q)
    lse = torch.empty(B, T, H, dtype=torch.float32, device=q.device)
    TQ = max(1, 128 // H)
    if splits is None:
        tiles = window // 128 + 2 if window else (N + 127) // 128
        splits = _splits_for(B * math.ceil(T / (2 * TQ)), tiles, sm_count(q.device))  # one item per tile pair
    part_o = part_lse = None
    # two splits with one work item per SM: the pair's splits combine as one
    # 2-CTA cluster in shared memory (no partials, no merge launch)
    cluster = (splits == 2 and PREFILL_CLUSTER and 2 * B * math.ceil(T / (2 * TQ)) <= sm_count(q.device))
    if splits > 1 and not cluster:
        part_o = torch.empty(splits, B * T * H, C, dtype=torch.float32, device=q.device)
        part_lse = torch.empty(splits, B * T * H, dtype=torch.float32, device=q.device)
    _lib.check(_lib.lib().wpt_attn_prefill(
        _lib.ptr(q), _lib.ptr(k), _lib.ptr(v), k.stride(0), k.stride(1), v.stride(0), v.stride(1),
        _lib.ptr(positions), _lib.ptr(floor), _lib.ptr(tree_bits), _lib.ptr(tree_base), _lib.ptr(sink),
        _lib.ptr(out), _lib.ptr(lse), _lib.ptr(part_o), _lib.ptr(part_lse), int(splits),
        B, T, H, C, N, int(window), float(scale), _lib.stream(q.device)))
    LAUNCHES[0] += 1 + (splits > 1 and not cluster)
    return out, lse


def _stream_shape(T, H, gather):
    """(columns per CTA, queries per CTA) of the key-stream kernel, as the C
    launcher derives them."""
    cols = H if gather else min(T * H, 64)
    ncol = 16 if cols <= 16 else 32 if cols <= 32 else 64
    return ncol, (1 if gather else ncol // H)


def uses_stream(T, H, C):
    """Whether the key-stream kernel computes this shape (few queries per row)."""
    return C == 128 and H <= 64 and T * H <= 64


_PLAN_CACHE = {}


def _stream_plan(B, T, H, N, K, window, gather, sms, chunk_tiles=None):
    """(chunk_tiles, splits, cluster) of a key-stream call: each query
    group's key slots are cut into chunks of chunk_tiles key tiles, one CTA
    per chunk; cluster: the splits of a group combine in shared memory as one
    thread-block cluster (2 to 8 splits on a grid of one wave) instead of
    through partials and a merge kernel. Remembered per shape (a decode loop
    asks the same question every step)."""
    key = (B, T, H, N, K, window, gather, sms, chunk_tiles)
    plan = _PLAN_CACHE.get(key)
    if plan is None:
        if len(_PLAN_CACHE) > 4096:
            _PLAN_CACHE.clear()
        plan = _PLAN_CACHE[key] = _stream_plan_for(B, T, H, N, K, window, gather, sms, chunk_tiles)
    return plan


def _stream_plan_for(B, T, H, N, K, window, gather, sms, chunk_tiles):
    _, TQ = _stream_shape(T, H, gather)
    groups = B * math.ceil(T / TQ)
    if gather:
        slots = K + max(window, 0)
    else:
        slots = min(N, window + TQ - 1) if window > 0 else N
    tiles = max(1, math.ceil(slots / 128))
    if chunk_tiles is None:
        chunk_tiles = CHUNK_TILES
    auto = not chunk_tiles
    if not chunk_tiles and gather:
        # every query gathers exactly `tiles` tiles: its slots split so that
        # the grid is about one CTA per SM
        chunk_tiles = math.ceil(tiles / max(1, sms // groups))
    elif not chunk_tiles:
        # at least 16 key tiles per CTA (a CTA's start-up costs about as much
        # as streaming a few tiles), more when that still gives two CTAs per
        # SM for rows of the table's full length (most rows are shorter)
        chunk_tiles = max(min(16, tiles), 16 * math.ceil(tiles * groups / (2 * sms) / 16))
        if tiles >= 64 and 2 * math.ceil(tiles / chunk_tiles) * groups < sms:
            # a few long rows (a GPU's shard of a long-context decode) that
            # would leave most SMs idle: about one CTA per SM
            chunk_tiles = max(2, math.ceil(tiles * groups / sms))
    chunk_tiles = max(1, min(int(chunk_tiles), tiles))
    splits = math.ceil(tiles / chunk_tiles)
    if auto and splits == 1 and tiles >= 2 and 2 * groups <= sms:
        # short rows (window rows) on fewer CTAs than SMs: each row's tiles
        # over a cluster of up to 8 CTAs, still one wave
        splits = min(8, tiles, sms // groups)
        chunk_tiles = math.ceil(tiles / splits)
        splits = math.ceil(tiles / chunk_tiles)
    return chunk_tiles, splits, 1 < splits <= 8 and groups * splits <= sms


def stream_forward(q, k, v, positions, scale, window=0, floor=None, idx=None, sink=None, chunk_tiles=None):
    """(out (B, T, H, C) bf16, lse (B, T, H) fp32) from the key-stream
    kernel. Range mode (idx None): as prefill_forward. Gather mode: each
    query reads rows idx[b, t, :] (-1 for none) and its last `window` rows."""
    _need_cuda(q, k, v, positions, floor, idx, sink)
    q = _bf16(q).contiguous()
    k, v = _table(k), _table(v)
    B, T, H, C = q.shape
    N = k.shape[1]
    positions = _rows(positions)
    floor = None if floor is None else _rows(floor)
    gather = idx is not None
    K = 0
    if gather:
        idx = _rows(idx)
        K = idx.shape[-1]
    if sink is not None and (sink.dtype != torch.float32 or not sink.is_contiguous()):
        sink = sink.float().contiguous()
    dev = q.device
    chunk_tiles, splits, cluster = _stream_plan(B, T, H, N, K, window, gather, sm_count(dev), chunk_tiles)
    out = torch.empty_like(q)
    lse = torch.empty((B, T, H), dtype=torch.float32, device=dev)
    part_o = part_lse = None
    if splits > 1 and not cluster:
        part_o = torch.empty((splits, B * T * H, C), dtype=torch.float32, device=dev)
        part_lse = torch.empty((splits, B * T * H), dtype=torch.float32, device=dev)
    ks, vs = k.stride(), v.stride()
    _lib.check(_lib.lib().wpt_attn_decode(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), ks[0], ks[1], vs[0], vs[1],
        positions.data_ptr(), _lib.ptr(floor), _lib.ptr(idx), K, _lib.ptr(sink), out.data_ptr(), lse.data_ptr(),
        _lib.ptr(part_o), _lib.ptr(part_lse), splits, chunk_tiles, B, T, H, C, N, int(window), float(scale),
        _lib.stream(dev)))
    LAUNCHES[0] += 1 + (splits > 1 and not cluster)
    return out, lse


def partials_plan(q_shape, N, device, window=0):
    """(splits, chunk_tiles) the key-stream kernel uses for partials of a
    (B, T, H, C) query block over N keys: at least two splits."""
    B, T, H, C = q_shape
    chunk_tiles, splits, _ = _stream_plan(B, T, H, N, 0, window, False, sm_count(device), None)
    if splits < 2:  # at least two partials, so that the caller always has partials to merge
        chunk_tiles, splits = max(1, math.ceil(chunk_tiles / 2)), 2
    return splits, chunk_tiles


def stream_partials(q, k, v, positions, scale, window=0, into=None, splits=None):
    """The key-stream kernel's split partials without the merge: (part_o
    (S, B*T*H, C) fp32, each split's output normalised by its own sum;
    part_lse (S, B*T*H) fp32, the natural log of that sum, -inf for a split
    with no visible row), S >= 2 (partials_plan). For callers that merge
    them with partials computed elsewhere (merge_partials, merge_groups),
    e.g. on the other GPUs of a long row. into=(part_o, part_lse): write
    there (contiguous fp32 of those shapes) instead of new tensors.
    splits: this many partials (>= 2) instead of partials_plan's count, the
    keys cut into that many equal chunks of whole tiles (splits with no key
    give -inf log-sums): ranks whose shards differ in length then still
    produce chunks of one layout."""
    _need_cuda(q, k, v, positions)
    q = _bf16(q).contiguous()
    k, v = _table(k), _table(v)
    B, T, H, C = q.shape
    N = k.shape[1]
    positions = _rows(positions)
    if splits is None:
        splits, chunk_tiles = partials_plan(q.shape, N, q.device, window)
    else:
        splits = max(2, int(splits))
        slots = min(N, window + 63) if window > 0 else N
        chunk_tiles = max(1, math.ceil(math.ceil(slots / 128) / splits))
    if into is None:
        part_o = torch.empty(splits, B * T * H, C, dtype=torch.float32, device=q.device)
        part_lse = torch.empty(splits, B * T * H, dtype=torch.float32, device=q.device)
    else:
        part_o, part_lse = into
        if (part_o.shape != (splits, B * T * H, C) or part_lse.shape != (splits, B * T * H)
                or not part_o.is_contiguous() or not part_lse.is_contiguous()):
            raise ValueError("stream_partials: `into` does not match partials_plan's shapes")
    _lib.check(_lib.lib().wpt_attn_decode(
        _lib.ptr(q), _lib.ptr(k), _lib.ptr(v), k.stride(0), k.stride(1), v.stride(0), v.stride(1),
        _lib.ptr(positions), None, None, 0, None, None, None, _lib.ptr(part_o), _lib.ptr(part_lse), splits,
        chunk_tiles, B, T, H, C, N, int(window), float(scale), _lib.stream(q.device)))
    LAUNCHES[0] += 1
    return part_o, part_lse


def merge_partial(part_o, part_lse, out_o=None, out_lse=None):
    """Merge of S split partials (part_o (S, rows, C), part_lse (S, rows)
    fp32) into one partial of the same kind, no sink: (out_o (rows, C) fp32,
    the splits' output normalised by their common sum; out_lse (rows,), its
    log). out_o / out_lse: write there (contiguous fp32) instead."""
    _need_cuda(part_o, part_lse, out_o, out_lse)
    S, rows, C = part_o.shape
    out_o = torch.empty(rows, C, dtype=torch.float32, device=part_o.device) if out_o is None else out_o
    out_lse = torch.empty(rows, dtype=torch.float32, device=part_o.device) if out_lse is None else out_lse
    _lib.check(_lib.lib().wpt_attn_merge_partial(_lib.ptr(part_o), _lib.ptr(part_lse), S, rows, rows, C,
                                                 _lib.ptr(out_o), _lib.ptr(out_lse), _lib.stream(part_o.device)))
    LAUNCHES[0] += 1
    return out_o, out_lse


def merge_groups(parts, per, rows, H, C, sink=None, out=None, lse=None):
    """Merge of partials gathered side by side: parts (G, group_floats) fp32,
    chunk g = `per` splits' output partials (per, rows, C) then their
    log-sums (per, rows). Returns (out (rows, C) bf16, lse (rows,) fp32)."""
    _need_cuda(parts, sink)
    G, group_floats = parts.shape
    if sink is not None:
        sink = sink.float().contiguous()
    out = torch.empty(rows, C, dtype=torch.bfloat16, device=parts.device) if out is None else out
    lse = torch.empty(rows, dtype=torch.float32, device=parts.device) if lse is None else lse
    _lib.check(_lib.lib().wpt_attn_merge_groups(_lib.ptr(parts), G, per, rows, group_floats, H, C, _lib.ptr(sink),
                                                _lib.ptr(out), _lib.ptr(lse), _lib.stream(parts.device)))
    LAUNCHES[0] += 1
    return out, lse


def exchange(part_o, part_lse, peers, world, rank, H, sink=None):
    """The long row's combine across GPUs in one kernel (wpt_attn_exchange):
    this rank's split partials (part_o (S, rows, C), part_lse (S, rows)
    fp32) are merged, stored into every rank's exchange buffer (peers: a
    ctypes array of the world buffers as mapped here), and, once every
    rank's result of the same call has landed, merged with the sink into
    (out (rows, C) bf16, lse (rows,) fp32)."""
    _need_cuda(part_o, part_lse, sink)
    S, rows, C = part_o.shape
    if sink is not None:
        sink = sink.float().contiguous()
    out = torch.empty(rows, C, dtype=torch.bfloat16, device=part_o.device)
    lse = torch.empty(rows, dtype=torch.float32, device=part_o.device)
    _lib.check(_lib.lib().wpt_attn_exchange(_lib.ptr(part_o), _lib.ptr(part_lse), S, rows, H, C, _lib.ptr(sink),
                                            peers, world, rank, _lib.ptr(out), _lib.ptr(lse),
                                            _lib.stream(part_o.device)))
    LAUNCHES[0] += 1
    return out, lse


def attention_forward(q, k, v, positions, scale, window=0, floor=None, sink=None):
    """Range attention by the kernel that suits the shape: the key-stream
    kernel for few queries per row, the prefill kernel otherwise."""
    B, T, H, C = q.shape
    if uses_stream(T, H, C):
        return stream_forward(q, k, v, positions, scale, window=window, floor=floor, sink=sink)
    return prefill_forward(q, k, v, positions, scale, window=window, floor=floor, sink=sink)


def select_rows(q, k, positions, lse, scale, K, window):
    """Each query's K chosen rows (B, T, K) int64 (pytorch_kernels.py:112-117):
    the top K by max_h (q_h . k_n * scale - lse_h) among rows 0 .. p - window,
    -1 padded. lse is the forward pass's (B, T, H)."""
    _need_cuda(q, k, positions, lse)
    q = _bf16(q).contiguous()
    k = _table(k)
    B, T, H, C = q.shape
    N = k.shape[1]
    positions = _rows(positions)
    lse = lse.float().contiguous()
    chosen = torch.empty(B, T, K, dtype=torch.int64, device=q.device)
    if K == 0:
        return chosen
    ld = (N + 3) // 4 * 4
    scores = torch.empty(B * T, ld, dtype=torch.float32, device=q.device)
    _lib.check(_lib.lib().wpt_attn_topk(
        _lib.ptr(q), _lib.ptr(k), k.stride(0), k.stride(1), _lib.ptr(positions), _lib.ptr(lse), _lib.ptr(scores),
        ld, _lib.ptr(chosen), int(K), B, T, H, C, N, int(window), float(scale), _lib.stream(q.device)))
    LAUNCHES[0] += 2
    return chosen


def merge_partials(part_o, part_lse, H, sink=None, out=None, lse=None):
    """Log-sum-exp merge of split partials: part_o (S, rows, C) fp32,
    part_lse (S, rows) -> (out (rows, C) bf16, lse (rows,) fp32)."""
    _need_cuda(part_o, part_lse, sink)
    S, rows, C = part_o.shape
    part_o, part_lse = part_o.float().contiguous(), part_lse.float().contiguous()
    if sink is not None:
        sink = sink.float().contiguous()
    out = torch.empty(rows, C, dtype=torch.bfloat16, device=part_o.device) if out is None else out
    lse = torch.empty(rows, dtype=torch.float32, device=part_o.device) if lse is None else lse
    _lib.check(_lib.lib().wpt_attn_merge(_lib.ptr(part_o), _lib.ptr(part_lse), S, rows, rows, H, C, _lib.ptr(sink),
                                         _lib.ptr(out), _lib.ptr(lse), _lib.stream(part_o.device)))
    LAUNCHES[0] += 1
    return out, lse


def attention_backward(q, k, v, positions, out, lse, d_out, scale, window=0, floor=None, sink=None, idx=None,
                       f32=False):
    """Gradients of range attention (each query reads rows max(0, p - window
    + 1, floor) .. min(p, N - 1)), plus its chosen rows idx (B, T, K) when
    given (sparse attention), sink (H,) in the denominators, from the forward
    pass's out (bf16) and lse: (dq (B, T, H, C), dk, dv (B, N, C) in bf16, or
    fp32 when f32; d_sink (H,) fp32 or None). Tensor-core kernels (bwd_prep,
    bwd_kv, bwd_q, and bwd_gather for chosen rows) on the current stream."""
    _need_cuda(q, k, v, positions, out, lse, d_out, floor, sink, idx)
    q = _bf16(q).contiguous()
    k, v = _table(k), _table(v)
    B, T, H, C = q.shape
    N = k.shape[1]
    positions = _rows(positions)
    floor = None if floor is None else _rows(floor)
    K = 0
    if idx is not None and idx.shape[-1] > 0:
        idx = _rows(idx)
        K = idx.shape[-1]
    else:
        idx = None
    out = _bf16(out).contiguous()
    d_out = d_out.to(torch.bfloat16).contiguous()
    lse = lse.float().contiguous()
    if sink is not None:
        sink = sink.float().contiguous()
    wide = f32 or K > 0  # chosen rows are added by fp32 atomics
    dtype = torch.float32 if wide else torch.bfloat16
    dq = torch.empty(B, T, H, C, dtype=dtype, device=q.device)
    dk = torch.empty(B, N, C, dtype=dtype, device=q.device)
    dv = torch.empty(B, N, C, dtype=dtype, device=q.device)
    d_sink = None if sink is None else torch.empty(H, dtype=torch.float32, device=q.device)
    nbytes = _lib.lib().wpt_attn_backward_scratch_bytes(B, T, H, C, N)
    if nbytes == 0:
        raise NotImplementedError(f"attention backward for B={B} T={T} H={H} C={C} N={N}: the kernels take "
                                  "head width 128 and up to 128 heads")
    scratch = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
    _lib.check(_lib.lib().wpt_attn_backward(
        _lib.ptr(q), _lib.ptr(k), _lib.ptr(v), k.stride(0), k.stride(1), v.stride(0), v.stride(1),
        _lib.ptr(positions), _lib.ptr(floor), _lib.ptr(idx), K, _lib.ptr(sink), _lib.ptr(out), _lib.ptr(lse),
        _lib.ptr(d_out), _lib.ptr(dq), _lib.ptr(dk), _lib.ptr(dv), _lib.ptr(d_sink), _lib.ptr(scratch),
        1 if wide else 0, B, T, H, C, N, int(window), float(scale), _lib.stream(q.device)))
    LAUNCHES[0] += 3 + (sink is not None) + (K > 0)
    if wide and not f32:
        dq, dk, dv = (to_bf16(x) for x in (dq, dk, dv))
    return dq, dk, dv, d_sink


def to_bf16(x):
    """A contiguous fp32 tensor rounded to bf16 by the library's kernel."""
    y = torch.empty(x.shape, dtype=torch.bfloat16, device=x.device)
    _lib.check(_lib.lib().wpt_f32_to_bf16(_lib.ptr(x), x.numel(), _lib.ptr(y), _lib.stream(x.device)))
    LAUNCHES[0] += 1
    return y


def cache_append(held, new, first, counts, need=None):
    """The generation cache's entries write (cache.py:110-128): row b's new
    entries new[b, :counts[b]] go to rows first[b] .. of the held table
    (B, capacity, ...), grown to max(need, 2 * capacity) rows (zeros) when
    `need` rows do not fit, as the reference grows it. Returns (held, the
    first `need` rows of it). need = max_b(first[b] + counts[b]) is what the
    reference reads back to the host; a caller that knows it (its own count
    of each row's tokens) passes it, and the call then launches one kernel
    and synchronises nothing."""
    _need_cuda(new, first, counts)
    B, n = new.shape[:2]
    first, counts = _rows(first), _rows(counts)
    if need is None:
        need = int((first + counts).max()) if B else 0  # the reference's own host read
    if held is None:
        held = new.new_zeros((B, 0) + tuple(new.shape[2:]))
    cap = held.shape[1]
    if need > cap:
        held = torch.cat([held, held.new_zeros((B, max(need, 2 * cap) - cap) + tuple(held.shape[2:]))], 1)
    held = held.to(new.dtype)
    if B and n:
        es = new.element_size()
        row_bytes = es * math.prod(new.shape[2:])
        if new.stride(-1) != 1 or (new.dim() > 3 and not new[0, 0].is_contiguous()):
            new = new.contiguous()
        _lib.check(_lib.lib().wpt_cache_append(
            _lib.ptr(new), new.stride(0) * es, new.stride(1) * es, _lib.ptr(held), held.stride(0) * es,
            held.stride(1) * es, _lib.ptr(first), _lib.ptr(counts), B, n, row_bytes, held.shape[1],
            _lib.stream(new.device)))
        LAUNCHES[0] += 1
    return held, held[:, :need]


def tree_bits(parents, B, base=None):
    """(n,) or (B, n) int64 parent indices on the GPU (-1 for a root,
    parents[i] < i) -> ((B, n) int64 ancestor masks: bit j of node i is set
    when node j is i or one of its ancestors; (B, n) positions base[b] + i
    when base (B,) is given, else None). One small kernel on the current
    stream: no host synchronisation, so verification can be captured in a
    CUDA graph. A parent that is not before its child ends that node's walk
    (the mask then holds the nodes met so far)."""
    n = parents.shape[-1]
    if n > 64:
        raise NotImplementedError(f"a tree of {n} nodes: the kernels take up to 64")
    _need_cuda(parents, base)
    par = _rows(parents)
    stride = 0 if par.dim() == 1 else n
    if stride and par.shape != (B, n):
        par = par.expand(B, n).contiguous()
    bits = torch.empty(B, n, dtype=torch.int64, device=par.device)
    positions = None if base is None else torch.empty(B, n, dtype=torch.int64, device=par.device)
    _lib.check(_lib.lib().wpt_tree_bits(_lib.ptr(par), stride, B, n, _lib.ptr(bits), _lib.ptr(base),
                                        _lib.ptr(positions), _lib.stream(par.device)))
    LAUNCHES[0] += 1
    return bits, positions


def head_scores(h, weight, round_bf16=True):
    """(R, V) fp32 scores = h (R, D) @ weight (V, D)^T from the tcgen05 head
    kernel (model.py:267,471: the output head, bias-free; with round_bf16 each
    score is rounded to bf16 first, as the reference's autocast head returns
    it). h and weight bf16 with contiguous rows; D a multiple of 64."""
    _need_cuda(h, weight)
    if h.dtype != torch.bfloat16 or weight.dtype != torch.bfloat16:
        raise NotImplementedError("the head kernel takes bf16 hidden states and weights")
    if h.stride(-1) != 1:
        h = h.contiguous()
    if weight.stride(-1) != 1:
        weight = weight.contiguous()
    R, D = h.shape
    V = weight.shape[0]
    if weight.shape[1] != D:
        raise ValueError(f"hidden width {D} against a head weight of {tuple(weight.shape)}")
    scores = torch.empty(R, V, dtype=torch.float32, device=h.device)
    _lib.check(_lib.lib().wpt_head_scores(h.data_ptr(), h.stride(0), weight.data_ptr(), weight.stride(0), R, D, V,
                                          1 if round_bf16 else 0, scores.data_ptr(), _lib.stream(h.device)))
    LAUNCHES[0] += math.ceil(R / 128)
    return scores


def accept(scores, drafted, q, uniforms, resample, temperature=1.0, top_k=None, lengths=None):
    """The acceptance step for R rows (wpt_inference/__init__.py:173-179,
    210-222) with explicit draws: returns (tokens (R, n + 1) int64, -1
    padded: each row's kept drafts then its drawn token; accepted (R,)
    int64: the drafts each row kept)."""
    _need_cuda(scores, drafted, q, uniforms, resample, lengths)
    scores = scores.float().contiguous()
    R, n1, V = scores.shape
    n = n1 - 1
    drafted = drafted.to(torch.int64).contiguous()
    q = q.float().contiguous()
    uniforms = uniforms.float().contiguous()
    resample = resample.float().reshape(R).contiguous()
    lengths = None if lengths is None else lengths.to(torch.int64).contiguous()
    scratch = torch.empty(_lib.lib().wpt_accept_scratch_bytes(R, n, V), dtype=torch.uint8, device=scores.device)
    tokens = torch.empty(R, n + 1, dtype=torch.int64, device=scores.device)
    accepted = torch.empty(R, dtype=torch.int64, device=scores.device)
    _lib.check(_lib.lib().wpt_accept(
        _lib.ptr(scores), _lib.ptr(drafted), _lib.ptr(q), _lib.ptr(uniforms), _lib.ptr(resample), _lib.ptr(lengths),
        _lib.ptr(scratch), _lib.ptr(tokens), _lib.ptr(accepted), R, n, V, float(temperature),
        0 if top_k is None else int(top_k), _lib.stream(scores.device)))
    LAUNCHES[0] += 2
    return tokens, accepted


# ------------------------------------------- the cache between two decode steps

BEAM_MAX = 64  # beams in and out of beam_select, and of cache_reorder
_current = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)  # the raw query, where there is one


def _one_device(*tensors):
    """Raises for tensors (None aside) that are not all on one CUDA device."""
    _need_cuda(*tensors)
    on = {t.device for t in tensors if t is not None}
    raise ValueError(f"tensors on {', '.join(map(str, on))}: a call takes one device")


def _call(device, fn, args):
    """fn(*args, stream) on `device`'s current stream, whichever device is current."""
    if device.index == _current():
        rc = fn(*args, _lib.stream(device))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _lib.stream(device))
    if rc:
        _lib.check(rc)


def _row_bytes(x):
    """Bytes of one (b, n) entry of a table (B, N, ...) whose entries are contiguous, or None."""
    size = es = x.element_size()
    shape = x.shape
    if len(shape) == 3:
        return es * shape[2] if x.stride(2) == 1 or shape[2] <= 1 else None
    stride = x.stride()
    for i in range(len(shape) - 1, 1, -1):
        if shape[i] > 1 and stride[i] * es != size:
            return None
        size *= shape[i]
    return size


def attention_weights(q, k, positions, lse, scale, weights, window=0, floor=None):
    """Adds to weights (B, N) fp32, in place, the attention weight that each
    row of k (B, N, C) gets from the queries q (B, T, H, C), summed over
    queries and heads: exp(scale q.k - lse) over the rows each query reads
    (those of prefill_forward), lse (B, T, H) the forward pass's. Up to 256
    columns T * H the keys stream past the queries (one launch), above that
    the queries past the keys (two, or three where a key's columns are summed
    in several runs)."""
    device = q.device
    if not (q.is_cuda and k.device == device and positions.device == device and lse.device == device and
            weights.device == device and (floor is None or floor.device == device)):
        _one_device(q, k, positions, lse, weights, floor)
    B, T, H, C = q.shape
    N = k.shape[1]
    if k.shape != (B, N, C) or lse.shape != (B, T, H) or positions.shape != (B, T) or \
            (floor is not None and floor.shape != (B, T)):
        raise ValueError(f"queries {tuple(q.shape)} with keys {tuple(k.shape)}, lse {tuple(lse.shape)}, positions "
                         f"{tuple(positions.shape)}")
    if weights.dtype != torch.float32 or weights.shape != (B, N):
        raise ValueError(f"weights must be float32 {(B, N)}")
    if window < 0 or (B | T | H | N) >> 31:  # past the library's 32-bit arguments
        raise ValueError(f"window={window}, or a shape past 2**31: {tuple(q.shape)}, {N} keys")
    window = min(window, 2 ** 31 - 1)  # past every table
    ld, step = weights.stride()
    if (step != 1 and N > 1) or (ld < N and B > 1):
        raise ValueError("weights must have contiguous rows: they are added to in place")
    if _bf16(q).data_ptr() % 16 or not q.is_contiguous():
        q = q.clone(memory_format=torch.contiguous_format)
    k = _table(k)
    positions = _rows(positions)
    if floor is not None:
        floor = _rows(floor)
    if lse.dtype != torch.float32 or not lse.is_contiguous():
        lse = lse.float().contiguous()
    if B * T * N == 0:
        return weights
    lib = _lib.lib()
    scratch = None
    if T * H > 256:
        scratch = torch.empty(lib.wpt_attn_weights_scratch_bytes(B, T, H, N), dtype=torch.uint8, device=device)
    sb, sn, _ = k.stride()
    _call(device, lib.wpt_attn_weights,
          (q.data_ptr(), k.data_ptr(), sb, sn, positions.data_ptr(), None if floor is None else floor.data_ptr(),
           lse.data_ptr(), weights.data_ptr(), ld, None if scratch is None else scratch.data_ptr(), B, T, H, C, N, window,
           scale))
    LAUNCHES[0] += 1 if scratch is None else 2
    return weights


def cache_evict(held, weights, lengths, keep, recent=0, first=0, capacity=None):
    """The rows of held (B, N, ...) that a budget of `keep` leaves: of row
    b's lengths[b] live ones the first `first`, the last `recent` and the
    others with the largest weights (B, N) (equal weights: the lowest row), in
    their order, as new tables of `capacity` rows (default `keep`), zeros
    after them. Returns (held (B, capacity, ...), weights (B, capacity), rows
    (B, keep) int64, -1 padded: the old places, counts (B,) int64)."""
    device = held.device
    if not (held.is_cuda and weights.device == device and lengths.device == device):
        _one_device(held, weights, lengths)
    if capacity is None:
        capacity = keep
    shape = held.shape
    B, N = shape[0], shape[1]
    if weights.shape != (B, N) or weights.dtype != torch.float32 or lengths.shape != (B,):
        raise ValueError(f"a table of {B} rows of {N} needs float32 weights {(B, N)} and lengths {(B,)}; got "
                         f"{weights.dtype} {tuple(weights.shape)} and {tuple(lengths.shape)}")
    if keep < 0 or recent < 0 or first < 0 or recent + first > keep or capacity < keep:
        raise ValueError(f"keep={keep} rows cannot hold first={first} and recent={recent}, or capacity={capacity} "
                         "cannot hold them")
    es = held.element_size()
    row_bytes = _row_bytes(held)
    apart = row_bytes is None
    if apart:
        row_bytes = es * math.prod(shape[2:])
    elif es < 4:  # the kernels copy units of 4 bytes
        apart = (held.data_ptr() | es * held.stride(0) | es * held.stride(1)) % 4 != 0
    if (B | N | capacity | row_bytes) >> 31:  # past the library's 32-bit arguments
        raise NotImplementedError(f"a table of {tuple(shape)} cut to keep={keep}, capacity={capacity}: too large")
    if apart:
        held = held.contiguous()
    ld, step = weights.stride()
    if step != 1 and N > 1 or ld < N and B > 1:
        weights = weights.contiguous()
        ld = N
    lengths = _rows(lengths)
    out = held.new_empty(B, capacity, *shape[2:])
    out_weights = weights.new_empty(B, capacity)
    rows = lengths.new_empty(B, keep)
    counts = torch.empty_like(lengths)
    stride = held.stride()
    _call(device, _lib.lib().wpt_cache_evict,
          (held.data_ptr(), stride[0] * es, stride[1] * es, weights.data_ptr(), ld, lengths.data_ptr(), out.data_ptr(),
           out_weights.data_ptr(), rows.data_ptr(), counts.data_ptr(), B, N, row_bytes, keep, recent, first, capacity))
    LAUNCHES[0] += 1  # and the copy's, for more than a little
    return out, out_weights, rows, counts


def beam_select(scores, totals, beams, done=None, end=None):
    """Beam search's selection: scores (R, W, V) fp32 or bf16 logits, totals
    (R, W) the beams' running log-probabilities; the `beams` largest of
    totals + log_softmax(scores) of each text (equal values: the lowest beam,
    then token). A beam in `done` (R, W) offers itself alone, total unchanged,
    with the token `end`. Returns (totals (R, beams) fp32, best first, parents
    and tokens (R, beams) int64); -inf, -1 and -1 where there are too few
    candidates."""
    device = scores.device
    if not (scores.is_cuda and totals.device == device and (done is None or done.device == device)):
        _one_device(scores, totals, done)
    bf16 = scores.dtype == torch.bfloat16
    if not bf16 and scores.dtype != torch.float32:
        raise NotImplementedError(f"the selection kernels take float32 or bfloat16 scores; got {scores.dtype}")
    R, W, V = scores.shape
    if beams < 1 or totals.shape != (R, W) or (done is not None and done.shape != (R, W)):
        raise ValueError(f"scores {tuple(scores.shape)} need totals (and done) {(R, W)}, and {beams} beams to pick")
    if W > BEAM_MAX or beams > BEAM_MAX or (R | V) >> 31:  # V: past the library's 32-bit arguments
        raise NotImplementedError(f"{beams} beams of scores {tuple(scores.shape)}: the selection kernels take up to "
                                  f"{BEAM_MAX} beams in and out, and vocabularies under 2**31")
    if done is None:
        end = 0  # not read
    else:
        if end is None or not 0 <= end < V:
            raise ValueError(f"ended beams need the token `end` of the vocabulary; got {end} of {V}")
        if done.dtype != torch.bool or not done.is_contiguous():
            done = done.to(torch.bool).contiguous()
    sr, sw, sv = scores.stride()
    if sv != 1 and V > 1:
        scores = scores.contiguous()
        sr, sw = W * V, V
    if totals.dtype != torch.float32 or not totals.is_contiguous():
        totals = totals.float().contiguous()
    out = torch.empty_like(totals) if beams == W else totals.new_empty(R, beams)
    parents = totals.new_empty(R, beams, dtype=torch.int64)
    tokens = torch.empty_like(parents)
    lib = _lib.lib()
    scratch = parents.new_empty(lib.wpt_beam_scratch_bytes(R, W, V, beams, bf16) // 8)
    _call(device, lib.wpt_beam_select,
          (scores.data_ptr(), bf16, sr, sw, totals.data_ptr(), None if done is None else done.data_ptr(),
           end, scratch.data_ptr(), out.data_ptr(), parents.data_ptr(), tokens.data_ptr(), R, W, V,
           beams))
    LAUNCHES[0] += 2
    return out, parents, tokens


def _places_overlap(rows, sb, sn, size, N, at=None, size2=0, N2=0):
    """Whether two of a table's places (b, n), `size` bytes at b * sb + n * sn (b
    under `rows`, n under N), share a byte; given `at`, whether one does with a place of
    a table of the same strides (places of size2 bytes, n under N2) that starts there."""
    same = at is None
    if same:
        at, size2, N2 = 0, size, N
    for b in range(1 - rows, rows):  # n2 * sn - n * sn in (-size2, size) - at - b * sb, over n2 - n
        low, high = -size2 - at - b * sb, size - at - b * sb
        if sn == 0:
            if low < 0 < high and not (same and b == 0 and N == 1):
                return True
            continue
        first, last = max(1 - N, low // sn + 1), min(N2 - 1, -(-high // sn) - 1)
        if last - first + 1 > (same and b == 0 and first <= 0 <= last):  # a place may share with itself
            return True
    return False


def _tables_overlap(rows, fields):
    """Whether tables, five numbers each (first byte, sb, sn, size, N), share memory, as
    far as that is told by their extents and, where these cross, by equal strides."""
    tables = sorted(zip(*(fields[i::5] for i in range(5))))
    tables = [t for t in tables if rows * t[3] * t[4]]
    for i, (start, sb, sn, size, N) in enumerate(tables):
        end = start + (rows - 1) * sb + (N - 1) * sn + size
        for start2, sb2, sn2, size2, N2 in tables[i + 1:]:
            if start2 >= end:
                break
            at = start2 - start
            if (sb, sn) != (sb2, sn2) and (rows, N, N2) != (1, 1, 1):
                continue
            # parts of the same wider entries, as keys and values: no need to look further
            wide = at + size2
            if size <= at and (wide <= sn and (rows == 1 or sb >= (max(N, N2) - 1) * sn + wide) or
                               wide <= sb and sn >= (rows - 1) * sb + wide):
                continue
            if _places_overlap(rows, sb, sn, size, N, at, size2, N2):
                return True
    return False


REORDER_TABLES = 32  # tables wpt_cache_reorder takes in one launch


def cache_reorder(tables, parents, lengths, first=None):
    """Reorders the beams' rows of one table or a list of tables (R * W, N,
    ...) in place: beam w of text r (row r * W + w) takes the table rows
    first[r] (default 0) .. lengths[r * W + p] - 1 of beam p = parents[r, w]
    (-1: it keeps its own); those before first[r], which have to be the same
    in all beams of the text, stay. Returns `tables`. A launch for every 32 tables,
    whatever their shapes."""
    every = [tables] if isinstance(tables, torch.Tensor) else tables
    device = parents.device
    if not (parents.is_cuda and lengths.device == device and (first is None or first.device == device)):
        _one_device(parents, lengths, first)
    R, W = parents.shape
    if lengths.shape != (R * W,) or (first is not None and first.shape != (R,)):
        raise ValueError(f"parents {(R, W)} need lengths {(R * W,)} (and first {(R,)})")
    parents, lengths = _rows(parents), _rows(lengths)
    if first is not None:
        first = _rows(first)
    fields, units = [], 0
    low, high, crossed = 0, 0, False  # the addresses of the tables so far; whether one lies among them
    for t in every:
        shape = t.shape
        if t.device != device:
            _one_device(t, parents)
        if len(shape) < 2 or shape[0] != R * W:
            raise ValueError(f"a table of {tuple(shape)} for {R} texts of {W} beams")
        size, es, stride = _row_bytes(t), t.element_size(), t.stride()
        sb, sn = stride[0] * es, stride[1] * es
        N = shape[1]
        if size is None or (t.numel() and not (sn >= size and sb >= (N - 1) * sn + size) and
                            not (sb >= size and sn >= (R * W - 1) * sb + size) and
                            _places_overlap(R * W, sb, sn, size, N)):
            raise ValueError("a reordered table's entries must be contiguous and its places must not overlap: it is "
                             "changed in place")
        at = t.data_ptr()
        fields += (at, sb, sn, size, N)
        units |= at | sb | sn | size
        end = at + (R * W - 1) * sb + (N - 1) * sn + size
        if not size * N:
            continue
        if at >= high:
            high, low = end, low or at
        elif end <= low:
            low = at
        else:
            crossed = True
    if crossed and _tables_overlap(R * W, fields):
        raise ValueError("two reordered tables share memory: they are changed in place")
    if units % 4 or (fields and W > BEAM_MAX):  # before the first launch: a call that is refused moves nothing
        raise NotImplementedError("the reordering kernel takes up to 64 beams and moves units of 4 bytes: tables, strides "
                                  "and entries must be multiples of 4 bytes")
    lib = _lib.lib()
    for i in range(0, len(fields), 5 * REORDER_TABLES):
        part = fields[i:i + 5 * REORDER_TABLES]
        _call(device, lib.wpt_cache_reorder,
              ((ctypes.c_int64 * len(part))(*part), len(part) // 5, parents.data_ptr(), lengths.data_ptr(),
               None if first is None else first.data_ptr(), R, W))
        LAUNCHES[0] += 1
    return tables


# ------------------------------------- rotary positions, the 8-bit paged cache

PAGE_BLOCK = 16  # cached entries that share a scale


def _whole(x, what):
    """x (...) contiguous int64. Numbers of a type that is not whole are
    refused: cut off, they would be other positions."""
    dtype = x.dtype
    if dtype is not torch.int64:
        if dtype.is_floating_point or dtype.is_complex or dtype is torch.bool:
            raise ValueError(f"{what} must be whole numbers; got {dtype}")
        x = x.to(torch.int64)
    return x if x.is_contiguous() else x.contiguous()


def rotary_frequencies(dims, base=10000.0, scaling=None, factor=1.0, original=None, low=1.0, high=32.0, device=None):
    """(dims / 2,) float64 angles a position, base ** (-2 i / dims), for rotate
    and paged_append. For a context `factor` times as long as the `original` one:
    scaling "linear" slows every pair by the factor, "base" enlarges the base so
    that the slowest pair slows by it and the fastest stays, "parts" slows the
    pairs that turn fewer than `low` times in the original context, leaves those
    over `high` times as they are and goes linearly between."""
    if dims < 0 or dims % 2:
        raise ValueError(f"an even number of channels turns; got {dims}")
    if scaling not in (None, "linear", "base", "parts"):
        raise ValueError(f"scaling {scaling!r}: None, 'linear', 'base' or 'parts'")
    if not base > 0 or not factor > 0 or (scaling == "parts" and (original is None or not high > low)):
        raise ValueError(f"base={base}, factor={factor}, original={original}, low={low}, high={high}")
    if scaling == "base":
        base = base * factor ** (dims / max(1, dims - 2))
    f = base ** (-torch.arange(0, dims, 2, dtype=torch.float64) / max(1, dims))
    if scaling == "linear":
        f = f / factor
    elif scaling == "parts":
        keep = ((original * f / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        f = f * keep + f / factor * (1 - keep)
    return f.to(device) if device is not None else f


def _frequencies(frequencies, C, start):
    """(contiguous fp32 or fp64 frequencies, dims, the first channel that turns) of heads of C channels."""
    if frequencies is None:
        return None, 0, 0
    shape, dtype = frequencies.shape, frequencies.dtype
    if len(shape) != 1 or not dtype.is_floating_point:
        raise ValueError(f"frequencies are (dims / 2,) floating-point angles; got {dtype} {tuple(shape)}")
    if dtype is not torch.float64 and dtype is not torch.float32:
        frequencies = frequencies.float()
    if not frequencies.is_contiguous():
        frequencies = frequencies.contiguous()
    dims = 2 * shape[0]
    if start is None:
        start = C - dims
    if start < 0 or start + dims > C:
        raise ValueError(f"{dims} turned channels from {start} on do not fit in {C}")
    return frequencies, dims, start


def rotate(x, positions, frequencies, start=None, interleaved=False, magnitude=1.0, inverse=False):
    """x (B, T, C) or (B, T, H, C), bf16 or fp32, with the channels start ..
    start + dims - 1 of each head (default: the last) turned by their positions
    (T,) or (B, T) times frequencies (dims / 2,), times magnitude; inverse turns
    the other way (the gradient). A new contiguous tensor."""
    device = x.device
    if not (x.is_cuda and positions.device == device and frequencies.device == device):
        _one_device(x, positions, frequencies)
    f32 = x.dtype is torch.float32
    if not f32 and x.dtype is not torch.bfloat16:
        raise NotImplementedError(f"the rotation kernel takes bfloat16 or float32; got {x.dtype}")
    shape, at = x.shape, positions.shape
    if len(shape) == 4:
        B, T, H, C = shape
    elif len(shape) == 3:
        B, T, C = shape
        H = 1
    else:
        raise ValueError(f"x must be (B, T, C) or (B, T, H, C); got {tuple(shape)}")
    each = len(at) == 2 and at[0] == B  # each row has positions of its own
    if at[-1:] != shape[1:2] or not (each or len(at) == 1 or (len(at) == 2 and at[0] == 1)):
        raise ValueError(f"positions must be {(T,)} or {(B, T)}; got {tuple(at)}")
    if (B | T | H | C) >> 31:
        raise NotImplementedError(f"x of {tuple(shape)}: past the library's 32-bit arguments")
    frequencies, dims, start = _frequencies(frequencies, C, start)
    if positions.dtype is not torch.int64 or positions.stride(-1) != 1:
        positions = _whole(positions, "positions")
    if x.is_contiguous():
        y = torch.empty_like(x)
    else:
        if x.stride(-1) != 1:
            x = x.contiguous()
        y = x.new_empty(shape)
    if B * T * H * C == 0:
        return y
    stride = x.stride()
    _call(device, _lib.lib().wpt_rotate,
          (x.data_ptr(), stride[0], stride[1], stride[2] if len(shape) == 4 else 0, positions.data_ptr(),
           positions.stride(0) if each else 0, frequencies.data_ptr(), frequencies.dtype is torch.float64, y.data_ptr(), f32,
           B, T, H, C, dims, start, interleaved, magnitude, inverse))
    LAUNCHES[0] += 1
    return y


_PAGE_LAYOUTS = {}  # what _pages found for shapes, strides and types that it has seen


def _pages(pages, scales, table):
    """Checks a paged cache's tensors; (P, S, C, B, M)."""
    ps, pt, ss, st, ts = pages.shape, pages.stride(), scales.shape, scales.stride(), table.shape
    key = ps, pt, ss, st, ts, pages.dtype, scales.dtype, table.dtype
    found = _PAGE_LAYOUTS.get(key)
    if found is None:
        if len(_PAGE_LAYOUTS) > 4096:
            _PAGE_LAYOUTS.clear()
        found = _PAGE_LAYOUTS[key] = _page_layout(ps, pt, ss, st, ts, pages.dtype, scales.dtype, table.dtype)
    if pages.data_ptr() % 16:
        raise ValueError("pages must be 16-byte aligned")
    return found


def _page_layout(ps, pt, ss, st, ts, pages_dtype, scales_dtype, table_dtype):
    if pages_dtype != torch.float8_e4m3fn or scales_dtype != torch.float32:
        raise NotImplementedError(f"the paged cache holds float8_e4m3fn with float32 scales; got {pages_dtype} and "
                                  f"{scales_dtype}")
    if len(ps) != 3 or ps[2] % 2 or ps[1] % PAGE_BLOCK or ss != (ps[0], ps[1] // PAGE_BLOCK, 2):
        raise ValueError(f"pages {tuple(ps)} must be (P, S, 2 C), S a multiple of {PAGE_BLOCK}, with scales (P, S / "
                         f"{PAGE_BLOCK}, 2); got {tuple(ss)}")
    P, S, C2 = ps
    if S not in (16, 32, 64) and (S % 128 or S == 0):
        raise NotImplementedError(f"pages of {S} entries: 16, 32, 64 or a multiple of 128")
    if len(ts) != 2 or table_dtype not in (torch.int32, torch.int64):
        raise ValueError(f"the page table must be (B, M) int32 or int64; got {table_dtype} {tuple(ts)}")
    if P * C2 and (pt[2] != 1 or pt[1] < C2 or (P > 1 and pt[0] < (S - 1) * pt[1] + C2) or (pt[0] | pt[1]) % 16):
        raise ValueError("pages must have contiguous entries, 16-byte aligned, and pages that do not overlap")
    if P and (st[2] != 1 or (st[1] != 2 and S > PAGE_BLOCK) or (P > 1 and st[0] < S // PAGE_BLOCK * 2)):
        raise ValueError("scales must be contiguous within a page")
    if (P | S | ts[1] | ts[1] * S) >> 31:
        raise NotImplementedError(f"{P} pages of {S} entries, {ts[1]} a row: past the library's 32-bit arguments")
    return P, S, C2 // 2, ts[0], ts[1]


def _table_rows(table):
    return table if table.shape[1] < 2 or table.stride(1) == 1 else table.contiguous()


def paged_cache(pages, page, width, device=None):
    """An empty paged cache for entries of `width` channels (a key, then a
    value, 2 * width): pages (pages, page, 2 * width) float8_e4m3fn and scales
    (pages, page / 16, 2) float32, zeros."""
    if page not in (16, 32, 64) and (page < 128 or page % 128):
        raise NotImplementedError(f"pages of {page} entries: 16, 32, 64 or a multiple of 128")
    if width < 16 or width % 16 or width > 512:
        raise NotImplementedError(f"entries of 2 x {width}: the paged cache takes multiples of 16 up to 512")
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else device
    return (torch.zeros(pages, page, 2 * width, dtype=torch.float8_e4m3fn, device=device),
            torch.zeros(pages, page // PAGE_BLOCK, 2, device=device))


def paged_append(pages, scales, table, new, first, counts, frequencies=None, positions=None, start=None,
                 interleaved=False, magnitude=1.0):
    """Writes new (B, n, 2 C), bf16 or fp32, to the paged cache, in place: row
    b's entries new[b, :counts[b]] become its entries first[b] .., entry i on
    page table[b, i // S]. With frequencies, keys are turned on the way, as
    rotate does, by positions (B, n) (default: their places first[b] + i). A
    block's scales become the least powers of two that hold its values; where it
    holds earlier entries of the row, not less than they were, and those are
    rounded again where a scale grows. What follows the new entries in their last
    block keeps its bytes, not its scale. Places outside the table or on no page
    (-1) are not written and set the status word's shape bit (with no page at all
    nothing is launched and it is not set)."""
    device = pages.device
    if not (pages.is_cuda and scales.device == device and table.device == device and new.device == device and
            first.device == device and counts.device == device and
            (frequencies is None or frequencies.device == device) and (positions is None or positions.device == device)):
        _one_device(pages, scales, table, new, first, counts, frequencies, positions)
    P, S, C, B, M = _pages(pages, scales, table)
    f32 = new.dtype is torch.float32
    if not f32 and new.dtype is not torch.bfloat16:
        raise NotImplementedError(f"the append kernel takes bfloat16 or float32 entries; got {new.dtype}")
    shape = new.shape
    if len(shape) != 3 or shape[0] != B or shape[2] != 2 * C or first.shape != (B,) or counts.shape != (B,):
        raise ValueError(f"entries {tuple(shape)} for a table of {B} rows and pages of 2 x {C}, with first "
                         f"{tuple(first.shape)} and counts {tuple(counts.shape)}")
    n = shape[1]
    if positions is not None and positions.shape != (B, n):
        raise ValueError(f"positions must be {(B, n)}; got {tuple(positions.shape)}")
    if (B | n) >> 31:
        raise NotImplementedError(f"entries {tuple(new.shape)}: past the library's 32-bit arguments")
    frequencies, dims, start = _frequencies(frequencies, C, start)
    first, counts = _whole(first, "first"), _whole(counts, "counts")
    positions = None if positions is None else _whole(positions, "positions")
    table = _table_rows(table)
    if new.stride(2) != 1:
        new = new.contiguous()
    if B * n * P * M == 0:
        return pages, scales
    ns, ps = new.stride(), pages.stride()
    _call(device, _lib.lib().wpt_paged_append,
          (new.data_ptr(), f32, ns[0], ns[1], pages.data_ptr(), ps[0], ps[1], scales.data_ptr(), scales.stride(0),
           table.data_ptr(), table.dtype is torch.int64, table.stride(0), first.data_ptr(), counts.data_ptr(),
           None if positions is None else positions.data_ptr(), None if frequencies is None else frequencies.data_ptr(),
           frequencies is not None and frequencies.dtype is torch.float64, B, n, C, M, P, S, dims, start, interleaved,
           magnitude))
    LAUNCHES[0] += 1
    return pages, scales


def _paged_plan(B, T, H, N, window, sms):
    """(splits, ctas) of a paged attention call over rows of up to N entries,
    remembered per shape."""
    key = ("paged", B, T, H, N, window, sms)
    plan = _PLAN_CACHE.get(key)
    if plan is None:
        if len(_PLAN_CACHE) > 4096:
            _PLAN_CACHE.clear()
        plan = _PLAN_CACHE[key] = _paged_plan_for(B, T, H, N, window, sms)
    return plan


def _paged_scratch(B, T, H, ctas):
    """The scratch of a balanced call in bf16 elements, remembered per shape."""
    key = ("paged scratch", B, T, H, ctas)
    size = _PLAN_CACHE.get(key)
    if size is None:
        size = _PLAN_CACHE[key] = (_lib.lib().wpt_paged_scratch_bytes(B, T, H, 0, ctas) + 1) // 2
    return size


def _paged_plan_for(B, T, H, N, window, sms):
    ncol = 16 if T * H <= 16 else 32
    chunks = math.ceil(H / 32)  # groups that a query's heads take
    TQ = max(1, ncol // H)
    groups = B * math.ceil(T / TQ) * chunks
    tiles = max(1, math.ceil(N / 128))
    if window:  # what neighbouring queries reach
        tiles = min(tiles, (window + TQ - 2) // 128 + 2)
    slots = 2 * sms  # CTAs at a time
    # Few tiles a CTA: one launch, a group's tiles over a cluster. A cluster's CTAs share a GPC (on B200 8 of 16 to 20
    # SMs), and more clusters than fit run in two waves: past two CTAs, 7/8 of the slots (33 clusters of 8 11.6 us, 34
    # 19.0; 44 of 6 11.7, 46 20.1). Rows of uneven lengths wait for the longest there; balanced, all CTAs end together,
    # but parts are written and merged in a second launch. Equal and ragged lengths (1/32 to all), us, cluster then
    # balanced: 16 rows of 4,096 12.3, 12.4 and 11.5, 11.7, of 8,192 15.6, 14.0 and 14.5, 12.5; where clusters fill the
    # SMs, 64 rows of 4,096 16.0, 19.6 and 15.3, 16.7, of 8,192 29.9, 33.8 and 22.7, 21.1.
    splits = next(s for s in range(min(8, tiles), 0, -1) if s == 1 or groups * s <= (slots if s == 2 else slots * 7 // 8))
    if tiles <= (10 if groups * splits > slots * 3 // 4 else 4) * splits:
        return splits, 1
    if groups <= 256 and groups * (math.ceil(N / 128) + 8) < 2 ** 31:
        return 0, min(slots, groups * tiles)
    return 1, 1  # more groups than CTAs at a time


def paged_attention(q, pages, scales, table, positions, scale, window=0, sink=None):
    """Attention of q (B, T, H, 128) bf16 over each row's entries 0 ..
    positions (B, T) of the paged cache (its last `window` ones, given a
    window), sink (H,) in the denominators: (out (B, T, H, 128) bf16, lse
    (B, T, H) fp32). Entries on no page (-1) are not read; a query without
    entries gives 0 and -inf (or its sink)."""
    device = q.device
    if not (q.is_cuda and pages.device == device and scales.device == device and table.device == device and
            positions.device == device and (sink is None or sink.device == device)):
        _one_device(q, pages, scales, table, positions, sink)
    P, S, C, rows, M = _pages(pages, scales, table)
    _bf16(q)
    shape, at = q.shape, positions.shape
    if len(shape) != 4 or shape[3] != C or rows != shape[0] or at[-1:] != shape[1:2] or \
            not (len(at) == 1 or len(at) == 2 and at[0] in (1, rows)):
        raise ValueError(f"queries {tuple(shape)} with pages of 2 x {C}, a table of {rows} rows and positions {tuple(at)}")
    B, T, H, _ = shape
    if sink is not None and sink.shape != (H,):
        raise ValueError(f"sink must be {(H,)}; got {tuple(sink.shape)}")
    if window < 0 or (B | T) >> 31:
        raise ValueError(f"window={window}, or a shape past 2**31: {tuple(q.shape)}")
    if C != 128 or H > 64:
        raise NotImplementedError(f"{H} heads of width {C}: the paged attention kernel takes head width 128 and up to 64 "
                                  "heads")
    window = min(window, 2 ** 31 - 1)  # past every table
    if not q.is_contiguous() or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)
    positions = _whole(positions if len(at) == 2 and at[0] == B else positions.expand(B, -1), "positions")
    table = _table_rows(table)
    if sink is not None and (sink.dtype is not torch.float32 or not sink.is_contiguous()):
        sink = sink.float().contiguous()
    out = torch.empty_like(q)
    lse = q.new_empty((B, T, H), dtype=torch.float32)
    if B * T * H == 0:
        return out, lse
    splits, ctas = _paged_plan(B, T, H, M * S, window, sm_count(device))
    lib = _lib.lib()
    scratch = None
    if splits == 0:
        scratch = q.new_empty(_paged_scratch(B, T, H, ctas))
    ps = pages.stride()
    _call(device, lib.wpt_paged_attention,
          (q.data_ptr(), pages.data_ptr(), ps[0], ps[1], scales.data_ptr(), scales.stride(0), table.data_ptr(),
           table.dtype is torch.int64, table.stride(0), positions.data_ptr(), None if sink is None else sink.data_ptr(),
           out.data_ptr(), lse.data_ptr(), None if scratch is None else scratch.data_ptr(), splits, ctas, B, T, H, C, M, P,
           S, window, scale))
    LAUNCHES[0] += 1 + (scratch is not None)
    return out, lse
