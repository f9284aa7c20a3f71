"""Float64 restatements of rotary positions and of the paged cache held in 8
bits (its append and the attention that reads it), for the tests of
wpt_b200.rotate, paged_append and paged_attention. The cache is a dict of
numpy arrays: "values" (P, S, 2 C), what the entries' e4m3 numbers are, and
"scales" (P, S // 16, 2)."""

import numpy as np

BLOCK = 16
TOP = 448.0


def e4m3_values():
    """The finite non-negative e4m3 numbers, in order."""
    out = [m * 2.0 ** -9 for m in range(8)]
    for e in range(1, 16):
        out += [(1 + m / 8) * 2.0 ** (e - 7) for m in range(8) if (e, m) != (15, 7)]
    return np.array(out)


_E4M3 = e4m3_values()


def to_e4m3(x):
    """Nearest e4m3 numbers (ties to the even one), NaN where x is; |x| <= 448."""
    x = np.asarray(x, np.float64)
    a = np.abs(x)
    hi = np.clip(np.searchsorted(_E4M3, a), 1, len(_E4M3) - 1)
    lo = hi - 1
    mid = (_E4M3[lo] + _E4M3[hi]) / 2
    pick = np.where((a > mid) | ((a == mid) & (hi % 2 == 0)), hi, lo)
    return np.where(np.isnan(x), np.nan, np.sign(x) * _E4M3[pick])


def rotate(x, positions, frequencies, start=None, interleaved=False, magnitude=1.0, inverse=False):
    """x (..., C) with positions of x.shape[:-1] (or broadcast to it): the pairs of its channels start ..
    start + 2 len(frequencies) - 1 (default: the last) as complex numbers times exp(i position frequency)."""
    y = np.array(x, np.float64)
    f = np.asarray(frequencies, np.float64)
    dims = 2 * len(f)
    start = y.shape[-1] - dims if start is None else start
    part = y[..., start:start + dims].copy()
    # angles modulo a turn in extended precision, as far positions need
    angle = np.mod(np.asarray(positions)[..., None].astype(np.longdouble) * f.astype(np.longdouble),
                   2 * np.pi * np.longdouble(1))
    turn = magnitude * np.exp(1j * (-1 if inverse else 1) * angle.astype(np.float64))
    if interleaved:
        z = (part[..., 0::2] + 1j * part[..., 1::2]) * turn
        part[..., 0::2], part[..., 1::2] = z.real, z.imag
    else:
        z = (part[..., :dims // 2] + 1j * part[..., dims // 2:]) * turn
        part = np.concatenate((z.real, z.imag), -1)
    y[..., start:start + dims] = part
    return y


def least_scale(amax):
    """The least power of two s, 2^-60 at least, with amax <= 448 s."""
    s = 2.0 ** -60
    while amax > TOP * s:
        s *= 2
    return s


def append(cache, table, new, first, counts, frequencies=None, positions=None, start=None, interleaved=False,
           magnitude=1.0):
    """The cache after appending, an entry and a block at a time, and the exact values of the entries written, in
    units of their block's scale, by (page, place)."""
    values, scales = cache["values"].copy(), cache["scales"].copy()
    P, S, C2 = values.shape
    C, M = C2 // 2, table.shape[1]
    exact = {}
    for b in range(len(first)):
        x = np.array(new[b, :max(0, min(counts[b], new.shape[1]))], np.float64)
        if frequencies is not None and len(x):
            pos = first[b] + np.arange(len(x)) if positions is None else positions[b, :len(x)]
            x[:, :C] = rotate(x[:, :C], pos, frequencies, start, interleaved, magnitude)
        x[np.abs(x) > TOP * 2.0 ** 60] = np.nan  # infinities too
        at = first[b] + np.arange(len(x))
        for block in sorted({n // BLOCK for n in at if 0 <= n < M * S}):
            page = table[b, block * BLOCK // S]
            if not 0 <= page < P:
                continue
            place, k = block * BLOCK % S, block % (S // BLOCK)
            mine = [i for i, n in enumerate(at) if n // BLOCK == block and n >= 0]
            older = max(0, max(first[b], 0) - block * BLOCK)
            for half in range(2):
                cols = slice(half * C, (half + 1) * C)
                part = x[mine][:, cols]
                finite = np.abs(part[np.isfinite(part)])
                s = least_scale(finite.max() if finite.size else 0.0)
                if older and scales[page, k, half] >= s:
                    s = scales[page, k, half]
                elif older:
                    old = values[page, place:place + older, cols] * (scales[page, k, half] / s)
                    values[page, place:place + older, cols] = to_e4m3(old)
                scales[page, k, half] = s
                for i in mine:
                    to = at[i] % S
                    exact.setdefault((page, to), np.zeros(C2))[cols] = x[i, cols] / s
                    values[page, to, cols] = to_e4m3(x[i, cols] / s)
    return dict(values=values, scales=scales), exact


def attention(q, cache, table, positions, scale, window=0, sink=None):
    """(out, lse) of q (B, T, H, C) over each row's entries 0 .. position, its last `window` ones given a window;
    entries on no page are not read. Only entries that are read are looked at."""
    B, T, H, C = q.shape
    values, scales = cache["values"], cache["scales"]
    P, S, _ = values.shape
    out, lse = np.zeros(q.shape), np.full((B, T, H), -np.inf)
    for b in range(B):
        for t in range(T):
            p = min(positions[b, t], table.shape[1] * S - 1)
            low = max(0, positions[b, t] - window + 1) if window else 0
            n = np.arange(low, p + 1)
            page = table[b, n // S] if len(n) else n
            n, page = n[(page >= 0) & (page < P)], page[(page >= 0) & (page < P)]
            e = values[page, n % S] * np.repeat(scales[page, n % S // BLOCK], C, -1)
            z = np.float64(scale) * (q[b, t].astype(np.float64) @ e[:, :C].T)
            if sink is not None:
                z = np.concatenate((z, np.asarray(sink, np.float64)[:, None]), 1)
            if not z.shape[1]:
                continue
            top = z.max(1, keepdims=True)
            top = np.where(np.isneginf(top), 0.0, top)
            w = np.exp(z - top)
            total = w.sum(1, keepdims=True)
            with np.errstate(divide="ignore"):
                lse[b, t] = (top + np.log(total))[:, 0]
            out[b, t] = (w[:, :len(n)] / np.where(total == 0, 1.0, total)) @ e[:, C:]
    return out, lse
