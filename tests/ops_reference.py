"""Plain restatements (numpy, 64 bits) of the operators of gemma_b200.ops, for their tests.

Written from the definitions in include/gemma_b200.h: loops over requests, blocks and rows, no code
shared with the kernels.
"""
import math

import numpy as np

MIN_EXP = -60
TOP = {"int8": 127.0, "e4m3": 448.0}


def blocks_of(n, B):
    return -(-n // B)


def plan(old, new, table, free, count, B, rows):
    """(outputs dict, table, free) after gg_plan_blocks; Python integers throughout."""
    table, free = table.copy(), free.copy()
    n, width = table.shape
    status = 0
    give = sum(max(0, blocks_of(a, B) - blocks_of(b, B)) for a, b in zip(old, new))
    take = sum(max(0, blocks_of(b, B) - blocks_of(a, B)) for a, b in zip(old, new))
    total = sum(max(0, b - a) for a, b in zip(old, new))
    if any(a < 0 or b < 0 or blocks_of(a, B) > width for a, b in zip(old, new)):
        status |= 8
    if any(blocks_of(b, B) > width for b in new):
        status |= 2
    if total > rows:
        status |= 4
    if not 0 <= count <= len(free) or count + give > len(free):
        status |= 16
    elif take > count + give:
        status |= 1
    out = dict(row_seq=np.full(rows, -1), positions=np.full(rows, -1), slots=np.full(rows, -1), status=status)
    if status:
        return dict(out, cu_rows=np.zeros(n + 1, int), lens=np.array(old), free_count=count), table, free
    top = count
    for i in range(n):
        for b in range(blocks_of(new[i], B), blocks_of(old[i], B)):
            free[top] = table[i, b]
            top += 1
    for i in range(n):
        for b in range(blocks_of(old[i], B), blocks_of(new[i], B)):
            top -= 1
            table[i, b] = free[top]
    cu, r = [0], 0
    for i in range(n):
        for p in range(old[i], new[i]):
            out["row_seq"][r], out["positions"][r], out["slots"][r] = i, p, table[i, p // B] * B + p % B
            r += 1
        cu.append(r)
    return dict(out, cu_rows=np.array(cu), lens=np.array(new), free_count=top), table, free


def rope(x, positions, freqs, layout, mscale, inverse):
    """x [rows][heads][dim] in float64."""
    y = x.astype(np.float64).copy()
    h = len(freqs)
    for r, p in enumerate(positions):
        if p < 0:
            continue
        ang = np.float64(p) * freqs
        c, s = mscale * np.cos(ang), mscale * np.sin(ang) * (-1 if inverse else 1)
        a, b = (y[r, :, :h].copy(), y[r, :, h:2 * h].copy()) if layout == "half" else (y[r, :, 0:2 * h:2].copy(), y[r, :, 1:2 * h:2].copy())
        u, v = a * c - b * s, b * c + a * s
        if layout == "half":
            y[r, :, :h], y[r, :, h:2 * h] = u, v
        else:
            y[r, :, 0:2 * h:2], y[r, :, 1:2 * h:2] = u, v
    return y


def e4m3_values():
    """Value of each of the 256 codes (NaN for 0x7f and 0xff)."""
    v = np.empty(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        x = m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
        v[c] = math.nan if c & 127 == 127 else (-x if c & 128 else x)
    return v


E4M3 = e4m3_values()


def decode(codes, code):
    """Raw bytes (uint8) -> values in float64."""
    return codes.astype(np.uint8).view(np.int8).astype(np.float64) if code == "int8" else E4M3[codes.astype(np.uint8)]


def encode(x, code):
    """Values within the code's range -> raw bytes, to nearest, ties to even."""
    if code == "int8":
        return np.rint(x).astype(np.int8).view(np.uint8)
    a = np.abs(x)
    step = 2.0 ** (np.floor(np.log2(np.maximum(a, 2.0 ** -6))) - 3)
    a = np.rint(a / step) * step
    pos = E4M3[:127]  # ascending
    return (np.searchsorted(pos, a).astype(np.uint8) | np.where(np.signbit(x), 128, 0).astype(np.uint8)).astype(np.uint8)


def exponent(amax, code):
    if amax == 0:
        return MIN_EXP
    e = math.floor(math.log2(amax / TOP[code])) - 1
    while amax > TOP[code] * 2.0 ** e:
        e += 1
    return max(e, MIN_EXP)


def append(codes, scale, x, slots, code):
    """In place on codes [blocks][heads][tokens][dim] (uint8) and scale [blocks][heads] (float64)."""
    nb, H, B, D = codes.shape
    r = 0
    while r < len(slots):
        s = slots[r]
        if not 0 <= s < nb * B:
            r += 1
            continue
        blk, m = s // B, 1
        while r + m < len(slots) and 0 <= slots[r + m] < nb * B and slots[r + m] // B == blk:
            m += 1
        last = {slots[r + j] % B: r + j for j in range(m)}
        first = min(last)
        for h in range(H):
            rows = {o: x[i, h].astype(np.float64) for o, i in last.items()}
            amax = max(np.max(np.abs(v)) if np.all(np.isfinite(v)) else math.inf for v in rows.values())
            old = scale[blk, h]
            if not math.isfinite(amax) or (first > 0 and not math.isfinite(old)):
                scale[blk, h] = math.nan
                for o in rows:
                    codes[blk, h, o] = 0
                continue
            e = exponent(amax, code)
            if first > 0:
                before = int(math.log2(old))
                if e > before:
                    codes[blk, h, :first] = encode(decode(codes[blk, h, :first], code) * 2.0 ** (before - e), code)
                e = max(e, before)
            scale[blk, h] = 2.0 ** e
            for o, v in rows.items():
                codes[blk, h, o] = encode(v * 2.0 ** -e, code)
        r += m


def attend(q, cu, lens, table, kv, B, scale, window, max_rows, max_len, xp=np):
    """(out, lse, pv, smax, least) in float64, the last three for error bounds: pv = sum_j p_j |v_j|,
    smax = max_j scale sum_d |q_d k_d|, least = max_j (p_j vs_j) sum_j |code_j|. kv(h, row, keys) ->
    k, v [keys][dim] and v's scales [keys] of key head h. Rows outside the batch stay NaN."""
    rows, heads, D = q.shape
    out, lse = np.full((rows, heads, D), np.nan), np.full((rows, heads), np.nan)
    pv, smax, least = np.zeros((rows, heads, D)), np.zeros((rows, heads)), np.zeros((rows, heads, D))
    H = kv.heads
    G = heads // H
    for i in range(len(lens)):
        n, keep = cu[i + 1] - cu[i], min(lens[i], max_len)
        for r in range(min(n, max_rows)):
            row = cu[i] + r
            if row >= rows:
                break
            p = lens[i] - n + r
            lo, hi = (max(0, p - window + 1) if window else 0), min(p, keep - 1)
            keys = np.array([j for j in range(lo, hi + 1) if 0 <= table[i, j // B] < kv.blocks], dtype=np.int64)
            for h in range(heads):
                if not len(keys):
                    out[row, h], lse[row, h] = 0, -math.inf
                    continue
                k, v, vs = kv(h // G, table[i], keys)
                z = k @ q[row, h] * scale
                m = z.max()
                w = np.exp(z - m)
                out[row, h] = w @ v / w.sum()
                lse[row, h] = m + math.log(w.sum())
                pv[row, h] = w @ np.abs(v) / w.sum()
                least[row, h] = (w * vs).max() / w.sum() * (np.abs(v) / vs[:, None]).sum(0)
                smax[row, h] = (np.abs(k) @ np.abs(q[row, h])).max() * abs(scale)
    return out, lse, pv, smax, least
