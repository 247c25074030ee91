"""Plain 64-bit restatements of the operators around the cache (rotary
positions, block-scaled pools, eviction, logits), from their formulas; numpy on
the host."""
from __future__ import annotations

import math

import numpy as np
import torch

BS = 16


# ---- rotary positions ----------------------------------------------------------------

def rope(x, positions, inv_freq, interleaved, magnitude=1.0):
    """x [T, H, D] -> float64 [T, H, D]."""
    y = x.astype(np.float64).copy()
    n = len(inv_freq)
    a = np.outer(positions.astype(np.longdouble), inv_freq.astype(np.longdouble))
    c, s = np.cos(a).astype(np.float64) * magnitude, np.sin(a).astype(np.float64) * magnitude
    first = np.arange(n) * 2 if interleaved else np.arange(n)
    second = first + (1 if interleaved else n)
    x0, x1 = y[..., first].copy(), y[..., second].copy()
    y[..., first] = x0 * c[:, None] - x1 * s[:, None]
    y[..., second] = x1 * c[:, None] + x0 * s[:, None]
    return y


def rope_bound(x, positions, inv_freq, interleaved, magnitude=1.0):
    """What 32-bit arithmetic may be off by, element by element: a fraction of a
    turn rounded to 24 bits (2^-26 turns, 2^-23 rad), sines within 2 ulp (2^-22)
    and their product with the magnitude (2^-24), on either element of the pair,
    then two roundings of the sum; and the angle's own 64-bit rounding."""
    b = np.zeros(x.shape)
    n = len(inv_freq)
    first = np.arange(n) * 2 if interleaved else np.arange(n)
    second = first + (1 if interleaved else n)
    size = (np.abs(x[..., first]) + np.abs(x[..., second])).astype(np.float64) * abs(magnitude)
    off = 2.0 ** -20.5 + np.abs(np.outer(positions, inv_freq)) * 2.0 ** -50
    b[..., first] = b[..., second] = size * off[:, None]
    return b


# ---- 8-bit pools with one scale a tile ---------------------------------------------------

def e4m3(x):
    """float64 -> the e4m3 byte nearest (ties to even), saturating at 448."""
    t = torch.from_numpy(np.clip(np.asarray(x, np.float64), -448, 448))
    # 64 -> 32 bits is exact for what the tests hand in (quotients by powers of two)
    return t.float().to(torch.float8_e4m3fn).view(torch.uint8).numpy()


def byte_values(b, fmt):
    if fmt.startswith("int8"):
        return b.view(np.int8).astype(np.float64)
    return torch.from_numpy(b.copy()).view(torch.float8_e4m3fn).float().numpy().astype(np.float64)


def tile_scale(amax, fmt):
    if amax < 2.0 ** -110:
        return np.float32(0)
    if fmt == "int8_block":
        return np.float32(amax) * (np.float32(1) / np.float32(127))
    s = 2.0 ** math.ceil(math.log2(float(amax) / 448.0))
    while float(amax) / s > 448:   # log2's rounding
        s *= 2
    while float(amax) / (s / 2) <= 448:
        s /= 2
    return np.float32(s)


def tile_bytes(x, s, fmt):
    """Bytes of x (float64) under scale s."""
    x = np.asarray(x, np.float64)
    if s == 0:
        y = np.zeros(x.shape, np.uint8)
    elif fmt == "int8_block":
        with np.errstate(invalid="ignore"):
            y = np.clip(np.rint(np.nan_to_num(x / np.float64(s), nan=0.0, posinf=127, neginf=-127)),
                        -127, 127).astype(np.int8).view(np.uint8)
    else:
        y = e4m3(x / np.float64(s))
    if fmt == "fp8_block":
        y = np.where(np.isnan(x), (y & 0x80) | 0x7f, y).astype(np.uint8)
    return y


def append_block(pool, scale, new, start, tables, ctx, fmt, max_new=None):
    """One layer's pool and scales, in place."""
    nb, hkv, _, d = pool.shape
    for b in range(len(ctx)):
        n = int(start[b + 1] - start[b])
        pos0 = int(ctx[b]) - n
        take = n if max_new is None else min(n, max_new)
        first, end = max(pos0, 0), pos0 + take
        for j in range(first // BS, -(-end // BS) if end > first else first // BS):
            if j >= tables.shape[1] or not 0 <= tables[b, j] < nb:
                continue
            blk, lo, hi = tables[b, j], max(first, j * BS), min(end, (j + 1) * BS)
            if lo >= hi:
                continue
            rows = new[int(start[b]) + lo - pos0:int(start[b]) + hi - pos0]
            for h in range(hkv):
                x = rows[:, h].astype(np.float64)
                fin = np.abs(x[np.isfinite(x)])
                r0 = lo - j * BS
                old = scale[blk, h] if r0 else np.float32(0)
                s = max(old, tile_scale(fin.max() if fin.size else 0.0, fmt))
                if r0 and s > old:
                    pool[blk, h, :r0] = tile_bytes(
                        byte_values(pool[blk, h, :r0], fmt) * np.float64(old), s, fmt)
                pool[blk, h, r0:r0 + hi - lo] = tile_bytes(x, s, fmt)
                scale[blk, h] = s


def dequantize(pool, scale, fmt):
    wide = scale[..., None, None] if fmt.endswith("block") else scale[..., None]
    return byte_values(pool, fmt) * wide.astype(np.float64)


# ---- attention -----------------------------------------------------------------------------

def rows_of(pool, tables, b, length):
    """Positions 0 .. length - 1 of sequence b (float64 [length, hkv, d]) and which
    of them have a valid block."""
    pos = np.arange(length)
    blk = tables[b, pos // BS].astype(np.int64)
    ok = (blk >= 0) & (blk < pool.shape[0])
    return pool[np.where(ok, blk, 0), :, pos % BS].astype(np.float64), ok


def attend(q, k, v, tables, ctx, scale, n_new=None, start=None):
    """Attention of every query row over its sequence's cache (float64 pools):
    out [rows, hq, d], the weights per sequence [hkv, length], and bounds of the
    error of a kernel that splits q and the weights into two bf16 parts: the
    parts leave 2^-16 of each q element, so a score is off by at most delta =
    2^-16 scale sum |q k| (2^-15 with what fp32 sums of 128 products add), every
    weight by a factor e^(2 delta), an output by 2 delta max |v|, and 2^-15
    max |v| for the weights' own parts and the sums."""
    hq, d = q.shape[1:]
    hkv = k.shape[1]
    g = hq // hkv
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    weights, wbound = [], []
    for b in range(len(ctx)):
        n = 1 if n_new is None else int(n_new[b])
        r0 = b if start is None else int(start[b])
        length = max(0, int(ctx[b]))
        w, wb = np.zeros((hkv, length)), np.zeros((hkv, length))
        if length and n:
            K, ok = rows_of(k, tables, b, length)
            V, _ = rows_of(v, tables, b, length)
            last = int(ctx[b]) - n + np.arange(n)
            seen = (np.arange(length)[None] <= last[:, None]) & ok
            for h in range(hq):
                x = q[r0:r0 + n, h].astype(np.float64)
                kk, vv = np.where(ok[:, None], K[:, h // g], 0), np.where(ok[:, None], V[:, h // g], 0)
                s = np.where(seen, x @ kk.T * scale, -np.inf)
                top = s.max(1, keepdims=True)
                e = np.where(seen, np.exp(s - np.where(np.isfinite(top), top, 0)), 0)
                l = e.sum(1, keepdims=True)
                p = np.where(l > 0, e / np.where(l > 0, l, 1), 0)
                out[r0:r0 + n, h] = p @ vv
                delta = 2.0 ** -15 * scale * (np.abs(x) @ np.abs(kk).T * seen).max(1, keepdims=True)
                bound[r0:r0 + n, h] = (2 * delta + 2.0 ** -15) * np.abs(vv).max()
                w[h // g] += p.sum(0)
                wb[h // g] += (p * (2 * delta + 2.0 ** -18)).sum(0)
        weights.append(w)
        wbound.append(wb)
    return out, bound, weights, wbound


def assert_within(got, want, bound, what=""):
    diff = np.abs(np.asarray(got, np.float64) - want)
    bad = ~(diff <= bound)
    if bad.any():
        i = np.unravel_index(np.argmax(np.where(bad, diff / np.maximum(bound, 1e-300), 0)), diff.shape)
        raise AssertionError(f"{what}: at {i}: got {np.asarray(got)[i]} want {want[i]}, off by "
                             f"{diff[i]:.3e}, bound {bound[i]:.3e}; {int(bad.sum())} of {bad.size}")


# ---- eviction ---------------------------------------------------------------------------------

def select(weights, tables, ctx, budget, sinks, recent, cap=None):
    """keep [B, hkv, budget], new_lens [B] for one layer's sums [nb, hkv, 16]."""
    nb, hkv, _ = weights.shape
    B = len(ctx)
    keep = np.full((B, hkv, budget), -1, np.int32)
    lens = np.zeros(B, np.int32)
    most = tables.shape[1] * BS if cap is None else min(cap, tables.shape[1] * BS)
    for b in range(B):
        length = min(max(int(ctx[b]), 0), most)
        pos = np.arange(length)
        blk = tables[b, pos // BS].astype(np.int64)
        ok = (blk >= 0) & (blk < nb)
        lens[b] = min(budget, int(ok.sum()))
        for h in range(hkv):
            def rank(p):
                w = weights[blk[p], h, p % BS]
                held = p < sinks or p >= length - recent
                return (not held, np.isnan(w), -float(w) if not np.isnan(w) else 0.0, p)
            chosen = sorted((int(p) for p in pos[ok]), key=rank)[:budget]
            keep[b, h, :len(chosen)] = sorted(chosen)
    return keep, lens


def compact(k, v, ks, vs, weights, keep, lens, src, dst, fmt):
    """One layer, in place; k / v in their storage type."""
    nb, hkv = k.shape[:2]
    for b in range(len(lens)):
        for h in range(hkv):
            for j in range(-(-int(lens[b]) // BS)):
                if j >= dst.shape[1] or not 0 <= dst[b, j] < nb:
                    continue
                to = dst[b, j]
                rows = []
                for r in range(BS):
                    i = j * BS + r
                    p = int(keep[b, h, i]) if i < lens[b] else -1
                    if 0 <= p < src.shape[1] * BS and 0 <= src[b, p // BS] < nb:
                        rows.append((r, src[b, p // BS], p % BS))
                if weights is not None:
                    for r, blk, at in rows:
                        weights[to, h, r] = weights[blk, h, at]
                for pool, scale in ((k, ks), (v, vs)):
                    if fmt is not None and fmt.endswith("block"):
                        if not rows:
                            continue
                        s = max(scale[blk, h] for _, blk, _ in rows)
                        for r, blk, at in rows:
                            x = pool[blk, h, at]
                            pool[to, h, r] = x if scale[blk, h] == s else tile_bytes(
                                byte_values(x, fmt) * np.float64(scale[blk, h]), s, fmt)
                        scale[to, h] = s
                        continue
                    for r, blk, at in rows:
                        pool[to, h, r] = pool[blk, h, at]
                        if scale is not None:
                            scale[to, h, r] = scale[blk, h, at]


# ---- logits -----------------------------------------------------------------------------------

def logits(x, history=None, start=None, prompt=None, repetition=None, frequency=None,
           presence=None, bias_ids=None, bias=None, bias_start=None, allowed=None):
    """Processed rows (float64), picks, and a bound of fp32's error: four
    roundings of 2^-24 on the terms' sizes."""
    rows, n = x.shape
    y, size = x.astype(np.float64).copy(), np.abs(x).astype(np.float64)
    picks = np.full(rows, -1, np.int32)
    penal = repetition is not None or frequency is not None or presence is not None
    for r in range(rows):
        if penal:
            ids = history[start[r]:start[r + 1]]
            made = ids[int(prompt[r]) if prompt is not None else 0:]
            rep = 1.0 if repetition is None else float(repetition[r])
            f = 0.0 if frequency is None else float(frequency[r])
            p = 0.0 if presence is None else float(presence[r])
            for t in set(int(t) for t in ids if 0 <= t < n):
                y[r, t] = y[r, t] / rep if y[r, t] > 0 else y[r, t] * rep
                size[r, t] = max(size[r, t], abs(y[r, t]))
                c = int((made == t).sum())
                if c:
                    y[r, t] -= f * c + p
                    size[r, t] += abs(f) * c + abs(p)
        if bias_ids is not None:
            last = {int(t): float(z) for t, z in zip(bias_ids[bias_start[r]:bias_start[r + 1]],
                                                     bias[bias_start[r]:bias_start[r + 1]])}
            for t, z in last.items():
                if 0 <= t < n:
                    y[r, t] += z
                    size[r, t] += abs(z)
        if allowed is not None:
            bits = (allowed[r].view(np.uint32)[np.arange(n) // 32] >> (np.arange(n) % 32)) & 1
            y[r, bits == 0] = -np.inf
        z = np.where(np.isnan(y[r]), -np.inf, y[r])
        if z.max() > -np.inf:
            picks[r] = np.nonzero(z == z.max())[0][-1]
    return y, picks, size * 2.0 ** -22
