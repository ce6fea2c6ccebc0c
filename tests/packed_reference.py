"""Packed-batch operators in 64 bits (numpy), and the bounds their results are held to.

A rounding is off by half a step at most, eps / 2 relative: bf16 2^-8, f16 2^-11, f32 2^-24.
"""
import numpy as np

from hologram_amd import DTYPE_BF16, DTYPE_F16, DTYPE_F32

HALF = {DTYPE_BF16: 2.0 ** -8, DTYPE_F16: 2.0 ** -11, DTYPE_F32: 2.0 ** -24}
ALL = [DTYPE_BF16, DTYPE_F16, DTYPE_F32]


def encode(x, dtype):
    """f64 / f32 values rounded to nearest into the dtype's array (bf16 as bits)."""
    x = np.asarray(x, np.float32)
    if dtype == DTYPE_F32:
        return x
    if dtype == DTYPE_F16:
        return x.astype(np.float16)
    u = np.ascontiguousarray(x).view(np.uint32)
    r = ((u.astype(np.uint64) + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r).astype(np.uint16)


def decode(a, dtype):
    if dtype == DTYPE_BF16:
        return (np.asarray(a).view(np.uint16).astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return np.asarray(a).view({DTYPE_F16: np.float16, DTYPE_F32: np.float32}[dtype]).astype(np.float64)


def attend(q, k, v, keys, heads, kv_heads, scale):
    """q [n, heads, d], k, v [m, kv_heads, d], row t over the first keys[t] keys: the result
    [n, heads, d] and the bound of each of its rows [n, heads, 1], given the size of the
    weights' rounding afterwards (see `bound`)."""
    n, _, d = q.shape
    out = np.zeros((n, heads, v.shape[2]))
    slack, top = np.zeros((n, heads, 1)), np.zeros((n, heads, 1))
    with np.errstate(all="ignore"):
        for h in range(heads):
            kh = h // (heads // kv_heads)
            for t in range(n):
                m = int(keys[t])
                if m == 0:
                    continue
                kk, vv = k[:m, kh], v[:m, kh]
                s = kk @ q[t, h] / scale
                p = np.exp(s - s.max())
                out[t, h] = p @ vv / p.sum()
                # a score: products of d + 8 sums in f32, q held to 23 bits of its largest
                mag = (np.abs(kk) @ np.abs(q[t, h])).max() / scale
                hold = np.abs(q[t, h]).max() * np.abs(kk).sum(axis=1).max() / scale
                slack[t, h] = 2 * ((d + 8) * 2.0 ** -24 * mag + 2.0 ** -23 * hold) + (m + 64) * 2.0 ** -23
                top[t, h] = np.abs(vv).max()
    return out, slack, top


def bound(slack, top, dtype):
    """Each weight and the result rounded once to the dtype (f32 weights to 22 bits at least),
    and the scores' and sums' own errors: all times the largest |v| that the row sees."""
    return (2 * HALF[dtype] + (2.0 ** -22 if dtype == DTYPE_F32 else 0) + slack) * top


def block_append(cache, scales, new, rows, pos, block):
    """cache int8 [batch, kv, bucket, d], scales f32 [batch, kv, nb], new f64 [tokens, kv, d]."""
    cache, scales = cache.astype(np.float64), scales.astype(np.float64)
    bucket, at = cache.shape[2], 0
    for b, (n, p) in enumerate(zip(rows, pos)):
        for kh in range(cache.shape[1]):
            for j in range(p // block, (p + n - 1) // block + 1 if n else 0):
                lo, hi = max(p, j * block), min(p + n, (j + 1) * block, bucket)
                if lo >= hi:
                    continue
                x = new[at + lo - p:at + hi - p, kh]
                top = np.abs(x).max()
                if not np.isfinite(top):
                    s = np.nan
                else:
                    s = 0.0 if top == 0 else max(2.0 ** np.ceil(np.log2(top / 127.0)), 2.0 ** -126)
                    while top > 127 * s:
                        s *= 2
                    while s > 2.0 ** -126 and top <= 127 * s / 2:
                        s /= 2
                if lo > j * block:
                    old = scales[b, kh, j]
                    if np.isnan(old) or abs(old) > s:
                        s = abs(old)
                    if not np.isnan(s) and s != old:
                        held = cache[b, kh, j * block:lo]
                        cache[b, kh, j * block:lo] = np.clip(np.rint(held * (old / s)), -127, 127)
                scales[b, kh, j] = s
                cache[b, kh, lo:hi] = np.clip(np.rint(x / s), -127, 127) if s > 0 else 0
        at += n
    return cache.astype(np.int8), scales.astype(np.float32)


def process_logits(x, history, spans, params, ids, values, mask):
    out = np.array(x, np.float64)
    rows, cols = out.shape
    with np.errstate(all="ignore"):
        for r in range(rows):
            if history is not None:
                h = history[r, :min(int(spans[r, 1]), history.shape[1])].astype(np.int64)
                gen = h[min(int(spans[r, 0]), len(h)):]
                rep, freq, pres = (float(v) for v in params[r])
                for c in np.unique(h[(h >= 0) & (h < cols)]):
                    v = out[r, c]
                    out[r, c] = v / rep if v > 0 else v * rep
                    times = int((gen == c).sum())
                    if times:
                        out[r, c] -= freq * times + pres
            if ids is not None:
                for c, v in zip(ids[r], values[r]):
                    if 0 <= c < cols:
                        out[r, c] += float(v)
            if mask is not None:
                allowed = (mask[r, np.arange(cols) // 32] >> (np.arange(cols) % 32).astype(np.uint32)) & 1
                out[r, allowed == 0] = -np.inf
    return out
