"""The operators of a long-context step in 64 bits (numpy): QkNormRotary, KvBlockBounds,
KvBlockSelect and AttentionI8Selected, with the bounds that computed results are held to."""
import numpy as np

from hologram_amd import DTYPE_F16
from packed_reference import HALF, attend


def rotary(x, gamma, eps, pos, freqs, rot, interleaved, magnitude, dtype):
    """x f64 [tokens, heads, d] at positions pos [tokens]: the result and its bound. gamma None
    with eps None: no norm."""
    d = x.shape[-1]
    y = x
    if eps is not None:
        y = x / np.sqrt((x * x).mean(axis=-1, keepdims=True) + eps)
        if gamma is not None:
            y = y * gamma
    out, mag = y.copy(), np.abs(y)
    if rot:
        ang = pos.astype(np.longdouble)[:, None] * freqs.astype(np.longdouble)
        c, s = (f(ang).astype(np.float64)[:, None] for f in (np.cos, np.sin))
        first, second = ((slice(0, rot, 2), slice(1, rot, 2)) if interleaved else
                         (slice(0, rot // 2), slice(rot // 2, rot)))
        a, b = y[..., first], y[..., second]
        out[..., first], out[..., second] = magnitude * (a * c - b * s), magnitude * (b * c + a * s)
        mag[..., first] = mag[..., second] = magnitude * (np.abs(a) + np.abs(b))
    # The root: a sum of d squares and four more operations, d + 8 roundings of half a step at
    # most. The norm two, cos and sin (their argument's rounding and the function's) 8, the
    # magnitude and the pair's sums 4. Then the result's own, and f16's step below its normals.
    tol = HALF[dtype] * np.abs(out) + mag * (d + 24) * 2.0 ** -24
    return out, tol + (2.0 ** -25 if dtype == DTYPE_F16 else 2.0 ** -130)


def block_bounds(cache, bounds, rows, pos, block):
    """cache int8 [batch, kv, bucket, d], bounds int8 [batch, kv, nb, 2, d]."""
    out, bucket = bounds.copy(), cache.shape[2]
    for b, (n, p) in enumerate(zip(rows, pos)):
        end = min(p + n, bucket)
        for j in range(p // block, -(-end // block)) if n and p < end else ():
            x = cache[b, :, j * block:min((j + 1) * block, end)]
            out[b, :, j, 0], out[b, :, j, 1] = x.min(axis=1), x.max(axis=1)
    return out


def eight_bits(q):
    """q f64 [..., heads, d] of one kv head as whole numbers, by the group's power of two."""
    q = np.where(np.isfinite(q), q, 0.0)
    top = np.abs(q).max()
    if top == 0:
        return q
    s = max(2.0 ** np.ceil(np.log2(top / 127.0)), 2.0 ** -126)
    while top > 127 * s:
        s *= 2
    while s > 2.0 ** -126 and top <= 127 * s / 2:
        s /= 2
    return np.rint(q / s)


def select_blocks(q, bounds, scales, lens, rows, kv, bucket, block, top, first, last):
    """q f64 [tokens, heads, d], bounds int8 [batch, kv, nb, 2, d], scales f32 [batch, kv, nb]:
    i32 [tokens, kv, top]."""
    g = q.shape[1] // kv
    out, at = np.full((q.shape[0], kv, top), -1, np.int32), 0
    with np.errstate(all="ignore"):
        for b, n in enumerate(rows):
            for t in range(n):
                v = min(max(int(lens[b]) - (n - 1 - t), 0), bucket)
                seen = -(-v // block)
                for kh in range(kv):
                    if seen <= top:
                        out[at + t, kh, :seen] = np.arange(seen)
                        continue
                    x = eight_bits(q[at + t, kh * g:(kh + 1) * g])[:, None]         # [g, 1, d]
                    j = np.arange(first, seen - last)
                    lo, hi = (bounds[b, kh, j, i].astype(np.float64) for i in (0, 1))
                    s = scales[b, kh, j].astype(np.float64)
                    most = np.maximum(x * lo, x * hi).sum(axis=(0, 2))
                    least = np.minimum(x * lo, x * hi).sum(axis=(0, 2))
                    score = np.where(s < 0, least, most) * s
                    score[np.isnan(score)] = np.inf
                    best = j[np.argsort(-score, kind="stable")[:top - first - last]]
                    out[at + t, kh] = np.sort(np.concatenate(
                        [np.arange(first), best, np.arange(seen - last, seen)]))
            at += n
    return out


def attend_listed(q, k, v, ks, vs, lists, lens, rows, kv, block, scale):
    """q f64 [tokens, heads, d], k, v int8 [batch, kv, bucket, d], ks, vs f32 [batch, kv, nb], lists
    [tokens, kv, top]: as packed_reference.attend."""
    g, bucket = q.shape[1] // kv, k.shape[2]
    nb = -(-bucket // block)
    out = np.zeros(q.shape)
    slack, top, at = np.zeros((*q.shape[:2], 1)), np.zeros((*q.shape[:2], 1)), 0
    for b, n in enumerate(rows):
        for t in range(n):
            sees = min(max(int(lens[b]) - (n - 1 - t), 0), bucket)
            for kh in range(kv):
                keys = [np.arange(j * block, min((j + 1) * block, sees))
                        for j in lists[at + t, kh].tolist() if 0 <= j < nb and j * block < sees]
                if not keys:
                    continue
                i = np.concatenate(keys)
                kk = k[b, kh, i].astype(np.float64) * ks[b, kh, i // block].astype(np.float64)[:, None]
                vv = v[b, kh, i].astype(np.float64) * vs[b, kh, i // block].astype(np.float64)[:, None]
                h = slice(kh * g, (kh + 1) * g)
                out[at + t, h], slack[at + t, h], top[at + t, h] = (
                    x[0] for x in attend(q[at + t:at + t + 1, h], kk[:, None], vv[:, None], [len(i)], g, 1, scale))
        at += n
    return out, slack, top
