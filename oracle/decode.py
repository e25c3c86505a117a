"""Float64 NumPy definitions of the cached-decoding kernels, with the error bounds their tests use."""

from __future__ import annotations

import numpy as np


def turned(x, positions, steps, scale, interleaved):
    """x [B, S, H, D] float64, positions [B, S] ints, steps int64 [R / 2]: pairs turned by
    position * step / 2**64 turns (product modulo 2**64), times scale."""
    x = np.array(x, np.float64)
    steps = np.asarray(steps, np.int64).view(np.uint64)
    phase = np.asarray(positions, np.int64).view(np.uint64)[:, :, None] * steps  # wraps
    angle = phase.astype(np.float64) * (2.0 * np.pi / 2.0 ** 64)
    c, s = np.cos(angle)[:, :, None] * scale, np.sin(angle)[:, :, None] * scale
    r = 2 * steps.size
    lo = slice(0, r, 2) if interleaved else slice(0, r // 2)
    hi = slice(1, r, 2) if interleaved else slice(r // 2, r)
    a, b = x[..., lo].copy(), x[..., hi].copy()
    x[..., lo], x[..., hi] = a * c - b * s, b * c + a * s
    return x


def pair_size(x, rotary, scale, interleaved):
    """scale * (|a| + |b|) at both elements of each pair, |x| behind the rotated part."""
    m = np.abs(np.array(x, np.float64))
    lo = slice(0, rotary, 2) if interleaved else slice(0, rotary // 2)
    hi = slice(1, rotary, 2) if interleaved else slice(rotary // 2, rotary)
    m[..., lo] = m[..., hi] = (m[..., lo] + m[..., hi]) * scale
    return m


def normed(x, weight, eps):
    x = np.asarray(x, np.float64)
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    return y if weight is None else y * np.asarray(weight, np.float64)


def tree_attention(q, k, v, lengths, mask, scale):
    """q [B, T, H, D], caches [B, Hk, C, D], mask [T, T], [B, T, T] or None (a chain).
    -> out, and per output the size sum_j p_j |v_j| and the row's largest score error in ulps of 2**-24."""
    q = np.asarray(q, np.float64)
    B, T, H, D = q.shape
    hk = k.shape[1]
    g = H // hk
    out, size = np.zeros((B, T, H, D)), np.zeros((B, T, H, D))
    ulps = np.zeros((B, T, H, 1))
    if mask is None:
        mask = np.tril(np.ones((T, T), bool))
    for b in range(B):
        n = int(lengths[b])
        if n < 0 or n + T > k.shape[2]:
            continue
        m = mask[b] if mask.ndim == 3 else mask
        for t in range(T):
            rows = np.concatenate([np.arange(n), n + np.nonzero(m[t])[0]])
            if not rows.size:
                continue
            for h in range(H):
                kk, vv = (np.asarray(c[b, h // g, rows], np.float64) for c in (k, v))
                s = kk @ q[b, t, h] * scale
                e = np.exp(s - s.max())
                p = e / e.sum()
                out[b, t, h], size[b, t, h] = p @ vv, p @ np.abs(vv)
                # D products and sums, the scale, the subtraction and the base-2 argument
                ulps[b, t, h] = (D + 4) * (np.abs(kk) @ np.abs(q[b, t, h]) * scale).max() + rows.size + 16
    return out, size, ulps


def commit(cache, lengths, path, accepted):
    cache = np.array(cache)
    for b, (n, m) in enumerate(zip(lengths, accepted)):
        cache[b, :, n:n + m] = cache[b][:, n + np.asarray(path[b][:m], np.int64)]
    return cache
