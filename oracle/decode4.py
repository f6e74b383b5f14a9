"""The 4-bit decode operators in float64 numpy: the group format (nsa_weight4 / nsa_kv4_cache of
include/nsattn.h), the linear over it, the cache step and the attention over cached rows.  Written from the
definitions, value by value where a layout is concerned; test infrastructure only."""

from __future__ import annotations

import numpy as np


def quantise(x, group):
    """x [..., n * group] -> codes (int, -7..7) of x's shape and float64 scales [..., n]."""
    x = np.asarray(x, np.float64)
    g = x.reshape(*x.shape[:-1], -1, group)
    amax = np.abs(g).max(-1)                       # NaN where the group holds one
    bad = ~np.isfinite(amax)
    amax = np.minimum(np.where(bad, 1.0, amax), 2.0 ** 120)
    m, e = np.frexp(amax / 7)                      # m in [0.5, 1): five bits are multiples of 1/32
    s = np.ldexp(np.ceil(m * 32) / 32, e)
    s = np.where(amax < 2.0 ** -110, 0.0, s)
    sat = np.where(bad[..., None], 0.0, np.clip(g, -(2.0 ** 120), 2.0 ** 120))
    c = np.where(s[..., None] > 0, np.rint(sat / np.where(s > 0, s, 1.0)[..., None]), 0.0)
    c = np.clip(c, -7, 7)
    s = np.where(bad, np.nan, s)
    return c.reshape(x.shape).astype(np.int64), s


def values(c, s):
    g = c.reshape(*s.shape, -1).astype(np.float64) * s[..., None]
    return g.reshape(c.shape)


def pack_weight(c, s, group):
    """Codes and scales of [N, K] (any N; K padded by the caller to the group) -> the tiled arrays."""
    N, K = c.shape
    T, C = -(-N // 16), -(-K // 128)
    codes = np.full((T, C, 16, 64), 0x88, np.uint8)
    scales = np.zeros((T, C, 16, 128 // group), np.float64)
    for k in range(K):
        r, e = k % 128, k % 8
        nib = e // 2 if e % 2 == 0 else 4 + (e - 1) // 2
        at = 16 * ((r // 8) % 4) + 4 * (r // 32) + nib // 2
        v = (c[:, k] + 8).astype(np.uint8)
        for n in range(N):
            old = codes[n // 16, k // 128, n % 16, at]
            codes[n // 16, k // 128, n % 16, at] = (old & 0xF0) | v[n] if nib % 2 == 0 else (old & 0x0F) | (v[n] << 4)
    for n in range(N):
        for j in range(s.shape[1]):
            scales[n // 16, j * group // 128, n % 16, j % (128 // group)] = s[n, j]
    return codes, scales


def norm_rope(x, w, cos, sin, eps):
    """x [..., D] float64, cos / sin [..., D/2] or None."""
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
    if cos is None:
        return y
    h = x.shape[-1] // 2
    a, b = y[..., :h], y[..., h:]
    return np.concatenate([a * cos - b * sin, b * cos + a * sin], -1)


def attention(q, k, v, pos, window, sinks, scale):
    """One query head [D] at position pos over cached rows k, v [n, D] (n > pos; NaN rows where a page is
    missing are masked through `np.isnan(k).all(-1)` by the caller).  Returns the row, the weights' sum of
    |v| and the largest sum of |q k| scale (the scores' error bound)."""
    j = np.arange(k.shape[0])
    see = j <= pos
    if window:
        see &= (j > pos - window) | (j < sinks)
    k, v = k[see], v[see]
    if not len(k):
        return np.zeros_like(q), np.zeros_like(q), 0.0
    s = (k @ q) * scale
    p = np.exp(s - s.max())
    p /= p.sum()
    return p @ v, p @ np.abs(v), float((np.abs(k) @ np.abs(q)).max() * abs(scale))
