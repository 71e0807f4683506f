"""The 4-bit KV cache and its attention from their definition, in NumPy and 64 bits.

Test infrastructure only.  A group is 64 consecutive dimensions of one head at one position:
codes c = 0..15 and two bf16 numbers z and h, value = fp32(z + h (2 c - 15)).
"""
from __future__ import annotations

import numpy as np


def bf16(x):
    """float32 -> the nearest bf16 (ties to even), as float32; NaN and infinities stay."""
    x = np.asarray(x, np.float32)
    u = x.view(np.uint32)
    r = ((u + np.uint32(0x7FFF) + ((u >> np.uint32(16)) & np.uint32(1))) & np.uint32(0xFFFF0000)).view(np.float32)
    return np.where(np.isfinite(x), r, x)


def quantise(x):
    """x fp32 [..., hd] -> (codes int [..., hd], z, h float64 [..., hd/64])."""
    with np.errstate(all="ignore"):
        g = np.asarray(x, np.float32).astype(np.float64).reshape(*x.shape[:-1], -1, 64)
        lo, hi = 0.5 * g.min(-1), 0.5 * g.max(-1)
        z = bf16((hi + lo).astype(np.float32)).astype(np.float64)
        h = bf16(((hi - lo) / 15.0).astype(np.float32)).astype(np.float64)
        lost = ~(np.isfinite(g).all(-1) & np.isfinite(z) & np.isfinite(h))
        z, h = np.where(lost, np.nan, z), np.where(lost, 0.0, h)
        t = np.where((h == 0.0)[..., None], 0.0, (g - z[..., None]) / h[..., None])
        c = np.clip(np.rint((t + 15.0) * 0.5), 0, 15).astype(np.int64)
    return c.reshape(x.shape), z, h


def values(c, z, h):
    """What codes and scales stand for: float32 [..., hd]."""
    u = (2 * c - 15).reshape(*z.shape, 64)
    return (z[..., None] + h[..., None] * u).astype(np.float32).reshape(c.shape)


def held(x):
    """fp32 [..., hd] -> the values the cache gives back, float32."""
    return values(*quantise(x))


def rope(x, table, p):
    """x fp32 [..., heads, hd] at positions p [...] -> fp32 (rotate-half, 64 bits, rounded once)."""
    half = x.shape[-1] // 2
    cs = table[p].astype(np.float64)[..., None, :, :]
    a, b, c, s = x[..., :half].astype(np.float64), x[..., half:].astype(np.float64), cs[..., 0], cs[..., 1]
    return np.concatenate([a * c - b * s, b * c + a * s], -1).astype(np.float32)


def attention(q, K, V, pos, Lmax=None):
    """q fp32 [B, M, H, hd], K and V [B, Hkv, L, hd], pos [B] -> float64 [B, M, H, hd]: keys 0..pos + m;
    rows outside [0, Lmax) (None: L) are zeros."""
    B, M, H, hd = q.shape
    Hkv, L = K.shape[1], K.shape[2] if Lmax is None else Lmax
    out = np.zeros((B, M, H, hd))
    for b in range(B):
        for m in range(M):
            p = int(pos[b]) + m
            if not 0 <= p < L:
                continue
            for n in range(H):
                k, v = (x[b, n // (H // Hkv), :p + 1].astype(np.float64) for x in (K, V))
                s = k @ q[b, m, n].astype(np.float64) / np.sqrt(hd)
                w = np.exp(s - s.max())
                out[b, m, n] = w @ v / w.sum()
    return out


def attention_bound(q, c, z, h, pos, Lmax=None):
    """How far the device's attention may be from attention(), elementwise (same shape), for keys and
    values given as (codes, z, h) pairs c = (ck, cv), .. [B, Hkv, L, ..].

    One fp32 rounding is e = 2^-24.  A score, with A = sum h |q u| + |z| |q| over its dimensions.  Few rows:
    q times its factor (1 e), in two fp16 terms (2^-22 = 4 e), 2 x 64 products summed in fp32 in any order
    (128 e of the sum of magnitudes, with levels c - 8 of no more than twice |u|, 2 x 128), joined with z's
    sums (63 additions, 5 more): at most 330 e of A.  Many rows: q and k in two fp16 terms each (4 e
    each and 4 e for the product left out, k's sum 1 e), 3 x 128 products summed: at most 400 e.  Then the
    difference to the maximum, both of at most A in base 2, and the exponential: 2 e A log2(e) ln 2 + 4 e.  So a
    weight is off by d = 2 (404 A + 4) e relative to the weights' mean error.  A sum over n keys: the
    products' terms (12 e), the weight's rounding and factors (4 e), the rescalings of up to n / 32 half
    blocks (2 each) and joins, and the additions: many rows 3 n; few rows 2 n of 2 h (c - 8), of no more
    than twice h |u|, and n of z + h, of no more than h |u| + |z|.  At most (5 n + n / 16 + 50) e of
    sum p (h |u| + |z|), and the sum of weights n e more."""
    B, M, H, hd = q.shape
    (ck, cv), (zk, zv), (hk, hv) = c, z, h
    Hkv, L = ck.shape[1], ck.shape[2] if Lmax is None else Lmax
    rep = lambda x: np.repeat(x, 64, -1)  # noqa: E731
    uk, uv = np.abs(2 * ck - 15) * rep(hk) + np.abs(rep(zk)), np.abs(2 * cv - 15) * rep(hv) + np.abs(rep(zv))
    K = rep(zk) + rep(hk) * (2 * ck - 15)
    out = np.zeros((B, M, H, hd))
    e = 2.0 ** -24
    for b in range(B):
        for m in range(M):
            p = int(pos[b]) + m
            if not 0 <= p < L:
                continue
            for n in range(H):
                j = n // (H // Hkv)
                x = q[b, m, n].astype(np.float64) / np.sqrt(hd)
                A = (uk[b, j, :p + 1] @ np.abs(x)).max()
                s = K[b, j, :p + 1] @ x
                w = np.exp(s - s.max())
                out[b, m, n] = (2 * (404 * A + 4) + 6 * (p + 1) + (p + 1) / 16 + 50) * e * (w @ uv[b, j, :p + 1] / w.sum())
    return out
