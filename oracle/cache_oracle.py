"""CPU oracle of the 8-bit key/value cache and the attention over it: the
definitions in 64 bits (numpy)."""
from __future__ import annotations

import numpy as np


def e4m3_values() -> np.ndarray:
    """The value of each e4m3 byte (1 sign, 4 exponent bits of bias 7, 3
    mantissa bits; the all-ones exponent and mantissa are NaN)."""
    c = np.arange(256)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e > 0, (1 + m / 8.0) * 2.0 ** (e - 7.0), m / 8.0 * 2.0 ** -6)
    v = np.where((e == 15) & (m == 7), np.nan, v)
    return np.where(c >= 128, -v, v)


def e8m0_values() -> np.ndarray:
    """The value of each scale byte."""
    v = 2.0 ** (np.arange(256) - 127.0)
    v[255] = np.nan
    return v


def quantise(x: np.ndarray):
    """(bytes (..., D), scale bytes (...,)) of rows x: the nearest e4m3 value of
    x / 2^e, ties to the even mantissa, 2^e >= 2^-126 the smallest power of two
    for which every magnitude is at most 448; rows with a NaN or an infinity:
    zeros and scale 255."""
    x = np.asarray(x, np.float64)
    bad = ~np.isfinite(x).all(-1)
    amax = np.abs(np.where(np.isfinite(x), x, 0.0)).max(-1)
    e = np.full(amax.shape, -126)
    for n in range(-126, 128):
        e = np.where(amax > 448.0 * 2.0 ** n, n + 1, e)
    y = np.where(bad[..., None], 0.0, x) / 2.0 ** e[..., None].astype(np.float64)
    grid = e4m3_values()[:127]  # 0 .. 448, increasing; the byte's low bit is the mantissa's
    mag = np.abs(y)
    hi = np.searchsorted(grid, mag).clip(0, 126)
    lo = (hi - 1).clip(0)
    d_hi, d_lo = grid[hi] - mag, mag - grid[lo]
    code = np.where((d_lo < d_hi) | ((d_lo == d_hi) & (lo % 2 == 0)), lo, hi)
    code = np.where(np.signbit(y) & ~bad[..., None], code + 128, code)
    return code.astype(np.uint8), np.where(bad, 255, e + 127).astype(np.uint8)


def values(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    """What cached rows stand for."""
    return e4m3_values()[codes] * e8m0_values()[scales][..., None]


def cached_attention(q, k, v, kv_len=None, q_len=None, slots=None, causal=True, scale=None, prefix=None,
                     prefix_len=None):
    """out and spread (B, Sq, H, D): softmax attention of q (B, Sq, H, D) over
    cached values k, v (slots, Hk, capacity, D), and over the rows' magnitudes
    |v| in v's place (how far errors of the weights can reach). prefix: (k, v) of
    the groups' shared keys."""
    B, Sq, H, D = q.shape
    n_slots, Hk, cap, _ = k.shape
    scale = D ** -0.5 if scale is None else scale
    out, spread = np.zeros(q.shape), np.zeros(q.shape)
    for b in range(B):
        m = Sq if q_len is None else min(max(int(q_len[b]), 0), Sq)
        n = cap if kv_len is None else min(max(int(kv_len[b]), 0), cap)
        slot = b if slots is None else int(slots[b])
        if not 0 <= slot < n_slots:
            slot, n = 0, 0
        p = 0
        if prefix is not None:
            at = b // (B // prefix[0].shape[0])
            p_cap = prefix[0].shape[2]
            p = p_cap if prefix_len is None else min(max(int(prefix_len[at]), 0), p_cap)
        if m == 0 or n + p == 0:
            continue
        own = np.full(m, n)
        if causal:  # (held to the keys that there are: those of a slot that is not there are none)
            length = cap if kv_len is None else min(max(int(kv_len[b]), 0), cap)
            own = np.minimum(n, np.maximum(length - m + np.arange(m) + 1, 0))
        seen = np.arange(n + p)[None, :] < (p + own)[:, None]
        for h in range(H):
            g = h // (H // Hk)
            kk, vv = (x[slot, g, :n] for x in (k, v))
            if p:
                kk, vv = (np.concatenate([x[at, g, :p], y]) for x, y in zip(prefix, (kk, vv)))
            s = np.where(seen, q[b, :m, h] @ kk.T * scale, -np.inf)
            w = np.exp(s - np.maximum(s.max(-1, keepdims=True), -1e300))
            total = w.sum(-1, keepdims=True)
            total[total == 0] = 1.0
            out[b, :m, h], spread[b, :m, h] = w @ vv / total, w @ np.abs(vv) / total
    return out, spread
