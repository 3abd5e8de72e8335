"""CPU oracle of the steps over the 8-bit key/value cache: rotary positions on
several axes, and attention with a sliding window or of a tree of drafted tokens,
from their definitions in 64 bits (numpy)."""
from __future__ import annotations

import math

import numpy as np


def angles(positions: np.ndarray, turns, axis) -> np.ndarray:
    """(..., pairs) angles in radians, whole turns left out, of positions (...,
    axes): exact products of integers modulo 2^64. A pair of an axis that there is
    not does not turn."""
    p = np.asarray(positions).astype(object)
    out = np.zeros(p.shape[:-1] + (len(turns),))
    for j, (t, a) in enumerate(zip(turns, axis)):
        if 0 <= a < p.shape[-1]:
            x = (p[..., a] * (int(t) % 2 ** 64)) % 2 ** 64
            out[..., j] = 2 * math.pi * (x.astype(np.float64) / 2.0 ** 64)
    return out


def axis_rope(x: np.ndarray, positions, turns, axis, halves: bool, inverse: bool = False):
    """Rows x (B, S, H, D) turned by positions (B, S, axes), and |u| + |w| of each
    value's pair (how far an error of a sine reaches)."""
    a = angles(positions, turns, axis)[:, :, None]
    c, s = np.cos(a), np.sin(a) * (-1 if inverse else 1)
    D = x.shape[-1]
    lo = slice(0, D // 2) if halves else slice(0, D, 2)
    hi = slice(D // 2, D) if halves else slice(1, D, 2)
    u, w = x[..., lo], x[..., hi]
    y, size = np.empty(x.shape), np.empty(x.shape)
    y[..., lo], y[..., hi] = u * c - w * s, u * s + w * c
    size[..., lo] = size[..., hi] = np.abs(u) + np.abs(w)
    return y, size


def window_sees(n: int, m: int, window: int, sinks: int, causal: bool) -> np.ndarray:
    """(m, n) truth values: query i of m sees key j of n."""
    e = (n - m + 1 + np.arange(m) if causal else np.full(m, n))[:, None]
    j = np.arange(n)[None, :]
    return (j < e) & ((j >= e - window) | (j < sinks))


def tree_sees(n: int, m: int, parents) -> np.ndarray:
    """(m, n) truth values for drafted tokens with these parents."""
    see = np.zeros((m, n), bool)
    base = n - m
    for i in range(m):
        if base + i < 0:
            continue  # (not in the cache, as its ancestors)
        see[i, :max(base, 0)] = True
        j = i
        while j >= 0 and base + j >= 0:
            see[i, base + j] = True
            j = int(parents[j]) if 0 <= parents[j] < j else -1
    return see


def masked_attention(q, k, v, sees, kv_len=None, q_len=None, slots=None, scale=None):
    """out and spread (B, Sq, H, D), as cache_oracle.cached_attention gives them;
    sees(b, n, m): what item b's m queries see of its n keys (where its slot is not
    there, of keys that are not there either)."""
    B, Sq, H, D = q.shape
    n_slots, Hk, cap, _ = k.shape
    scale = D ** -0.5 if scale is None else scale
    out, spread = np.zeros(q.shape), np.zeros(q.shape)
    for b in range(B):
        m = Sq if q_len is None else min(max(int(q_len[b]), 0), Sq)
        n = cap if kv_len is None else min(max(int(kv_len[b]), 0), cap)
        slot = b if slots is None else int(slots[b])
        if not 0 <= slot < n_slots or m == 0 or n == 0:
            continue
        see = sees(b, n, m)
        for h in range(H):
            g = h // (H // Hk)
            s = np.where(see, q[b, :m, h] @ k[slot, g, :n].T * scale, -np.inf)
            w = np.exp(s - np.maximum(s.max(-1, keepdims=True), -1e300))
            total = w.sum(-1, keepdims=True)
            total[total == 0] = 1.0
            out[b, :m, h], spread[b, :m, h] = w @ v[slot, g, :n] / total, w @ np.abs(v[slot, g, :n]) / total
    return out, spread
