"""An 8-bit key/value cache and the attention over it, on the GPU.

A cache keeps the keys and values of sequences whose attention is called again
and again: the text or image states that every denoising step's cross-attention
reads, the past tokens of an autoregressive rollout or a causal text encoder, a
prompt template that a whole batch shares. (The reference recomputes or holds
such states in bf16: cross-attention context `src/vidax/models/wan/wan2_1/
dit.py:119-127`, causal text pathway `src/vidax/models/cosmos3/
dit_layers.py:114-135`.)

`kv_cache_write` quantises new tokens into it (e4m3 with one power-of-two scale
per token and head), `kv_cache_read` gives them back in bf16, `cached_attention`
attends over it (any number of queries per sequence, grouped heads, causal or
not), and `shared_prefix_attention` attends over a prefix that the items of a
batch share, read once for all of them, and each item's own tokens. Every call
launches HIP kernels on torch's current stream and never waits for the GPU;
lengths, positions and slots are device tensors, so a captured graph may be
replayed while they change.
"""
from __future__ import annotations

import functools
from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib
from .attention import _aligned, _strides3

__all__ = ["KVCache", "create_kv_cache", "kv_cache_write", "kv_cache_read", "cached_attention",
           "shared_prefix_attention"]

_E4M3 = torch.float8_e4m3fn
_E8M0 = torch.float8_e8m0fnu


class KVCache(NamedTuple):
    """Cached keys and values: k and v (slots, num_kv_heads, capacity,
    head_dim) float8_e4m3fn, k_scale and v_scale (slots, num_kv_heads,
    capacity) float8_e8m0fnu, all contiguous; capacity a multiple of 64,
    head_dim 64 or 128. The row at [s, h, p] stands for k[s, h, p] *
    k_scale[s, h, p]; scale NaN marks a row that held a NaN or an infinity."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor


def create_kv_cache(num_slots: int, capacity: int, num_kv_heads: int, head_dim: int, device=None) -> KVCache:
    """A cache of num_slots sequences of up to `capacity` tokens (rounded up to
    a multiple of 64), every position holding zeros."""
    if num_slots < 1 or capacity < 1 or num_kv_heads < 1:
        raise ValueError("num_slots, capacity and num_kv_heads must be >= 1")
    if head_dim not in (64, 128):
        raise NotImplementedError(f"head_dim {head_dim} is not supported (64 and 128 are)")
    shape = (num_slots, num_kv_heads, (capacity + 63) // 64 * 64)
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else device
    k, v = (torch.zeros(shape + (head_dim,), dtype=torch.uint8, device=device).view(_E4M3) for _ in range(2))
    ks, vs = (torch.full(shape, 127, dtype=torch.uint8, device=device).view(_E8M0) for _ in range(2))
    return KVCache(k, v, ks, vs)


def _check_cache(cache: KVCache, name: str) -> None:
    k, v, ks, vs = cache
    if (k.dtype == v.dtype == _E4M3 and ks.dtype == vs.dtype == _E8M0 and k.dim() == 4 and k.shape == v.shape and
            ks.shape == vs.shape == k.shape[:3] and k.is_cuda and k.device == v.device == ks.device == vs.device and
            k.is_contiguous() and v.is_contiguous() and ks.is_contiguous() and vs.is_contiguous()):
        return  # (the checks below say what is wrong; the C ABI checks sizes and alignment)
    parts = (("k", k, _E4M3, 4), ("v", v, _E4M3, 4), ("k_scale", ks, _E8M0, 3), ("v_scale", vs, _E8M0, 3))
    for n, t, dtype, dims in parts:
        if t.dtype != dtype:
            raise TypeError(f"{name}.{n} must be {dtype}; got {t.dtype}")
        if t.dim() != dims or t.shape != k.shape[:dims]:
            raise ValueError(f"{name}.{n} of shape {tuple(t.shape)} does not go with {name}.k {tuple(k.shape)}: k and "
                             "v are (slots, num_kv_heads, capacity, head_dim), the scales the first three")
    for n, t, _, _ in parts:
        if not t.is_cuda:
            raise ValueError(f"{name}.{n} must be a GPU tensor")
        if t.device != k.device:
            raise ValueError(f"{name}'s tensors must be on one device")
        if not t.is_contiguous():
            raise ValueError(f"{name}.{n} must be contiguous")


def _check_rows(x: torch.Tensor, name: str, cache: KVCache) -> None:
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if x.dim() != 4:
        raise ValueError(f"{name} must be (B, S, H, D); got shape {tuple(x.shape)}")
    if x.dtype != torch.bfloat16:
        raise TypeError(f"{name} must be bfloat16; got {x.dtype}")
    if x.device != cache.k.device:
        raise ValueError(f"{name} must be on the cache's device")
    if x.shape[3] != cache.k.shape[3]:
        raise ValueError(f"{name} has head dim {x.shape[3]}, the cache {cache.k.shape[3]}")


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x as the kernels read it: its values in memory, the head dim contiguous,
    16-byte aligned, strides multiples of 8 (a copy where it is not so)."""
    if x.is_neg():
        x = x.resolve_neg()
    x = _aligned(x) if x.stride(3) == 1 else x.contiguous()
    return x if x.data_ptr() % 16 == 0 else x.clone(memory_format=torch.contiguous_format)


def _ints(x, n: int, dev: torch.device, name: str) -> Optional[torch.Tensor]:
    """int32 (n,) on dev, or None."""
    if x is None:
        return None
    if not (isinstance(x, torch.Tensor) and x.dtype == torch.int32 and x.device == dev and x.is_contiguous()):
        x = torch.as_tensor(x, device=dev)
        if x.is_floating_point() or x.is_complex() or x.dtype == torch.bool:
            raise TypeError(f"{name} must hold integers; got {x.dtype}")
        # (values past 32 bits are held at its ends, outside any cache)
        x = x.clamp(-(1 << 31), (1 << 31) - 1).to(torch.int32).contiguous() if x.dtype == torch.int64 else \
            x.to(torch.int32).contiguous()
    if x.numel() != n:
        raise ValueError(f"{name} must hold {n} integers; got shape {tuple(x.shape)}")
    return x


def _ptr(x: Optional[torch.Tensor]) -> Optional[int]:
    return None if x is None else x.data_ptr()


def _cache_args(c: Optional[KVCache]):
    if c is None:
        return None, None, None, None, 0, 0
    return (c.k.data_ptr(), c.v.data_ptr(), c.k_scale.data_ptr(), c.v_scale.data_ptr(), c.k.shape[0], c.k.shape[2])


def kv_cache_write(cache: KVCache, k: torch.Tensor, v: torch.Tensor, start=None, *, num=None, slots=None) -> None:
    """Quantises new tokens into the cache: token t of batch item b goes to
    position start[b] + t of slot slots[b].

    k and v are (B, S, num_kv_heads, head_dim) bf16. start (B,): the first
    position (default 0). num (B,): how many of an item's S tokens are real;
    the others are padding and not written (default all). slots (B,): the
    items' slots (default 0, 1, ...). A row is stored as e4m3 times the smallest
    power of two that fits its largest magnitude, each value rounded once (by at
    most 2^-4 of itself; by at most 2^-10 of the scale below 2^-6 of it); a row
    with a NaN or an infinity is stored as NaN.
    Tokens outside the cache (a position past its capacity, a negative one, an
    unknown slot) are dropped. Where two items name the same slot and position,
    the later item's token is kept.
    """
    _check_cache(cache, "cache")
    for n, x in (("k", k), ("v", v)):
        _check_rows(x, n, cache)
        if x.shape[2] != cache.k.shape[1]:
            raise ValueError(f"{n} has {x.shape[2]} heads, the cache {cache.k.shape[1]}")
    if k.shape != v.shape:
        raise ValueError(f"k and v shapes differ: {tuple(k.shape)} vs {tuple(v.shape)}")
    B, S, Hk, D = k.shape
    dev = k.device
    start, num, slots = (_ints(x, B, dev, n) for x, n in ((start, "start"), (num, "num"), (slots, "slots")))
    if B == 0 or S == 0:
        return
    k, v = _rows(k), _rows(v)
    ck, cv, ks, vs, n_slots, cap = _cache_args(cache)
    _lib.launch(dev, _lib.lib().vx_kv_write_fwd, k.data_ptr(), v.data_ptr(), _strides3(k), _strides3(v), ck, cv, ks,
                vs, n_slots, cap, _ptr(start), _ptr(num), _ptr(slots), B, S, Hk, D)


def kv_cache_read(cache: KVCache, length: int, start=None, *, slots=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(k, v), each (B, length, num_kv_heads, head_dim) bf16: positions start[b]
    .. start[b] + length - 1 of slot slots[b], as they are stored (bf16 holds
    every such value; magnitudes below 2^-126 give zero). B is the length of
    `slots`, else of `start`, else the number of slots; defaults as in
    kv_cache_write. Positions outside the cache give zeros."""
    _check_cache(cache, "cache")
    length = int(length)
    if length < 0:
        raise ValueError(f"length must be >= 0; got {length}")
    dev = cache.k.device
    n_slots, Hk, _, D = cache.k.shape
    slots = None if slots is None else torch.as_tensor(slots, device=dev)
    start = None if start is None else torch.as_tensor(start, device=dev)
    B = slots.numel() if slots is not None else start.numel() if start is not None else n_slots
    start, slots = _ints(start, B, dev, "start"), _ints(slots, B, dev, "slots")
    k, v = (torch.empty((B, length, Hk, D), dtype=torch.bfloat16, device=dev) for _ in range(2))
    if B == 0 or length == 0:
        return k, v
    ck, cv, ks, vs, n_slots, cap = _cache_args(cache)
    _lib.launch(dev, _lib.lib().vx_kv_read_fwd, ck, cv, ks, vs, n_slots, cap, _ptr(start), _ptr(slots), B, length, Hk,
                D, k.data_ptr(), v.data_ptr())
    return k, v


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(device_index: int, *sizes: int) -> int:
    with torch.cuda.device(device_index):
        return max(int(_lib.lib().vx_cached_attn_workspace_size(*sizes)), 0)  # (sizes it refuses: the launch says why)


def _attend(q: torch.Tensor, cache: KVCache, prefix: Optional[KVCache], kv_len, prefix_len, q_len, slots,
            causal: bool, scale: Optional[float], out: Optional[torch.Tensor]) -> torch.Tensor:
    _check_cache(cache, "cache")
    _check_rows(q, "q", cache)
    B, Sq, H, D = q.shape
    dev = q.device
    n_slots, Hk, cap, _ = cache.k.shape
    n_prefix = p_cap = 0
    if prefix is not None:
        _check_cache(prefix, "prefix")
        if prefix.k.shape[1] != Hk or prefix.k.shape[3] != D or prefix.k.device != dev:
            raise ValueError("prefix and cache must agree on heads, head dim and device")
        n_prefix, p_cap = prefix.k.shape[0], prefix.k.shape[2]
        prefix_len = _ints(prefix_len, n_prefix, dev, "prefix_len")
    kv_len, q_len, slots = (_ints(x, B, dev, n) for x, n in ((kv_len, "kv_len"), (q_len, "q_len"), (slots, "slots")))
    if out is None:
        out = torch.empty((B, Sq, H, D), dtype=q.dtype, device=dev)
    elif (out.shape != q.shape or out.dtype != q.dtype or out.stride(-1) != 1 or out.device != dev):
        raise ValueError("out must be a (B, Sq, H, D) bf16 tensor with a contiguous head dim, on q's device")
    if B == 0 or Sq == 0 or H == 0:
        return out
    q = _rows(q)
    ws_bytes = _workspace_bytes(dev.index, cap, n_prefix, p_cap, B, Sq, H, Hk, D)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if ws_bytes > 0 else None
    _lib.launch(dev, _lib.lib().vx_cached_attn_fwd, q.data_ptr(), out.data_ptr(), _strides3(q), _strides3(out),
                *_cache_args(cache), *_cache_args(prefix), _ptr(kv_len), _ptr(q_len), _ptr(slots), _ptr(prefix_len),
                B, Sq, H, Hk, D, int(bool(causal)), D ** -0.5 if scale is None else float(scale), _ptr(ws), ws_bytes)
    return out


def cached_attention(q: torch.Tensor, cache: KVCache, kv_len=None, *, q_len=None, slots=None, causal: bool = True,
                     scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of q (B, Sq, H, D) bf16 over cached keys and values; returns
    (B, Sq, H, D) bf16. H is a multiple of the cache's heads: query head h reads
    cached head h // (H / num_kv_heads).

    kv_len (B,): an item's cached tokens, its new ones among them (write them
    first); default the capacity. q_len (B,): how many of its Sq queries are
    real (default all); the other rows of the output are zeros. slots (B,): the
    items' slots (default 0, 1, ...). causal: the queries are the sequence's
    last tokens, query i of q_len at position kv_len - q_len + i, and see no
    later one; False: every query sees every cached token (cross-attention to
    an encoder's states). scale defaults to 1/sqrt(D).
    Lengths are held to [0, capacity] and [0, Sq]; an item whose slot the cache
    does not have sees no keys, and a query that sees no key gives zeros. A
    cached row of scale NaN makes NaN the outputs of exactly the queries of its
    head that see it.
    """
    return _attend(q, cache, None, kv_len, None, q_len, slots, causal, scale, out)


def shared_prefix_attention(q: torch.Tensor, prefix: KVCache, cache: KVCache, kv_len=None, *, prefix_len=None,
                            q_len=None, slots=None, causal: bool = True, scale: Optional[float] = None,
                            out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """cached_attention of a batch whose items share a prefix: every query sees
    the whole prefix, then its own item's cached tokens as in cached_attention
    (kv_len, and the positions of causal, count those alone).

    prefix: a cache whose slot g holds the prefix of the batch items g * n ..
    g * n + n - 1, n = B / (its number of slots): one slot for a prefix that all
    share, two for a guided batch's halves. prefix_len (slots,): its tokens
    (default its capacity), held to [0, capacity]. The queries of a group read
    each prefix row once for all of them.
    """
    if prefix is None:
        raise TypeError("prefix must be a KVCache")
    return _attend(q, cache, prefix, kv_len, prefix_len, q_len, slots, causal, scale, out)
