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
replayed while they change. (Lists, arrays and host tensors are copied there
behind the stream's earlier work, which a capture refuses.)
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
_MOST = (1 << 31) - 1  # sizes are 32-bit numbers in the C ABI


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


def _check_cache(cache: KVCache, name: str) -> Tuple[int, int, int, int, int]:
    """(slots, num_kv_heads, capacity, head_dim, device index) of a cache whose
    tensors go together (the C ABI checks sizes and alignment)."""
    if not isinstance(cache, KVCache):
        raise TypeError(f"{name} must be a KVCache")
    try:
        k, v, ks, vs = cache
        shape = k.shape
        n, h, c, d = shape
        index = k.get_device()
        if (k.dtype is _E4M3 and v.dtype is _E4M3 and ks.dtype is _E8M0 and vs.dtype is _E8M0 and v.shape == shape and
                ks.shape == (n, h, c) and vs.shape == (n, h, c) and index >= 0 and v.get_device() == index and
                ks.get_device() == index and vs.get_device() == index and k.is_contiguous() and v.is_contiguous() and
                ks.is_contiguous() and vs.is_contiguous()):
            return n, h, c, d, index
    except (AttributeError, TypeError, ValueError):
        pass
    # what is wrong
    if not all(isinstance(t, torch.Tensor) for t in cache):
        raise TypeError(f"{name} must be a KVCache of four tensors")
    parts = tuple(zip(("k", "v", "k_scale", "v_scale"), cache, (_E4M3, _E4M3, _E8M0, _E8M0), (4, 4, 3, 3)))
    k = cache[0]
    for part, t, dtype, dims in parts:
        if t.dtype != dtype:
            raise TypeError(f"{name}.{part} must be {dtype}; got {t.dtype}")
        if t.dim() != dims or t.shape != k.shape[:dims]:
            raise ValueError(f"{name}.{part} of shape {tuple(t.shape)} does not go with {name}.k {tuple(k.shape)}: k "
                             "and v are (slots, num_kv_heads, capacity, head_dim), the scales the first three")
    for part, t, _, _ in parts:
        if not t.is_cuda:
            raise ValueError(f"{name}.{part} must be a GPU tensor")
        if t.device != k.device:
            raise ValueError(f"{name}'s tensors must be on one device")
        if not t.is_contiguous():
            raise ValueError(f"{name}.{part} must be contiguous")
    raise ValueError(f"{name} is not a KVCache that the kernels take")


def _check_rows(x: torch.Tensor, name: str, index: int, head_dim: int) -> Tuple[int, int, int, int]:
    """The shape of queries, keys or values (B, S, H, D), checked."""
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    shape = x.shape
    if len(shape) != 4:
        raise ValueError(f"{name} must be (B, S, H, D); got shape {tuple(shape)}")
    if x.dtype is not torch.bfloat16:
        raise TypeError(f"{name} must be bfloat16; got {x.dtype}")
    if x.get_device() != index:
        raise ValueError(f"{name} must be on the cache's device")
    if shape[3] != head_dim:
        raise ValueError(f"{name} has head dim {shape[3]}, the cache {head_dim}")
    if shape[1] > _MOST:
        raise NotImplementedError(f"{name} has {shape[1]} tokens per item (at most 2^31 - 1)")
    return shape


def _rows(x: torch.Tensor):
    """(x as the kernels read it, its address, its C ABI strides): its values in
    memory, the head dim contiguous, 16-byte aligned, strides multiples of 8 (a
    copy where it is not so)."""
    if x.is_neg():
        x = x.resolve_neg()
    at = x.data_ptr()
    if at % 16 == 0 and x.is_contiguous():
        return x, at, None
    x = _aligned(x) if x.stride(3) == 1 else x.contiguous()
    if x.data_ptr() % 16 != 0:
        x = x.clone(memory_format=torch.contiguous_format)
    return x, x.data_ptr(), _strides3(x)


def _ints(x, n: int, index: int, name: str):
    """(int32 tensor of n values on the device, its address), or (None, None)."""
    if x is None:
        return None, None
    if not (isinstance(x, torch.Tensor) and x.dtype is torch.int32 and x.get_device() == index and x.is_contiguous()):
        if not isinstance(x, torch.Tensor):
            x = torch.as_tensor(x)
            if x.numel() == 0:  # (an empty list has no integers to tell its type)
                x = x.to(torch.int32)
        if x.is_floating_point() or x.is_complex() or x.dtype == torch.bool:
            raise TypeError(f"{name} must hold integers; got {x.dtype}")
        # (values past 32 bits are held at its ends, outside any cache)
        if x.dtype == torch.uint32:
            x = x.to(torch.int64)
        elif x.dtype == torch.uint64:
            x = x.view(torch.int64)
            x = x.masked_fill(x < 0, (1 << 31) - 1)
        if x.dtype == torch.int64:
            x = x.clamp(-(1 << 31), (1 << 31) - 1)
        x = _on_device(x.to(torch.int32), index, name).contiguous()
    if x.numel() != n:
        raise ValueError(f"{name} must hold {n} integers; got shape {tuple(x.shape)}")
    return x, x.data_ptr()


def _on_device(x: torch.Tensor, index: int, name: str) -> torch.Tensor:
    """x on the device. Host values go by way of pinned memory of the call's own:
    the copy waits its turn on the stream, the call does not, and the caller may
    change x at once. (A captured copy would read that memory again at every replay.)"""
    if x.device.type != "cpu":
        return x.to(torch.device("cuda", index))
    with torch.cuda.device(index):
        if torch.cuda.is_current_stream_capturing():
            raise ValueError(f"{name} must be a device tensor while a graph is captured")
        held = torch.empty(x.shape, dtype=x.dtype, pin_memory=True)
        held.copy_(x)
        return held.to(torch.device("cuda", index), non_blocking=True)


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
    n_slots, Hk, cap, D, index = _check_cache(cache, "cache")
    shape = _check_rows(k, "k", index, D)
    vshape = _check_rows(v, "v", index, D)
    B, S, heads, _ = shape
    if heads != Hk or vshape[2] != Hk:
        raise ValueError(f"k and v have {heads} and {vshape[2]} heads, the cache {Hk}")
    if shape != vshape:
        raise ValueError(f"k and v shapes differ: {tuple(shape)} vs {tuple(vshape)}")
    start, start_at = _ints(start, B, index, "start")
    num, num_at = _ints(num, B, index, "num")
    slots, slots_at = _ints(slots, B, index, "slots")
    if B == 0 or S == 0:
        return
    k, k_at, k_strides = _rows(k)
    v, v_at, v_strides = _rows(v)
    _lib.launch(cache.k.device, _lib.lib().vx_kv_write_fwd, k_at, v_at, k_strides, v_strides, cache.k.data_ptr(),
                cache.v.data_ptr(), cache.k_scale.data_ptr(), cache.v_scale.data_ptr(), n_slots, cap, start_at, num_at,
                slots_at, B, S, Hk, D)


def kv_cache_read(cache: KVCache, length: int, start=None, *, slots=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(k, v), each (B, length, num_kv_heads, head_dim) bf16: positions start[b]
    .. start[b] + length - 1 of slot slots[b], as they are stored, rounded to bf16
    (which holds all such values of magnitudes 2^-126 to below 2^128). B is the length of
    `slots`, else of `start`, else the number of slots; defaults as in
    kv_cache_write. Positions outside the cache give zeros."""
    n_slots, Hk, cap, D, index = _check_cache(cache, "cache")
    length = int(length)
    if length < 0:
        raise ValueError(f"length must be >= 0; got {length}")
    dev = cache.k.device
    items = slots if slots is not None else start
    B = n_slots if items is None else (items if isinstance(items, torch.Tensor) else torch.as_tensor(items)).numel()
    start, start_at = _ints(start, B, index, "start")
    slots, slots_at = _ints(slots, B, index, "slots")
    k = torch.empty((B, length, Hk, D), dtype=torch.bfloat16, device=dev)
    v = torch.empty_like(k)
    if B == 0 or length == 0:
        return k, v
    _lib.launch(dev, _lib.lib().vx_kv_read_fwd, cache.k.data_ptr(), cache.v.data_ptr(), cache.k_scale.data_ptr(),
                cache.v_scale.data_ptr(), n_slots, cap, start_at, slots_at, B, length, Hk, D, k.data_ptr(),
                v.data_ptr())
    return k, v


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(device_index: int, *sizes: int) -> int:
    with torch.cuda.device(device_index):
        return max(int(_lib.lib().vx_cached_attn_workspace_size(*sizes)), 0)  # (sizes it refuses: the launch says why)


def _attend(q: torch.Tensor, cache: KVCache, prefix: Optional[KVCache], kv_len, prefix_len, q_len, slots,
            causal: bool, scale: Optional[float], out: Optional[torch.Tensor]) -> torch.Tensor:
    n_slots, Hk, cap, D, index = _check_cache(cache, "cache")
    B, Sq, H, _ = shape = _check_rows(q, "q", index, D)
    kv_len, kv_len_at = _ints(kv_len, B, index, "kv_len")
    q_len, q_len_at = _ints(q_len, B, index, "q_len")
    slots, slots_at = _ints(slots, B, index, "slots")
    n_prefix = p_cap = 0
    p_k = p_v = p_ks = p_vs = p_len_at = None
    if prefix is not None:
        n_prefix, p_heads, p_cap, p_dim, p_index = _check_cache(prefix, "prefix")
        if p_heads != Hk or p_dim != D or p_index != index:
            raise ValueError("prefix and cache must agree on heads, head dim and device")
        prefix_len, p_len_at = _ints(prefix_len, n_prefix, index, "prefix_len")
        p_k, p_v, p_ks, p_vs = (prefix.k.data_ptr(), prefix.v.data_ptr(), prefix.k_scale.data_ptr(),
                                prefix.v_scale.data_ptr())
    dev = q.device
    empty = B == 0 or Sq == 0 or H == 0
    if not empty:
        q, q_at, q_strides = _rows(q)
    out_strides = None
    if out is None:
        out = torch.empty_like(q) if not empty and q_strides is None else torch.empty(shape, dtype=q.dtype, device=dev)
    elif out.shape != shape or out.dtype != q.dtype or out.stride(-1) != 1 or out.device != dev:
        raise ValueError("out must be a (B, Sq, H, D) bf16 tensor with a contiguous head dim, on q's device")
    elif out.is_neg() or any(st == 0 and n > 1 for st, n in zip(out.stride(), shape)):
        raise ValueError("out must be a tensor that holds its values as they are, each in memory of its own")
    else:
        out_strides = _strides3(out)
    if empty:
        return out
    ws_bytes = _workspace_bytes(index, cap, n_prefix, p_cap, B, Sq, H, Hk, D,
                                int(not causal and q_len is None))
    ws = ws_at = None
    if ws_bytes > 0:
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
        ws_at = ws.data_ptr()
    _lib.launch(dev, _lib.lib().vx_cached_attn_fwd, q_at, out.data_ptr(), q_strides, out_strides, cache.k.data_ptr(),
                cache.v.data_ptr(), cache.k_scale.data_ptr(), cache.v_scale.data_ptr(), n_slots, cap, p_k, p_v, p_ks,
                p_vs, n_prefix, p_cap, kv_len_at, q_len_at, slots_at, p_len_at, B, Sq, H, Hk, D, 1 if causal else 0,
                D ** -0.5 if scale is None else float(scale), ws_at, ws_bytes)
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
