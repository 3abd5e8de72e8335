"""The steps of a rollout or a decoding loop over the 8-bit key/value cache.

A rollout that makes a video block by block, or a text pathway that makes it token
by token, turns its new queries and keys by their positions, writes the keys and
values to the cache, and attends over what the cache holds. (The reference's rotary
tables cover a whole grid from position 0, `src/vidax/core/rope3d.py:45-111`, and
its causal text pathway recomputes all tokens, `src/vidax/models/cosmos3/
dit_layers.py:114-135`.)

`apply_axis_rope` turns rows by integer positions per token and axis (time, height,
width), `kv_cache_write_rope` does so to keys on their way into the cache,
`windowed_attention` attends over a sliding window behind a few first tokens, and
`tree_attention` lets drafted tokens see their ancestors only. As in the cache's
other calls, each launches HIP kernels on torch's current stream and never waits for
the GPU; positions, lengths, parents and slots are device tensors, so a captured
graph may be replayed while they change.
"""
from __future__ import annotations

import decimal
import functools
import math
from decimal import Decimal
from typing import NamedTuple, Optional, Sequence

import torch

from . import _lib
from .kv_cache import _MOST, KVCache, _check_cache, _check_rows, _ints, _out_for, _rows

__all__ = ["AxisRope", "create_axis_rope", "apply_axis_rope", "kv_cache_write_rope", "windowed_attention",
           "tree_attention"]


class AxisRope(NamedTuple):
    """How the pairs of a head's channels turn. turns (head_dim / 2,) int64: turns
    per position in units of 2^-64 turns, modulo 2^64 (the tensor's values as
    unsigned ones; 0: the pair stays as it is). axis (head_dim / 2,) int32: the axis
    whose position turns the pair. axes: their number, 1 to 4. halves: pair j is
    channels (j, j + head_dim / 2) rather than (2 j, 2 j + 1)."""
    turns: torch.Tensor
    axis: torch.Tensor
    axes: int
    halves: bool


@functools.lru_cache(maxsize=8)
def _two_pi(digits: int) -> Decimal:
    """2 pi to that many digits: pi / 4 = 4 arctan(1/5) - arctan(1/239) (Machin)."""
    one = 10 ** (digits + 10)

    def arctan_of_inverse(n: int) -> int:
        total, power, k = 0, one // n, 1
        while power:
            total += power // k if k % 4 == 1 else -(power // k)
            power, k = power // (n * n), k + 2
        return total

    return Decimal(8 * (4 * arctan_of_inverse(5) - arctan_of_inverse(239))) / one


def _turns_of(base: float, ladder: Sequence[tuple]) -> list:
    """scale * base^-(n / d) / 2 pi for each (scale, n, d), in units of 2^-64, whole turns
    left out, rounded once: 53 bits of a float would leave position * 2^-56 of a turn, and
    as much times the scale. (n < d, so what is largest are the scale and 1 / base.)"""
    largest = max((abs(scale) for scale, _, _ in ladder), default=0.0)
    # (those of the whole turns, and 20 behind the point, with room for roundings)
    digits = 60 + sum(int(math.log10(x)) + 1 for x in (largest, 1 / max(base, 1e-308)) if x > 1)
    with decimal.localcontext(decimal.Context(prec=digits, rounding=decimal.ROUND_HALF_EVEN, Emin=-99999, Emax=99999,
                                              traps=[])):
        unit, log = Decimal(2 ** 64) / _two_pi(digits), Decimal(base).ln()
        return [int((Decimal(scale) * (log * -n / d).exp() * unit).to_integral_value()) % 2 ** 64
                for scale, n, d in ladder]


def create_axis_rope(head_dim: int, split: Sequence[int], base: float = 10000.0, *, shared: bool = False,
                     halves: bool = False, axis_scale: Optional[Sequence[float]] = None, device=None) -> AxisRope:
    """The turns of a head whose channels are split over axes: split[a] channels
    (an even number) to axis a, in order; channels past their sum do not turn.

    Pair i of an axis's own ones turns by position * base^(-2 i / split[a]) radians
    (the ladder of create_rope3d_freqs and create_abs_rope3d_freqs); shared: pair j
    of the head by position * base^(-2 j / head_dim). axis_scale: a factor of each
    axis's positions (frames per second, a coarser grid). halves as in AxisRope
    (default: adjacent channels, as in apply_rope3d). The turns are rounded once, to
    the nearest 2^-64 of a turn: at any position the angle is that of base and
    axis_scale, as the numbers they are, to within 2^-34 of a turn.
    """
    if head_dim not in (64, 128):
        raise NotImplementedError(f"head_dim {head_dim} is not supported (64 and 128 are)")
    split = [int(d) for d in split]
    if not 1 <= len(split) <= 4:
        raise NotImplementedError(f"{len(split)} axes are not supported (1 to 4 are)")
    if any(d < 0 or d % 2 for d in split) or sum(split) > head_dim:
        raise ValueError(f"split {split} must be even numbers of at most head_dim {head_dim} together")
    scales = [1.0] * len(split) if axis_scale is None else [float(x) for x in axis_scale]
    if len(scales) != len(split) or not all(math.isfinite(x) for x in scales):
        raise ValueError(f"axis_scale must hold {len(split)} finite numbers")
    base = float(base)
    if not (base > 0 and math.isfinite(base)):
        raise ValueError(f"base must be positive and finite; got {base}")
    ladder, axis = [], []
    for a, (channels, scale) in enumerate(zip(split, scales)):
        for i in range(channels // 2):
            ladder.append((scale, 2 * len(ladder), head_dim) if shared else (scale, 2 * i, channels))
            axis.append(a)
    turns = _turns_of(base, ladder)
    still = head_dim // 2 - len(turns)
    turns = [t - 2 ** 64 if t >= 2 ** 63 else t for t in turns] + [0] * still
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else device
    return AxisRope(torch.tensor(turns, dtype=torch.int64, device=device),
                    torch.tensor(axis + [0] * still, dtype=torch.int32, device=device), len(split), bool(halves))


def _check_rope(rope: AxisRope, head_dim: int, index: int):
    """(turns' address, axis's address, number of axes, halves) of a rope that goes
    with rows of this head dim on this device."""
    if not isinstance(rope, AxisRope):
        raise TypeError("rope must be an AxisRope")
    turns, axis, axes, halves = rope
    try:
        if (turns.dtype is torch.int64 and axis.dtype is torch.int32 and
                turns.shape == axis.shape == (head_dim // 2,) and turns.get_device() == index and
                axis.get_device() == index and turns.is_contiguous() and axis.is_contiguous()):
            return turns.data_ptr(), axis.data_ptr(), int(axes), int(bool(halves))
    except AttributeError:
        pass
    # what is wrong
    for name, t, dtype in (("turns", turns, torch.int64), ("axis", axis, torch.int32)):
        if not isinstance(t, torch.Tensor) or t.dtype != dtype:
            raise TypeError(f"rope.{name} must be a tensor of {dtype}")
        if t.shape != (head_dim // 2,):
            raise ValueError(f"rope.{name} has shape {tuple(t.shape)}, a head of {head_dim} channels has "
                             f"{head_dim // 2} pairs")
        if t.get_device() != index or not t.is_contiguous():
            raise ValueError(f"rope.{name} must be contiguous and on the rows' device")
    raise ValueError("rope is not an AxisRope that the kernels take")


def _positions(positions, batch: int, seq: int, axes: int, index: int):
    """(positions as the kernels read them, their address, their C ABI strides)."""
    if (isinstance(positions, torch.Tensor) and positions.shape == (batch, seq, axes) and
            positions.dtype is torch.int32 and positions.get_device() == index):
        if positions.is_contiguous():
            return positions, positions.data_ptr(), None
    else:
        if not isinstance(positions, torch.Tensor):
            positions = torch.as_tensor(positions)
        shape = positions.shape
        if shape not in ((batch, seq, axes), (seq, axes)):
            raise ValueError(f"positions must be ({batch}, {seq}, {axes}) or ({seq}, {axes}); got {tuple(shape)}")
        if not (positions.dtype is torch.int32 and positions.get_device() == index):
            positions = _ints(positions, positions.numel(), index, "positions")[0].reshape(shape)
        positions = positions.expand(batch, seq, axes)
    return positions, positions.data_ptr(), _lib.strides3(positions.stride())


def apply_axis_rope(x: torch.Tensor, positions, rope: AxisRope, *, inverse: bool = False) -> torch.Tensor:
    """Turns every head's pairs of x (B, S, H, D) bf16 by their tokens' positions
    (B, S, axes) int32 (or (S, axes), shared by the batch; any strides): pair j,
    (u, w), becomes (u cos a - w sin a, u sin a + w cos a) with a the pair's turns
    times position[axis[j]]. Returns a new contiguous tensor, turned in fp32 and
    rounded once. D is 64 or 128.

    inverse: by as much the other way. That undoes a turn (cached keys that move to
    other positions), and is its gradient: of x, from that of the output.
    Angles are formed modulo a turn in integers, so far positions turn as exactly as
    near ones; positions past 32 bits are held at its ends.
    """
    if not isinstance(x, torch.Tensor):
        raise TypeError("x must be a torch.Tensor")
    if not x.is_cuda:
        raise ValueError("x must be a GPU tensor")
    index = x.get_device()
    B, S, H, D = shape = _check_rows(x, "x", index, x.shape[-1] if x.dim() else 0)
    if D not in (64, 128):
        raise NotImplementedError(f"head_dim {D} is not supported (64 and 128 are)")
    turns_at, axis_at, axes, halves = _check_rope(rope, D, index)
    positions, positions_at, strides = _positions(positions, B, S, axes, index)
    if B == 0 or S == 0 or H == 0:
        return torch.empty(shape, dtype=x.dtype, device=x.device)
    x, x_at, x_strides = _rows(x)
    out = torch.empty_like(x) if x_strides is None else torch.empty(shape, dtype=x.dtype, device=x.device)
    _lib.launch(out.device, _lib.lib().vx_axis_rope_fwd, x_at, out.data_ptr(), x_strides, positions_at, strides, axes,
                turns_at, axis_at, halves, int(bool(inverse)), B, S, H, D)
    return out


def kv_cache_write_rope(cache: KVCache, k: torch.Tensor, v: torch.Tensor, positions, rope: AxisRope, start=None, *,
                        num=None, slots=None) -> None:
    """kv_cache_write of keys turned as by apply_axis_rope (one pass; turned in fp32
    and rounded once, to the cache's 8 bits) and of values as they are. positions
    (B, S, axes) or (S, axes) are those of the tokens of k, wherever in the cache
    they go; the other arguments as in kv_cache_write."""
    n_slots, Hk, cap, D, index = _check_cache(cache, "cache")
    shape = _check_rows(k, "k", index, D)
    vshape = _check_rows(v, "v", index, D)
    B, S, heads, _ = shape
    if heads != Hk or vshape[2] != Hk:
        raise ValueError(f"k and v have {heads} and {vshape[2]} heads, the cache {Hk}")
    if shape != vshape:
        raise ValueError(f"k and v shapes differ: {tuple(shape)} vs {tuple(vshape)}")
    turns_at, axis_at, axes, halves = _check_rope(rope, D, index)
    positions, positions_at, strides = _positions(positions, B, S, axes, index)
    start, start_at = _ints(start, B, index, "start")
    num, num_at = _ints(num, B, index, "num")
    slots, slots_at = _ints(slots, B, index, "slots")
    if B == 0 or S == 0:
        return
    k, k_at, k_strides = _rows(k)
    v, v_at, v_strides = _rows(v)
    _lib.launch(cache.k.device, _lib.lib().vx_kv_write_rope_fwd, k_at, v_at, k_strides, v_strides,
                cache.k.data_ptr(), cache.v.data_ptr(), cache.k_scale.data_ptr(), cache.v_scale.data_ptr(), n_slots,
                cap, start_at, num_at, slots_at, positions_at, strides, axes, turns_at, axis_at, halves, B, S, Hk, D)


@functools.lru_cache(maxsize=1024)
def _window_bytes(device_index: int, *sizes: int) -> int:
    with torch.cuda.device(device_index):
        return max(int(_lib.lib().vx_window_attn_workspace_size(*sizes)), 0)  # (what it refuses: the launch says why)


@functools.lru_cache(maxsize=1024)
def _tree_bytes(device_index: int, *sizes: int) -> int:
    with torch.cuda.device(device_index):
        return max(int(_lib.lib().vx_tree_attn_workspace_size(*sizes)), 0)


def _attend_args(q: torch.Tensor, cache: KVCache, kv_len, q_len, slots, out: Optional[torch.Tensor]):
    """What windowed_attention and tree_attention have alike: (sizes, tensors that
    the call reads, output, the C ABI's arguments up to slots). Where there is
    nothing to compute, the arguments are None."""
    n_slots, Hk, cap, D, index = _check_cache(cache, "cache")
    B, Sq, H, _ = shape = _check_rows(q, "q", index, D)
    kv_len, kv_len_at = _ints(kv_len, B, index, "kv_len")
    q_len, q_len_at = _ints(q_len, B, index, "q_len")
    slots, slots_at = _ints(slots, B, index, "slots")
    dev = q.device
    sizes = (index, cap, B, Sq, H, Hk, D)
    if B == 0 or Sq == 0 or H == 0:
        return sizes, None, _out_for(out, shape, dev, None)[0], None
    q, q_at, q_strides = _rows(q)
    out, out_strides = _out_for(out, shape, dev, q if q_strides is None else None)
    k, v, ks, vs = cache
    return sizes, (q, kv_len, q_len, slots), out, (q_at, out.data_ptr(), q_strides, out_strides, k.data_ptr(),
                                                   v.data_ptr(), ks.data_ptr(), vs.data_ptr(), n_slots, cap,
                                                   kv_len_at, q_len_at, slots_at)


def _workspace(nbytes: int, dev: torch.device):
    """(a workspace, its address), or (None, None)."""
    if nbytes == 0:
        return None, None
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    return ws, ws.data_ptr()


def windowed_attention(q: torch.Tensor, cache: KVCache, kv_len=None, *, window: int, sinks: int = 0, q_len=None,
                       slots=None, causal: bool = True, scale: Optional[float] = None,
                       out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """cached_attention whose queries see the last `window` tokens up to theirs and
    the first `sinks` ones; returns (B, Sq, H, D) bf16.

    causal: query i of q_len sits at position p = kv_len - q_len + i and sees
    positions p - window + 1 .. p and, of 0 .. sinks - 1, those up to p (single
    tokens, prompts in chunks). False: the queries are one block whose tokens see
    each other: all of them see the last `window` of the kv_len tokens, their own
    among them, and the first `sinks` (a block of a rollout over the frames before
    it). What the cache holds at positions that no query sees may be anything, as
    past kv_len. The other arguments, lengths outside their range, queries without a
    visible key and rows of scale NaN are as in cached_attention.
    """
    window, sinks = int(window), int(sinks)
    if window < 1 or sinks < 0:
        raise ValueError(f"window ({window}) must be >= 1 and sinks ({sinks}) >= 0")
    window, sinks, causal = min(window, _MOST), min(sinks, _MOST), 1 if causal else 0  # (more than any cache holds)
    sizes, held, out, args = _attend_args(q, cache, kv_len, q_len, slots, out)
    if args is not None:
        index, cap, B, Sq, H, Hk, D = sizes
        nbytes = _window_bytes(index, cap, B, Sq, H, Hk, D, window, sinks, causal)
        ws, ws_at = _workspace(nbytes, out.device)
        _lib.launch(out.device, _lib.lib().vx_window_attn_fwd, *args, B, Sq, H, Hk, D, window, sinks, causal,
                    D ** -0.5 if scale is None else float(scale), ws_at, nbytes)
    return out


def tree_attention(q: torch.Tensor, cache: KVCache, parents, kv_len=None, *, q_len=None, slots=None,
                   scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """cached_attention of drafted tokens that form a tree; returns (B, Sq, H, D) bf16.

    The last q_len of an item's kv_len cached tokens are drafted (write them first),
    and the queries are theirs, in the same order. parents (B, Sq) int32 (or (Sq,),
    one tree for all items): the drafted token that a drafted token follows, an
    earlier one; any value that is not 0 .. i - 1 stands for none: such a token
    follows the last one in front of the drafted ones. Query i sees all tokens in
    front of the drafted ones, its ancestors and itself. Sq is at most 512; with
    parents i - 1 this is cached_attention. The other arguments, lengths outside
    their range, queries without a visible key and rows of scale NaN are as there.
    """
    if parents is None:
        raise TypeError("parents must hold integers")
    sizes, held, out, args = _attend_args(q, cache, kv_len, q_len, slots, out)
    index, cap, B, Sq, H, Hk, D = sizes
    shape = parents.shape if isinstance(parents, torch.Tensor) else torch.as_tensor(parents).shape
    if shape != (B, Sq) and shape != (Sq,):
        raise ValueError(f"parents must be ({B}, {Sq}) or ({Sq},); got {tuple(shape)}")
    one = len(shape) == 1
    parents, parents_at = _ints(parents, Sq if one else B * Sq, index, "parents")
    if args is not None:
        nbytes = _tree_bytes(index, cap, B, Sq, H, Hk, D)
        ws, ws_at = _workspace(nbytes, out.device)
        _lib.launch(out.device, _lib.lib().vx_tree_attn_fwd, *args, parents_at, 0 if one else Sq, B, Sq, H, Hk, D,
                    D ** -0.5 if scale is None else float(scale), ws_at, nbytes)
    return out
