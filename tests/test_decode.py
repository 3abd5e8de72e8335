"""Rotary positions on several axes, and attention over the 8-bit cache with a
sliding window or of a tree of drafted tokens.

Attention is compared with the oracle (64 bits, on the stored values) under the bound
that tests/test_kv_cache.py derives from what the kernels round. A turned value
y = u c - w s is off by at most
  2^-20 (|u| + |w|)   sine and cosine (2^-21 each) and the fp32 products and sum
  2^-8 |y|            the output to bf16
before it is stored in 8 bits: half a step of e4m3 and the first of these.
"""
import ctypes
import decimal
import math
import os
import re
from decimal import Decimal as D_

import numpy as np
import pytest
import torch

import vidax_amd as vx
from oracle import cache_oracle as CO
from oracle import decode_oracle as O
from vidax_amd import _lib

A = 1 << 20  # a 16-byte aligned fake device address (never dereferenced)
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
INVALID, UNSUPPORTED = _lib.VX_ERR_INVALID_ARGUMENT, _lib.VX_ERR_UNSUPPORTED


# ------------------------------------------------------------------ refusals (CPU)
def test_decode_symbols_are_exported():
    text = open(os.path.join(os.path.dirname(__file__), "..", "include", "vx_decode.h")).read()
    names = set(re.findall(r"\b(vx_\w+)\s*\(", re.sub(r"/\*.*?\*/", "", text, flags=re.S)))
    assert names == set(_lib.DECODE_SYMBOLS)
    assert all(hasattr(_lib.lib(), n) for n in names)
    assert _lib.lib().vx_decode_abi_version() == 10000


def _s3(s):
    return None if s is None else _lib.strides3(s)


def _rope_check(**kw):
    a = dict(x=A, o=A, xst=None, pos=A, pst=(6, 3, 1), axes=3, turns=A, axis=A, halves=0, inverse=0, B=2, S=2, H=3,
             D=128)
    a.update(kw)
    return _lib.lib().vx_axis_rope_check(a["x"], a["o"], _s3(a["xst"]), a["pos"], _s3(a["pst"]), a["axes"],
                                         a["turns"], a["axis"], a["halves"], a["inverse"], a["B"], a["S"], a["H"],
                                         a["D"])


def _write_check(**kw):
    a = dict(k=A, v=A, kst=None, vst=None, ck=A, cv=A, ks=A, vs=A, slots_n=4, cap=128, start=None, num=None,
             slots=None, pos=A, pst=(6, 3, 1), axes=3, turns=A, axis=A, halves=0, B=2, S=3, Hk=2, D=64)
    a.update(kw)
    return _lib.lib().vx_kv_write_rope_check(
        a["k"], a["v"], _s3(a["kst"]), _s3(a["vst"]), a["ck"], a["cv"], a["ks"], a["vs"], a["slots_n"], a["cap"],
        a["start"], a["num"], a["slots"], a["pos"], _s3(a["pst"]), a["axes"], a["turns"], a["axis"], a["halves"],
        a["B"], a["S"], a["Hk"], a["D"])


ATTN_ARGS = dict(q=A, o=A, qst=None, ost=None, ck=A, cv=A, ks=A, vs=A, slots_n=4, cap=128, kv_len=None, q_len=None,
                 slots=None, B=2, S=3, H=4, Hk=2, D=64, scale=0.125)


def _window_check(**kw):
    a = dict(ATTN_ARGS, window=5, sinks=1, causal=1)
    a.update(kw)
    return _lib.lib().vx_window_attn_check(
        a["q"], a["o"], _s3(a["qst"]), _s3(a["ost"]), a["ck"], a["cv"], a["ks"], a["vs"], a["slots_n"], a["cap"],
        a["kv_len"], a["q_len"], a["slots"], a["B"], a["S"], a["H"], a["Hk"], a["D"], a["window"], a["sinks"],
        a["causal"], ctypes.c_float(a["scale"]))


def _tree_check(**kw):
    a = dict(ATTN_ARGS, parents=A, pstride=3)
    a.update(kw)
    return _lib.lib().vx_tree_attn_check(
        a["q"], a["o"], _s3(a["qst"]), _s3(a["ost"]), a["ck"], a["cv"], a["ks"], a["vs"], a["slots_n"], a["cap"],
        a["kv_len"], a["q_len"], a["slots"], a["parents"], a["pstride"], a["B"], a["S"], a["H"], a["Hk"], a["D"],
        ctypes.c_float(a["scale"]))


def test_checks_accept_valid_arguments():
    assert _rope_check() == _rope_check(pst=None) == _lib.VX_OK
    assert _rope_check(pst=(0, 1, 0), axes=4, D=64, xst=(8, 8, 8), halves=1, inverse=1) == _lib.VX_OK
    assert _write_check() == _write_check(slots=A, B=9, pst=(0, 0, 0), halves=1) == _lib.VX_OK
    assert _window_check() == _window_check(window=2 ** 31 - 1, sinks=2 ** 31 - 1, causal=0) == _lib.VX_OK
    assert _tree_check() == _tree_check(S=512, pstride=0) == _lib.VX_OK
    assert _lib.last_error() == ""


ROPE = [
    (dict(pos=None), INVALID, "non-NULL"),
    (dict(turns=None), INVALID, "non-NULL"),
    (dict(axis=None), INVALID, "non-NULL"),
    (dict(pos=A + 2), INVALID, "aligned"),
    (dict(turns=A + 4), INVALID, "aligned"),
    (dict(axis=A + 1), INVALID, "aligned"),
    (dict(axes=0), UNSUPPORTED, "num_axes"),
    (dict(axes=5), UNSUPPORTED, "num_axes"),
    (dict(halves=2), INVALID, "halves"),
    (dict(pst=(6, -1, 1)), INVALID, "position_strides"),
    (dict(D=96), UNSUPPORTED, "head_dim"),
    (dict(B=0), INVALID, "batch"),
    (dict(B=65536, slots=A), INVALID, "batch"),
    (dict(S=0), INVALID, "seq"),
]
ATTN = [
    (dict(q=None), INVALID, "non-NULL"),
    (dict(o=A + 8), INVALID, "aligned"),
    (dict(ck=None), INVALID, "non-NULL"),
    (dict(vs=A + 4), INVALID, "aligned"),
    (dict(cap=100), INVALID, "capacity"),
    (dict(D=80), UNSUPPORTED, "head_dim"),
    (dict(B=5), INVALID, "slots"),
    (dict(S=0), INVALID, "seq"),
    (dict(H=5), INVALID, "multiple of num_kv_heads"),
    (dict(scale=0.0), INVALID, "scale"),
    (dict(qst=(8, 8, 4)), INVALID, "multiple of 8"),
    (dict(kv_len=A + 2), INVALID, "4-byte"),
]


@pytest.mark.parametrize("check,kw,code,frag", [(c, *r) for c in (_rope_check, _write_check) for r in ROPE] +
                         [(c, *r) for c in (_window_check, _tree_check) for r in ATTN] + [
    (_rope_check, dict(x=None), INVALID, "non-NULL"),
    (_rope_check, dict(o=A + 8), INVALID, "aligned"),
    (_rope_check, dict(xst=(8, 8, 4)), INVALID, "multiple of 8"),
    (_rope_check, dict(H=0), INVALID, "num_heads"),
    (_rope_check, dict(inverse=2), INVALID, "inverse"),
    (_write_check, dict(k=None), INVALID, "non-NULL"),
    (_write_check, dict(vst=(8, -8, 8)), INVALID, "negative"),
    (_write_check, dict(cap=65), INVALID, "capacity"),
    (_write_check, dict(B=5), INVALID, "slots"),
    (_window_check, dict(window=0), INVALID, "window"),
    (_window_check, dict(sinks=-1), INVALID, "sinks"),
    (_window_check, dict(causal=2), INVALID, "causal"),
    (_window_check, dict(S=2 ** 30), UNSUPPORTED, "too many"),
    (_tree_check, dict(S=513), UNSUPPORTED, "drafted"),
    (_tree_check, dict(parents=None), INVALID, "parents"),
    (_tree_check, dict(parents=A + 2), INVALID, "parents"),
    (_tree_check, dict(pstride=-1), INVALID, "parents_stride"),
])
def test_checks_refuse(check, kw, code, frag):
    kw = {n: x for n, x in kw.items() if n != "slots" or check is not _rope_check}
    assert check(**kw) == code
    assert frag in _lib.last_error()


@pytest.mark.parametrize("check,fits,refused", [
    (_rope_check, dict(S=2 ** 21, H=31 * 32), dict(S=2 ** 21, H=31 * 32 + 1)),  # 64 threads for 32 heads of a token
    (_write_check, dict(S=2 ** 21, Hk=511), dict(S=2 ** 21, Hk=512)),
    (_window_check, dict(B=1, S=2 ** 22, H=127, Hk=127), dict(B=1, S=2 ** 22, H=128, Hk=128)),
    (_tree_check, dict(B=65535, S=1, H=255, Hk=255, slots=A), dict(B=65535, S=1, H=256, Hk=256, slots=A)),
])
def test_checks_refuse_grids_past_32_bits(check, fits, refused):
    assert check(**fits) == _lib.VX_OK, _lib.last_error()
    assert check(**refused) == UNSUPPORTED and "too" in _lib.last_error()


def test_workspaces_are_of_what_is_seen():
    """A window's ranges and their partial results follow the window, not the
    capacity; sizes that the calls refuse give -1."""
    L = _lib.lib()
    size = lambda cap, window, sinks=0: L.vx_window_attn_workspace_size(cap, 1, 1, 8, 8, 128, window, sinks, 1)
    assert size(131072, 500) == size(1024, 500) == 0 < size(131072, 5000) == size(8192, 5000)
    assert size(131072, 10 ** 9) == size(131072, 2 ** 31 - 1, 2 ** 31 - 1) == \
        L.vx_cached_attn_workspace_size(131072, 0, 0, 1, 1, 8, 8, 128, 0)
    assert L.vx_tree_attn_workspace_size(131072, 1, 1, 8, 8, 128) == size(131072, 10 ** 9)
    assert size(100, 5) == size(128, 0) == size(128, 5, -1) == -1
    assert L.vx_tree_attn_workspace_size(128, 1, 513, 8, 8, 128) == -1


def test_injected_error_is_reported():
    L = _lib.lib()
    L.vx_debug_inject_error(_lib.VX_ERR_LAUNCH)
    s = _lib.strides3((6, 3, 1))
    try:
        assert L.vx_axis_rope_fwd(A, A, None, A, s, 3, A, A, 0, 0, 2, 2, 3, 128, None) == _lib.VX_ERR_LAUNCH
        assert L.vx_kv_write_rope_fwd(A, A, None, None, A, A, A, A, 4, 128, None, None, None, A, s, 3, A, A, 0, 2, 3,
                                      2, 64, None) == _lib.VX_ERR_LAUNCH
        f = ctypes.c_float(0.1)
        assert L.vx_window_attn_fwd(A, A, None, None, A, A, A, A, 4, 128, None, None, None, 2, 3, 4, 2, 64, 5, 1, 1, f,
                                    A, 1 << 40, None) == _lib.VX_ERR_LAUNCH
        assert L.vx_tree_attn_fwd(A, A, None, None, A, A, A, A, 4, 128, None, None, None, A, 3, 2, 3, 4, 2, 64, f, A,
                                  1 << 40, None) == _lib.VX_ERR_LAUNCH
        assert "injected" in _lib.last_error()
    finally:
        L.vx_debug_inject_error(0)


def test_turning_in_place_needs_contiguous_rows():
    """out is written contiguously: where x is the same memory at other strides, rows
    would be overwritten before they are read. (Strides of a single item, token or head
    say nothing.) Refused before anything is launched."""
    L, positions = _lib.lib(), _lib.strides3((6, 3, 1))
    call = lambda x, o, st, B=2, S=3, H=4: L.vx_axis_rope_fwd(x, o, _s3(st), A, positions, 3, A, A, 0, 0, B, S, H, 64,
                                                              None)
    L.vx_debug_inject_error(_lib.VX_ERR_LAUNCH)  # (what is not refused)
    try:
        for st in ((0, 256, 64), (768, 0, 64), (768, 256, 0), (768, 64, 192), (2304, 768, 64), (256, 512, 64)):
            assert call(A, A, st) == INVALID, st
            assert "in-place" in _lib.last_error()
            assert call(A, A + (1 << 20), st) == _lib.VX_ERR_LAUNCH
        for sizes, st in ((dict(), None), (dict(), (768, 256, 64)), (dict(B=1), (8, 256, 64)),
                          (dict(B=1, S=1), (8, 16, 64)), (dict(S=1), (256, 8, 64)), (dict(H=1), (192, 64, 8)),
                          (dict(B=1, S=1, H=1), (0, 0, 0))):
            assert call(A, A, st, **sizes) == _lib.VX_ERR_LAUNCH, (sizes, st)
    finally:
        L.vx_debug_inject_error(0)


def test_a_missing_workspace_is_refused():
    L, f = _lib.lib(), ctypes.c_float(0.1)
    for ws, n in ((None, 1 << 40), (A + 4, 1 << 40), (A, 16)):
        assert L.vx_window_attn_fwd(A, A, None, None, A, A, A, A, 4, 8192, None, None, None, 2, 1, 4, 2, 64, 5000, 1, 1,
                                    f, ws, n, None) == INVALID
        assert "workspace" in _lib.last_error()
        assert L.vx_tree_attn_fwd(A, A, None, None, A, A, A, A, 4, 8192, None, None, None, A, 3, 2, 1, 4, 2, 64, f, ws,
                                  n, None) == INVALID
        assert "workspace" in _lib.last_error()


# ------------------------------------------------------------------ the turns
@pytest.mark.parametrize("D,split,shared", [(128, (44, 42, 42), False), (128, (32, 48, 48), True),
                                            (64, (16, 16, 16), False), (64, (64,), False),
                                            (64, (8, 0, 24, 32), True)])
@pytest.mark.parametrize("base,scale", [(10000.0, None), (5e6, (0.25, 1.0, 3.0, 1e6))])
def test_turns_are_the_ladders(D, split, shared, base, scale):
    """turns / 2^64 is scale * base^-e / 2 pi modulo 1, as far as 64 bits tell."""
    scale = None if scale is None else scale[:len(split)]
    rope = vx.create_axis_rope(D, split, base, shared=shared, halves=True, axis_scale=scale, device="cpu")
    assert rope.axes == len(split) and rope.halves and rope.turns.shape == rope.axis.shape == (D // 2,)
    at = 0
    for a, channels in enumerate(split):
        for i in range(channels // 2):
            e = 2 * at / D if shared else 2 * i / channels
            want = (1.0 if scale is None else scale[a]) * base ** -e / (2 * math.pi)
            got = (int(rope.turns[at]) % 2 ** 64) / 2.0 ** 64
            off = (got - want) % 1.0
            assert min(off, 1 - off) <= 2.0 ** -51 * max(1.0, want) and int(rope.axis[at]) == a
            at += 1
    assert (rope.turns[at:] == 0).all()


def _pi(digits):
    """By the arithmetic-geometric mean (Gauss and Legendre), in a context of that precision."""
    a, b, t, p = D_(1), 1 / D_(2).sqrt(), D_(1) / 4, D_(1)
    for _ in range(digits.bit_length() + 2):
        a, b, t, p = (a + b) / 2, (a * b).sqrt(), t - p * ((a - b) / 2) ** 2, 2 * p
    return (a + b) ** 2 / (4 * t)


@pytest.mark.parametrize("D,split,shared", [(128, (44, 42, 42), False), (64, (64,), False), (64, (8, 0, 24, 32), True)])
@pytest.mark.parametrize("base,scale", [(10000.0, None), (5e6, (24.0, 1.0, 0.1, 1e6)), (500000.0, (-1 / 3, 24, 1e-9, 7)),
                                        (1e-300, (1.0, 2.0, 3.0, 4.0)), (1.5e308, (1e300, -1e308, 5e-324, 2.0 ** 80))])
def test_turns_are_rounded_once(D, split, shared, base, scale):
    """turns is scale * base^-e / 2 pi modulo 1 to the nearest of 2^64 steps: base and
    scale are taken as the numbers they are, so positions of 2^31 are off by 2^-34 of a
    turn at most whatever the scale."""
    scale = (1.0,) * len(split) if scale is None else scale[:len(split)]
    rope = vx.create_axis_rope(D, split, base, shared=shared, axis_scale=scale, device="cpu")
    digits = 120 if 1 < base < 1e9 else 800
    with decimal.localcontext(decimal.Context(prec=digits, traps=[])):
        two_pi, at = 2 * _pi(digits), 0
        for a, channels in enumerate(split):
            for i in range(channels // 2):
                e = D_(2 * at) / D if shared else D_(2 * i) / channels
                want = D_(scale[a]) * D_(base) ** -e / two_pi * 2 ** 64
                off = (int(rope.turns[at]) - want) % 2 ** 64  # (Decimal's remainder keeps the sign)
                off = min(abs(off), 2 ** 64 - abs(off))
                assert off <= D_("0.5000001"), (at, off)
                at += 1
    assert (rope.turns[at:] == 0).all()


def test_create_axis_rope_refuses():
    make = lambda *a, **kw: vx.create_axis_rope(*a, device="cpu", **kw)
    with pytest.raises(NotImplementedError, match="head_dim"):
        make(96, (96,))
    with pytest.raises(NotImplementedError, match="axes"):
        make(64, ())
    with pytest.raises(NotImplementedError, match="axes"):
        make(64, (2,) * 5)
    for split in ((3, 3), (-2, 4), (64, 2)):
        with pytest.raises(ValueError, match="split"):
            make(64, split)
    for scale in ((1.0,), (1.0, math.inf)):
        with pytest.raises(ValueError, match="axis_scale"):
            make(64, (2, 2), axis_scale=scale)
    for base in (0.0, -1.0, math.nan, math.inf):
        with pytest.raises(ValueError, match="base"):
            make(64, (2, 2), base)


def test_python_refusals_on_the_host():
    c = vx.create_kv_cache(1, 64, 1, 64, device="cpu")
    q = torch.zeros((1, 1, 1, 64), dtype=torch.bfloat16)
    rope = vx.create_axis_rope(64, (16, 16), device="cpu")
    p = torch.zeros((1, 1, 2), dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU tensor"):
        vx.apply_axis_rope(q, p, rope)
    with pytest.raises(TypeError, match="torch.Tensor"):
        vx.apply_axis_rope([1.0], p, rope)
    for call in (lambda: vx.kv_cache_write_rope(c, q, q, p, rope), lambda: vx.windowed_attention(q, c, window=4),
                 lambda: vx.tree_attention(q, c, [-1])):
        with pytest.raises(ValueError, match="GPU tensor"):
            call()
    for call in (lambda: vx.kv_cache_write_rope(tuple(c), q, q, p, rope),
                 lambda: vx.windowed_attention(q, tuple(c), window=4), lambda: vx.tree_attention(q, tuple(c), [-1])):
        with pytest.raises(TypeError, match="cache must be a KVCache"):
            call()
    for window, sinks in ((0, 0), (-1, 0), (1, -1)):
        with pytest.raises(ValueError, match="window"):
            vx.windowed_attention(q, c, window=window, sinks=sinks)
    with pytest.raises(TypeError, match="parents"):
        vx.tree_attention(q, c, None)


def test_oracle_sees():
    assert O.window_sees(6, 2, 2, 1, True).astype(int).tolist() == [[1, 0, 0, 1, 1, 0], [1, 0, 0, 0, 1, 1]]
    assert O.window_sees(5, 2, 2, 1, False).astype(int).tolist() == [[1, 0, 0, 1, 1]] * 2
    assert O.window_sees(2, 4, 9, 9, True).astype(int).tolist() == [[0, 0], [0, 0], [1, 0], [1, 1]]
    assert O.tree_sees(5, 3, [-1, 0, 0]).astype(int).tolist() == [[1, 1, 1, 0, 0], [1, 1, 1, 1, 0], [1, 1, 1, 0, 1]]
    assert O.tree_sees(4, 4, [-1, 0, 7, 1]).astype(int).tolist() == [[1, 0, 0, 0], [1, 1, 0, 0], [0, 0, 1, 0],
                                                                     [1, 1, 0, 1]]
    assert O.tree_sees(2, 3, [-1, 0, 1]).astype(int).tolist() == [[0, 0], [1, 0], [1, 1]]


# ------------------------------------------------------------------ turning on the GPU
def _bf16(x, gpu):
    return torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(gpu).to(torch.bfloat16)


def _ints(x, gpu):
    return None if x is None else torch.tensor(x, dtype=torch.int32, device=gpu)


def _f64(t):
    return t.double().cpu().numpy()


def _bytes(cache):
    return [t.view(torch.uint8).cpu().numpy() for t in cache]


def _assert_turned(got, x, positions, rope, inverse=False):
    y, size = O.axis_rope(_f64(x), positions, rope.turns.tolist(), rope.axis.tolist(), rope.halves, inverse)
    tol = 2.0 ** -8 * np.abs(y) + 2.0 ** -20 * size
    err = np.abs(_f64(got) - y)
    at = np.unravel_index(np.argmax(err - tol), err.shape)
    assert (err <= tol).all(), (at, err[at], tol[at], y[at])


TURNS = [
    # B, S, H, D, split, shared, far
    (1, 1, 1, 64, (64,), False, 10),
    (1, 1, 1, 128, (44, 42, 42), False, 100),
    (8, 1, 32, 128, (32, 48, 48), True, 2 ** 31 - 1),
    (2, 5, 3, 64, (16, 16, 16), False, 2 ** 20),
    (1, 33, 9, 128, (128,), False, 2 ** 31 - 1),
    (3, 7, 40, 128, (44, 42, 42), False, 50),
    (1, 3, 71, 64, (8, 0, 24, 32), True, 1000),
    (2, 130, 33, 64, (24, 20, 20), False, 50),
    (1, 2, 130, 128, (2, 4), False, 2 ** 16),
]


@pytest.mark.gpu
@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("case", TURNS, ids=[str(c) for c in TURNS])
def test_apply_axis_rope(gpu, case, inverse, halves):
    B, S, H, D, split, shared, far = case
    print(f"[case] apply_axis_rope {case} inverse={inverse} halves={halves}", flush=True)
    rng = np.random.default_rng(B * S + H)
    rope = vx.create_axis_rope(D, split, shared=shared, halves=halves, device=gpu)
    x = _bf16(rng.standard_normal((B, S, H, D)) * np.exp(2 * rng.standard_normal((B, S, H, 1))), gpu)
    positions = rng.integers(-far - 1, far + 1, (B, S, len(split)))
    got = vx.apply_axis_rope(x, _ints(positions.tolist(), gpu), rope, inverse=inverse)
    assert _lib.last_launch() == f"axis_rope_kernel<{D}, {'halves' if halves else 'adjacent'}>"
    assert got.shape == x.shape and got.is_contiguous()
    _assert_turned(got, x, positions, rope, inverse)


@pytest.mark.gpu
def test_turning_at_every_eighth(gpu):
    """Angles at and beside the borders of the quarters, and those that are whole
    quarters exactly: (u, w) turned by n quarters is what swapping and negating gives."""
    turns = [(n * 2 ** 61 + d) % 2 ** 64 for n in range(8) for d in (-(2 ** 32), -1, 0, 1, 2 ** 31, 2 ** 32)]
    turns = (turns + [0] * 64)[:64]
    signed = [t - 2 ** 64 if t >= 2 ** 63 else t for t in turns]
    rope = vx.AxisRope(torch.tensor(signed, device=gpu), _ints([0] * 64, gpu), 1, True)
    x = _bf16(np.random.default_rng(2).standard_normal((1, 3, 2, 128)), gpu)
    got = vx.apply_axis_rope(x, _ints([[[0], [1], [-1]]], gpu), rope)
    assert torch.equal(got[:, 0], x[:, 0])
    _assert_turned(got, x, np.array([[[0], [1], [-1]]]), rope)
    quarters = [j for j, t in enumerate(turns) if t % 2 ** 62 == 0]
    u, w = _f64(x)[0, 1, :, :64], _f64(x)[0, 1, :, 64:]
    y = _f64(got)[0, 1]
    for j in quarters:
        n = turns[j] // 2 ** 62
        c, s = ((1, 0), (0, 1), (-1, 0), (0, -1))[n]
        assert (y[:, j] == c * u[:, j] - s * w[:, j]).all() and (y[:, 64 + j] == s * u[:, j] + c * w[:, j]).all()


@pytest.mark.gpu
def test_positions_and_rows_of_any_layout(gpu):
    """Positions shared by the batch, by the axes, transposed, of other integer types
    and from the host, and strided rows, give what contiguous int32 ones give."""
    g = torch.Generator(device=gpu).manual_seed(3)
    rope = vx.create_axis_rope(64, (16, 24, 24), device=gpu)
    fused = torch.randn((2, 21, 3, 4, 64), generator=g, device=gpu).bfloat16()
    x = fused[:, :, 1]
    p = torch.randint(0, 900, (2, 21, 3), generator=g, device=gpu, dtype=torch.int32)
    want = vx.apply_axis_rope(x.contiguous(), p, rope)
    odd = torch.zeros(x.numel() + 1, dtype=torch.bfloat16, device=gpu)[1:].reshape(x.shape).copy_(x)
    for rows in (x, odd, x.transpose(1, 2).contiguous().transpose(1, 2),
                 x.transpose(2, 3).contiguous().transpose(2, 3)):
        assert torch.equal(vx.apply_axis_rope(rows, p, rope), want)
    for q in (p.permute(2, 0, 1).contiguous().permute(1, 2, 0), p.long(), p.cpu(), p.to(torch.int16), p.tolist()):
        assert torch.equal(vx.apply_axis_rope(x, q, rope), want)
    shared = p[0]
    want = vx.apply_axis_rope(x, shared[None].repeat(2, 1, 1), rope)
    for q in (shared, shared.cpu(), shared[None].expand(2, 21, 3), shared.tolist()):
        assert torch.equal(vx.apply_axis_rope(x, q, rope), want)
    text = p[..., :1]
    want = vx.apply_axis_rope(x, text.repeat(1, 1, 3), rope)
    assert torch.equal(vx.apply_axis_rope(x, text.expand(2, 21, 3), rope), want)
    far = torch.full((2, 21, 3), 2 ** 40, device=gpu)  # held at 32 bits' end
    assert torch.equal(vx.apply_axis_rope(x, far, rope), vx.apply_axis_rope(x, far.clamp_max(2 ** 31 - 1).int(), rope))
    assert vx.apply_axis_rope(x[:0], p[:0], rope).shape == (0, 21, 4, 64)
    assert vx.apply_axis_rope(x[:, :0], p[:, :0], rope).shape == (2, 0, 4, 64)
    assert vx.apply_axis_rope(x[:, :, :0], p, rope).shape == (2, 21, 0, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("halves", [0, 1])
@pytest.mark.parametrize("B,S,H,D", [(1, 1, 1, 64), (3, 37, 71, 64), (2, 130, 40, 128)])
def test_turning_in_place(gpu, B, S, H, D, halves):
    """The C entry with out = x gives what it gives elsewhere, bit for bit."""
    print(f"[case] in place B={B} S={S} H={H} D={D} halves={halves}", flush=True)
    rope = vx.create_axis_rope(D, (D // 4, D // 4, D // 4), halves=bool(halves), device=gpu)
    g = torch.Generator(device=gpu).manual_seed(S)
    x = torch.randn((B, S, H, D), generator=g, device=gpu).bfloat16()
    p = torch.randint(0, 5000, (B, S, 3), generator=g, device=gpu, dtype=torch.int32)
    want = vx.apply_axis_rope(x, p, rope)
    _lib.launch(x.device, _lib.lib().vx_axis_rope_fwd, x.data_ptr(), x.data_ptr(), None, p.data_ptr(), None, 3,
                rope.turns.data_ptr(), rope.axis.data_ptr(), halves, 0, B, S, H, D)
    assert torch.equal(x, want)


@pytest.mark.gpu
def test_axes_that_are_not_there_do_not_turn(gpu):
    rope = vx.create_axis_rope(64, (32, 32), device=gpu)
    x = torch.randn((1, 5, 2, 64), device=gpu).bfloat16()
    p = torch.randint(1, 99, (1, 5, 2), device=gpu, dtype=torch.int32)
    for value in (2, -1, 2 ** 31 - 1):
        out = vx.apply_axis_rope(x, p, rope._replace(axis=torch.where(rope.axis == 1, value, rope.axis)))
        assert torch.equal(out[..., 32:], x[..., 32:])
        assert torch.equal(out[..., :32], vx.apply_axis_rope(x, p, rope)[..., :32])


@pytest.mark.gpu
@pytest.mark.parametrize("halves", [False, True])
def test_the_gradient_is_the_turn_back(gpu, halves):
    """The gradient of sum(turned * g) is g turned back: against the formula's (its
    matrix transposed, from unit vectors) and against differences, which are exact
    up to rounding, for the turn is linear."""
    D, S = 64, 6
    rope = vx.create_axis_rope(D, (24, 20, 20), halves=halves, device=gpu)
    rng = np.random.default_rng(8)
    p = rng.integers(0, 5000, (1, S, 3))
    positions = _ints(p.tolist(), gpu)
    x, g = (_bf16(rng.standard_normal((1, S, 1, D)), gpu) for _ in range(2))
    back = _f64(vx.apply_axis_rope(g, positions, rope, inverse=True))[0, :, 0]
    turns, axis = rope.turns.tolist(), rope.axis.tolist()
    units = np.broadcast_to(np.eye(D)[None, None], (1, S, D, D))  # head n: unit vector n
    matrix = O.axis_rope(units, p, turns, axis, halves)[0][0]      # [token][n] = the turned unit vector
    want = np.einsum("snd,sd->sn", matrix, _f64(g)[0, :, 0])
    tol = 2.0 ** -8 * np.abs(want) + 2.0 ** -20 * 2 * np.abs(_f64(g)).max()
    assert (np.abs(back - want) <= tol).all()
    # differences of sum(turned * g) for steps of one channel
    h = 4.0
    for n in (0, 1, 31, 32, 63):
        up, down = x.clone(), x.clone()
        up[..., n] = h
        down[..., n] = -h
        gain = _f64(vx.apply_axis_rope(up, positions, rope)) - _f64(vx.apply_axis_rope(down, positions, rope))
        slope = (gain * _f64(g))[0, :, 0].sum(-1) / (2 * h)
        # (two values of the pair change; each of the four is rounded by 2^-8 of at most h + max|x|)
        off = 2 * 2 * 2.0 ** -8 * (h + np.abs(_f64(x)).max()) * np.abs(_f64(g)).max() / (2 * h)
        assert (np.abs(slope - back[:, n]) <= off + 2.0 ** -7 * np.abs(back[:, n])).all()
    # a whole turn and back
    y = vx.apply_axis_rope(vx.apply_axis_rope(x, positions, rope), positions, rope, inverse=True)
    size = np.abs(_f64(x)).max() * math.sqrt(2)
    assert np.abs(_f64(y) - _f64(x)).max() <= (2 * 2.0 ** -8 + 2.0 ** -8) * size


def test_the_grid_tables_are_a_case_of_it():
    """create_rope3d_freqs's tables (fp32 angles) are this rope at grid positions."""
    t, h, w, D = 3, 4, 5, 128
    cos, sin = vx.create_rope3d_freqs(t, h, w, D)
    c = D // 2
    split = tuple(2 * n for n in (c - 2 * (c // 3), c // 3, c // 3))
    rope = vx.create_axis_rope(D, split, device="cpu")
    p = np.stack(np.meshgrid(np.arange(t), np.arange(h), np.arange(w), indexing="ij"), -1).reshape(-1, 3)
    a = O.angles(p, rope.turns.tolist(), rope.axis.tolist())
    # (fp32 angles of at most 4 radians: the power, the division and the product are each half a step off)
    assert np.abs(np.cos(a) - cos[0, :, 0].double().numpy()).max() <= 4 * 4 * 2.0 ** -23
    assert np.abs(np.sin(a) - sin[0, :, 0].double().numpy()).max() <= 4 * 4 * 2.0 ** -23


@pytest.mark.gpu
@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("D", [64, 128])
def test_pairs_that_do_not_turn_keep_their_values(gpu, D, halves):
    """Bit for bit, with infinities, NaN and zeros of either sign beside them: pairs past
    the split at any position, and all pairs at position 0."""
    rope = vx.create_axis_rope(D, (D // 4,), halves=halves, device=gpu)
    x = np.random.default_rng(D).standard_normal((1, 2, 3, D))
    special = np.array([np.inf, -np.inf, np.nan, 0.0, -0.0, 3.0])
    u, w = np.meshgrid(special, special)
    still = [j for j in range(D // 2) if rope.turns[j] == 0]
    assert len(still) == D // 2 - D // 8
    at = lambda j: (j, j + D // 2) if halves else (2 * j, 2 * j + 1)
    for i, (p, q) in enumerate(zip(u.ravel(), w.ravel())):
        x[:, :, i % 3, list(at(still[i // 3]))] = p, q
        x[:, 1, i % 3, list(at(i // 3 % (D // 8)))] = p, q
    x = _bf16(x, gpu)
    for inverse in (False, True):
        y = vx.apply_axis_rope(x, _ints([[123457], [0]], gpu), rope, inverse=inverse)
        assert (x.isnan() == y.isnan()).all(), inverse
        same = (x.view(torch.int16) == y.view(torch.int16)) | x.isnan()
        assert same[:, 1].all(), inverse
        for j in still:
            assert same[:, 0, :, list(at(j))].all(), (inverse, j)


WRITES = [
    # B, S, Hk, D, cap, start, num, slots, split
    (1, 1, 1, 64, 64, None, None, None, (16, 24, 24)),
    (3, 17, 2, 128, 128, [0, 5, 111], None, [2, 0, 3], (44, 42, 42)),
    (2, 33, 3, 64, 128, [1, 95], [33, 20], None, (64,)),
    (4, 50, 1, 64, 64, [30, -10, 64, -60], None, [0, 1, 2, 3], (8, 8, 8, 8)),
    (3, 9, 2, 128, 128, [4, 4, 4], [9, 9, 12], [5, -1, 1], (32, 48, 48)),
    (3, 20, 2, 64, 64, [0, 10, 5], None, [1, 1, 1], (32, 32)),       # the same slot and positions twice
    (1, 700, 5, 128, 1024, [123], [651], None, (44, 42, 42)),
    # heads in fours: a workgroup's waves share their tokens' angles
    (1, 1, 4, 64, 64, [63], None, None, (64,)),
    (2, 33, 4, 128, 128, [1, 95], [33, 20], None, (44, 42, 42)),
    (3, 17, 8, 64, 64, [0, 5, 47], [17, 0, 9], [5, 2, 1], (16, 24, 24)),
    (2, 100, 12, 128, 128, [0, 30], [100, 65], [1, 1], (32, 48, 48)),
]


@pytest.mark.gpu
@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("case", WRITES, ids=[str(c) for c in WRITES])
def test_kv_cache_write_rope(gpu, case, halves):
    """Values are stored as kv_cache_write stores them, turned keys within half a
    step of e4m3 under the smallest scale that fits, and the rest stays as it was."""
    B, S, Hk, D, cap, start, num, slots, split = case
    print(f"[case] write_rope {case} halves={halves}", flush=True)
    rng = np.random.default_rng(B * S + D)
    raw = [rng.integers(0, 256, (4, Hk, cap, D), np.uint8) for _ in range(2)]
    raw += [rng.integers(0, 256, (4, Hk, cap), np.uint8) for _ in range(2)]
    types = (E4M3, E4M3, E8M0, E8M0)
    make = lambda: vx.KVCache(*(torch.from_numpy(x.copy()).to(gpu).view(t) for x, t in zip(raw, types)))
    rope = vx.create_axis_rope(D, split, halves=halves, device=gpu)
    k, v = (_bf16(rng.standard_normal((B, S, Hk, D)) * np.exp(3 * rng.standard_normal((B, S, Hk, 1))), gpu)
            for _ in range(2))
    p = rng.integers(-50, 100000, (B, S, len(split)))
    at = dict(start=_ints(start, gpu), num=_ints(num, gpu), slots=_ints(slots, gpu))
    cache, plain, still = make(), make(), make()
    vx.kv_cache_write_rope(cache, k, v, _ints(p.tolist(), gpu), rope, **at)
    assert _lib.last_launch() == f"kv_write_rope_kernel<{D}, {'halves' if halves else 'adjacent'}>"
    vx.kv_cache_write(plain, k, v, **at)
    vx.kv_cache_write_rope(still, k, v, torch.zeros_like(_ints(p.tolist(), gpu)), rope, **at)
    got, want, same = _bytes(cache), _bytes(plain), _bytes(still)
    assert all((x == y).all() for x, y in zip(same, want))   # positions 0: nothing turns
    assert (got[1] == want[1]).all() and (got[3] == want[3]).all()
    y, size = O.axis_rope(_f64(k), p, rope.turns.tolist(), rope.axis.tolist(), halves)
    slack = 2.0 ** -20 * size
    rows = {}  # what a position holds: the last item's token
    for b in range(B):
        slot = b if slots is None else slots[b]
        for t in range(S if num is None else min(num[b], S)):
            pos = (0 if start is None else start[b]) + t
            if 0 <= slot < 4 and 0 <= pos < cap:
                rows[slot, pos] = (b, t)
    untouched = np.ones((4, cap), bool)
    stored = CO.values(got[0], got[2])
    for (slot, pos), (b, t) in rows.items():
        untouched[slot, pos] = False
        for h in range(Hk):
            top = np.abs(y[b, t, h]).max()
            most = slack[b, t, h].max()
            fits = {int(CO.quantise(np.array([[m]]))[1][0]) for m in (top - most, top + most)}
            s = int(got[2][slot, h, pos])
            assert s in fits, (slot, pos, h, s, fits)
            tol = np.maximum(2.0 ** -4 * np.abs(y[b, t, h]), 2.0 ** (s - 127 - 10)) + (1 + 2.0 ** -4) * slack[b, t, h]
            assert (np.abs(stored[slot, h, pos] - y[b, t, h]) <= tol).all(), (slot, pos, h)
    for x, before in zip(got, raw):
        x, before = np.moveaxis(x, 1, 2), np.moveaxis(before, 1, 2)
        assert (x[untouched] == before[untouched]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("halves", [False, True])
def test_turned_rows_that_are_not_finite(gpu, halves):
    """A NaN or an infinity in a key row, or a pair whose turn passes fp32, makes it a
    NaN row; rows of the largest and smallest magnitudes keep their scales."""
    rope = vx.create_axis_rope(64, (32, 32), halves=halves, device=gpu)
    x = np.random.default_rng(4).standard_normal((1, 8, 1, 64))
    x[0, 0, 0, 3], x[0, 1, 0, 40], x[0, 2, 0, 63] = np.nan, np.inf, -np.inf
    x[0, 3] = 3.38e38
    x[0, 4] = 0.0
    x[0, 5] *= 2.0 ** -130
    x[0, 6] *= 2.0 ** 120
    k = _bf16(x, gpu)
    c = vx.create_kv_cache(1, 64, 1, 64, device=gpu)
    p = _ints([[[1, 7]] * 8], gpu)
    vx.kv_cache_write_rope(c, k, k.nan_to_num(0.0, 0.0, 0.0), p, rope)
    scales = _bytes(c)[2][0, 0, :8]
    y = O.axis_rope(np.nan_to_num(_f64(k), nan=0.0, posinf=0.0, neginf=0.0), np.array([[[1, 7]] * 8]),
                    rope.turns.tolist(), rope.axis.tolist(), halves)[0][0, :, 0]
    assert (scales[:3] == 255).all() and (_bytes(c)[0][0, 0, :3] == 0).all()
    assert np.abs(y[3]).max() > 3.4028235e38 and scales[3] == 255
    assert scales[4] == 1 and (_bytes(c)[0][0, 0, 4] & 127 == 0).all() and scales[5] == 1
    assert scales[6] == CO.quantise(y[6:7])[1][0] and scales[7] == CO.quantise(y[7:8])[1][0]


# ------------------------------------------------------------------ attention on the GPU
def _cache_of(rng, slots, Hk, cap, D, gpu, lens=None, std=1.0):
    """A cache of random tokens; positions from lens[slot] on hold arbitrary
    bytes (NaN codes and scales among them)."""
    raw = [rng.integers(0, 256, (slots, Hk, cap, D), np.uint8) for _ in range(2)]
    raw += [rng.integers(0, 256, (slots, Hk, cap), np.uint8) for _ in range(2)]
    cache = vx.KVCache(*(torch.from_numpy(x).to(gpu).view(t) for x, t in zip(raw, (E4M3, E4M3, E8M0, E8M0))))
    k = _bf16(std * rng.standard_normal((slots, cap, Hk, D)), gpu)
    v = _bf16(rng.standard_normal((slots, cap, Hk, D)) * np.exp(rng.standard_normal((slots, cap, Hk, 1))), gpu)
    vx.kv_cache_write(cache, k, v, num=None if lens is None else np.minimum(lens, cap))
    return cache


def _held(cache, lens=None):
    """Stored values (k, v) in 64 bits, what lies past lens replaced by zeros."""
    raw, out = _bytes(cache), []
    for codes, scales in ((raw[0], raw[2]), (raw[1], raw[3])):
        x = CO.values(codes, scales)
        for s in range(x.shape[0] if lens is not None else 0):
            x[s, :, max(int(lens[s]), 0):] = 0.0
        out.append(x)
    return out


def _assert_close(got, q, held, sees, **kw):
    q64 = _f64(q)
    ref, spread = O.masked_attention(q64, *held, sees, **kw)
    D = q.shape[3]
    scale = kw.get("scale") or D ** -0.5
    L = scale * np.abs(q64).sum(-1).max() * np.abs(held[0]).max()
    n = held[0].shape[2]
    tol = 2 * 2.0 ** -8 * np.abs(ref) + spread * (2.0 ** -8 + 2 * (D + 2) * 2.0 ** -24 * L + 2 * (n + 64) * 2.0 ** -24)
    err = np.abs(_f64(got) - ref)
    assert not np.isnan(err).any()
    at = np.unravel_index(np.argmax(err - tol), err.shape)
    assert (err <= tol).all(), (at, err[at], tol[at], ref[at])


def _by_slot(n_slots, cap, kv_len, slots):
    lens = np.zeros(n_slots, int)
    for b, n in enumerate(kv_len):
        slot = b if slots is None else slots[b]
        if 0 <= slot < n_slots:
            lens[slot] = max(lens[slot], min(max(n, 0), cap))
    return lens


WINDOWS = [
    # B, Sq, H, Hk, D, cap, kv_len, q_len, slots, window, sinks, causal
    (1, 1, 1, 1, 128, 64, [1], None, None, 1, 0, True),
    (1, 1, 1, 1, 64, 64, [0], None, None, 1, 1, True),
    (2, 1, 4, 2, 128, 128, [128, 5], None, None, 1, 0, True),              # a query sees itself
    (3, 1, 8, 1, 64, 320, [300, 0, 31], None, [2, 0, 1], 70, 3, True),
    (5, 1, 16, 2, 128, 1024, [1000, 1, 33, 64, 700], None, None, 200, 4, True),
    (1, 1, 12, 12, 128, 2048, [1999], None, None, 64, 64, True),           # tiles and sinks that are whole
    (1, 1, 12, 12, 128, 2048, [1984], None, None, 96, 32, True),
    (2, 1, 8, 8, 64, 4096, [4001, 4096], None, None, 3000, 33, True),      # in parts
    (1, 1, 71, 1, 64, 448, [447], None, None, 100, 5, True),
    (2, 4, 6, 2, 64, 192, [150, 4], None, None, 3, 2, True),
    (2, 7, 10, 2, 128, 192, [190, 100], [7, 3], None, 33, 0, True),
    (2, 33, 2, 2, 128, 128, [97, 33], None, None, 10, 1, True),            # a whole prompt and a chunk
    (3, 70, 3, 1, 64, 256, [256, 70, 130], [70, 0, 1], [1, 2, 0], 20, 7, True),
    (1, 130, 4, 4, 128, 320, [300], None, None, 65, 30, True),
    (1, 300, 4, 1, 128, 512, [512], None, None, 100, 40, True),            # many rows; sinks inside some windows
    (2, 500, 2, 1, 64, 704, [700, 555], [500, 333], None, 128, 64, True),
    (1, 600, 3, 3, 128, 640, [600], None, None, 64, 0, True),              # prompts shorter and longer than it
    (2, 20, 2, 1, 128, 64, [3, 0], [20, 20], None, 2, 1, True),            # queries before the first key
    (2, 200, 2, 1, 128, 64, [3, 60], [200, 120], None, 2, 1, True),
    (2, 40, 4, 2, 64, 128, [77, 128], None, None, 50, 8, False),           # a block
    (1, 300, 2, 2, 128, 512, [512], None, None, 333, 60, False),
    (2, 257, 3, 3, 128, 320, [1, 300], [257, 129], None, 129, 0, False),
    (1, 200, 8, 8, 64, 2048, [1999], None, None, 1, 1, False),
    (4, 2, 2, 1, 64, 64, [10, 20, 30, 40], None, [0, 7, -1, 3], 5, 1, True),  # slots that are not there
    (3, 1, 4, 4, 128, 64, [1000, -3, 64], [9, 1, -2], None, 6, 2, True),   # lengths held to the sizes
    (2, 3, 4, 2, 128, 192, [190, 64], None, None, 2 ** 31 - 1, 0, True),
    (2, 3, 4, 2, 128, 192, [190, 64], None, None, 1, 2 ** 31 - 1, True),   # sinks past all keys
    (1, 150, 4, 1, 64, 1024, [1000], None, None, 40, 870, True),           # sinks up to and past the windows
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", WINDOWS, ids=[str(c) for c in WINDOWS])
def test_windowed_attention(gpu, case):
    B, Sq, H, Hk, D, cap, kv_len, q_len, slots, window, sinks, causal = case
    print(f"[case] windowed_attention {case}", flush=True)
    rng = np.random.default_rng(Sq * H + cap)
    n_slots = max(B, 4)
    lens = _by_slot(n_slots, cap, kv_len, slots)
    cache = _cache_of(rng, n_slots, Hk, cap, D, gpu, lens)
    q = _bf16(2 * rng.standard_normal((B, Sq, H, D)), gpu)
    out = torch.full_like(q, 7.0)
    got = vx.windowed_attention(q, cache, _ints(kv_len, gpu), window=window, sinks=sinks, q_len=_ints(q_len, gpu),
                                slots=_ints(slots, gpu), causal=causal, out=out)
    assert got is out
    print(f"  launched {_lib.last_launch()}", flush=True)
    _assert_close(got, q, _held(cache, lens), lambda b, n, m: O.window_sees(n, m, window, sinks, causal),
                  kv_len=kv_len, q_len=q_len, slots=slots)


def _lens(rng, B, most):
    x = rng.integers(0, most + 1, B)
    x[rng.random(B) < 0.2] = 0
    x[0] = most
    return [int(v) for v in x]


@pytest.mark.gpu
@pytest.mark.parametrize("B,Sq,H,Hk,D,cap,window,sinks,causal", [
    (70, 1, 8, 2, 128, 2048, 1100, 5, True),     # more streams than lanes
    (130, 1, 2, 1, 64, 1536, 1200, 40, True),
    (9, 3, 4, 1, 64, 4096, 2000, 33, True),
    (5, 40, 8, 2, 128, 2048, 300, 20, True),
    (3, 70, 8, 2, 64, 2048, 1500, 0, True),
    (2, 200, 4, 1, 128, 2560, 1000, 100, True),
    (2, 150, 2, 1, 128, 2560, 1400, 100, False),
    (66, 9, 4, 2, 64, 320, 31, 3, True),
])
def test_windows_over_many_lengths(gpu, B, Sq, H, Hk, D, cap, window, sinks, causal):
    print(f"[case] windows B={B} Sq={Sq} H={H}/{Hk} D={D} cap={cap} window={window} sinks={sinks}", flush=True)
    rng = np.random.default_rng(B + cap)
    kv_len, q_len = _lens(rng, B, cap), _lens(rng, B, Sq)
    cache = _cache_of(rng, B, Hk, cap, D, gpu, np.array(kv_len))
    q = _bf16(2 * rng.standard_normal((B, Sq, H, D)), gpu)
    got = vx.windowed_attention(q, cache, _ints(kv_len, gpu), window=window, sinks=sinks, q_len=_ints(q_len, gpu),
                                causal=causal)
    print(f"  launched {_lib.last_launch()}", flush=True)
    _assert_close(got, q, _held(cache, kv_len), lambda b, n, m: O.window_sees(n, m, window, sinks, causal),
                  kv_len=kv_len, q_len=q_len)


def _tree(rng, B, Sq, kind):
    if kind == "chain":
        return np.broadcast_to(np.arange(-1, Sq - 1), (B, Sq)).copy()
    if kind == "roots":
        return np.full((B, Sq), -1)
    if kind == "star":
        return np.where(np.arange(Sq) == 0, -1, 0) + np.zeros((B, 1), int)
    if kind == "wild":  # anything, most of it no parent
        return rng.integers(-2 ** 31, 2 ** 31, (B, Sq)) >> rng.integers(0, 28, (B, Sq))
    p = (np.arange(Sq) * np.sqrt(rng.random((B, Sq)))).astype(int)
    return np.where(rng.random((B, Sq)) < 0.1, -1, np.minimum(p, np.arange(Sq) - 1))


TREES = [
    # B, Sq, H, Hk, D, cap, kv_len, q_len, slots, kind
    (1, 1, 1, 1, 64, 64, [1], None, None, "any"),
    (1, 1, 1, 1, 128, 64, [0], None, None, "any"),
    (1, 5, 1, 1, 128, 64, [5], None, None, "any"),                         # nothing in front
    (2, 26, 12, 12, 128, 1024, [700, 26], None, None, "any"),
    (2, 26, 12, 12, 128, 1024, [700, 26], None, None, "wild"),
    (3, 31, 8, 2, 64, 320, [300, 31, 200], [31, 0, 7], [2, 0, 1], "any"),
    (2, 32, 4, 1, 128, 320, [320, 64], None, None, "chain"),
    (2, 33, 4, 1, 64, 320, [319, 65], [33, 32], None, "star"),
    (2, 64, 8, 2, 128, 448, [400, 128], None, None, "roots"),
    (2, 65, 8, 2, 64, 448, [400, 97], [65, 64], None, "any"),
    (3, 61, 8, 2, 128, 4096, [4000, 100, 61], [61, 30, 61], None, "any"),  # in parts
    (1, 250, 8, 1, 64, 1024, [1000], None, None, "any"),
    (2, 250, 4, 1, 128, 512, [512, 300], [250, 201], None, "wild"),
    (1, 512, 2, 2, 128, 640, [600], None, None, "any"),
    (1, 512, 2, 1, 64, 576, [512], None, None, "chain"),
    (1, 511, 1, 1, 128, 576, [573], None, None, "any"),
    (2, 20, 2, 1, 128, 64, [3, 0], [20, 20], None, "any"),                 # drafted tokens before the first position
    (2, 200, 4, 2, 64, 256, [130, 0], [200, 200], None, "chain"),
    (4, 6, 2, 1, 64, 64, [10, 20, 30, 40], None, [0, 7, -1, 3], "any"),    # slots that are not there
    (3, 4, 4, 4, 128, 64, [1000, -3, 64], [9, 1, -2], None, "any"),        # lengths held to the sizes
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", TREES, ids=[str(c) for c in TREES])
def test_tree_attention(gpu, case):
    B, Sq, H, Hk, D, cap, kv_len, q_len, slots, kind = case
    print(f"[case] tree_attention {case}", flush=True)
    rng = np.random.default_rng(Sq * H + cap)
    n_slots = max(B, 4)
    lens = _by_slot(n_slots, cap, kv_len, slots)
    cache = _cache_of(rng, n_slots, Hk, cap, D, gpu, lens)
    q = _bf16(2 * rng.standard_normal((B, Sq, H, D)), gpu)
    parents = _tree(rng, B, Sq, kind)
    out = torch.full_like(q, 7.0)
    got = vx.tree_attention(q, cache, _ints(parents.tolist(), gpu), _ints(kv_len, gpu), q_len=_ints(q_len, gpu),
                            slots=_ints(slots, gpu), out=out)
    assert got is out
    print(f"  launched {_lib.last_launch()}", flush=True)
    held, kw = _held(cache, lens), dict(kv_len=kv_len, q_len=q_len, slots=slots)
    _assert_close(got, q, held, lambda b, n, m: O.tree_sees(n, m, parents[b]), **kw)
    if kind == "chain":  # what causal attention computes
        _assert_close(vx.cached_attention(q, cache, _ints(kv_len, gpu), q_len=_ints(q_len, gpu),
                                          slots=_ints(slots, gpu)), q, held,
                      lambda b, n, m: O.tree_sees(n, m, parents[b]), **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("B,Sq,H,Hk,D,cap", [(70, 5, 8, 2, 128, 1536), (9, 30, 4, 1, 64, 4096),
                                             (3, 100, 8, 2, 128, 2048), (130, 9, 2, 1, 64, 192)])
def test_trees_over_many_lengths(gpu, B, Sq, H, Hk, D, cap):
    print(f"[case] trees B={B} Sq={Sq} H={H}/{Hk} D={D} cap={cap}", flush=True)
    rng = np.random.default_rng(B + cap)
    kv_len, q_len = _lens(rng, B, cap), _lens(rng, B, Sq)
    cache = _cache_of(rng, B, Hk, cap, D, gpu, np.array(kv_len))
    q = _bf16(2 * rng.standard_normal((B, Sq, H, D)), gpu)
    parents = _tree(rng, 1, Sq, "any")[0]
    got = vx.tree_attention(q, cache, _ints(parents.tolist(), gpu), _ints(kv_len, gpu), q_len=_ints(q_len, gpu))
    print(f"  launched {_lib.last_launch()}", flush=True)
    _assert_close(got, q, _held(cache, kv_len), lambda b, n, m: O.tree_sees(n, m, parents), kv_len=kv_len, q_len=q_len)


# each kernel of the plan: name, B, Sq, H, Hk, D, cap, kv_len
PLANS = [
    ("few_masked_kernel<{D}, 8, {mask}>", 1, 1, 12, 12, 700, [690]),
    ("few_masked_kernel<{D}, 4, {mask}>", 40, 1, 8, 8, 128, [100] * 40),
    ("few_masked_kernel<{D}, 4, {mask}>", 2, 3, 4, 2, 4096, [4090, 2000]),   # in parts
    ("many_masked_kernel<{D}, {mask}>", 2, 500, 50, 25, 704, [704, 600]),
    # with heads of 64 (named first) 2000 rows' 63 small tiles take 0.4125 x 63 x 0.54 us, 16 large ones
    # 1.05 x 16 x 0.54 and their start of 5: as long
    ("few_masked_kernel<64, 4, {mask}> many_masked_kernel<128, 8, {mask}>", 1, 500, 100, 25, 704, [700]),
    ("many_masked_kernel<64, {mask}> many_masked_kernel<128, 8, {mask}>", 2, 256, 32, 8, 4096, [4000, 3001]),  # in parts
]


def _kernel(name, D, mask):
    both = name.split("> ")
    return (both[0] + ">" if len(both) == 2 and D == 64 else both[-1]).format(D=D, mask=mask)


def _plan_call(mask, gpu, rng, q, cache, kv_len, **kw):
    B, Sq = q.shape[:2]
    if mask == "window":
        window, sinks = max(kv_len) - 30, 3
        sees = lambda b, n, m: O.window_sees(n, m, window, sinks, True)
        return sees, lambda: vx.windowed_attention(q, cache, _ints(kv_len, gpu), window=window, sinks=sinks, **kw)
    parents = _tree(rng, B, Sq, "any")
    on = _ints(parents.tolist(), gpu)
    lens = _ints(kv_len, gpu)
    return (lambda b, n, m: O.tree_sees(n, m, parents[b])), lambda: vx.tree_attention(q, cache, on, lens, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("mask", ["window", "tree"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("plan", PLANS, ids=[f"{p[0]} {p[5]}" for p in PLANS])
def test_every_kernel_of_the_plan(gpu, plan, D, mask):
    """Each kernel, by name, against the oracle, with a scale of its own, strided
    queries and outputs; rows of scale NaN reach exactly the queries that see them;
    two runs give the same bits."""
    name, B, Sq, H, Hk, cap, kv_len = plan
    print(f"[case] {plan} D={D} {mask}", flush=True)
    rng = np.random.default_rng(D + cap)
    cap = (cap + 63) // 64 * 64
    cache = _cache_of(rng, B, Hk, cap, D, gpu, np.array(kv_len))
    fused = _bf16(2 * rng.standard_normal((B, Sq, H, 2, D)), gpu)
    q = fused[:, :, :, 1]
    wide = torch.full((B, Sq, H, 3, D), 5.0, dtype=torch.bfloat16, device=gpu)
    sees, call = _plan_call(mask, gpu, rng, q, cache, kv_len, scale=0.11, out=wide[:, :, :, 1])
    got = call().clone()
    assert _lib.last_launch() == _kernel(name, D, mask)
    assert (wide[:, :, :, 0] == 5).all() and (wide[:, :, :, 2] == 5).all()
    _assert_close(got, q, _held(cache, kv_len), sees, kv_len=kv_len, scale=0.11)
    assert torch.equal(call(), got)
    for which in (2, 3):  # a key's scale, then a value's; the row's bytes are zeros
        bad = [min(n - 1, x) for n, x in zip(kv_len, (5, 40, 9, 17) * 10)]
        n0 = kv_len[0]
        bad[0] = n0 - 31  # at the border of the windows, among the last tiles
        held = cache[which].view(torch.uint8).clone(), cache[which - 2].view(torch.uint8).clone()
        for b in range(B):
            cache[which].view(torch.uint8)[b, 0, bad[b]] = 255
            cache[which - 2].view(torch.uint8)[b, 0, bad[b]] = 0
        nan = call().isnan().cpu().numpy()
        want = np.zeros(nan.shape, bool)
        for b in range(B):
            see = sees(b, kv_len[b], Sq)[:, bad[b]]
            want[b, see, :H // Hk] = True
        assert (nan == want).all(), which
        cache[which].view(torch.uint8).copy_(held[0])
        cache[which - 2].view(torch.uint8).copy_(held[1])


@pytest.mark.gpu
@pytest.mark.parametrize("mask", ["window", "tree"])
@pytest.mark.parametrize("plan", PLANS, ids=[f"{p[0]} {p[5]}" for p in PLANS])
@pytest.mark.parametrize("size", [2.0 ** 25, -2.0 ** 40, 2.0 ** 100])
def test_logits_of_any_size(gpu, plan, mask, size):
    """Keys so large that a query sees, as good as alone, the keys of its largest
    logit: their values' mean. (Keys +-size in one channel, the others 0.)"""
    name, B, Sq, H, Hk, cap, kv_len = plan
    D = 128
    rng = np.random.default_rng(31)
    cap = (cap + 63) // 64 * 64
    sign = rng.integers(0, 2, (B, cap, Hk)) * 2 - 1
    k = np.zeros((B, cap, Hk, D))
    k[..., 0] = sign * size
    v = rng.standard_normal((B, cap, Hk, D))
    cache = vx.create_kv_cache(B, cap, Hk, D, device=gpu)
    vx.kv_cache_write(cache, _bf16(k, gpu), _bf16(v, gpu))
    q = np.zeros((B, Sq, H, D))
    q[..., 0] = 1.0
    q = _bf16(q, gpu)
    sees, call = _plan_call(mask, gpu, rng, q, cache, kv_len, scale=1.0)
    got = _f64(call())
    assert _lib.last_launch() == _kernel(name, D, mask)
    held = _held(cache)[1]
    for b in range(B):
        see = sees(b, kv_len[b], Sq)
        for h in range(H):
            g = h // (H // Hk)
            up = sign[b, :kv_len[b], g] * np.sign(size) > 0
            best = np.where((see & up).any(-1, keepdims=True), see & up, see)
            w = best / np.maximum(best.sum(-1, keepdims=True), 1)
            x = held[b, g, :kv_len[b]]
            ref, spread = w @ x, w @ np.abs(x)
            tol = 2 * 2.0 ** -8 * np.abs(ref) + spread * (2.0 ** -8 + 2 * (cap + 64) * 2.0 ** -24)
            assert (np.abs(got[b, :, h] - ref) <= tol).all(), (b, h)


@pytest.mark.gpu
@pytest.mark.parametrize("mask", ["window", "tree"])
@pytest.mark.parametrize("plan", PLANS, ids=[f"{p[0]} {p[5]}" for p in PLANS])
def test_queries_that_are_not_finite(gpu, plan, mask):
    """A NaN in a query makes NaN that query's output alone; in padding rows it is
    not looked at, and they give zeros."""
    name, B, Sq, H, Hk, cap, kv_len = plan
    rng = np.random.default_rng(cap)
    cap = (cap + 63) // 64 * 64
    cache = _cache_of(rng, B, Hk, cap, 128, gpu, np.array(kv_len))
    q = _bf16(rng.standard_normal((B, Sq, H, 128)), gpu)
    q_len = [Sq - min(b, Sq - 1) * (Sq // 3 + 1) if Sq > 2 else Sq for b in range(B)]
    q_len = [max(m, 1) for m in q_len]
    sees, call = _plan_call(mask, gpu, rng, q, cache, kv_len, q_len=_ints(q_len, gpu))
    want = call()
    for b in range(B):
        q[b, q_len[b]:] = float("nan")
    assert torch.equal(call(), want) and _lib.last_launch() == _kernel(name, 128, mask)
    assert all((want[b, q_len[b]:] == 0).all() for b in range(B))
    q[0, Sq // 2, H - 1, 5] = float("nan")
    q[B - 1, 0, 0, 127] = float("nan")
    got = call()
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[0, Sq // 2, H - 1] = hit[B - 1, 0, 0] = True
    assert got[hit].isnan().all() and torch.equal(got[~hit], want[~hit])


@pytest.mark.gpu
@pytest.mark.parametrize("Sq,cap", [(1, 8192), (64, 1024), (600, 704)])
def test_a_window_of_everything_is_causal_attention(gpu, Sq, cap):
    """With every position in its window, or among its sinks, a call gives what
    cached_attention gives: the same tiles in the same order, bit for bit."""
    rng = np.random.default_rng(Sq)
    cache = _cache_of(rng, 2, 2, cap, 128, gpu)
    q = _bf16(rng.standard_normal((2, Sq, 4, 128)), gpu)
    n = _ints([cap, cap - 77], gpu)
    want = vx.cached_attention(q, cache, n)
    assert torch.equal(vx.windowed_attention(q, cache, n, window=cap), want)
    assert torch.equal(vx.windowed_attention(q, cache, n, window=1, sinks=cap), want)
    want = vx.cached_attention(q, cache, n, causal=False)
    assert torch.equal(vx.windowed_attention(q, cache, n, window=2 ** 40, causal=False), want)


@pytest.mark.gpu
def test_unseen_positions_are_not_read(gpu):
    """What lies outside every query's view, a tile and more from it, may be
    anything: NaN codes and scales there change nothing."""
    rng = np.random.default_rng(12)
    cap, n = 4096, 4000
    cache = _cache_of(rng, 1, 2, cap, 128, gpu, [n])
    for Sq, window, sinks in ((1, 500, 10), (40, 900, 70), (300, 128, 0)):
        q = _bf16(rng.standard_normal((1, Sq, 8, 128)), gpu)
        want = vx.windowed_attention(q, cache, [n], window=window, sinks=sinks)
        junk = vx.KVCache(*(t.clone() for t in cache))
        lo, hi = (sinks + 63) // 64 * 64, (n - Sq + 1 - window) // 64 * 64
        junk.k.view(torch.uint8)[:, :, lo:hi] = 0x7f
        junk.v.view(torch.uint8)[:, :, lo:hi] = 0xff
        junk.v_scale.view(torch.uint8)[:, :, lo:hi] = 255
        assert torch.equal(vx.windowed_attention(q, junk, [n], window=window, sinks=sinks), want)


UNSEEN = [
    # kernels with heads of 64 and of 128, B, Sq, H, Hk, cap, kv_len, window, sinks, causal
    ("few 8, few 8", 1, 1, 12, 12, 704, [690], 500, 10, True),            # both borders inside tiles
    ("few 8, few 8", 1, 1, 12, 12, 704, [690], 640, 35, True),            # ... of the same tile: 35 .. 49
    ("few 4, few 4", 1, 1, 4, 4, 704, [690], 1, 0, True),                 # one key of a tile
    ("few 8, few 8", 1, 1, 4, 4, 704, [690], 34, 1, True),
    ("few 4, few 4", 40, 1, 8, 8, 128, [100] * 39 + [33], 30, 2, True),
    ("few 4, few 4", 2, 3, 8, 8, 8192, [8190, 5000], 4000, 70, True),     # in parts
    ("few 8, few 8", 2, 40, 4, 1, 512, [500, 300], 100, 31, True),        # tiles of rows with windows of their own
    ("few 8, few 8", 2, 20, 4, 1, 512, [500, 300], 77, 5, False),
    ("many 4, many 4", 2, 256, 64, 16, 2048, [2000, 1400], 1000, 70, True),
    ("many 4, many 4", 2, 600, 64, 32, 1024, [1000, 960], 300, 33, True),  # (the second item's: 33 .. 60)
    ("few 4, many 8", 1, 600, 64, 32, 1024, [999], 300, 33, True),
    ("many 4, many 4", 2, 700, 64, 32, 1024, [1000, 701], 500, 5, False),
    ("many 4, many 8", 2, 256, 32, 8, 4096, [4000, 3001], 2500, 100, True),  # in parts
]


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("case", UNSEEN, ids=[str(c) for c in UNSEEN])
def test_what_unseen_positions_hold_is_nothing(gpu, case, D):
    """Whatever lies at positions that no query sees, up to the borders of the sinks and
    of the window and behind the last token, changes no bit: NaN codes under scales of
    NaN, the largest values under the largest scale, any bytes."""
    kernels, B, Sq, H, Hk, cap, kv_len, window, sinks, causal = case
    print(f"[case] unseen {case} D={D}", flush=True)
    rng = np.random.default_rng(Sq + window)
    cache = _cache_of(rng, B, Hk, cap, D, gpu)
    q = _bf16(2 * rng.standard_normal((B, Sq, H, D)), gpu)
    call = lambda c: vx.windowed_attention(q, c, _ints(kv_len, gpu), window=window, sinks=sinks, causal=causal)
    want = call(cache)
    print(f"  launched {_lib.last_launch()}", flush=True)
    kind, waves = kernels.split(", ")[D // 128].split()
    assert _lib.last_launch() == f"{kind}_masked_kernel<{D}, {waves}, window>".replace(", 4" * (kind == "many"), "")
    assert not want.isnan().any()
    seen = torch.zeros((B, cap), dtype=torch.bool)
    for b, n in enumerate(kv_len):
        seen[b, :n] = torch.from_numpy(O.window_sees(n, Sq, window, sinks, causal).any(0))
        assert not seen[b, sinks:n].all()
    hidden = (~seen).to(gpu)[:, None].expand(B, Hk, cap)
    for code, scale in ((0xff, 255), (0x7e, 254), (None, None)):
        junk = vx.KVCache(*(t.clone() for t in cache))
        for t, x in zip(junk, (code, code, scale, scale)):
            held = t.view(torch.uint8)
            at = hidden[..., None].expand_as(held) if held.dim() == 4 else hidden
            held[at] = x if x is not None else torch.from_numpy(rng.integers(0, 256, int(at.sum()), np.uint8)).to(gpu)
        assert torch.equal(call(junk), want), code


@pytest.mark.gpu
def test_offsets_past_32_bits(gpu):
    """Positions of a slot that lies more than 2^32 bytes into the cache, written
    turned and attended over in both ways, as those of a small one."""
    slots, Hk, cap, D = 9, 8, 524288, 128  # 4.8e9 bytes of keys
    big = vx.KVCache(*(torch.empty(s, dtype=torch.uint8, device=gpu).view(t) for s, t in
                       (((slots, Hk, cap, D), E4M3),) * 2 + (((slots, Hk, cap), E8M0),) * 2))
    small = vx.create_kv_cache(1, 1024, Hk, D, device=gpu)
    rope = vx.create_axis_rope(D, (44, 42, 42), device=gpu)
    g = torch.Generator(device=gpu).manual_seed(9)
    k, v = (torch.randn((1, 1000, Hk, D), generator=g, device=gpu).bfloat16() for _ in range(2))
    p = torch.arange(1000, dtype=torch.int32, device=gpu)[:, None].expand(1000, 3)
    vx.kv_cache_write_rope(small, k, v, p, rope)
    q = torch.randn((1, 9, 16, D), generator=g, device=gpu).bfloat16()
    parents = torch.arange(9, dtype=torch.int32, device=gpu) // 2 - 1
    at = cap - 1000
    vx.kv_cache_write_rope(big, k, v, p, rope, [at], slots=[slots - 1])
    # sees the last 700 of either
    want = vx.windowed_attention(q, small, [1000], window=600)
    got = vx.windowed_attention(q, big, [cap], window=600, slots=[slots - 1])
    tol = 2 * 2.0 ** -8 * want.abs().double() + 2.0 ** -7 * float(v.abs().max())
    assert ((got.double() - want.double()).abs() <= tol).all()
    vx.kv_cache_write_rope(big, k, v, p, rope, [0], slots=[slots - 1])
    want = vx.tree_attention(q, small, parents, [1000])
    got = vx.tree_attention(q, big, parents, [1000], slots=[slots - 1])
    assert ((got.double() - want.double()).abs() <= tol.max()).all()


# ------------------------------------------------------------------ as they are used together
def _rollout(gpu, on_stream=None):
    """Blocks of a rollout through the cache, then drafted tokens and the accepted
    ones: every step's attention against the oracle on what the cache holds."""
    rng = np.random.default_rng(77)
    H, Hk, D, cap, block, blocks = 8, 4, 64, 512, 60, 6
    rope = vx.create_axis_rope(D, (16, 24, 24), device=gpu)
    cache = vx.create_kv_cache(2, cap, Hk, D, device=gpu)
    slots = [1, 0]
    new = lambda S, heads: _bf16(rng.standard_normal((2, S, heads, D)), gpu)
    grid = np.stack(np.meshgrid(np.arange(3), np.arange(4), np.arange(5), indexing="ij"), -1).reshape(-1, 3)
    n = 0
    window, sinks = 2 * block, block
    for step in range(blocks):  # three frames of 4 x 5 a block
        p = _ints((grid + [3 * step, 0, 0]).tolist(), gpu)
        q, k, v = new(block, H), new(block, Hk), new(block, Hk)
        turned = vx.apply_axis_rope(q, p, rope)
        _assert_turned(turned, q, np.broadcast_to(p.cpu().numpy(), (2, block, 3)), rope)
        vx.kv_cache_write_rope(cache, k, v, p, rope, _ints([n, n], gpu), slots=_ints(slots, gpu))
        n += block
        got = vx.windowed_attention(turned, cache, _ints([n, n], gpu), window=window, sinks=sinks, causal=False,
                                    slots=_ints(slots, gpu))
        _assert_close(got, turned, _held(cache), lambda b, n, m: O.window_sees(n, m, window, sinks, False),
                      kv_len=[n, n], slots=slots)
    # nine drafted tokens behind the blocks, at the positions of their depths
    parents = np.array([-1, 0, 0, 1, 1, 2, 3, 6, 6])
    depth = np.array([0, 1, 1, 2, 2, 2, 3, 4, 4])
    p = _ints((np.repeat(depth[:, None], 3, 1) + 100).tolist(), gpu)
    q, k, v = new(9, H), new(9, Hk), new(9, Hk)
    turned = vx.apply_axis_rope(q, p, rope)
    vx.kv_cache_write_rope(cache, k, v, p, rope, _ints([n, n], gpu), slots=_ints(slots, gpu))
    drafted = vx.tree_attention(turned, cache, _ints(parents.tolist(), gpu), _ints([n + 9] * 2, gpu),
                                slots=_ints(slots, gpu))
    _assert_close(drafted, turned, _held(cache), lambda b, n, m: O.tree_sees(n, m, parents), kv_len=[n + 9] * 2,
                  slots=slots)
    # the path 0 - 1 - 3 - 6 - 8 is accepted: written as the sequence's next tokens, its queries see what they saw
    path = [0, 1, 3, 6, 8]
    vx.kv_cache_write_rope(cache, k[:, path], v[:, path], p[path], rope, _ints([n, n], gpu), slots=_ints(slots, gpu))
    n += len(path)
    taken = vx.cached_attention(turned[:, path], cache, _ints([n, n], gpu), slots=_ints(slots, gpu))
    _assert_close(taken, turned[:, path], _held(cache), lambda b, n, m: O.window_sees(n, m, n, 0, True), kv_len=[n, n],
                  slots=slots)
    spread = float(v.abs().max()) * 2
    assert ((taken.double() - drafted[:, path].double()).abs() <= 2.0 ** -6 * spread).all()
    # next tokens, one by one
    for _ in range(3):
        p = _ints([[[200 + n] * 3]] * 2, gpu)
        q, k, v = new(1, H), new(1, Hk), new(1, Hk)
        turned = vx.apply_axis_rope(q, p, rope)
        vx.kv_cache_write_rope(cache, k, v, p, rope, _ints([n, n], gpu), slots=_ints(slots, gpu))
        n += 1
        got = vx.windowed_attention(turned, cache, _ints([n, n], gpu), window=50, sinks=4, slots=_ints(slots, gpu))
        _assert_close(got, turned, _held(cache), lambda b, n, m: O.window_sees(n, m, 50, 4, True), kv_len=[n, n],
                      slots=slots)


@pytest.mark.gpu
def test_a_rollout(gpu):
    _rollout(gpu)


@pytest.mark.gpu
def test_a_rollout_on_another_stream(gpu):
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        _rollout(gpu)
    s.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("Sq,cap", [(1, 4096), (40, 2048), (300, 640)])
def test_graph_replays(gpu, Sq, cap):
    """A captured step (turn, write, both attentions), replayed while positions,
    lengths, parents and queries change and eager steps run between the replays:
    every replay equals the eager result bit for bit. Two graphs of one pool side by
    side keep their results."""
    B, H, Hk, D = 3, 8, 4, 128
    rope = vx.create_axis_rope(D, (32, 48, 48), shared=True, halves=True, device=gpu)
    cache = _cache_of(np.random.default_rng(5), B, Hk, cap, D, gpu)
    q, k, v = (torch.empty((B, Sq, h, D), dtype=torch.bfloat16, device=gpu) for h in (H, Hk, Hk))
    kv_len, m, start = (torch.zeros(B, dtype=torch.int32, device=gpu) for _ in range(3))
    p, parents = (torch.zeros(s, dtype=torch.int32, device=gpu) for s in ((B, Sq, 3), (B, Sq)))

    def step():
        turned = vx.apply_axis_rope(q, p, rope)
        vx.kv_cache_write_rope(cache, k, v, p, rope, start, num=m)
        return (turned, vx.windowed_attention(turned, cache, kv_len, window=cap // 2, sinks=9, q_len=m),
                vx.tree_attention(turned, cache, parents, kv_len, q_len=m))

    def set_inputs(seed, share):
        r = np.random.default_rng(seed)
        for t in (q, k, v):
            t.copy_(torch.from_numpy(r.standard_normal(t.shape).astype(np.float32)))
        n = [int(cap * share) // (i + 1) for i in range(B)]
        used = [max(int(Sq * share), 1) if i else Sq for i in range(B)]
        kv_len.copy_(torch.tensor(n))
        m.copy_(torch.tensor(used))
        start.copy_(torch.tensor([a - b for a, b in zip(n, used)]))
        p.copy_(torch.from_numpy(r.integers(0, 9999, p.shape)))
        parents.copy_(torch.from_numpy(_tree(r, B, Sq, "any")))

    side = torch.cuda.Stream()
    set_inputs(0, 1.0)
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(first):
        out = step()
    with torch.cuda.graph(second, pool=first.pool()):
        other = step()
    for seed, share in ((1, 1.0), (2, 0.4), (3, 0.0), (4, 0.9)):
        print(f"  replay at {share}", flush=True)
        set_inputs(seed, share)
        want = [x.clone() for x in step()]
        torch.cuda.synchronize()
        for graph, outs in ((first, out), (second, other)):
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs, want))


@pytest.mark.gpu
def test_two_streams_at_once(gpu):
    """Calls of two streams at a time have workspaces of their own."""
    rng = np.random.default_rng(6)
    cache = _cache_of(rng, 4, 4, 8192, 128, gpu)
    q = [_bf16(rng.standard_normal((4, 3, 8, 128)), gpu) for _ in range(2)]
    parents = _ints([-1, 0, 0], gpu)
    calls = [lambda: vx.windowed_attention(q[0], cache, window=6000, sinks=8),
             lambda: vx.tree_attention(q[1], cache, parents)]
    want = [c() for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for s, c, o in zip(streams, calls, got):
            with torch.cuda.stream(s):
                o.append(c())
    torch.cuda.synchronize()
    for w, o in zip(want, got):
        assert all(torch.equal(x, w) for x in o)


@pytest.mark.gpu
def test_host_integers_and_captures(gpu):
    """Parents and positions from the host, as lists, arrays or tensors of any integer
    type; under a capture they are refused."""
    cache = _cache_of(np.random.default_rng(1), 2, 2, 128, 64, gpu)
    q = torch.randn((2, 3, 4, 64), device=gpu).bfloat16()
    par = [[-1, 0, 0], [-1, -1, 1]]
    want = vx.tree_attention(q, cache, _ints(par, gpu), _ints([50, 60], gpu))
    for x in (par, np.array(par), torch.tensor(par), torch.tensor(par, device=gpu),
              torch.tensor(par, dtype=torch.int8)):
        assert torch.equal(vx.tree_attention(q, cache, x, [50, 60]), want)
    want = vx.tree_attention(q, cache, _ints([par[0]] * 2, gpu))
    assert torch.equal(vx.tree_attention(q, cache, par[0]), want)
    assert torch.equal(vx.tree_attention(q, cache, _ints(par[0], gpu)), want)
    rope = vx.create_axis_rope(64, (32, 32), device=gpu)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(ValueError, match="captured"):
            vx.tree_attention(q, cache, par)
        with pytest.raises(ValueError, match="captured"):
            vx.apply_axis_rope(q, [[0, 0]] * 3, rope)
        roots = torch.full((3,), -1, dtype=torch.int32, device=gpu)
        out = vx.tree_attention(q, cache, roots)
    for _ in range(3):
        out.fill_(9.0)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, vx.tree_attention(q, cache, [-1] * 3))


@pytest.mark.gpu
def test_refusals_of_gpu_calls(gpu):
    cache = vx.create_kv_cache(2, 128, 2, 64, device=gpu)
    q = torch.zeros((2, 3, 4, 64), dtype=torch.bfloat16, device=gpu)
    k = q[:, :, :2]
    rope = vx.create_axis_rope(64, (32, 32), device=gpu)
    p = torch.zeros((2, 3, 2), dtype=torch.int32, device=gpu)
    with pytest.raises(TypeError, match="bfloat16"):
        vx.apply_axis_rope(q.float(), p, rope)
    with pytest.raises(ValueError, match="B, S, H, D"):
        vx.apply_axis_rope(q[0], p, rope)
    with pytest.raises(NotImplementedError, match="head_dim"):
        vx.apply_axis_rope(q[..., :32], p, rope)
    with pytest.raises(TypeError, match="AxisRope"):
        vx.apply_axis_rope(q, p, tuple(rope))
    with pytest.raises(TypeError, match="turns"):
        vx.apply_axis_rope(q, p, rope._replace(turns=rope.turns.int()))
    with pytest.raises(TypeError, match="axis"):
        vx.apply_axis_rope(q, p, rope._replace(axis=rope.axis.long()))
    with pytest.raises(ValueError, match="pairs"):
        vx.apply_axis_rope(q, p, vx.create_axis_rope(128, (64, 64), device=gpu))
    with pytest.raises(ValueError, match="device"):
        vx.apply_axis_rope(q, p, vx.create_axis_rope(64, (32, 32), device="cpu"))
    with pytest.raises(NotImplementedError, match="num_axes"):
        vx.apply_axis_rope(q, torch.zeros((2, 3, 5), dtype=torch.int32, device=gpu), rope._replace(axes=5))
    for bad in (p[:1], p[:, :2], p[..., :1], p[0, 0], torch.zeros((3, 2, 3), dtype=torch.int32)):
        with pytest.raises(ValueError, match="positions must be"):
            vx.apply_axis_rope(q, bad, rope)
    with pytest.raises(TypeError, match="integers"):
        vx.apply_axis_rope(q, p.float(), rope)
    with pytest.raises(ValueError, match="heads"):
        vx.kv_cache_write_rope(cache, q, q, p, rope)
    with pytest.raises(ValueError, match="shapes differ"):
        vx.kv_cache_write_rope(cache, k, k[:, :2], p, rope)
    with pytest.raises(ValueError, match="positions must be"):
        vx.kv_cache_write_rope(cache, k, k, p[:1], rope)
    with pytest.raises(ValueError, match="start must hold"):
        vx.kv_cache_write_rope(cache, k, k, p, rope, [0])
    with pytest.raises(ValueError, match="parents must be"):
        vx.tree_attention(q, cache, [[-1, 0, 0]])
    with pytest.raises(TypeError, match="integers"):
        vx.tree_attention(q, cache, [0.0, 1.0, 2.0])
    long = torch.zeros((1, 513, 2, 64), dtype=torch.bfloat16, device=gpu)
    with pytest.raises(NotImplementedError, match="drafted"):
        vx.tree_attention(long, cache, [-1] * 513)
    with pytest.raises(ValueError, match="multiple of num_kv_heads"):
        vx.windowed_attention(q[:, :, :3], cache, window=4)
    with pytest.raises(ValueError, match="out must be"):
        vx.windowed_attention(q, cache, window=4, out=q.float())
    with pytest.raises(ValueError, match="out must be"):
        vx.tree_attention(q, cache, [-1, 0, 0], out=q[:1].expand(2, 3, 4, 64))
    assert vx.windowed_attention(q[:0], cache, window=4).shape == (0, 3, 4, 64)
    assert vx.windowed_attention(q[:, :0], cache, window=4).shape == (2, 0, 4, 64)
    assert vx.tree_attention(q[:, :0], cache, torch.zeros((2, 0), dtype=torch.int32)).shape == (2, 0, 4, 64)
