"""The 8-bit key/value cache and the attention over it.

Stored values are compared exactly. Attention is compared with the oracle (64
bits, on the stored values) under a bound per output value that follows from
what the kernels round. With o the exact output and A the same weights over
|v|:
  2^-8 |o|                         the output to bf16
  2^-8 (A + |o|)                   the weights to bf16: w_j (1 + d_j), |d_j| <= 2^-8, over their own
                                   sum is off by sum_j w_j d_j (v_j - o) at most
  2 (D + 2) 2^-24 L A              fp32 logits: D products and sums of at most
                                   L = max_j scale sum_d |q_d k_jd| in all; a
                                   logit off by x moves weights by at most 2 x
  2 (n + 64) 2^-24 A               fp32 sums over n keys, exponentials, merges
"""
import ctypes

import numpy as np
import pytest
import torch

import vidax_amd as vx
from oracle import cache_oracle as O
from vidax_amd import _lib

A = 1 << 20  # a 16-byte aligned fake device address (never dereferenced)
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


# ------------------------------------------------------------------ refusals (CPU)
def test_cache_symbols_are_exported():
    import os
    import re
    text = open(os.path.join(os.path.dirname(__file__), "..", "include", "vx_cache.h")).read()
    names = set(re.findall(r"\b(vx_\w+)\s*\(", re.sub(r"/\*.*?\*/", "", text, flags=re.S)))
    assert names == set(_lib.CACHE_SYMBOLS)
    assert all(hasattr(_lib.lib(), n) for n in names)


def test_cache_abi_version():
    assert _lib.lib().vx_cache_abi_version() == 10000


def _write_check(**kw):
    a = dict(k=A, v=A, kst=None, vst=None, ck=A, cv=A, ks=A, vs=A, slots_n=4, cap=128, start=None, num=None,
             slots=None, B=2, S=3, Hk=2, D=64)
    a.update(kw)
    s3 = lambda s: None if s is None else _lib.strides3(s)
    return _lib.lib().vx_kv_write_check(a["k"], a["v"], s3(a["kst"]), s3(a["vst"]), a["ck"], a["cv"], a["ks"],
                                        a["vs"], a["slots_n"], a["cap"], a["start"], a["num"], a["slots"], a["B"],
                                        a["S"], a["Hk"], a["D"])


def _read_check(**kw):
    a = dict(ck=A, cv=A, ks=A, vs=A, slots_n=4, cap=128, start=None, slots=None, B=2, S=3, Hk=2, D=64, ko=A, vo=A)
    a.update(kw)
    return _lib.lib().vx_kv_read_check(a["ck"], a["cv"], a["ks"], a["vs"], a["slots_n"], a["cap"], a["start"],
                                       a["slots"], a["B"], a["S"], a["Hk"], a["D"], a["ko"], a["vo"])


def _attn_check(**kw):
    a = dict(q=A, o=A, qst=None, ost=None, ck=A, cv=A, ks=A, vs=A, slots_n=4, cap=128, pk=None, pv=None, pks=None,
             pvs=None, p_n=0, p_cap=0, kv_len=None, q_len=None, slots=None, p_len=None, B=2, S=3, H=4, Hk=2, D=64,
             causal=1, scale=0.125)
    a.update(kw)
    s3 = lambda s: None if s is None else _lib.strides3(s)
    return _lib.lib().vx_cached_attn_check(
        a["q"], a["o"], s3(a["qst"]), s3(a["ost"]), a["ck"], a["cv"], a["ks"], a["vs"], a["slots_n"], a["cap"],
        a["pk"], a["pv"], a["pks"], a["pvs"], a["p_n"], a["p_cap"], a["kv_len"], a["q_len"], a["slots"], a["p_len"],
        a["B"], a["S"], a["H"], a["Hk"], a["D"], a["causal"], ctypes.c_float(a["scale"]))


PREFIX = dict(pk=A, pv=A, pks=A, pvs=A, p_n=1, p_cap=64)


def test_checks_accept_valid_arguments():
    assert _write_check() == _write_check(slots=A, B=9) == _write_check(D=128, kst=(8, 8, 8)) == _lib.VX_OK
    assert _read_check() == _read_check(slots=A, B=9, start=A) == _lib.VX_OK
    assert _attn_check() == _attn_check(slots=A, B=9) == _attn_check(**PREFIX) == _lib.VX_OK
    assert _attn_check(**{**PREFIX, "p_n": 2, "p_len": A}) == _lib.VX_OK
    assert _lib.last_error() == ""


INVALID, UNSUPPORTED = _lib.VX_ERR_INVALID_ARGUMENT, _lib.VX_ERR_UNSUPPORTED
CACHE_REFUSALS = [
    (dict(ck=None), INVALID, "non-NULL"),
    (dict(ks=None), INVALID, "non-NULL"),
    (dict(cv=A + 8), INVALID, "aligned"),
    (dict(vs=A + 4), INVALID, "aligned"),
    (dict(cap=100), INVALID, "capacity"),
    (dict(cap=0), INVALID, "capacity"),
    (dict(slots_n=0), INVALID, ">= 1"),
    (dict(D=96), UNSUPPORTED, "head_dim"),
    (dict(B=0), INVALID, "batch"),
    (dict(B=65536, slots=A), INVALID, "batch"),
    (dict(B=5), INVALID, "slots"),
    (dict(S=0), INVALID, "seq"),
    (dict(slots=A + 2), INVALID, "4-byte"),
]


@pytest.mark.parametrize("check,kw,code,frag", [(c, *r) for c in (_write_check, _read_check, _attn_check)
                                                for r in CACHE_REFUSALS] + [
    (_write_check, dict(k=None), INVALID, "non-NULL"),
    (_write_check, dict(v=A + 2), INVALID, "aligned"),
    (_write_check, dict(Hk=0), INVALID, "num_kv_heads"),
    (_write_check, dict(kst=(1, 8, 8)), INVALID, "multiple of 8"),
    (_write_check, dict(vst=(8, -8, 8)), INVALID, "negative"),
    (_write_check, dict(num=A + 1), INVALID, "4-byte"),
    (_write_check, dict(S=2 ** 31 - 1, Hk=65535), UNSUPPORTED, "too large"),
    (_read_check, dict(ko=None), INVALID, "non-NULL"),
    (_read_check, dict(vo=A + 8), INVALID, "aligned"),
    (_read_check, dict(start=A + 2), INVALID, "4-byte"),
    (_attn_check, dict(q=None), INVALID, "non-NULL"),
    (_attn_check, dict(o=A + 8), INVALID, "aligned"),
    (_attn_check, dict(H=5), INVALID, "multiple of num_kv_heads"),
    (_attn_check, dict(scale=0.0), INVALID, "scale"),
    (_attn_check, dict(scale=float("nan")), INVALID, "scale"),
    (_attn_check, dict(causal=2), INVALID, "causal"),
    (_attn_check, dict(qst=(8, 8, 4)), INVALID, "multiple of 8"),
    (_attn_check, dict(kv_len=A + 2), INVALID, "4-byte"),
    (_attn_check, dict(S=2 ** 30), UNSUPPORTED, "too many"),
    (_attn_check, dict(p_n=1), INVALID, "prefix"),
    (_attn_check, dict(p_len=A), INVALID, "prefix"),
    (_attn_check, dict(PREFIX, pks=None), INVALID, "prefix"),
    (_attn_check, dict(PREFIX, p_n=3, B=4), INVALID, "multiple of num_prefixes"),
    (_attn_check, dict(PREFIX, p_cap=65), INVALID, "capacity"),
    (_attn_check, dict(PREFIX, p_len=A + 2), INVALID, "4-byte"),
    (_attn_check, dict(PREFIX, B=4, S=2 ** 28), UNSUPPORTED, "too many"),
])
def test_checks_refuse(check, kw, code, frag):
    assert check(**kw) == code
    assert frag in _lib.last_error()


@pytest.mark.parametrize("check,fits,refused", [
    (_write_check, dict(S=2 ** 21, Hk=511), dict(S=2 ** 21, Hk=512)),
    (_read_check, dict(S=2 ** 21, Hk=511), dict(S=2 ** 21, Hk=512)),
    # 65535 items of one query: a tile per item and head
    (_attn_check, dict(B=65535, S=1, H=255, Hk=255, slots=A), dict(B=65535, S=1, H=256, Hk=256, slots=A)),
    (_attn_check, dict(B=1, S=2 ** 22, H=127, Hk=127), dict(B=1, S=2 ** 22, H=128, Hk=128)),
    # (a prefix's tiles beside the items' own; its merge's rows)
    (_attn_check, dict(PREFIX, B=2, p_n=2, S=2 ** 21, H=63, Hk=63), dict(PREFIX, B=2, p_n=2, S=2 ** 21, H=64, Hk=64)),
    (_attn_check, dict(PREFIX, B=1, p_n=1, S=2 ** 21, H=63, Hk=63), dict(PREFIX, B=1, p_n=1, S=2 ** 21, H=64, Hk=64)),
])
def test_checks_refuse_grids_past_32_bits(check, fits, refused):
    """The threads of a launch, 64 for 16 positions and 256 for 32 rows, are counted in 32 bits."""
    assert check(**fits) == _lib.VX_OK, _lib.last_error()
    assert check(**refused) == UNSUPPORTED and "too" in _lib.last_error()


@pytest.mark.parametrize("cap,p_cap", [(64, 2 ** 31 - 64), (2 ** 31 - 64, 64), (2 ** 30, 2 ** 30), (1024, 64)])
def test_capacities_whose_sum_passes_32_bits_are_long(cap, p_cap):
    """A prefix and items of more than 1024 positions together are cut into parts, which need a workspace;
    shorter ones take one pass without any."""
    size = _lib.lib().vx_cached_attn_workspace_size
    assert size(cap, 1, p_cap, 1, 1, 1, 1, 64, 0) > 0
    assert size(960, 1, 64, 1, 1, 1, 1, 64, 0) == 0


def test_injected_error_is_reported():
    L = _lib.lib()
    L.vx_debug_inject_error(_lib.VX_ERR_LAUNCH)
    try:
        rc = L.vx_kv_read_fwd(A, A, A, A, 4, 128, None, None, 2, 3, 2, 64, A, A, None)
        assert rc == _lib.VX_ERR_LAUNCH and "injected" in _lib.last_error()
        rc = L.vx_kv_write_fwd(A, A, None, None, A, A, A, A, 4, 128, None, None, None, 2, 3, 2, 64, None)
        assert rc == _lib.VX_ERR_LAUNCH
        rc = L.vx_cached_attn_fwd(A, A, None, None, A, A, A, A, 4, 128, None, None, None, None, 0, 0, None, None, None,
                                  None, 2, 3, 4, 2, 64, 1, ctypes.c_float(0.1), A, 1 << 40, None)
        assert rc == _lib.VX_ERR_LAUNCH
    finally:
        L.vx_debug_inject_error(0)


def test_python_refusals_on_the_host():
    with pytest.raises(ValueError, match="GPU tensor"):
        c = vx.create_kv_cache(2, 64, 2, 64, device="cpu")
        vx.kv_cache_read(c, 4)
    with pytest.raises(TypeError, match="e4m3"):
        vx.kv_cache_read(c._replace(k=c.k.view(torch.uint8)), 4)
    with pytest.raises(ValueError, match="does not go with"):
        vx.kv_cache_read(c._replace(v_scale=c.v_scale[:1]), 4)
    with pytest.raises(NotImplementedError, match="head_dim"):
        vx.create_kv_cache(2, 64, 2, 80, device="cpu")
    with pytest.raises(ValueError, match=">= 1"):
        vx.create_kv_cache(2, 0, 2, 64, device="cpu")
    assert vx.create_kv_cache(2, 65, 3, 128, device="cpu").k.shape == (2, 3, 128, 128)


@pytest.mark.parametrize("make", [tuple, list, lambda c: c._replace(v_scale=None), lambda c: c[:3], lambda c: None])
def test_what_is_no_cache_is_refused(make):
    c = vx.create_kv_cache(1, 64, 1, 64, device="cpu")
    q = torch.zeros((1, 1, 1, 64), dtype=torch.bfloat16)
    for call, name in ((lambda x: vx.kv_cache_write(x, q, q), "cache"), (lambda x: vx.kv_cache_read(x, 1), "cache"),
                       (lambda x: vx.cached_attention(q, x), "cache"),
                       (lambda x: vx.shared_prefix_attention(q, c, x), "cache")):
        with pytest.raises(TypeError, match=f"{name} must be a KVCache"):
            call(make(c))


@pytest.mark.gpu
def test_a_plain_tuple_is_no_prefix(gpu):
    c = vx.create_kv_cache(1, 64, 1, 64, device=gpu)
    q = torch.zeros((1, 1, 1, 64), dtype=torch.bfloat16, device=gpu)
    with pytest.raises(TypeError, match="prefix must be a KVCache"):
        vx.shared_prefix_attention(q, tuple(c), c)


def test_oracle_rounding():
    """The oracle's rows against torch's conversion of the same scaled values."""
    rng = np.random.default_rng(1)
    x = torch.from_numpy(rng.standard_normal((300, 64)) * np.exp(4 * rng.standard_normal((300, 1)))).bfloat16()
    codes, scales = O.quantise(x.double().numpy())
    f = torch.from_numpy(2.0 ** (scales.astype(np.float64) - 127))[:, None]
    want = (x.double() / f).float().to(E4M3).view(torch.uint8).numpy()
    assert (codes == want).all()
    y = np.abs(O.e4m3_values()[codes]).max(-1)
    assert (y <= 448).all() and (y >= 224).all()  # the smallest scale that fits
    assert O.quantise(np.array([[0.0, np.inf], [0.0, 0.0], [448.0, 1.0], [464.0, 464.0]]))[1].tolist() == \
        [255, 1, 127, 128]


# ------------------------------------------------------------------ on the GPU
def _bf16(x, gpu):
    return torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(gpu).to(torch.bfloat16)


def _ints(x, gpu):
    return None if x is None else torch.tensor(x, dtype=torch.int32, device=gpu)


def _rand_rows(rng, *shape):
    """Rows of widely differing magnitudes, some of them zero."""
    x = rng.standard_normal(shape) * np.exp(3 * rng.standard_normal(shape[:-1] + (1,)))
    return x * (rng.random(shape[:-1] + (1,)) > 0.05)


def _bytes(cache):
    return [t.view(torch.uint8).cpu().numpy() for t in cache]


def _noise_cache(rng, slots, Hk, cap, D, gpu):
    """A cache of arbitrary bytes, NaN codes and NaN scales among them."""
    raw = [rng.integers(0, 256, (slots, Hk, cap, D), np.uint8) for _ in range(2)]
    raw += [rng.integers(0, 256, (slots, Hk, cap), np.uint8) for _ in range(2)]
    t = [torch.from_numpy(x).to(gpu) for x in raw]
    return vx.KVCache(t[0].view(E4M3), t[1].view(E4M3), t[2].view(E8M0), t[3].view(E8M0)), raw


@pytest.mark.gpu
@pytest.mark.parametrize("B,S,Hk,D,cap,start,num,slots", [
    (1, 1, 1, 64, 64, None, None, None),
    (1, 1, 1, 128, 64, [63], None, None),
    (3, 17, 2, 128, 128, [0, 5, 111], None, [2, 0, 3]),
    (2, 33, 3, 64, 128, [1, 95], [33, 20], None),
    (2, 16, 12, 128, 64, [48, 0], [0, 16], [1, 0]),
    (4, 50, 1, 64, 64, [30, -10, 64, -60], None, [0, 1, 2, 3]),      # past the end, before the start
    (3, 9, 2, 128, 64, [4, 4, 4], [9, 9, 12], [5, -1, 1]),          # slots that are not there, num past S
    (2, 3, 1, 64, 64, [2 ** 31 - 1, -2 ** 31], None, None),
    (1, 700, 5, 128, 1024, [123], [651], None),
])
def test_write_is_exact_and_leaves_the_rest(gpu, B, S, Hk, D, cap, start, num, slots):
    print(f"[case] write B={B} S={S} Hk={Hk} D={D} cap={cap} start={start} num={num} slots={slots}", flush=True)
    rng = np.random.default_rng(B * S + D)
    cache, want = _noise_cache(rng, 4, Hk, cap, D, gpu)
    k, v = _bf16(_rand_rows(rng, B, S, Hk, D), gpu), _bf16(_rand_rows(rng, B, S, Hk, D), gpu)
    vx.kv_cache_write(cache, k, v, _ints(start, gpu), num=_ints(num, gpu), slots=_ints(slots, gpu))
    torch.cuda.synchronize()
    for x, codes, scales in ((k, want[0], want[2]), (v, want[1], want[3])):
        y, s = O.quantise(x.double().cpu().numpy())
        for b in range(B):
            slot = b if slots is None else slots[b]
            for t in range(S if num is None else min(num[b], S)):
                pos = (0 if start is None else start[b]) + t
                if 0 <= slot < 4 and 0 <= pos < cap:
                    codes[slot, :, pos], scales[slot, :, pos] = y[b, t], s[b, t]
    for got, w, n in zip(_bytes(cache), want, ("k", "v", "k_scale", "v_scale")):
        assert (got == w).all(), (n, np.argwhere(got != w)[:5])


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_write_every_magnitude(gpu, D):
    """Rows scaled over all of bf16's exponents, their largest value on every
    side of a power of two's border, and rows with NaN and infinities."""
    rng = np.random.default_rng(5)
    n = 512
    x = rng.uniform(-1, 1, (1, n, 1, D))
    top = np.array([1.0, 1.75, 1.7578125, 1.9921875])[rng.integers(0, 4, n)] * 2.0 ** np.linspace(-120, 127, n).astype(int)
    x *= top[None, :, None, None]
    x[0, np.arange(n), 0, rng.integers(0, D, n)] = top
    x[0, 7] = 0.0
    x[0, 9, 0, 3] = np.nan
    x[0, 10, 0, D - 1] = np.inf
    x[0, 11, 0, 0] = -np.inf
    x[0, 12] = -0.0
    k = _bf16(x, gpu)
    cache = vx.create_kv_cache(1, n, 1, D, device=gpu)
    vx.kv_cache_write(cache, k, k)
    y, s = O.quantise(k.double().cpu().numpy())
    got = _bytes(cache)
    for at in (0, 1):
        assert (got[at][0, 0] == y[0, :, 0]).all() and (got[2 + at][0, 0] == s[0, :, 0]).all()
    back, _ = vx.kv_cache_read(cache, n)
    want = O.values(y, s)
    # what bf16 holds as a subnormal value may read as zero
    ref = torch.from_numpy(want).to(torch.bfloat16).to(gpu)
    same = (back == ref) | (back.isnan() & ref.isnan()) | ((back == 0) & (ref.abs() < 2.0 ** -126))
    assert same.all()
    assert int(back.isnan().all(-1).sum()) == int(back.isnan().any(-1).sum()) == 3


@pytest.mark.gpu
def test_write_strided_rows(gpu):
    """Slices of a fused projection, a transposed layout and a misaligned view
    give what their contiguous copies give."""
    g = torch.Generator(device=gpu).manual_seed(3)
    fused = torch.randn((2, 21, 3, 4, 64), generator=g, device=gpu).bfloat16()
    heads_first = torch.randn((2, 4, 21, 64), generator=g, device=gpu).bfloat16()
    odd = torch.randn(2 * 21 * 4 * 64 + 1, generator=g, device=gpu).bfloat16()[1:].reshape(2, 21, 4, 64)
    wide = torch.randn((2, 21, 4, 66), generator=g, device=gpu).bfloat16()[..., :64]
    last = torch.randn((2, 21, 64, 4), generator=g, device=gpu).bfloat16().transpose(2, 3)
    one = torch.randn((1, 1, 4, 64), generator=g, device=gpu).bfloat16().expand(2, 21, 4, 64)
    for k, v in ((fused[:, :, 0], fused[:, :, 2]), (heads_first.transpose(1, 2), odd), (wide, last), (one, wide)):
        a, b = (vx.create_kv_cache(2, 64, 4, 64, device=gpu) for _ in range(2))
        vx.kv_cache_write(a, k, v, [3, 40])
        vx.kv_cache_write(b, k.contiguous(), v.contiguous(), [3, 40])
        assert all((x == y).all() for x, y in zip(_bytes(a), _bytes(b)))


@pytest.mark.gpu
def test_same_slot_twice_keeps_the_later_item(gpu):
    rng = np.random.default_rng(11)
    B, S, Hk, D, cap = 70, 20, 2, 128, 256  # (more items than a wave has lanes)
    slots = rng.integers(0, 3, B)
    start = rng.integers(-5, 250, B)
    num = rng.integers(0, S + 1, B)
    k, v = _bf16(_rand_rows(rng, B, S, Hk, D), gpu), _bf16(_rand_rows(rng, B, S, Hk, D), gpu)
    a, b = (vx.create_kv_cache(3, cap, Hk, D, device=gpu) for _ in range(2))
    vx.kv_cache_write(a, k, v, start, num=num, slots=slots)
    for i in range(B):
        vx.kv_cache_write(b, k[i:i + 1], v[i:i + 1], start[i:i + 1], num=num[i:i + 1], slots=slots[i:i + 1])
    for x, y in zip(_bytes(a), _bytes(b)):
        assert (x == y).all()


@pytest.mark.gpu
@pytest.mark.parametrize("B,S,Hk,D,cap,start,slots", [
    (1, 1, 1, 128, 64, [63], None),
    (4, 40, 3, 64, 64, None, None),
    (5, 77, 2, 128, 128, [0, -30, 100, 128, -2 ** 31], [3, 0, 1, 1, 2]),
    (3, 5, 2, 64, 64, [1, 2, 3], [4, -1, 3]),
])
def test_read(gpu, B, S, Hk, D, cap, start, slots):
    print(f"[case] read B={B} S={S} Hk={Hk} D={D} cap={cap} start={start} slots={slots}", flush=True)
    rng = np.random.default_rng(B + S)
    cache = vx.create_kv_cache(4, cap, Hk, D, device=gpu)
    vx.kv_cache_write(cache, _bf16(_rand_rows(rng, 4, cap, Hk, D), gpu), _bf16(_rand_rows(rng, 4, cap, Hk, D), gpu))
    raw = _bytes(cache)
    for got, codes, scales in zip(vx.kv_cache_read(cache, S, _ints(start, gpu), slots=_ints(slots, gpu)), raw, raw[2:]):
        held = O.values(codes, scales)
        want = np.zeros((B, S, Hk, D))
        for b in range(B):
            slot = b if slots is None else slots[b]
            for t in range(S):
                pos = (0 if start is None else start[b]) + t
                if 0 <= slot < 4 and 0 <= pos < cap:
                    want[b, t] = held[slot, :, pos]
        assert (got.double().cpu().numpy() == want).all()


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_read_every_byte(gpu, D):
    """Every value byte but the NaN codes under every scale byte, as a cache made elsewhere may hold them."""
    raw = np.delete(np.arange(256), [0x7f, 0xff]).astype(np.uint8)
    codes = np.stack([np.roll(np.resize(raw, 256 * D), 7 * s).reshape(1, 256, D) for s in range(256)])
    scales = np.broadcast_to(np.arange(256, dtype=np.uint8)[:, None, None], (256, 1, 256)).copy()
    codes[255] = 0
    t = [torch.from_numpy(x).to(gpu) for x in (codes, scales)]
    cache = vx.KVCache(t[0].view(E4M3), t[0].clone().view(E4M3), t[1].view(E8M0), t[1].clone().view(E8M0))
    want = torch.from_numpy(O.values(codes, scales)).transpose(1, 2)  # (slots, positions, 1, D)
    for got in vx.kv_cache_read(cache, 256):
        x = got.double().cpu()
        ref = want.float().bfloat16().double()  # (values have four bits: exact in fp32; in bf16 down to 2^-130)
        same = (x == ref) | (x.isnan() & ref.isnan())
        assert same.all(), [(int(s), float(want[s][~same[s]][0]), float(x[s][~same[s]][0]))
                            for s in (~same).any(-1).any(-1).any(-1).nonzero()[:5, 0]]
        assert ((ref == want) | want.isnan() | (want.abs() < 2.0 ** -126) | (want.abs() >= 2.0 ** 128)).all()


def _cache_of(rng, slots, Hk, cap, D, gpu, lens=None, std=1.0):
    """A cache of random tokens; positions from lens[slot] on hold arbitrary
    bytes (NaN codes and scales among them)."""
    cache, _ = _noise_cache(rng, slots, Hk, cap, D, gpu)
    k = _bf16(std * rng.standard_normal((slots, cap, Hk, D)), gpu)
    v = _bf16(rng.standard_normal((slots, cap, Hk, D)) * np.exp(rng.standard_normal((slots, cap, Hk, 1))), gpu)
    vx.kv_cache_write(cache, k, v, num=None if lens is None else np.minimum(lens, cap))
    return cache


def _held(cache, lens=None):
    """Stored values (k, v) in 64 bits, what lies past lens replaced by zeros."""
    raw = _bytes(cache)
    out = []
    for codes, scales in ((raw[0], raw[2]), (raw[1], raw[3])):
        x = O.values(codes, scales)
        for s in range(x.shape[0] if lens is not None else 0):
            x[s, :, max(int(lens[s]), 0):] = 0.0
        out.append(x)
    return out


def _assert_close(got, q, held, prefix, **kw):
    """The bound of the module's docstring."""
    q64 = q.double().cpu().numpy()
    ref, spread = O.cached_attention(q64, *held, prefix=prefix, **kw)
    D = q.shape[3]
    scale = kw.get("scale") or D ** -0.5
    top = max([np.abs(x[0]).max() for x in (held, prefix) if x is not None and x[0].size] or [0.0])
    L = scale * np.abs(q64).sum(-1).max() * top
    n = held[0].shape[2] + (prefix[0].shape[2] if prefix is not None else 0)
    tol = 2 * 2.0 ** -8 * np.abs(ref) + spread * (2.0 ** -8 + 2 * (D + 2) * 2.0 ** -24 * L + 2 * (n + 64) * 2.0 ** -24)
    err = np.abs(got.double().cpu().numpy() - ref)
    assert not np.isnan(err).any()
    at = np.unravel_index(np.argmax(err - tol), err.shape)
    assert (err <= tol).all(), (at, err[at], tol[at], ref[at])


ATTN = [
    # B, Sq, H, Hk, D, cap, kv_len, q_len, slots, causal
    (1, 1, 1, 1, 128, 64, [1], None, None, True),
    (1, 1, 1, 1, 64, 64, [0], None, None, True),
    (2, 1, 4, 2, 128, 128, [128, 5], None, None, True),
    (3, 1, 8, 1, 64, 320, [300, 0, 31], None, [2, 0, 1], True),
    (5, 1, 16, 2, 128, 1024, [1000, 1, 33, 64, 700], None, None, True),
    (1, 1, 12, 12, 128, 2048, [1999], None, None, True),
    (1, 1, 71, 1, 64, 448, [447], None, None, True),               # more heads per cached head than a tile has rows
    (2, 4, 6, 2, 64, 192, [150, 4], None, None, True),             # a few tokens at once
    (2, 7, 10, 2, 128, 192, [190, 100], [7, 3], None, True),
    (2, 33, 2, 2, 128, 128, [97, 33], None, None, True),           # a whole prompt and a chunk
    (3, 70, 3, 1, 64, 256, [256, 70, 130], [70, 0, 1], [1, 2, 0], True),
    (1, 130, 4, 4, 128, 320, [300], None, None, True),
    (2, 20, 2, 1, 128, 64, [3, 0], [20, 20], None, True),          # queries before the first key
    (2, 40, 4, 2, 64, 128, [77, 128], None, None, False),          # cross attention
    (1, 300, 2, 2, 128, 512, [512], None, None, False),
    (2, 257, 3, 3, 128, 64, [1, 64], [257, 129], None, False),
    (4, 2, 2, 1, 64, 64, [10, 20, 30, 40], None, [0, 7, -1, 3], True),  # slots that are not there
    (3, 1, 4, 4, 128, 64, [1000, -3, 64], [9, 1, -2], None, True),  # lengths held to the sizes
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", ATTN, ids=[str(c) for c in ATTN])
def test_cached_attention(gpu, case):
    B, Sq, H, Hk, D, cap, kv_len, q_len, slots, causal = case
    print(f"[case] cached_attention {case}", flush=True)
    rng = np.random.default_rng(Sq * H + cap)
    n_slots = max(B, 4)
    by_slot = np.zeros(n_slots, int)
    for b in range(B):
        slot = b if slots is None else slots[b]
        if 0 <= slot < n_slots:
            by_slot[slot] = max(by_slot[slot], min(max(kv_len[b], 0), cap))
    cache = _cache_of(rng, n_slots, Hk, cap, D, gpu, by_slot)
    q = _bf16(2 * rng.standard_normal((B, Sq, H, D)), gpu)
    kw = dict(kv_len=kv_len, q_len=q_len, slots=slots, causal=causal)
    got = vx.cached_attention(q, cache, **{k: _ints(x, gpu) if k != "causal" else x for k, x in kw.items()})
    again = vx.cached_attention(q, cache, **kw)
    torch.cuda.synchronize()
    assert torch.equal(got, again)  # the same bits
    _assert_close(got, q, _held(cache, by_slot), None, **kw)


def _lens(rng, B, most):
    """Lengths from none to the most, a third of them very short."""
    n = rng.integers(0, most + 1, B)
    short = rng.random(B) < 0.33
    n[short] = rng.integers(0, 4, short.sum())
    n[rng.integers(0, B)] = most
    return n


@pytest.mark.gpu
@pytest.mark.parametrize("B,Sq,H,Hk,D,cap,causal", [
    (130, 1, 2, 1, 64, 2048, True),       # more items than a wave has lanes, tiles in ranges
    (70, 3, 3, 1, 128, 1088, True),
    (9, 1, 32, 4, 128, 4096, True),
    (1, 1, 4, 1, 64, 16384, True),        # one long sequence over the whole chip
    (66, 20, 4, 1, 64, 1536, True),       # the same with more rows than a tile
    (3, 50, 4, 2, 128, 4096, True),
    (2, 100, 2, 1, 64, 8192, False),
    (1, 700, 5, 1, 128, 2048, True),
])
def test_ranges_over_many_lengths(gpu, B, Sq, H, Hk, D, cap, causal):
    """Batches whose tiles are cut into ranges that end inside streams and span
    empty ones."""
    print(f"[case] ranges B={B} Sq={Sq} H={H} Hk={Hk} D={D} cap={cap} causal={causal}", flush=True)
    rng = np.random.default_rng(B + Sq + cap)
    lens = _lens(rng, B, cap)
    q_len = rng.integers(0, Sq + 1, B) if Sq > 1 else None
    cache = _cache_of(rng, B, Hk, cap, D, gpu, lens)
    q = _bf16(2 * rng.standard_normal((B, Sq, H, D)), gpu)
    kw = dict(kv_len=lens, q_len=q_len, causal=causal)
    got = vx.cached_attention(q, cache, **kw)
    assert torch.equal(got, vx.cached_attention(q, cache, **kw))
    _assert_close(got, q, _held(cache, lens), None, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("B,Sq,H,Hk,D,groups,p_cap,cap", [
    (130, 1, 2, 1, 64, 65, 1024, 1088),   # two sharers each, more groups than a wave has lanes
    (12, 1, 8, 2, 128, 1, 4096, 128),     # 48 rows on one prefix
    (12, 1, 8, 2, 64, 3, 2048, 2048),     # ranges on both sides
    (4, 30, 4, 2, 128, 2, 1536, 1536),
    (64, 1, 1, 1, 128, 64, 128, 64),      # every item a prefix of its own, in one pass
    (2, 600, 8, 8, 128, 2, 64, 2048),     # a short prefix in front of long prompts
    (2, 300, 4, 4, 64, 1, 4096, 320),     # the other way
])
def test_prefixes_over_many_lengths(gpu, B, Sq, H, Hk, D, groups, p_cap, cap):
    print(f"[case] prefixes B={B} Sq={Sq} H={H} Hk={Hk} D={D} groups={groups} p_cap={p_cap} cap={cap}", flush=True)
    rng = np.random.default_rng(B + Sq + p_cap)
    lens, p_len = _lens(rng, B, cap), _lens(rng, groups, p_cap)
    q_len = rng.integers(0, Sq + 1, B) if Sq > 1 else None
    cache, prefix = _cache_of(rng, B, Hk, cap, D, gpu, lens), _cache_of(rng, groups, Hk, p_cap, D, gpu, p_len)
    q = _bf16(2 * rng.standard_normal((B, Sq, H, D)), gpu)
    kw = dict(kv_len=lens, prefix_len=p_len, q_len=q_len)
    got = vx.shared_prefix_attention(q, prefix, cache, **kw)
    assert torch.equal(got, vx.shared_prefix_attention(q, prefix, cache, **kw))
    _assert_close(got, q, _held(cache, lens), _held(prefix, p_len), **kw)


@pytest.mark.gpu
def test_cached_attention_defaults_strides_and_out(gpu):
    """Full caches, a scale of the caller's, strided and misaligned queries and
    an output of the caller's."""
    rng = np.random.default_rng(2)
    cache = _cache_of(rng, 3, 2, 192, 64, gpu)
    fused = _bf16(rng.standard_normal((3, 5, 3, 8, 64)), gpu)
    odd = _bf16(rng.standard_normal(3 * 5 * 8 * 64 + 3), gpu)[3:].reshape(3, 5, 8, 64)
    spread = _bf16(rng.standard_normal((3, 5, 64, 8)), gpu).transpose(2, 3)
    for q in (fused[:, :, 1], odd, spread, fused[:, :1, 2], fused[:1, :1, 0, :1].expand(3, 5, 8, 64)):
        out = torch.full((3, q.shape[1] + 2, 10, 64), 7.0, dtype=torch.bfloat16, device=gpu)
        got = vx.cached_attention(q, cache, causal=False, scale=0.3, out=out[:, 1:-1, 1:9])
        assert got.data_ptr() == out[:, 1:-1, 1:9].data_ptr()
        _assert_close(got, q, _held(cache), None, causal=False, scale=0.3)
        rest = out.clone()
        rest[:, 1:-1, 1:9] = 7.0
        assert (rest == 7.0).all()  # nothing beside the output rows


PLANS = [
    # kernel, parts (the workspace holds some); B, Sq, H, Hk, D, cap, kv_len, q_len, causal; groups, prefix cap, prefix_len
    ("many_kernel<128>", False, 2, 500, 32, 4, 128, 640, [640, 577], [500, 333], True, 0, 0, None),
    ("many_kernel<64>", False, 4, 500, 32, 4, 64, 640, [601, 1, 0, 640], [499, 500, 17, 0], True, 0, 0, None),
    ("many_kernel<128>", False, 2, 500, 32, 4, 128, 640, [63, 640], [500, 500], False, 0, 0, None),
    ("many_kernel<64>", False, 4, 500, 32, 4, 64, 640, [601, 1, 0, 640], [499, 500, 17, 0], False, 0, 0, None),
    ("many_kernel<128>", True, 3, 300, 8, 8, 128, 3520, [3500, 0, 1777], [300, 7, 299], True, 0, 0, None),
    ("many_kernel<64>", True, 3, 300, 8, 8, 64, 7040, [7040, 129, 3333], [299, 300, 1], True, 0, 0, None),
    ("many_kernel<128>", True, 3, 300, 8, 8, 128, 3520, [1, 3520, 65], None, False, 0, 0, None),
    ("many_kernel<64>", True, 3, 300, 8, 8, 64, 7040, [0, 5001, 7000], [200, 300, 300], False, 0, 0, None),
    ("prefix_kernel<128, false, true>", True, 16, 16, 16, 8, 128, 128, [3 + 8 * i for i in range(16)], None, True, 1, 4288,
     [4201]),
    ("prefix_kernel<64, false, true>", True, 16, 16, 16, 8, 64, 128, [8 * i for i in range(16)], [i + 1 for i in range(16)],
     True, 2, 8576, [8576, 31]),
    ("prefix_kernel<128, false, false>", True, 2, 500, 32, 4, 128, 640, [600, 501], [499, 500], True, 1, 640, [601]),
    ("prefix_kernel<64, false, false>", True, 4, 500, 32, 4, 64, 640, [600, 0, 640, 1], [499, 500, 1, 77], True, 2, 1280,
     [1201, 0]),
    ("prefix_kernel<128, true, false>", True, 2, 500, 32, 4, 128, 640, [600, 501], [499, 500], True, 1, 64, [33]),
    ("prefix_kernel<64, true, false>", True, 4, 500, 32, 4, 64, 640, [600, 0, 640, 1], None, False, 1, 64, [64]),
    ("prefix_kernel<128, true, true>", True, 4, 5, 8, 2, 128, 2048, [2048, 5, 0, 700], [5, 1, 2, 4], True, 2, 192, [192, 1]),
    ("prefix_kernel<64, true, true>", True, 4, 5, 8, 2, 64, 64, [64, 5, 0, 33], None, True, 1, 2048, [2001]),
    ("few_kernel<128, 4, false>", True, 4, 1, 8, 2, 128, 2048, [2048, 5, 0, 700], None, True, 0, 0, None),
    ("few_kernel<64, 4, false>", True, 2, 9, 8, 2, 64, 4096, [4001, 9], [9, 8], True, 0, 0, None),
    ("few_kernel<64, 8, false>", False, 3, 5, 4, 2, 64, 320, [320, 5, 100], [5, 5, 2], True, 0, 0, None),
    ("few_kernel<64, 4, true>", False, 40, 1, 16, 8, 64, 64, [i % 65 for i in range(40)], None, True, 2, 192, [190, 1]),
    ("few_kernel<64, 8, true>", False, 2, 3, 4, 2, 64, 64, [64, 3], [3, 2], True, 1, 192, [190]),
    ("few_kernel<128, 8, false>", False, 3, 5, 4, 2, 128, 320, [320, 5, 100], [5, 5, 2], True, 0, 0, None),
    ("few_kernel<128, 4, true>", False, 40, 1, 16, 8, 128, 64, [i % 65 for i in range(40)], None, True, 2, 192, [190, 1]),
    ("few_kernel<128, 8, true>", False, 2, 3, 4, 2, 128, 64, [64, 3], [3, 2], True, 1, 192, [190]),
    ("few_kernel<128, 4, false>", False, 3, 1, 4, 2, 128, 128, [100, 0, 128], None, True, 0, 0, None),
    ("few_kernel<64, 4, false>", False, 3, 40, 4, 2, 64, 128, [100, 0, 128], [40, 3, 39], False, 0, 0, None),
]


def _attend(case, gpu, cache, prefix, q):
    """The call of a case of PLANS, on the kernel that it is there for."""
    kernel, parts, B, Sq, H, Hk, D, cap, kv_len, q_len, causal, groups, p_cap, p_len = case
    kw = dict(q_len=_ints(q_len, gpu), causal=causal)
    size = _lib.lib().vx_cached_attn_workspace_size(cap, groups, p_cap, B, Sq, H, Hk, D, int(not causal and q_len is None))
    assert (size > 0) == parts
    if groups:
        got = vx.shared_prefix_attention(q, prefix, cache, _ints(kv_len, gpu), prefix_len=_ints(p_len, gpu), **kw)
    else:
        got = vx.cached_attention(q, cache, _ints(kv_len, gpu), **kw)
    assert _lib.last_launch() == kernel
    return got


PLAN_IDS = [f"{c[0]}{' parts' if c[1] else ''}{'' if c[10] else ' cross'}" for c in PLANS]


@pytest.mark.gpu
@pytest.mark.parametrize("case", PLANS, ids=PLAN_IDS)
def test_every_kernel_of_the_plan(gpu, case):
    kernel, _, B, Sq, H, Hk, D, cap, kv_len, q_len, causal, groups, p_cap, p_len = case
    print(f"[case] {case}", flush=True)
    rng = np.random.default_rng(Sq + cap + p_cap + D)
    cache = _cache_of(rng, B, Hk, cap, D, gpu, kv_len)
    prefix = _cache_of(rng, groups, Hk, p_cap, D, gpu, p_len) if groups else None
    q = _bf16(2 * rng.standard_normal((B, Sq, H, D)), gpu)
    if q_len is not None:  # (padding rows may hold anything)
        for b, n in enumerate(q_len):
            q[b, n:] = float("nan")
    got = _attend(case, gpu, cache, prefix, q)
    assert torch.equal(got, _attend(case, gpu, cache, prefix, q))
    if q_len is not None:
        for b, n in enumerate(q_len):
            q[b, n:] = 0.0
    _assert_close(got, q, _held(cache, kv_len), _held(prefix, p_len) if groups else None, kv_len=kv_len, q_len=q_len,
                  causal=causal, **(dict(prefix_len=p_len) if groups else {}))


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("case", PLANS, ids=PLAN_IDS)
def test_nan_rows_in_every_kernel_of_the_plan(gpu, case, which):
    """A NaN token of the cache, then one of the prefix, reaches the queries of its
    head that see it and no others, through ranges and merges too."""
    kernel, _, B, Sq, H, Hk, D, cap, kv_len, q_len, causal, groups, p_cap, p_len = case
    print(f"[case] NaN in {which}, {case}", flush=True)
    rng = np.random.default_rng(9)
    b, head = int(np.argmax(np.minimum(kv_len, q_len or [Sq] * B))), Hk - 1
    m, n = (q_len[b] if q_len else Sq), kv_len[b]
    for where in ("own", "prefix") if groups else ("own",):
        at = n - (m + 1) // 2 if where == "own" else p_len[0] // 2
        caches = []
        for slots, positions, spot in ((B, cap, b if where == "own" else -1),
                                       (groups, p_cap, 0 if where == "prefix" else -1)):
            if slots == 0:
                caches.append(None)
                continue
            x = {i: rng.standard_normal((slots, positions, Hk, D)) for i in "kv"}
            if spot >= 0:
                x[which][spot, max(at, 0), head, 11] = np.nan
            caches.append(vx.create_kv_cache(slots, positions, Hk, D, device=gpu))
            vx.kv_cache_write(caches[-1], _bf16(x["k"], gpu), _bf16(x["v"], gpu))
        q = _bf16(rng.standard_normal((B, Sq, H, D)), gpu)
        got = _attend(case, gpu, *caches, q)
        want = torch.zeros((B, Sq, H, D), dtype=torch.bool, device=gpu)
        G = H // Hk
        if where == "own":
            first = max(at, 0) - n + m if causal else 0  # the first query that sees it
            want[b, max(first, 0):m, head * G:] = True
        else:
            for i in range(B // groups):
                want[i, :q_len[i] if q_len else Sq, head * G:] = True
        assert torch.equal(got.isnan(), want), where


@pytest.mark.gpu
@pytest.mark.parametrize("case", PLANS, ids=PLAN_IDS)
def test_queries_that_are_not_finite(gpu, case):
    """A NaN and an infinite query row become NaN, whatever their neighbours in a tile."""
    kernel, _, B, Sq, H, Hk, D, cap, kv_len, q_len, causal, groups, p_cap, p_len = case
    print(f"[case] {case}", flush=True)
    rng = np.random.default_rng(Sq + cap + p_cap)
    cache = _cache_of(rng, B, Hk, cap, D, gpu, kv_len)
    prefix = _cache_of(rng, groups, Hk, p_cap, D, gpu, p_len) if groups else None
    q = _bf16(2 * rng.standard_normal((B, Sq, H, D)), gpu)
    b = int(np.argmax(np.minimum(kv_len, q_len or [Sq] * B)))
    last = (q_len[b] if q_len else Sq) - 1
    q[b, last, 0], q[b, last, H - 1] = 0.0, 0.0
    finite = _attend(case, gpu, cache, prefix, q)
    bad = q.clone()
    bad[b, last, 0, 5], bad[b, last, H - 1] = float("nan"), float("inf")
    got = _attend(case, gpu, cache, prefix, bad)
    want = torch.zeros(got.shape, dtype=torch.bool, device=gpu)
    want[b, last, 0], want[b, last, H - 1] = True, True
    assert torch.equal(got.isnan(), want)
    _assert_close(torch.where(want, finite, got), q, _held(cache, kv_len), _held(prefix, p_len) if groups else None,
                  kv_len=kv_len, q_len=q_len, causal=causal, **(dict(prefix_len=p_len) if groups else {}))


@pytest.mark.gpu
@pytest.mark.parametrize("case", [PLANS[0], PLANS[4], PLANS[11], None], ids=["many", "many in parts", "prefix", "expanded"])
def test_graph_replays_of_long_calls(gpu, case):
    """Captured calls of many queries (with prefixes, in parts, expanded to bf16),
    replayed while lengths, queries and eager calls between the replays change;
    every replay equals the eager result bit for bit."""
    if case is None:
        case = ("flash", True, 1, 4224, 72, 72, 64, 128, [128], None, False, 0, 0, None)
    kernel, _, B, Sq, H, Hk, D, cap, _, q_len, causal, groups, p_cap, _ = case
    print(f"[case] replays of {case}", flush=True)
    rng = np.random.default_rng(10)
    cache = _cache_of(rng, B, Hk, cap, D, gpu)
    prefix = _cache_of(rng, groups, Hk, p_cap, D, gpu) if groups else None
    q = torch.empty((B, Sq, H, D), dtype=torch.bfloat16, device=gpu)
    kv_len, m = (torch.zeros(B, dtype=torch.int32, device=gpu) for _ in range(2))
    p_len = torch.zeros(max(groups, 1), dtype=torch.int32, device=gpu)

    def call():
        kw = dict(q_len=m if q_len is not None else None, causal=causal)
        if groups:
            return vx.shared_prefix_attention(q, prefix, cache, kv_len, prefix_len=p_len, **kw)
        return vx.cached_attention(q, cache, kv_len, **kw)

    def set_inputs(share):
        for t, most in ((kv_len, cap), (m, Sq), (p_len, p_cap)):
            t.copy_(torch.tensor([int(most * share) // (i + 1) for i in range(t.numel())], dtype=torch.int32))
        q.copy_(torch.randn(q.shape, device=gpu))

    set_inputs(1.0)
    call()  # warm-up
    assert _lib.last_launch().startswith(kernel)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for share in (1.0, 0.37, 0.0, 0.9):
        set_inputs(share)
        want = call()  # eager work between the replays
        torch.cuda.synchronize()
        out.fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        print(f"  replay at {share}", flush=True)
        assert torch.equal(out, want)


PREFIXES = [
    # B, Sq, H, Hk, D, groups, prefix cap, prefix_len, cap, kv_len, q_len, slots, causal
    (1, 1, 1, 1, 64, 1, 64, [64], 64, [1], None, None, True),
    (4, 1, 8, 2, 128, 1, 320, [300], 64, [0, 1, 20, 64], None, None, True),
    (6, 1, 4, 4, 64, 2, 192, [190, 0], 64, [5, 0, 64, 0, 0, 7], None, None, True),  # a group without a prefix
    (6, 3, 6, 2, 128, 3, 128, [128, 1, 65], 128, [3, 9, 100, 128, 3, 4], [3, 1, 2, 3, 0, 3], [5, 4, 3, 2, 1, 0], True),
    (2, 50, 4, 1, 64, 1, 448, [401], 64, [50, 60], [50, 33], None, True),
    (40, 1, 16, 2, 128, 1, 704, [701], 64, [i % 65 for i in range(40)], None, None, True),
    (4, 20, 3, 3, 128, 2, 64, [33, 2000], 64, [64, 1, 5, 9], None, [0, 9, 1, 2], False),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", PREFIXES, ids=[str(c[:9]) for c in PREFIXES])
def test_shared_prefix_attention(gpu, case):
    B, Sq, H, Hk, D, groups, p_cap, p_len, cap, kv_len, q_len, slots, causal = case
    print(f"[case] shared_prefix_attention {case}", flush=True)
    rng = np.random.default_rng(B + Sq + p_cap)
    by_slot = np.zeros(B, int)
    for b in range(B):
        slot = b if slots is None else slots[b]
        if 0 <= slot < B:
            by_slot[slot] = kv_len[b]
    cache = _cache_of(rng, B, Hk, cap, D, gpu, by_slot)
    p_held = np.minimum(p_len, p_cap)
    prefix = _cache_of(rng, groups, Hk, p_cap, D, gpu, p_held)
    q = _bf16(2 * rng.standard_normal((B, Sq, H, D)), gpu)
    kw = dict(kv_len=kv_len, prefix_len=p_len, q_len=q_len, slots=slots, causal=causal)
    got = vx.shared_prefix_attention(q, prefix, cache, **kw)
    again = vx.shared_prefix_attention(q, prefix, cache, **kw)
    torch.cuda.synchronize()
    assert torch.equal(got, again)
    _assert_close(got, q, _held(cache, by_slot), _held(prefix, p_held), **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("Sq", [1, 5, 40])
@pytest.mark.parametrize("which", ["k", "v"])
def test_nan_rows_reach_only_the_queries_that_see_them(gpu, Sq, which):
    """A NaN token makes NaN the outputs of its head's queries from its position
    on, and no other's, though they share tiles; the same for a prefix's."""
    rng = np.random.default_rng(4)
    B, H, Hk, D, cap, n = 2, 4, 2, 128, 128, 100
    k, v = (rng.standard_normal((B, cap, Hk, D)) for _ in range(2))
    at = n - (Sq + 1) // 2  # seen by the last queries of item 0, head group 1
    (k if which == "k" else v)[0, at, 1, 17] = np.inf
    cache = vx.create_kv_cache(B, cap, Hk, D, device=gpu)
    vx.kv_cache_write(cache, _bf16(k, gpu), _bf16(v, gpu))
    q = _bf16(rng.standard_normal((B, Sq, H, D)), gpu)
    got = vx.cached_attention(q, cache, [n, n])
    want = torch.zeros((B, Sq, H, D), dtype=torch.bool, device=gpu)
    want[0, at - n + Sq:, 2:] = True
    assert torch.equal(got.isnan(), want)
    own = vx.create_kv_cache(B, 64, Hk, D, device=gpu)
    got = vx.shared_prefix_attention(q, cache, own, [0, 0], prefix_len=[n, n])
    want[0, :, 2:] = True
    assert torch.equal(got.isnan(), want)


@pytest.mark.gpu
def test_large_logits_and_rows(gpu):
    """Logits far apart (one key takes all the weight) and values of 2^110: no
    overflow on the way."""
    D, n = 128, 300
    rng = np.random.default_rng(8)
    q = _bf16(40 * rng.standard_normal((1, 1, 2, D)), gpu)
    k = 40 * rng.standard_normal((1, n, 1, D))
    v = np.where(rng.random((1, n, 1, D)) < 0.5, -1, 1) * 2.0 ** 110
    cache = vx.create_kv_cache(1, n, 1, D, device=gpu)
    vx.kv_cache_write(cache, _bf16(k, gpu), _bf16(v, gpu))
    got = vx.cached_attention(q, cache, [n]).double().cpu().numpy()
    hk, hv = _held(cache)
    ref, _ = O.cached_attention(q.double().cpu().numpy(), hk, hv, kv_len=[n])
    # logits of ~1e4: fp32 sums are off by up to (D + 2) 2^-24 of sum |q k|, ~0.1, which moves a
    # weight by at most 20 %; one key holds nearly all of it
    assert np.isfinite(got).all() and np.abs(got - ref).max() <= 0.25 * 2.0 ** 110


LARGE = [  # B, Sq, H, Hk, D, cap, kv_len, prefix capacity, kernel
    (2, 1, 4, 2, 128, 128, [128, 77], 0, "few_kernel<128"),
    (2, 3, 4, 2, 64, 2048, [2048, 1999], 0, "few_kernel<64"),           # in ranges
    (2, 512, 32, 4, 128, 576, [576, 500], 0, "many_kernel<128>"),
    (4, 512, 32, 4, 64, 576, [576, 500, 1, 64], 0, "many_kernel<64>"),
    (2, 1, 4, 2, 128, 64, [64, 20], 192, "few_kernel<128, 8, true>"),
    (2, 5, 8, 2, 64, 64, [64, 20], 2048, "prefix_kernel<64"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("size", [-2.0 ** 125, -2.0 ** 105, -2.0 ** 40, -2.0 ** 25, 2.0 ** 25, 2.0 ** 40, 2.0 ** 125])
@pytest.mark.parametrize("case", LARGE, ids=[c[-1] + ("" if c[5] < 2048 else " in ranges") for c in LARGE])
def test_logits_of_any_size(gpu, case, size):
    """Logits of 2^25 to 2^125 of either sign: all weight on the keys of the largest
    one, evenly. (The products are exact, one dim each, and the logits differ by an
    eighth or more of their size, so the weights are equal or nothing, and their
    rounding is one common factor of at most 2^-8: the bound of the module's docstring
    without its term for inexact logits.)"""
    B, Sq, H, Hk, D, cap, kv_len, p_cap, kernel = case
    print(f"[case] logits of {size} in {case}", flush=True)
    rng = np.random.default_rng(17)

    def cache_of(n, positions):
        k = np.zeros((n, positions, Hk, D))
        k[..., 5] = rng.choice([1.0, 1.125, 1.25, 1.5, 1.75], (n, positions, Hk))
        c = vx.create_kv_cache(n, positions, Hk, D, device=gpu)
        vx.kv_cache_write(c, _bf16(k * 2.0 ** 60, gpu), _bf16(rng.standard_normal(k.shape), gpu))
        return c

    cache, q = cache_of(B, cap), np.zeros((B, Sq, H, D))
    q[..., 5] = size / 2.0 ** 60
    q = _bf16(q, gpu)
    kw = dict(kv_len=kv_len, causal=True, scale=1.0)
    prefix = None
    if p_cap:
        prefix = cache_of(1, p_cap)
        got = vx.shared_prefix_attention(q, prefix, cache, _ints(kv_len, gpu), prefix_len=_ints([p_cap - 30], gpu), scale=1.0)
        kw["prefix_len"] = [p_cap - 30]
    else:
        got = vx.cached_attention(q, cache, _ints(kv_len, gpu), scale=1.0)
    assert _lib.last_launch().startswith(kernel)
    ref, spread = O.cached_attention(q.double().cpu().numpy(), *_held(cache), prefix=_held(prefix) if p_cap else None, **kw)
    tol = 2 * 2.0 ** -8 * np.abs(ref) + spread * (2.0 ** -8 + 2 * (cap + p_cap + 64) * 2.0 ** -24)
    err = np.abs(got.double().cpu().numpy() - ref)
    assert (err <= tol).all(), (np.argwhere(~(err <= tol))[:3], np.isnan(err).sum())


EVEN = LARGE + [(2, 257, 3, 3, 64, 320, [320, 77], 0, "few_kernel<64"), (1, 4096, 74, 74, 128, 128, [100], 0, "flash_")]


@pytest.mark.gpu
@pytest.mark.parametrize("case", EVEN, ids=[c[-1] + f" {c[5]}" for c in EVEN])
def test_the_weights_sum_to_one(gpu, case):
    """Values that are the same for all keys come out as they are, bit for bit: the
    sum that divides is that of the weights that multiply them. Here all weights but
    one of 32 are 2^-0.99609, which bf16 rounds down by 0.27 %: over the sum of the
    unrounded ones, a value 1 would become 1 - 2^-8. (fp32 sums of 2^12 terms are off by
    2^-12 at most, half a step of bf16 below 1 is 2^-9.)"""
    B, Sq, H, Hk, D, cap, kv_len, p_cap, kernel = case
    print(f"[case] weights of {case}", flush=True)

    def cache_of(n, positions):
        c = vx.create_kv_cache(n, positions, Hk, D, device=gpu)
        k, v = np.zeros((n, positions, Hk, D)), np.ones((n, positions, Hk, D))
        k[..., 3] = -1.0
        k[:, ::32] = 0.0
        vx.kv_cache_write(c, _bf16(k, gpu), _bf16(v * 2.0 ** np.arange(-3, Hk - 3)[:, None], gpu))
        return c

    cache = cache_of(B, cap)
    q, n = torch.full((B, Sq, H, D), 0.99609375, dtype=torch.bfloat16, device=gpu), _ints(kv_len, gpu)
    scale = float(np.log(2.0))  # (logits in log2 units)
    if p_cap:
        got = vx.shared_prefix_attention(q, cache_of(1, p_cap), cache, n, prefix_len=_ints([p_cap - 30], gpu), scale=scale)
    else:
        got = vx.cached_attention(q, cache, n, causal=kernel != "flash_", scale=scale)
    assert _lib.last_launch().startswith(kernel)
    want = vx.kv_cache_read(cache, 1)[1][:1].repeat_interleave(H // Hk, 2).expand(B, Sq, H, D).clone()
    if kernel != "flash_" and not p_cap:  # (causal queries in front of the first key see none)
        for b, m in enumerate(kv_len):
            want[b, :max(Sq - m, 0)] = 0
    assert torch.equal(got, want), int((got != want).sum())


@pytest.mark.gpu
def test_offsets_past_32_bits(gpu):
    """The last slot of a cache whose arrays are above 4 GiB."""
    n_slots, Hk, cap, D = 34, 8, 131072, 128
    shape = (n_slots, Hk, cap)
    cache = vx.KVCache(*(torch.empty(shape + (D,), dtype=torch.uint8, device=gpu).view(E4M3) for _ in range(2)),
                       *(torch.empty(shape, dtype=torch.uint8, device=gpu).view(E8M0) for _ in range(2)))
    assert cache.k.numel() > 1 << 32
    rng = np.random.default_rng(3)
    S, first = 200, cap - 200
    k, v = _bf16(rng.standard_normal((1, S, Hk, D)), gpu), _bf16(rng.standard_normal((1, S, Hk, D)), gpu)
    vx.kv_cache_write(cache, k, v, [first], slots=[n_slots - 1])
    bk, bv = vx.kv_cache_read(cache, S, [first], slots=[n_slots - 1])
    for got, x in ((bk, k), (bv, v)):
        assert (got.double().cpu().numpy() == O.values(*O.quantise(x.double().cpu().numpy()))).all()
    # all positions but the last 200 given scale 1, bytes 0: weight exp(0) on zero values
    for t in cache[:2]:
        t[n_slots - 1, :, :first].view(torch.uint8).zero_()
    for t in cache[2:]:
        t[n_slots - 1, :, :first].view(torch.uint8).fill_(127)
    q = _bf16(3 * rng.standard_normal((1, 1, 2 * Hk, D)), gpu)
    got = vx.cached_attention(q, cache, [cap], slots=[n_slots - 1])
    s = torch.einsum("hd,shd->hs", q[0, 0].double(), bk[0].double().repeat_interleave(2, 1)) * D ** -0.5
    w = s.exp()
    total = w.sum(-1) + first
    ref = torch.einsum("hs,shd->hd", w, bv[0].double().repeat_interleave(2, 1)) / total[:, None]
    spread = torch.einsum("hs,shd->hd", w, bv[0].double().abs().repeat_interleave(2, 1)) / total[:, None]
    L = float((q[0, 0].double().abs().sum(-1) * bk.double().abs().max()).max() * D ** -0.5)
    tol = 2.0 ** -8 * ref.abs() + spread * (2.0 ** -8 + 2 * (D + 2) * 2.0 ** -24 * L + 2 * (cap + 64) * 2.0 ** -24)
    assert ((got[0, 0].double() - ref).abs() <= tol).all()


@pytest.mark.gpu
def test_rollout_on_another_stream(gpu):
    """The operators together, as a rollout uses them: a template written once
    for all samples, each sample's prompt in a padded chunk, then tokens one by
    one, on a stream of its own; every step against the oracle on the stored
    values, and kv_cache_read against the cache."""
    rng = np.random.default_rng(21)
    B, H, Hk, D, P = 5, 8, 2, 128, 150
    prefix = vx.create_kv_cache(1, P, Hk, D, device=gpu)
    cache = vx.create_kv_cache(B, 64, Hk, D, device=gpu)
    stream = torch.cuda.Stream(gpu)
    with torch.cuda.stream(stream):
        pk, pv = _bf16(rng.standard_normal((1, P, Hk, D)), gpu), _bf16(rng.standard_normal((1, P, Hk, D)), gpu)
        vx.kv_cache_write(prefix, pk, pv)
        lens = np.zeros(B, np.int64)
        for Sq, num in ((30, [30, 12, 1, 25, 17]), (1, [1] * B), (1, [1] * B), (2, [2, 1, 2, 0, 1]), (1, [1] * B)):
            k, v = (_bf16(rng.standard_normal((B, Sq, Hk, D)), gpu) for _ in range(2))
            q = _bf16(2 * rng.standard_normal((B, Sq, H, D)), gpu)
            vx.kv_cache_write(cache, k, v, _ints(lens, gpu), num=_ints(num, gpu))
            lens = lens + num
            got = vx.shared_prefix_attention(q, prefix, cache, _ints(lens, gpu), prefix_len=[P], q_len=_ints(num, gpu))
            alone = vx.cached_attention(q, cache, _ints(lens, gpu), q_len=_ints(num, gpu))
            back = vx.kv_cache_read(cache, 64)
            stream.synchronize()
            held, shared = _held(cache, lens), _held(prefix, [P])
            _assert_close(got, q, held, shared, kv_len=lens, prefix_len=[P], q_len=num)
            _assert_close(alone, q, held, None, kv_len=lens, q_len=num)
            for x, h in zip(back, _held(cache)):
                assert (x.double().cpu().numpy() == h.transpose(0, 2, 1, 3)).all()


@pytest.mark.gpu
def test_graph_replays_follow_the_lengths(gpu):
    """A decoding step (write, then attention with and without a prefix)
    captured once and replayed while positions, lengths, tokens and eager calls
    between the replays change; two graphs live at once. Every replay equals the
    eager result bit for bit."""
    rng = np.random.default_rng(6)
    B, H, Hk, D, cap = 6, 16, 2, 128, 2048
    prefix = _cache_of(rng, 2, Hk, 320, D, gpu)
    base = _cache_of(rng, B, Hk, cap, D, gpu)
    dup = lambda c: vx.KVCache(*(t.clone() for t in c))
    live = dup(base)
    q = torch.empty((B, 1, H, D), dtype=torch.bfloat16, device=gpu)
    k, v = (torch.empty((B, 1, Hk, D), dtype=torch.bfloat16, device=gpu) for _ in range(2))
    start, kv_len = (torch.zeros(B, dtype=torch.int32, device=gpu) for _ in range(2))
    p_len = torch.zeros(2, dtype=torch.int32, device=gpu)

    def step(cache):
        vx.kv_cache_write(cache, k, v, start)
        return (vx.cached_attention(q, cache, kv_len),
                vx.shared_prefix_attention(q, prefix, cache, kv_len, prefix_len=p_len))

    def set_inputs(lens, p):
        n = torch.tensor(lens, dtype=torch.int32, device=gpu)
        start.copy_(n - 1)
        kv_len.copy_(n)
        p_len.copy_(torch.tensor(p, dtype=torch.int32, device=gpu))
        for t in (q, k, v):
            t.copy_(_bf16(rng.standard_normal(tuple(t.shape)), gpu))

    set_inputs([1] * B, [1, 1])
    step(live)  # warm-up
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(live))
        graphs.append(g)
    for r, (lens, p) in enumerate([([2048, 1, 7, 700, 64, 65], [320, 0]), ([1] * B, [0, 0]),
                                   ([2000] * B, [1, 319]), ([33, 2048, 1, 2, 3, 1500], [64, 65])]):
        set_inputs(lens, p)
        for t, s in zip(live, base):
            t.copy_(s)
        ref = step(dup(base))  # eager work between the replays
        torch.cuda.synchronize()
        for g, out in zip(graphs, outs):
            for o in out:
                o.fill_(9.0)
            g.replay()
            torch.cuda.synchronize()
            print(f"  replay {r}", flush=True)
            assert all(torch.equal(o, e) for o, e in zip(out, ref))


def _step_with_host_integers(cache, x, host):
    """Every operator once, its integers on the host."""
    vx.kv_cache_write(cache, x, x, host([3, 9]), num=host([1, 1]), slots=host([1, 0]))
    return (*vx.kv_cache_read(cache, 64, slots=host([1, 0])), vx.cached_attention(x, cache, host([4, 20])),
            vx.shared_prefix_attention(x, cache, cache, host([20, 4]), prefix_len=host([7, 8]), q_len=host([1, 0])))


HOST = {"list": list, "numpy": np.array, "tensor": torch.tensor, "int32": lambda v: torch.tensor(v, dtype=torch.int32),
        "pinned": lambda v: torch.tensor(v, dtype=torch.int32).pin_memory()}


@pytest.mark.gpu
@pytest.mark.parametrize("host", HOST.values(), ids=list(HOST))
def test_host_integers_wait_for_nothing(gpu, host):
    """Calls whose lengths, positions and slots are host values return while the
    stream is still at work, and give what device tensors give; the caller may
    change its values as soon as the call returns."""
    g = torch.Generator(device=gpu).manual_seed(12)
    x = torch.randn((2, 1, 2, 64), generator=g, device=gpu).bfloat16()
    caches = [vx.create_kv_cache(2, 64, 2, 64, device=gpu) for _ in range(3)]
    work = torch.randn((8192, 8192), generator=g, device=gpu).bfloat16()
    want = _step_with_host_integers(caches[0], x, lambda v: _ints(v, gpu))
    made = []

    def given(v):
        made.append(host(v))
        return made[-1]

    for c in caches[1:]:  # (the first pass may still allocate)
        torch.cuda.synchronize()
        for _ in range(40):  # about 35 ms
            torch.matmul(work, work)
        busy = torch.cuda.Event()
        busy.record()
        got = _step_with_host_integers(c, x, given)
        waited = busy.query()
        for m in made:
            for i in range(2):
                m[i] = 63
        made.clear()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert all((a == b).all() for a, b in zip(_bytes(c), _bytes(caches[0])))
    assert not waited


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.uint8, torch.int16, torch.uint16, torch.uint32, torch.int64, torch.uint64])
@pytest.mark.parametrize("on", ["host", "gpu"])
def test_integers_of_any_type(gpu, dtype, on):
    """Integers of other types than int32 count as what they are: the largest of their type as a length past
    the capacity and a position past the end."""
    g = torch.Generator(device=gpu).manual_seed(14)
    x = torch.randn((2, 1, 2, 64), generator=g, device=gpu).bfloat16()
    k = torch.randn((2, 64, 2, 64), generator=g, device=gpu).bfloat16()
    cache = vx.create_kv_cache(2, 64, 2, 64, device=gpu)
    vx.kv_cache_write(cache, k, k)
    before = _bytes(cache)
    top = torch.from_numpy(np.array([np.iinfo(str(dtype).split(".")[1]).max, 5], str(dtype).split(".")[1]))
    top = top.to(gpu) if on == "gpu" else top
    assert top.dtype == dtype
    assert torch.equal(vx.cached_attention(x, cache, top), vx.cached_attention(x, cache, _ints([64, 5], gpu)))
    assert (vx.kv_cache_read(cache, 1, top)[0][0] == 0).all()
    vx.kv_cache_write(cache, x, x, top)
    after = _bytes(cache)
    assert all((a[0] == b[0]).all() for a, b in zip(after, before)) and (after[0][1, :, 5] != before[0][1, :, 5]).any()


@pytest.mark.gpu
@pytest.mark.parametrize("none", [[], (), np.array([], np.int64), torch.tensor([], dtype=torch.int64)], ids=repr)
def test_integers_of_no_items(gpu, none):
    c = vx.create_kv_cache(2, 64, 2, 64, device=gpu)
    x = torch.zeros((0, 3, 2, 64), dtype=torch.bfloat16, device=gpu)
    vx.kv_cache_write(c, x, x, none, num=none, slots=none)
    assert vx.kv_cache_read(c, 3, none, slots=none)[0].shape == (0, 3, 2, 64)
    assert vx.cached_attention(x, c, none, q_len=none, slots=none).shape == x.shape
    with pytest.raises(ValueError, match="kv_len must hold 2"):
        vx.cached_attention(x.new_zeros((2, 1, 2, 64)), c, none)


@pytest.mark.gpu
def test_host_integers_are_refused_under_capture(gpu):
    c = vx.create_kv_cache(2, 64, 2, 64, device=gpu)
    x = torch.ones((2, 1, 2, 64), dtype=torch.bfloat16, device=gpu)
    want = vx.cached_attention(x, c, _ints([4, 5], gpu))  # (and the library is loaded)
    n = _ints([4, 5], gpu)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for call, name in ((lambda: vx.kv_cache_write(c, x, x, [1, 2]), "start"),
                           (lambda: vx.kv_cache_read(c, 3, slots=[0, 1]), "slots"),
                           (lambda: vx.cached_attention(x, c, torch.tensor([4, 5])), "kv_len"),
                           (lambda: vx.shared_prefix_attention(x, c, c, prefix_len=np.array([4, 5])), "prefix_len")):
            with pytest.raises(ValueError, match=f"{name} must be a device tensor"):
                call()
        got = vx.cached_attention(x, c, n)
    for _ in range(3):
        got.fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


@pytest.mark.gpu
def test_more_tokens_than_32_bits_count_are_refused(gpu):
    """(an expanded row: 2^32 + 3 tokens in 128 bytes)"""
    c = vx.create_kv_cache(1, 64, 1, 64, device=gpu)
    x = torch.ones((1, 1, 1, 64), dtype=torch.bfloat16, device=gpu)
    for n in (2 ** 31, 2 ** 32 + 3):
        with pytest.raises(NotImplementedError, match="tokens per item"):
            vx.kv_cache_write(c, x.expand(1, n, 1, 64), x.expand(1, n, 1, 64))
    assert (_bytes(c)[0] == 0).all()


@pytest.mark.gpu
def test_outputs_that_cannot_hold_the_values_are_refused(gpu):
    """Views that negate what they hold, or hold several values in one place."""
    c = vx.create_kv_cache(2, 64, 2, 64, device=gpu)
    x = torch.ones((2, 3, 2, 64), dtype=torch.bfloat16, device=gpu)
    vx.kv_cache_write(c, x, x)
    out = torch.full_like(x, 7.0)
    for bad in (torch._neg_view(out), out[:1].expand(2, 3, 2, 64), out[:, :1].expand(2, 3, 2, 64)):
        with pytest.raises(ValueError, match="out must be"):
            vx.cached_attention(x, c, [3, 3], out=bad)
    assert (out == 7.0).all()
    assert vx.cached_attention(x[:1], c, [3], out=out[:1].expand(1, 3, 2, 64)).data_ptr() == out.data_ptr()
    assert (out[0] == 1.0).all()


@pytest.mark.gpu
def test_refusals_of_gpu_calls(gpu):
    c = vx.create_kv_cache(2, 64, 2, 64, device=gpu)
    x = torch.zeros((2, 3, 2, 64), dtype=torch.bfloat16, device=gpu)
    for bad, err, frag in ((x.float(), TypeError, "bfloat16"), (x[0], ValueError, r"\(B, S, H, D\)"),
                           (x.cpu(), ValueError, "device"), (x[..., :32], ValueError, "head dim"),
                           (x[:, :, :1], ValueError, "heads"), (x[:, :2], ValueError, "differ")):
        with pytest.raises(err, match=frag):
            vx.kv_cache_write(c, bad, x)
    with pytest.raises(ValueError, match="slots"):
        vx.kv_cache_write(c, x[:1].expand(3, 3, 2, 64), x[:1].expand(3, 3, 2, 64))
    with pytest.raises(ValueError, match="start"):
        vx.kv_cache_write(c, x, x, [1, 2, 3])
    with pytest.raises(TypeError, match="integers"):
        vx.kv_cache_write(c, x, x, [1.0, 2.0])
    with pytest.raises(ValueError, match="length"):
        vx.kv_cache_read(c, -1)
    with pytest.raises(ValueError, match="multiple of num_kv_heads"):
        vx.cached_attention(torch.zeros((2, 1, 3, 64), dtype=torch.bfloat16, device=gpu), c)
    with pytest.raises(ValueError, match="kv_len"):
        vx.cached_attention(x, c, [1])
    with pytest.raises(ValueError, match="scale"):
        vx.cached_attention(x, c, scale=0.0)
    with pytest.raises(ValueError, match="out must be"):
        vx.cached_attention(x, c, out=x[:, :2])
    with pytest.raises(ValueError, match="contiguous"):
        vx.cached_attention(x, c._replace(k=c.k.transpose(1, 2).contiguous().transpose(1, 2)))
    with pytest.raises(TypeError, match="prefix"):
        vx.shared_prefix_attention(x, None, c)
    with pytest.raises(ValueError, match="agree"):
        vx.shared_prefix_attention(x, vx.create_kv_cache(1, 64, 1, 64, device=gpu), c)
    with pytest.raises(ValueError, match="multiple of num_prefixes"):
        vx.shared_prefix_attention(x, vx.create_kv_cache(4, 64, 2, 64, device=gpu), c)
    # nothing to do
    assert vx.cached_attention(x[:0], c).shape == (0, 3, 2, 64)
    assert vx.cached_attention(x[:, :0], c).shape == (2, 0, 2, 64)
    assert vx.kv_cache_read(c, 0)[0].shape == (2, 0, 2, 64)
    vx.kv_cache_write(c, x[:, :0], x[:, :0])


@pytest.mark.gpu
@pytest.mark.parametrize("D,slots", [(128, None), (64, [2, 7, 0])])
def test_long_cross_attention(gpu, D, slots):
    """Queries long enough for the expansion to bf16: sampled rows against the
    oracle, all rows against the same call in shorter pieces; a NaN token makes
    its head's rows NaN, and an item without a slot or a key gives zeros."""
    print(f"[case] long cross attention D={D} slots={slots}", flush=True)
    rng = np.random.default_rng(31)
    B, Sq, H, cap, lens = 3, 33400, 3, 192, [150, 192, 0 if slots is None else 33]
    by_slot = np.zeros(3, int)
    for b in range(B):
        slot = b if slots is None else slots[b]
        if slot < 3:
            by_slot[slot] = lens[b]
    k = rng.standard_normal((3, cap, H, D))
    k[0 if slots is None else 2, 17, 1, 3] = np.nan
    cache, _ = _noise_cache(rng, 3, H, cap, D, gpu)
    vx.kv_cache_write(cache, _bf16(k, gpu), _bf16(rng.standard_normal((3, cap, H, D)), gpu), num=by_slot)
    q = _bf16(2 * rng.standard_normal((B, Sq, H, D)), gpu)
    kw = dict(slots=_ints(slots, gpu), causal=False)
    got = vx.cached_attention(q, cache, _ints(lens, gpu), **kw)
    assert _lib.last_launch().startswith("flash_")
    pieces = torch.cat([vx.cached_attention(q[:, i:i + 2050], cache, _ints(lens, gpu), **kw) for i in range(0, Sq, 2050)], 1)
    want_nan = torch.zeros_like(got, dtype=torch.bool)
    want_nan[0, :, 1] = True
    assert torch.equal(got.isnan(), want_nan) and torch.equal(pieces.isnan(), want_nan)
    empty = 2 if slots is None else 1
    assert (got[empty] == 0).all() and (pieces[empty] == 0).all()
    rows = np.unique(np.linspace(0, Sq - 1, 40).astype(int))
    keep = [0, 2]  # (head 1 of item 0 is NaN)
    held = [x[:, keep] for x in _held(cache, by_slot)]
    for y in (got, pieces):
        sub, qs = y[:, rows][:, :, keep], q[:, rows][:, :, keep]
        _assert_close(sub, qs, held, None, kv_len=lens, slots=slots, causal=False)
