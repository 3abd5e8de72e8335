"""Operators of decoding and rollout steps over an 8-bit key/value cache: rotary
positions on several axes (alone, and on the way into the cache), attention with
a sliding window and first tokens that stay visible, attention of a tree of
drafted tokens.

A case is a dict of plain values; `listed()` holds the named ones, `draw(rng)`
makes another one of the same ranges. Kinds:

rope    pairs of channels turned by the token's positions (time, height, width),
        or back (the gradient of the turn, and how cached keys are moved)
write   keys turned the same way, written to the cache with their values, and
        read back
window  attention over the cached tokens within `window` of the query and the
        first `sinks` ones: single tokens, prompts in chunks (causal), or a
        block of tokens that see each other (not causal)
tree    attention of drafted tokens: each sees all tokens in front of the
        drafted ones, its ancestors and itself

A cache holds keys and values as float8_e4m3fn in (slot, kv head, position,
head dim) order, with one power-of-two scale (float8_e8m0fnu) per row: a row x is
stored as x / 2^e rounded to e4m3, 2^e the smallest power of two for which
max|x| / 2^e <= 448.

`run` computes a case in its plain form or, where `own` is true, through the
entry points of vidax_amd. `exact` computes the same from the definitions in 64
bits.
"""
import math
import random

import torch

own = False

BF16 = torch.bfloat16
E4M3 = torch.float8_e4m3fn
E8M0 = torch.float8_e8m0fnu
AXES = 3


def listed():
    return [
        # the queries of eight sequences' next tokens
        dict(name="rope_tokens_8", kind="rope", B=8, S=1, H=32, D=128, ct=32, ch=48, cw=48, halves=True, shared=True,
             back=False, grid=False, far=131072),
        # a whole video's queries (21 latent frames of 30 x 52), adjacent pairs
        dict(name="rope_32760", kind="rope", B=1, S=32760, H=40, D=128, ct=44, ch=42, cw=42, halves=False,
             shared=False, back=False, grid=True, far=0),
        # the gradient of a padded batch's queries, heads of 64, some channels not turned
        dict(name="rope_back_2x5003", kind="rope", B=2, S=5003, H=16, D=64, ct=16, ch=16, cw=16, halves=True,
             shared=False, back=True, grid=False, far=1000000),
        # one new token of each of 64 sequences: what every decoding step writes
        dict(name="write_tokens_64", kind="write", B=64, S=1, lo=1, Hk=8, D=128, cap=4096, slots=True,
             ct=32, ch=48, cw=48, halves=True, shared=True, grid=False, far=131072),
        # a block of three latent frames of 30 x 52, behind the frames before it
        dict(name="write_4680", kind="write", B=2, S=4680, lo=4680, Hk=12, D=128, cap=32768, slots=False,
             ct=44, ch=42, cw=42, halves=False, shared=False, grid=True, far=0),
        # one prompt's next token
        dict(name="window_1x700", kind="window", B=1, Sq=1, q_lo=1, H=12, Hk=12, D=128, lo=700, hi=700, cap=1024,
             window=256, sinks=4, causal=True, slots=False),
        # a serving batch of prompts of all lengths, its slots in the order of arrival
        dict(name="window_64x8192", kind="window", B=64, Sq=1, q_lo=1, H=32, Hk=8, D=128, lo=150, hi=8192, cap=8192,
             window=2048, sinks=4, causal=True, slots=True),
        # the next chunk of two prompts, one of them shorter (a padded batch)
        dict(name="window_2x1000x5003", kind="window", B=2, Sq=1000, q_lo=777, H=32, Hk=8, D=128, lo=4000, hi=5003,
             cap=8192, window=1500, sinks=100, causal=True, slots=False),
        # a block of three latent frames over the last twelve and the first one
        dict(name="window_4680x32760", kind="window", B=1, Sq=4680, q_lo=4680, H=12, Hk=12, D=128, lo=32760,
             hi=32760, cap=32768, window=18720, sinks=1560, causal=False, slots=False),
        # one prompt's drafted tokens
        dict(name="tree_1x26x700", kind="tree", B=1, Sq=26, q_lo=26, H=12, Hk=12, D=128, lo=700, hi=700, cap=1024,
             slots=False),
        # a serving batch, each with up to 61 drafted tokens
        dict(name="tree_16x61x8192", kind="tree", B=16, Sq=61, q_lo=30, H=32, Hk=8, D=128, lo=150, hi=8192, cap=8192,
             slots=True),
        # two long contexts under a wide tree, heads of 64
        dict(name="tree_2x250x30000", kind="tree", B=2, Sq=250, q_lo=201, H=32, Hk=4, D=64, lo=20001, hi=30000,
             cap=30016, slots=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _capacity(n):
    return (n + 63) // 64 * 64


def _rope_of(rng, D):
    split = rng.choice([[D // 4, D // 8 * 3, D // 8 * 3], [D - 4 * (D // 6), 2 * (D // 6), 2 * (D // 6)],
                        [D // 4, D // 4, D // 4], [D, 0, 0]])
    grid = rng.random() < 0.4
    return dict(ct=split[0], ch=split[1], cw=split[2], halves=rng.random() < 0.5, shared=rng.random() < 0.5, grid=grid,
                far=0 if grid else _log_int(rng, 100, 1000000))


def draw(rng):
    kind = rng.choice(["rope", "rope", "write", "write", "window", "window", "window", "tree", "tree"])
    D = rng.choice([128, 128, 64])
    while True:
        Hk = rng.choice([1, 2, 4, 8, 8, 12, 16, 40])
        if kind in ("rope", "write"):
            B, S = _log_int(rng, 1, 64), _log_int(rng, 1, 32760)
            if kind == "rope":
                c = dict(kind=kind, B=B, S=S, H=Hk * rng.choice([1, 1, 2, 4]), D=D, back=rng.random() < 0.3)
            else:
                c = dict(kind=kind, B=B, S=S, lo=rng.randint((S + 1) // 2, S), Hk=Hk, D=D,
                         cap=_capacity(S + rng.randint(0, 500)), slots=rng.random() < 0.5)
            c.update(_rope_of(rng, D))
            if B * S * c.get("H", Hk) * D <= (32760 * 40 * 128 if kind == "rope" else 32760 * 12 * 128):
                return c
            continue
        H = Hk * rng.choice([1, 1, 2, 3, 4, 5, 8])
        form = rng.choice(["token", "token", "few", "chunk", "block"]) if kind == "window" else "tree"
        B = _log_int(rng, 1, 64) if form in ("token", "few") else rng.randint(1, 16 if form == "tree" else 4)
        Sq = {"token": 1, "few": rng.randint(2, 9), "chunk": _log_int(rng, 10, 2000),
              "block": _log_int(rng, 100, 4680), "tree": _log_int(rng, 2, 300)}[form]
        hi = Sq + _log_int(rng, 1, 32760 if form == "block" else 131000)
        lo = rng.randint(Sq, hi)
        c = dict(kind=kind, B=B, Sq=Sq, q_lo=rng.randint((Sq + 1) // 2, Sq), H=H, Hk=Hk, D=D, lo=lo, hi=hi,
                 cap=_capacity(hi + rng.randint(0, 300)), slots=rng.random() < 0.5)
        if kind == "window":
            c.update(window=_log_int(rng, 1, 20000), sinks=rng.choice([0, 1, 4, 100, _log_int(rng, 1, 2000)]),
                     causal=form != "block")
        if B * c["cap"] * Hk * D <= 64 * 8192 * 8 * 128 and B * Sq * H * hi <= 4680 * 12 * 32760:
            return c


# ------------------------------------------------------------------ the inputs
def _spread(n, lo, hi):
    """n lengths in lo..hi, the same ones for every seed, hi among them."""
    r = random.Random(n * 1000003 + 31 * hi + lo)
    return [hi] + [r.randint(lo, hi) for _ in range(n - 1)]


def _lengths(case):
    """(query lengths, key lengths) of the batch items."""
    q, kv = _spread(case["B"], case["q_lo"], case["Sq"]), _spread(case["B"], case["lo"], case["hi"])
    return q, [max(n, m) for n, m in zip(kv, q)]  # the queries are the sequence's last tokens


def _frequencies(case):
    """(angle per position in radians, axis) of each pair of channels: on its
    own axis's ladder base^(-2 i / channels), or on one of the whole head; pairs
    past the axes' channels do not turn."""
    freq, axis, D = [], [], case["D"]
    for a, channels in enumerate((case["ct"], case["ch"], case["cw"])):
        for i in range(channels // 2):
            freq.append(10000.0 ** (-2.0 * len(freq) / D if case["shared"] else -2.0 * i / channels))
            axis.append(a)
    freq += [0.0] * (D // 2 - len(freq))
    axis += [0] * (D // 2 - len(axis))
    return freq, axis


def _turns(freq):
    """Turns per position in units of 2^-64 turns, whole turns left out."""
    t = [round(f / (2.0 * math.pi) * 2.0 ** 64) % 2 ** 64 for f in freq]
    return torch.tensor([x - 2 ** 64 if x >= 2 ** 63 else x for x in t], dtype=torch.int64, device="cuda")


def _positions(case, g):
    """(B, S, 3) positions: latent frames of 30 x 52 behind others, or text with
    images among it: tokens whose axes agree, and some whose axes do not."""
    B, S = case["B"], case["S"]
    at = torch.arange(S, device="cuda")
    if case["grid"]:
        p = torch.stack([at // 1560, at // 52 % 30, at % 52], dim=-1).expand(B, S, AXES).clone()
        p[..., 0] += 3 * torch.randint(0, 7, (B, 1), generator=g, device="cuda")
    else:
        p = (at + torch.randint(0, case["far"] + 1, (B, 1), generator=g, device="cuda"))[..., None].repeat(1, 1, AXES)
        off = torch.randint(0, 50, (B, S, 2), generator=g, device="cuda")
        p[..., 1:] += off * (at // 97 % 3 == 1)[:, None]
    return p.to(torch.int32)


def _quantised(x):
    """(e4m3 values, e8m0 scales) of rows x (..., D), fp32."""
    amax = x.abs().amax(-1)
    m, e = torch.frexp(amax)  # amax = m 2^e with m in [0.5, 1); 448 = 0.875 * 2^9
    e = torch.clamp_min(e - 9 + (m > 0.875).to(e.dtype), -126)
    y = x * ((127 - e) << 23).view(torch.float32)[..., None]  # 2^-e, by its bits
    return y.to(E4M3), (e + 127).to(torch.uint8).view(E8M0)


def _cache(g, n, Hk, cap, D):
    """A cache of n slots whose every position holds a token: rows of the
    spread that normed keys and projected values have, some of them large."""
    def rows(std):
        x = torch.randn((n, Hk, cap, D), generator=g, device="cuda")
        x *= std * torch.exp(0.5 * torch.randn((n, Hk, cap, 1), generator=g, device="cuda"))
        return _quantised(x.to(BF16).float())
    (k, ks), (v, vs) = rows(1.0), rows(0.7)
    return [k, v, ks, vs]


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind, B, D = case["kind"], case["B"], case["D"]
    st = dict(case=case)
    order = torch.randperm(B, generator=g, device="cuda").to(torch.int32)
    st["slots"] = order if case.get("slots") else None
    if kind in ("rope", "write"):
        S = case["S"]
        freq, axis = _frequencies(case)
        st["freq"] = torch.tensor(freq, dtype=torch.float64, device="cuda")
        st["axis"] = _ints(axis)
        st["turns"] = _turns(freq)
        st["positions"] = _positions(case, g)
        if kind == "rope":
            st["x"] = torch.randn((B, S, case["H"], D), generator=g, device="cuda").to(BF16)
            return st
        Hk = case["Hk"]
        st["start"] = torch.randint(0, case["cap"] - S + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
        shape = (B, Hk, case["cap"], D)
        st["cache"] = [torch.zeros(shape, device="cuda").to(E4M3) for _ in range(2)]
        st["cache"] += [torch.full(shape[:3], 127, dtype=torch.uint8, device="cuda").view(E8M0) for _ in range(2)]
        st["k"] = torch.randn((B, S, Hk, D), generator=g, device="cuda").to(BF16)
        st["v"] = (0.7 * torch.randn((B, S, Hk, D), generator=g, device="cuda")).to(BF16)
        st["num"] = _ints(_spread(B, case["lo"], S)) if case["lo"] < S else None
        return st
    Sq = case["Sq"]
    st["cache"] = _cache(g, B, case["Hk"], case["cap"], D)
    q_len, kv_len = _lengths(case)
    st["q"] = torch.randn((B, Sq, case["H"], D), generator=g, device="cuda").to(BF16)
    st["q_len"] = _ints(q_len) if case["q_lo"] < Sq else None
    st["kv_len"] = _ints(kv_len)
    if kind == "tree":
        # a token's parent is one of the drafted tokens in front of it, mostly a near one; some are roots
        at = torch.arange(Sq, device="cuda")
        parent = (at * torch.rand((B, Sq), generator=g, device="cuda").sqrt()).long().clamp_max(at - 1)
        root = torch.rand((B, Sq), generator=g, device="cuda") < 0.05
        st["parents"] = torch.where(root | (at == 0), -1, parent).to(torch.int32)
    return st


# ------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    kind = case["kind"]
    if own:
        import vidax_amd as vx
        if kind in ("rope", "write"):
            rope = vx.AxisRope(state["turns"], state["axis"], AXES, case["halves"])
            if kind == "rope":
                return vx.apply_axis_rope(state["x"], state["positions"], rope, inverse=case["back"])
            cache, slots = vx.KVCache(*state["cache"]), state["slots"]
            vx.kv_cache_write_rope(cache, state["k"], state["v"], state["positions"], rope, state["start"],
                                   num=state["num"], slots=slots)
            return vx.kv_cache_read(cache, case["S"], state["start"], slots=slots)
        cache = vx.KVCache(*state["cache"])
        if kind == "window":
            return vx.windowed_attention(state["q"], cache, state["kv_len"], window=case["window"],
                                         sinks=case["sinks"], q_len=state["q_len"], slots=state["slots"],
                                         causal=case["causal"])
        return vx.tree_attention(state["q"], cache, state["parents"], state["kv_len"], q_len=state["q_len"],
                                 slots=state["slots"])
    if kind == "rope":
        return _plain_rope(state, state["x"], case["back"]).to(BF16)
    if kind == "write":
        return _plain_write(state)
    return _plain_attention(state)


def _plain_rope(state, x, back=False):
    angle = state["positions"].double()[..., state["axis"].long()] * state["freq"]  # (B, S, D / 2)
    cos, sin = torch.cos(angle).float()[:, :, None], torch.sin(angle).float()[:, :, None]
    if back:
        sin = -sin
    x = x.float()
    half = x.shape[-1] // 2
    if state["case"]["halves"]:
        a, b = x[..., :half], x[..., half:]
        return torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)


def _plain_write(state):
    case = state["case"]
    slot = state["slots"].long() if state["slots"] is not None else torch.arange(case["B"], device="cuda")
    pos = state["start"].long()[:, None] + torch.arange(case["S"], device="cuda")
    slot = slot[:, None].expand_as(pos)
    out = []
    for held, scale, x in zip(state["cache"][:2], state["cache"][2:], (_plain_rope(state, state["k"]), state["v"])):
        held, scale = held.view(torch.uint8), scale.view(torch.uint8)
        y, s = (t.view(torch.uint8) for t in _quantised(x.float()))
        if state["num"] is not None:  # tokens past num stay as they are
            keep = (torch.arange(pos.shape[1], device="cuda") < state["num"][:, None])[..., None]
            y = torch.where(keep[..., None], y, held[slot, :, pos])
            s = torch.where(keep, s, scale[slot, :, pos])
        held[slot, :, pos] = y
        scale[slot, :, pos] = s
        out.append((held[slot, :, pos].view(E4M3).float() * scale[slot, :, pos].view(E8M0).float()[..., None]).to(BF16))
    return out


def _ancestors(parents):
    """(B, Sq, Sq) truth values: column j is row i's ancestor, or itself."""
    n = parents.shape[1]
    at = torch.arange(n, device="cuda")
    reach = ((parents[..., None] == at) | (at[:, None] == at)).float()
    for _ in range(max(1, (n - 1).bit_length())):  # paths of twice the length
        reach = torch.matmul(reach, reach.contiguous()).clamp_max(1.0)
    return reach > 0


def _plain_attention(state):
    case = state["case"]
    B, Sq, H, Hk, D = (case[n] for n in ("B", "Sq", "H", "Hk", "D"))
    G = H // Hk
    cache = [x.view(torch.uint8) for x in state["cache"]]
    if state["slots"] is not None:
        cache = [x[state["slots"].long()] for x in cache]
    n = int(max(case["hi"], Sq))
    k, v, ks, vs = [x.view(t)[:, :, :n].float() for x, t in zip(cache, (E4M3, E4M3, E8M0, E8M0))]
    k, v = k * ks[..., None], v * vs[..., None]
    keys, rows = torch.arange(n, device="cuda"), torch.arange(Sq, device="cuda")
    kv_len = state["kv_len"].long()[:, None]
    q_len = state["q_len"].long()[:, None] if state["q_len"] is not None else torch.full((B, 1), Sq, device="cuda")
    bound = kv_len - q_len + rows + 1 if case.get("causal", True) else kv_len.expand(B, Sq)
    seen = keys < bound[..., None]  # (B, Sq, n)
    if case["kind"] == "window":
        seen &= (keys >= bound[..., None] - case["window"]) | (keys < case["sinks"])
    else:
        at = keys - (kv_len - q_len)  # (B, n): the drafted token that lies there
        kin = torch.gather(_ancestors(state["parents"]), 2, at[:, None].clamp(0, Sq - 1).expand(B, Sq, n))
        seen &= (at < 0)[:, None] | kin
    q = state["q"].float().reshape(B, Sq, Hk, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, G * Sq, D) * D ** -0.5
    s = torch.matmul(q, k.transpose(2, 3)).reshape(B, Hk, G, Sq, n).masked_fill_(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp_(s.sub_(torch.where(top == -math.inf, 0.0, top)))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.reshape(B, Hk, G * Sq, n), v).reshape(B, Hk, G, Sq, D)
    o = o / torch.where(total == 0, 1.0, total) * (rows < q_len)[:, None, None, :, None]
    return o.permute(0, 3, 1, 2, 4).reshape(B, Sq, H, D).to(BF16)


# ------------------------------------------------------------------ its work
def work(case):
    kind, B, D = case["kind"], case["B"], case["D"]
    row = D + 1  # bytes of a cached row and its scale
    if kind == "rope":
        n = B * case["S"] * case["H"] * D
        return {"bytes": 4 * n + 4 * AXES * B * case["S"], "flops": 3 * n}
    if kind == "write":
        held, new = 2 * B * case["S"] * case["Hk"], sum(_spread(B, case["lo"], case["S"]))
        return {"bytes": held * (row + 2 * D) + 2 * new * case["Hk"] * (2 * D + row) + 4 * AXES * new,
                "flops": held * D + 3 * new * case["Hk"] * D}
    read = pairs = 0
    for m, n in zip(*_lengths(case)):
        if kind == "tree":
            read += n
            pairs += m * (n - m) + m  # (and what its ancestors are)
            continue
        causal, w, s = case["causal"], case["window"], case["sinks"]
        low = max(0, (n - m + 1 if causal else n) - w)  # the first key within some query's window
        read += min(s, low) + n - low
        for bound in (range(n - m + 1, n + 1) if causal else (n,)):
            pairs += (1 if causal else m) * (min(s, max(0, bound - w)) + min(w, bound))
    return {"bytes": 2 * row * case["Hk"] * read + 4 * D * case["H"] * B * case["Sq"],
            "flops": 4 * D * case["H"] * pairs}


# ------------------------------------------------------------------ in 64 bits
def _turned(x, positions, case, back):
    """Rows x (B, S, H, D) in 64 bits, each pair turned by its axis's position
    times its frequency."""
    y = x.double().clone()
    D = case["D"]
    for j, (f, a) in enumerate(zip(*_frequencies(case))):
        lo, hi = (j, j + D // 2) if case["halves"] else (2 * j, 2 * j + 1)
        t = positions[..., a].double() * (-f if back else f)
        c, s = torch.cos(t)[..., None], torch.sin(t)[..., None]
        u, w = x[..., lo].double(), x[..., hi].double()
        y[..., lo], y[..., hi] = u * c - w * s, w * c + u * s
    return y


def _e4m3(y):
    """Values y (64 bits, |y| <= 448) rounded to e4m3: three bits behind the
    leading one, steps of 2^-9 below 2^-6, ties to even."""
    step = torch.exp2(torch.clamp_min(torch.floor(torch.log2(torch.clamp_min(y.abs(), 2.0 ** -20))), -6) - 3)
    return torch.round(y / step) * step


def _stored(x):
    """The values that rows x (..., D) stand for once they are stored."""
    amax = x.abs().amax(-1, keepdim=True)
    e = torch.full_like(amax, -126.0)
    for n in range(-126, 12):  # the smallest e with amax <= 448 * 2^e; inputs here stay below 448 * 2^11
        e = torch.where(amax > 448.0 * 2.0 ** n, n + 1.0, e)
    return _e4m3(x / torch.exp2(e)) * torch.exp2(e)


def exact(case, seed):
    st = prepare(case, seed)
    B, D = case["B"], case["D"]
    if case["kind"] == "rope":
        return _turned(st["x"], st["positions"], case, case["back"])
    if case["kind"] == "write":
        out = [_stored(_turned(st["k"], st["positions"], case, False)), _stored(st["v"].double())]
        for y in out:
            for b in range(B if st["num"] is not None else 0):
                y[b, int(st["num"][b]):] = 0.0  # never written: the cache was empty
        return out
    slots = st["slots"].tolist() if st["slots"] is not None else list(range(B))
    q_len, kv_len = _lengths(case)
    Sq, H, G = case["Sq"], case["H"], case["H"] // case["Hk"]
    out = torch.zeros((B, Sq, H, D), dtype=torch.float64, device="cuda")
    for b in range(B):
        m, n = q_len[b], kv_len[b]
        k, v = (x[slots[b], :, :n].double() * s[slots[b], :, :n].double()[..., None]
                for x, s in zip(st["cache"][:2], st["cache"][2:]))
        see = torch.zeros((m, n), dtype=torch.bool, device="cuda")
        if case["kind"] == "tree":
            see[:, :n - m] = True
            for i, parent in enumerate(st["parents"][b, :m].tolist()):
                if parent >= 0:
                    see[i] = see[parent]
                see[i, n - m + i] = True
        else:
            for i in range(m if case["causal"] else 1):
                row = see[i] if case["causal"] else see
                end = n - m + 1 + i if case["causal"] else n
                row[..., :min(case["sinks"], end)] = True
                row[..., max(0, end - case["window"]):end] = True
        for h in range(H):
            logits = (st["q"][b, :m, h].double() @ k[h // G].T) / math.sqrt(D)
            logits[~see] = -math.inf
            w = torch.exp(logits - logits.amax(-1, keepdim=True).clamp_min(-1e300))
            out[b, :m, h] = (w @ v[h // G]) / w.sum(-1, keepdim=True)
    return out
