"""Operators of an 8-bit key/value cache: writing and reading it, attention over
it, and attention of a batch that shares a long prefix.

A cache holds keys and values as float8_e4m3fn in (slot, kv head, position,
head dim) order, with one power-of-two scale (float8_e8m0fnu) per slot, kv
head and position: a row x of head dim values is stored as x / 2^e rounded to
e4m3, 2^e the smallest power of two for which max|x| / 2^e <= 448.

A case is a dict of plain values; `listed()` holds the named ones, `draw(rng)`
makes another one of the same ranges. Kinds:

write   new tokens' keys and values written to the cache, and read back
read    a stretch of the cache read back as bf16
attn    attention over the cached keys: single tokens, prompts in chunks
        (causal), or cross attention to an encoder's states (not causal)
prefix  the same for batch items that share a prefix, one per group

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


def listed():
    return [
        # one new token of each of eight sequences: what every decoding step writes
        dict(name="write_tokens_8", kind="write", B=8, S=1, lo=1, Hk=8, D=128, cap=4096, slots=True),
        # a whole video's tokens (five latent frames, 12 heads) for later steps
        dict(name="write_7800", kind="write", B=1, S=7800, lo=7800, Hk=12, D=128, cap=7808, slots=False),
        # two prompts' text states, read back for a bf16 consumer
        dict(name="read_512", kind="read", B=2, S=512, Hk=40, D=128, cap=512, slots=False),
        # the keys and values of a full video self-attention
        dict(name="read_32760", kind="read", B=1, S=32760, Hk=40, D=128, cap=32768, slots=False),
        # one prompt's next token
        dict(name="decode_1x700", kind="attn", B=1, Sq=1, q_lo=1, H=12, Hk=12, D=128, lo=700, hi=700, cap=1024,
             causal=True, slots=False),
        # a serving batch of prompts of all lengths, its slots in the order of arrival
        dict(name="decode_64x8192", kind="attn", B=64, Sq=1, q_lo=1, H=32, Hk=8, D=128, lo=150, hi=8192, cap=8192,
             causal=True, slots=True),
        # two long contexts
        dict(name="decode_2x131000", kind="attn", B=2, Sq=1, q_lo=1, H=32, Hk=8, D=128, lo=90001, hi=131000,
             cap=131072, causal=True, slots=False),
        # the next chunk of two prompts, one of them shorter (a padded batch)
        dict(name="chunk_2x1000x5003", kind="attn", B=2, Sq=1000, q_lo=777, H=32, Hk=8, D=128, lo=4000, hi=5003,
             cap=8192, causal=True, slots=False),
        # video tokens against two padded prompts whose states stay in the cache over all denoising steps
        dict(name="cross_32760x512", kind="attn", B=2, Sq=32760, q_lo=32760, H=40, Hk=40, D=128, lo=148, hi=512,
             cap=512, causal=False, slots=False),
        # a few samples behind one short instruction, heads of 64
        dict(name="prefix_4x226", kind="prefix", B=4, Sq=1, q_lo=1, H=16, Hk=16, D=64, lo=1, hi=60, cap=64,
             groups=1, p_lo=226, p_hi=226, p_cap=256, causal=True),
        # many samples behind one long prompt: one decoding step
        dict(name="prefix_32x8192", kind="prefix", B=32, Sq=1, q_lo=1, H=32, Hk=8, D=128, lo=0, hi=500, cap=512,
             groups=1, p_lo=8192, p_hi=8192, p_cap=8192, causal=True),
        # the samples' own prompts behind a guided pair of templates, in one chunk
        dict(name="prefix_16x64x4001", kind="prefix", B=16, Sq=64, q_lo=20, H=16, Hk=8, D=128, lo=64, hi=200,
             cap=256, groups=2, p_lo=1500, p_hi=4001, p_cap=4096, causal=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _capacity(n):
    return (n + 63) // 64 * 64


def draw(rng):
    kind = rng.choice(["write", "read", "attn", "attn", "attn", "prefix", "prefix"])
    D = rng.choice([128, 128, 64])
    while True:
        Hk = rng.choice([1, 2, 4, 8, 8, 12, 16, 40])
        if kind in ("write", "read"):
            B, S = _log_int(rng, 1, 64), _log_int(rng, 1, 32760)
            c = dict(kind=kind, B=B, S=S, Hk=Hk, D=D, cap=_capacity(S + rng.randint(0, 500)),
                     slots=rng.random() < 0.5)
            if kind == "write":
                c["lo"] = rng.randint((S + 1) // 2, S)
        else:
            H = Hk * rng.choice([1, 1, 2, 3, 4, 5, 8])
            form = rng.choice(["token", "token", "few", "chunk"] + (["cross"] if kind == "attn" else []))
            B = _log_int(rng, 1, 64) if form in ("token", "few") else rng.randint(1, 4)
            Sq = {"token": 1, "few": rng.randint(2, 9), "chunk": _log_int(rng, 10, 2000),
                  "cross": _log_int(rng, 200, 32760)}[form]
            if kind == "attn":
                hi = _log_int(rng, 20, 2000) if form == "cross" else Sq + _log_int(rng, 1, 131000)
            else:
                hi = Sq + _log_int(rng, 1, 1000)
            lo = rng.randint(min(Sq if form != "cross" else 1, hi), hi)
            c = dict(kind=kind, B=B, Sq=Sq, q_lo=rng.randint((Sq + 1) // 2, Sq), H=H, Hk=Hk, D=D, lo=lo, hi=hi,
                     cap=_capacity(hi + rng.randint(0, 300)), causal=form != "cross")
            if kind == "attn":
                c["slots"] = rng.random() < 0.5
            else:
                p_hi = _log_int(rng, 20, 30000)
                c.update(groups=rng.choice([g for g in (1, 1, 2, 4) if B % g == 0]), p_hi=p_hi,
                         p_lo=rng.randint(p_hi // 2, p_hi), p_cap=_capacity(p_hi))
        held = c.get("groups", 0) * c.get("p_cap", 0) + B * c["cap"]  # cached positions
        scores = B * c["Sq"] * c["H"] * (c["hi"] + c.get("p_hi", 0)) if "Sq" in c else 0
        if held * Hk * D <= 64 * 8192 * 8 * 128 and work(c)["flops"] <= 6e11 and scores <= 2 * 32760 * 40 * 512:
            if kind in ("attn", "prefix") or B * c["S"] * Hk * D <= 32760 * 40 * 128:
                return c


# ------------------------------------------------------------------ the inputs
def _spread(n, lo, hi):
    """n lengths in lo..hi, the same ones for every seed, hi among them."""
    r = random.Random(n * 1000003 + 31 * hi + lo)
    return [hi] + [r.randint(lo, hi) for _ in range(n - 1)]


def _lengths(case):
    """(query lengths, key lengths, prefix lengths) of the batch items and groups."""
    B = case["B"]
    q = _spread(B, case["q_lo"], case["Sq"])
    kv = _spread(B, case["lo"], case["hi"])
    if case["causal"]:  # the queries are the sequence's last tokens
        kv = [max(n, m) if case["kind"] == "attn" else n for n, m in zip(kv, q)]
    return q, kv, _spread(case["groups"], case["p_lo"], case["p_hi"]) if "groups" in case else []


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
    kind, B, Hk, D = case["kind"], case["B"], case["Hk"], case["D"]
    st = dict(case=case)
    order = torch.randperm(B, generator=g, device="cuda").to(torch.int32)
    st["slots"] = order if case.get("slots") else None
    if kind in ("write", "read"):
        S = case["S"]
        st["start"] = torch.randint(0, case["cap"] - S + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
    if kind == "write":
        shape = (B, Hk, case["cap"], D)
        st["cache"] = [torch.zeros(shape, device="cuda").to(E4M3) for _ in range(2)]
        st["cache"] += [torch.full(shape[:3], 127, dtype=torch.uint8, device="cuda").view(E8M0) for _ in range(2)]
        st["k"] = torch.randn((B, S, Hk, D), generator=g, device="cuda").to(BF16)
        st["v"] = (0.7 * torch.randn((B, S, Hk, D), generator=g, device="cuda")).to(BF16)
        st["num"] = _ints(_spread(B, case["lo"], S)) if case["lo"] < S else None
        return st
    st["cache"] = _cache(g, B, Hk, case["cap"], D)
    if kind == "read":
        return st
    q_len, kv_len, p_len = _lengths(case)
    st["q"] = torch.randn((B, case["Sq"], case["H"], D), generator=g, device="cuda").to(BF16)
    st["q_len"] = _ints(q_len) if case["q_lo"] < case["Sq"] else None
    st["kv_len"] = _ints(kv_len)
    if kind == "prefix":
        st["prefix"] = _cache(g, case["groups"], Hk, case["p_cap"], D)
        st["p_len"] = _ints(p_len)
    return st


# ------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    kind = case["kind"]
    if own:
        import vidax_amd as vx
        cache, slots = vx.KVCache(*state["cache"]), state["slots"]
        if kind == "write":
            vx.kv_cache_write(cache, state["k"], state["v"], state["start"], num=state["num"], slots=slots)
        if kind in ("write", "read"):
            return vx.kv_cache_read(cache, case["S"], state["start"], slots=slots)
        if kind == "attn":
            return vx.cached_attention(state["q"], cache, state["kv_len"], q_len=state["q_len"], slots=slots,
                                       causal=case["causal"])
        return vx.shared_prefix_attention(state["q"], vx.KVCache(*state["prefix"]), cache, state["kv_len"],
                                          prefix_len=state["p_len"], q_len=state["q_len"], causal=case["causal"])
    if kind == "write":
        _plain_write(state)
    if kind in ("write", "read"):
        return _plain_read(state)
    return _plain_attention(state)


def _positions(state):
    """(slot, position) index tensors, (B, S), of the tokens written or read."""
    case = state["case"]
    slot = state["slots"].long() if state["slots"] is not None else torch.arange(case["B"], device="cuda")
    pos = state["start"].long()[:, None] + torch.arange(case["S"], device="cuda")
    return slot[:, None].expand_as(pos), pos


def _plain_write(state):
    slot, pos = _positions(state)
    for held, scale, x in zip(state["cache"][:2], state["cache"][2:], (state["k"], state["v"])):
        held, scale = held.view(torch.uint8), scale.view(torch.uint8)
        y, s = (t.view(torch.uint8) for t in _quantised(x.float()))
        if state["num"] is not None:  # tokens past num stay as they are
            keep = (torch.arange(pos.shape[1], device="cuda") < state["num"][:, None])[..., None]
            y = torch.where(keep[..., None], y, held[slot, :, pos])
            s = torch.where(keep, s, scale[slot, :, pos])
        held[slot, :, pos] = y
        scale[slot, :, pos] = s


def _plain_read(state):
    slot, pos = _positions(state)
    k, v, ks, vs = state["cache"]
    return [(x.view(torch.uint8)[slot, :, pos].view(E4M3).float() *
             s.view(torch.uint8)[slot, :, pos].view(E8M0).float()[..., None]).to(BF16)
            for x, s in ((k, ks), (v, vs))]


def _values(x, s, n):
    """The first n positions of cached rows as fp32."""
    return x[:, :, :n].float() * s[:, :, :n].float()[..., None]


def _plain_attention(state):
    case = state["case"]
    B, Sq, H, Hk, D = (case[n] for n in ("B", "Sq", "H", "Hk", "D"))
    G = H // Hk
    cache = [x.view(torch.uint8) for x in state["cache"]]
    if state["slots"] is not None:
        cache = [x[state["slots"].long()] for x in cache]
    k, v, ks, vs = [x.view(t) for x, t in zip(cache, (E4M3, E4M3, E8M0, E8M0))]
    n = int(case["hi"] if case["kind"] == "prefix" else max(case["hi"], case["Sq"] if case["causal"] else 0))
    keys = torch.arange(n, device="cuda")
    rows = torch.arange(Sq, device="cuda")
    kv_len = state["kv_len"][:, None, None]
    q_len = state["q_len"][:, None] if state["q_len"] is not None else torch.full((B, 1), Sq, device="cuda")
    bound = kv_len
    if case["causal"]:  # query i of q_len is position kv_len - q_len + i
        bound = torch.minimum(kv_len, (state["kv_len"][:, None] - q_len + rows + 1)[..., None])
    seen = keys < bound  # (B, Sq or 1, n)
    q = state["q"].float().reshape(B, Sq, Hk, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, G * Sq, D) * D ** -0.5
    s = torch.matmul(q, _values(k, ks, n).transpose(2, 3)).reshape(B, Hk, G, Sq, n)
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    if case["kind"] == "prefix":
        P, m = case["groups"], case["p_hi"]
        pk, pv, pks, pvs = state["prefix"]
        qp = q.reshape(P, B // P, Hk, G * Sq, D).transpose(1, 2).reshape(P, Hk, (B // P) * G * Sq, D)
        sp = torch.matmul(qp, _values(pk, pks, m).transpose(2, 3))
        sp = sp.masked_fill((torch.arange(m, device="cuda") >= state["p_len"][:, None])[:, None, None], -math.inf)
        sp = sp.reshape(P, Hk, B // P, G, Sq, m).transpose(1, 2).reshape(B, Hk, G, Sq, m)
        s = torch.cat([sp, s], dim=-1)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    if case["kind"] == "prefix":
        pp, p = p[..., :m], p[..., m:]
        pp = pp.reshape(P, B // P, Hk, G * Sq, m).transpose(1, 2).reshape(P, Hk, (B // P) * G * Sq, m)
        op = torch.matmul(pp, _values(pv, pvs, m))
        op = op.reshape(P, Hk, B // P, G, Sq, D).transpose(1, 2).reshape(B, Hk, G, Sq, D)
    o = torch.matmul(p.reshape(B, Hk, G * Sq, n), _values(v, vs, n)).reshape(B, Hk, G, Sq, D)
    o = (o + op if case["kind"] == "prefix" else o) / torch.where(total == 0, 1.0, total)
    o = o * (rows < q_len)[:, None, None, :, None]
    return o.permute(0, 3, 1, 2, 4).reshape(B, Sq, H, D).to(BF16)


# ------------------------------------------------------------------ its work
def work(case):
    kind, B, Hk, D = case["kind"], case["B"], case["Hk"], case["D"]
    row = D + 1  # bytes of a cached row and its scale
    if kind in ("write", "read"):
        held = 2 * B * case["S"] * Hk  # rows of k and of v read back
        nbytes = held * (row + 2 * D)
        if kind == "write":
            nbytes += 2 * sum(_spread(B, case["lo"], case["S"])) * Hk * (2 * D + row)
        return {"bytes": nbytes, "flops": held * D}
    q_len, kv_len, p_len = _lengths(case)
    nbytes = 2 * row * Hk * (sum(kv_len) + sum(p_len)) + 2 * 2 * D * case["H"] * B * case["Sq"]
    pairs = 0
    for b in range(B):
        n, m = kv_len[b], q_len[b]
        if case["causal"]:
            first = n - m + 1  # keys that query 0 sees
            hidden = max(0, -first + 1)  # queries before the first key
            a, c = max(first, 0), n
            pairs += (a + c) * (min(m, m - hidden + 1) if first < 0 else m) // 2
        else:
            pairs += n * m
        if p_len:
            pairs += p_len[b // (B // len(p_len))] * m
    return {"bytes": nbytes, "flops": 4 * D * case["H"] * pairs}


# ------------------------------------------------------------------ in 64 bits
def _e4m3(y):
    """Values y (64 bits, |y| <= 448) rounded to e4m3: three bits behind the
    leading one, steps of 2^-9 below 2^-6, ties to even."""
    step = torch.exp2(torch.clamp_min(torch.floor(torch.log2(torch.clamp_min(y.abs(), 2.0 ** -20))), -6) - 3)
    return torch.round(y / step) * step


def _stored(x):
    """The values that rows x (..., D) stand for once they are stored."""
    x = x.double()
    amax = x.abs().amax(-1, keepdim=True)
    e = torch.full_like(amax, -126.0)
    for n in range(-126, 12):  # the smallest e with amax <= 448 * 2^e; inputs here stay below 448 * 2^11
        e = torch.where(amax > 448.0 * 2.0 ** n, n + 1.0, e)
    return _e4m3(x / torch.exp2(e)) * torch.exp2(e)


def _held(cache, slot):
    """Keys and values of one slot, (Hk, cap, D) each, in 64 bits."""
    return [x[slot].double() * s[slot].double()[..., None] for x, s in ((cache[0], cache[2]), (cache[1], cache[3]))]


def exact(case, seed):
    st = prepare(case, seed)
    B = case["B"]
    slots = st["slots"].tolist() if st["slots"] is not None else list(range(B))
    if case["kind"] in ("write", "read"):
        S, out = case["S"], [[], []]
        for b, at in enumerate(st["start"].tolist()):
            if case["kind"] == "read":
                for o, x in zip(out, _held(st["cache"], slots[b])):
                    o.append(x[:, at:at + S].transpose(0, 1))
            else:
                m = int(st["num"][b]) if st["num"] is not None else S
                for o, x in zip(out, (st["k"], st["v"])):
                    y = _stored(x[b])
                    y[m:] = 0.0  # never written: the cache was empty
                    o.append(y)
        return [torch.stack(o) for o in out]
    q_len, kv_len, p_len = _lengths(case)
    Sq, H, Hk, D = (case[n] for n in ("Sq", "H", "Hk", "D"))
    G = H // Hk
    out = torch.zeros((B, Sq, H, D), dtype=torch.float64, device="cuda")
    for b in range(B):
        m, n = q_len[b], kv_len[b]
        k, v = (x[:, :n] for x in _held(st["cache"], slots[b]))
        last = torch.full((m,), n, device="cuda")
        if case["causal"]:
            last = n - m + 1 + torch.arange(m, device="cuda")  # keys below this are seen
        if p_len:
            group = b // (B // case["groups"])
            pk, pv = (x[:, :p_len[group]] for x in _held(st["prefix"], group))
            k, v = torch.cat([pk, k], dim=1), torch.cat([pv, v], dim=1)
            last = last.clamp_min(0) + p_len[group]
        hide = torch.arange(k.shape[1], device="cuda")[None, :] >= last[:, None]
        for h in range(H):
            logits = (st["q"][b, :m, h].double() @ k[h // G].T) / math.sqrt(D)
            logits[hide] = -math.inf
            w = torch.exp(logits - logits.amax(-1, keepdim=True).clamp_min(-1e300))
            z = w.sum(-1, keepdim=True)
            out[b, :m, h] = (w @ v[h // G]) / torch.where(z == 0, 1.0, z)
    return out
