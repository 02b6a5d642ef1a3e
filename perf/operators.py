"""The operators of the 4-bit KV cache, measured: quantising append, RoPE fused with it, read-back, decode attention.

A cache row is one (position, kv head): `d` codes of 4 bits and, for every `group` consecutive dims, a (scale, base) pair of fp16;
value = code * scale + base.  The row's d/4 units of four codes (unit u = 8 j + r holds dims 4u .. 4u + 3) are stored at place
r * (d / 32) + j, eight codes to an int32 word.  Head-major caches are [batch, heads, max_len, ...], paged pools
[blocks, heads, block_size, ...] with a block table [batch, blocks per sequence].
"""
import importlib
import math
import random

import torch

own = False

LIMIT = 65440.0          # values are clamped to it before they are quantised, so that 15 * scale + base is finite in fp16
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


# ---- cases ---------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one user, a short chat: the whole call is latency
        dict(name="attn_b1_len777", kind="attn", paged=False, dtype="f16", batch=1, hq=32, hkv=8, d=128, group=64, lo=777, hi=777,
             max_len=800, block=0, spread=1, empty=False),
        # the decode step of the benchmark: 64 sequences at context 4096
        dict(name="attn_b64_ctx4096", kind="attn", paged=False, dtype="f16", batch=64, hq=32, hkv=8, d=128, group=64, lo=4096, hi=4096,
             max_len=4097, block=0, spread=2, empty=False),
        # ragged batch of 32 up to 8192 positions, the finest groups, bf16
        dict(name="attn_b32_ragged8192_bf16", kind="attn", paged=False, dtype="bf16", batch=32, hq=32, hkv=8, d=128, group=32, lo=512,
             hi=8192, max_len=8192, block=0, spread=3, empty=False),
        # a paged server with small heads, odd lengths, one slot of the batch empty
        dict(name="attn_paged_b24_d64_bf16", kind="attn", paged=True, dtype="bf16", batch=24, hq=16, hkv=2, d=64, group=64, lo=1, hi=2100,
             max_len=2112, block=16, spread=4, empty=True),
        # one very long document, paged, the coarsest groups
        dict(name="attn_paged_b1_len131071", kind="attn", paged=True, dtype="f16", batch=1, hq=32, hkv=8, d=128, group=128, lo=131071,
             hi=131071, max_len=131072, block=64, spread=5, empty=False),
        # a decode step's new rows of 64 sequences, written and read back
        dict(name="write_b64_t1", kind="write", paged=False, dtype="f16", batch=64, tokens=1, heads=8, d=128, group=64, max_len=4097,
             block=0, spread=6, ragged=False),
        # the prefill of one long prompt
        dict(name="write_b1_t8192_bf16", kind="write", paged=False, dtype="bf16", batch=1, tokens=8192, heads=8, d=128, group=128,
             max_len=8200, block=0, spread=7, ragged=False),
        # a padded batch of prompts of different lengths into a paged pool, a head_dim that is no power of two
        dict(name="write_paged_b8_t1000", kind="write", paged=True, dtype="f16", batch=8, tokens=1000, heads=8, d=96, group=32,
             max_len=1040, block=16, spread=8, ragged=True),
        # the context of four sequences expanded for the next chunk of their prefill
        dict(name="read_b4_ctx8192", kind="read", paged=False, dtype="f16", batch=4, heads=8, d=128, group=64, lo=8192, hi=8192,
             max_len=8192, block=0, spread=9, empty=False),
        # short odd contexts out of a paged pool
        dict(name="read_paged_b16_bf16", kind="read", paged=True, dtype="bf16", batch=16, heads=4, d=128, group=32, lo=1, hi=1333,
             max_len=1360, block=16, spread=10, empty=True),
        # a decode step's fused QKV rows: rotated, quantised, stored
        dict(name="rope_b64", kind="rope", dtype="f16", batch=64, hq=32, hkv=8, d=128, group=64, max_len=4097, spread=11),
        # a large decode batch in bf16 with the finest groups
        dict(name="rope_b512_bf16", kind="rope", dtype="bf16", batch=512, hq=32, hkv=8, d=128, group=32, max_len=1025, spread=12),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    d = rng.choice([64, 96, 128, 128, 128, 192, 256])
    group = rng.choice([g for g in (32, 64, 128) if d % g == 0])
    dtype, paged, spread = rng.choice(["f16", "bf16"]), rng.random() < 0.5, rng.randrange(1 << 20)
    block = rng.choice([8, 16, 32, 64, 48, 100]) if paged else 0
    kind = rng.choice(["attn", "attn", "write", "read", "rope"])
    heads = rng.choice([1, 2, 4, 8, 8])
    cap = 32 * 8 * 4096 * 128                 # elements of a cache tensor: half of the largest listed case's
    if kind == "attn":
        batch = _log(rng, 1, 64)
        hi = max(1, min(_log(rng, 1, 65536), cap // (batch * heads * d)))
        c = dict(kind=kind, paged=paged, dtype=dtype, batch=batch, hq=heads * rng.choice([1, 2, 3, 4, 4, 7, 8, 16]), hkv=heads, d=d,
                 group=group, lo=rng.randint(1, hi), hi=hi, max_len=hi + rng.randint(0, 40), block=block, spread=spread,
                 empty=batch > 1 and rng.random() < 0.3)
    elif kind == "write":
        batch = _log(rng, 1, 64)
        tokens = max(1, min(_log(rng, 1, 8192), 8192 // batch))
        c = dict(kind=kind, paged=paged, dtype=dtype, batch=batch, tokens=tokens, heads=heads, d=d, group=group,
                 max_len=tokens + rng.randint(8, 200), block=block, spread=spread, ragged=rng.random() < 0.5)
    elif kind == "read":
        batch = _log(rng, 1, 32)
        hi = max(1, min(_log(rng, 1, 16384), cap // 4 // (batch * heads * d)))
        c = dict(kind=kind, paged=paged, dtype=dtype, batch=batch, heads=heads, d=d, group=group, lo=rng.randint(1, hi), hi=hi,
                 max_len=hi + rng.randint(0, 40), block=block, spread=spread, empty=batch > 1 and rng.random() < 0.3)
    else:
        c = dict(kind=kind, dtype=dtype, batch=_log(rng, 1, 512), hq=heads * rng.choice([1, 2, 4, 4, 7, 8]), hkv=heads, d=d, group=group,
                 max_len=rng.randint(16, 2000), spread=spread)
    if c.get("paged"):                        # whole blocks
        c["max_len"] = -(-c["max_len"] // block) * block
    return c


def _lens(c):
    r = random.Random(c["spread"])
    lens = [r.randint(c["lo"], c["hi"]) for _ in range(c["batch"])]
    if c["empty"]:
        lens[r.randrange(len(lens))] = 0
    return lens


def _writes(c):
    """(first position, new tokens) of every sequence of an append."""
    r = random.Random(c["spread"])
    first = [r.randint(0, c["max_len"] - c["tokens"]) for _ in range(c["batch"])]
    count = [r.randint(0, c["tokens"]) if c["ragged"] else c["tokens"] for _ in range(c["batch"])]
    if c["ragged"]:
        count[0] = c["tokens"]
    return first, count


def work(case):
    c = case
    d, row = c["d"], c["d"] // 2 + 4 * (c["d"] // c["group"])       # bytes of one row of K or V in 4 bits
    if c["kind"] == "attn":
        n = sum(_lens(c))
        return {"bytes": 2 * n * c["hkv"] * row + 4 * c["batch"] * c["hq"] * d + 4 * c["batch"], "flops": 4 * n * c["hq"] * d}
    if c["kind"] == "write":                  # new rows in, codes out, and the values that they stand for
        n = 2 * sum(_writes(c)[1]) * c["heads"]
        return {"bytes": n * (2 * d + row + 2 * d), "flops": 8 * n * d}
    if c["kind"] == "read":
        n = 2 * sum(_lens(c)) * c["heads"]
        return {"bytes": n * (row + 2 * d), "flops": 2 * n * d}
    n = 2 * c["batch"] * c["hkv"]
    return {"bytes": 2 * c["batch"] * (2 * c["hq"] + 2 * c["hkv"]) * d + 4 * c["batch"] * d + n * (row + 2 * d),
            "flops": 3 * c["batch"] * (c["hq"] + c["hkv"]) * d + 8 * n * d}


# ---- the plain form ------------------------------------------------------------------------------------------------
def _shifts(device):
    return torch.arange(0, 32, 4, dtype=torch.int32, device=device)


def _quantise(x, group):
    """x [..., d] -> codes [..., d] int32, params [..., d / group, 2] fp16."""
    x = x.float().clamp(-LIMIT, LIMIT).unflatten(-1, (-1, group))
    base = x.amin(-1).half()
    scale = ((x.amax(-1) - base.float()) / 15).half()
    # in 64 bits: a quotient that lies on the border of two codes goes to the even one
    s, b = scale.double().unsqueeze(-1), base.double().unsqueeze(-1)
    codes = torch.where(s > 0, torch.round((x.double() - b) / torch.where(s > 0, s, 1.0)), 0.0).clamp(0, 15)
    return codes.int().flatten(-2), torch.stack((scale, base), -1)


def _pack(codes):
    u = codes.unflatten(-1, (-1, 8, 4)).transpose(-3, -2).flatten(-3).unflatten(-1, (-1, 8))
    return (u << _shifts(codes.device)).sum(-1).int()


def _values(words, params):
    """The cache rows as fp32: words [..., d / 8], params [..., d / group, 2]."""
    codes = ((words.unsqueeze(-1) >> _shifts(words.device)) & 15).flatten(-2)
    codes = codes.unflatten(-1, (8, -1, 4)).transpose(-3, -2).flatten(-3)
    p = params.float()
    codes = codes.unflatten(-1, (params.shape[-2], -1)).float()
    return (codes * p[..., 0:1] + p[..., 1:2]).flatten(-2)


def _context(cache, table):
    """[batch, heads, positions, ...] of a cache tensor, gathered through the block table where there is one."""
    return cache if table is None else cache[table.long()].transpose(1, 2).flatten(2, 3)


def _rows(s):
    """(index tensors of the rows that an append writes) for [batch, heads, tokens]."""
    c = s["case"]
    pos = s["first"].long()[:, None] + torch.arange(c["tokens"], device="cuda")[None]
    h = torch.arange(c["heads"], device="cuda")[None, :, None]
    if s["table"] is None:
        return torch.arange(c["batch"], device="cuda")[:, None, None], h, pos[:, None]
    return torch.gather(s["table"].long(), 1, pos // c["block"])[:, None], h, (pos % c["block"])[:, None]


def _plain_attn(s):
    c, t = s["case"], s["table"]
    k = _values(_context(s["kc"], t), _context(s["kp"], t))
    v = _values(_context(s["vc"], t), _context(s["vp"], t))
    q = s["q"].float().unflatten(1, (c["hkv"], -1))
    scores = (q @ k.transpose(-1, -2)) * s["scale"]
    seen = torch.arange(k.shape[2], device="cuda") < s["lens"][:, None, None, None]
    scores = torch.where(seen, scores, -torch.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=-3e38)          # a sequence without positions has no largest score
    p = torch.exp(scores - top)
    out = (p @ v) / p.sum(-1, keepdim=True).clamp(min=1e-30)
    return out.flatten(1, 2).to(s["q"].dtype)


def _plain_store(x, codes, params, at, new, group):
    """Rows x go into a cache at the places `at` where `new` says so; what they read back as."""
    w, p = _quantise(x, group)
    w, p = torch.where(new, _pack(w), codes[at]), torch.where(new[..., None], p, params[at])
    codes[at], params[at] = w, p
    return torch.where(new, _values(w, p), 0.0).to(x.dtype)


def _plain_write(s):
    c, at = s["case"], _rows(s)
    new = torch.arange(c["tokens"], device="cuda")[None] < s["count"][:, None]
    new = new[:, None, :, None]                                    # [batch, 1, tokens, 1]
    return [_plain_store(s["k"].transpose(1, 2), s["kc"], s["kp"], at, new, c["group"]),
            _plain_store(s["v"].transpose(1, 2), s["vc"], s["vp"], at, new, c["group"])]


def _plain_read(s):
    c, t = s["case"], s["table"]
    seen = (torch.arange(c["max_len"], device="cuda")[None] < s["lens"][:, None])[:, None, :, None]
    read = lambda w, p: torch.where(seen, _values(_context(w, t), _context(p, t)), 0.0).to(TYPES[c["dtype"]])  # noqa: E731
    return [read(s["kc"], s["kp"]), read(s["vc"], s["vp"])]


def _plain_rope(s):
    c = s["case"]
    d, hq, hkv = c["d"], c["hq"], c["hkv"]
    rows = s["qkv"].unflatten(-1, (-1, d))
    cos, sin = s["cos"][s["pos"].long()][:, None], s["sin"][s["pos"].long()][:, None]
    lo, hi = rows[:, :hq + hkv, :d // 2].float(), rows[:, :hq + hkv, d // 2:].float()
    rot = torch.cat((lo * cos - hi * sin, hi * cos + lo * sin), -1).to(rows.dtype)
    at = torch.arange(c["batch"], device="cuda")[:, None], torch.arange(hkv, device="cuda")[None], s["pos"].long()[:, None]
    new = torch.ones(c["batch"], hkv, 1, dtype=torch.bool, device="cuda")
    return [rot[:, :hq], _plain_store(rot[:, hq:], s["kc"], s["kp"], at, new, c["group"])[:, :, None],
            _plain_store(rows[:, hq + hkv:], s["vc"], s["vp"], at, new, c["group"])[:, :, None]]


# ---- the framework's calls -----------------------------------------------------------------------------------------
def _kernels():
    return importlib.import_module("triton-rs_b200").prelude


def _own(s):
    c, P = s["case"], _kernels()
    fn = lambda name: getattr(P, name + "_" + c["dtype"])          # noqa: E731
    cache = (s["kc"], s["kp"], s["vc"], s["vp"])
    if c["kind"] == "attn":
        if s["table"] is None:
            fn("batched_decode_attention_hm_int4")(s["q"], *cache, s["lens"], s["out"], c["batch"], c["hq"], c["hkv"], c["d"], c["group"],
                                                   c["max_len"], s["scale"])
        else:
            fn("batched_decode_attention_paged_int4")(s["q"], *cache, s["table"], s["lens"], s["out"], c["batch"], c["hq"], c["hkv"], c["d"],
                                                      c["group"], c["block"], s["blocks"], s["table"].shape[1], s["scale"])
        return s["out"]
    if c["kind"] == "write":
        st = c["heads"] * c["d"]
        if s["table"] is None:
            fn("kv_cache_append_hm_int4")(s["k"], s["v"], *cache, s["first"], s["count"], c["heads"], c["d"], c["group"], c["max_len"],
                                          c["batch"], c["tokens"], st, st)
        else:
            fn("kv_cache_append_paged_int4")(s["k"], s["v"], *cache, s["table"], s["first"], s["count"], c["heads"], c["d"], c["group"],
                                             c["block"], s["blocks"], s["table"].shape[1], c["batch"], c["tokens"], st, st)
    if c["kind"] == "rope":
        fn("rope_kv_append_hm_int4")(s["qkv"], s["cos"], s["sin"], s["pos"], s["out"], *cache, c["hq"], c["hkv"], c["d"], c["group"],
                                     c["max_len"], c["batch"])
        fn("kv_cache_read_hm_int4")(*cache, s["pos"], s["lens"], s["ko"], s["vo"], c["hkv"], c["d"], c["group"], c["max_len"], c["batch"], 1)
        return [s["out"], s["ko"], s["vo"]]
    first = s["first"] if c["kind"] == "write" else None
    if s["table"] is None:
        fn("kv_cache_read_hm_int4")(*cache, first, s["lens"], s["ko"], s["vo"], c["heads"], c["d"], c["group"], c["max_len"], c["batch"],
                                    s["ko"].shape[2])
    else:
        fn("kv_cache_read_paged_int4")(*cache, s["table"], first, s["lens"], s["ko"], s["vo"], c["heads"], c["d"], c["group"], c["block"],
                                       s["blocks"], s["table"].shape[1], c["batch"], s["ko"].shape[2])
    return [s["ko"], s["vo"]]


def run(state):
    if own:
        return _own(state)
    return {"attn": _plain_attn, "write": _plain_write, "read": _plain_read, "rope": _plain_rope}[state["case"]["kind"]](state)


# ---- inputs --------------------------------------------------------------------------------------------------------
def _cache(c, heads, g, dtype, fill):
    """(codes, params) of an empty cache, or of one that holds N(0, 1) rows with a spread that differs from dim to dim."""
    lead = (c["batch"], heads, c["max_len"]) if not c.get("paged") else (c["batch"] * (c["max_len"] // c["block"]) + 3, heads, c["block"])
    d, n = c["d"], c["d"] // c["group"]
    codes = torch.zeros(lead + (d // 8,), dtype=torch.int32, device="cuda")
    params = torch.zeros(lead + (n, 2), dtype=torch.float16, device="cuda")
    if fill:
        width = torch.exp(0.3 * torch.randn(heads, 1, d, device="cuda", generator=g))
        for i in range(0, lead[0], 64):       # a part at a time: the 64-bit quotients take room
            for j in range(0, lead[2], 8192):
                part = codes[i:i + 64, :, j:j + 8192]
                x = torch.randn(part.shape[:3] + (d,), device="cuda", generator=g).mul_(width).to(dtype)
                w, p = _quantise(x, c["group"])
                codes[i:i + 64, :, j:j + 8192], params[i:i + 64, :, j:j + 8192] = _pack(w), p
    return codes, params


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 + c["spread"])
    dt = TYPES[c["dtype"]]
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")                                   # noqa: E731
    randn = lambda *shape: torch.randn(*shape, device="cuda", generator=g).to(dt)                       # noqa: E731
    s = {"case": c, "table": None}
    heads = c.get("heads") or c["hkv"]
    if c.get("paged"):
        per = c["max_len"] // c["block"]
        s["blocks"] = c["batch"] * per + 3
        s["table"] = torch.randperm(s["blocks"], device="cuda", generator=g)[:c["batch"] * per].int().view(c["batch"], per).contiguous()
    filled = c["kind"] in ("attn", "read")
    s["kc"], s["kp"] = _cache(c, heads, g, dt, filled)
    s["vc"], s["vp"] = _cache(c, heads, g, dt, filled)
    if c["kind"] == "attn":
        s["q"], s["lens"], s["scale"] = randn(c["batch"], c["hq"], c["d"]), ints(_lens(c)), c["d"] ** -0.5
        s["out"] = torch.zeros_like(s["q"])
    elif c["kind"] == "write":
        first, count = _writes(c)
        s["first"], s["count"], s["lens"] = ints(first), ints(count), ints([a + b for a, b in zip(first, count)])
        s["k"], s["v"] = (randn(c["batch"], c["tokens"], heads, c["d"]) for _ in range(2))
        s["ko"], s["vo"] = (torch.zeros(c["batch"], heads, c["tokens"], c["d"], dtype=dt, device="cuda") for _ in range(2))
    elif c["kind"] == "read":
        s["lens"] = ints(_lens(c))
        s["ko"], s["vo"] = (torch.zeros(c["batch"], heads, c["max_len"], c["d"], dtype=dt, device="cuda") for _ in range(2))
    else:
        r = random.Random(c["spread"])
        pos = [r.randrange(c["max_len"]) for _ in range(c["batch"])]
        s["pos"], s["lens"] = ints(pos), ints([p + 1 for p in pos])
        # angles in 64 bits: position * frequency loses its fraction in 32 at far positions
        turn = torch.arange(c["max_len"], device="cuda").double()[:, None] * 500000.0 ** (-torch.arange(0, c["d"], 2, device="cuda").double() / c["d"])
        s["cos"], s["sin"] = turn.cos().float().contiguous(), turn.sin().float().contiguous()
        s["qkv"] = randn(c["batch"], (c["hq"] + 2 * heads) * c["d"])
        s["out"] = torch.zeros(c["batch"], c["hq"], c["d"], dtype=dt, device="cuda")
        s["ko"], s["vo"] = (torch.zeros(c["batch"], heads, 1, c["d"], dtype=dt, device="cuda") for _ in range(2))
    return s


# ---- from the definition, in 64 bits ---------------------------------------------------------------------------------
def _exact_rows(words, params, d):
    """Rows in 64 bits, dim by dim: dim e of unit u = e // 4 stands at place (u % 8) * (d / 32) + u // 8 of the row."""
    e = torch.arange(d, device="cuda")
    u = e // 4
    place = (u % 8) * (d // 32) + u // 8
    code = (words[..., place // 2].long() >> (16 * (place % 2) + 4 * (e % 4))) & 15
    of = e // (d // params.shape[-2])
    return code.double() * params[..., of, 0].double() + params[..., of, 1].double()


def _exact_stored(x, group):
    """What a row reads back as, in 64 bits: the two roundings of scale and base belong to the format."""
    x = x.double().clamp(-LIMIT, LIMIT)
    y = x.reshape(x.shape[:-1] + (x.shape[-1] // group, group))
    low = y.min(-1, keepdim=True).values.half().double()
    step = ((y.max(-1, keepdim=True).values - low) / 15).half().double()
    n = torch.where(step == 0, torch.zeros_like(y), ((y - low) / step.clamp(min=1e-30)).round().clamp(0, 15))
    return (n * step + low).reshape(x.shape)


def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    d = c["d"]
    if c["kind"] in ("attn", "read"):
        heads = s["kc"].shape[1]
        outs = [torch.zeros_like(s["out"], dtype=torch.float64)] if c["kind"] == "attn" else [torch.zeros_like(s["ko"], dtype=torch.float64) for _ in range(2)]
        for b, n in enumerate(_lens(c)):
            if n == 0:
                continue
            if s["table"] is None:
                pick = lambda a: a[b, :, :n]                                                             # noqa: E731
            else:
                p = torch.arange(n, device="cuda")
                blk = s["table"][b].long()[p // c["block"]]
                pick = lambda a: a[blk, :, p % c["block"]].movedim(0, 1)                                 # noqa: E731
            k, v = (_exact_rows(pick(s[x + "c"]), pick(s[x + "p"]), d) for x in "kv")
            if c["kind"] == "read":
                outs[0][b, :, :n], outs[1][b, :, :n] = k, v
                continue
            q = s["q"][b].double().reshape(heads, -1, d)
            z = torch.einsum("hgd,hpd->hgp", q, k) * s["scale"]
            outs[0][b] = torch.einsum("hgp,hpd->hgd", torch.softmax(z, -1), v).reshape(-1, d)
        return outs[0] if c["kind"] == "attn" else outs
    if c["kind"] == "write":
        new = (torch.arange(c["tokens"], device="cuda") < s["count"][:, None])[:, None, :, None]
        return [torch.where(new, _exact_stored(s[x], c["group"]).transpose(1, 2), 0.0) for x in "kv"]
    x = s["qkv"].double().reshape(c["batch"], -1, d)
    r = x[:, :c["hq"] + c["hkv"]]
    z = torch.complex(r[..., :d // 2], r[..., d // 2:])
    at = s["pos"].long()
    z = z * torch.complex(s["cos"][at].double(), s["sin"][at].double())[:, None]
    r = torch.cat((z.real, z.imag), -1)
    k = r[:, c["hq"]:].to(s["qkv"].dtype)      # the rotated key is rounded to its type before it is quantised, as the unfused calls round it
    return [r[:, :c["hq"]], _exact_stored(k, c["group"])[:, :, None], _exact_stored(x[:, c["hq"] + c["hkv"]:], c["group"])[:, :, None]]
