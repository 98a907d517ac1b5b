"""The operators between a decoder layer's qkv linear and its output linear: rotary positions, a paged key-value cache
that is quantised as it is written and read back, and the attention of one new token a sequence over that cache.

`own` is False: every operator in its plain form, elementary torch operations in 32 bits.  `own` is True: the calls a
program makes of kairos_amd.ops.

A cache is a uint8 tensor [pages, kv_heads, tiles a page, bytes a tile]; a tile is 32 consecutive tokens of one head, and
holds their keys, then their values, then (8- and 4-bit kinds) their fp16 factors, in the order in which the lanes of a
matrix instruction take them:
  keys    [unit groups][lane group g 4][row 16][n units][8 elements], n = 1 / 2 / 4 for f16 / int8 / int4; unit
          (h, kk) is elements 32 kk + 8 g .. + 7 of token 8 (row // 4) + 4 h + row % 4; int4: element e of a unit is
          nibble e // 2 + 4 (e % 2) of the unit's 32-bit word
  values  [D / 16 n][token // 8][16][token % 8] words of 16 bits, each n neighbouring elements of a token, low bits first
  factors [32] fp16 each: int8: key scale, value scale; int4: key scale, key offset, value scale, value offset
int8 holds u = code + 128 and stands for scale * (u - 128); int4 stands for scale * u + offset.
"""
import math

import torch

own = False

TILE = 32
PER_WORD = {"f16": 1, "int8": 2, "int4": 4}                      # elements in 16 bits
TABLES = {"f16": 0, "int8": 2, "int4": 4}                        # fp16 factors a token


# ---- cases ------------------------------------------------------------------------------------------------------------
def _case(name, op, batch, heads, kv_heads, head_dim, **more):
    return dict(name=name, op=op, batch=batch, heads=heads, kv_heads=kv_heads, head_dim=head_dim, **more)


def listed():
    return [
        # queries and keys of one decode step, eight sequences at unequal positions: a call of launch latency
        _case("rotary decode 8", "rotary", 8, 32, 8, 128, tokens=1, start=2047, rotary_dim=128, interleaved=False, scaling="llama3"),
        # a prefill batch of odd length, neighbouring pairs, half of the head rotated, positions far into a long context
        _case("rotary prefill 4x4001", "rotary", 4, 28, 4, 128, tokens=4001, start=100000, rotary_dim=64, interleaved=True, scaling="yarn"),
        # one decode step of a serving batch: its keys rotated and quantised into the cache, as they then stand in it
        _case("append decode 32 int8", "append", 32, 32, 8, 128, tokens=1, start=1500, rotary_dim=128, interleaved=False,
              scaling="none", kind="int8", page=64),
        # a chunk of a prompt behind one already cached: odd start and length, so tiles and pages begin and end inside it
        _case("append chunk 3x777 f16", "append", 3, 64, 8, 128, tokens=777, start=333, rotary_dim=128, interleaved=False,
              scaling="linear", kind="f16", page=32),
        # a whole prefill at the batch of the decoder command, four bits a value
        _case("append prefill 32x1024 int4", "append", 32, 32, 8, 128, tokens=1024, start=0, rotary_dim=128, interleaved=False,
              scaling="llama3", kind="int4", page=128),
        # a cached prefix handed back to a chunked prefill
        _case("read 2x5003 int8", "read", 2, 32, 8, 128, tokens=5003, start=0, kind="int8", page=64),
        # the cached prompts of a batch, narrow heads
        _case("read 16x8000 int4", "read", 16, 8, 8, 64, tokens=8000, start=17, kind="int4", page=256),
        # the first answers of a chat: one sequence, a short context
        _case("attend 1x200 f16", "attend", 1, 32, 8, 128, length=200, ragged=False, window=0, kind="f16", page=64),
        # the decoder command's batch at its last token, eight bits
        _case("attend 32x1536 int8", "attend", 32, 32, 8, 128, length=1536, ragged=False, window=0, kind="int8", page=64),
        # a serving batch of very unequal lengths, seven query heads to a key head
        _case("attend 64 ragged 8192 f16", "attend", 64, 28, 4, 128, length=8192, ragged=True, window=0, kind="f16", page=32),
        # few sequences in a very long context, four bits, eight query heads to a key head
        _case("attend 4x100001 int4", "attend", 4, 64, 8, 128, length=100001, ragged=False, window=0, kind="int4", page=128),
        # one document of the longest context
        _case("attend 2x131072 f16", "attend", 2, 32, 8, 128, length=131072, ragged=False, window=0, kind="f16", page=256),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(("rotary", "append", "read", "attend", "attend"))
    heads, kv, d = rng.choice(((32, 8, 128), (64, 8, 128), (28, 4, 128), (40, 8, 128), (8, 8, 64), (20, 1, 64), (16, 2, 256)))
    kind = rng.choice(("f16", "int8", "int4"))
    page = 32 * rng.choice((1, 2, 3, 4, 8))
    if op == "attend":
        b = _log(rng, 1, 64)
        most = 2 * 131072 * 8 * 512 // (b * kv * d * 4)           # as many elements as the longest listed cache
        length = _log(rng, 1, min(131072, most))
        return dict(op=op, batch=b, heads=heads, kv_heads=kv, head_dim=d, length=length, ragged=rng.random() < 0.5,
                    window=rng.choice((0, 0, 0, _log(rng, 1, 4096))), kind=kind, page=page)
    b = _log(rng, 1, 32)
    most = 32768 * 48 * 128 // (b * (heads + 2 * kv) * d) if op != "read" else 16 * 8000 * 8 * 64 // (b * kv * d)
    s = _log(rng, 1, min(4096, most)) if rng.random() < 0.75 else 1
    c = dict(op=op, batch=b, heads=heads, kv_heads=kv, head_dim=d, tokens=s, start=rng.choice((0, _log(rng, 1, 8000))))
    if op != "read":
        c.update(rotary_dim=rng.choice((d, d, d // 2, 32)), interleaved=rng.random() < 0.4,
                 scaling=rng.choice(("none", "linear", "llama3", "yarn")))
    if op != "rotary":
        c.update(kind=kind, page=page)
    return c


# ---- what a program has in hand ----------------------------------------------------------------------------------------
def _table(positions, dim, scaling):
    """cos, sin fp32 [positions, dim / 2, 2] of base 500000, from 64-bit angles."""
    f = 500000.0 ** (-torch.arange(0, dim, 2, dtype=torch.float64, device="cuda") / dim)
    gain = 1.0
    if scaling == "linear":
        f = f / 4.0
    elif scaling == "llama3":                                     # long wavelengths divided by 8, a ramp in between
        turns = 8192 * f / (2 * math.pi)
        keep = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        f = f * keep + f / 8.0 * (1 - keep)
    elif scaling == "yarn":
        turns = 8192 * f / (2 * math.pi)
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0, 1)
        f = f * keep + f / 16.0 * (1 - keep)
        gain = 0.1 * math.log(16.0) + 1.0
    t = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * f
    return torch.stack((torch.cos(t) * gain, torch.sin(t) * gain), dim=-1).float().contiguous()


def _spread(n, b):
    """n for the first sequence, then lengths spread over 1 .. n."""
    return [n] + [1 + int((n - 1) * ((0.6180339887 * i) % 1.0)) for i in range(1, b)]


def _starts(case):
    """Sequences do not stand at the same position: up to 30 before the given one."""
    return [max(0, case["start"] - (7 * i) % 31) for i in range(case["batch"])]


def _lens(case):
    return _spread(case["length"], case["batch"]) if case["ragged"] else [case["length"]] * case["batch"]


def _tile_bytes(kind, d):
    return 4 * TILE * d // PER_WORD[kind] + 2 * TILE * TABLES[kind]


def _pages(case, lens, g):
    """Page table int32 [batch, widest] over a pool in random order (-1 behind a sequence's pages), and the pool's size."""
    page = case["page"]
    need = torch.tensor([-(-n // page) for n in lens], device="cuda")
    pool = int(need.sum()) + 3
    order = torch.randperm(pool, generator=g, device="cuda")
    at = torch.arange(max(1, int(need.max())), device="cuda")[None, :]
    first = torch.cumsum(need, 0) - need
    entry = order[(first[:, None] + at).clamp(max=pool - 1)]
    return torch.where(at < need[:, None], entry, -1).to(torch.int32).contiguous(), pool


def _random_cache(case, pool, g):
    """Codes and factors as rows of normal values leave them."""
    d, kind, tiles = case["head_dim"], case["kind"], case["page"] // TILE
    shape = (pool, case["kv_heads"], tiles)
    if kind == "f16":
        return torch.randn(shape + (2 * TILE * d,), generator=g, device="cuda", dtype=torch.float16).view(torch.uint8)
    cache = torch.empty(shape + (_tile_bytes(kind, d),), dtype=torch.uint8, device="cuda")
    codes = cache.shape[-1] - 2 * TILE * TABLES[kind]
    size = torch.empty(shape + (TABLES[kind], TILE), device="cuda").uniform_(0.7, 1.4, generator=g)
    if kind == "int8":
        u = torch.randn(shape + (codes,), generator=g, device="cuda", dtype=torch.float16).mul_(45.0).round_().clamp_(-127, 127).add_(128)
        cache[..., :codes] = u.to(torch.uint8)
        size *= 2.8 / 127.0
    else:
        u = torch.randn(shape + (codes, 2), generator=g, device="cuda", dtype=torch.float16).mul_(2.8).add_(7.5).round_().clamp_(0, 15)
        u = u.to(torch.uint8)
        cache[..., :codes] = u[..., 0] + 16 * u[..., 1]
        size[..., 0::2, :] *= 5.4 / 15.0
        size[..., 1::2, :] = size[..., 0::2, :] * -7.5
    cache[..., codes:] = size.to(torch.float16).view(torch.uint8).reshape(shape + (-1,))
    return cache


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    b, h, kv, d = case["batch"], case["heads"], case["kv_heads"], case["head_dim"]
    st = dict(case)
    if case["op"] == "attend":
        lens = _lens(case)
        st["page_table"], pool = _pages(case, lens, g)
        st["cache"] = _random_cache(case, pool, g)
        st["q"] = torch.randn((b, h, d), generator=g, device="cuda", dtype=torch.float16) * 2.0
        st["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        return st
    starts = _starts(case)
    st["start_at"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    if case["op"] != "read":
        # the output of the fused qkv linear; queries, keys and values are views of it
        qkv = torch.randn((b, case["tokens"], h + 2 * kv, d), generator=g, device="cuda", dtype=torch.float16)
        st["q"], st["k"], st["v"] = qkv[:, :, :h], qkv[:, :, h:h + kv], qkv[:, :, h + kv:]
        st["table"] = _table(max(starts) + case["tokens"], case["rotary_dim"], case["scaling"])
    if case["op"] != "rotary":
        st["page_table"], pool = _pages(case, [s + case["tokens"] for s in starts], g)
        if case["op"] == "read":
            st["cache"] = _random_cache(case, pool, g)
        else:
            st["cache"] = torch.zeros((pool, kv, case["page"] // TILE, _tile_bytes(case["kind"], d)), dtype=torch.uint8, device="cuda")
    return st


# ---- the plain forms ---------------------------------------------------------------------------------------------------
def _rotate(x, st):
    """x fp16 [B, S, heads, D]; the first rotary_dim elements of every head turned by their token's angles."""
    r, s = st["rotary_dim"], x.shape[1]
    pos = st["start_at"].long()[:, None] + torch.arange(s, device=x.device)
    cs = st["table"][pos][:, :, None]                             # [B, S, 1, R / 2, 2]
    cos, sin = cs[..., 0], cs[..., 1]
    t = x[..., :r].float()
    if st["interleaved"]:
        a, b = t[..., 0::2], t[..., 1::2]
        t = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = t[..., : r // 2], t[..., r // 2:]
        t = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((t.half(), x[..., r:]), dim=-1)


def _scale_up(width, steps):
    """The fp16 next to width / steps, one step up where `steps` of it would fall short of the width."""
    s = (width.double() / steps).float().half()
    return torch.where(s.float() * steps < width, (s.view(torch.int16) + 1).view(torch.float16), s)


def _inverse(s):
    return torch.where(s > 0, (1.0 / s.double()).float(), torch.zeros_like(s, dtype=torch.float32))


def _held(x, kind):
    """The values that a cache of this kind holds for the rows x fp16 [..., D]."""
    if kind == "f16":
        return x
    t = x.float()
    if kind == "int8":
        s = _scale_up(t.abs().amax(-1, keepdim=True), 127)
        v = torch.round(t * _inverse(s)).clamp(-127, 127) * s.float()
    else:
        lo = t.amin(-1, keepdim=True)
        s = _scale_up(t.amax(-1, keepdim=True) - lo, 15)
        v = torch.round((t - lo) * _inverse(s)).clamp(0, 15) * s.float() + lo
    return v.clamp(-65504, 65504).half()


def _values(tiles, kind, d):
    """Keys and values fp32 [..., 32, D] of tiles uint8 [..., bytes a tile]."""
    lead, n, part = tiles.shape[:-1], PER_WORD[kind], 2 * TILE * d // PER_WORD[kind]
    keys, vals, fac = tiles[..., :part], tiles[..., part:2 * part], tiles[..., 2 * part:].contiguous()
    if kind == "f16":
        k = keys.contiguous().view(torch.float16).float().reshape(lead + (2, d // 32, 4, 4, 4, 8))
        v = vals.contiguous().view(torch.float16).float().reshape(lead + (d // 16, 4, 16, 8, 1))
    elif kind == "int8":
        k = (keys.float() - 128.0).reshape(lead + (d // 32, 64, 2, 8)).transpose(-3, -2).reshape(lead + (2, d // 32, 4, 4, 4, 8))
        v = (vals.float() - 128.0).reshape(lead + (d // 32, 4, 16, 8, 2))
    else:
        nib = torch.stack((keys & 15, keys >> 4), dim=-1).reshape(lead + (d // 64, 64, 4, 2, 4))      # [.., unit, e % 2, e // 2]
        k = nib.transpose(-2, -1).reshape(lead + (d // 64, 64, 4, 8)).transpose(-3, -2).reshape(lead + (2, d // 32, 4, 4, 4, 8)).float()
        v = torch.stack((vals & 15, vals >> 4), dim=-1).reshape(lead + (d // 64, 4, 16, 8, 4)).float()
    z = len(lead)
    k = k.permute(*range(z), z + 3, z, z + 4, z + 1, z + 2, z + 5).reshape(lead + (TILE, d))
    v = v.permute(*range(z), z + 1, z + 3, z, z + 2, z + 4).reshape(lead + (TILE, d))
    if kind != "f16":
        f = fac.view(torch.float16).float().reshape(lead + (TABLES[kind], TILE, 1))
        k, v = (k * f[..., 0, :, :], v * f[..., 1, :, :]) if kind == "int8" else (
            k * f[..., 0, :, :] + f[..., 1, :, :], v * f[..., 2, :, :] + f[..., 3, :, :])
    return k, v


def _dense(st, tokens):
    """Keys and values fp32 [B, kv_heads, >= tokens, D] of the sequences' first tokens, whole pages of them."""
    table = st["page_table"][:, : -(-tokens // st["page"])].long().clamp(min=0)
    k, v = _values(st["cache"][table].transpose(1, 2), st["kind"], st["head_dim"])     # [B, heads, pages, tiles, 32, D]
    return k.flatten(2, 4), v.flatten(2, 4)


def _plain_attend(st):
    b, h, d = st["q"].shape
    kv, lens = st["kv_heads"], st["lens"].long()
    k, v = _dense(st, st["length"])
    q = st["q"].float().reshape(b, kv, h // kv, d)
    s = torch.matmul(q, k.transpose(2, 3).contiguous()) * d ** -0.5
    t = torch.arange(k.shape[2], device=s.device)
    seen = t[None, :] < lens[:, None]
    if st["window"]:
        seen = seen & (t[None, :] >= (lens - st["window"])[:, None])
    seen = seen[:, None, None, :]
    s = s.masked_fill(~seen, float("-inf"))
    p = torch.exp(s - s.amax(-1, keepdim=True))
    return (torch.matmul(p, v) / p.sum(-1, keepdim=True)).reshape(b, h, d).half()


def _plain_read(st):
    k, v = _dense(st, st["page"] * st["page_table"].shape[1])
    b, s = st["batch"], st["tokens"]
    at = st["start_at"].long()[:, None] + torch.arange(s, device=k.device)
    row = torch.arange(b, device=k.device)[:, None]
    return [k.transpose(1, 2)[row, at].half(), v.transpose(1, 2)[row, at].half()]


def run(state):
    st = state
    if own:
        from kairos_amd import ops
        if st["op"] == "attend":
            return ops.paged_attention(st["q"], st["cache"], st["page_table"], st["lens"], window=st["window"])
        if st["op"] == "read":
            return list(ops.kv_read(st["cache"], st["page_table"], st["start_at"], st["tokens"]))
        if st["op"] == "rotary":
            return list(ops.rotary(st["q"], st["k"], st["start_at"], st["table"], interleaved=st["interleaved"]))
        q = ops.kv_append(st["cache"], st["page_table"], st["start_at"], st["k"], st["v"], st["table"], q=st["q"],
                          interleaved=st["interleaved"])
        return [q, *ops.kv_read(st["cache"], st["page_table"], st["start_at"], st["tokens"])]
    if st["op"] == "attend":
        return _plain_attend(st)
    if st["op"] == "read":
        return _plain_read(st)
    q, k = _rotate(st["q"], st), _rotate(st["k"], st)
    if st["op"] == "rotary":
        return [q, k]
    return [q, _held(k, st["kind"]), _held(st["v"], st["kind"])]


# ---- what a pass cannot do without --------------------------------------------------------------------------------------
def work(case):
    b, h, kv, d = case["batch"], case["heads"], case["kv_heads"], case["head_dim"]
    token = _tile_bytes(case["kind"], d) / TILE if "kind" in case else 0         # cache bytes of a token's key and value
    if case["op"] == "attend":
        lens = [min(n, case["window"] or n) for n in _lens(case)]
        return {"bytes": sum(lens) * kv * token + 4 * b * h * d, "flops": 4.0 * sum(lens) * h * d}
    rows = b * case["tokens"]
    if case["op"] == "read":
        return {"bytes": rows * kv * (token + 4 * d), "flops": 4.0 * rows * kv * d}
    table = case["tokens"] * case["rotary_dim"] * 4
    if case["op"] == "rotary":
        return {"bytes": rows * (h + kv) * d * 4 + table, "flops": 3.0 * rows * (h + kv) * case["rotary_dim"]}
    # queries in and out; keys and values in, into the cache, out of it, and out as they stand there
    return {"bytes": rows * (4 * h * d + kv * (8 * d + 2 * token)) + table,
            "flops": 3.0 * rows * (h + kv) * case["rotary_dim"] + 8.0 * rows * kv * d}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------
def _exact_rotate(x, st):
    r, s, x = st["rotary_dim"], x.shape[1], x.double()
    i = torch.arange(r // 2, device=x.device)
    first, second = (2 * i, 2 * i + 1) if st["interleaved"] else (i, i + r // 2)
    out = x.clone()
    for b in range(x.shape[0]):
        p = int(st["start_at"][b])
        z = torch.view_as_complex(st["table"][p:p + s].double())[:, None]
        w = torch.complex(x[b][..., first], x[b][..., second]) * z
        out[b][..., first], out[b][..., second] = w.real, w.imag
    return out


def _exact_held(x, kind):
    if kind == "f16":
        return x
    lo = torch.zeros_like(x[..., :1]) if kind == "int8" else x.amin(-1, keepdim=True)
    steps = 127 if kind == "int8" else 15
    width = (x - lo).abs().amax(-1, keepdim=True).float().double()
    s = (width / steps).half().double()
    e = torch.floor(torch.log2(s.clamp(min=2.0 ** -14)))
    s = torch.where(s * steps < width, s + torch.exp2(e - 10), s)
    u = torch.round((x - lo) / torch.where(s > 0, s, torch.ones_like(s)))
    return u * s + lo


def _exact_tokens(st, b, head, first, last):
    """Keys and values fp64 [last - first, D] of one head of one sequence, by the byte address of every element."""
    d, kind, page, dev = st["head_dim"], st["kind"], st["page"], st["cache"].device
    n, part = PER_WORD[kind], 2 * TILE * d // PER_WORD[kind]
    at = torch.arange(first, last, device=dev)
    flat, tile_bytes = st["cache"].view(-1), st["cache"].shape[-1]
    tiles = page // TILE
    tile = (st["page_table"][b].long()[at // page] * st["kv_heads"] + head) * tiles + at % page // TILE
    base, tok, e = (tile * tile_bytes)[:, None], (at % TILE)[:, None], torch.arange(d, device=dev)[None, :]
    row, half = 4 * (tok // 8) + tok % 4, tok // 4 % 2
    unit = half * (d // 32) + e // 32
    chunk = (unit // n) * 1024 + (e % 32 // 8 * 16 + row) * 16
    word = part + ((e // (16 * n) * 4 + tok // 8) * 16 + e % (16 * n) // n) * 16 + tok % 8 * 2

    def half_at(o):
        return flat.view(torch.float16)[o // 2].double()

    def fac(i):
        return half_at(base + 2 * part + 2 * (TILE * i + tok))

    if kind == "f16":
        return half_at(base + chunk + e % 8 * 2), half_at(base + word)
    if kind == "int8":
        k = flat[base + chunk + unit % 2 * 8 + e % 8].double() - 128
        return k * fac(0), (flat[base + word + e % 2].double() - 128) * fac(1)
    place = e % 8 // 2 + 4 * (e % 2)
    k = (flat[base + chunk + unit % 4 * 4 + place // 2].long() >> (4 * (place % 2))) & 15
    v = (flat[base + word + e % 4 // 2].long() >> (4 * (e % 2))) & 15
    return k.double() * fac(0) + fac(1), v.double() * fac(2) + fac(3)


def exact(case, seed):
    st = prepare(case, seed)
    b, h, kv, d = case["batch"], case["heads"], case["kv_heads"], case["head_dim"]
    if case["op"] == "attend":
        out = torch.zeros((b, h, d), dtype=torch.float64, device="cuda")
        for i, n in enumerate(_lens(case)):
            first = max(0, n - case["window"]) if case["window"] else 0
            for j in range(kv):
                k, v = _exact_tokens(st, i, j, first, n)
                q = st["q"][i, j * (h // kv):(j + 1) * (h // kv)].double()
                out[i, j * (h // kv):(j + 1) * (h // kv)] = torch.softmax(q @ k.T.contiguous() / math.sqrt(d), dim=-1) @ v
        return out
    if case["op"] == "read":
        k = torch.empty((b, case["tokens"], kv, d), dtype=torch.float64, device="cuda")
        v = torch.empty_like(k)
        for i, s in enumerate(_starts(case)):
            for j in range(kv):
                k[i, :, j], v[i, :, j] = _exact_tokens(st, i, j, s, s + case["tokens"])
        return [k, v]
    q, k = _exact_rotate(st["q"], st), _exact_rotate(st["k"], st)
    if case["op"] == "rotary":
        return [q, k]
    return [q, _exact_held(k.half().double(), case["kind"]), _exact_held(st["v"].double(), case["kind"])]
