"""CPU restatement (numpy) of the decoder operators behind the qkv linear: rotary positions, the paged key-value cache's codes and
byte layout, attention of one token over it.  Written from the formulas, element by element; used by the tests only."""
import numpy as np

TILE = 32
PER_WORD = {"f16": 1, "int8": 2, "int4": 4}
FACTORS = {"f16": 0, "int8": 2, "int4": 4}


def tile_bytes(D, kind):
    return 4 * TILE * D // PER_WORD[kind] + 2 * TILE * FACTORS[kind]


def rotate(x, pos, table, interleaved, dtype=np.float64):
    """x fp16 [..., heads, D], pos int [...]: turned in `dtype`, every product and sum rounded to it; not rounded to fp16."""
    R = 2 * table.shape[1]
    c, s = table[pos].astype(dtype)[..., None, :, 0], table[pos].astype(dtype)[..., None, :, 1]
    y = x.astype(dtype)
    i = np.arange(R // 2)
    first, second = (2 * i, 2 * i + 1) if interleaved else (i, i + R // 2)
    a, b = y[..., first].copy(), y[..., second].copy()
    y[..., first] = a * c - b * s
    y[..., second] = b * c + a * s
    return y


def _scale_up(width, steps):
    s = (width / np.float32(steps)).astype(np.float32).astype(np.float16)
    short = s.astype(np.float32) * np.float32(steps) < width
    return np.where(short, (s.view(np.uint16) + 1).view(np.float16), s)


def quantise(x, kind):
    """x fp16 [..., D] -> (codes uint8 [..., D], scale fp16 [...], offset fp16 [...])."""
    f = x.astype(np.float32)
    if kind == "int8":
        z = np.zeros(x.shape[:-1], np.float16)
        s = _scale_up(np.abs(f).max(-1), 127)
    else:
        z = x.min(-1) + np.float16(0)             # never -0
        s = _scale_up(f.max(-1) - f.min(-1), 15)
    with np.errstate(divide="ignore"):
        r = np.where(s > 0, np.float32(1.0) / s.astype(np.float32), np.float32(0.0)).astype(np.float32)
    t = np.rint((f - z.astype(np.float32)[..., None]) * r[..., None])
    u = np.clip(t, -127, 127) + 128 if kind == "int8" else np.clip(t, 0, 15)
    return u.astype(np.uint8), s, z


def values_of(u, s, z, kind, dtype=np.float64):
    u = u.astype(dtype)
    if kind == "int8":
        return (u - 128) * s.astype(dtype)[..., None]
    return u * s.astype(dtype)[..., None] + z.astype(dtype)[..., None]


def to_f16(v):
    return np.clip(v, -65504.0, 65504.0).astype(np.float16)


# ---- the tile's bytes ---------------------------------------------------------------------------------------------------
def key_place(tau, d, D, kind):
    """(byte, shift) of key element d of token tau in its tile."""
    n = PER_WORD[kind]
    row, half, kk, g, e = 4 * (tau // 8) + tau % 4, tau // 4 % 2, d // 32, d // 8 % 4, d % 8
    unit = half * (D // 32) + kk
    at = unit // n * 1024 + (16 * g + row) * 16 + unit % n * (16 // n)
    if kind == "f16":
        return at + 2 * e, 0
    if kind == "int8":
        return at + e, 0
    nib = e // 2 + 4 * (e % 2)
    return at + nib // 2, 4 * (nib % 2)


def value_place(tau, d, D, kind):
    n = PER_WORD[kind]
    c, dl, a = d // (16 * n), d % (16 * n) // n, d % n
    at = 2 * TILE * D // n + (c * 64 + tau // 8 * 16 + dl) * 16 + tau % 8 * 2
    if kind == "f16":
        return at, 0
    if kind == "int8":
        return at + a, 0
    return at + a // 2, 4 * (a % 2)


def factor_place(tau, i, D, kind):
    return 4 * TILE * D // PER_WORD[kind] + 2 * (TILE * i + tau)


def _put_f16(tile, at, h):
    tile[at:at + 2] = np.array([h], np.float16).view(np.uint8)


def _get_f16(tile, at):
    return tile[at:at + 2].copy().view(np.float16)[0]


def put_token(tile, tau, k, v, kind):
    """Writes fp16 rows k, v [D] of one token into a tile (uint8 [tile_bytes])."""
    D = k.shape[0]
    if kind == "f16":
        for d in range(D):
            _put_f16(tile, key_place(tau, d, D, kind)[0], k[d])
            _put_f16(tile, value_place(tau, d, D, kind)[0], v[d])
        return
    for part, (x, place) in enumerate(((k, key_place), (v, value_place))):
        u, s, z = quantise(x, kind)
        for d in range(D):
            at, shift = place(tau, d, D, kind)
            if kind == "int8":
                tile[at] = u[d]
            else:
                tile[at] = (int(tile[at]) & (0xF0 >> shift)) | (int(u[d]) << shift)
        per = FACTORS[kind] // 2
        _put_f16(tile, factor_place(tau, per * part, D, kind), s)
        if kind == "int4":
            _put_f16(tile, factor_place(tau, per * part + 1, D, kind), z)


def get_tile(tile, D, kind):
    """Keys and values fp64 [32, D] that a tile stands for."""
    out = np.empty((2, TILE, D))
    for part, place in enumerate((key_place, value_place)):
        for tau in range(TILE):
            at = [place(tau, d, D, kind) for d in range(D)]
            if kind == "f16":
                idx = np.array([a for a, _ in at])
                raw = np.stack((tile[idx], tile[idx + 1]), -1).copy().view(np.float16)[:, 0]
                out[part, tau] = raw
                continue
            u = np.array([(int(tile[a]) >> s) & (255 if kind == "int8" else 15) for a, s in at], np.uint8)
            per = FACTORS[kind] // 2
            s = _get_f16(tile, factor_place(tau, per * part, D, kind))
            z = _get_f16(tile, factor_place(tau, per * part + 1, D, kind)) if kind == "int4" else np.float16(0)
            out[part, tau] = values_of(u, np.float16(s), np.float16(z), kind)
    return out[0], out[1]


_PLACES = {}


def get_tiles(tiles, D, kind):
    """Keys and values fp64 [n, 32, D] of tiles uint8 [n, tile_bytes]: get_tile by whole index arrays."""
    if (D, kind) not in _PLACES:
        _PLACES[D, kind] = [np.array([[place(tau, d, D, kind) for d in range(D)] for tau in range(TILE)]) for place in (key_place, value_place)]
    out = []
    for part, at in enumerate(_PLACES[D, kind]):
        byte, shift = at[..., 0], at[..., 1]
        if kind == "f16":
            out.append(np.stack((tiles[:, byte], tiles[:, byte + 1]), -1).view(np.float16)[..., 0].astype(np.float64))
            continue
        u = (tiles[:, byte].astype(np.int64) >> shift) & (255 if kind == "int8" else 15)
        per = FACTORS[kind] // 2

        def factor(i):
            lo = np.array([factor_place(tau, i, D, kind) for tau in range(TILE)])
            return np.stack((tiles[:, lo], tiles[:, lo + 1]), -1).view(np.float16)[..., 0]

        out.append(values_of(u, factor(per * part), factor(per * part + 1) if kind == "int4" else np.float16(0), kind))
    return out


def sequence(cache, page_row, length, head, D, kind):
    """Keys and values fp64 [length, D] of one head of one sequence."""
    if not length:
        return np.zeros((0, D)), np.zeros((0, D))
    per = cache.shape[2]
    t = np.arange(-(-length // TILE))
    k, v = get_tiles(cache[np.asarray(page_row)[t // per], head, t % per], D, kind)
    return k.reshape(-1, D)[:length], v.reshape(-1, D)[:length]


def attend(q, k, v, scale):
    """q fp16 [G, D], k, v fp64 [T, D] -> (o fp64 [G, D], sum p |v| / sum p, sum p with p relative to the largest, p / sum p)."""
    if not len(k):
        return np.zeros(q.shape), np.zeros(q.shape), np.zeros((len(q), 1)), np.zeros((len(q), 0))
    s = q.astype(np.float64) @ k.T * scale
    p = np.exp(s - s.max(-1, keepdims=True))
    t = p.sum(-1, keepdims=True)
    return p @ v / t, p @ np.abs(v) / t, t, p / t


# ---- how far the kernel may be off ----------------------------------------------------------------------------------------
MIDDLE = {"f16": 0.0, "int8": 128.0, "int4": 7.5}


def sequence_codes(cache, page_row, first, length, head, D, kind):
    """What the cache holds for positions first .. length - 1 of one head, taken apart: for keys and for values (codes [T, D], scale
    [T], offset [T]), all fp64, so that the value is scale * (code - 128) (int8), scale * code + offset (int4), code (f16)."""
    per = cache.shape[2]
    t = np.arange(-(-length // TILE))
    tiles = cache[np.asarray(page_row)[t // per], head, t % per]
    get_tiles(tiles[:1], D, kind)
    out = []
    for part, at in enumerate(_PLACES[D, kind]):
        byte, shift = at[..., 0], at[..., 1]
        per_part = FACTORS[kind] // 2

        def factor(i):
            lo = np.array([factor_place(tau, i, D, kind) for tau in range(TILE)])
            return np.stack((tiles[:, lo], tiles[:, lo + 1]), -1).view(np.float16)[..., 0].astype(np.float64).reshape(-1)[first:length]

        if kind == "f16":
            u = np.stack((tiles[:, byte], tiles[:, byte + 1]), -1).view(np.float16)[..., 0].astype(np.float64)
            s, z = np.ones(length - first), np.zeros(length - first)
        else:
            u = ((tiles[:, byte].astype(np.int64) >> shift) & (255 if kind == "int8" else 15)).astype(np.float64)
            s = factor(per_part * part)
            z = factor(per_part * part + 1) if kind == "int4" else np.zeros(length - first)
        out.append((u.reshape(-1, D)[first:length], s, z))
    return out


def attend_bound(q, keys, values, scale, kind, o, weights):
    """How far decode attention may be off the exact outputs o [G, D] for the parts that sequence_codes gives; counts what the
    kernel does, code by code:

    A matrix instruction adds 32 products to an accumulator: taken as 33 terms brought to the largest one's exponent and cut to 24
    bits, 33 * 2^-23 of the largest of them and of the sums before and behind.  A subnormal factor (codes enter as u * 2^-24, nibbles
    as u * 2^-20) stands for 2^-14 in this: u as at least 1024, or 64.
    Scores: D / 32 instructions, then the scale, and for codes the middle or the offset times the sum of q (D / 4 + 8 additions);
    the exponent is rounded once or twice, exp2 and the references' changes cost 8 steps.  A score's error moves a weight by
    as much, relative, and an output by that times the distance of the token's value.
    Weights enter as two fp16 numbers: off by 2^-22 relative, or 2^-33 of the largest weight.
    Sums: at least two waves take the tiles in turn, so T / 64 + 1 steps, each as above, over what is summed: the codes, and their
    middle as often; the sums of p and of the offsets in fp32, 8 additions a step, and 16 for the joins.
    Last the output's rounding."""
    (ku, ks, kz), (vu, vs, vz) = keys, values
    T, D = ku.shape
    if T == 0:
        return np.zeros(o.shape)
    one, cut, mid = 2.0 ** -24, 33 * 2.0 ** -23, MIDDLE[kind]
    least = {"f16": 2.0 ** -14, "int8": 1024.0, "int4": 64.0}[kind]
    qd = q.astype(np.float64)
    k = {"f16": ku, "int8": (ku - 128) * ks[:, None], "int4": ku * ks[:, None] + kz[:, None]}[kind]
    v = {"f16": vu, "int8": (vu - 128) * vs[:, None], "int4": vu * vs[:, None] + vz[:, None]}[kind]
    x = qd @ k.T * scale                                              # [G, T]
    qn, kn = np.maximum(np.abs(qd), 2.0 ** -14), np.maximum(np.abs(ku), least)
    run, err = np.zeros(x.shape), np.zeros(x.shape)
    for at in range(0, D, 32):
        before, run = run, run + qd[:, at:at + 32] @ ku[:, at:at + 32].T
        term = (qn[:, None, at:at + 32] * kn[None, :, at:at + 32]).max(-1)
        err += cut * np.maximum(term, np.maximum(np.abs(before), np.abs(run)))
    offset = {"f16": 0.0 * ks, "int8": 128.0 * ks, "int4": np.abs(kz)}[kind]
    err = scale * (ks * err + (D / 4 + 8) * one * np.abs(qd).sum(-1, keepdims=True) * offset
                   + 8 * one * (ks * np.abs(run) + np.abs(qd.sum(-1, keepdims=True)) * offset))
    err = err + one * (np.abs(x) + (x.max(-1, keepdims=True) - x) + 48) + 8 * 2 * one
    assert (weights * err).max() < 0.1, "bound not meant for scores this coarse"
    steps = T // 64 + 2
    summed = weights @ (vs[:, None] * (np.abs(vu) + mid))
    term = weights @ (vs[:, None] * np.maximum(np.abs(vu), least))
    offsets = weights @ (mid * vs + np.abs(vz))
    far = np.stack([(w * e) @ np.abs(v - c) for w, e, c in zip(weights, err, o)])
    width = (vs[:, None] * np.abs(vu - mid)).max()
    return (np.abs(o) * 2.0 ** -11 + 2.0 ** -25 + 1.1 * far + 2.0 ** -22 * (weights @ (vs[:, None] * np.abs(vu - mid))) + T * 2.0 ** -33 * width
            + cut * (steps * summed + term) + (8 * steps + 16) * one * (np.abs(o) + offsets[:, None]))
