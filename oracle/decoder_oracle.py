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
