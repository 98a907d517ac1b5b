"""GPU parity of the decoder operators behind the qkv linear (rotary positions, the paged key-value cache's writer and reader, decode
attention over it) against the numpy oracle: rotation and cache bytes bit for bit, attention against 64 bits with a bound that counts
the kernel's roundings."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
from oracle import decoder_oracle as DO

pytestmark = pytest.mark.gpu

KINDS = ["f16", "int8", "int4"]


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from kairos_amd import ops as _ops
    return _ops


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def i32(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def bits(t):
    return t.cpu().numpy().view(np.uint16)


def table_of(positions, R, base=10000.0):
    from kairos_amd.rotary import rotary_table
    t = rotary_table(positions, R, base, device="cpu")
    return t.numpy(), t.cuda()


def rotated(x, pos, table, inter):
    """What the operator gives, bit for bit: fp32 products and sums rounded one by one, then fp16."""
    with np.errstate(over="ignore", invalid="ignore"):
        return DO.rotate(x, pos, table, inter, np.float32).astype(np.float16)


def qkv_views(rng, B, S, H, KV, D):
    qkv = rng.standard_normal((B, S, H + 2 * KV, D)).astype(np.float16)
    t = dev(qkv)
    return (qkv[:, :, :H], qkv[:, :, H:H + KV], qkv[:, :, H + KV:]), (t[:, :, :H], t[:, :, H:H + KV], t[:, :, H + KV:])


# ---- rotary positions -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("D, R", [(64, 64), (64, 32), (128, 128), (128, 80), (128, 16), (256, 256), (256, 48)])
@pytest.mark.parametrize("B, S, H, KV", [(1, 1, 4, 4), (3, 5, 7, 1), (2, 67, 8, 2)])
def test_rotary_bit_for_bit(ops, B, S, H, KV, D, R, inter):
    rng = np.random.default_rng(B * 1000 + S + D + R)
    (q, k, _), (qd, kd, _) = qkv_views(rng, B, S, H, KV, D)
    table, td = table_of(S + 40, R)
    start = rng.integers(0, 40, B).astype(np.int32)
    pos = start[:, None] + np.arange(S)
    for a, b in ((qd, kd), (qd.contiguous(), kd.contiguous())):
        qo, ko = ops.rotary(a, b, dev(start), td, interleaved=inter)
        assert qo.is_contiguous() and qo.shape == q.shape and ko.shape == k.shape
        assert np.array_equal(bits(qo), rotated(q, pos, table, inter).view(np.uint16))
        assert np.array_equal(bits(ko), rotated(k, pos, table, inter).view(np.uint16))
    # against the formula in 64 bits: half an fp16 step, and an fp32 step for each of three operations on |a| + |b|
    exact = DO.rotate(q, pos, table, inter)
    size = np.abs(q.astype(np.float64)).max() * 2
    assert (np.abs(qo.cpu().numpy().astype(np.float64) - exact) <= np.abs(exact) * 2.0 ** -11 + 2.0 ** -25 + size * 3 * 2.0 ** -24).all()


def test_rotary_keeps_lengths_and_undoes_itself(ops):
    """A table with sines negated turns back: off by the two fp16 roundings of a pair."""
    q = torch.randn((2, 9, 4, 128), dtype=torch.float16, device="cuda")
    _, td = table_of(64, 128)
    there, _ = ops.rotary(q, q, i32(3, 50), td)
    back, _ = ops.rotary(there, there, i32(3, 50), td * torch.tensor([1.0, -1.0], device="cuda"))
    a, b = q.float()[..., :64], q.float()[..., 64:]
    size = torch.sqrt(a * a + b * b).repeat(1, 1, 1, 2)
    # each turn rounds both halves of a pair by half a step (2^-11 of at most the pair's length)
    assert ((back.float() - q.float()).abs() <= size * (2 ** 0.5 * 2.0 ** -11 + 2.0 ** -11 + 1e-6) + 2.0 ** -23).all()


def test_rotary_padding_positions_and_empty_calls(ops):
    q = torch.randn((3, 6, 4, 64), dtype=torch.float16, device="cuda")
    table, td = table_of(10, 32)
    qo, ko = ops.rotary(q, q[:, :, :2], i32(0, 7, -2), td, count=i32(4, 99, 6))
    assert not qo[0, 4:].any() and not ko[0, 4:].any()
    want = rotated(q.cpu().numpy()[0:1, :4], np.arange(4)[None], table, False)
    assert np.array_equal(bits(qo[0:1, :4]), want.view(np.uint16))
    # positions 7, 8, 9 are in the table, 10 .. 12 and -2, -1 are not: NaN in the turned elements, the others copied
    assert torch.isfinite(qo[1, :3]).all() and torch.isnan(qo[1, 3:, :, :32]).all() and torch.isnan(qo[2, :2, :, :32]).all()
    assert torch.equal(qo[1, 3:, :, 32:], q[1, 3:, :, 32:]) and torch.isfinite(qo[2, 2:]).all()
    for shape in ((0, 4, 2, 64), (2, 0, 2, 64)):
        e = torch.zeros(shape, dtype=torch.float16, device="cuda")
        a, b = ops.rotary(e, e, torch.zeros(shape[0], dtype=torch.int32, device="cuda"), td)
        assert a.shape == shape and b.shape == shape
    # count 0 and below: all padding
    a, _ = ops.rotary(q, q, i32(0, 0, 0), td, count=i32(0, -3, 1))
    assert not a[:2].any() and not a[2, 1:].any() and a[2, 0].any()


# ---- the cache's writer and reader ------------------------------------------------------------------------------------------
def make_pages(rng, B, tokens, page, spare=2):
    """int32 [B, width] over distinct pages in random order, and their number."""
    width = -(-max(tokens, 1) // page)
    pool = B * width + spare
    return rng.permutation(pool)[:B * width].reshape(B, width).astype(np.int32), pool


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("S, page, starts", [(1, 32, (0, 31, 70)), (1, 96, (95, 96, 5)), (13, 32, (29, 0, 3)), (75, 64, (0, 21, 40)), (130, 160, (0, 7, 32))])
def test_append_writes_the_oracle_s_bytes_and_read_returns_them(ops, S, page, starts, D, kind):
    B, H, KV = 3, 4, 2
    rng = np.random.default_rng(S + D)
    (q, k, v), (qd, kd, vd) = qkv_views(rng, B, S, H, KV, D)
    k[0, 0, 0] = 0; k[1, 0, 1] = 3.0; v[2, 0, 0] = -65504.0; v[0, 0, 1, ::2] = np.float16(6e-8); k[2, 0, 0, 5] = 65504.0
    kd.copy_(dev(k)); vd.copy_(dev(v))
    R = D // 2
    table, td = table_of(S + 100, R)
    pages, pool = make_pages(rng, B, max(starts) + S, page)
    count = np.array([S, max(1, S - 3), S], np.int32)
    start = np.array(starts, np.int32)
    cache = rng.integers(0, 256, size=(pool, KV, page // 32, DO.tile_bytes(D, kind))).astype(np.uint8)
    want = cache.copy()
    pos = start[:, None] + np.arange(S)
    kr, qr = rotated(k, pos, table, True), rotated(q, pos, table, True)
    for b in range(B):
        for s in range(count[b]):
            p = pos[b, s]
            for h in range(KV):
                DO.put_token(want[pages[b, p // page], h, p % page // 32], p % 32, kr[b, s, h], v[b, s, h], kind)
    cd = dev(cache)
    qo, ko = ops.kv_append(cd, dev(pages), dev(start), kd, vd, td, q=qd, interleaved=True, count=dev(count), want_k=True)
    got = cd.cpu().numpy()
    assert np.array_equal(got, want), np.argwhere(got != want)[:5]         # nothing else in the pool is touched
    for b in range(B):
        n = count[b]
        assert np.array_equal(bits(qo[b, :n]), qr[b, :n].view(np.uint16)) and np.array_equal(bits(ko[b, :n]), kr[b, :n].view(np.uint16))
        assert not qo[b, n:].any() and not ko[b, n:].any()
    rk, rv = ops.kv_read(cd, dev(pages), dev(start), S, count=dev(count))
    for b in range(B):
        n = count[b]
        for x, got in ((kr, rk), (v, rv)):
            ref = x[b, :n] if kind == "f16" else DO.to_f16(DO.values_of(*DO.quantise(x[b, :n], kind), kind, np.float32))
            assert np.array_equal(got[b, :n].cpu().numpy().astype(np.float32), ref.astype(np.float32))
            assert not got[b, n:].any()
    # without queries or a table: keys as they are
    cd = dev(cache)
    assert ops.kv_append(cd, dev(pages), dev(start), kd, vd, count=dev(count)) is None
    rk, _ = ops.kv_read(cd, dev(pages), dev(start), 1)
    ref = k[:, :1] if kind == "f16" else DO.to_f16(DO.values_of(*DO.quantise(k[:, :1], kind), kind, np.float32))
    assert np.array_equal(rk.cpu().numpy().astype(np.float32), ref.astype(np.float32))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("count", [-2 ** 31, -1, 0, 1, 2, 7, 2 ** 31 - 1])
def test_append_of_any_count(ops, count, kind):
    """Counts from the least to the largest int32, starts that leave one or a few tokens in the first group of eight: the tokens that are
    there stand in the cache as if appended one by one, the others come back as zeros and leave the cache as it was."""
    B, S, H, KV, D = 3, 19, 4, 2, 64
    rng = np.random.default_rng(6)
    q, k, v = (dev(rng.standard_normal((B, S, n, D)).astype(np.float16)) for n in (H, KV, KV))
    pages, start = i32(*range(6)).reshape(3, 2), i32(7, 6, 2)
    table = torch.from_numpy(rng.standard_normal((64, D // 2, 2)).astype(np.float32)).cuda()
    both = [torch.full((6, KV, 1, ops.kv_tile_bytes(D, kind)), 9, dtype=torch.uint8, device="cuda") for _ in range(2)]
    got, turned = ops.kv_append(both[0], pages, start, k, v, table, q=q, count=i32(count, count, count), want_k=True)
    there = min(max(count, 0), S)
    for s in range(there):
        one, k1 = ops.kv_append(both[1], pages, start + s, k[:, s:s + 1], v[:, s:s + 1], table, q=q[:, s:s + 1], want_k=True)
        assert torch.equal(got[:, s:s + 1], one) and torch.equal(turned[:, s:s + 1], k1)
    assert torch.equal(both[0], both[1]) and not got[:, there:].any() and not turned[:, there:].any()


@pytest.mark.parametrize("kind", KINDS)
def test_pages_outside_the_cache_are_never_followed(ops, kind):
    """Entries of -1, of the pool's size and of 2^31 - 1, and positions past the row of the page table: writes are dropped, reads give
    NaN, neighbours are untouched."""
    D, KV, page, pool = 64, 2, 32, 4
    pages = i32(2, -1, pool, 2 ** 31 - 1).reshape(1, 4)
    cache = torch.randint(0, 256, (pool, KV, 1, ops.kv_tile_bytes(D, kind)), dtype=torch.uint8, device="cuda")
    before = cache.clone()
    S = 150                                                        # positions 10 .. 159; the row ends at 128
    k = torch.randn((1, S, KV, D), dtype=torch.float16, device="cuda")
    ops.kv_append(cache, pages, i32(10), k, k)
    changed = (cache != before).flatten(1).any(1)
    assert changed.tolist() == [False, False, True, False]
    rk, rv = ops.kv_read(cache, pages, i32(10), S)
    assert torch.isfinite(rk[0, :22]).all() and torch.isnan(rk[0, 22:]).all() and torch.isnan(rv[0, 22:]).all()
    rk, _ = ops.kv_read(cache, pages, i32(-3), 4)
    assert torch.isnan(rk[0, :3]).all()
    before = cache.clone()
    ops.kv_append(cache, pages, i32(-5), k[:, :5], k[:, :5])       # positions -5 .. -1
    assert torch.equal(cache, before)


@pytest.mark.parametrize("kind", ["int8", "int4"])
def test_rows_that_are_not_finite_read_as_nan(ops, kind):
    cache = torch.zeros((1, 1, 1, ops.kv_tile_bytes(64, kind)), dtype=torch.uint8, device="cuda")
    k = torch.randn((1, 4, 1, 64), dtype=torch.float16, device="cuda")
    k[0, 1, 0, 3] = float("inf"); k[0, 2, 0, 60] = float("nan")
    ops.kv_append(cache, i32(0).reshape(1, 1), i32(0), k, k)
    rk, rv = ops.kv_read(cache, i32(0).reshape(1, 1), i32(0), 4)
    for r in (rk, rv):
        assert torch.isnan(r[0, 1:3]).all() and torch.isfinite(r[0, 0]).all() and torch.isfinite(r[0, 3]).all()


# ---- attention --------------------------------------------------------------------------------------------------------------
def attention_bound(q, k, v, scale, kind, o, mean_v, total, weights):
    """How far the kernel may be off: the output's rounding (2^-11), the weights' rounding to fp16 (2^-11 of each, half a subnormal
    step of the smallest), and the scores' error -- D products added in fp32, codes with their offset (at most 1152 + 127, or
    1024 + 15) in front of the subtraction -- which moves a weight by as much, relative.  The sums over tokens are fp32: T * 2^-24
    of the mean size.
    Codes: what is summed are the codes themselves, 0..255 or 0..15, not the values, and the offsets come off the sums: T + 8 additions
    (the join and the subtraction among them), each off by 2^-24 of a sum of at most p times the row's width, 255 s = 2 max|v| for
    int8 and 15 s + |z| + 8 s <= 4 max|v| for int4.  An element that is zero in the row with all the weight shows it: there mean_v is nothing."""
    T, D = k.shape
    if T == 0:
        return np.zeros(o.shape)
    aq = np.abs(q.astype(np.float64)).sum(-1, keepdims=True)
    kmax = np.abs(k).max()
    big = {"f16": kmax, "int8": kmax / 100 * 1300, "int4": kmax * 1200}[kind]
    err = scale * aq * big * (D / 8 + 8) * 2.0 ** -24 + 2.0 ** -20
    width = 0.0 if kind == "f16" else (weights @ np.abs(v).max(-1))[:, None] * {"int8": 2, "int4": 4}[kind]
    return ((np.abs(o) + mean_v) * 2.0 ** -11 + 2 * mean_v * (err + T * 2.0 ** -24) + T * 2.0 ** -25 * np.abs(v).max() / total + 2.0 ** -24
            + (T + 8) * 2.0 ** -24 * width)


def random_cache(rng, pool, KV, tiles, D, kind):
    """A pool with garbage (NaN patterns among it) everywhere; tokens are put in by the caller."""
    return rng.integers(0, 256, size=(pool, KV, tiles, DO.tile_bytes(D, kind))).astype(np.uint8)


def filled(rng, lens, KV, D, kind, page, size=1.0):
    """A cache written token by token by the oracle, its page table (entries behind a sequence's pages: -1), and nothing else in it
    but garbage."""
    need = [-(-n // page) for n in lens]
    width = max(max(need), 1)
    pool = sum(need) + 2
    order = rng.permutation(pool)
    pages = np.full((len(lens), width), -1, np.int32)
    cache = random_cache(rng, pool, KV, page // 32, D, kind)
    at = 0
    for b, n in enumerate(lens):
        pages[b, :need[b]] = order[at:at + need[b]]
        at += need[b]
        k, v = ((rng.standard_normal((n, KV, D)) * size).astype(np.float16) for _ in range(2))
        for t in range(n):
            for h in range(KV):
                DO.put_token(cache[pages[b, t // page], h, t % page // 32], t % 32, k[t, h], v[t, h], kind)
    return cache, pages


def check_attention(ops, cache, pages, lens, q, KV, D, kind, window=0, scale=None, got=None):
    H = q.shape[1]
    G = H // KV
    if got is None:
        got = ops.paged_attention(dev(q), dev(cache), dev(pages), dev(np.array(lens, np.int32)), scale=scale, window=window)
    assert got.shape == q.shape and got.dtype == torch.float16
    got = got.cpu().numpy().astype(np.float64)
    sc = D ** -0.5 if scale is None else scale
    for b, n in enumerate(lens):
        lo = max(0, n - window) if window else 0
        for h in range(KV):
            k, v = DO.sequence(cache, pages[b], n, h, D, kind)
            k, v = k[lo:], v[lo:]
            o, mean_v, total, weights = DO.attend(q[b, h * G:(h + 1) * G], k, v, sc)
            bound = attention_bound(q[b, h * G:(h + 1) * G], k, v, sc, kind, o, mean_v, total, weights)
            off = np.abs(got[b, h * G:(h + 1) * G] - o)
            assert (off <= bound).all(), (b, h, n, float((off / np.maximum(bound, 1e-30)).max()))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D, H, KV", [(64, 4, 4), (64, 20, 1), (128, 7, 1), (128, 8, 2), (128, 33, 1), (256, 16, 1), (256, 4, 2)])
def test_attention_ragged_lengths(ops, D, H, KV, kind):
    """Lengths around the tile (32), a page's end inside it, none at all, one token; query groups of 1, 4, 7, 8, 16, 20, 33."""
    lens = [1, 0, 31, 32, 33, 100, 129]
    rng = np.random.default_rng(D + H)
    cache, pages = filled(rng, lens, KV, D, kind, 64)
    q = (rng.standard_normal((len(lens), H, D)) * 2).astype(np.float16)
    check_attention(ops, cache, pages, lens, q, KV, D, kind)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("window", [1, 5, 32, 64, 77, 1000])
def test_attention_window(ops, window, kind):
    lens = [200, 64, 3, 0]
    rng = np.random.default_rng(window)
    cache, pages = filled(rng, lens, 2, 64, kind, 96)
    q = (rng.standard_normal((4, 8, 64)) * 2).astype(np.float16)
    check_attention(ops, cache, pages, lens, q, 2, 64, kind, window=window, scale=0.2)


@pytest.mark.parametrize("kind", KINDS)
def test_attention_split_over_a_long_sequence(ops, kind):
    """One long sequence next to short ones: its tokens are shared out over workgroups and joined."""
    lens = [2500, 1, 40]
    rng = np.random.default_rng(9)
    cache, pages = filled(rng, lens, 1, 64, kind, 32)
    q = (rng.standard_normal((3, 4, 64)) * 2).astype(np.float16)
    check_attention(ops, cache, pages, lens, q, 1, 64, kind)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("size, qsize", [(1e-3, 1.0), (300.0, 0.05), (1.0, 30.0)])
def test_attention_sizes_of_values_and_scores(ops, size, qsize, kind):
    """Values far from 1 (their scales subnormal in fp16 or large), and scores so wide that one token takes all the weight."""
    lens = [90, 33]
    rng = np.random.default_rng(4)
    cache, pages = filled(rng, lens, 2, 64, kind, 32, size)
    q = (rng.standard_normal((2, 4, 64)) * qsize).astype(np.float16)
    check_attention(ops, cache, pages, lens, q, 2, 64, kind)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("H", [4, 12])
def test_attention_small_values_beside_large_ones_without_weight(ops, H, kind):
    """All weight on a token whose value is 1e-4, tokens with 60000 and a weight of e^-128 in its tile and the next: the small value's
    weight keeps its 11 bits.  Off by its rounding and the output's, 2^-11 each of the row's largest, and half a subnormal step; the
    codes' sums add 48 * 2^-24 of four times that."""
    n, D = 40, 64
    rng = np.random.default_rng(5)
    cache, pages = random_cache(rng, 3, 1, 1, D, kind), np.array([[2, 0]], np.int32)
    for t in range(n):
        k = np.full(D, 4.0 if t == 5 else -4.0, np.float16)
        v = (rng.standard_normal(D) * (1e-4 if t == 5 else 20000.0)).clip(-60000, 60000).astype(np.float16)
        DO.put_token(cache[pages[0, t // 32], 0, 0], t % 32, k, v, kind)
    q = np.full((1, H, D), 2.0, np.float16)
    got = ops.paged_attention(dev(q), dev(cache), dev(pages), i32(n)).cpu().numpy().astype(np.float64)[0]
    held = DO.sequence(cache, pages[0], n, 0, D, kind)[1][5].astype(np.float64)
    assert np.abs(got - held).max() <= np.abs(held).max() * (2 * 2.0 ** -11 + 4 * 48 * 2.0 ** -24) + 2.0 ** -25


def test_attention_strided_queries_and_4d(ops):
    rng = np.random.default_rng(2)
    lens = [70, 45]
    cache, pages = filled(rng, lens, 2, 64, "int8", 32)
    qkv = (rng.standard_normal((2, 1, 8, 64)) * 2).astype(np.float16)
    qd = dev(qkv)[:, :, :4]
    got = ops.paged_attention(qd, dev(cache), dev(pages), i32(*lens))
    assert got.shape == (2, 1, 4, 64) and got.is_contiguous()
    check_attention(ops, cache, pages, lens, qkv[:, 0, :4], 2, 64, "int8", got=got[:, 0])


@pytest.mark.parametrize("kind", KINDS)
def test_attention_errors_of_device_data_stay_in_their_sequence(ops, kind):
    """A page that is not one of the cache and a length past the row of the page table give NaN for that sequence only."""
    rng = np.random.default_rng(5)
    lens = [70, 70, 70, 70]
    cache, pages = filled(rng, lens, 2, 64, kind, 32)
    q = rng.standard_normal((4, 4, 64)).astype(np.float16)
    pages[1, 1] = len(cache); pages[2, 0] = -7
    given = np.array([70, 70, 70, 97], np.int32)                    # the row holds 96
    got = ops.paged_attention(dev(q), dev(cache), dev(pages), dev(given))
    assert torch.isnan(got[1:]).all() and torch.isfinite(got[0]).all()
    check_attention(ops, cache, pages[:1], lens[:1], q[:1], 2, 64, kind, got=got[:1])
    neg = ops.paged_attention(dev(q), dev(cache), dev(pages), i32(-1, 0, -2 ** 31, 0))
    assert not neg.any()
    e = ops.paged_attention(torch.zeros((0, 4, 64), dtype=torch.float16, device="cuda"), dev(cache), dev(pages[:0]), dev(given[:0]))
    assert e.shape == (0, 4, 64)


@pytest.mark.parametrize("kind", KINDS)
def test_cache_beyond_32_bit_offsets(ops, kind):
    """Pages whose bytes lie past 4 GiB, written, read and attended to as those at the start."""
    D, KV, page = 256, 8, 256
    per = KV * (page // 32) * ops.kv_tile_bytes(D, kind)
    pool = (5 << 30) // per
    cache = torch.empty((pool, KV, page // 32, ops.kv_tile_bytes(D, kind)), dtype=torch.uint8, device="cuda")
    S = 300
    k, v = (torch.randn((1, S, KV, D), dtype=torch.float16, device="cuda") for _ in range(2))
    q = torch.randn((1, 16, D), dtype=torch.float16, device="cuda")
    near, far = i32(0, 1).reshape(1, 2), i32(pool - 1, pool - 2).reshape(1, 2)
    outs = []
    for pages in (near, far):
        ops.kv_append(cache, pages, i32(0), k, v)
        outs.append(ops.kv_read(cache, pages, i32(0), S) + (ops.paged_attention(q, cache, pages, i32(S)),))
    for a, b in zip(*outs):
        assert torch.isfinite(a).all() and torch.equal(a, b)
    del cache


def appended(ops, rng, lens, KV, D, kind, page, width=None, size=1.0):
    """A cache filled by kv_append (whose bytes the oracle has checked), its page table (-1 behind a sequence's pages) as numpy."""
    need = [-(-n // page) for n in lens]
    pool = sum(need) + 2
    order, at = rng.permutation(pool), 0
    pages = np.full((len(lens), width or max(max(need), 1)), -1, np.int32)
    for b, n in enumerate(need):
        pages[b, :n] = order[at:at + n]
        at += n
    cache = torch.full((pool, KV, page // 32, ops.kv_tile_bytes(D, kind)), 255, dtype=torch.uint8, device="cuda")      # NaN patterns
    S = max(max(lens), 1)
    k, v = (dev((rng.standard_normal((len(lens), S, KV, D)) * size).astype(np.float16)) for _ in range(2))
    ops.kv_append(cache, dev(pages), torch.zeros(len(lens), dtype=torch.int32, device="cuda"), k, v, count=i32(*lens))
    return cache, pages


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("B, KV, lens", [
    (130, 4, lambda i: (i * 37) % 41),                            # more tasks than shares, sequences of no tokens among them
    (70, 8, lambda i: 1 + (i * 53) % 200),
    (3, 2, lambda i: (5000, 1, 1700)[i]),                         # pieces of equal length
    (40, 8, lambda i: 9000 if i == 7 else 1 + (i * 11) % 60),    # one long sequence among short ones: a row cut anywhere
    (257, 1, lambda i: i),                                         # more than 64 lengths, tasks of every length up to 256
])
def test_attention_work_shared_out(ops, B, KV, lens, kind):
    """Every way the tiles are shared out over workgroups: whole tasks, equal pieces, a row of tasks cut anywhere."""
    D, H = 64, 4 * KV
    lens = [lens(i) for i in range(B)]
    rng = np.random.default_rng(B)
    cache, pages = appended(ops, rng, lens, KV, D, kind, 32)
    q = (rng.standard_normal((B, H, D)) * 2).astype(np.float16)
    got = ops.paged_attention(dev(q), cache, dev(pages), i32(*lens))
    again = ops.paged_attention(dev(q), cache, dev(pages), i32(*lens))
    assert torch.equal(got.view(torch.int16), again.view(torch.int16))          # whichever workgroup joins
    ws = ops.gemv_workspace_for("cuda")
    assert not ws[:65536].any()                                                 # arrival counters left zero
    some = sorted(set([0, B - 1, int(np.argmax(lens))] + list(rng.choice(B, min(B, 24), replace=False))))
    check_attention(ops, cache.cpu().numpy(), pages[some], [lens[i] for i in some], q[some], KV, D, kind, got=got[some])
    none = [i for i, n in enumerate(lens) if n == 0]
    assert not got[none].any()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D, G, B, KV", [(128, 4, 40, 8), (128, 12, 40, 8), (64, 12, 40, 8), (64, 4, 135, 8), (128, 4, 260, 8), (64, 3, 260, 8), (128, 12, 130, 16),
                                         (64, 12, 130, 16), (256, 2, 130, 16), (64, 1, 1100, 2)])
def test_attention_of_many_tasks(ops, D, G, B, KV, kind):
    """From a task more than CUs up to many thousands, short ones, none, and one so long that it is cut among them; over 1024 lengths."""
    lens = [0 if i % 9 == 4 else 700 if i == 17 else 1 + (i * 23) % 45 for i in range(B)]
    rng = np.random.default_rng(B + G)
    cache, pages = appended(ops, rng, lens, KV, D, kind, 32)
    q = (rng.standard_normal((B, G * KV, D)) * 2).astype(np.float16)
    got = ops.paged_attention(dev(q), cache, dev(pages), i32(*lens))
    again = ops.paged_attention(dev(q), cache, dev(pages), i32(*lens))
    assert torch.equal(got.view(torch.int16), again.view(torch.int16))
    host = cache.cpu().numpy()
    some = [4, 17, B // 2, B - 1]
    check_attention(ops, host, pages[some], [lens[b] for b in some], q[some], KV, D, kind, got=got[some])
    # the others against the same sequences shared out differently: twice (|o| + mean |v|) 2^-11 with |v| < 6, 2^-6.4, and as much for scores and codes
    for at in range(0, B, 64):
        part = ops.paged_attention(dev(q[at:at + 64]), cache, dev(pages[at:at + 64]), i32(*lens[at:at + 64]))
        assert (part.float() - got[at:at + 64].float()).abs().max() <= 2.0 ** -5


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D, G, B, KV, width", [(128, 16, 1, 1, 1), (128, 16, 130, 16, 2), (64, 16, 130, 16, 2), (64, 8, 130, 16, 2), (128, 8, 40, 8, 2), (256, 16, 2, 2, 1), (128, 32, 16, 2, 400)])
def test_the_stated_workspace_suffices(ops, D, G, B, KV, width, kind):
    """64 KiB of counters and 17 MiB, as the header says, for whatever share of the work the shape asks for; counters left zero."""
    from kairos_amd import _lib
    cache = torch.zeros((4, KV, 1, ops.kv_tile_bytes(D, kind)), dtype=torch.uint8, device="cuda")
    pages, lens = torch.ones((B, width), dtype=torch.int32, device="cuda"), torch.full((B,), 32 * width, dtype=torch.int32, device="cuda")
    q = torch.ones((B, G * KV, D), dtype=torch.float16, device="cuda")
    out = torch.full_like(q, 7.0)
    ws = torch.zeros(65536 + (17 << 20), dtype=torch.uint8, device="cuda")
    args = ops._paged_attn_args.pack(out.data_ptr(), q.data_ptr(), cache.data_ptr(), pages.data_ptr(), lens.data_ptr(), ws.data_ptr(), ws.numel(),
                                     G * KV * D, 0.1, B, G * KV, KV, D, ops.KV_KINDS[kind], 4, 1, width, 0)
    assert _lib.load().kmi_paged_attn(args, torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert not out.any() and not ws[:65536].any()              # a cache of zeros: int8 stands for 0 * (0 - 128)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D, G", [(64, 17), (64, 32), (64, 33), (128, 20), (128, 64), (256, 20)])
def test_attention_many_heads_on_a_wide_page_table(ops, D, G, kind):
    """Page tables with room for far longer sequences: 32 query heads at once where more than 16 share a key head, one sequence cut."""
    lens = [2200, 70, 0]
    rng = np.random.default_rng(G)
    cache, pages = appended(ops, rng, lens, 1, D, kind, 32, width=5000)
    q = (rng.standard_normal((3, G, D)) * 2).astype(np.float16)
    got = ops.paged_attention(dev(q), cache, dev(pages), i32(*lens))
    check_attention(ops, cache.cpu().numpy(), pages, lens, q, 1, D, kind, got=got)


@pytest.mark.parametrize("kind", KINDS)
def test_attention_flat_and_peaked_over_many_tokens(ops, kind):
    """20000 equal scores (every token counts alike: sums of many small weights) and one token far above the others."""
    D, n = 128, 20000
    rng = np.random.default_rng(8)
    cache, pages = appended(ops, rng, [n, n], 1, D, kind, 64)
    q = np.zeros((2, 8, D), np.float16)
    k, _ = DO.sequence(cache.cpu().numpy(), pages[1], n, 0, D, kind)
    q[1] = (k[12345] * 3).astype(np.float16)
    got = ops.paged_attention(dev(q), cache, dev(pages), i32(n, n))
    check_attention(ops, cache.cpu().numpy(), pages, [n, n], q, 1, D, kind, got=got)


def test_attention_values_that_are_infinite_where_no_token_counts(ops):
    """f16: infinities and NaN in keys and values in front of the window and behind the end."""
    rng = np.random.default_rng(3)
    D, n, w = 64, 75, 20
    cache, pages = filled(rng, [n], 1, D, "f16", 32)
    for t in (0, 31, 40, n - w - 1):
        bad = np.full(D, np.inf if t % 2 else np.nan, np.float16)
        DO.put_token(cache[pages[0, t // 32], 0, 0], t % 32, bad, bad, "f16")
    q = rng.standard_normal((1, 4, D)).astype(np.float16)
    check_attention(ops, cache, pages, [n], q, 1, D, "f16", window=w)


@pytest.mark.parametrize("kind", KINDS)
def test_two_graphs_of_cut_sequences_on_one_scratch(ops, kind):
    """Captured calls whose sequences are cut into shares, two graphs in turn on the scratch that they share, eager calls in between."""
    rng = np.random.default_rng(6)
    D, H, KV = 128, 8, 2
    lens = i32(4000, 2600)
    cache, pages = appended(ops, rng, [4000, 2600], KV, D, kind, 64)
    pd = dev(pages)
    qs = [torch.randn((2, H, D), dtype=torch.float16, device="cuda") for _ in range(2)]
    scratch, side = ops.Scratch(), torch.cuda.Stream()
    graphs = []
    side.wait_stream(torch.cuda.current_stream())
    for q in qs:
        with torch.cuda.stream(side), scratch:
            ops.paged_attention(q, cache, pd, lens)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with scratch, torch.cuda.graph(g, stream=side):
            out = ops.paged_attention(q, cache, pd, lens)
        graphs.append((g, out))
    for i in range(4):
        for q in qs:
            q.copy_(torch.randn(q.shape, dtype=torch.float16, device="cuda"))
        for g, _ in graphs:
            g.replay()
        want = [ops.paged_attention(q, cache, pd, lens) for q in qs]
        torch.cuda.synchronize()
        for (_, out), w in zip(graphs, want):
            assert torch.equal(out.view(torch.int16), w.view(torch.int16)), i
        lens.sub_(i32(100, 700))
    assert not scratch.gemv[:65536].any()


def test_capture_without_a_scratch_is_refused(ops):
    """As every call of the library that needs one: creating a scratch inside a capture would record a fill into the graph."""
    s = torch.cuda.Stream()
    cache = torch.zeros((2, 2, 1, ops.kv_tile_bytes(64, "int8")), dtype=torch.uint8, device="cuda")
    q = torch.zeros((1, 4, 64), dtype=torch.float16, device="cuda")
    pages, lens = i32(0).reshape(1, 1), i32(5)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    ops.release_workspace("cuda", s.cuda_stream)
    with pytest.raises(RuntimeError, match="scratch"):
        with torch.cuda.graph(g, stream=s):
            ops.paged_attention(q, cache, pages, lens)


# ---- together, streams, graphs -----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", KINDS)
def test_a_generation_step_by_step(ops, kind):
    """Prefill of unequal prompts (padded batch), then tokens one by one: rotate, append and attend as a decoder layer does, against the
    attention of the oracle over everything the cache holds so far."""
    from kairos.kv_cache import PagedKVCache
    from kairos.rotary import rotary_table
    B, H, KV, D, page = 2, 8, 2, 64, 32
    rng = np.random.default_rng(1)
    count = np.array([37, 20], np.int32)
    S = int(count.max())
    table = rotary_table(128, D, 500000.0, {"rope_type": "yarn", "factor": 2.0, "original_max_position_embeddings": 64})
    c = PagedKVCache(8, KV, D, kind, page)
    pages, _ = make_pages(rng, B, 96, page)
    _, (q, k, v) = qkv_views(rng, B, S, H, KV, D)
    c.append(dev(pages), i32(0, 0), k, v, table, q=q, count=dev(count))
    lens = count.copy()
    for step in range(4):
        _, (q, k, v) = qkv_views(rng, B, 1, H, KV, D)
        qo = c.append(dev(pages), dev(lens), k, v, table, q=q)
        want_q = rotated(q.cpu().numpy(), lens[:, None], table.cpu().numpy(), False)
        assert np.array_equal(bits(qo), want_q.view(np.uint16))
        lens = lens + 1
        out = c.attend(qo, dev(pages), dev(lens))
        check_attention(ops, c.data.cpu().numpy(), pages, list(lens), want_q[:, 0], KV, D, kind, got=out[:, 0])
        rk, _ = c.read(dev(pages), dev(lens - 1), 1)
        key = rotated(k.cpu().numpy(), (lens - 1)[:, None], table.cpu().numpy(), False)
        ref = key if kind == "f16" else DO.to_f16(DO.values_of(*DO.quantise(key, kind), kind, np.float32))
        assert np.array_equal(rk.cpu().numpy().astype(np.float32), ref.astype(np.float32))


@pytest.mark.parametrize("kind", KINDS)
def test_captured_step_replays_as_eager(ops, kind):
    """One decode step (append + attend, position on the device) captured once and replayed with the program's own eager work in
    between; every replay equals the eager step bit for bit, also where two graphs replay in turn on one stream."""
    from kairos.rotary import rotary_table
    B, H, KV, D, page = 3, 8, 2, 128, 64
    table = rotary_table(2048, D)
    pages = torch.randperm(B * 20, device="cuda")[:B * 20].to(torch.int32).reshape(B, 20).contiguous()
    shape = (B * 20, KV, page // 32, ops.kv_tile_bytes(D, kind))
    seed = torch.randn((B, 1000, KV, D), dtype=torch.float16, device="cuda")
    caches = [torch.zeros(shape, dtype=torch.uint8, device="cuda") for _ in range(3)]
    for c in caches:
        ops.kv_append(c, pages, i32(0, 0, 0), seed, seed)
    qkv = torch.randn((B, 1, H + 2 * KV, D), dtype=torch.float16, device="cuda")
    pos = i32(1000, 40, 0)

    def step(cache):
        q = ops.kv_append(cache, pages, pos, qkv[:, :, H:H + KV], qkv[:, :, H + KV:], table, q=qkv[:, :, :H])
        return ops.paged_attention(q, cache, pages, pos + 1)

    side = torch.cuda.Stream()
    scratch = ops.Scratch()
    graphs, outs = [], []
    side.wait_stream(torch.cuda.current_stream())
    for c in caches[:2]:
        with torch.cuda.stream(side), scratch:
            step(c)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with scratch, torch.cuda.graph(g, stream=side):
            outs.append(step(c))
        graphs.append(g)
    for i in range(4):
        qkv.copy_(torch.randn(qkv.shape, dtype=torch.float16, device="cuda"))
        for g in graphs:
            g.replay()
        want = step(caches[2])
        torch.cuda.synchronize()
        for o, c in zip(outs, caches):
            assert torch.equal(o.view(torch.int16), want.view(torch.int16)), i
            assert torch.equal(c, caches[2])
        pos.add_(1)


def test_streams_of_their_own(ops):
    """Calls on two streams at once, each ordered behind its inputs: the results of one stream alone."""
    D, KV, H, page = 128, 4, 16, 64
    cache = torch.randn((80, KV, page // 32, ops.kv_tile_bytes(D, "f16") // 2), device="cuda").half().view(torch.uint8)
    pages = torch.arange(80, dtype=torch.int32, device="cuda").reshape(2, 40)
    qs = [torch.randn((2, H, D), dtype=torch.float16, device="cuda") for _ in range(8)]
    lens = i32(2500, 77)
    want = [ops.paged_attention(q, cache, pages, lens) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None] * len(qs)
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for i, q in enumerate(qs):
        with torch.cuda.stream(streams[i % 2]):
            got[i] = ops.paged_attention(q, cache, pages, lens)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))


@pytest.mark.parametrize("kind", KINDS)
def test_decoder_command_s_stack(ops, kind):
    """The decoder command's layer (fused qkv, matched norms, switched linears) on the paged cache against the same layer on its static
    fp16 cache and PyTorch attention, given the keys and values that a cache of this kind holds: prefill and decode logits, and graph
    replays against eager steps token for token.  Both layers' keys and values are the same bits (same linears, same inputs), so
    what differs are the roundings of attention and behind it: fp16 weights, attention output, three linears' outputs and the
    activations between them, under 40 times 2^-11 of the largest logit."""
    from kairos.dynamic_linear import DynamicLinear
    from kairos.perf_profiler import Profiler
    from kairos_amd.bench_extra import Decoder
    from oracle import kairos_oracle as O
    dev_ = torch.device("cuda:0")
    hidden, heads, kv, mlp, vocab = 1024, 8, 2, 2048, 2048
    d = hidden // heads
    shapes = [((heads + 2 * kv) * d, hidden), (hidden, hidden), (2 * mlp, hidden), (hidden, mlp)]
    prof = Profiler(shapes)
    for sh in shapes:
        for r, name in [(16, "w4a16_gemv"), (1 << 20, "w4a16_gemm")]:
            prof.record_best_comp(sh, r, name)
    old, DynamicLinear.prof = DynamicLinear.prof, prof
    try:
        lins = []
        for layer in range(1):
            ql = []
            for i, (N, K) in enumerate(shapes):
                lin = torch.nn.Linear(K, N, bias=False, dtype=torch.float16)
                with torch.no_grad():
                    lin.weight.copy_(torch.from_numpy(O.synth_weights(N, K, seed=300 + 10 * layer + i) * np.float16(2.0)))
                ql.append(DynamicLinear.from_module(lin.cuda(), "cuda"))
            lins.append(ql)
        B, prompt, t_max = 3, 45, 160
        paged = Decoder(lins, dev_, hidden, heads, kv, vocab, t_max=t_max, seed=1, kv_cache=kind)
        glue = Decoder(lins, dev_, hidden, heads, kv, vocab, t_max=t_max, seed=1)
        ids = torch.randint(0, vocab, (B, prompt), device=dev_, generator=torch.Generator(device=dev_).manual_seed(2))
        tol = 40 * 2.0 ** -11
        table = table_of(t_max, d, 500000.0)[0]

        def held_qkv(layer):
            def qkv_of(x, delta, cs):
                x, qkv = layer._heads(x, delta)
                pos = np.arange(qkv.shape[1])[None] if qkv.shape[1] > 1 else glue.pos.cpu().numpy()[None]
                pos = np.broadcast_to(pos, qkv.shape[:2])
                q, k, v = (t.cpu().numpy() for t in qkv.split((heads, kv, kv), dim=2))
                q, k = rotated(q, pos, table, False), rotated(k, pos, table, False)
                if kind != "f16":
                    k, v = (DO.to_f16(DO.values_of(*DO.quantise(t, kind), kind, np.float32)) for t in (k, v))
                return (x,) + tuple(dev(t).transpose(1, 2) for t in (q, k, v))
            return qkv_of


        def rel(a, b):
            return ((a.float() - b.float()).abs().max() / b.float().abs().max()).item()

        for layer in glue.layers:
            layer._qkv = held_qkv(layer)
        for dec in (paged, glue):
            dec.alloc(B)
        got, want = paged.prefill_logits(ids), glue.prefill_logits(ids)
        assert torch.isfinite(got).all() and rel(got, want) < tol, rel(got, want)
        first = want.argmax(-1)
        eager = []
        for dec in (paged, glue):
            dec.start(first, prompt)
        for t in range(4):
            paged.step()
            glue.step()
            assert rel(paged.logits, glue.logits) < tol, (t, rel(paged.logits, glue.logits))
            eager.append((paged.tok.clone(), paged.logits.clone()))
            nxt = glue.tok                                          # both continue with the glue's token
            paged.x_in.copy_(paged.emb[nxt])
        paged.prefill(ids)
        graph = paged.capture()
        paged.start(first, prompt)
        paged.prefill(ids)                                          # eager work between capture and replay
        glue.start(first, prompt)
        for t in range(4):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(paged.tok, eager[t][0]) and torch.equal(paged.logits, eager[t][1]), t
            glue.step()
            paged.x_in.copy_(paged.emb[glue.tok])
        paged.free()
        assert all(L.cache is None for L in paged.layers)
    finally:
        DynamicLinear.prof = old


# ---- refusals -------------------------------------------------------------------------------------------------------------------
def test_refusals(ops):
    q = torch.zeros((2, 3, 4, 64), dtype=torch.float16, device="cuda")
    k = torch.zeros((2, 3, 2, 64), dtype=torch.float16, device="cuda")
    start, pages = i32(0, 0), i32(0, 1).reshape(2, 1)
    table = torch.zeros((8, 32, 2), device="cuda")
    cache = torch.zeros((2, 2, 1, ops.kv_tile_bytes(64, "int8")), dtype=torch.uint8, device="cuda")
    cases = [
        (lambda: ops.rotary(q.float(), k, start, table), TypeError), (lambda: ops.rotary(q, k, start.long(), table), TypeError),
        (lambda: ops.rotary(q, k, start[:1], table), ValueError), (lambda: ops.rotary(q[:1], k, start, table), ValueError),
        (lambda: ops.rotary(q, k, start, table.half()), TypeError), (lambda: ops.rotary(q, k, start, table[..., :1]), ValueError),
        (lambda: ops.rotary(q, k, start, table[:, :30].contiguous()), Exception), (lambda: ops.rotary(q.transpose(2, 3), k, start, table), ValueError),
        (lambda: ops.rotary(q[..., 4:36], k[..., 4:36], start, table), ValueError), (lambda: ops.rotary(q, k, start, table, count=i32(1)), ValueError),
        (lambda: ops.rotary(q[..., :32].contiguous(), k[..., :32].contiguous(), start, table), Exception),
        (lambda: ops.kv_append(cache, pages, start, k[:, :, :1], k[:, :, :1]), ValueError), (lambda: ops.kv_append(cache, pages[:1], start, k, k), ValueError),
        (lambda: ops.kv_append(cache, pages.long(), start, k, k), TypeError), (lambda: ops.kv_append(cache[..., :100].contiguous(), pages, start, k, k), ValueError),
        (lambda: ops.kv_append(cache, pages, start, k, k[:, :2]), ValueError), (lambda: ops.kv_append(cache.to(torch.int8), pages, start, k, k), TypeError),
        (lambda: ops.kv_append(cache.transpose(0, 1), pages, start, k, k), ValueError), (lambda: ops.kv_append(cache, pages, start, k.cpu(), k), ValueError),
        (lambda: ops.kv_read(cache, pages, start, -1), ValueError), (lambda: ops.kv_read(cache, pages, start[:1], 3), ValueError),
        (lambda: ops.kv_read(cache, pages, start, 3, count=start.float()), TypeError),
        (lambda: ops.rotary(q, k[:, :, :0], start, table), ValueError),          # nothing would turn q
        (lambda: ops.paged_attention(q[:, :2], cache, pages, start), ValueError), (lambda: ops.paged_attention(q[:, 0, :3], cache, pages, start), ValueError),
        (lambda: ops.paged_attention(q[:, 0], cache, pages, start, scale=0.0), Exception), (lambda: ops.paged_attention(q[:, 0], cache, pages, start, window=-1), Exception),
        (lambda: ops.paged_attention(q[:, 0], cache, pages, i32(1)), ValueError), (lambda: ops.paged_attention(q[:, 0].cpu(), cache, pages, start), ValueError),
    ]
    for i, (call, err) in enumerate(cases):
        with pytest.raises(err):
            call()
            print("accepted", i)
