"""How exact the decode attention over the paged cache is, against 64 bits: what it may add to the rounding of its outputs."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
from oracle import decoder_oracle as DO
from test_gpu_decoder_operators import KINDS, appended, dev, i32, ops  # noqa: F401

pytestmark = pytest.mark.gpu


def in_64_bits(cache, pages, lens, q, KV, D, kind, scale):
    """fp64 [B, H, D] from the bytes of the cache."""
    G = q.shape[1] // KV
    out = np.zeros(q.shape)
    for b, n in enumerate(lens):
        for h in range(KV):
            k, v = DO.sequence(cache, pages[b], n, h, D, kind)
            out[b, h * G:(h + 1) * G] = DO.attend(q[b, h * G:(h + 1) * G], k, v, scale)[0]
    return out


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D, KV, G", [(64, 4, 4), (128, 2, 4), (128, 1, 12), (128, 1, 20), (256, 2, 8)])
def test_nothing_but_the_output_is_rounded_to_11_bits(ops, D, KV, G, kind):  # noqa: F811
    """The error's root mean square against that of the outputs' own rounding, which is evenly spread over a step: step / sqrt(12).
    The sums in fp32 (scores 2^-18, 25 steps of accumulation 2^-17 relative) add under 2^-16 of the outputs, which is 2^-4 of the
    rounding and 0.2 % in squares.  Weights of 11 bits would add random errors of their own, the root mean square of
    2^-11 / sqrt(3) of a weight, over independent values 0.6 to 0.8 of the rounding, 17 % and more in all.  10 % parts the two."""
    lens = [1536, 1500, 777, 1536]
    rng = np.random.default_rng(D + G)
    cache, pages = appended(ops, rng, lens, KV, D, kind, 64)
    q = (rng.standard_normal((4, KV * G, D)) * 2).astype(np.float16)
    got = ops.paged_attention(dev(q), cache, dev(pages), i32(*lens)).cpu().numpy()
    want = in_64_bits(cache.cpu().numpy(), pages, lens, q, KV, D, kind, D ** -0.5)
    step = np.spacing(np.abs(want).astype(np.float16)).astype(np.float64)
    off, rounding = np.sqrt(((got - want) ** 2).mean()), np.sqrt((step ** 2).mean() / 12)
    assert off <= 1.1 * rounding, (off, rounding)


def check_close(cache, pages, lens, q, KV, D, kind, got, scale=None, window=0):
    """Every output within what DO.attend_bound counts."""
    G, sc = q.shape[1] // KV, D ** -0.5 if scale is None else scale
    got = got.cpu().numpy().astype(np.float64)
    for b, n in enumerate(lens):
        lo = max(0, n - window) if window else 0
        for h in range(KV):
            if n == 0:
                assert not got[b].any()
                continue
            k, v = DO.sequence(cache, pages[b], n, h, D, kind)
            at = slice(h * G, (h + 1) * G)
            o, _, _, w = DO.attend(q[b, at], k[lo:], v[lo:], sc)
            bound = DO.attend_bound(q[b, at], *DO.sequence_codes(cache, pages[b], lo, n, h, D, kind), sc, kind, o, w)
            off = np.abs(got[b, at] - o)
            assert (off <= bound).all(), (b, h, n, float((off / bound).max()))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D, G", [(64, 4), (128, 12), (256, 8)])
@pytest.mark.parametrize("size, ksize", [(1e-3, 1.0), (3e-4, 12000.0), (2e-4, 1.0), (5e-5, 1.0), (1e-5, 1.0)])
def test_small_queries_under_a_large_scale(ops, size, ksize, D, G, kind):  # noqa: F811
    """Queries down to fp16's subnormal numbers, the scale (or the keys) as much larger: scores of a normal spread."""
    lens = [300, 64]
    rng = np.random.default_rng(D)
    cache, pages = appended(ops, rng, lens, 1, D, kind, 32, size=ksize)
    q = (rng.standard_normal((2, G, D)) * size).astype(np.float16)
    scale = float(np.float32(2.0 / (size * ksize * D ** 0.5)))
    got = ops.paged_attention(dev(q), cache, dev(pages), i32(*lens), scale=scale)
    check_close(cache.cpu().numpy(), pages, lens, q, 1, D, kind, got, scale)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D, H, KV", [(64, 4, 4), (64, 20, 1), (128, 7, 1), (128, 8, 2), (128, 33, 1), (256, 16, 1), (256, 4, 2)])
def test_ragged_lengths(ops, D, H, KV, kind):  # noqa: F811
    """One token, none, a tile's edges, several tiles; query groups of 1, 4, 7, 16, 20 and 33."""
    lens = [1, 0, 31, 32, 33, 100, 129]
    rng = np.random.default_rng(D + H)
    cache, pages = appended(ops, rng, lens, KV, D, kind, 64)
    q = (rng.standard_normal((len(lens), H, D)) * 2).astype(np.float16)
    got = ops.paged_attention(dev(q), cache, dev(pages), i32(*lens))
    check_close(cache.cpu().numpy(), pages, lens, q, KV, D, kind, got)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("window", [1, 5, 77])
def test_windows(ops, window, kind):  # noqa: F811
    lens = [200, 64, 3, 0]
    rng = np.random.default_rng(window)
    cache, pages = appended(ops, rng, lens, 2, 64, kind, 96)
    q = (rng.standard_normal((4, 8, 64)) * 2).astype(np.float16)
    got = ops.paged_attention(dev(q), cache, dev(pages), i32(*lens), scale=0.2, window=window)
    check_close(cache.cpu().numpy(), pages, lens, q, 2, 64, kind, got, 0.2, window)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D, G, width", [(64, 4, None), (128, 8, None), (128, 20, 5000), (256, 4, None)])
def test_sequences_cut_into_shares(ops, D, G, width, kind):  # noqa: F811
    """Long ones cut and joined next to short ones; with a wide page table 32 query heads of a key head at once."""
    lens = [2500, 1, 40, 1801]
    rng = np.random.default_rng(D + G)
    cache, pages = appended(ops, rng, lens, 1, D, kind, 32, width=width)
    q = (rng.standard_normal((4, G, D)) * 2).astype(np.float16)
    got = ops.paged_attention(dev(q), cache, dev(pages), i32(*lens))
    check_close(cache.cpu().numpy(), pages, lens, q, 1, D, kind, got)


@pytest.mark.parametrize("kind", KINDS)
def test_many_tasks(ops, kind):  # noqa: F811
    """Two-wave workgroups: thousands of short tasks, one long one cut among them."""
    D, G, B, KV = 64, 4, 260, 8
    lens = [0 if i % 9 == 4 else 700 if i == 17 else 1 + (i * 23) % 45 for i in range(B)]
    rng = np.random.default_rng(B)
    cache, pages = appended(ops, rng, lens, KV, D, kind, 32)
    q = (rng.standard_normal((B, G * KV, D)) * 2).astype(np.float16)
    got = ops.paged_attention(dev(q), cache, dev(pages), i32(*lens))
    some = [0, 4, 17, 100, B - 1]
    check_close(cache.cpu().numpy(), pages[some], [lens[b] for b in some], q[some], KV, D, kind, got[some])


@pytest.mark.parametrize("D, G, width, size", [(64, 1, None, 2.0), (64, 4, None, 30.0), (128, 20, 5000, 2.0), (128, 4, None, 6.0), (256, 4, None, 2.0)])
def test_infinite_values_come_through(ops, D, G, width, size):  # noqa: F811
    """f16: an infinity that counts gives that infinity however small its weight -- in another wave's or share's tiles than a score e^300 times
    as large, a lone token's whose weight is a power of two -- both signs or a NaN give NaN; the elements beside it stay as exact as ever."""
    lens = [1, 40, 300, 2500]
    rng = np.random.default_rng(D + G)
    cache, pages = appended(ops, rng, lens, 1, D, "f16", 32, width=width)
    host, q = cache.cpu().numpy(), (rng.standard_normal((4, G, D)) * size).astype(np.float16)
    plain = {}
    for b, n in enumerate(lens):
        k, v = (x.astype(np.float16) for x in DO.sequence(host, pages[b], n, 0, D, "f16"))
        plain[b] = v.copy()
        if n > 1:                                                     # one token e^300 above the others for the first head
            first = q[b, 0].astype(np.float64)
            k[7] = (first * 300 * D ** 0.5 / (first @ first)).astype(np.float16)
        low = int((q[b, -1].astype(np.float64) @ k.T.astype(np.float64)).argmin())
        v[rng.integers(n), 0] = np.inf
        v[low, 1] = -np.inf
        v[n // 2, 2] = -np.inf; v[n - 1, 3] = np.inf
        v[:, 4] = np.inf
        v[n // 3, 5] = np.nan
        v[0, 6] = np.inf; v[n - 1, 6] = -np.inf if n > 1 else np.inf
        for t in range(n):
            DO.put_token(host[pages[b, t // 32], 0, 0], t % 32, k[t], v[t], "f16")
    got = ops.paged_attention(dev(q), dev(host), dev(pages), i32(*lens)).cpu().numpy().astype(np.float64)
    for b, n in enumerate(lens):
        k, v = DO.sequence(host, pages[b], n, 0, D, "f16")
        with np.errstate(invalid="ignore"):
            o, _, _, w = DO.attend(q[b], k, v, D ** -0.5)
        assert (w > 0).all()
        assert np.isposinf(o[:, [0, 3, 4]]).all() and np.isneginf(o[:, 1:3]).all() and np.isnan(o[:, 5]).all()
        assert np.array_equal(got[b, :, :7], o[:, :7], equal_nan=True), (b, got[b, :, :7])
        parts = [(k, np.ones(n), np.zeros(n)), (np.where(np.isfinite(v), v, 0.0), np.ones(n), np.zeros(n))]
        o = w @ parts[1][0]
        bound = DO.attend_bound(q[b], *parts, D ** -0.5, "f16", o, w)
        assert (np.abs(got[b] - o)[:, 7:] <= bound[:, 7:]).all(), b


def test_scores_of_minus_infinity(ops):  # noqa: F811
    """f16: a token whose score is -inf has no weight at all; where every token's is, the output is NaN, not zero."""
    D, G, lens = 64, 4, [1, 33, 33, 1700]
    rng = np.random.default_rng(8)
    cache, pages = appended(ops, rng, lens, 1, D, "f16", 32)
    host, q = cache.cpu().numpy(), (rng.standard_normal((4, G, D)) * 2).astype(np.float16)
    q[:, :, 0] = np.abs(q[:, :, 0]) + np.float16(1)
    for b, n in enumerate(lens):
        k, v = (x.astype(np.float16) for x in DO.sequence(host, pages[b], n, 0, D, "f16"))
        out = slice(0, n) if b != 2 else slice(0, n - 1, 3)
        k[out, 0] = -np.inf
        for t in range(n):
            DO.put_token(host[pages[b, t // 32], 0, 0], t % 32, k[t], v[t], "f16")
    got = ops.paged_attention(dev(q), dev(host), dev(pages), i32(*lens))
    assert torch.isnan(got[[0, 1, 3]]).all()
    n = lens[2]
    k, v = DO.sequence(host, pages[2], n, 0, D, "f16")
    keep = np.isfinite(k[:, 0])
    assert not keep[0] and keep[1]
    parts = [(x[keep], np.ones(keep.sum()), np.zeros(keep.sum())) for x in (k, v)]
    o, _, _, w = DO.attend(q[2], k[keep], v[keep], D ** -0.5)
    assert (np.abs(got[2].cpu().numpy() - o) <= DO.attend_bound(q[2], *parts, D ** -0.5, "f16", o, w)).all()


def test_a_row_of_over_a_billion_tiles(ops):  # noqa: F811
    """1000 sequences of 34 million tokens that share their pages, 256 shares of the work for 512 workgroups: twice the quota times
    256 passes 2^31, so the workgroups past the last share must not multiply by it.  Equal scores, value scales and codes that are
    powers of two: every sum is exact (at most 2^24 equal terms a lane), and so is the output."""
    B, D, G, tiles, width = 1000, 64, 8, 1024, 1055
    length = 32 * (tiles * width - 256)
    units = B * (length // 32)
    assert 2 ** 30 < units and 511 * (units // 256) >= 2 ** 31 and B * (tiles * width + 6) <= 0x7FFF0000
    cache = torch.full((2, 1, tiles, ops.kv_tile_bytes(D, "int8")), 64, dtype=torch.uint8, device="cuda")
    for page in range(2):
        factors = torch.tensor([1.0, 2.0 ** (page - 6)], dtype=torch.float16, device="cuda").repeat_interleave(32)
        cache[page, 0, :, 4 * 32 * D // 2:] = factors.view(torch.uint8)
    pages = (torch.arange(B, dtype=torch.int32, device="cuda") % 2)[:, None].repeat(1, width)
    q, lens = torch.zeros((B, G, D), dtype=torch.float16, device="cuda"), torch.full((B,), length, dtype=torch.int32, device="cuda")
    got = ops.paged_attention(q, cache, pages, lens)
    want = -(2.0 ** (torch.arange(B, device="cuda") % 2))                  # (64 - 128) * 2^(page - 6)
    assert (got.float() == want[:, None, None]).all()
    assert not ops.gemv_workspace_for("cuda")[:65536].any()
