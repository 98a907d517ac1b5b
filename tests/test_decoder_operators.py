"""CPU side of the decoder operators behind the qkv linear: the oracle's cache layout and quantiser against their own
definitions, the rotary tables, and every refusal of the C entries and of the Python layer (nothing here launches)."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
from oracle import decoder_oracle as DO


@pytest.fixture(scope="module")
def lib():
    import os
    from kairos_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        from kairos_amd import build
        build.build(verbose=False)
    return _lib.load()


@pytest.mark.parametrize("kind", ["f16", "int8", "int4"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_tile_layout_uses_every_byte_once(lib, D, kind):
    from kairos_amd import ops
    n = ops.kv_tile_bytes(D, kind)
    assert n == DO.tile_bytes(D, kind) and n % 128 == 0
    used = np.zeros(n, np.int64)                                   # bits used of every byte
    for tau in range(32):
        for place in (DO.key_place, DO.value_place):
            words = {}
            for d in range(D):
                at, shift = place(tau, d, D, kind)
                if kind == "f16":
                    used[at] += 8; used[at + 1] += 8
                else:
                    used[at] += 8 if kind == "int8" else 4
                words.setdefault(at // 2, set()).add(d)
            assert all(len(w) == DO.PER_WORD[kind] for w in words.values())      # a token owns whole 16-bit words
        for i in range(DO.FACTORS[kind]):
            at = DO.factor_place(tau, i, D, kind)
            used[at] += 8; used[at + 1] += 8
    assert (used == 8).all()


def test_cache_forms_are_told_apart_by_their_tile_bytes(lib):
    assert len({DO.tile_bytes(D, k) for D in (64, 128, 256) for k in DO.PER_WORD}) == 9


@pytest.mark.parametrize("kind", ["int8", "int4"])
def test_quantiser_is_off_by_at_most_half_a_step(kind):
    """u = rint(x / s) off by half a step s, plus the rounding of the fp32 quotient (2^-23 of at most 127 steps); the widest rows
    included: no element is clipped although s is rounded to fp16, subnormal rows among them."""
    rng = np.random.default_rng(3)
    size = np.exp2(rng.integers(-24, 14, size=(400, 1))).astype(np.float32)
    x = np.clip(rng.standard_normal((400, 128)).astype(np.float32) * size, -65504, 65504).astype(np.float16)
    x[0] = 0; x[1] = 65504; x[2, ::2] = -65504; x[3] = np.float16(6e-8); x[4, 7] = 1.0
    u, s, z = DO.quantise(x, kind)
    assert np.isfinite(s.astype(np.float64)).all()
    v = DO.values_of(u, s, z, kind)
    half = s.astype(np.float64)[:, None] * (0.5 + 128 * 2.0 ** -23)
    if kind == "int4":                                              # max - min rounds to fp32 before it is divided
        half = half + (x.max(-1) .astype(np.float64) - x.min(-1))[:, None] * 2.0 ** -23
    assert (np.abs(v - x.astype(np.float64)) <= half).all()


def test_oracle_token_round_trip():
    rng = np.random.default_rng(0)
    for kind in ("f16", "int8", "int4"):
        tile = rng.integers(0, 256, size=DO.tile_bytes(64, kind)).astype(np.uint8)
        k, v = (rng.standard_normal((32, 64)).astype(np.float16) for _ in range(2))
        for tau in range(32):
            DO.put_token(tile, tau, k[tau], v[tau], kind)
        gk, gv = DO.get_tile(tile, 64, kind)
        assert all(np.array_equal(a[0], b) for a, b in zip(DO.get_tiles(tile[None], 64, kind), (gk, gv)))
        for x, got in ((k, gk), (v, gv)):
            if kind == "f16":
                assert np.array_equal(got, x.astype(np.float64))
            else:
                assert np.array_equal(got, DO.values_of(*DO.quantise(x, kind), kind))


# ---- rotary tables ------------------------------------------------------------------------------------------------------
def test_rotary_table_against_mpmath_free_angles():
    """fp32 of the exact cosine: off by half a step (2^-24 relative, 2^-25 absolute near 1) plus the 64-bit angle's rounding
    (position 10^6: 2^-33 radians)."""
    from kairos_amd.rotary import rotary_table
    t = rotary_table(1000, 32, base=500000.0, device="cpu")
    assert t.shape == (1000, 16, 2) and t.dtype == torch.float32
    for p in (0, 1, 31, 999):
        for i in range(16):
            a = p * 500000.0 ** (-2 * i / 32)
            for j, f in enumerate((math.cos, math.sin)):
                assert abs(float(t[p, i, j]) - f(a)) <= 2.0 ** -25 + 1e-12, (p, i)


def test_rotary_scalings():
    from kairos_amd.rotary import rotary_frequencies
    plain, one = rotary_frequencies(64, 10000.0)
    assert one == 1.0 and plain.dtype == torch.float64 and float(plain[0]) == 1.0
    lin, _ = rotary_frequencies(64, 10000.0, {"rope_type": "linear", "factor": 4.0})
    assert torch.allclose(lin, plain / 4, rtol=1e-15)
    ntk, _ = rotary_frequencies(64, 10000.0, {"type": "ntk", "factor": 4.0})
    assert float(ntk[0]) == 1.0 and abs(float(ntk[-1]) / float(plain[-1]) - 0.25) < 1e-12     # the slowest pair slows by the factor
    l3, _ = rotary_frequencies(128, 500000.0, {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
                                               "original_max_position_embeddings": 8192})
    base, _ = rotary_frequencies(128, 500000.0)
    wave = 2 * math.pi / base
    assert torch.equal(l3[wave < 8192 / 4], base[wave < 8192 / 4])
    assert torch.allclose(l3[wave > 8192], base[wave > 8192] / 8, rtol=1e-15)
    mid = (wave >= 8192 / 4) & (wave <= 8192)
    ramp = (8192 / wave[mid] - 1.0) / 3.0
    assert mid.any() and torch.allclose(l3[mid], (1 - ramp) * base[mid] / 8 + ramp * base[mid], rtol=1e-12)
    yarn, gain = rotary_frequencies(64, 10000.0, {"rope_type": "yarn", "factor": 16.0, "original_max_position_embeddings": 4096})
    turns = 4096 * plain / (2 * math.pi)
    assert abs(gain - (0.1 * math.log(16.0) + 1.0)) < 1e-15
    assert torch.equal(yarn[turns > 40], plain[turns > 40]) and torch.allclose(yarn[turns < 0.5], plain[turns < 0.5] / 16, rtol=1e-12)
    assert ((yarn <= plain * (1 + 1e-15)) & (yarn >= plain / 16 * (1 - 1e-15))).all()
    assert rotary_frequencies(64, 10000.0, {"rope_type": "yarn", "factor": 16.0, "original_max_position_embeddings": 4096,
                                            "attention_factor": 1.0})[1] == 1.0
    for bad in ({"rope_type": "other", "factor": 2.0}, {"rope_type": "linear"}, {"rope_type": "linear", "factor": 0.5}, {"factor": 2.0}):
        with pytest.raises(ValueError):
            rotary_frequencies(64, 10000.0, bad)
    for R in (0, 8, 20, -16):
        with pytest.raises(ValueError):
            rotary_frequencies(R)
    with pytest.raises(ValueError):
        rotary_frequencies(64, 1.0)


# ---- refusals of the C entries -------------------------------------------------------------------------------------------
ROPE = dict(q_out=16, k_out=16, cache=16, q=16, k=16, v=16, table=16, start=16, count=0, page_table=16, q_batch=0, q_token=0,
            k_batch=0, k_token=0, v_batch=0, v_token=0, B=1, S=1, H=4, KV=2, D=64, rotary_dim=64, table_rows=8, interleaved=0,
            kind=0, num_pages=4, page_tiles=1, max_pages=4)
READ = dict(k_out=16, v_out=16, cache=16, start=16, count=0, page_table=16, B=1, S=1, KV=2, D=64, kind=0, num_pages=4, page_tiles=1,
            max_pages=4)
ATTN = dict(out=16, q=16, cache=16, page_table=16, lens=16, workspace=16, workspace_bytes=1 << 30, q_batch=0, scale=0.125, B=1, H=4, KV=2, D=64, kind=0, num_pages=4,
            page_tiles=1, max_pages=4, window=0)


def _pack(form, base, change):
    return form.pack(*dict(base, **change).values())


@pytest.mark.parametrize("change, code", [
    (dict(start=0), -1), (dict(k=0), -1), (dict(q=0), -1), (dict(q_out=0), -1), (dict(cache=0, k_out=0), -1), (dict(v=0), -1),
    (dict(page_table=0), -1), (dict(q=8), -5), (dict(k=24), -5), (dict(v=2), -5), (dict(cache=8), -5), (dict(table=4), -5),
    (dict(k_out=8), -5), (dict(q_out=4), -5), (dict(q_token=4), -5), (dict(v_batch=12), -5),
    (dict(D=96), -2), (dict(D=0), -2), (dict(B=-1), -2), (dict(B=65536), -2), (dict(S=-1), -2), (dict(KV=0), -2), (dict(H=0), -2),
    (dict(H=70000), -2), (dict(rotary_dim=72), -2), (dict(rotary_dim=24), -2), (dict(rotary_dim=-16), -2), (dict(table=0), -2),
    (dict(table_rows=0), -2), (dict(kind=3), -2), (dict(kind=-1), -2), (dict(num_pages=0), -2), (dict(page_tiles=0), -2),
    (dict(max_pages=0), -2), (dict(max_pages=1 << 20, page_tiles=1 << 10), -2), (dict(max_pages=1 << 26), -2),
    (dict(num_pages=1 << 28, KV=8), -2), (dict(S=(1 << 26) + 1), -2), (dict(B=0), 0), (dict(S=0), 0),
])
def test_rope_kv_refusals(lib, change, code):
    from kairos_amd import ops
    assert lib.kmi_rope_kv(_pack(ops._rope_kv_args, ROPE, change), None) == code
    if code < 0:
        assert b"kmi_" in lib.kmi_get_last_error_string()
    assert lib.kmi_rope_kv(None, None) == -1


@pytest.mark.parametrize("change, code", [
    (dict(k_out=0), -1), (dict(v_out=0), -1), (dict(start=0), -1), (dict(cache=0), -1), (dict(page_table=0), -1), (dict(k_out=8), -5),
    (dict(cache=8), -5), (dict(D=32), -2), (dict(kind=4), -2), (dict(S=-1), -2), (dict(KV=0), -2), (dict(B=70000), -2),
    (dict(num_pages=0), -2), (dict(max_pages=0), -2), (dict(S=0x7FFFFFFF, KV=65535), -2), (dict(S=(1 << 26) + 1), -2), (dict(B=0), 0), (dict(S=0), 0),
])
def test_kv_read_refusals(lib, change, code):
    from kairos_amd import ops
    assert lib.kmi_kv_read(_pack(ops._kv_read_args, READ, change), None) == code
    assert lib.kmi_kv_read(None, None) == -1


@pytest.mark.parametrize("change, code", [
    (dict(out=0), -1), (dict(q=0), -1), (dict(lens=0), -1), (dict(cache=0), -1), (dict(page_table=0), -1), (dict(out=8), -5), (dict(q=8), -5),
    (dict(q_batch=4), -5), (dict(H=5), -2), (dict(H=0), -2), (dict(KV=3), -2), (dict(D=80), -2), (dict(kind=9), -2), (dict(window=-1), -2),
    (dict(scale=0.0), -2), (dict(scale=-1.0), -2), (dict(scale=float("nan")), -2), (dict(scale=float("inf")), -2), (dict(scale=1e16), -2), (dict(workspace=0), -2),
    (dict(workspace_bytes=1 << 16), -2), (dict(workspace=8), -5), (dict(B=65535, KV=2, H=4, max_pages=1 << 20), -2), (dict(B=0), 0),
])
def test_paged_attn_refusals(lib, change, code):
    from kairos_amd import ops
    assert lib.kmi_paged_attn(_pack(ops._paged_attn_args, ATTN, change), None) == code
    assert lib.kmi_paged_attn(None, None) == -1


def test_structs_have_the_header_s_size():
    """struct.Struct formats of the binding against the C layout (pointers and int64 first, then 32-bit fields)."""
    from kairos_amd import ops
    assert ops._rope_kv_args.size == 10 * 8 + 6 * 8 + 12 * 4
    assert ops._kv_read_args.size == 6 * 8 + 8 * 4
    assert ops._paged_attn_args.size == 7 * 8 + 8 + 4 + 9 * 4


def test_python_layer_refuses_cpu_tensors_and_wrong_forms(lib):
    from kairos_amd import ops
    from kairos.kv_cache import PagedKVCache
    h = torch.zeros((1, 2, 4, 64), dtype=torch.float16)
    i = torch.zeros(1, dtype=torch.int32)
    cache = torch.zeros((2, 4, 1, ops.kv_tile_bytes(64, "int8")), dtype=torch.uint8)
    with pytest.raises(ValueError):
        ops.rotary(h, h, i, torch.zeros((4, 32, 2)))
    with pytest.raises(TypeError):
        ops.rotary(h.float(), h.float(), i, torch.zeros((4, 32, 2)))
    with pytest.raises(ValueError):
        ops.kv_read(cache, torch.zeros((1, 1), dtype=torch.int32), i, 4)
    with pytest.raises(ValueError):
        ops.paged_attention(h[:, 0], cache, torch.zeros((1, 1), dtype=torch.int32), i)
    with pytest.raises(ValueError):
        ops.kv_tile_bytes(64, "int2")
    with pytest.raises(Exception):
        ops.kv_tile_bytes(96, "int8")
    for bad in (dict(page_size=48), dict(page_size=0), dict(kind="fp8")):
        with pytest.raises(ValueError):
            PagedKVCache(4, 2, 64, device="cpu", **bad)
    with pytest.raises(ValueError):
        PagedKVCache(0, 2, 64, device="cpu")
    c = PagedKVCache(4, 2, 128, "int4", 64, device="cpu")
    assert c.data.shape == (4, 2, 2, 4352) and c.bytes_per_token == 2 * 136
