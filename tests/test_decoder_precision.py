"""The bound that decode attention is held to, on the CPU: it lets the exact answer's rounding pass and turns down mistakes planted in
the oracle's."""
import numpy as np
import pytest

from oracle import decoder_oracle as DO

KINDS = ["f16", "int8", "int4"]


def case(D, T, kind, G=4, seed=0):
    """Normal rows quantised by the oracle, q times 2: what the GPU tests attend to."""
    rng = np.random.default_rng(seed + D + T)
    parts = []
    for _ in range(2):
        x = rng.standard_normal((T, D)).astype(np.float16)
        if kind == "f16":
            parts.append((x.astype(np.float64), np.ones(T), np.zeros(T)))
        else:
            u, s, z = DO.quantise(x, kind)
            parts.append((u.astype(np.float64), s.astype(np.float64), z.astype(np.float64)))
    k, v = (DO.values_of(u, s, z, kind) if kind != "f16" else u for u, s, z in parts)
    q = (rng.standard_normal((G, D)) * 2).astype(np.float16)
    o, _, _, w = DO.attend(q, k, v, D ** -0.5)
    return q, k, v, parts, o, w, DO.attend_bound(q, *parts, D ** -0.5, kind, o, w)


def half(x):
    return x.astype(np.float16).astype(np.float64)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D, T", [(64, 1), (64, 129), (128, 129), (256, 129), (64, 2500), (128, 1536), (256, 700)])
def test_the_rounded_answer_passes_and_mistakes_do_not(D, T, kind):
    q, k, v, parts, o, w, bound = case(D, T, kind)
    assert (np.abs(half(o) - o) <= bound).all()
    scale = D ** -0.5

    def refused(x):
        return (np.abs(half(x) - o) > bound).mean()

    assert refused(0 * o) > 0.9
    assert refused(o * 1.02) > 0.5                                            # every value 2 % too large
    if T > 1:
        assert refused(DO.attend(q, k, v, scale * 1.02)[0]) > 0.5
        assert refused(DO.attend(q, k[:-32], v[:-32], scale)[0]) > 0.5
        assert refused(DO.attend(q, k[1:], v[:-1], scale)[0]) > 0.9           # keys beside their neighbours' values
    if 1 < T <= 129:
        assert refused(DO.attend(q, k[:-1], v[:-1], scale)[0]) > 0            # one token left out


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_the_bound_is_a_small_part_of_the_outputs(D, kind):
    """Median over the outputs' root mean square, 129 tokens: the output's rounding is 2^-12 to 2^-11 of it."""
    q, k, v, parts, o, w, bound = case(D, 129, kind)
    assert np.median(bound) < 2.0 ** -8 * np.sqrt((o ** 2).mean())


def test_the_bound_turns_down_queries_rounded_on_their_way():
    """int4: half of the elements divided by 16 in fp16, where they are subnormal, moves outputs past the bound."""
    rng = np.random.default_rng(1)
    q, k, v, parts, o, w, _ = case(64, 300, "int4")
    q = (rng.standard_normal((4, 64)) * 1e-5).astype(np.float16)
    scale = 2.0 / (1e-5 * 8)
    o, _, _, w = DO.attend(q, k, v, scale)
    bound = DO.attend_bound(q, *parts, scale, "int4", o, w)
    (u, s, z), _ = parts
    high = np.arange(64) % 4 >= 2
    lossy = np.where(high, (q / np.float16(16)).astype(np.float64) * 16, q.astype(np.float64))
    x = (lossy @ (u * s[:, None]).T + q.astype(np.float64).sum(-1, keepdims=True) * z) * scale
    p = np.exp(x - x.max(-1, keepdims=True))
    assert (np.abs(half(o) - o) <= bound).all() and (np.abs(p @ v / p.sum(-1, keepdims=True) - o) > bound).mean() > 0.5


@pytest.mark.parametrize("kind", KINDS)
def test_codes_taken_apart_are_the_values(kind):
    rng = np.random.default_rng(7)
    D, KV = 64, 2
    cache = np.zeros((3, KV, 2, DO.tile_bytes(D, kind)), np.uint8)
    for t in range(100):
        for h in range(KV):
            k, v = (rng.standard_normal(D).astype(np.float16) for _ in range(2))
            DO.put_token(cache[(2, 0)[t // 64], h, t % 64 // 32], t % 32, k, v, kind)
    whole = DO.sequence(cache, [2, 0], 100, 1, D, kind)
    for (u, s, z), x in zip(DO.sequence_codes(cache, [2, 0], 13, 100, 1, D, kind), whole):
        got = u if kind == "f16" else DO.values_of(u, s, z, kind)
        assert np.array_equal(got, x[13:])
