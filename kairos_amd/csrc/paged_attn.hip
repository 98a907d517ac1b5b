// Attention of one new token a sequence over the paged cache:
//   o[b, h] = sum_t p_t v_t / sum_t p_t,   p_t = exp(scale q[b, h] . k_t - m),   t over the sequence's (window's) tokens
// One pass over the cache with a running reference m and sum of the softmax.  The G = H / KV query heads that share a key
// head are the 16 columns of a matrix instruction, 32 tokens a step:
//   S^T [token x head] = K Q^T      (16x16x32 MFMA, two row halves of 16 tokens)
//   O^T [d x head]    += V^T P^T    (16x16x32 MFMA, a step's 32 tokens deep)
// The cache's tile order makes the result registers of the first product, lane (head, g) = tokens 8 g .. 8 g + 7, the operand
// registers of the second: nothing passes through LDS or between lanes but the maximum over the four lane groups, where m is raised.
// The weights enter the second product as two fp16 numbers that add up to 22 bits, an instruction each.
// Codes enter the products masked where they stand, as fp16 subnormals (the MFMA takes them exactly): one instruction for two.  A key's
// factors meet its score in fp32, with the sum of q for the offset.  A value's scale multiplies p, in fp32 before the split in two; m is
// one reference a head for p and for that product, so that both stay in range.  The codes' middle is taken off the sums at the end by
// the sum of the same split weights (two more MFMAs a tile against a row of ones), and the offsets of the int4 kind add up to one scalar
// a head.
//
// Bound by the reading of the cache (a plain read past the caches: 7.0 TB/s): 2 x 131072 f16 (1074 MB) 162 us, 6.6 TB/s; 64 ragged up to 8192
// f16 95 us, 5.8 TB/s; 32 x 1536 int8 20.4 us; over int4 by its arithmetic as well: 4 x 100001 (64 heads on 8 of 128) 76-77 us for 435 MB,
// 5.7 TB/s.  One sequence of 200 tokens: 6.7-6.9 us, all of it latency (the schedule 2, the first loads 1, the joins 2).
#include "kv_parts.h"

// Waves of a workgroup.  Loads are short of flight where tiles are small, so there eight waves (two a SIMD, one computing while the other
// waits): int4 (4 x 100001: 77 us, four waves 85), int8 with heads of 64 (8 x 60000: 82 us, 97), and 32 query heads a wave, for their
// arithmetic (64 x up to 62479 int8, 20 heads of 64: 66 us, 78).  Else four read as fast and start and end a share sooner (1 x 4096 int8:
// 11.5 us, 14.2).  More tasks than CUs: small workgroups, several a CU, so that one task's end hides behind another's middle:
// int4 of 128 with over 256 tasks four waves (64 x up to 1000, 8 key heads: 15.4 us, 28 with eight; up to 8000: 63, 83; but 256
// tasks, 32 x 1536: 23.5, 15.6 with eight); from 2048 on, or 1024 of codes with heads of 64, two (256 x up to 300, 8 key heads of 128,
// int8: 29 us, 40 with four; 1000 x up to 100 int4: 63, 86; against it 256 x up to 2000 f16: 184, 172).  Heads of 256 fill a SIMD's
// registers with one wave.
static constexpr bool pa_codes64(int D, int kind, int pack) { return kind != KMI_KV_F16 && D == 64 && pack == 2; }
static int pa_waves(int D, int kind, int pack, int columns, long long tasks) {
    if (columns == 32) return 8;
    if (D < 256 && tasks >= (pa_codes64(D, kind, pack) ? 1024 : 2048)) return 2;
    if (pa_codes64(D, kind, pack)) return 8;
    return kind == KMI_KV_INT4 && (D == 256 || tasks <= 256) ? 8 : 4;
}
static constexpr int pa_a_cu(int D, int kind, int pack, int waves) {         // workgroups that fit a CU's registers
    const int most = D == 256 ? 4 : pa_codes64(D, kind, pack) ? 16 : kind == KMI_KV_INT4 && pack == 2 ? 12 : 8;      // waves
    return most < waves ? 1 : most / waves;
}
// Shares.  256 at a time, one a CU, read a long cache 4 % faster than 512 (164 us against 170 for 2 x 131072 f16: fewer places of
// memory at once), more hide the starts and ends of short tasks (64 x up to 1000 int8, 8 key heads: 19 us, 28 with 256 workgroups).
static constexpr int PA_LONG = 96;            // tiles a share from which 256 uneven ones are taken all the same
// Being cut costs a task about 3 us (hand-off and join): none of up to nine tiles a wave is (2 x 1152 f16, 36 tiles: 9.6 us
// whole, 10.6 cut), and no share is smaller than three (1 x 4096 f16: 11.8 us, 13.2 with six).
static constexpr int PA_WHOLE_STEPS = 9, PA_MIN_STEPS = 3;
static constexpr int PA_SMALL_BYTES = 320 << 10;   // of a task that no row of tasks is cut in (256 x up to 300 f16: 42 us, 46 with such cuts)
static constexpr int PA_HELD = 1024;          // sequences whose lengths the schedule keeps in LDS
static constexpr int PA_TASK_COST = 6;        // tiles' worth of a task's start and end; 3 and 12 measured the same
// Tiles of the page table from which a wave takes 32 query heads at once (more than 16 share a key head; not int4, whose arithmetic
// then spills: 40 us against 30): the cache is read once (16 x up to 20000 f16, 64 heads on 2: 44 us against 63; int8 34 and 41), but
// there are half as many shares (13 x up to 7411 int4: 21 us against 14).  By the table's room, since the lengths are on the device: short
// sequences under a wide table take this form too.
static constexpr long long PA_WIDE = 12288;

// The largest weight starts at 2^8: weights down to 2^-22 of it are then normal numbers of fp16, and the two numbers together are off by
// at most 2^-33 of the largest weight where they are smaller still.
static constexpr float PA_LIFT = 8.0f;
static constexpr float PA_NEG = -1e30f;       // the reference before the first token: below every x, finite, so differences stay numbers

// Over the four lane groups g that hold a head's tokens: the row swaps leave a pair of neighbouring groups' values in both.
template <typename F>
__device__ __forceinline__ float over_groups(float v, F f) {
    uint32_t u = __builtin_bit_cast(uint32_t, v);
    auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const uint32_t a0 = a[0], a1 = a[1];
    u = __builtin_bit_cast(uint32_t, f(__builtin_bit_cast(float, a0), __builtin_bit_cast(float, a1)));
    auto b = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const uint32_t b0 = b[0], b1 = b[1];
    return f(__builtin_bit_cast(float, b0), __builtin_bit_cast(float, b1));
}
__device__ __forceinline__ float group_max(float v) { return over_groups(v, [](float a, float b) { return fmaxf(a, b); }); }
__device__ __forceinline__ float group_sum(float v) { return over_groups(v, [](float a, float b) { return a + b; }); }
// What a sum is worth relative to a higher reference, 2^x.  Never zero: an infinite sum stays one, and 2^-126 of a finite one is nothing.
__device__ __forceinline__ float decay(float x) { return fmaxf(__builtin_amdgcn_exp2f(x), 0x1p-126f); }

// Eight halves of unit u (0 .. n - 1) of a 16-byte key chunk: the elements, or their codes u as subnormals, u * 2^-24 (int8) or u * 2^-20
// (int4, for the low bits that sums of subnormals lose: see value_unit).  All at one place, so that q enters as it is: a query is never
// rounded (q / 16 for the nibbles that stand higher saves two shifts a unit, 32 x 1536 14.7 us for 14.9, but lost bits of queries
// below 2^-10: outputs off by 3 % where all of q was about 1e-5).
template <int KIND>
__device__ __forceinline__ h8_t key_unit(const u4_t& c, int u) {
    u4_t o = c;
    if constexpr (KIND == KMI_KV_INT8) {
        o[0] = __builtin_amdgcn_perm(0u, c[2 * u], 0x0C010C00u);
        o[1] = __builtin_amdgcn_perm(0u, c[2 * u], 0x0C030C02u);
        o[2] = __builtin_amdgcn_perm(0u, c[2 * u + 1], 0x0C010C00u);
        o[3] = __builtin_amdgcn_perm(0u, c[2 * u + 1], 0x0C030C02u);
    } else if constexpr (KIND == KMI_KV_INT4) {
        const uint32_t w = c[u];
        o[0] = w << 4 & 0x00F000F0u;
        o[1] = w & 0x00F000F0u;
        o[2] = w >> 4 & 0x00F000F0u;
        o[3] = w >> 8 & 0x00F000F0u;
    }
    return __builtin_bit_cast(h8_t, o);
}

// Value a (0 .. n - 1) of the eight tokens of a 16-byte value chunk: the element, or its code u as the subnormal u * 2^-24, for int4
// u * 2^-20: measured, the sum of a product's terms loses low bits of subnormals (nibbles at 2^-24: outputs 3.6e-4 of their root mean
// square too low over 100001 tokens, 1e-5 at 2^-20; bytes at 2^-24: 2e-5).
template <int KIND>
__device__ __forceinline__ h8_t value_unit(const u4_t& c, int a) {
    u4_t o = c;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (KIND == KMI_KV_INT8) o[i] = a ? __builtin_amdgcn_perm(0u, c[i], 0x0C030C01u) : c[i] & 0x00FF00FFu;
        if constexpr (KIND == KMI_KV_INT4) o[i] = (a == 0 ? c[i] << 4 : c[i] >> (4 * a - 4)) & 0x00F000F0u;
    }
    return __builtin_bit_cast(h8_t, o);
}

// Infinities and NaN to fp16's largest numbers, by the bits: as integers with a sign the positive ones stand highest, without one the negative.
__device__ __forceinline__ h8_t in_range(h8_t x) {
    typedef int16_t s8_t __attribute__((ext_vector_type(8)));
    typedef uint16_t us8_t __attribute__((ext_vector_type(8)));
    const s8_t p = __builtin_elementwise_min(__builtin_bit_cast(s8_t, x), (s8_t)(int16_t)0x7BFF);
    return __builtin_bit_cast(h8_t, __builtin_elementwise_min(__builtin_bit_cast(us8_t, p), (us8_t)(uint16_t)0xFBFF));
}

// One wave's share of one head's tokens.  PACK = 2 (at most 8 query heads): columns 0-7 of the product are the heads on the tokens of
// the tile's half h = 0, columns 8-15 the same heads on half 1, each with a running maximum of its own: q stands twice in
// the operand, zero in the other half's columns, and every lane has four scores a tile instead of eight.
template <int D, int KIND, int PACK>
struct PaWave {
    static constexpr int n = kv_per_word(KIND), CH = D / 16 / n, KSTEPS = D / 32, OT = D / 16, NF = kv_factors(KIND);
    static constexpr int TILE_BYTES = kv_tile_bytes(D, KIND), PART = kv_part_bytes(D, KIND);
    static constexpr int NS = 8 / PACK;                        // scores a lane holds of a tile
    static constexpr bool CODES = KIND != KMI_KV_F16;
    static constexpr float UNIT = !CODES ? 1.0f : KIND == KMI_KV_INT4 ? 0x1p20f : 0x1p24f;      // what a code's place divides it by
    typedef _Float16 fac_t __attribute__((ext_vector_type(NS)));
    h8_t q[PACK][KSTEPS];       // lane (column, g): q[32 kk + 8 g ..]
    f4_t acc[OT];               // lane (column, g): tile T = n c + a, rows dl = 4 g + r, d = 16 n c + n dl + a
    f4_t psum;                  // sum of the weights that entered acc (every row the same)
    float m;                    // the column's reference: weights are p = 2^(x - m), x = score * scale * log2(e)
    float l, zsum;              // this lane's share of the sums of p and of p * offset
    float c, qc;                // scale * log2(e) times UNIT; sum of q, times scale * log2(e)

    __device__ __forceinline__ void load_q(const half_t* qrow, bool used, int g) {
#pragma unroll
        for (int kk = 0; kk < KSTEPS; ++kk) q[0][kk] = used ? *reinterpret_cast<const h8_t*>(qrow + 32 * kk + 8 * g) : h8_t{};
    }
    __device__ __forceinline__ void start(int col, float scale) {
        float s = 0.0f;
#pragma unroll
        for (int kk = 0; kk < KSTEPS; ++kk) {
            const h8_t x = q[0][kk];
            if constexpr (CODES) {
#pragma unroll
                for (int e = 0; e < 8; ++e) s += (float)x[e];
            }
            if constexpr (PACK == 1) {
                q[0][kk] = x;
            } else {
                q[0][kk] = col < 8 ? x : h8_t{};
                q[1][kk] = col < 8 ? h8_t{} : x;
            }
        }
        c = scale * UNIT;
        qc = CODES ? group_sum(s) * scale : 0.0f;
#pragma unroll
        for (int t = 0; t < OT; ++t) acc[t] = f4_t{};
        psum = f4_t{};
        m = PA_NEG; l = 0.0f; zsum = 0.0f;
    }

    struct Factors {
        fac_t f[NF ? NF : 1];
    };
    struct Tile {
        u4_t k[CH], v[CH];
        Factors f;
    };
    struct Scores {
        float s[NS];
    };
    // The weights in two numbers of fp16, 22 bits, so that nothing but the output is rounded to 11: off by 2.0e-4 to 2.1e-4 of the output's
    // norm, as the output's rounding alone; with one number f16 2.7e-4, codes 2.2e-4 to 2.5e-4.  In the same time over f16 and int8 (2 x 131072
    // f16 163 us; 32 x 1536 int8 20.3 us, 20.2 with one), dearer over int4 (4 x 100001 77.3 us, 76.6; 32 x 1536 14.7 us, 13.9).
    struct Weights {
        h8_t high, low;
    };
    // The first of the lane's NS tokens in a tile.
    static __device__ __forceinline__ int first_token(int lane) { return 8 * (lane >> 4) + (PACK == 2 ? (lane >> 1) & 4 : 0); }

    // A cache is read once a step: loads that leave nothing behind in the caches (2 x 131072 f16: 162 us, 182 with ordinary ones; 64 ragged up
    // to 8192: 93, 107; against it a cache small enough to stay: 8 x up to 3000 f16, heads of 256: 27, 20).
    static __device__ __forceinline__ void load_keys(Tile& t, const char* tile, int lane) {
#pragma unroll
        for (int i = 0; i < CH; ++i) t.k[i] = __builtin_nontemporal_load(reinterpret_cast<const u4_t*>(tile + i * 1024 + lane * 16));
#pragma unroll
        for (int i = 0; i < NF; ++i) t.f.f[i] = *reinterpret_cast<const fac_t*>(tile + 2 * PART + 64 * i + 2 * first_token(lane));
    }
    static __device__ __forceinline__ void load_values(Tile& t, const char* tile, int lane) {
#pragma unroll
        for (int i = 0; i < CH; ++i) t.v[i] = __builtin_nontemporal_load(reinterpret_cast<const u4_t*>(tile + PART + i * 1024 + lane * 16));
    }

    // Raw scores of the lane's tokens and column.
    __device__ __forceinline__ Scores scores(const Tile& t, int lane) const {
        f4_t s4[2] = {f4_t{}, f4_t{}};
#pragma unroll
        for (int kk = 0; kk < KSTEPS; ++kk) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int unit = h * KSTEPS + kk;
                s4[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(key_unit<KIND>(t.k[unit / n], unit % n), q[PACK == 2 ? h : 0][kk], s4[h], 0, 0, 0);
            }
        }
        if constexpr (PACK == 2) {                             // a choice, no sum: zero times a masked token's contents may be NaN
#pragma unroll
            for (int r = 0; r < 4; ++r) s4[0][r] = lane & 8 ? s4[1][r] : s4[0][r];
        }
        Scores o;
#pragma unroll
        for (int j = 0; j < NS; ++j) o.s[j] = s4[j >> 2][j & 3];
        return o;
    }
    // x - less of a product's result: the score in powers of two.
    __device__ __forceinline__ float exponent(float s, const Factors& fac, int j, float less) const {
        if constexpr (KIND == KMI_KV_F16) return __builtin_fmaf(s, c, -less);
        if constexpr (KIND == KMI_KV_INT8) return __builtin_fmaf(__builtin_fmaf(s, c, -128.0f * qc), (float)fac.f[0][j], -less);
        return __builtin_fmaf(s * c, (float)fac.f[0][j], __builtin_fmaf(qc, (float)fac.f[1][j], -less));
    }
    // The weights that meet the values -- p, for codes p times the token's value scale -- from the products' results, as fp16
    // operands; the reference, the sums and the accumulators are brought to them.  The reference is raised (so that the largest weight
    // is 2^8, or the largest p 2^40 where every value scale is tiny) only where a weight would pass 2^15 or p 2^48, which is seldom
    // after a wave's first tile: no reduction over lanes otherwise.  fac: the tile's factors, tok: its first token, [lo, hi) the
    // tokens that count, bad: no page of this cache.
    template <bool CAREFUL>
    __device__ __forceinline__ Weights weights(const Scores& sc, Tile& tile, Factors& fac, int tok, int lo, int hi, bool bad, int lane) {
        float vs[NS], y[NS], p[NS], wt[NS];
#pragma unroll
        for (int j = 0; j < NS; ++j) {
            vs[j] = CODES ? (float)fac.f[NF / 2][j] : 1.0f;
            y[j] = exponent(sc.s[j], fac, j, m);
        }
        if (tok < lo || tok + KV_TILE > hi) {
            // tokens outside: no weight, and nothing that stands in their place may reach a product
#pragma unroll
            for (int j = 0; j < NS; ++j) {
                const int t = tok + first_token(lane) + j;
                const bool in = t >= lo && t < hi;
                y[j] = in ? y[j] : -__builtin_inff();
                vs[j] = in ? vs[j] : 0.0f;
                if constexpr (KIND == KMI_KV_INT4) fac.f[3][j] = in ? fac.f[3][j] : (half_t)0.0f;
            }
            if constexpr (!CODES) {
                u4_t keep = {};
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int t = tok + 8 * (lane >> 4) + j;
                    keep[j >> 1] |= t >= lo && t < hi ? 0xFFFFu << (16 * (j & 1)) : 0u;
                }
#pragma unroll
                for (int i = 0; i < CH; ++i) tile.v[i] &= keep;
            }
        }
        if (bad) {
#pragma unroll
            for (int j = 0; j < NS; ++j) y[j] = __builtin_nanf("");
        }
        float wtop = 0.0f, ytop = PA_NEG;
#pragma unroll
        for (int j = 0; j < NS; ++j) {
            p[j] = __builtin_amdgcn_exp2f(y[j]);
            wt[j] = CODES ? p[j] * vs[j] : p[j];
            wtop = fmaxf(wtop, wt[j]);
            if constexpr (CODES) ytop = fmaxf(ytop, y[j]);
        }
        if (__any(wtop > 32768.0f || ytop > 48.0f)) {
            float top = -__builtin_inff(), wide = top;             // largest x, largest x + log2(value scale)
#pragma unroll
            for (int j = 0; j < NS; ++j) {
                // from the products again: y is what m left of x
                y[j] = y[j] == -__builtin_inff() ? y[j] : bad ? __builtin_nanf("") : exponent(sc.s[j], fac, j, 0.0f);
                top = fmaxf(top, y[j]);
                if constexpr (CODES) wide = fmaxf(wide, y[j] + __builtin_amdgcn_logf(vs[j]));
            }
            top = group_max(top);
            const float m2 = fmaxf(m, CODES ? fmaxf(group_max(wide) - PA_LIFT, top - 40.0f) : top - PA_LIFT);
            const float a = decay(m - m2);
            m = m2;
            l *= a; zsum *= a;
            if constexpr (CODES) psum = psum * a;
#pragma unroll
            for (int i = 0; i < OT; ++i) acc[i] = acc[i] * a;
#pragma unroll
            for (int j = 0; j < NS; ++j) {
                p[j] = __builtin_amdgcn_exp2f(y[j] - m);
                wt[j] = CODES ? p[j] * vs[j] : p[j];
            }
        }
        h8_t pf = {}, rest = {};
#pragma unroll
        for (int j = 0; j < NS; ++j) {
            l += p[j];
            if constexpr (KIND == KMI_KV_INT4) zsum = __builtin_fmaf(p[j], __builtin_fmaf(7.5f, vs[j], (float)fac.f[3][j]), zsum);
            pf[j] = (half_t)wt[j];
            // careful: a token that counts has some weight, however low its score, so that an infinite value's never rounds to 0 (0 * inf)
            if constexpr (CAREFUL) pf[j] = y[j] > -__builtin_inff() ? __builtin_fmaxf16(pf[j], (half_t)0x1p-24f) : pf[j];
            rest[j] = (half_t)(wt[j] - (float)pf[j]);
        }
        if constexpr (PACK == 2) {                             // the lane's tokens are its column's half of the operand's eight
            const uint32_t first = lane & 8 ? 0u : 0xFFFFFFFFu;
            auto placed = [&](h8_t x) {
                const u4_t w = __builtin_bit_cast(u4_t, x);
                return __builtin_bit_cast(h8_t, u4_t{w[0] & first, w[1] & first, w[0] & ~first, w[1] & ~first});
            };
            pf = placed(pf);
            rest = placed(rest);
        }
        return {pf, rest};
    }
    // Careful: the low numbers are of either sign or zero, so they meet the values brought into fp16's range, and an infinite value comes
    // through the high numbers alone (as it is; of both signs NaN).
    template <bool CAREFUL>
    __device__ __forceinline__ void add(const Tile& tile, const Weights& w) {
#pragma unroll
        for (int T = 0; T < OT; ++T) {
            const h8_t v = value_unit<KIND>(tile.v[T / n], T % n);
            acc[T] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, w.high, acc[T], 0, 0, 0);
            acc[T] = __builtin_amdgcn_mfma_f32_16x16x32_f16(CAREFUL ? in_range(v) : v, w.low, acc[T], 0, 0, 0);
        }
        if constexpr (CODES) {
            const half_t one = (half_t)1.0f;
            const h8_t ones = {one, one, one, one, one, one, one, one};
            psum = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, w.high, psum, 0, 0, 0);
            psum = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, w.low, psum, 0, 0, 0);
        }
    }
    // Is there a sum that is not finite while the weights are numbers?
    __device__ __forceinline__ bool not_finite() const {
        f4_t s = f4_t{};
#pragma unroll
        for (int T = 0; T < OT; ++T) s = s + acc[T] * 0.0f;
        return __any(!(s[0] + s[1] + s[2] + s[3] == 0.0f) && l == l);
    }
    // What the join needs besides m and acc: the sums over the lane groups, and what is added to every output: the offsets (of the
    // codes' middle), less the middle times the very weights that entered acc, so that their rounding cancels.
    __device__ __forceinline__ void totals(float& sum, float& add) const {
        sum = group_sum(l);
        add = 0.0f;
        if constexpr (KIND == KMI_KV_INT8) add = -128.0f * psum[0];
        if constexpr (KIND == KMI_KV_INT4) add = group_sum(zsum) - 7.5f * psum[0];
    }
    static __device__ __forceinline__ float other_half(float v) {          // row_ror 8: column c ^ 8 of the same lane group
        return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x128, 0xF, 0xF, false));
    }
    static __device__ __forceinline__ int d_of(int T, int dl) { return 16 * n * (T / n) + n * dl + T % n; }
};

// Work is shared out by tiles.  The lengths are on the device, so every workgroup works the shares out itself, the same way:
//   quota q = tiles of all tasks (sequence, 16 query heads of a key head) / workgroups, at least min_quota;
//   if the tasks, cut into pieces of q (or of 9/8 q), are no more pieces than workgroups: one piece each;
//   else all tasks stand in a row, each with PA_TASK_COST further tiles for what a task costs besides its tiles, and workgroup w takes the
//   run [w q, (w + 1) q) of the row, whatever the lengths are.
// A task that lies in one share is finished there; one that is cut leaves a partial sum per workgroup (at most two each: the
// task that a share begins in the middle of, and the one that it ends in the middle of), and whichever workgroup of a task
// arrives last joins them in order.
struct PaSplit {
    uint32_t* counters;             // [gridDim.x] arrivals of the task that begins in share w and ends behind it; zero between calls
    float* partial;                 // [gridDim.x][2][slot], slot: m[16], l[16], o[used][D]
    int slot;
    int tasks_a_sequence, head_tiles;
    float c;
};

// Inclusive sum over the wave's lanes.
__device__ __forceinline__ int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);        // row_shr 1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);        // row_bcast 15: the row in front
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);        // row_bcast 31: the two rows in front
    return v;
}

struct PaSequence {
    int lo, hi, first, tiles;       // tokens that count, first tile, number of tiles
    bool over;
};
__device__ __forceinline__ PaSequence pa_sequence(const kmi_paged_attn_args& p, int len) {
    const long capacity = (long)p.max_pages * p.page_tiles * KV_TILE;
    PaSequence s;
    s.over = len > capacity;
    s.hi = s.over || len < 0 ? 0 : len;
    s.lo = p.window > 0 ? max(0, s.hi - p.window) : 0;
    s.first = s.lo / KV_TILE;
    s.tiles = (s.hi + KV_TILE - 1) / KV_TILE - s.first;
    return s;
}

template <bool V>
struct Flag {
    static constexpr bool value = V;
};

// The waves' sums, each relative to its own reference.
template <int D, int NW>
struct PaJoin {
    float m[NW][16], l[NW][16], add[NW][16];
    f4_t o[NW][D / 16][64];
};

// Slot of share v of a task that begins in share w0.
__device__ __forceinline__ size_t pa_slot(int w0, int v, int slot) { return ((size_t)(w0 + v) * 2 + (v == 0)) * slot; }

// n shares' sums to the task's outputs, by all 64 NW threads: four outputs a thread and share, the shares dealt over the threads that
// are left, their references and sums in LDS first.  One workgroup reads slowly past its caches (about 10 GB/s): all loads of a
// thread are in flight at once.
template <int D, int HT, int NW>
__device__ __forceinline__ void join_shares(const float* partial, int slot, int w0, int n, int used, half_t* out, float* lds, int room) {
    constexpr int COLS = 16 * HT, THREADS = 64 * NW, FLIGHT = 8;
    const int quads = used * D / 4;                              // groups of four outputs
    const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(partial), 0, -1, 0x00020000);
    const int most = room / 2 / (2 * COLS);                      // shares whose references fit half of the LDS at once
    float* held = lds;                                           // [share][column] reference, sum
    f4_t* outs = reinterpret_cast<f4_t*>(lds + room / 2);        // [dealt][quads] partial outputs
    const int dealt = max(1, min(min(THREADS / quads, n), room / 2 / (4 * quads)));
    for (int q0 = 0; q0 < quads; q0 += THREADS) {
        const int q = dealt > 1 ? threadIdx.x % quads : q0 + threadIdx.x, first = dealt > 1 ? threadIdx.x / quads : 0;
        const int c = min(4 * q / D, used - 1), at = c / 16 * (32 + 16 * D) + 32 + 4 * q - c / 16 * 16 * D;
        const bool mine = q < quads && first < dealt;
        float top = PA_NEG, sum = 0.0f;
        f4_t o = {};
        for (int v0 = 0; v0 < n; v0 += most) {
            const int here = min(most, n - v0);
            __syncthreads();
            for (int i = threadIdx.x; i < here * COLS; i += THREADS) {
                const int k = i % COLS;
                if (k >= used) continue;
                const float* s = partial + pa_slot(w0, v0 + i / COLS, slot) + k / 16 * (32 + 16 * D) + k % 16;
                held[2 * i] = __hip_atomic_load(s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                held[2 * i + 1] = __hip_atomic_load(s + 16, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
            __syncthreads();
            if (!mine) continue;
            for (int v = first; v < here; v += FLIGHT * dealt) {
                f4_t y[FLIGHT];
#pragma unroll
                for (int k = 0; k < FLIGHT; ++k) {              // 16 = sc1: performed at the memory side, as the stores were
                    const int share = v0 + min(v + k * dealt, here - 1);
                    y[k] = __builtin_bit_cast(f4_t, __builtin_amdgcn_raw_buffer_load_b128(rsrc, (int)((pa_slot(w0, share, slot) + at) * 4), 0, 16));
                }
                float next = top, m[FLIGHT];
#pragma unroll
                for (int k = 0; k < FLIGHT; ++k) {
                    m[k] = v + k * dealt < here ? held[2 * ((v + k * dealt) * COLS + c)] : PA_NEG;
                    next = fmaxf(next, m[k]);
                }
                const float keep = decay(top - next);
                sum *= keep; o = o * keep; top = next;
#pragma unroll
                for (int k = 0; k < FLIGHT; ++k) {
                    if (v + k * dealt >= here) continue;
                    const float f = decay(m[k] - next);
                    sum += f * held[2 * ((v + k * dealt) * COLS + c) + 1];
                    o = o + y[k] * f;
                }
            }
        }
        if (dealt > 1) {                                         // the threads that share an output, in order
            float* tops = held;                                  // [dealt][quads] reference, sum
            __syncthreads();
            if (mine) {
                outs[first * quads + q] = o;
                tops[2 * (first * quads + q)] = top;
                tops[2 * (first * quads + q) + 1] = sum;
            }
            __syncthreads();
            if (mine && first == 0) {
                for (int k = 1; k < dealt; ++k) {
                    const float m = tops[2 * (k * quads + q)], next = fmaxf(top, m);
                    const float keep = decay(top - next), f = decay(m - next);
                    sum = sum * keep + f * tops[2 * (k * quads + q) + 1];
                    o = o * keep + outs[k * quads + q] * f;
                    top = next;
                }
            }
        }
        if (mine && first == 0) {
            const float norm = 1.0f / sum;
            typedef _Float16 h4 __attribute__((ext_vector_type(4)));
            *reinterpret_cast<h4*>(out + 4 * q) = h4{(half_t)(o[0] * norm), (half_t)(o[1] * norm), (half_t)(o[2] * norm), (half_t)(o[3] * norm)};
        }
        if (dealt > 1) break;
    }
}

template <int D, int KIND, int PACK, int HT, int NW>
__global__ __launch_bounds__(64 * NW, NW * pa_a_cu(D, KIND, PACK, NW) / 4) void paged_attn_kernel(kmi_paged_attn_args p, PaSplit sp) {
    constexpr int MINE = D / 16 / NW > 0 ? D / 16 / NW : 1;         // MINE: output tiles that a wave joins
    using W = PaWave<D, KIND, PACK>;
    __shared__ PaJoin<D, NW> join;
    __shared__ int last;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, g = lane >> 4, col = lane & 15;
    const int G = p.H / p.KV, run = blockIdx.x;
    half_t* out0 = static_cast<half_t*>(p.out);

    __shared__ int held_lens[PA_HELD];
    const int lens0 = lane < p.B ? p.lens[lane] : 0;                       // of the first 64 sequences: most often all
    if (p.B > 64) {
        for (int b = threadIdx.x; b < min(p.B, PA_HELD); b += 64 * NW) held_lens[b] = p.lens[b];
        __syncthreads();
    }
    auto length = [&](int b) { return b < PA_HELD ? held_lens[b] : p.lens[b]; };
    auto tiles_of = [&](int b0) {                                          // of sequence b0 + lane
        const int b = b0 + lane;
        return b < p.B ? pa_sequence(p, b0 == 0 ? lens0 : length(b)).tiles : 0;
    };
    auto sum_over = [&](auto f) {                                          // over the sequences, f(tiles), times the tasks of one
        int v = 0;
        for (int b0 = 0; b0 < p.B; b0 += 64) v += __builtin_amdgcn_readlane(wave_scan(f(tiles_of(b0))), 63);
        return v * sp.tasks_a_sequence;
    };
    // One workgroup a CU where the shares come out even or are long, else as many as there are.
    const int units = sum_over([](int n) { return n; }), most = gridDim.x;
    auto quota_of = [&](int units, int shares) { return (max((units + shares - 1) / shares, PA_MIN_STEPS * NW) + NW - 1) / NW * NW; };
    auto pieces_of = [](int n, int q) { return n <= PA_WHOLE_STEPS * NW ? (n > 0 ? 1 : 0) : (n + q - 1) / q; };
    auto pieces = [&](int q) { return sum_over([&](int n) { return pieces_of(n, q); }); };
    int shares = NW == 2 || (KIND == KMI_KV_INT4 && NW == 4) ? most : min(most, 256), quota = quota_of(units, shares);
    bool even = pieces(quota) <= shares;
    for (int pass = 0; !even; ++pass) {
        const int more = (quota + quota / 8 + NW - 1) / NW * NW;
        even = pieces(more) <= shares;
        if (even) {
            quota = more;
        } else if (pass == 1 || quota >= PA_LONG || shares == most) {
            quota = quota_of(sum_over([](int n) { return n ? n + PA_TASK_COST : 0; }), shares);
            break;
        } else {
            shares = most;
            quota = quota_of(units, shares);
            even = pieces(quota) <= shares;
        }
    }
    // the row that the shares are cut from: pieces, one a share, or tiles and PA_TASK_COST a task, `quota` a share
    auto room = [&](int n) { return n == 0 ? 0 : even ? pieces_of(n, quota) : n + PA_TASK_COST; };     // a task's, in the row
    constexpr int SMALL = PA_WHOLE_STEPS * NW < PA_SMALL_BYTES / W::TILE_BYTES ? PA_WHOLE_STEPS * NW : PA_SMALL_BYTES / W::TILE_BYTES;
    // (workgroups past the last share own nothing: a multiple of their number would pass 2^31 where the row holds over 2^30 tiles)
    const int per_share = even ? 1 : quota, begin = min(run, shares) * per_share, end = run < shares ? begin + per_share : begin;
    int b = p.B, before = 0;                                               // before: the room of the sequences in front
    for (int b0 = 0; b0 < p.B; b0 += 64) {
        const int mine = room(tiles_of(b0)) * sp.tasks_a_sequence, upto = wave_scan(mine);
        const uint64_t behind = __ballot(before + upto > begin);
        if (behind) {
            const int at = __builtin_ctzll(behind);
            b = b0 + at;
            before += __builtin_amdgcn_readlane(upto, at) - __builtin_amdgcn_readlane(mine, at);
            break;
        }
        before += __builtin_amdgcn_readlane(upto, 63);
    }
    auto len_of = [&](int b) { return b < 64 ? __builtin_amdgcn_readlane(lens0, b & 63) : __builtin_amdgcn_readfirstlane(length(b)); };

    for (int unit = begin; unit < end && b < p.B;) {
        const PaSequence seq = pa_sequence(p, len_of(b));
        const int space = room(seq.tiles);
        if (unit >= before + space * sp.tasks_a_sequence) {
            before += space * sp.tasks_a_sequence;
            ++b;
            continue;
        }
        const int task = (unit - before) / space, task0 = before + task * space;
        int ta = unit - task0, tb, first_share = run, parts = 1;           // the share's tiles of the task; the task's shares
        if (even) {
            first_share = task0;
            parts = space;
            tb = (int)((long)(ta + 1) * seq.tiles / space);
            ta = (int)((long)ta * seq.tiles / space);
            unit = end;
        } else if (seq.tiles <= SMALL) {
            const int middle = task0 + space / 2;
            unit = task0 + space;
            if (middle < begin || middle >= end) continue;
            ta = 0;
            tb = seq.tiles;
        } else {
            tb = min(seq.tiles, end - task0);
            unit = task0 + min(space, end - task0);
            if (ta >= tb) continue;
            first_share = task0 / quota;
            parts = (task0 + seq.tiles - 1) / quota - first_share + 1;
        }
        const int head = task / sp.head_tiles, h0 = (task - head * sp.head_tiles) * 16 * HT, used = min(16 * HT, G - h0);

        W w[HT];
#pragma unroll
        for (int x = 0; x < HT; ++x) {
            const int hcol = (PACK == 2 ? col & 7 : col) + 16 * x;         // the column's query head
            w[x].load_q(static_cast<const half_t*>(p.q) + b * p.q_batch + (size_t)(head * G + h0 + min(hcol, used - 1)) * D, hcol < used, g);
        }
        // this wave's tiles: ta + wave + NW i; their places in the pool: 64 at a time, one a lane
        const int count = (tb - ta - wave + NW - 1) / NW;
        const char* cache = static_cast<const char*>(p.cache);
        int places = -1;
        auto place_of = [&](int i) {
            if ((i & 63) == 0) {
                const int t = seq.first + min(ta + (i + lane) * NW + wave, tb - 1), page = t / p.page_tiles;
                const int id = p.page_table[(size_t)b * p.max_pages + page];
                places = id >= 0 && id < p.num_pages ? (id * p.KV + head) * p.page_tiles + t - page * p.page_tiles : -1;
            }
            return __builtin_amdgcn_readlane(places, i & 63);
        };
        // the registers of a tile's keys, then of its values, are loaded for the next tile as soon as they are used up
        typename W::Tile tile;
        int place = 0;
        auto fetch_keys = [&](int i) {
            place = place_of(i);
            W::load_keys(tile, cache + (size_t)max(place, 0) * W::TILE_BYTES, lane);
        };
        auto fetch_values = [&]() { W::load_values(tile, cache + (size_t)max(place, 0) * W::TILE_BYTES, lane); };
        if (count > 0) {
            fetch_keys(0);
            fetch_values();
        }
#pragma unroll
        for (int x = 0; x < HT; ++x) w[x].start(col, sp.c);
        // (a load under a condition would make the compiler wait for every load wherever it waits for one)
        auto step = [&](auto more, auto careful, int i) {
            typename W::Scores sc[HT];
#pragma unroll
            for (int x = 0; x < HT; ++x) sc[x] = w[x].scores(tile, lane);
            typename W::Factors fac = tile.f;
            const bool bad = place < 0;
            if constexpr (more.value) fetch_keys(i + 1);
            __builtin_amdgcn_sched_barrier(0);
            typename W::Weights o[HT];
#pragma unroll
            for (int x = 0; x < HT; ++x)
                o[x] = w[x].template weights<careful.value>(sc[x], tile, fac, (seq.first + ta + wave + NW * i) * KV_TILE, seq.lo, seq.hi, bad, lane);
            __builtin_amdgcn_sched_barrier(0);                 // values are decoded where they are used: not before, into registers
#pragma unroll
            for (int x = 0; x < HT; ++x) w[x].template add<careful.value>(tile, o[x]);
            if constexpr (more.value) fetch_values();
            __builtin_amdgcn_sched_barrier(0);
        };
        int i = 0;
        for (; i + 1 < count; ++i) step(Flag<true>(), Flag<false>(), i);
        if (i < count) step(Flag<false>(), Flag<false>(), i);
        if constexpr (!W::CODES) {
            // f16: infinities or NaN among the values.  The wave's tiles once more, carefully: two packed instructions for two values, which
            // one wave a SIMD does not hide (1 x 1152 11.4 us for 10.2 if all tiles were taken so), and no loads ahead.
            bool again = false;
#pragma unroll
            for (int x = 0; x < HT; ++x) again |= w[x].not_finite();
            if (again) {
#pragma unroll
                for (int x = 0; x < HT; ++x) w[x].start(col, sp.c);
                for (i = 0; i < count; ++i) {
                    fetch_keys(i);
                    fetch_values();
                    step(Flag<false>(), Flag<true>(), i);
                }
            }
        }

        // the waves' sums, joined
        const bool complete = parts == 1;
        float* slot = sp.partial + ((size_t)run * 2 + (ta == 0)) * sp.slot;
        half_t* out = out0 + ((size_t)b * p.H + head * G + h0) * D;
#pragma unroll
        for (int x = 0; x < HT; ++x) {
            if (x > 0) __syncthreads();                        // the arrays are written again
            float sum, add;
            w[x].totals(sum, add);
            if (g == 0) { join.m[wave][col] = w[x].m; join.l[wave][col] = sum; join.add[wave][col] = add; }
#pragma unroll
            for (int T = 0; T < W::OT; ++T) join.o[wave][T][lane] = w[x].acc[T];
            __syncthreads();
            float mm = PA_NEG, ll = 0.0f, plus = 0.0f, a[NW];
#pragma unroll
            for (int v = 0; v < NW; ++v) mm = fmaxf(mm, join.m[v][col]);
            if constexpr (PACK == 2) mm = fmaxf(mm, W::other_half(mm));
#pragma unroll
            for (int v = 0; v < NW; ++v) {
                a[v] = decay(join.m[v][col] - mm);
                ll += a[v] * join.l[v][col];
                plus += a[v] * join.add[v][col];
            }
            if constexpr (PACK == 2) { ll += W::other_half(ll); plus += W::other_half(plus); }
            const float norm = 1.0f / ll;                      // 0 / 0 = NaN where every score is -inf
            float* part = slot + x * (32 + 16 * D);
            if (wave * MINE < W::OT) {
#pragma unroll
                for (int i = 0; i < MINE; ++i) {
                    const int T = wave * MINE + i;
                    f4_t o = {};
#pragma unroll
                    for (int v = 0; v < NW; ++v) o = o + join.o[v][T][lane] * a[v];
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        float y = o[r];
                        if constexpr (PACK == 2) y += W::other_half(y);
                        if constexpr (W::CODES) y = __builtin_fmaf(y, W::UNIT, plus);
                        if ((PACK == 2 && col >= 8) || col + 16 * x >= used) continue;
                        const int d = W::d_of(T, 4 * g + r);
                        if (complete) out[(size_t)(col + 16 * x) * D + d] = (half_t)(y * norm);
                        else __hip_atomic_store(part + 32 + col * D + d, y, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                    }
                }
                if (!complete && wave == 0 && g == 0 && col + 16 * x < used && !(PACK == 2 && col >= 8)) {
                    __hip_atomic_store(part + col, mm, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                    __hip_atomic_store(part + 16 + col, ll, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                }
            }
        }
        if (!complete) {
            // Hand-off without fences: partial sums travel by agent-scope stores and loads, performed at the memory side; every
            // thread waits for its own to be performed, the barrier for every thread, and only then the arrival is counted there.
            const int w0 = first_share, n = parts;
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            if (threadIdx.x == 0) last = __hip_atomic_fetch_add(sp.counters + w0, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)(n - 1);
            __syncthreads();
            if (last) {
                join_shares<D, HT, NW>(sp.partial, sp.slot, w0, n, used, out, reinterpret_cast<float*>(join.o), sizeof(join.o) / sizeof(float));
                if (threadIdx.x == 0) __hip_atomic_store(sp.counters + w0, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);     // for the next call
            }
        }
        __syncthreads();                                       // the next task writes the shared arrays again
    }

    // sequences without a tile: zeros, or NaN where the length does not fit the page table
    for (int b = run; b < p.B; b += gridDim.x) {
        const PaSequence s = pa_sequence(p, len_of(b));
        if (s.tiles) continue;
        const uint32_t fill = s.over ? 0x7E007E00u : 0u;
        u4_t* o = reinterpret_cast<u4_t*>(out0 + (size_t)b * p.H * D);
        for (int i = threadIdx.x; i < p.H * D / 8; i += 64 * NW) o[i] = u4_t{fill, fill, fill, fill};
    }
}

int kv_check_cache(const char* fn, const void* cache, const void* page_table, int B, int KV, int D, int kind, int num_pages,
                   int page_tiles, int max_pages);

extern "C" int kmi_paged_attn(const kmi_paged_attn_args* args, void* stream) {
    const char* fn = "kmi_paged_attn";
    if (!args) return kmi_set_error(KMI_E_NULL, "%s: args is NULL", fn);
    const kmi_paged_attn_args& p = *args;
    if (!p.out || !p.q || !p.lens) return kmi_set_error(KMI_E_NULL, "%s: out, q and lens must not be NULL", fn);
    if (!kmi_aligned16(p.out) || !kmi_aligned16(p.q) || !kmi_aligned16(p.workspace) || (p.q_batch & 7))
        return kmi_set_error(KMI_E_ALIGN, "%s: out, q and the workspace must be 16-byte aligned, q's stride a multiple of 8 elements", fn);
    const int rc = kv_check_cache(fn, p.cache, p.page_table, p.B, p.KV, p.D, p.kind, p.num_pages, p.page_tiles, p.max_pages);
    if (rc < 0) return rc;
    if (p.H <= 0 || p.H % p.KV || p.H > 65535 || p.window < 0 || !(p.scale > 0.0f) || !(p.scale < 1e16f))
        return kmi_set_error(KMI_E_SHAPE, "%s: need H a multiple of KV, window>=0 and 0<scale<1e16, which no score leaves fp32 with (H=%d KV=%d window=%d scale=%g)",
                             fn, p.H, p.KV, p.window, (double)p.scale);
    if (p.B == 0) return KMI_OK;
    const long long pool = (long long)p.B * p.KV * p.max_pages * p.page_tiles;
    const int G = p.H / p.KV, columns = G > 16 && p.D < 256 && p.kind != KMI_KV_INT4 && pool >= PA_WIDE ? 32 : 16, used = G < columns ? G : columns;
    PaSplit sp;
    sp.head_tiles = (G + columns - 1) / columns;
    sp.tasks_a_sequence = p.KV * sp.head_tiles;
    sp.c = p.scale * 1.44269504088896340736f;
    sp.slot = used > 16 ? 2 * (32 + 16 * p.D) : 32 + used * p.D;
    sp.counters = static_cast<uint32_t*>(p.workspace);
    sp.partial = reinterpret_cast<float*>(static_cast<char*>(p.workspace) + KMI_GEMV_WS_HEADER);
    // as many workgroups as the kernel may want, never more than the tasks can be cut into
    const long long most = (long long)p.B * sp.tasks_a_sequence * ((long long)p.max_pages * p.page_tiles + PA_TASK_COST);
    if (most > 0x7FFF0000ll)
        return kmi_set_error(KMI_E_SHAPE, "%s: %d sequences of %d pages hold more than 2^31 tiles", fn, p.B, p.max_pages);
    const long long pieces = (long long)p.B * sp.tasks_a_sequence * (((long long)p.max_pages * p.page_tiles + 7) / 8);
    const int pack = G > 8 || p.kind == KMI_KV_F16 ? 1 : 2, waves = pa_waves(p.D, p.kind, pack, columns, (long long)p.B * sp.tasks_a_sequence);
    const int most_runs = 256 * pa_a_cu(p.D, p.kind, pack, waves), runs = (int)(pieces < most_runs ? pieces : most_runs);
    const size_t need = KMI_GEMV_WS_HEADER + (size_t)most_runs * 2 * sp.slot * sizeof(float);
    if (!p.workspace || p.workspace_bytes < need)
        return kmi_set_error(KMI_E_SHAPE, "%s: the workspace must hold %zu bytes (has %zu)", fn, need, p.workspace ? (size_t)p.workspace_bytes : (size_t)0);
    const dim3 grid(runs), block(waves * 64);
    hipStream_t st = static_cast<hipStream_t>(stream);
#define KMI_PA(D_, K_, PACK_, HT_, NW_) hipLaunchKernelGGL((paged_attn_kernel<D_, K_, PACK_, HT_, NW_>), grid, block, 0, st, p, sp)
#define KMI_PA_WAVES(D_, K_, PACK_, NW_)                                             \
    if (D_ < 256 && waves == 2) KMI_PA(D_, K_, PACK_, 1, D_ == 256 ? NW_ : 2);       \
    else KMI_PA(D_, K_, PACK_, 1, NW_)
#define KMI_PA_WIDE(D_, K_) if (D_ < 256 && columns == 32) KMI_PA(D_, K_, 1, D_ == 256 ? 1 : 2, D_ == 256 ? 4 : 8)
#define KMI_PA_F16(D_)                                             \
    KMI_PA_WIDE(D_, KMI_KV_F16);                                   \
    else KMI_PA_WAVES(D_, KMI_KV_F16, 1, 4)
#define KMI_PA_INT8(D_)                                            \
    KMI_PA_WIDE(D_, KMI_KV_INT8);                                  \
    else if (pack == 1) { KMI_PA_WAVES(D_, KMI_KV_INT8, 1, 4); }   \
    else KMI_PA_WAVES(D_, KMI_KV_INT8, 2, D_ == 64 ? 8 : 4)
#define KMI_PA_INT4(D_)                                                                   \
    if (pack == 1 && waves == 8) KMI_PA(D_, KMI_KV_INT4, 1, 1, 8);                        \
    else if (pack == 1) { KMI_PA_WAVES(D_, KMI_KV_INT4, 1, D_ == 256 ? 8 : 4); }          \
    else if (waves == 8) KMI_PA(D_, KMI_KV_INT4, 2, 1, 8);                                \
    else KMI_PA_WAVES(D_, KMI_KV_INT4, 2, D_ == 128 ? 4 : 8)
#define KMI_PA_LAUNCH(D_)                                  \
    switch (p.kind) {                                      \
        case KMI_KV_F16: KMI_PA_F16(D_); break;            \
        case KMI_KV_INT8: KMI_PA_INT8(D_); break;          \
        default: KMI_PA_INT4(D_);                          \
    }
    if (p.D == 64) { KMI_PA_LAUNCH(64) }
    else if (p.D == 128) { KMI_PA_LAUNCH(128) }
    else { KMI_PA_LAUNCH(256) }
#undef KMI_PA_LAUNCH
#undef KMI_PA_INT4
#undef KMI_PA_INT8
#undef KMI_PA_F16
#undef KMI_PA_WIDE
#undef KMI_PA_WAVES
#undef KMI_PA
    return kmi_check_launch(fn);
}
