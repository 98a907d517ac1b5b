// Rotary positions, the cache's writer (fused with them) and its reader.
//
// Rotation, per pair (a, b) of a head's first R elements -- (i, i + R/2) or (2i, 2i + 1) -- with the table's fp32 cosine and
// sine of the token's position (products and sums rounded one by one in fp32, the result once to fp16):
//   a' = a cos - b sin,   b' = b cos + a sin
// Quantisation of a row x (one token of one key or value head), per kind:
//   int8  s = up(max|x| / 127, 127), u = rint(x * (1 / s)) + 128          stands for s * (u - 128)
//   int4  z = min x, s = up((max x - z) / 15, 15), u = rint((x - z) * (1 / s))   stands for s * u + z
// up(s, n): s rounded to fp16, one fp16 step up where n * s would fall short of the row's width, so that no element of a
// tiny row (subnormal s) is clipped.  The quotients and the reciprocal are IEEE divisions, every step is rounded to fp32
// once: the codes are the same on any machine.  A row with an infinity or NaN gets the scale NaN and reads as NaN.
// Traffic: every row read once and written once, plus the table's R * 4 bytes a token; bound by the memory.  Measured: rotation
// alone, 4 x 4001 tokens, 28 + 4 heads of 128: 51 us for 263 MB, 5.2 TB/s (a large copy: 5.0); into the cache, 32 x 1024 tokens, 32 + 8 + 8
// heads of 128: int4 164 us (155 at best) for 707 MB, 4.3 TB/s; 3 x 777 tokens, 64 + 8 + 8 heads, f16: 23 us for 96 MB, 4.2 TB/s; one token of
// 32 sequences: 4 us.
#include "kv_parts.h"
#include <type_traits>

struct RowFactors {
    half_t s, z;
    float r;                       // 1 / s, 0 for a row of equal elements
};

__device__ __forceinline__ half_t scale_up(float width, float steps) {
    half_t s = (half_t)(width / steps);
    if ((float)s * steps < width) s = __builtin_bit_cast(half_t, (uint16_t)(__builtin_bit_cast(uint16_t, s) + 1));
    return s;
}

typedef uint16_t us2_t __attribute__((ext_vector_type(2)));

// v joined by f over LPR neighbouring lanes (4, 8 or 16), in all of them.
template <int LPR, typename T, typename F>
__device__ __forceinline__ T over_row(T v, F f) {
    auto step = [&](auto ctrl) {
        const int o = __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), ctrl.value, 0xF, 0xF, false);
        v = f(v, __builtin_bit_cast(T, o));
    };
    step(std::integral_constant<int, 0xB1>());                 // quad_perm 1 0 3 2
    step(std::integral_constant<int, 0x4E>());                 // quad_perm 2 3 0 1
    if constexpr (LPR >= 8) step(std::integral_constant<int, 0x141>());       // row_half_mirror: the other four of eight
    if constexpr (LPR >= 16) step(std::integral_constant<int, 0x140>());      // row_mirror: the other eight of sixteen
    return v;
}

// Factors of a row spread over LPR neighbouring lanes, two chunks of eight elements each.
template <int LPR, int KIND>
__device__ __forceinline__ RowFactors row_factors(h8_t a, h8_t b) {
#pragma clang fp contract(off)
    RowFactors f = {};
    if constexpr (KIND == KMI_KV_F16) return f;
    const u4_t wa = __builtin_bit_cast(u4_t, a), wb = __builtin_bit_cast(u4_t, b);
    us2_t top = {};                                     // largest |x| as bits: orders infinities and NaN above all
    h2_t lo = as_h2(wa[0]), hi = lo;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t w = i < 4 ? wa[i & 3] : wb[i & 3];
        top = __builtin_elementwise_max(top, __builtin_bit_cast(us2_t, w & 0x7FFF7FFFu));
        if constexpr (KIND == KMI_KV_INT4) {
            lo = __builtin_elementwise_min(lo, as_h2(w));
            hi = __builtin_elementwise_max(hi, as_h2(w));
        }
    }
    top = over_row<LPR>(top, [](us2_t x, us2_t y) { return __builtin_elementwise_max(x, y); });
    const uint16_t most = top[0] > top[1] ? top[0] : top[1];
    if constexpr (KIND == KMI_KV_INT8) {
        f.s = scale_up((float)__builtin_bit_cast(half_t, most), 127.0f);
    } else {
        const half_t l = lo[0] < lo[1] ? lo[0] : lo[1], h = hi[0] > hi[1] ? hi[0] : hi[1];
        h2_t ends = {l, -h};
        ends = over_row<LPR>(ends, [](h2_t x, h2_t y) { return __builtin_elementwise_min(x, y); });
        const float flo = (float)ends[0] + 0.0f;        // never -0: which of two zeros is the smallest is left open
        f.z = (half_t)flo;
        f.s = scale_up(-(float)ends[1] - flo, 15.0f);
    }
    if (most >= 0x7C00) f.s = __builtin_bit_cast(half_t, (uint16_t)0x7E00);
    f.r = (float)f.s > 0.0f ? 1.0f / (float)f.s : 0.0f;
    return f;
}

// Eight elements of a row as the cache holds them: elements, or codes (bytes; nibbles), in order.  NPW = 32-bit words.
// A code is rounded by adding 1.5 * 2^23 (+ 128): its bits are then the low ones of the sum, the others a constant that is taken
// off the packed word once.  up() leaves no code outside its range, so nothing is clamped.
template <int KIND>
struct Packed {
    static constexpr int NPW = 4 / kv_per_word(KIND);
    uint32_t w[NPW];
};
template <int KIND>
__device__ __forceinline__ Packed<KIND> pack_row(h8_t x, const RowFactors& f) {
#pragma clang fp contract(off)
    Packed<KIND> o;
    if constexpr (KIND == KMI_KV_F16) {
        const u4_t w = __builtin_bit_cast(u4_t, x);
#pragma unroll
        for (int i = 0; i < 4; ++i) o.w[i] = w[i];
    } else {
        constexpr int bits = KIND == KMI_KV_INT8 ? 8 : 4, per = 32 / bits;
        constexpr uint32_t base = 0x4B400000u;          // of 1.5 * 2^23
#pragma unroll
        for (int i = 0; i < Packed<KIND>::NPW; ++i) {
            uint32_t w = 0;
#pragma unroll
            for (int e = 0; e < per; ++e) {
                const float v = KIND == KMI_KV_INT8 ? (float)x[per * i + e] * f.r + 12583040.0f
                                                    : ((float)x[per * i + e] - (float)f.z) * f.r + 12582912.0f;
                w += (__builtin_bit_cast(uint32_t, v)) << (bits * e);
            }
            uint32_t off = 0;
#pragma unroll
            for (int e = 0; e < per; ++e) off += base << (bits * e);
            o.w[i] = w - off;
        }
    }
    return o;
}
// Four items of four lanes (a quad) turned over: item i of lane k becomes item k of lane i.
template <typename T>
__device__ __forceinline__ void turn_quad(T (&x)[4], int lane) {
    constexpr int N = sizeof(T) / 4;
    struct Words {
        uint32_t w[N];
    };
    Words v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __builtin_bit_cast(Words, x[i]);
    auto swap = [&](auto ctrl, int i, int j, bool upper) {     // item j of the lower lanes with item i of the upper ones
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const uint32_t give = upper ? v[i].w[n] : v[j].w[n];
            const uint32_t got = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)give, ctrl.value, 0xF, 0xF, false);
            v[i].w[n] = upper ? got : v[i].w[n];
            v[j].w[n] = upper ? v[j].w[n] : got;
        }
    };
    const bool odd = lane & 1, high = lane & 2;
    swap(std::integral_constant<int, 0xB1>(), 0, 1, odd);
    swap(std::integral_constant<int, 0xB1>(), 2, 3, odd);
    swap(std::integral_constant<int, 0x4E>(), 0, 2, high);
    swap(std::integral_constant<int, 0x4E>(), 1, 3, high);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __builtin_bit_cast(T, v[i]);
}
// Nibble e of a key unit stands at place e / 2 + 4 (e % 2): even elements in the low half, odd ones in the high.
__device__ __forceinline__ uint32_t nibbles_apart(uint32_t w) {
    uint32_t e = w & 0x0F0F0F0Fu, o = (w >> 4) & 0x0F0F0F0Fu;
    e = (e | e >> 4) & 0x00FF00FFu; e = (e | e >> 8) & 0xFFFFu;
    o = (o | o >> 4) & 0x00FF00FFu; o = (o | o >> 8) & 0xFFFFu;
    return e | o << 16;
}
__device__ __forceinline__ uint32_t nibbles_together(uint32_t w) {
    uint32_t e = w & 0xFFFFu, o = w >> 16;
    e = (e | e << 8) & 0x00FF00FFu; e = (e | e << 4) & 0x0F0F0F0Fu;
    o = (o | o << 8) & 0x00FF00FFu; o = (o | o << 4) & 0x0F0F0F0Fu;
    return e | o << 4;
}

template <int D, int KIND>
__device__ __forceinline__ void store_factors(char* tile, int tau, int first, const RowFactors& f) {
    if constexpr (KIND != KMI_KV_F16) *reinterpret_cast<half_t*>(tile + kv_factor_offset<D, KIND>(tau, first)) = f.s;
    if constexpr (KIND == KMI_KV_INT4) *reinterpret_cast<half_t*>(tile + kv_factor_offset<D, KIND>(tau, first + 1)) = f.z;
}

template <int D, int KIND>
__device__ __forceinline__ void store_key(char* tile, int tau, int d0, const Packed<KIND>& w) {
    char* at = tile + kv_key_offset<D, KIND>(tau, d0);
    if constexpr (KIND == KMI_KV_F16) *reinterpret_cast<u4_t*>(at) = u4_t{w.w[0], w.w[1], w.w[2], w.w[3]};
    else if constexpr (KIND == KMI_KV_INT8) *reinterpret_cast<u2_t*>(at) = u2_t{w.w[0], w.w[1]};
    else *reinterpret_cast<uint32_t*>(at) = nibbles_apart(w.w[0]);
}

// One token's value: its words stand 16 bytes apart.
template <int D, int KIND>
__device__ __forceinline__ void store_value(char* tile, int tau, int d0, const Packed<KIND>& w) {
    constexpr int n = kv_per_word(KIND);
#pragma unroll
    for (int i = 0; i < 8 / n; ++i)
        *reinterpret_cast<uint16_t*>(tile + kv_value_offset<D, KIND>(tau, d0 + n * i)) = (uint16_t)(w.w[i / 2] >> (16 * (i & 1)));
}
// Eight tokens tau0 .. tau0 + 7 (tau0 % 8 == 0): whole 16-byte chunks, 128 / n bytes in a row; d0s: the quad's lanes' d0.
// f16 and int8: four chunks of a quad at a time change hands, so that a store writes 64 bytes in a row instead of 16.
template <int D, int KIND>
__device__ __forceinline__ void store_values8(char* tile, int tau0, const int (&d0s)[4], int lane, const Packed<KIND> (&w)[8]) {
    constexpr int n = kv_per_word(KIND), CHUNKS = 8 / n;
    u4_t c[CHUNKS];
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) c[i][j] = __builtin_amdgcn_perm(w[2 * j + 1].w[i / 2], w[2 * j].w[i / 2], i & 1 ? 0x07060302u : 0x05040100u);
    if constexpr (CHUNKS >= 4) {
#pragma unroll
        for (int q = 0; q < CHUNKS / 4; ++q) {
            u4_t x[4] = {c[4 * q], c[4 * q + 1], c[4 * q + 2], c[4 * q + 3]};
            turn_quad(x, lane);
#pragma unroll
            for (int k = 0; k < 4; ++k) reinterpret_cast<u4_t*>(tile + kv_value_offset<D, KIND>(tau0, d0s[k]))[4 * q + (lane & 3)] = x[k];
        }
    } else {
        const int d0 = lane & 2 ? (lane & 1 ? d0s[3] : d0s[2]) : (lane & 1 ? d0s[1] : d0s[0]);
        u4_t* at = reinterpret_cast<u4_t*>(tile + kv_value_offset<D, KIND>(tau0, d0));
#pragma unroll
        for (int i = 0; i < CHUNKS; ++i) at[i] = c[i];
    }
}
// The same of keys: tokens tau0 + 4 h .. + 3 of a unit lie behind each other, 16 bytes apart, so four units of a quad change hands.
template <int D, int KIND>
__device__ __forceinline__ void store_keys8(char* tile, int tau0, const int (&d0s)[4], int lane, const Packed<KIND> (&w)[8]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        Packed<KIND> x[4] = {w[4 * h], w[4 * h + 1], w[4 * h + 2], w[4 * h + 3]};
        turn_quad(x, lane);
#pragma unroll
        for (int k = 0; k < 4; ++k) store_key<D, KIND>(tile, tau0 + 4 * h + (lane & 3), d0s[k], x[k]);
    }
}

// A lane has two chunks of eight elements of a row, at da and db.  Half layout: in the turned part da and db = da + R/2 are
// partners, element by element; interleaved: they are neighbours.  Behind the turned part they are neighbours.
template <bool INTERLEAVED>
struct Chunks {
    int da, db;
    bool turned;
    int pair0;                                                  // first of the lane's eight pairs
    __device__ __forceinline__ Chunks(int c, int R) {
        turned = 16 * c < R;
        da = !INTERLEAVED && turned ? 8 * c : 16 * c;
        db = !INTERLEAVED && turned ? 8 * c + R / 2 : 16 * c + 8;
        pair0 = 8 * c;
    }
};

// Turns a lane's two chunks by the angles of a position (NaN beyond the table).
template <bool INTERLEAVED>
__device__ __forceinline__ void turn(h8_t& a, h8_t& b, const float* table, int rows, int R, int pos, const Chunks<INTERLEAVED>& at) {
#pragma clang fp contract(off)
    if (!at.turned) return;
    const bool inside = pos >= 0 && pos < rows;
    const f4_t* p = reinterpret_cast<const f4_t*>(table + (size_t)(inside ? pos : 0) * R + 2 * at.pair0);
    f4_t cs[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) cs[i] = p[i];
    if (!inside) {
        const float nan = __builtin_nanf("");
#pragma unroll
        for (int i = 0; i < 4; ++i) cs[i] = f4_t{nan, nan, nan, nan};
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float c = cs[i / 2][2 * (i & 1)], s = cs[i / 2][2 * (i & 1) + 1];
        const float x = INTERLEAVED ? (float)(i < 4 ? a[2 * i & 7] : b[2 * i & 7]) : (float)a[i];
        const float y = INTERLEAVED ? (float)(i < 4 ? a[(2 * i + 1) & 7] : b[(2 * i + 1) & 7]) : (float)b[i];
        const half_t u = (half_t)(x * c - y * s), v = (half_t)(y * c + x * s);
        if constexpr (INTERLEAVED) {
            if (i < 4) { a[2 * i & 7] = u; a[(2 * i + 1) & 7] = v; }
            else { b[2 * i & 7] = u; b[(2 * i + 1) & 7] = v; }
        } else {
            a[i] = u; b[i] = v;
        }
    }
}

// One workgroup: eight neighbouring positions 8 i .. 8 i + 7 of one sequence, 4096 / D rows (heads of queries, keys or values) of each;
// a lane has sixteen elements of one row, both halves of its pairs.  Where all eight tokens are there, all loads are in flight
// before the first use, and the values leave as whole chunks of the cache, turned over in registers.  (One token a lane group, values
// stored by 16-bit words: 83 us for 3 x 777 f16 with its reading back, 30 so; 32 x 1024 int4 253 us, 190 so.)
template <int D, int KIND, bool INTERLEAVED>
__global__ __launch_bounds__(256) void rope_kv_kernel(kmi_rope_kv_args p) {
    constexpr int LPR = D / 16, ROWS = 256 / LPR, K_ = KIND < 0 ? 0 : KIND;
    const int b = blockIdx.y, R = p.rotary_dim, c = threadIdx.x % LPR;
    const int r = (p.q ? 0 : p.H) + blockIdx.z * ROWS + threadIdx.x / LPR;
    if (r >= p.H + p.KV + (KIND >= 0 ? p.KV : 0)) return;
    const bool is_q = r < p.H, is_v = r >= p.H + p.KV;
    const int head = is_q ? r : is_v ? r - p.H - p.KV : r - p.H;
    const int start = p.start[b], count = p.count ? max(0, min(p.count[b], p.S)) : p.S;
    const int pos0 = (int)((unsigned)((start >> 3) + (int)blockIdx.x) << 3), s0 = (int)((unsigned)pos0 - (unsigned)start);
    if (s0 >= p.S) return;

    const Chunks<INTERLEAVED> at(c, R);
    int das[4], dbs[4];                                         // of the quad's lanes
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const Chunks<INTERLEAVED> o((c & ~3) + k, R);
        das[k] = o.da; dbs[k] = o.db;
    }
    const int heads = is_q ? p.H : p.KV;
    const half_t* row = is_q ? static_cast<const half_t*>(p.q) + b * p.q_batch : is_v ? static_cast<const half_t*>(p.v) + b * p.v_batch
                                                                                     : static_cast<const half_t*>(p.k) + b * p.k_batch;
    const int64_t step = is_q ? p.q_token : is_v ? p.v_token : p.k_token;
    row += (size_t)head * D;
    half_t* out = static_cast<half_t*>(is_q ? p.q_out : is_v ? nullptr : p.k_out);
    if (out) out += ((size_t)b * p.S * heads + head) * D;
    const size_t out_step = (size_t)heads * D;
    const KvPlace place = {static_cast<char*>(p.cache), p.page_table, p.num_pages, p.page_tiles, p.max_pages, p.KV};
    char* tile = nullptr;                                       // the eight positions lie in one tile
    if constexpr (KIND >= 0) tile = is_q || pos0 < 0 ? nullptr : kv_tile_at<kv_tile_bytes(D, K_)>(place, b, head, pos0 / KV_TILE);
    const int tau0 = pos0 & (KV_TILE - 1);
    const float* table = static_cast<const float*>(p.table);
    auto load = [&](int s, int d) { return *reinterpret_cast<const h8_t*>(row + s * step + d); };
    auto store = [&](int s, int d, h8_t x) { *reinterpret_cast<h8_t*>(out + s * out_step + d) = x; };

    if (s0 >= 0 && s0 + 8 <= count) {
        h8_t xa[8], xb[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) { xa[j] = load(s0 + j, at.da); xb[j] = load(s0 + j, at.db); }
        if (is_v) {
            if constexpr (KIND >= 0) {
                if (!tile) return;
                Packed<K_> wa[8], wb[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const RowFactors f = row_factors<LPR, K_>(xa[j], xb[j]);
                    wa[j] = pack_row<K_>(xa[j], f);
                    wb[j] = pack_row<K_>(xb[j], f);
                    if (c == 0) store_factors<D, K_>(tile, tau0 + j, kv_factors(K_) / 2, f);
                }
                store_values8<D, K_>(tile, tau0, das, c, wa);
                store_values8<D, K_>(tile, tau0, dbs, c, wb);
            }
            return;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            turn(xa[j], xb[j], table, p.table_rows, R, pos0 + j, at);
            if (out) { store(s0 + j, at.da, xa[j]); store(s0 + j, at.db, xb[j]); }
        }
        if constexpr (KIND >= 0) {
            if (!tile) return;
            Packed<K_> wa[8], wb[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const RowFactors f = row_factors<LPR, K_>(xa[j], xb[j]);
                wa[j] = pack_row<K_>(xa[j], f);
                wb[j] = pack_row<K_>(xb[j], f);
                if (c == 0) store_factors<D, K_>(tile, tau0 + j, 0, f);
            }
            store_keys8<D, K_>(tile, tau0, das, c, wa);
            store_keys8<D, K_>(tile, tau0, dbs, c, wb);
        }
        return;
    }
    const int lo = max(0, -s0), hi = min(8, count - s0);       // the tokens that are there
    if (out) {
        for (int j = max(lo, hi); j < 8 && s0 + j < p.S; ++j) { // rows behind the sequence: zeros out, nothing into the cache
            store(s0 + j, at.da, h8_t{});
            store(s0 + j, at.db, h8_t{});
        }
    }
    auto put = [&](int j, h8_t xa, h8_t xb) {
        if (out) { store(s0 + j, at.da, xa); store(s0 + j, at.db, xb); }
        if constexpr (KIND >= 0) {
            if (!tile) return;
            const RowFactors f = row_factors<LPR, K_>(xa, xb);
            const Packed<K_> wa = pack_row<K_>(xa, f), wb = pack_row<K_>(xb, f);
            if (is_v) {
                store_value<D, K_>(tile, tau0 + j, at.da, wa);
                store_value<D, K_>(tile, tau0 + j, at.db, wb);
            } else {
                store_key<D, K_>(tile, tau0 + j, at.da, wa);
                store_key<D, K_>(tile, tau0 + j, at.db, wb);
            }
            if (c == 0) store_factors<D, K_>(tile, tau0 + j, is_v ? kv_factors(K_) / 2 : 0, f);
        }
    };
    if (hi <= lo) return;
    if (hi == lo + 1) {                                         // a decode step
        h8_t xa = load(s0 + lo, at.da), xb = load(s0 + lo, at.db);
        if (!is_v) turn(xa, xb, table, p.table_rows, R, pos0 + lo, at);
        put(lo, xa, xb);
        return;
    }
    // a few: one after the other, each would wait for its own loads; so eight are loaded and turned, some of them twice
    h8_t xa[8], xb[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int there = min(max(j, lo), hi - 1);
        xa[j] = load(s0 + there, at.da); xb[j] = load(s0 + there, at.db);
    }
    if (!is_v) {
#pragma unroll
        for (int j = 0; j < 8; ++j) turn(xa[j], xb[j], table, p.table_rows, R, pos0 + min(max(j, lo), hi - 1), at);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        if (j >= lo && j < hi) put(j, xa[j], xb[j]);
    }
}

template <int KIND>
__device__ __forceinline__ half_t value_of(int u, float s, float z) {
#pragma clang fp contract(off)
    const float v = KIND == KMI_KV_INT8 ? (float)(u - 128) * s : (float)u * s + z;
    return (half_t)(v > 65504.0f ? 65504.0f : v < -65504.0f ? -65504.0f : v);
}

// Eight packed elements to fp16.
template <int KIND>
__device__ __forceinline__ h8_t unpack_row(const Packed<KIND>& w, float s, float z) {
    if constexpr (KIND == KMI_KV_F16) {
        return __builtin_bit_cast(h8_t, u4_t{w.w[0], w.w[1], w.w[2], w.w[3]});
    } else {
        h8_t o;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if constexpr (KIND == KMI_KV_INT8) o[e] = value_of<KIND>((w.w[e / 4] >> (8 * (e % 4))) & 255, s, 0.0f);
            else o[e] = value_of<KIND>((w.w[0] >> (4 * e)) & 15, s, z);
        }
        return o;
    }
}

// One workgroup: eight neighbouring positions 8 i .. 8 i + 7 of one sequence, 2048 / D rows (key heads, then value heads); a lane
// reads eight elements of one row of all eight tokens (whole chunks of values, turned over in registers).  Bound by the memory: 16 x
// 8000 tokens, 8 heads of 64, int4: 61 us for 336 MB, 5.5 TB/s (107 us a token at a time; 76 with stores that stay in the caches, against
// loads past them 117: two lanes' loads share a line).
template <int D, int KIND>
__global__ __launch_bounds__(256) void kv_read_kernel(kmi_kv_read_args p) {
    constexpr int LPR = D / 8, ROWS = 256 / LPR, n = kv_per_word(KIND), NF = kv_factors(KIND);
    const int b = blockIdx.y, d0 = (threadIdx.x % LPR) * 8;
    const int r = blockIdx.z * ROWS + threadIdx.x / LPR;
    if (r >= 2 * p.KV) return;
    const bool is_v = r >= p.KV;
    const int head = is_v ? r - p.KV : r;
    const int start = p.start[b], count = p.count ? min(p.count[b], p.S) : p.S;
    const int pos0 = (int)((unsigned)((start >> 3) + (int)blockIdx.x) << 3), s0 = (int)((unsigned)pos0 - (unsigned)start);
    if (s0 >= p.S) return;
    half_t* out = static_cast<half_t*>(is_v ? p.v_out : p.k_out) + ((size_t)b * p.S * p.KV + head) * D + d0;
    const size_t out_step = (size_t)p.KV * D;
    const KvPlace place = {static_cast<char*>(const_cast<void*>(p.cache)), p.page_table, p.num_pages, p.page_tiles, p.max_pages, p.KV};
    const char* tile = pos0 < 0 ? nullptr : kv_tile_at<kv_tile_bytes(D, KIND)>(place, b, head, pos0 / KV_TILE);
    const int tau0 = pos0 & (KV_TILE - 1);

    Packed<KIND> w[8] = {};
    h8_t fs = {}, fz = {};                                      // scales and offsets of the eight tokens
    if (tile) {
        if constexpr (NF > 0) {
            const int first = is_v ? NF / 2 : 0;
            fs = *reinterpret_cast<const h8_t*>(tile + kv_factor_offset<D, KIND>(tau0, first));
            if constexpr (NF == 4) fz = *reinterpret_cast<const h8_t*>(tile + kv_factor_offset<D, KIND>(tau0, first + 1));
        }
        if (is_v) {
            const u4_t* at = reinterpret_cast<const u4_t*>(tile + kv_value_offset<D, KIND>(tau0, d0));
            u4_t c[8 / n];
#pragma unroll
            for (int i = 0; i < 8 / n; ++i) c[i] = at[i];
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int k = 0; k < Packed<KIND>::NPW; ++k)
                    w[j].w[k] = __builtin_amdgcn_perm(c[2 * k + 1][j / 2], c[2 * k][j / 2], j & 1 ? 0x07060302u : 0x05040100u);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const char* at = tile + kv_key_offset<D, KIND>(tau0 + j, d0);
                if constexpr (KIND == KMI_KV_F16) {
                    const u4_t v = *reinterpret_cast<const u4_t*>(at);
#pragma unroll
                    for (int k = 0; k < 4; ++k) w[j].w[k] = v[k];
                } else if constexpr (KIND == KMI_KV_INT8) {
                    const u2_t v = *reinterpret_cast<const u2_t*>(at);
                    w[j].w[0] = v[0]; w[j].w[1] = v[1];
                } else {
                    w[j].w[0] = nibbles_together(*reinterpret_cast<const uint32_t*>(at));
                }
            }
        }
    }
    const half_t nan = __builtin_bit_cast(half_t, (uint16_t)0x7E00);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int s = s0 + j;
        if (s < 0 || s >= p.S) continue;
        h8_t x = unpack_row<KIND>(w[j], (float)fs[j], (float)fz[j]);
        if (!tile) x = h8_t{nan, nan, nan, nan, nan, nan, nan, nan};
        if (s >= count) x = h8_t{};
        __builtin_nontemporal_store(x, reinterpret_cast<h8_t*>(out + s * out_step));
    }
}

static constexpr int KV_MOST_TOKENS = 1 << 26;                  // of a call and sequence: a launch holds under 2^32 threads in a row

// ---- C entries ---------------------------------------------------------------------------------------------------------
extern "C" int kmi_kv_tile_bytes(int D, int kind) {
    if (!kv_head_dim_ok(D) || kind < KMI_KV_F16 || kind > KMI_KV_INT4)
        return kmi_set_error(KMI_E_SHAPE, "kmi_kv_tile_bytes: need a head dimension of 64, 128 or 256 and a kind of 0..2 (D=%d kind=%d)", D, kind);
    return kv_tile_bytes(D, kind);
}

int kv_check_cache(const char* fn, const void* cache, const void* page_table, int B, int KV, int D, int kind, int num_pages,
                   int page_tiles, int max_pages) {
    if (!cache || !page_table) return kmi_set_error(KMI_E_NULL, "%s: cache and page_table must not be NULL", fn);
    if (!kmi_aligned16(cache)) return kmi_set_error(KMI_E_ALIGN, "%s: the cache must be 16-byte aligned", fn);
    if (kmi_kv_tile_bytes(D, kind) < 0) return KMI_E_SHAPE;
    if (B < 0 || B > 65535 || KV <= 0 || num_pages <= 0 || page_tiles <= 0 || max_pages <= 0 ||
        (long long)max_pages * page_tiles >= (1ll << 26) || (double)num_pages * KV * page_tiles > 2147483647.0)
        return kmi_set_error(KMI_E_SHAPE, "%s: need 0<=B<=65535, KV>0, num_pages>0, page_tiles>0, max_pages>0, under 2^31 tokens a sequence "
                             "and under 2^31 tiles (B=%d KV=%d num_pages=%d page_tiles=%d max_pages=%d)", fn, B, KV, num_pages, page_tiles, max_pages);
    return KMI_OK;
}

extern "C" int kmi_rope_kv(const kmi_rope_kv_args* args, void* stream) {
    const char* fn = "kmi_rope_kv";
    if (!args) return kmi_set_error(KMI_E_NULL, "%s: args is NULL", fn);
    const kmi_rope_kv_args& p = *args;
    const bool cached = p.cache != nullptr;
    if (!p.start || !p.k) return kmi_set_error(KMI_E_NULL, "%s: start and k must not be NULL", fn);
    if (!p.q != !p.q_out) return kmi_set_error(KMI_E_NULL, "%s: q and q_out go together", fn);
    if (!cached && !p.k_out) return kmi_set_error(KMI_E_NULL, "%s: k_out is needed without a cache", fn);
    if (cached && !p.v) return kmi_set_error(KMI_E_NULL, "%s: a cache needs v", fn);
    if (!kmi_aligned16(p.q) || !kmi_aligned16(p.q_out) || !kmi_aligned16(p.k) || !kmi_aligned16(p.k_out) || !kmi_aligned16(p.v) ||
        !kmi_aligned16(p.table))
        return kmi_set_error(KMI_E_ALIGN, "%s: every tensor must be 16-byte aligned", fn);
    if (!kv_head_dim_ok(p.D) || p.B < 0 || p.B > 65535 || p.S < 0 || p.S > KV_MOST_TOKENS || p.H < 0 || p.KV <= 0 || (p.q && p.H <= 0) ||
        (long long)p.H + 2ll * p.KV > 65535)
        return kmi_set_error(KMI_E_SHAPE, "%s: need a head dimension of 64, 128 or 256, 0<=B<=65535, 0<=S<=2^26, H, KV>0 (B=%d S=%d H=%d KV=%d D=%d)",
                             fn, p.B, p.S, p.H, p.KV, p.D);
    if (p.rotary_dim < 0 || p.rotary_dim > p.D || (p.rotary_dim & 15) || (p.rotary_dim && (!p.table || p.table_rows <= 0)))
        return kmi_set_error(KMI_E_SHAPE, "%s: rotary_dim must be a multiple of 16 up to the head dimension, with a table of rows (rotary_dim=%d rows=%d)",
                             fn, p.rotary_dim, p.table_rows);
    if ((p.q_batch | p.q_token | p.k_batch | p.k_token | p.v_batch | p.v_token) & 7)
        return kmi_set_error(KMI_E_ALIGN, "%s: strides must be multiples of 8 elements", fn);
    if (cached) {
        const int rc = kv_check_cache(fn, p.cache, p.page_table, p.B, p.KV, p.D, p.kind, p.num_pages, p.page_tiles, p.max_pages);
        if (rc < 0) return rc;
    }
    if (p.B == 0 || p.S == 0) return KMI_OK;
    const int rows = (p.q ? p.H : 0) + p.KV + (cached ? p.KV : 0), at_once = 4096 / p.D;
    const dim3 grid((unsigned)(((long long)p.S + 14) / 8), p.B, (rows + at_once - 1) / at_once), block(256);
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int kind = cached ? p.kind : -1;
#define KMI_ROPE_LAUNCH(D_, K_) \
    hipLaunchKernelGGL((p.interleaved ? rope_kv_kernel<D_, K_, true> : rope_kv_kernel<D_, K_, false>), grid, block, 0, st, p)
#define KMI_ROPE_KIND(D_)                                                                                             \
    switch (kind) {                                                                                                   \
        case KMI_KV_F16: KMI_ROPE_LAUNCH(D_, KMI_KV_F16); break;                                                      \
        case KMI_KV_INT8: KMI_ROPE_LAUNCH(D_, KMI_KV_INT8); break;                                                    \
        case KMI_KV_INT4: KMI_ROPE_LAUNCH(D_, KMI_KV_INT4); break;                                                    \
        default: KMI_ROPE_LAUNCH(D_, -1);                                                                             \
    }
    if (p.D == 64) { KMI_ROPE_KIND(64) }
    else if (p.D == 128) { KMI_ROPE_KIND(128) }
    else { KMI_ROPE_KIND(256) }
#undef KMI_ROPE_KIND
#undef KMI_ROPE_LAUNCH
    return kmi_check_launch(fn);
}

extern "C" int kmi_kv_read(const kmi_kv_read_args* args, void* stream) {
    const char* fn = "kmi_kv_read";
    if (!args) return kmi_set_error(KMI_E_NULL, "%s: args is NULL", fn);
    const kmi_kv_read_args& p = *args;
    if (!p.k_out || !p.v_out || !p.start) return kmi_set_error(KMI_E_NULL, "%s: k_out, v_out and start must not be NULL", fn);
    if (!kmi_aligned16(p.k_out) || !kmi_aligned16(p.v_out)) return kmi_set_error(KMI_E_ALIGN, "%s: outputs must be 16-byte aligned", fn);
    const int rc = kv_check_cache(fn, p.cache, p.page_table, p.B, p.KV, p.D, p.kind, p.num_pages, p.page_tiles, p.max_pages);
    if (rc < 0) return rc;
    if (p.S < 0 || p.S > KV_MOST_TOKENS) return kmi_set_error(KMI_E_SHAPE, "%s: need 0<=S<=2^26 (S=%d)", fn, p.S);
    if (p.B == 0 || p.S == 0) return KMI_OK;
    const int at_once = 2048 / p.D;
    if (p.KV > 32767) return kmi_set_error(KMI_E_SHAPE, "%s: need KV<=32767 (KV=%d)", fn, p.KV);
    const dim3 grid((unsigned)(((long long)p.S + 14) / 8), p.B, (2 * p.KV + at_once - 1) / at_once), block(256);
    hipStream_t st = static_cast<hipStream_t>(stream);
#define KMI_READ_LAUNCH(D_)                                                                                           \
    switch (p.kind) {                                                                                                 \
        case KMI_KV_F16: hipLaunchKernelGGL((kv_read_kernel<D_, KMI_KV_F16>), grid, block, 0, st, p); break;          \
        case KMI_KV_INT8: hipLaunchKernelGGL((kv_read_kernel<D_, KMI_KV_INT8>), grid, block, 0, st, p); break;        \
        default: hipLaunchKernelGGL((kv_read_kernel<D_, KMI_KV_INT4>), grid, block, 0, st, p);                        \
    }
    if (p.D == 64) { KMI_READ_LAUNCH(64) }
    else if (p.D == 128) { KMI_READ_LAUNCH(128) }
    else { KMI_READ_LAUNCH(256) }
#undef KMI_READ_LAUNCH
    return kmi_check_launch(fn);
}
