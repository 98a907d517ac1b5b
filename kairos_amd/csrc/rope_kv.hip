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
// Traffic: every row read once and written once, plus the table's R * 4 bytes a token; a memory-bound kernel.
#include "kv_parts.h"

struct RowFactors {
    half_t s, z;
    float r;                       // 1 / s, 0 for a row of equal elements
};

__device__ __forceinline__ half_t scale_up(float width, float steps) {
    half_t s = (half_t)(width / steps);
    if ((float)s * steps < width) s = __builtin_bit_cast(half_t, (uint16_t)(__builtin_bit_cast(uint16_t, s) + 1));
    return s;
}

// Factors of a row spread over LPR neighbouring lanes, eight elements each.
template <int LPR, int KIND>
__device__ __forceinline__ RowFactors row_factors(h8_t x) {
#pragma clang fp contract(off)
    int top = 0;                                        // largest |x| as bits: orders infinities and NaN above all
    half_t lo = x[0], hi = x[0];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const half_t v = x[e];                          // a copy: a bit cast of a vector's element reads element 0
        const int bits = __builtin_bit_cast(uint16_t, v) & 0x7FFF;
        top = bits > top ? bits : top;
        lo = x[e] < lo ? x[e] : lo;
        hi = x[e] > hi ? x[e] : hi;
    }
    float flo = (float)lo, fhi = (float)hi;
#pragma unroll
    for (int off = LPR / 2; off > 0; off >>= 1) {
        const int t = __shfl_xor(top, off, 64);
        top = t > top ? t : top;
        if constexpr (KIND == KMI_KV_INT4) {
            flo = fminf(flo, __shfl_xor(flo, off, 64));
            fhi = fmaxf(fhi, __shfl_xor(fhi, off, 64));
        }
    }
    RowFactors f;
    f.z = (half_t)0.0f;
    if constexpr (KIND == KMI_KV_INT8) {
        f.s = scale_up((float)__builtin_bit_cast(half_t, (uint16_t)top), 127.0f);
    } else {
        f.z = (half_t)(flo + 0.0f);                     // never -0: which of two zeros is the smallest is left open
        f.s = scale_up(fhi - flo, 15.0f);
    }
    if (top >= 0x7C00) f.s = __builtin_bit_cast(half_t, (uint16_t)0x7E00);
    f.r = (float)f.s > 0.0f ? 1.0f / (float)f.s : 0.0f;
    return f;
}

__device__ __forceinline__ int code_of(float x, float z, float r, float lo, float hi) {
#pragma clang fp contract(off)
    return (int)fminf(fmaxf(rintf((x - z) * r), lo), hi);      // the clamp also turns a NaN into a number
}

// Eight elements of a row as the cache holds them: elements, or codes (bytes; nibbles), in order.  NPW = 32-bit words.
template <int KIND>
struct Packed {
    static constexpr int NPW = 4 / kv_per_word(KIND);
    uint32_t w[NPW];
};
template <int KIND>
__device__ __forceinline__ Packed<KIND> pack_row(h8_t x, const RowFactors& f) {
    Packed<KIND> o;
    if constexpr (KIND == KMI_KV_F16) {
        const u4_t w = __builtin_bit_cast(u4_t, x);
#pragma unroll
        for (int i = 0; i < 4; ++i) o.w[i] = w[i];
    } else {
#pragma unroll
        for (int i = 0; i < Packed<KIND>::NPW; ++i) o.w[i] = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if constexpr (KIND == KMI_KV_INT8) o.w[e / 4] |= (uint32_t)(code_of((float)x[e], 0.0f, f.r, -127.0f, 127.0f) + 128) << (8 * (e % 4));
            else o.w[0] |= (uint32_t)code_of((float)x[e], (float)f.z, f.r, 0.0f, 15.0f) << (4 * e);
        }
    }
    return o;
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
__device__ __forceinline__ void store_factors(char* tile, int tau, int d0, int first, const RowFactors& f) {
    if constexpr (KIND != KMI_KV_F16) {
        if (d0 != 0) return;
        *reinterpret_cast<half_t*>(tile + kv_factor_offset<D, KIND>(tau, first)) = f.s;
        if constexpr (KIND == KMI_KV_INT4) *reinterpret_cast<half_t*>(tile + kv_factor_offset<D, KIND>(tau, first + 1)) = f.z;
    }
}

template <int D, int KIND>
__device__ __forceinline__ void store_key(char* tile, int tau, int d0, h8_t x) {
    RowFactors f = {};
    if constexpr (KIND != KMI_KV_F16) f = row_factors<D / 8, KIND>(x);
    const Packed<KIND> w = pack_row<KIND>(x, f);
    char* at = tile + kv_key_offset<D, KIND>(tau, d0);
    if constexpr (KIND == KMI_KV_F16) *reinterpret_cast<u4_t*>(at) = u4_t{w.w[0], w.w[1], w.w[2], w.w[3]};
    else if constexpr (KIND == KMI_KV_INT8) *reinterpret_cast<u2_t*>(at) = u2_t{w.w[0], w.w[1]};
    else *reinterpret_cast<uint32_t*>(at) = nibbles_apart(w.w[0]);
    store_factors<D, KIND>(tile, tau, d0, 0, f);
}

// One token's value: its words stand 16 bytes apart.
template <int D, int KIND>
__device__ __forceinline__ void store_value(char* tile, int tau, int d0, const Packed<KIND>& w) {
    constexpr int n = kv_per_word(KIND);
#pragma unroll
    for (int i = 0; i < 8 / n; ++i)
        *reinterpret_cast<uint16_t*>(tile + kv_value_offset<D, KIND>(tau, d0 + n * i)) = (uint16_t)(w.w[i / 2] >> (16 * (i & 1)));
}
// Eight tokens tau0 .. tau0 + 7 (tau0 % 8 == 0): whole 16-byte chunks, 128 / n bytes in a row.
template <int D, int KIND>
__device__ __forceinline__ void store_values8(char* tile, int tau0, int d0, const Packed<KIND> (&w)[8]) {
    constexpr int n = kv_per_word(KIND);
    u4_t* at = reinterpret_cast<u4_t*>(tile + kv_value_offset<D, KIND>(tau0, d0));
#pragma unroll
    for (int i = 0; i < 8 / n; ++i) {
        u4_t c;
#pragma unroll
        for (int j = 0; j < 4; ++j) c[j] = __builtin_amdgcn_perm(w[2 * j + 1].w[i / 2], w[2 * j].w[i / 2], i & 1 ? 0x07060302u : 0x05040100u);
        at[i] = c;
    }
}

// Cosines and sines of the pairs that a lane's eight elements d0 .. d0 + 7 belong to; NaN beyond the table.
template <bool INTERLEAVED>
struct Angles {
    static constexpr int PAIRS = INTERLEAVED ? 4 : 8;
    float c[PAIRS], s[PAIRS];
    __device__ __forceinline__ void load(const float* table, int rows, int R, int pos, int d0) {
        if (d0 >= R) return;
        const bool inside = pos >= 0 && pos < rows;
        const int i0 = INTERLEAVED ? d0 / 2 : d0 % (R / 2);
        const f4_t* p = reinterpret_cast<const f4_t*>(table + (size_t)(inside ? pos : 0) * R + 2 * i0);
#pragma unroll
        for (int i = 0; i < PAIRS / 2; ++i) {
            const f4_t v = p[i];
            const float nan = __builtin_nanf("");
            c[2 * i] = inside ? v[0] : nan; s[2 * i] = inside ? v[1] : nan;
            c[2 * i + 1] = inside ? v[2] : nan; s[2 * i + 1] = inside ? v[3] : nan;
        }
    }
    // x: the lane's elements; o: their partners (half layout)
    __device__ __forceinline__ h8_t turn(h8_t x, h8_t o, int R, int d0) const {
#pragma clang fp contract(off)
        if (d0 >= R) return x;
        h8_t y;
        if constexpr (INTERLEAVED) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float a = (float)x[2 * i], b = (float)x[2 * i + 1];
                y[2 * i] = (half_t)(a * c[i] - b * s[i]);
                y[2 * i + 1] = (half_t)(b * c[i] + a * s[i]);
            }
        } else {
            const bool first = d0 < R / 2;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float a = (float)x[e], b = (float)o[e];
                const float t = b * s[e];
                y[e] = (half_t)(a * c[e] + (first ? -t : t));
            }
        }
        return y;
    }
};

// One workgroup: eight neighbouring positions 8 i .. 8 i + 7 of one sequence, 2048 / D rows (heads of queries, keys or values) of each;
// a lane has eight elements of one row.  Where all eight tokens are there, all loads are in flight before the first use,
// and the values leave as whole chunks of the cache, turned over in registers.
template <int D, int KIND, bool INTERLEAVED>
__global__ __launch_bounds__(256) void rope_kv_kernel(kmi_rope_kv_args p) {
    constexpr int LPR = D / 8, ROWS = 256 / LPR, K_ = KIND < 0 ? 0 : KIND;
    const int b = blockIdx.y, d0 = (threadIdx.x % LPR) * 8, R = p.rotary_dim;
    const int r = (p.q ? 0 : p.H) + blockIdx.z * ROWS + threadIdx.x / LPR;
    if (r >= p.H + p.KV + (KIND >= 0 ? p.KV : 0)) return;
    const bool is_q = r < p.H, is_v = r >= p.H + p.KV;
    const int head = is_q ? r : is_v ? r - p.H - p.KV : r - p.H;
    const int start = p.start[b], count = p.count ? min(p.count[b], p.S) : p.S;
    const int pos0 = (int)((unsigned)((start >> 3) + (int)blockIdx.x) << 3), s0 = (int)((unsigned)pos0 - (unsigned)start);
    if (s0 >= p.S) return;

    const int heads = is_q ? p.H : p.KV;
    const half_t* row = is_q ? static_cast<const half_t*>(p.q) + b * p.q_batch : is_v ? static_cast<const half_t*>(p.v) + b * p.v_batch
                                                                                     : static_cast<const half_t*>(p.k) + b * p.k_batch;
    const int64_t step = is_q ? p.q_token : is_v ? p.v_token : p.k_token;
    row += (size_t)head * D;
    half_t* out = static_cast<half_t*>(is_q ? p.q_out : is_v ? nullptr : p.k_out);
    if (out) out += ((size_t)b * p.S * heads + head) * D + d0;
    const size_t out_step = (size_t)heads * D;
    const KvPlace place = {static_cast<char*>(p.cache), p.page_table, p.num_pages, p.page_tiles, p.max_pages, p.KV};
    char* tile = nullptr;                                       // the eight positions lie in one tile
    if constexpr (KIND >= 0) tile = is_q || pos0 < 0 ? nullptr : kv_tile_at<kv_tile_bytes(D, K_)>(place, b, head, pos0 / KV_TILE);
    const int tau0 = pos0 & (KV_TILE - 1);
    const int partner = INTERLEAVED || d0 >= R ? d0 : d0 < R / 2 ? d0 + R / 2 : d0 - R / 2;
    const float* table = static_cast<const float*>(p.table);
    Angles<INTERLEAVED> ang;

    if (s0 >= 0 && s0 + 8 <= count) {
        h8_t x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = *reinterpret_cast<const h8_t*>(row + (s0 + j) * step + d0);
        if (is_v) {
            if constexpr (KIND >= 0) {
                if (!tile) return;
                Packed<K_> w[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    RowFactors f = {};
                    if constexpr (K_ != KMI_KV_F16) f = row_factors<LPR, K_>(x[j]);
                    w[j] = pack_row<K_>(x[j], f);
                    store_factors<D, K_>(tile, tau0 + j, d0, kv_factors(K_) / 2, f);
                }
                store_values8<D, K_>(tile, tau0, d0, w);
            }
            return;
        }
        h8_t o[8];
        if constexpr (!INTERLEAVED) {
#pragma unroll
            for (int j = 0; j < 8; ++j) o[j] = *reinterpret_cast<const h8_t*>(row + (s0 + j) * step + partner);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            ang.load(table, p.table_rows, R, pos0 + j, d0);
            const h8_t y = ang.turn(x[j], INTERLEAVED ? x[j] : o[j], R, d0);
            if (out) *reinterpret_cast<h8_t*>(out + (s0 + j) * out_step) = y;
            if constexpr (KIND >= 0) {
                if (tile) store_key<D, K_>(tile, tau0 + j, d0, y);
            }
        }
        return;
    }
    for (int j = 0; j < 8; ++j) {
        const int s = s0 + j;
        if (s < 0 || s >= p.S) continue;
        if (s >= count) {                                       // rows behind the sequence: zeros out, nothing into the cache
            if (out) *reinterpret_cast<h8_t*>(out + s * out_step) = h8_t{};
            continue;
        }
        h8_t x = *reinterpret_cast<const h8_t*>(row + s * step + d0);
        if (!is_v) {
            const h8_t o = *reinterpret_cast<const h8_t*>(row + s * step + partner);
            ang.load(table, p.table_rows, R, pos0 + j, d0);
            x = ang.turn(x, o, R, d0);
        }
        if (out) *reinterpret_cast<h8_t*>(out + s * out_step) = x;
        if constexpr (KIND >= 0) {
            if (!tile) continue;
            if (is_v) {
                RowFactors f = {};
                if constexpr (K_ != KMI_KV_F16) f = row_factors<LPR, K_>(x);
                store_value<D, K_>(tile, tau0 + j, d0, pack_row<K_>(x, f));
                store_factors<D, K_>(tile, tau0 + j, d0, kv_factors(K_) / 2, f);
            } else {
                store_key<D, K_>(tile, tau0 + j, d0, x);
            }
        }
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
// reads eight elements of one row of all eight tokens (whole chunks of values, turned over in registers).
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
        *reinterpret_cast<h8_t*>(out + s * out_step) = x;
    }
}

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
        (long long)max_pages * page_tiles > (1ll << 26))
        return kmi_set_error(KMI_E_SHAPE, "%s: need 0<=B<=65535, KV>0, num_pages>0, page_tiles>0, max_pages>0 and at most 2^31 tokens a "
                             "sequence (B=%d KV=%d num_pages=%d page_tiles=%d max_pages=%d)", fn, B, KV, num_pages, page_tiles, max_pages);
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
    if (!kv_head_dim_ok(p.D) || p.B < 0 || p.B > 65535 || p.S < 0 || p.H < 0 || p.KV <= 0 || (p.q && p.H <= 0) ||
        (long long)p.H + 2ll * p.KV > 65535)
        return kmi_set_error(KMI_E_SHAPE, "%s: need a head dimension of 64, 128 or 256, 0<=B<=65535, S>=0, H, KV>0 (B=%d S=%d H=%d KV=%d D=%d)",
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
    const int rows = (p.q ? p.H : 0) + p.KV + (cached ? p.KV : 0), at_once = 2048 / p.D;
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
    if (p.S < 0) return kmi_set_error(KMI_E_SHAPE, "%s: need S>=0 (S=%d)", fn, p.S);
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
