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

// Codes of eight elements: int8 two words of four bytes, int4 element e in nibble e / 2 + 4 (e % 2) of one word.
template <int KIND>
__device__ __forceinline__ void row_codes(h8_t x, const RowFactors& f, int (&u)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        if constexpr (KIND == KMI_KV_INT8) u[e] = code_of((float)x[e], 0.0f, f.r, -127.0f, 127.0f) + 128;
        else u[e] = code_of((float)x[e], (float)f.z, f.r, 0.0f, 15.0f);
    }
}

template <int D, int KIND>
__device__ __forceinline__ void store_key(char* tile, int tau, int d0, h8_t x) {
    char* at = tile + kv_key_offset<D, KIND>(tau, d0);
    if constexpr (KIND == KMI_KV_F16) {
        *reinterpret_cast<h8_t*>(at) = x;
    } else {
        const RowFactors f = row_factors<D / 8, KIND>(x);
        int u[8];
        row_codes<KIND>(x, f, u);
        if constexpr (KIND == KMI_KV_INT8) {
            u2_t w;
            w[0] = u[0] | u[1] << 8 | u[2] << 16 | u[3] << 24;
            w[1] = u[4] | u[5] << 8 | u[6] << 16 | u[7] << 24;
            *reinterpret_cast<u2_t*>(at) = w;
        } else {
            uint32_t w = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) w |= (uint32_t)u[e] << (4 * (e / 2 + 4 * (e & 1)));
            *reinterpret_cast<uint32_t*>(at) = w;
        }
        if (d0 == 0) {
            *reinterpret_cast<half_t*>(tile + kv_factor_offset<D, KIND>(tau, 0)) = f.s;
            if constexpr (KIND == KMI_KV_INT4) *reinterpret_cast<half_t*>(tile + kv_factor_offset<D, KIND>(tau, 1)) = f.z;
        }
    }
}

template <int D, int KIND>
__device__ __forceinline__ void store_value(char* tile, int tau, int d0, h8_t x) {
    if constexpr (KIND == KMI_KV_F16) {
#pragma unroll
        for (int e = 0; e < 8; ++e) *reinterpret_cast<half_t*>(tile + kv_value_offset<D, KIND>(tau, d0 + e)) = x[e];
    } else {
        const RowFactors f = row_factors<D / 8, KIND>(x);
        int u[8];
        row_codes<KIND>(x, f, u);
        constexpr int n = kv_per_word(KIND);
#pragma unroll
        for (int w = 0; w < 8 / n; ++w) {
            int bits = 0;
#pragma unroll
            for (int a = 0; a < n; ++a) bits |= u[n * w + a] << (16 / n * a);
            *reinterpret_cast<uint16_t*>(tile + kv_value_offset<D, KIND>(tau, d0 + n * w)) = (uint16_t)bits;
        }
        if (d0 == 0) {
            constexpr int i = kv_factors(KIND) / 2;
            *reinterpret_cast<half_t*>(tile + kv_factor_offset<D, KIND>(tau, i)) = f.s;
            if constexpr (KIND == KMI_KV_INT4) *reinterpret_cast<half_t*>(tile + kv_factor_offset<D, KIND>(tau, 3)) = f.z;
        }
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
    // x: the lane's elements; row: the row's first element (for the partner of the half layout)
    __device__ __forceinline__ h8_t turn(h8_t x, const half_t* row, int R, int d0) const {
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
            const h8_t o = *reinterpret_cast<const h8_t*>(row + (first ? d0 + R / 2 : d0 - R / 2));
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

// One workgroup: `span` neighbouring tokens of one sequence, all their rows (queries, keys, values), eight elements a lane.
// A lane keeps the angles of its elements for all rows of a token.
template <int D, int KIND, bool INTERLEAVED>
__global__ __launch_bounds__(256) void rope_kv_kernel(kmi_rope_kv_args p, int span) {
    constexpr int LPR = D / 8, ROWS = 256 / LPR;
    constexpr int TILE_BYTES = KIND < 0 ? 0 : kv_tile_bytes(D, KIND < 0 ? 0 : KIND);
    const int b = blockIdx.y;
    const int d0 = (threadIdx.x % LPR) * 8, r0 = threadIdx.x / LPR;
    const int start = p.start[b], count = p.count ? min(p.count[b], p.S) : p.S;
    const int first = p.q ? 0 : p.H, rows = p.H + p.KV + (KIND >= 0 ? p.KV : 0);
    const KvPlace place = {static_cast<char*>(p.cache), p.page_table, p.num_pages, p.page_tiles, p.max_pages, p.KV};
    half_t* q_out = static_cast<half_t*>(p.q_out);
    half_t* k_out = static_cast<half_t*>(p.k_out);
    Angles<INTERLEAVED> ang;
    for (int s = blockIdx.x * span; s < min((int)(blockIdx.x + 1) * span, p.S); ++s) {
        const bool valid = s < count;
        const int pos = valid ? (int)((unsigned)start + (unsigned)s) : 0;
        if (valid) ang.load(static_cast<const float*>(p.table), p.table_rows, p.rotary_dim, pos, d0);
        const size_t token = (size_t)b * p.S + s;
        for (int r = first + r0; r < rows; r += ROWS) {
            const bool is_q = r < p.H, is_k = !is_q && r < p.H + p.KV;
            const int head = is_q ? r : is_k ? r - p.H : r - p.H - p.KV;
            half_t* out = is_q ? q_out + (token * p.H + head) * D : is_k && k_out ? k_out + (token * p.KV + head) * D : nullptr;
            if (!valid) {                                       // rows behind the sequence: zeros out, nothing into the cache
                if (out) *reinterpret_cast<h8_t*>(out + d0) = h8_t{};
                continue;
            }
            const half_t* row = is_q ? static_cast<const half_t*>(p.q) + b * p.q_batch + s * p.q_token
                              : is_k ? static_cast<const half_t*>(p.k) + b * p.k_batch + s * p.k_token
                                     : static_cast<const half_t*>(p.v) + b * p.v_batch + s * p.v_token;
            row += (size_t)head * D;
            h8_t x = *reinterpret_cast<const h8_t*>(row + d0);
            if (is_q || is_k) x = ang.turn(x, row, p.rotary_dim, d0);
            if (out) *reinterpret_cast<h8_t*>(out + d0) = x;
            if constexpr (KIND >= 0) {
                if (is_q) continue;
                // the lanes of a row go together: the row's factors are joined over them
                char* tile = pos < 0 ? nullptr : kv_tile_at<TILE_BYTES>(place, b, head, pos / KV_TILE);
                if (!tile) continue;
                if (is_k) store_key<D, KIND>(tile, pos % KV_TILE, d0, x);
                else store_value<D, KIND>(tile, pos % KV_TILE, d0, x);
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

// Eight elements a lane of one token of one head, keys and values.
template <int D, int KIND>
__global__ __launch_bounds__(256) void kv_read_kernel(kmi_kv_read_args p) {
    constexpr int LPR = D / 8, n = kv_per_word(KIND);
    const int b = blockIdx.y;
    const long item = (long)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;       // (token, head)
    if (item >= (long)p.S * p.KV) return;
    const int s = (int)(item / p.KV), head = (int)(item - (long)s * p.KV), d0 = (threadIdx.x % LPR) * 8;
    const size_t at = (((size_t)b * p.S + s) * p.KV + head) * D + d0;
    h8_t k = {}, v = {};
    const int count = p.count ? p.count[b] : p.S;
    if (s < count) {
        const KvPlace place = {static_cast<char*>(const_cast<void*>(p.cache)), p.page_table, p.num_pages, p.page_tiles, p.max_pages, p.KV};
        const int pos = (int)((unsigned)p.start[b] + (unsigned)s), tau = pos & (KV_TILE - 1);
        const char* tile = pos < 0 ? nullptr : kv_tile_at<kv_tile_bytes(D, KIND)>(place, b, head, pos / KV_TILE);
        if (!tile) {
            const half_t nan = __builtin_bit_cast(half_t, (uint16_t)0x7E00);
            k = h8_t{nan, nan, nan, nan, nan, nan, nan, nan};
            v = k;
        } else if constexpr (KIND == KMI_KV_F16) {
            k = *reinterpret_cast<const h8_t*>(tile + kv_key_offset<D, KIND>(tau, d0));
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = *reinterpret_cast<const half_t*>(tile + kv_value_offset<D, KIND>(tau, d0 + e));
        } else {
            float f[4] = {};
#pragma unroll
            for (int i = 0; i < kv_factors(KIND); ++i) f[i] = (float)*reinterpret_cast<const half_t*>(tile + kv_factor_offset<D, KIND>(tau, i));
            const char* kp = tile + kv_key_offset<D, KIND>(tau, d0);
            if constexpr (KIND == KMI_KV_INT8) {
                const u2_t w = *reinterpret_cast<const u2_t*>(kp);
#pragma unroll
                for (int e = 0; e < 8; ++e) k[e] = value_of<KIND>((w[e / 4] >> (8 * (e % 4))) & 255, f[0], 0.0f);
            } else {
                const uint32_t w = *reinterpret_cast<const uint32_t*>(kp);
#pragma unroll
                for (int e = 0; e < 8; ++e) k[e] = value_of<KIND>((w >> (4 * (e / 2 + 4 * (e & 1)))) & 15, f[0], f[1]);
            }
#pragma unroll
            for (int w = 0; w < 8 / n; ++w) {
                const int bits = *reinterpret_cast<const uint16_t*>(tile + kv_value_offset<D, KIND>(tau, d0 + n * w));
#pragma unroll
                for (int a = 0; a < n; ++a)
                    v[n * w + a] = value_of<KIND>((bits >> (16 / n * a)) & (KIND == KMI_KV_INT8 ? 255 : 15),
                                                  KIND == KMI_KV_INT8 ? f[1] : f[2], f[3]);
            }
        }
    }
    *reinterpret_cast<h8_t*>(static_cast<half_t*>(p.k_out) + at) = k;
    *reinterpret_cast<h8_t*>(static_cast<half_t*>(p.v_out) + at) = v;
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
    const int span = p.S >= 64 ? 8 : 1;
    const dim3 grid((p.S + span - 1) / span, p.B), block(256);
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int kind = cached ? p.kind : -1;
#define KMI_ROPE_LAUNCH(D_, K_) \
    hipLaunchKernelGGL((p.interleaved ? rope_kv_kernel<D_, K_, true> : rope_kv_kernel<D_, K_, false>), grid, block, 0, st, p, span)
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
    const long per = 256 / (p.D / 8), blocks = ((long)p.S * p.KV + per - 1) / per;
    if (blocks > 0x7FFFFFFF) return kmi_set_error(KMI_E_SHAPE, "%s: S * KV is too large (S=%d KV=%d)", fn, p.S, p.KV);
    const dim3 grid((unsigned)blocks, p.B), block(256);
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
