// Attention of one new token a sequence over the paged cache:
//   o[b, h] = sum_t p_t v_t / sum_t p_t,   p_t = exp(scale q[b, h] . k_t - m),   t over the sequence's (window's) tokens
// One pass over the cache with the running maximum m and sum of the softmax.  The G = H / KV query heads that share a key
// head are the 16 columns of a matrix instruction, 32 tokens a step:
//   S^T [token x head] = K Q^T      (16x16x32 MFMA, two row halves of 16 tokens)
//   O^T [d x head]    += V^T P^T    (16x16x32 MFMA, a step's 32 tokens deep)
// The cache's tile order makes the result registers of the first product, lane (head, g) = tokens 8 g .. 8 g + 7, the operand
// registers of the second: nothing passes through LDS or between lanes but the maximum over the four lane groups.
// Codes enter the products as fp16 integers.  Keys go in as 1024 + u (one byte permute or mask, no subtraction); the offset
// times the sum of q is taken off in fp32, where the score's factor is applied.  Values go in as small signed integers; the
// token's scale multiplies p, relative to a running power of two so that p stays normal in fp16, and the offsets of the int4
// kind add up to one scalar a head.
#include "kv_parts.h"

static constexpr float PA_NEG = -1e30f;       // running maximum before the first token: finite, so differences stay numbers

__device__ __forceinline__ float group_max(float v) {      // over the four lane groups g that hold a head's tokens
    v = fmaxf(v, __shfl_xor(v, 16, 64));
    return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float group_sum(float v) {
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}

// Eight halves of unit u (0 .. n - 1) of a 16-byte key chunk: the element itself, or 1024 + code.
template <int KIND>
__device__ __forceinline__ h8_t key_unit(const u4_t& c, int u) {
    if constexpr (KIND == KMI_KV_F16) {
        return __builtin_bit_cast(h8_t, c);
    } else if constexpr (KIND == KMI_KV_INT8) {
        u4_t o;
        o[0] = __builtin_amdgcn_perm(0x64646464u, c[2 * u], 0x04010400u);
        o[1] = __builtin_amdgcn_perm(0x64646464u, c[2 * u], 0x04030402u);
        o[2] = __builtin_amdgcn_perm(0x64646464u, c[2 * u + 1], 0x04010400u);
        o[3] = __builtin_amdgcn_perm(0x64646464u, c[2 * u + 1], 0x04030402u);
        return __builtin_bit_cast(h8_t, o);
    } else {
        u4_t o;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = ((c[u] >> (4 * i)) & 0x000F000Fu) | 0x64006400u;
        return __builtin_bit_cast(h8_t, o);
    }
}

// Value a (0 .. n - 1) of the eight tokens of a 16-byte value chunk: the element, or code - 128 / code - 8.
template <int KIND>
__device__ __forceinline__ h8_t value_unit(const u4_t& c, int a) {
    if constexpr (KIND == KMI_KV_F16) {
        return __builtin_bit_cast(h8_t, c);
    } else {
        u4_t o;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            h2_t v;
            if constexpr (KIND == KMI_KV_INT8) {
                const h2_t off = {(half_t)1152.0f, (half_t)1152.0f};
                v = as_h2(__builtin_amdgcn_perm(0x64646464u, c[i], a ? 0x04030401u : 0x04020400u)) - off;
            } else {
                const uint32_t w = a & 2 ? c[i] >> 8 : c[i];
                const h2_t off = {(half_t)1032.0f, (half_t)1032.0f}, off16 = {(half_t)-72.0f, (half_t)-72.0f};
                const h2_t sixteenth = {(half_t)0.0625f, (half_t)0.0625f};
                v = a & 1 ? pk_fma(as_h2((w & 0x00F000F0u) | 0x64006400u), sixteenth, off16)
                          : as_h2((w & 0x000F000Fu) | 0x64006400u) - off;
            }
            o[i] = as_u32(v);
        }
        return __builtin_bit_cast(h8_t, o);
    }
}

// One wave's share of one head's tokens.
template <int D, int KIND>
struct PaWave {
    static constexpr int n = kv_per_word(KIND), CH = D / 16 / n, KSTEPS = D / 32, OT = D / 16, NF = kv_factors(KIND);
    static constexpr int TILE_BYTES = kv_tile_bytes(D, KIND), PART = kv_part_bytes(D, KIND);
    h8_t q[KSTEPS];             // lane (head, g): q[32 kk + 8 g ..]
    f4_t acc[OT];               // lane (head, g): tile T = n c + a, rows dl = 4 g + r, d = 16 n c + n dl + a
    float m, l, zsum;           // running maximum (raw scores; the head's), this lane's share of the sums of p and p * offset
    float ref;                  // power of two that the value scales are relative to
    float qsum;

    __device__ __forceinline__ void start(const half_t* qrow, bool used, int g) {
        float s = 0.0f;
#pragma unroll
        for (int kk = 0; kk < KSTEPS; ++kk) {
            q[kk] = used ? *reinterpret_cast<const h8_t*>(qrow + 32 * kk + 8 * g) : h8_t{};
#pragma unroll
            for (int e = 0; e < 8; ++e) s += (float)q[kk][e];
        }
        qsum = KIND == KMI_KV_F16 ? 0.0f : group_sum(s);
#pragma unroll
        for (int t = 0; t < OT; ++t) acc[t] = f4_t{};
        m = PA_NEG; l = 0.0f; zsum = 0.0f; ref = 0x1p-24f;
    }

    struct Tile {
        u4_t k[CH], v[CH];
        h8_t f[NF ? NF : 1];
    };
    __device__ __forceinline__ void load_keys(Tile& t, const char* tile, int lane) const {
#pragma unroll
        for (int i = 0; i < CH; ++i) t.k[i] = *reinterpret_cast<const u4_t*>(tile + i * 1024 + lane * 16);
#pragma unroll
        for (int i = 0; i < NF; ++i) t.f[i] = *reinterpret_cast<const h8_t*>(tile + 2 * PART + 64 * i + (lane >> 4) * 16);
    }
    __device__ __forceinline__ void load_values(Tile& t, const char* tile, int lane) const {
#pragma unroll
        for (int i = 0; i < CH; ++i) t.v[i] = *reinterpret_cast<const u4_t*>(tile + PART + i * 1024 + lane * 16);
    }

    // Scores of the tile's tokens and the weights p (fp16 operand `pf`); tok0 = the lane's first token, [lo, hi) the tokens
    // that count, whole = the tile lies inside.  bad: no page of this cache.  c = scale * log2(e).
    __device__ __forceinline__ h8_t weights(Tile& t, int tok0, int lo, int hi, bool whole, bool bad, float c) {
        f4_t s4[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            s4[h] = f4_t{};
#pragma unroll
            for (int kk = 0; kk < KSTEPS; ++kk) {
                const int unit = h * KSTEPS + kk;
                s4[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(key_unit<KIND>(t.k[unit / n], unit % n), q[kk], s4[h], 0, 0, 0);
            }
        }
        float s[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            s[j] = s4[j >> 2][j & 3];
            if constexpr (KIND == KMI_KV_INT8) s[j] = (s[j] - 1152.0f * qsum) * (float)t.f[0][j];
            if constexpr (KIND == KMI_KV_INT4) s[j] = (s[j] - 1024.0f * qsum) * (float)t.f[0][j] + qsum * (float)t.f[1][j];
            if (bad) s[j] = __builtin_nanf("");
        }
        float vs[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) vs[j] = KIND == KMI_KV_F16 ? 1.0f : (float)t.f[NF / 2][j];
        if (!whole) {
            // tokens outside: no weight, and nothing that stands in their place may reach a product
            u4_t keep;
#pragma unroll
            for (int i = 0; i < 4; ++i) keep[i] = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const bool in = tok0 + j >= lo && tok0 + j < hi;
                s[j] = in ? s[j] : -__builtin_inff();
                vs[j] = in ? vs[j] : 0.0f;
                if constexpr (KIND == KMI_KV_INT4) t.f[3][j] = in ? t.f[3][j] : (half_t)0.0f;
                keep[j >> 1] |= in ? 0xFFFFu << (16 * (j & 1)) : 0u;
            }
            if constexpr (KIND == KMI_KV_F16) {
#pragma unroll
                for (int i = 0; i < CH; ++i) t.v[i] &= keep;
            }
        }
        float top = s[0];
#pragma unroll
        for (int j = 1; j < 8; ++j) top = fmaxf(top, s[j]);
        top = group_max(top);
        float vtop = 0.0f;
        if constexpr (KIND != KMI_KV_F16) {
#pragma unroll
            for (int j = 0; j < 8; ++j) vtop = fmaxf(vtop, vs[j]);
            vtop = group_max(vtop);
        }
        if (__any(top > m) || vtop > ref) {
            const float m2 = fmaxf(m, top);
            float a = __builtin_amdgcn_exp2f((m - m2) * c);
            l *= a; zsum *= a;
            m = m2;
            if (KIND != KMI_KV_F16 && vtop > ref) {                // the next power of two: products with it are exact
                const float r2 = __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, vtop) + 0x7FFFFFu) & 0x7F800000u);
                a *= ref / r2;
                ref = r2;
            }
#pragma unroll
            for (int i = 0; i < OT; ++i) acc[i] = acc[i] * a;
        }
        const float inv = 1.0f / ref, mc = m * c;
        h8_t pf;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j], c, -mc));
            l += p;
            if constexpr (KIND == KMI_KV_INT4) zsum += p * ((float)t.f[3][j] + 8.0f * vs[j]);
            pf[j] = (half_t)(KIND == KMI_KV_F16 ? p : p * (vs[j] * inv));
        }
        return pf;
    }
    // The sums as they stand: value scales' unit and the offsets' sum applied.
    __device__ __forceinline__ void unscale() {
        if constexpr (KIND == KMI_KV_F16) return;
#pragma unroll
        for (int T = 0; T < OT; ++T) acc[T] = acc[T] * ref + zsum;
    }
    static __device__ __forceinline__ int d_of(int T, int dl) { return 16 * n * (T / n) + n * dl + T % n; }
    __device__ __forceinline__ void add(const Tile& t, const h8_t& pf) {
#pragma unroll
        for (int T = 0; T < OT; ++T)
            acc[T] = __builtin_amdgcn_mfma_f32_16x16x32_f16(value_unit<KIND>(t.v[T / n], T % n), pf, acc[T], 0, 0, 0);
    }
};

// One workgroup: 16 query heads of one key head of one sequence; its waves take the sequence's tiles in turn and are joined.
template <int D, int KIND>
__global__ __launch_bounds__(256) void paged_attn_kernel(kmi_paged_attn_args p, int head_tiles, float c) {
    using W = PaWave<D, KIND>;
    constexpr int NW = 4;
    __shared__ float red_m[NW][16], red_l[NW][16];
    __shared__ f4_t red_o[NW][W::OT / NW * (NW - 1)][64];       // every wave's tiles but those that it writes itself
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, g = lane >> 4, col = lane & 15;
    const int b = blockIdx.y, head = blockIdx.x / head_tiles, h0 = (blockIdx.x - head * head_tiles) * 16;
    const int G = p.H / p.KV, used = min(16, G - h0);
    const long capacity = (long)p.max_pages * p.page_tiles * KV_TILE;
    int hi = p.lens[b];
    const bool over = hi > capacity;
    hi = over ? 0 : max(hi, 0);
    const int lo = p.window > 0 ? max(0, hi - p.window) : 0;
    const KvPlace place = {static_cast<char*>(const_cast<void*>(p.cache)), p.page_table, p.num_pages, p.page_tiles, p.max_pages, p.KV};

    W w;
    w.start(static_cast<const half_t*>(p.q) + b * p.q_batch + (size_t)(head * G + h0 + min(col, used - 1)) * D, col < used, g);
    const int t1 = (hi + KV_TILE - 1) / KV_TILE;
    for (int t = lo / KV_TILE + wave; t < t1; t += NW) {
        const char* at = kv_tile_at<W::TILE_BYTES>(place, b, head, t);
        const bool bad = at == nullptr;
        if (bad) at = place.cache;
        typename W::Tile tile;
        w.load_keys(tile, at, lane);
        w.load_values(tile, at, lane);
        const bool whole = t * KV_TILE >= lo && (t + 1) * KV_TILE <= hi;
        const h8_t pf = w.weights(tile, t * KV_TILE + 8 * g, lo, hi, whole, bad, c);
        w.add(tile, pf);
    }

    // join: wave v adds up and writes the output tiles T = v * OT / NW .. of all waves
    constexpr int MINE = W::OT / NW;
    w.l = group_sum(w.l);
    if constexpr (KIND == KMI_KV_INT4) w.zsum = group_sum(w.zsum);
    if (g == 0) { red_m[wave][col] = w.m; red_l[wave][col] = w.l; }
    w.unscale();
    if (col < used) {
#pragma unroll
        for (int T = 0; T < W::OT; ++T)
            if (T / MINE != wave) red_o[wave][T - (T / MINE > wave ? MINE : 0)][lane] = w.acc[T];
    }
    __syncthreads();
    if (col >= used) return;
    float mm = PA_NEG, ll = 0.0f, a[NW];
#pragma unroll
    for (int v = 0; v < NW; ++v) mm = fmaxf(mm, red_m[v][col]);
#pragma unroll
    for (int v = 0; v < NW; ++v) {
        a[v] = __builtin_amdgcn_exp2f((red_m[v][col] - mm) * c);
        ll += a[v] * red_l[v][col];
    }
    half_t* out = static_cast<half_t*>(p.out) + ((size_t)b * p.H + head * G + h0 + col) * D;
#pragma unroll
    for (int T = 0; T < W::OT; ++T) {
        if (T / MINE != wave) continue;
        f4_t o = {};
#pragma unroll
        for (int v = 0; v < NW; ++v) {
            const f4_t x = v == wave ? w.acc[T] : red_o[v][T - (T / MINE > v ? MINE : 0)][lane];
            o = o + x * a[v];
        }
#pragma unroll
        for (int r = 0; r < 4; ++r)
            out[W::d_of(T, 4 * g + r)] = over ? __builtin_bit_cast(half_t, (uint16_t)0x7E00) : ll == 0.0f ? (half_t)0.0f : (half_t)(o[r] / ll);
    }
}

int kv_check_cache(const char* fn, const void* cache, const void* page_table, int B, int KV, int D, int kind, int num_pages,
                   int page_tiles, int max_pages);

extern "C" int kmi_paged_attn(const kmi_paged_attn_args* args, void* stream) {
    const char* fn = "kmi_paged_attn";
    if (!args) return kmi_set_error(KMI_E_NULL, "%s: args is NULL", fn);
    const kmi_paged_attn_args& p = *args;
    if (!p.out || !p.q || !p.lens) return kmi_set_error(KMI_E_NULL, "%s: out, q and lens must not be NULL", fn);
    if (!kmi_aligned16(p.out) || !kmi_aligned16(p.q) || (p.q_batch & 7))
        return kmi_set_error(KMI_E_ALIGN, "%s: out and q must be 16-byte aligned, q's stride a multiple of 8 elements", fn);
    const int rc = kv_check_cache(fn, p.cache, p.page_table, p.B, p.KV, p.D, p.kind, p.num_pages, p.page_tiles, p.max_pages);
    if (rc < 0) return rc;
    if (p.H <= 0 || p.H % p.KV || p.H > 65535 || p.window < 0 || !(p.scale > 0.0f) || !(p.scale < 1e30f))
        return kmi_set_error(KMI_E_SHAPE, "%s: need H a multiple of KV, window>=0 and a positive finite scale (H=%d KV=%d window=%d scale=%g)",
                             fn, p.H, p.KV, p.window, (double)p.scale);
    if (p.B == 0) return KMI_OK;
    const int G = p.H / p.KV, head_tiles = (G + 15) / 16;
    const float c = p.scale * 1.44269504088896340736f;
    const dim3 grid(p.KV * head_tiles, p.B), block(256);
    hipStream_t st = static_cast<hipStream_t>(stream);
#define KMI_PA_LAUNCH(D_)                                                                                             \
    switch (p.kind) {                                                                                                 \
        case KMI_KV_F16: hipLaunchKernelGGL((paged_attn_kernel<D_, KMI_KV_F16>), grid, block, 0, st, p, head_tiles, c); break;   \
        case KMI_KV_INT8: hipLaunchKernelGGL((paged_attn_kernel<D_, KMI_KV_INT8>), grid, block, 0, st, p, head_tiles, c); break; \
        default: hipLaunchKernelGGL((paged_attn_kernel<D_, KMI_KV_INT4>), grid, block, 0, st, p, head_tiles, c);    \
    }
    if (p.D == 64) { KMI_PA_LAUNCH(64) }
    else if (p.D == 128) { KMI_PA_LAUNCH(128) }
    else { KMI_PA_LAUNCH(256) }
#undef KMI_PA_LAUNCH
    return kmi_check_launch(fn);
}
