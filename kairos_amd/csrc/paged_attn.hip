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

#ifndef KMI_PA_RUNS
#define KMI_PA_RUNS 512
#endif
#ifndef KMI_PA_MIN_QUOTA
#define KMI_PA_MIN_QUOTA 8
#endif

static constexpr float PA_NEG = -1e30f;       // running maximum before the first token: finite, so differences stay numbers

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

    struct Factors {
        h8_t f[NF ? NF : 1];
    };
    struct Tile {
        u4_t k[CH], v[CH];
        Factors f;
    };
    struct Scores {
        float s[8];
    };
    __device__ __forceinline__ void load_keys(Tile& t, const char* tile, int lane) const {
#pragma unroll
        for (int i = 0; i < CH; ++i) t.k[i] = *reinterpret_cast<const u4_t*>(tile + i * 1024 + lane * 16);
#pragma unroll
        for (int i = 0; i < NF; ++i) t.f.f[i] = *reinterpret_cast<const h8_t*>(tile + 2 * PART + 64 * i + (lane >> 4) * 16);
    }
    __device__ __forceinline__ void load_values(Tile& t, const char* tile, int lane) const {
#pragma unroll
        for (int i = 0; i < CH; ++i) t.v[i] = *reinterpret_cast<const u4_t*>(tile + PART + i * 1024 + lane * 16);
    }

    // Raw scores of the lane's tokens 8 g + j and head.
    __device__ __forceinline__ Scores scores(const Tile& t) const {
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
        Scores o;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            o.s[j] = s4[j >> 2][j & 3];
            if constexpr (KIND == KMI_KV_INT8) o.s[j] = (o.s[j] - 1152.0f * qsum) * (float)t.f.f[0][j];
            if constexpr (KIND == KMI_KV_INT4) o.s[j] = (o.s[j] - 1024.0f * qsum) * (float)t.f.f[0][j] + qsum * (float)t.f.f[1][j];
        }
        return o;
    }
    // The weights p (fp16 operand) from the scores, and the running maximum, sums and accumulators brought to them; v: the
    // tile's values, fac: its factors.  tok0 = the lane's first token, [lo, hi) the tokens that count, whole = the tile lies
    // inside.  bad: no page of this cache.  c = scale * log2(e).
    __device__ __forceinline__ h8_t weights(Scores& sc, u4_t (&val)[CH], Factors& fac, int tok0, int lo, int hi, bool whole, bool bad, float c) {
        float (&s)[8] = sc.s;
        if (bad) {
#pragma unroll
            for (int j = 0; j < 8; ++j) s[j] = __builtin_nanf("");
        }
        float vs[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) vs[j] = KIND == KMI_KV_F16 ? 1.0f : (float)fac.f[NF / 2][j];
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
                if constexpr (KIND == KMI_KV_INT4) fac.f[3][j] = in ? fac.f[3][j] : (half_t)0.0f;
                keep[j >> 1] |= in ? 0xFFFFu << (16 * (j & 1)) : 0u;
            }
            if constexpr (KIND == KMI_KV_F16) {
#pragma unroll
                for (int i = 0; i < CH; ++i) val[i] &= keep;
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
            if constexpr (KIND == KMI_KV_INT4) zsum += p * ((float)fac.f[3][j] + 8.0f * vs[j]);
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
    __device__ __forceinline__ void add(const u4_t (&val)[CH], const h8_t& pf) {
#pragma unroll
        for (int T = 0; T < OT; ++T)
            acc[T] = __builtin_amdgcn_mfma_f32_16x16x32_f16(value_unit<KIND>(val[T / n], T % n), pf, acc[T], 0, 0, 0);
    }
};

// Work is shared out by tiles: the tiles of all tasks (sequence, 16 query heads of a key head) stand in a row, sequence by
// sequence, and workgroup w takes the run [w * quota, (w + 1) * quota) of them, whatever the lengths are -- the lengths are on the
// device, so every workgroup adds them up itself.  A task that lies in one run is finished there; one cut by run borders leaves a
// partial sum per workgroup (at most two each: the task that a run begins in the middle of, and the one that it ends in the
// middle of), and whichever workgroup of a task arrives last joins them in order.
struct PaSplit {
    uint32_t* counters;             // [gridDim.x] arrivals of the task that begins in run w and ends behind it; zero between calls
    float* partial;                 // [gridDim.x][2][slot], slot: m[16], l[16], o[used][D]
    int slot;
    int min_quota;
    int tasks_a_sequence, head_tiles;
    float c;
};

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

// Sums relative to a maximum, joined over NW waves: wave v adds up the output tiles T = v * OT / NW .. of all of them.
template <int D, int KIND>
struct PaJoin {
    using W = PaWave<D, KIND>;
    static constexpr int NW = 4, MINE = W::OT / NW;
    float m[NW][16], l[NW][16];
    f4_t o[NW][MINE * (NW - 1)][64];            // every wave's tiles but those that it adds up itself
};

template <int D, int KIND>
__global__ __launch_bounds__(256) void paged_attn_kernel(kmi_paged_attn_args p, PaSplit sp) {
    using W = PaWave<D, KIND>;
    using J = PaJoin<D, KIND>;
    constexpr int NW = J::NW, MINE = J::MINE;
    __shared__ J join;
    __shared__ int last;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, g = lane >> 4, col = lane & 15;
    const int G = p.H / p.KV, run = blockIdx.x;
    half_t* out0 = static_cast<half_t*>(p.out);

    // sequences without a tile: zeros, or NaN where the length does not fit the page table
    for (int b = run; b < p.B; b += gridDim.x) {
        const PaSequence s = pa_sequence(p, p.lens[b]);
        if (s.tiles) continue;
        const uint32_t fill = s.over ? 0x7E007E00u : 0u;
        u4_t* o = reinterpret_cast<u4_t*>(out0 + (size_t)b * p.H * D);
        for (int i = threadIdx.x; i < p.H * D / 8; i += 256) o[i] = u4_t{fill, fill, fill, fill};
    }

    // all tiles, the run's share, and the sequence that it begins in
    int total = 0;
    for (int b0 = 0; b0 < p.B; b0 += 64) total += b0 + lane < p.B ? pa_sequence(p, p.lens[b0 + lane]).tiles : 0;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) total += __shfl_xor(total, off, 64);
    const int U = __builtin_amdgcn_readfirstlane(total) * sp.tasks_a_sequence;
    int quota = (U + (int)gridDim.x - 1) / (int)gridDim.x;
    quota = (max(quota, sp.min_quota) + NW - 1) / NW * NW;
    const int begin = run * quota, end = min(U, begin + quota);
    if (run > (U - 1) / quota || U == 0) return;
    int b = 0, before = 0;                                      // before: tiles of the sequences in front, times tasks
    for (int b0 = 0; b0 < p.B; b0 += 64) {
        const int mine = b0 + lane < p.B ? pa_sequence(p, p.lens[b0 + lane]).tiles * sp.tasks_a_sequence : 0;
        int upto = mine;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int v = __shfl_up(upto, off, 64);
            if (lane >= off) upto += v;
        }
        const uint64_t behind = __ballot(before + upto > begin);
        if (behind) {
            const int at = __builtin_ctzll(behind);
            b = b0 + at;
            before += __builtin_amdgcn_readlane(upto, at) - __builtin_amdgcn_readlane(mine, at);
            break;
        }
        before += __builtin_amdgcn_readlane(upto, 63);
    }

    for (int unit = begin; unit < end && b < p.B;) {
        const PaSequence seq = pa_sequence(p, p.lens[b]);
        if (unit >= before + seq.tiles * sp.tasks_a_sequence) {
            before += seq.tiles * sp.tasks_a_sequence;
            ++b;
            continue;
        }
        const int task = (unit - before) / seq.tiles, ta = unit - before - task * seq.tiles;
        const int tb = min(seq.tiles, ta + end - unit);
        const int task0 = before + task * seq.tiles;                       // the task's first unit
        const int head = task / sp.head_tiles, h0 = (task - head * sp.head_tiles) * 16, used = min(16, G - h0);
        unit += tb - ta;

        W w;
        w.start(static_cast<const half_t*>(p.q) + b * p.q_batch + (size_t)(head * G + h0 + min(col, used - 1)) * D, col < used, g);
        // this wave's tiles ta + wave + NW i; their places in the pool, 64 at a time, one a lane
        const int count = (tb - ta - wave + NW - 1) / NW;
        const char* cache = static_cast<const char*>(p.cache);
        int places = -1;
        auto place_of = [&](int i) {
            if ((i & 63) == 0) {
                const int t = seq.first + ta + wave + NW * (i + lane);
                places = -1;
                if (i + lane < count) {
                    const int page = t / p.page_tiles;
                    const int id = p.page_table[(size_t)b * p.max_pages + page];
                    if (id >= 0 && id < p.num_pages) places = (id * p.KV + head) * p.page_tiles + t - page * p.page_tiles;
                }
            }
            return __builtin_amdgcn_readlane(places, i & 63);
        };
        typename W::Tile tile;
        int place = 0;
        if (count > 0) {
            place = place_of(0);
            const char* at = cache + (size_t)max(place, 0) * W::TILE_BYTES;
            w.load_keys(tile, at, lane);
            w.load_values(tile, at, lane);
        }
        for (int i = 0; i < count; ++i) {
            typename W::Scores sc = w.scores(tile);
            typename W::Factors fac = tile.f;
            const bool bad = place < 0;
            const char* next = nullptr;
            if (i + 1 < count) {
                place = place_of(i + 1);
                next = cache + (size_t)max(place, 0) * W::TILE_BYTES;
                w.load_keys(tile, next, lane);
            }
            const int t = seq.first + ta + wave + NW * i;
            const bool whole = t * KV_TILE >= seq.lo && (t + 1) * KV_TILE <= seq.hi;
            const h8_t pf = w.weights(sc, tile.v, fac, t * KV_TILE + 8 * g, seq.lo, seq.hi, whole, bad, sp.c);
            w.add(tile.v, pf);
            if (next) w.load_values(tile, next, lane);
        }

        // the waves' sums, joined
        w.l = group_sum(w.l);
        if constexpr (KIND == KMI_KV_INT4) w.zsum = group_sum(w.zsum);
        if (g == 0) { join.m[wave][col] = w.m; join.l[wave][col] = w.l; }
        w.unscale();
        if (col < used) {
#pragma unroll
            for (int T = 0; T < W::OT; ++T)
                if (T / MINE != wave) join.o[wave][T - (T / MINE > wave ? MINE : 0)][lane] = w.acc[T];
        }
        __syncthreads();
        float mm = PA_NEG, ll = 0.0f, a[NW];
#pragma unroll
        for (int v = 0; v < NW; ++v) mm = fmaxf(mm, join.m[v][col]);
#pragma unroll
        for (int v = 0; v < NW; ++v) {
            a[v] = __builtin_amdgcn_exp2f((join.m[v][col] - mm) * sp.c);
            ll += a[v] * join.l[v][col];
        }
        const bool complete = ta == 0 && tb == seq.tiles;
        float* slot = sp.partial + ((size_t)run * 2 + (ta == 0)) * sp.slot;
        half_t* out = out0 + ((size_t)b * p.H + head * G + h0) * D;
        const float norm = ll == 0.0f ? 0.0f : 1.0f / ll;
        if (col < used) {
#pragma unroll
            for (int T = 0; T < W::OT; ++T) {
                if (T / MINE != wave) continue;
                f4_t o = {};
#pragma unroll
                for (int v = 0; v < NW; ++v) {
                    const f4_t x = v == wave ? w.acc[T] : join.o[v][T - (T / MINE > v ? MINE : 0)][lane];
                    o = o + x * a[v];
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int d = W::d_of(T, 4 * g + r);
                    const float x = o[r];
                    if (complete) out[(size_t)col * D + d] = (half_t)(x * norm);
                    else __hip_atomic_store(slot + 32 + col * D + d, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                }
            }
            if (!complete && wave == 0 && g == 0) {
                __hip_atomic_store(slot + col, mm, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                __hip_atomic_store(slot + 16 + col, ll, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
        }
        if (!complete) {
            // Hand-off without fences: partial sums travel by agent-scope stores and loads, performed at the memory side; every
            // thread waits for its own to be performed, the barrier for every thread, and only then the arrival is counted there.
            const int w0 = task0 / quota, n = (task0 + seq.tiles - 1) / quota - w0 + 1;
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            if (threadIdx.x == 0) last = __hip_atomic_fetch_add(sp.counters + w0, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)(n - 1);
            __syncthreads();
            if (last) {
                auto slot_of = [&](int v) { return sp.partial + ((size_t)(w0 + v) * 2 + (v == 0)) * sp.slot; };
                for (int i = threadIdx.x; i < used * D; i += 256) {
                    const int hc = i / D;
                    float top = PA_NEG, sum = 0.0f, o = 0.0f;
#pragma unroll 8
                    for (int v = 0; v < n; ++v) top = fmaxf(top, __hip_atomic_load(slot_of(v) + hc, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
#pragma unroll 8
                    for (int v = 0; v < n; ++v) {
                        const float* s = slot_of(v);
                        const float f = __builtin_amdgcn_exp2f((__hip_atomic_load(s + hc, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) - top) * sp.c);
                        sum += f * __hip_atomic_load(s + 16 + hc, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                        o += f * __hip_atomic_load(s + 32 + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                    }
                    out[i] = (half_t)(sum == 0.0f ? 0.0f : o / sum);
                }
                if (threadIdx.x == 0) __hip_atomic_store(sp.counters + w0, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);     // for the next call
            }
        }
        __syncthreads();                                       // the next task writes the shared arrays again
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
    if (p.H <= 0 || p.H % p.KV || p.H > 65535 || p.window < 0 || !(p.scale > 0.0f) || !(p.scale < 1e30f))
        return kmi_set_error(KMI_E_SHAPE, "%s: need H a multiple of KV, window>=0 and a positive finite scale (H=%d KV=%d window=%d scale=%g)",
                             fn, p.H, p.KV, p.window, (double)p.scale);
    if (p.B == 0) return KMI_OK;
    const int G = p.H / p.KV, used = G < 16 ? G : 16;
    PaSplit sp;
    sp.head_tiles = (G + 15) / 16;
    sp.tasks_a_sequence = p.KV * sp.head_tiles;
    sp.c = p.scale * 1.44269504088896340736f;
    sp.slot = 32 + used * p.D;
    sp.min_quota = KMI_PA_MIN_QUOTA;
    sp.counters = static_cast<uint32_t*>(p.workspace);
    sp.partial = reinterpret_cast<float*>(static_cast<char*>(p.workspace) + KMI_GEMV_WS_HEADER);
    // as many runs as the GPU holds at once, never more than the tasks have room for
    const long long most = (long long)p.B * sp.tasks_a_sequence * p.max_pages * p.page_tiles;
    if (most > 0x7FFFFFFFll)
        return kmi_set_error(KMI_E_SHAPE, "%s: %d sequences of %d pages hold more than 2^31 tiles", fn, p.B, p.max_pages);
    const long long by_quota = (most + sp.min_quota - 1) / sp.min_quota;
    const int runs = (int)(by_quota < KMI_PA_RUNS ? by_quota : KMI_PA_RUNS);
    const size_t need = KMI_GEMV_WS_HEADER + (size_t)KMI_PA_RUNS * 2 * sp.slot * sizeof(float);
    if (!p.workspace || p.workspace_bytes < need)
        return kmi_set_error(KMI_E_SHAPE, "%s: the workspace must hold %zu bytes (has %zu)", fn, need, p.workspace ? (size_t)p.workspace_bytes : (size_t)0);
    const dim3 grid(runs), block(256);
    hipStream_t st = static_cast<hipStream_t>(stream);
#define KMI_PA_LAUNCH(D_)                                                                                             \
    switch (p.kind) {                                                                                                 \
        case KMI_KV_F16: hipLaunchKernelGGL((paged_attn_kernel<D_, KMI_KV_F16>), grid, block, 0, st, p, sp); break;   \
        case KMI_KV_INT8: hipLaunchKernelGGL((paged_attn_kernel<D_, KMI_KV_INT8>), grid, block, 0, st, p, sp); break; \
        default: hipLaunchKernelGGL((paged_attn_kernel<D_, KMI_KV_INT4>), grid, block, 0, st, p, sp);                 \
    }
    if (p.D == 64) { KMI_PA_LAUNCH(64) }
    else if (p.D == 128) { KMI_PA_LAUNCH(128) }
    else { KMI_PA_LAUNCH(256) }
#undef KMI_PA_LAUNCH
    return kmi_check_launch(fn);
}
