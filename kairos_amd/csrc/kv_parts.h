// The paged key-value cache's tile: what its writer, its reader and the attention kernel share.
//
// A cache is [num_pages][kv_heads][page_tiles][tile_bytes]; a tile holds 32 consecutive tokens of one head, contiguous:
// keys, values, factors.  Inside, everything lies in the order in which the lanes of a 16x16x32 MFMA take it, so the
// attention kernel reads a tile with whole 1 KiB wave loads and feeds them to the matrix unit without moving anything
// between lanes.  n = elements in 16 bits: 1 (f16), 2 (int8), 4 (int4).
//   keys     unit (h, kk, g, row) = elements 32 kk + 8 g .. + 7 of token 8 (row / 4) + 4 h + row % 4: the A operand of
//            Q K^T, row = token, so that lane (head, g) of the product holds tokens 8 g .. 8 g + 7 over its two halves h.
//            [units (h, kk), n at a time][lane 16 g + row][n units of 16 / n bytes]
//   values   the A operand of V^T P: lane (dl, g) holds tokens 8 g + j of n neighbouring elements d = 16 n c + n dl + a.
//            [c][lane 16 g + dl][token j = 0..7] words of 16 bits, value a in bits 16 a / n
//   factors  fp16 [32] each: int8: key scale, value scale; int4: key scale, key offset, value scale, value offset
// A token of one head owns whole 16-bit words everywhere, so writers of different tokens never share one.
#ifndef KMI_KV_PARTS_H
#define KMI_KV_PARTS_H
#include "kmi_common.h"

#define KV_TILE 32

static constexpr int kv_per_word(int kind) { return kind == KMI_KV_F16 ? 1 : kind == KMI_KV_INT8 ? 2 : 4; }
static constexpr int kv_factors(int kind) { return kind == KMI_KV_F16 ? 0 : kind == KMI_KV_INT8 ? 2 : 4; }
static constexpr int kv_part_bytes(int D, int kind) { return 2 * KV_TILE * D / kv_per_word(kind); }     // keys or values
static constexpr int kv_tile_bytes(int D, int kind) { return 2 * kv_part_bytes(D, kind) + 2 * KV_TILE * kv_factors(kind); }
static inline bool kv_head_dim_ok(int D) { return D == 64 || D == 128 || D == 256; }

#ifdef __HIPCC__
// Byte offset in a tile of the eight key elements d0 .. d0 + 7 (d0 % 8 == 0) of token tau; 16 / n bytes.
template <int D, int KIND>
__device__ __forceinline__ int kv_key_offset(int tau, int d0) {
    constexpr int n = kv_per_word(KIND);
    const int row = 4 * (tau >> 3) + (tau & 3), h = (tau >> 2) & 1;
    const int unit = h * (D / 32) + (d0 >> 5), g = (d0 >> 3) & 3;
    return (unit / n) * 1024 + (g * 16 + row) * 16 + (unit % n) * (16 / n);
}
// Byte offset in a tile of the word that holds element d (d % n == 0) of token tau's value.
template <int D, int KIND>
__device__ __forceinline__ int kv_value_offset(int tau, int d) {
    constexpr int n = kv_per_word(KIND);
    return kv_part_bytes(D, KIND) + ((d / (16 * n)) * 64 + (tau >> 3) * 16 + (d % (16 * n)) / n) * 16 + (tau & 7) * 2;
}
template <int D, int KIND>
__device__ __forceinline__ int kv_factor_offset(int tau, int i) {
    return 2 * kv_part_bytes(D, KIND) + 2 * (KV_TILE * i + tau);
}

// A tile's address, or nullptr where the page table has no page of this cache for it.
struct KvPlace {
    char* cache;
    const int32_t* page_table;      // [B][max_pages]
    int num_pages, page_tiles, max_pages, kv_heads;
};
template <int TILE_BYTES>
__device__ __forceinline__ char* kv_tile_at(const KvPlace& p, int b, int head, int tile) {
    const int page = tile / p.page_tiles;
    if (tile < 0 || page >= p.max_pages) return nullptr;
    const int id = p.page_table[(size_t)b * p.max_pages + page];
    if (id < 0 || id >= p.num_pages) return nullptr;
    return p.cache + (((size_t)id * p.kv_heads + head) * p.page_tiles + (tile - page * p.page_tiles)) * TILE_BYTES;
}
#endif  // __HIPCC__
#endif
