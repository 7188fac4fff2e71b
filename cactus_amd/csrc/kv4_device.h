// kv4_device.h -- page layout of the 4-bit KV cache, shared by the kernels
// that write and move pages (kv4.hip) and those that attend over them
// (attention_kv4.hip).
//
// pages[layer][page][kv head][16-key tile]; a tile holds 16 keys and values of
// one head in 18 d bytes, in the operand order of the 16x16x32 FP16 matrix
// instruction (lane = 16 h + row, eight contraction steps per lane), so that
// the attention feeds the instruction from its loads without a transpose:
//   K codes  [h 4][key 16][d/64][t 8]  byte: dim 64 p + 8 h + t in the low
//            nibble, dim 64 p + 32 + 8 h + t in the high one (K Q^T: row =
//            key, the contraction runs over 32 dims, 8 per lane)
//   K scales [h 4][d/32][i 4] fp16 of key 4 h + i (the rows of the product's
//            lane), one per 32 dims
//   V codes  [h 4][x 16][d/32][i 4]    byte: dim 32 g + x of key 4 h + i in
//            the low nibble, dim 32 g + 16 + x in the high one (V^T P^T: row
//            = dim, the contraction runs over the keys that the score
//            product left in the lane)
//   V scales like the K scales
// Codes are stored as code + 8.  Every key has bytes of its own, so a single
// token is appended without reading what is there.
#pragma once
#include "hip_common.h"

namespace cactus_hip {

constexpr int KV4_GROUP = CACTUS_HIP_KV4_GROUP;   // dims per scale
constexpr int KV4_TILE = 16;                      // keys per tile
constexpr size_t KV4_MAX_SEQS = 65536;            // slots: a bit each in LDS (duplicate check)

// what the kernels take of cactus_hip_kv4_cache
struct Kv4View {
    uint8_t* pages;          // the layer's (or, for the page operations, layer 0's)
    int32_t* table;
    int32_t* lens;
    int32_t* refs;
    int32_t* state;
    int Hkv, d, ps_log2;     // page size: 1 << ps_log2 tokens
    int num_pages, max_seqs, max_pages;
    int layers;
    size_t layer_bytes, page_bytes;
};

enum { KV4_FREE = 0, KV4_HINT = 1, KV4_STATUS = 2 };   // state words

__host__ __device__ inline int kv4_tile_bytes(int d) { return 18 * d; }

// bytes of (page, head): tiles of 16 keys
__device__ __forceinline__ uint8_t* kv4_tile(const Kv4View& c, int page, int head, int tile) {
    return c.pages + (size_t)page * c.page_bytes +
           (size_t)((head << (c.ps_log2 - 4)) + tile) * (unsigned)kv4_tile_bytes(c.d);
}
__device__ __forceinline__ bool kv4_page_ok(const Kv4View& c, int page) { return (unsigned)page < (unsigned)c.num_pages; }

// tokens of a slot, within what its table row can hold
__device__ __forceinline__ int kv4_len(const Kv4View& c, int slot) {
    const int cap = c.max_pages << c.ps_log2;
    const int n = c.lens[slot];
    return n < 0 ? 0 : (n > cap ? cap : n);
}
__device__ __forceinline__ int kv4_pages_of(const Kv4View& c, int len) { return (len + (1 << c.ps_log2) - 1) >> c.ps_log2; }
// slot of request i; -1: no such slot
__device__ __forceinline__ int kv4_slot(const Kv4View& c, const int32_t* seqs, int i) {
    const int s = seqs ? seqs[i] : i;
    return (unsigned)s < (unsigned)c.max_seqs ? s : -1;
}
// rows of request i, of at most seq_len
__device__ __forceinline__ int kv4_count(const int32_t* counts, int i, int seq_len) {
    const int n = counts ? counts[i] : seq_len;
    return n < 0 ? 0 : (n > seq_len ? seq_len : n);
}

// checks the descriptor and fills the view; `layer`: whose pages (page
// operations take all layers from layer 0 on)
int kv4_view(const cactus_hip_kv4_cache* c, size_t layer, const char* what, Kv4View* out);

}  // namespace cactus_hip
