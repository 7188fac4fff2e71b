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

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 h16x2 __attribute__((ext_vector_type(2)));

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

// ------------------------------------------------------------ quantization (kv4.hip, kv4_rope.hip)
// Per value: x / s to the nearest integer, ties to even.  x has 11 significant
// bits and (k + 1/2) s at most 12, so x / s is either exactly k + 1/2 or at least
// 2^-13 away from it; x times the FP32 reciprocal of s is within 2^-20 of x / s, and
// rounded to a multiple of 2^-14 it falls on the same side, ties included (an
// exact division took twice the instructions).

// Scale of a group from the bits of its largest magnitude: a / 7 rounded to 8
// significant bits (bf16) and then to fp16, which only rounds again where the
// scale is an fp16 subnormal.  NaN for a NaN or an infinity.
__device__ __forceinline__ uint16_t kv4_scale(uint32_t abits) {
    const float q = h2f((uint16_t)abits) / 7.0f;
    uint32_t b = __builtin_bit_cast(uint32_t, q);
    b = (b + 0x7FFFu + ((b >> 16) & 1u)) & 0xFFFF0000u;   // finite: to nearest, ties to even
    return abits >= 0x7C00u ? (uint16_t)0x7E00u : f2h(bits_f(b));
}
// code + 8 in the low byte of the result; inv: 1 / s, 0 where every code is 0
__device__ __forceinline__ uint32_t kv4_code(uint16_t x, float inv) {
    const float v = __builtin_fmaf(h2f(x), inv, 768.0f) - 768.0f;    // a multiple of 2^-14 (|v| < 16)
    const float w = __builtin_amdgcn_fmed3f(v, -7.0f, 7.0f);
    return __builtin_bit_cast(uint32_t, w + 12582920.0f);  // 3 2^22 + 8: the integer in the low bits
}
__device__ __forceinline__ uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __builtin_amdgcn_perm(b, a, 0x0C0C0400u) | __builtin_amdgcn_perm(d, c, 0x04000C0Cu);
}
template <int CTRL>
__device__ __forceinline__ uint32_t quad(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, true);
}
// byte j of lane i's result: byte i of lane j's v, within each quad of lanes
__device__ __forceinline__ uint32_t quad_transpose(uint32_t v, int i) {
    // bytes (0, 1) and (2, 3) change places between lanes 1 apart, then pairs between lanes 2 apart
    uint32_t o = quad<0xB1>(v);
    v = i & 1 ? __builtin_amdgcn_perm(v, o, 0x07030501u) : __builtin_amdgcn_perm(o, v, 0x06020400u);
    o = quad<0x4E>(v);
    return i & 2 ? __builtin_amdgcn_perm(v, o, 0x07060302u) : __builtin_amdgcn_perm(o, v, 0x05040100u);
}
// N dwords at p, 4 N bytes aligned up to 16
template <int N>
__device__ __forceinline__ void load_dwords(uint32_t (&w)[N], const uint8_t* p) {
    if constexpr (N == 2) {
        const uint2 u = *reinterpret_cast<const uint2*>(p);
        w[0] = u.x, w[1] = u.y;
    } else {
#pragma unroll
        for (int k = 0; k < N / 4; k++) {
            const uint4 u = reinterpret_cast<const uint4*>(p)[k];
            w[4 * k] = u.x, w[4 * k + 1] = u.y, w[4 * k + 2] = u.z, w[4 * k + 3] = u.w;
        }
    }
}
template <int N>
__device__ __forceinline__ void store_dwords(uint8_t* p, const uint32_t (&w)[N]) {
    if constexpr (N == 2) {
        *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    } else {
#pragma unroll
        for (int k = 0; k < N / 4; k++)
            reinterpret_cast<uint4*>(p)[k] = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
    }
}

// Quantizes and writes a wave's share of a tile: x[g], dims 32 g + 8 h to + 7 of token `key` (lane
// 16 h + key), the keys or (vals) the values of one head; out: their part of the tile.
// `mine`: the lane's token is new; `whole`: all 16 are (the same for the wave).
template <int D>
__device__ __forceinline__ void kv4_write_tile(const uint4 (&x)[D / 32], uint8_t* out, bool vals, bool mine, bool whole) {
    constexpr int NG = D / 32;
    const int lane = threadIdx.x & 63, key = lane & 15, h = lane >> 4, i = lane & 3;
    // the groups' largest magnitudes, as fp16 bits (a NaN's or an infinity's are above every number's)
    uint32_t amax[NG];
#pragma unroll
    for (int g = 0; g < NG; g++) {
        const uint32_t m = 0x7FFF7FFFu;
        u16x2 y = __builtin_bit_cast(u16x2, x[g].x & m);
        y = __builtin_elementwise_max(y, __builtin_bit_cast(u16x2, x[g].y & m));
        y = __builtin_elementwise_max(y, __builtin_bit_cast(u16x2, x[g].z & m));
        y = __builtin_elementwise_max(y, __builtin_bit_cast(u16x2, x[g].w & m));
        amax[g] = max((uint32_t)y[0], (uint32_t)y[1]);
    }
#pragma unroll
    for (int g = 0; g < NG; g++) amax[g] = max(amax[g], (uint32_t)__shfl_xor((int)amax[g], 16, 64));
#pragma unroll
    for (int g = 0; g < NG; g++) amax[g] = max(amax[g], (uint32_t)__shfl_xor((int)amax[g], 32, 64));
    uint32_t c0[NG], c1[NG];                                 // codes of dims 0-3 and 4-7, a byte each
#pragma unroll
    for (int g = 0; g < NG; g++) {
        const uint16_t sb = kv4_scale(amax[g]);
        const float s = h2f(sb), inv = s > 0.0f ? 1.0f / s : 0.0f;      // (NaN: codes 0)
        // (a NaN or infinite value times 0 is NaN: its code is 0 too)
        const bool zero = !(s > 0.0f);
        const uint32_t w[4] = {x[g].x, x[g].y, x[g].z, x[g].w};
        uint32_t u[8];
#pragma unroll
        for (int t = 0; t < 8; t++) u[t] = kv4_code((uint16_t)(t & 1 ? w[t / 2] >> 16 : w[t / 2]), inv);
        c0[g] = zero ? 0x08080808u : low_bytes(u[0], u[1], u[2], u[3]);
        c1[g] = zero ? 0x08080808u : low_bytes(u[4], u[5], u[6], u[7]);
        if (mine && h == (g & 3))
            reinterpret_cast<uint16_t*>(out + 8 * D)[((key >> 2) * NG + g) * 4 + (key & 3)] = sb;
    }
    if (!vals) {
        uint32_t b[NG];
#pragma unroll
        for (int p = 0; p < NG / 2; p++) {
            b[2 * p] = c0[2 * p] | c0[2 * p + 1] << 4;
            b[2 * p + 1] = c1[2 * p] | c1[2 * p + 1] << 4;
        }
        if (mine) store_dwords(out + lane * (D / 8), b);
        return;
    }
    // lanes h and h + 2 hold dims x and x + 16, which share a byte: lane h < 2 takes
    // x = 8 h to 8 h + 3, lane h + 2 the four dims behind them
    uint32_t b[NG];
#pragma unroll
    for (int g = 0; g < NG; g++) {
        const uint32_t got = (uint32_t)__shfl_xor((int)(h < 2 ? c1[g] : c0[g]), 32, 64);
        b[g] = h < 2 ? c0[g] | got << 4 : got | c1[g] << 4;
    }
    const int x0 = 8 * (h & 1) + (h < 2 ? 0 : 4);
    if (whole) {
#pragma unroll
        for (int g = 0; g < NG; g++) b[g] = quad_transpose(b[g], i);
        store_dwords(out + (key >> 2) * 2 * D + (x0 + i) * (D / 8), b);
    } else if (mine) {
        // other tokens of the tile stay: a byte at a time
#pragma unroll
        for (int g = 0; g < NG; g++)
#pragma unroll
            for (int t = 0; t < 4; t++)
                out[(key >> 2) * 2 * D + (x0 + t) * (D / 8) + 4 * g + i] = (uint8_t)(b[g] >> (8 * t));
    }
}

// checks the descriptor and fills the view; `layer`: whose pages (page
// operations take all layers from layer 0 on)
int kv4_view(const cactus_hip_kv4_cache* c, size_t layer, const char* what, Kv4View* out);

}  // namespace cactus_hip
