// kv4_rope.hip -- appending to the paged 4-bit KV cache with the head norms and
// the position rotation applied on the way, and the table of the rotations.
//
//   y = x / sqrt(mean(x^2) + eps) w,   halves a, b of y at position p:
//   a cos(p f_i) - b sin(p f_i),  b cos(p f_i) + a sin(p f_i)
// Keys are computed in 64 bits and rounded once, to FP16, which keeps their 4-bit
// codes what the formula says: an FP32 sum that falls on the other side of an
// FP16 value's border moves a key by 2^-11, and where that crosses the border of
// two codes, by a seventh of its group's largest.  Queries have no codes: 64 bits
// where a wave has one row, 32 where it has many, rounded once too.
//
// Single rows are bound by the chain of loads (length, position, rotation and page), prompts by
// memory with the vector units 60% busy.  Four prompts of up to 2048 rows (6427 in all), 16 query
// and 8 KV heads of 128 dims with norms: 24.7 us in a graph, 26.4 traced; 89.7 MB, 3.6 TB/s (16 more
// query heads add 52.6 MB in 11.6 us, 4.5 TB/s; the keys' 64-bit sums are what the rest waits
// for).  The same with 64 dims 13.6 us (3.3 TB/s), with 256 dims 47.1 (3.8), with 4 and 1 heads of 256
// dims 11.8 (3.5).  64 single rows 4.3 us traced, one row of 4 and 1 heads of 256 dims 3.9.  Queries
// go past the caches: 39.9 -> 38.4 us with the read of the keys and values.
#include "kv4_device.h"

namespace cactus_hip {

// One rounding from 64 bits to FP16 (nearest, ties to even; FP32 in between would
// round twice): of the 52 fraction bits the upper 20 stay, the lowest of them
// set if any behind it is, which FP32 holds exactly and FP16 rounds as the whole.
__device__ __forceinline__ uint16_t f64_to_h(double x) {
    const uint64_t b = __builtin_bit_cast(uint64_t, x);
    const uint32_t hi = (uint32_t)(b >> 32) | min((uint32_t)b, 1u);
    return f2h((float)__builtin_bit_cast(double, (uint64_t)hi << 32));
}
// 1 / sqrt(v): the approximation's 2^-24 or so squared twice by Newton's steps; 0 for
// infinity and infinity for 0, as the formula has them
__device__ __forceinline__ double rsqrt_f64(double v) {
    const double y0 = __builtin_amdgcn_rsq(v);
    double y = y0;
#pragma unroll
    for (int i = 0; i < 2; i++) y = __builtin_fma(0.5 * y, __builtin_fma(-(v * y), y, 1.0), y);
    return v > 0.0 && v < __builtin_inf() ? y : y0;
}
template <int CTRL>
__device__ __forceinline__ double dpp_f64(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, 0xF, 0xF, true);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CTRL, 0xF, 0xF, true);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double wave_sum_f64(double v) {
    v += dpp_f64<0xB1>(v);        // within rows of 16 lanes
    v += dpp_f64<0x4E>(v);
    v += dpp_f64<0x141>(v);
    v += dpp_f64<0x140>(v);
    const auto of = [&](int l) {
        const uint64_t b = __builtin_bit_cast(uint64_t, v);
        const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, l), hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), l);
        return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
    };
    return (of(0) + of(16)) + (of(32) + of(48));
}

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct RopeArgs {
    Kv4View c;
    const int32_t* seqs;
    const int32_t* counts;
    const uint16_t* q;
    uint16_t* q_out;
    const uint16_t* k;
    const uint16_t* v;
    const uint16_t* q_norm;
    const uint16_t* k_norm;
    const float* table;      // [position][cos, sin][d / 2]
    size_t q_stride, kv_stride;
    int Hq, S;
    double eps;
};

// A wave takes a head's row: dims 64 e + lane, e < D / 64, so that the halves of a
// rotation are in one lane (D 128, 256) or in lanes 32 apart (D 64).
// grid (row, 4 heads each, request), heads in the order q, k, v
constexpr int ROW_WAVES = 4;
template <int D>
__global__ void __launch_bounds__(64 * ROW_WAVES) kv4_rope_row_kernel(RopeArgs a) {
    constexpr int E = D / 64, NG = D / 32;
    const Kv4View& c = a.c;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int item = (int)blockIdx.y * ROW_WAVES + wave, row = blockIdx.x, req = blockIdx.z;
    if (item >= a.Hq + 2 * c.Hkv) return;
    const bool is_q = item < a.Hq, is_v = item >= a.Hq + c.Hkv;
    const int head = is_q ? item : is_v ? item - a.Hq - c.Hkv : item - a.Hq;
    const size_t r = (size_t)req * a.S + row;
    const uint16_t* src = (is_q ? a.q + r * a.q_stride : (is_v ? a.v : a.k) + r * a.kv_stride) + (size_t)head * D + lane;
    const uint16_t* w = is_q ? a.q_norm : is_v ? nullptr : a.k_norm;
    // what does not hang on the position is on its way while the slot's length is looked up
    uint16_t x[E], wn[E] = {};
#pragma unroll
    for (int e = 0; e < E; e++) x[e] = src[64 * e];
    if (w) {
#pragma unroll
        for (int e = 0; e < E; e++) wn[e] = w[64 * e + lane];
    }
    const int status = c.state[KV4_STATUS];
    const int slot = kv4_slot(c, a.seqs, req);
    if (slot < 0) return;
    const int len = kv4_len(c, slot), m = kv4_count(a.counts, req, a.S);
    const int pos = len - m + row;
    if (status != 0 || row >= m || pos < 0) return;
    const int page = is_q ? 0 : c.table[(size_t)slot * c.max_pages + (pos >> c.ps_log2)];
    if (!is_v) {
        double y[E];
#pragma unroll
        for (int e = 0; e < E; e++) y[e] = (double)h2f(x[e]);
        if (w) {
            double ss = 0;
#pragma unroll
            for (int e = 0; e < E; e++) ss = __builtin_fma(y[e], y[e], ss);
            const double inv = rsqrt_f64(wave_sum_f64(ss) * (1.0 / D) + a.eps);
#pragma unroll
            for (int e = 0; e < E; e++) y[e] = y[e] * (double)h2f(wn[e]) * inv;
        }
        const float* t = a.table + (size_t)pos * D;
        if constexpr (E == 1) {
            const double co = t[lane & 31], si = t[32 + (lane & 31)], o = __shfl_xor(y[0], 32, 64);
            x[0] = f64_to_h(__builtin_fma(y[0], co, lane < 32 ? -(o * si) : o * si));
        } else {
#pragma unroll
            for (int e = 0; e < E / 2; e++) {
                const double co = t[64 * e + lane], si = t[D / 2 + 64 * e + lane], u = y[e], v = y[e + E / 2];
                x[e] = f64_to_h(__builtin_fma(u, co, -(v * si)));
                x[e + E / 2] = f64_to_h(__builtin_fma(v, co, u * si));
            }
        }
    }
    if (is_q) {
        uint16_t* dst = a.q_out + (r * a.Hq + head) * D + lane;
#pragma unroll
        for (int e = 0; e < E; e++) dst[64 * e] = x[e];
        return;
    }
    if (!kv4_page_ok(c, page)) return;
    uint8_t* out = kv4_tile(c, page, head, (pos & ((1 << c.ps_log2) - 1)) >> 4) + (is_v ? 9 * D : 0);
    const int key = pos & 15, l = lane & 31;
#pragma unroll
    for (int e = 0; e < E; e++) {
        // group 2 e + lane / 32
        const uint16_t sb = kv4_scale((uint32_t)half_wave_max((float)(x[e] & 0x7FFFu)));     // (bits as numbers)
        const float s = h2f(sb), inv = s > 0.0f ? 1.0f / s : 0.0f;
        const uint32_t code = s > 0.0f ? kv4_code(x[e], inv) & 15u : 8u;
        const int g = 2 * e + (lane >> 5);
        if (l == 0) reinterpret_cast<uint16_t*>(out + 8 * D)[((key >> 2) * NG + g) * 4 + (key & 3)] = sb;
        if (is_v) {      // dims x and x + 16 of a group share a byte
            const uint32_t b = code | (uint32_t)__shfl_xor((int)code, 16, 64) << 4;
            if (!(lane & 16)) out[(key >> 2) * 2 * D + (lane & 15) * NG * 4 + g * 4 + (key & 3)] = (uint8_t)b;
        } else {         // dims of neighbouring groups do
            const uint32_t b = code | (uint32_t)__shfl_xor((int)code, 32, 64) << 4;
            if (lane < 32) out[(l >> 3) * 2 * D + key * (D / 8) + e * 8 + (l & 7)] = (uint8_t)b;
        }
    }
}

// Prompts.  Queries and keys: D / 16 lanes take a token, each two pieces of 8 dims that a rotation
// pairs (so that neighbouring lanes load neighbouring bytes: with a lane per token, as the pages
// have them, the L1 took a row's piece at a time), and a wave 1024 / D tokens of several heads one after
// the other, the rotations staying in registers.  In each 8 lanes the pieces are 0 1 2 3 7 6 5 4:
// the four of a scale's group are a quad, and the two whose codes share bytes mirror each other.
// Values: a 16-token tile per wave in the pages' order, as the append without rotation.
// grid (tile, 4 units each, request); units: TPT token groups times ceil(q and k heads / heads),
// then ceil(v heads / heads)
constexpr int TILE_WAVES = 4;
// Rows of a call from which tiles are faster than a wave per row and head (8 sequences of 8 rows 5.8
// against 6.2 us, of 16 rows 6.7 against 6.4; 64 of 4 rows 8.5 against 10.0, of 8 rows 11.6
// against 10.9: shorter sequences leave tiles too empty), and waves from which one takes two
// heads, by them one and two heads per wave (us):
//   waves        16 / 8 of 64     16 / 8 of 128    16 / 8 of 256    32 / 8 of 128    4 / 1 of 256
//   2000          4.6   5.5        4.9   6.7        6.4   9.7        4.7   5.8        6.3   5.7
//   6100          9.2   7.3        9.4   9.0       10.8  10.8        9.0   8.9       10.8   9.3
//   8200         10.5  10.7       11.1  11.5       13.1  13.2       10.7  11.1       13.0  11.3
//   12300        14.2  13.4       14.4  14.1       17.1  17.1       14.0  13.3       16.7  14.6
//   28000        26.9  24.8       32.3  29.2       34.7  32.0       30.7  27.6       36.1  30.5
constexpr size_t ROPE_TILE_ROWS = 128, ROPE_TILE_SEQ = 8, ROPE_TWO_HEADS = 8192;
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, true);
}
template <int D>
__global__ void __launch_bounds__(64 * TILE_WAVES, 3) kv4_rope_tile_kernel(RopeArgs a, int heads) {
    constexpr int NG = D / 32, LPT = D / 16, TPW = 64 / LPT, TPT = 16 / TPW;
    const Kv4View& c = a.c;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int req = blockIdx.z, rot = a.Hq + c.Hkv, chunks = (rot + heads - 1) / heads;
    const int unit = (int)blockIdx.y * TILE_WAVES + wave;
    if (unit >= TPT * chunks) {
        const int h0 = (unit - TPT * chunks) * heads;
        if (h0 >= c.Hkv) return;
        const int status = c.state[KV4_STATUS];
        const int slot = kv4_slot(c, a.seqs, req);
        if (slot < 0 || status != 0) return;
        const int len = kv4_len(c, slot), first = len - kv4_count(a.counts, req, a.S);   // (negative: rows without a token)
        const int lo = max(first, 0);
        const int pos0 = (lo & ~15) + 16 * (int)blockIdx.x;
        if (pos0 >= len) return;
        const int key = lane & 15, h = lane >> 4, pos = pos0 + key;
        const int page = c.table[(size_t)slot * c.max_pages + (pos0 >> c.ps_log2)];
        if (!kv4_page_ok(c, page)) return;
        const bool mine = pos >= lo && pos < len, whole = pos0 >= lo && pos0 + 16 <= len;
        const uint16_t* src = a.v + ((size_t)req * a.S + ((mine ? pos : lo) - first)) * a.kv_stride + 8 * h;
        for (int head = h0; head < min(h0 + heads, c.Hkv); head++) {
            uint4 x[NG];
#pragma unroll
            for (int g = 0; g < NG; g++) x[g] = *reinterpret_cast<const uint4*>(src + (size_t)head * D + 32 * g);
            kv4_write_tile<D>(x, kv4_tile(c, page, head, (pos0 & ((1 << c.ps_log2) - 1)) >> 4) + 9 * D, true, mine, whole);
        }
        return;
    }
    const int s = lane & (LPT - 1), j = LPT == 4 || !(s & 4) ? s : s ^ 3;       // piece (the other is j + LPT)
    const int r0 = 16 * (int)blockIdx.x + unit / chunks * TPW, in_s = r0 + lane / LPT;
    if (r0 >= a.S) return;
    const size_t row = (size_t)req * a.S + min(in_s, a.S - 1);
    const int item0 = unit % chunks * heads, item1 = min(item0 + heads, rot);
    const auto source = [&](int item) {
        return (item < a.Hq ? a.q + row * a.q_stride + (size_t)item * D : a.k + row * a.kv_stride + (size_t)(item - a.Hq) * D) + 8 * j;
    };
    const u32x4 ones = {0x3C003C00u, 0x3C003C00u, 0x3C003C00u, 0x3C003C00u};      // the weights of no norm
    // the first rows do not hang on the position: on their way while the slot's length is looked up
    u32x4 next[2];
    {
        const uint16_t* p = source(item0);
        next[0] = *reinterpret_cast<const u32x4*>(p);
        next[1] = *reinterpret_cast<const u32x4*>(p + D / 2);
    }
    const int status = c.state[KV4_STATUS];
    const int slot = kv4_slot(c, a.seqs, req);
    if (slot < 0) return;
    const int len = kv4_len(c, slot), m = kv4_count(a.counts, req, a.S);
    if (status != 0 || r0 >= m) return;
    const int pos = len - m + in_s;
    const bool mine = in_s < m && pos >= 0;
    const int at = mine ? pos : 0;
    float co[8], si[8];
    {
        const float* t = a.table + (size_t)at * D + 8 * j;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const f32x4 u = *reinterpret_cast<const f32x4*>(t + 4 * i), v = *reinterpret_cast<const f32x4*>(t + D / 2 + 4 * i);
#pragma unroll
            for (int k = 0; k < 4; k++) co[4 * i + k] = u[k], si[4 * i + k] = v[k];
        }
    }
    // the tile of the lane's token
    const int page = item1 > a.Hq ? c.table[(size_t)slot * c.max_pages + (at >> c.ps_log2)] : 0;
    const bool keeps = mine && kv4_page_ok(c, page);
    const int key = at & 15;
    uint8_t* tile = kv4_tile(c, keeps ? page : 0, 0, (at & ((1 << c.ps_log2) - 1)) >> 4);
    const size_t head_bytes = (size_t)(18 * D) << (c.ps_log2 - 4);
    for (int item = item0; item < item1; item++) {
        u32x4 x[2] = {next[0], next[1]}, w[2] = {ones, ones};
        if (item + 1 < item1) {
            const uint16_t* p = source(item + 1);
            next[0] = *reinterpret_cast<const u32x4*>(p);
            next[1] = *reinterpret_cast<const u32x4*>(p + D / 2);
        }
        const uint16_t* norm = item < a.Hq ? a.q_norm : a.k_norm;
        if (norm) {
            w[0] = *reinterpret_cast<const u32x4*>(norm + 8 * j);
            w[1] = *reinterpret_cast<const u32x4*>(norm + D / 2 + 8 * j);
        }
        const auto xh = [&](int u, int i) { return h2f((uint16_t)(x[u][i / 2] >> 16 * (i & 1))); };
        float xw[2][8];                           // times the weights, exact (fma_mix takes FP16 operands as they are)
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
            for (int i = 0; i < 8; i++) xw[u][i] = __builtin_fmaf(xh(u, i), h2f((uint16_t)(w[u][i / 2] >> 16 * (i & 1))), -0.0f);
        if (item < a.Hq) {
            // in 32 bits: an FP16 result has no border that 2^-22 beside it matters for
            float f = 1.0f;
            if (norm) {
                float ss = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; i++) ss = __builtin_fmaf(xh(0, i), xh(0, i), __builtin_fmaf(xh(1, i), xh(1, i), ss));
                ss += dpp_move_keep<0xB1>(ss);
                ss += dpp_move_keep<0x4E>(ss);
                if constexpr (LPT >= 8) ss += dpp_move_keep<0x141>(ss);
                if constexpr (LPT >= 16) ss += dpp_move_keep<0x140>(ss);
                f = __builtin_amdgcn_rsqf(ss * (1.0f / D) + (float)a.eps);
            }
            h16x2 r[2][4];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float cf = co[i] * f, sf = si[i] * f;
                r[0][i / 2][i & 1] = (_Float16)__builtin_fmaf(xw[0][i], cf, -(xw[1][i] * sf));
                r[1][i / 2][i & 1] = (_Float16)__builtin_fmaf(xw[1][i], cf, xw[0][i] * sf);
            }
            if (mine) {
                uint16_t* dst = a.q_out + (row * a.Hq + item) * D + 8 * j;
#pragma unroll
                for (int u = 0; u < 2; u++)
                    __builtin_nontemporal_store((u32x4){__builtin_bit_cast(uint32_t, r[u][0]), __builtin_bit_cast(uint32_t, r[u][1]),
                                                        __builtin_bit_cast(uint32_t, r[u][2]), __builtin_bit_cast(uint32_t, r[u][3])},
                                                reinterpret_cast<u32x4*>(dst + u * (D / 2)));
            }
            continue;
        }
        double f = 1.0;
        if (norm) {
            double ss = 0.0;
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int i = 0; i < 8; i++) ss += (double)__builtin_fmaf(xh(u, i), xh(u, i), 0.0f);      // (exact in FP32)
            ss += dpp_f64<0xB1>(ss);
            ss += dpp_f64<0x4E>(ss);
            if constexpr (LPT >= 8) ss += dpp_f64<0x141>(ss);
            if constexpr (LPT >= 16) ss += dpp_f64<0x140>(ss);
            f = rsqrt_f64(ss * (1.0 / D) + a.eps);
        }
        uint16_t r[2][8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const double u = (double)xw[0][i] * f, v = (double)xw[1][i] * f, cs = co[i], sn = si[i];
            r[0][i] = f64_to_h(__builtin_fma(u, cs, -(v * sn)));
            r[1][i] = f64_to_h(__builtin_fma(v, cs, u * sn));
        }
        uint8_t* out = tile + (size_t)(item - a.Hq) * head_bytes;
        uint32_t b[2][2];                         // codes of a piece, a byte each
        uint16_t sb[2];
#pragma unroll
        for (int u = 0; u < 2; u++) {
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < 8; i++) m = max(m, (uint32_t)(r[u][i] & 0x7FFFu));
            m = max(m, dpp<0xB1>(m));
            m = max(m, dpp<0x4E>(m));
            sb[u] = kv4_scale(m);
            const float sc = h2f(sb[u]), inv = sc > 0.0f ? 1.0f / sc : 0.0f;
            uint32_t k[8];
#pragma unroll
            for (int i = 0; i < 8; i++) k[i] = kv4_code(r[u][i], inv);
            b[u][0] = sc > 0.0f ? low_bytes(k[0], k[1], k[2], k[3]) : 0x08080808u;
            b[u][1] = sc > 0.0f ? low_bytes(k[4], k[5], k[6], k[7]) : 0x08080808u;
        }
        uint2 bytes;
        int p = 0;                                // 64-dim block of the bytes
        if constexpr (LPT == 4) {
            bytes = make_uint2(b[0][0] | b[1][0] << 4, b[0][1] | b[1][1] << 4);
        } else {
            // lanes with the low nibbles' pieces finish the first half's block, their mirrors the second's
            const bool high = s & 4;
            const uint32_t g0 = dpp<0x141>(high ? b[0][0] : b[1][0]), g1 = dpp<0x141>(high ? b[0][1] : b[1][1]);
            bytes = high ? make_uint2(g0 | b[1][0] << 4, g1 | b[1][1] << 4) : make_uint2(b[0][0] | g0 << 4, b[0][1] | g1 << 4);
            p = (j >> 3) + (high ? LPT / 8 : 0);
        }
        if (keeps) {
            *reinterpret_cast<uint2*>(out + (j & 3) * 2 * D + key * (D / 8) + 8 * p) = bytes;
            if ((s & 3) < 2) {
                const int g = (j >> 2) + (s & 1 ? LPT / 4 : 0);
                reinterpret_cast<uint16_t*>(out + 8 * D)[((key >> 2) * NG + g) * 4 + (key & 3)] = s & 1 ? sb[1] : sb[0];
            }
        }
    }
}

// angles in 64 bits: p f up to 2^31 has 21 bits behind the point left
__global__ void __launch_bounds__(256) rope_table_kernel(float* table, size_t positions, int half, double log2_theta) {
    const size_t n = positions * half;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) {
        const size_t p = i / half;
        const int j = (int)(i % half);
        const double angle = (double)p * exp2(-log2_theta * j / half);
        double s, co;
        sincos(angle, &s, &co);
        table[p * 2 * half + j] = (float)co;
        table[p * 2 * half + half + j] = (float)s;
    }
}

}  // namespace cactus_hip

using namespace cactus_hip;

extern "C" {

int cactus_hip_rope_table_f32(float* table, size_t positions, size_t head_dim, float theta, void* stream) {
    CH_REQUIRE(head_dim >= 2 && head_dim % 2 == 0 && head_dim <= 65536, "rope_table: head_dim is even, from 2 to 65536");
    CH_REQUIRE(theta > 0.0f && theta < __builtin_inff(), "rope_table: theta is a positive number");
    CH_REQUIRE(positions < (1ull << 31), "rope_table: positions out of range");
    if (positions == 0) return CACTUS_HIP_OK;
    CH_REQUIRE(table, "rope_table: null pointer");
    const size_t blocks = (positions * (head_dim / 2) + 255) / 256;
    hipLaunchKernelGGL(rope_table_kernel, dim3((unsigned)(blocks < 8192 ? blocks : 8192)), dim3(256), 0, as_stream(stream), table,
                       positions, (int)(head_dim / 2), log2((double)theta));
    return check_launch("rope_table");
}

int cactus_hip_kv4_append_rope_f16(const cactus_hip_kv4_cache* cache, size_t layer, const int32_t* seqs,
                                   const int32_t* counts, const uint16_t* q, size_t q_stride, uint16_t* q_out,
                                   size_t num_q_heads, const uint16_t* k, const uint16_t* v, size_t kv_stride,
                                   const uint16_t* q_norm, const uint16_t* k_norm, float eps, const float* table,
                                   size_t table_positions, size_t batch, size_t seq_len, void* stream) {
    RopeArgs a;
    int rc = kv4_view(cache, layer, "kv4_append_rope", &a.c);
    if (rc) return rc;
    if (batch == 0 || seq_len == 0) return CACTUS_HIP_OK;
    CH_REQUIRE(k && v && table && (num_q_heads == 0 || (q && q_out)), "kv4_append_rope: null pointer");
    CH_REQUIRE(num_q_heads <= 16384, "kv4_append_rope: num_q_heads out of range");
    const auto aligned = [](const void* p) { return ((uintptr_t)p & 15) == 0; };
    CH_REQUIRE(aligned(k) && aligned(v) && kv_stride % 8 == 0 &&
                   (num_q_heads == 0 || (aligned(q) && aligned(q_out) && q_stride % 8 == 0)),
               "kv4_append_rope: rows are not 16-byte aligned");
    CH_REQUIRE(aligned(table) && aligned(q_norm) && aligned(k_norm), "kv4_append_rope: norms or table not 16-byte aligned");
    CH_REQUIRE(kv_stride >= cache->kv_heads * cache->head_dim, "kv4_append_rope: kv_stride is shorter than a row");
    CH_REQUIRE(num_q_heads == 0 || q_stride >= num_q_heads * cache->head_dim, "kv4_append_rope: q_stride is shorter than a row");
    CH_REQUIRE(num_q_heads == 0 || q_out != q || q_stride == num_q_heads * cache->head_dim,
               "kv4_append_rope: q in place are dense rows");
    CH_REQUIRE(eps >= 0.0f && eps < __builtin_inff(), "kv4_append_rope: eps is a number from 0 on");
    CH_REQUIRE(table_positions >= cache->max_pages * cache->page_size,
               "kv4_append_rope: table_positions is less than a slot's tokens, max_pages * page_size");
    CH_REQUIRE(batch <= cache->max_seqs && batch <= 65535, "kv4_append_rope: more requests than slots, or than 65535");
    CH_REQUIRE(seq_len < (1u << 24), "kv4_append_rope: seq_len out of range");
    a.seqs = seqs;
    a.counts = counts;
    a.q = q;
    a.q_out = q_out;
    a.k = k;
    a.v = v;
    a.q_norm = q_norm;
    a.k_norm = k_norm;
    a.table = table;
    a.q_stride = q_stride;
    a.kv_stride = kv_stride;
    a.Hq = (int)num_q_heads;
    a.S = (int)seq_len;
    a.eps = eps;
    const size_t items = num_q_heads + 2 * cache->kv_heads;
    if (seq_len >= ROPE_TILE_SEQ && batch * seq_len >= ROPE_TILE_ROWS) {
        const auto units = [&](size_t heads) {
            return cache->head_dim / 64 * ceil_div(num_q_heads + cache->kv_heads, heads) + ceil_div(cache->kv_heads, heads);
        };
        const int heads = batch * ceil_div(seq_len, 16) * units(1) < ROPE_TWO_HEADS ? 1 : 2;
        const dim3 grid(ceil_div(seq_len + 15, 16), ceil_div(units(heads), TILE_WAVES), (unsigned)batch);
        switch (a.c.d) {
            case 64: hipLaunchKernelGGL(kv4_rope_tile_kernel<64>, grid, dim3(64 * TILE_WAVES), 0, as_stream(stream), a, heads); break;
            case 128: hipLaunchKernelGGL(kv4_rope_tile_kernel<128>, grid, dim3(64 * TILE_WAVES), 0, as_stream(stream), a, heads); break;
            default: hipLaunchKernelGGL(kv4_rope_tile_kernel<256>, grid, dim3(64 * TILE_WAVES), 0, as_stream(stream), a, heads);
        }
        return check_launch("kv4_append_rope");
    }
    const dim3 grid((unsigned)seq_len, ceil_div(items, ROW_WAVES), (unsigned)batch);
    switch (a.c.d) {
        case 64: hipLaunchKernelGGL(kv4_rope_row_kernel<64>, grid, dim3(64 * ROW_WAVES), 0, as_stream(stream), a); break;
        case 128: hipLaunchKernelGGL(kv4_rope_row_kernel<128>, grid, dim3(64 * ROW_WAVES), 0, as_stream(stream), a); break;
        default: hipLaunchKernelGGL(kv4_rope_row_kernel<256>, grid, dim3(64 * ROW_WAVES), 0, as_stream(stream), a);
    }
    return check_launch("kv4_append_rope");
}

}  // extern "C"
