// kv4_rope.hip -- appending to the paged 4-bit KV cache with the head norms and
// the position rotation applied on the way, and the table of the rotations.
//
//   y = x / sqrt(mean(x^2) + eps) w,   halves a, b of y at position p:
//   a cos(p f_i) - b sin(p f_i),  b cos(p f_i) + a sin(p f_i)
// Queries and keys are computed in 64 bits and rounded once, to FP16.  For the
// keys that keeps the 4-bit codes what the formula says: an FP32 sum that falls
// on the other side of an FP16 value's border moves a key by 2^-11, and where
// that crosses the border of two codes, by a seventh of its group's largest.
#include "kv4_device.h"

namespace cactus_hip {

// One rounding from 64 bits to FP16 (nearest, ties to even; FP32 in between would
// round twice): of the 52 fraction bits the upper 20 stay, the lowest of them
// set if any behind it is, which FP32 holds exactly and FP16 rounds as the whole.
__device__ __forceinline__ uint16_t f64_to_h(double x) {
    const uint64_t b = __builtin_bit_cast(uint64_t, x);
    const uint32_t hi = (uint32_t)(b >> 32) | ((uint32_t)b != 0 ? 1u : 0u);
    return f2h((float)__builtin_bit_cast(double, (uint64_t)hi << 32));
}
__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

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
    const int status = c.state[KV4_STATUS];
    const int slot = kv4_slot(c, a.seqs, req);
    if (slot < 0 || status != 0) return;
    const int len = kv4_len(c, slot), m = kv4_count(a.counts, req, a.S);
    const int pos = len - m + row;
    if (row >= m || pos < 0) return;
    const bool is_q = item < a.Hq, is_v = item >= a.Hq + c.Hkv;
    const int head = is_q ? item : is_v ? item - a.Hq - c.Hkv : item - a.Hq;
    const size_t r = (size_t)req * a.S + row;
    const uint16_t* src = (is_q ? a.q + r * a.q_stride : (is_v ? a.v : a.k) + r * a.kv_stride) + (size_t)head * D + lane;
    uint16_t x[E];
#pragma unroll
    for (int e = 0; e < E; e++) x[e] = src[64 * e];
    if (!is_v) {
        const uint16_t* w = is_q ? a.q_norm : a.k_norm;
        double y[E];
#pragma unroll
        for (int e = 0; e < E; e++) y[e] = (double)h2f(x[e]);
        if (w) {
            double ss = 0;
#pragma unroll
            for (int e = 0; e < E; e++) ss = __builtin_fma(y[e], y[e], ss);
            const double inv = 1.0 / sqrt(wave_sum_f64(ss) * (1.0 / D) + a.eps);
#pragma unroll
            for (int e = 0; e < E; e++) y[e] = y[e] * inv * (double)h2f(w[64 * e + lane]);
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
    const int page = c.table[(size_t)slot * c.max_pages + (pos >> c.ps_log2)];
    if (!kv4_page_ok(c, page)) return;
    uint8_t* out = kv4_tile(c, page, head, (pos & ((1 << c.ps_log2) - 1)) >> 4) + (is_v ? 9 * D : 0);
    const int key = pos & 15, l = lane & 31;
#pragma unroll
    for (int e = 0; e < E; e++) {
        // group 2 e + lane / 32
        uint32_t am = x[e] & 0x7FFFu;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) am = max(am, (uint32_t)__shfl_xor((int)am, o, 64));
        const uint16_t sb = kv4_scale(am);
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

// A wave takes one 16-token tile of several heads, lane 16 h + token with dims 8 h to 8 h + 7 of
// each 32-dim group, the order in which the append writes pages: the halves of a rotation are in
// one lane, and the table's values stay in registers from head to head (read anew for each they
// were twice the bytes of the rows).
// grid (tile, TILE_WAVES * heads_per_wave heads, request)
constexpr int TILE_WAVES = 4;
constexpr size_t ROPE_TILE_ROWS = 8;
constexpr int ROPE_PER_WAVE = 4;
template <int D>
__global__ void __launch_bounds__(64 * TILE_WAVES) kv4_rope_tile_kernel(RopeArgs a, int per_wave) {
    constexpr int NG = D / 32, NP = NG / 2;
    const Kv4View& c = a.c;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), key = lane & 15, h = lane >> 4;
    const int req = blockIdx.z, items = a.Hq + 2 * c.Hkv;
    const int status = c.state[KV4_STATUS];
    const int slot = kv4_slot(c, a.seqs, req);
    if (slot < 0 || status != 0) return;
    const int len = kv4_len(c, slot), first = len - kv4_count(a.counts, req, a.S);   // (negative: rows without a token)
    const int lo = max(first, 0);
    const int pos0 = (lo & ~15) + 16 * (int)blockIdx.x;
    if (pos0 >= len) return;
    const int pos = pos0 + key;
    const bool mine = pos >= lo && pos < len, whole = pos0 >= lo && pos0 + 16 <= len;
    const int at = mine ? pos : lo;
    const size_t row = (size_t)req * a.S + (at - first);
    float co[NP][8], si[NP][8];
    {
        const float* t = a.table + (size_t)at * D + 8 * h;
#pragma unroll
        for (int g = 0; g < NP; g++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const f32x4 u = *reinterpret_cast<const f32x4*>(t + 32 * g + 4 * j), v = *reinterpret_cast<const f32x4*>(t + D / 2 + 32 * g + 4 * j);
#pragma unroll
                for (int i = 0; i < 4; i++) co[g][4 * j + i] = u[i], si[g][4 * j + i] = v[i];
            }
    }
    const int page = c.table[(size_t)slot * c.max_pages + (pos0 >> c.ps_log2)];
    const int tile = (pos0 & ((1 << c.ps_log2) - 1)) >> 4;
    const int item0 = (int)blockIdx.y * TILE_WAVES * per_wave + wave;
    const auto source = [&](int item) {
        const bool is_q = item < a.Hq, is_v = item >= a.Hq + c.Hkv;
        return (is_q ? a.q + row * a.q_stride : (is_v ? a.v : a.k) + row * a.kv_stride) +
               (size_t)(is_q ? item : is_v ? item - a.Hq - c.Hkv : item - a.Hq) * D + 8 * h;
    };
    uint4 next[NG];
    if (item0 < items) {
        const uint16_t* src = source(item0);
#pragma unroll
        for (int g = 0; g < NG; g++) next[g] = *reinterpret_cast<const uint4*>(src + 32 * g);
    }
    for (int n = 0; n < per_wave; n++) {
        const int item = item0 + TILE_WAVES * n;
        if (item >= items) return;
        uint4 x[NG];
#pragma unroll
        for (int g = 0; g < NG; g++) x[g] = next[g];
        if (n + 1 < per_wave && item + TILE_WAVES < items) {
            const uint16_t* src = source(item + TILE_WAVES);
#pragma unroll
            for (int g = 0; g < NG; g++) next[g] = *reinterpret_cast<const uint4*>(src + 32 * g);
        }
        const bool is_q = item < a.Hq, is_v = item >= a.Hq + c.Hkv;
        const auto half_of = [&](int g, int j) { return h2f((uint16_t)((&x[g].x)[j / 2] >> 16 * (j & 1))); };
        if (is_q) {
            // in 32 bits: an FP16 result has no border that 2^-22 beside it matters for
            float f = 1.0f;
            if (a.q_norm) {
                float ss = 0.0f;
#pragma unroll
                for (int g = 0; g < NG; g++)
#pragma unroll
                    for (int j = 0; j < 8; j++) ss = __builtin_fmaf(half_of(g, j), half_of(g, j), ss);
                ss += __shfl_xor(ss, 16, 64);
                ss += __shfl_xor(ss, 32, 64);
                f = 1.0f / sqrtf(ss * (1.0f / D) + (float)a.eps);
            }
            uint16_t* dst = a.q_out + (row * a.Hq + item) * D + 8 * h;
#pragma unroll
            for (int g = 0; g < NP; g++) {
                uint4 wa = make_uint4(0, 0, 0, 0), wb = wa;
                if (a.q_norm) {
                    wa = *reinterpret_cast<const uint4*>(a.q_norm + 32 * g + 8 * h);
                    wb = *reinterpret_cast<const uint4*>(a.q_norm + D / 2 + 32 * g + 8 * h);
                }
                uint32_t ra[4], rb[4];
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    float u = half_of(g, j), v = half_of(g + NP, j);
                    if (a.q_norm) {
                        u = u * f * h2f((uint16_t)((&wa.x)[j / 2] >> 16 * (j & 1)));
                        v = v * f * h2f((uint16_t)((&wb.x)[j / 2] >> 16 * (j & 1)));
                    }
                    const uint32_t p = f2h(__builtin_fmaf(u, co[g][j], -(v * si[g][j]))), r = f2h(__builtin_fmaf(v, co[g][j], u * si[g][j]));
                    if (j & 1) ra[j / 2] |= p << 16, rb[j / 2] |= r << 16;
                    else ra[j / 2] = p, rb[j / 2] = r;
                }
                if (mine) {
                    *reinterpret_cast<uint4*>(dst + 32 * g) = make_uint4(ra[0], ra[1], ra[2], ra[3]);
                    *reinterpret_cast<uint4*>(dst + D / 2 + 32 * g) = make_uint4(rb[0], rb[1], rb[2], rb[3]);
                }
            }
            continue;
        }
        if (!kv4_page_ok(c, page)) return;        // (heads go up: keys and values are all that is left)
        if (!is_v) {
            double f = 1.0;
            if (a.k_norm) {
                double ss = 0.0;
#pragma unroll
                for (int g = 0; g < NG; g++)
#pragma unroll
                    for (int j = 0; j < 8; j++) ss += (double)(half_of(g, j) * half_of(g, j));     // (exact in FP32)
                ss += __shfl_xor(ss, 16, 64);
                ss += __shfl_xor(ss, 32, 64);
                f = 1.0 / sqrt(ss * (1.0 / D) + a.eps);
            }
#pragma unroll
            for (int g = 0; g < NP; g++) {
                uint4 wa = make_uint4(0, 0, 0, 0), wb = wa;
                if (a.k_norm) {
                    wa = *reinterpret_cast<const uint4*>(a.k_norm + 32 * g + 8 * h);
                    wb = *reinterpret_cast<const uint4*>(a.k_norm + D / 2 + 32 * g + 8 * h);
                }
                uint32_t ra[4], rb[4];
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    double u = half_of(g, j), v = half_of(g + NP, j);
                    if (a.k_norm) {
                        // (x w is exact in FP32)
                        u = (double)(half_of(g, j) * h2f((uint16_t)((&wa.x)[j / 2] >> 16 * (j & 1)))) * f;
                        v = (double)(half_of(g + NP, j) * h2f((uint16_t)((&wb.x)[j / 2] >> 16 * (j & 1)))) * f;
                    }
                    const double cs = co[g][j], sn = si[g][j];
                    const uint32_t p = f64_to_h(__builtin_fma(u, cs, -(v * sn))), r = f64_to_h(__builtin_fma(v, cs, u * sn));
                    if (j & 1) ra[j / 2] |= p << 16, rb[j / 2] |= r << 16;
                    else ra[j / 2] = p, rb[j / 2] = r;
                }
                x[g] = make_uint4(ra[0], ra[1], ra[2], ra[3]);
                x[g + NP] = make_uint4(rb[0], rb[1], rb[2], rb[3]);
            }
        }
        const int head = is_v ? item - a.Hq - c.Hkv : item - a.Hq;
        kv4_write_tile<D>(x, kv4_tile(c, page, head, tile) + (is_v ? 9 * D : 0), is_v, mine, whole);
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
    CH_REQUIRE(num_q_heads <= 65536, "kv4_append_rope: num_q_heads out of range");
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
    if (seq_len >= ROPE_TILE_ROWS) {
        const int per_wave = ROPE_PER_WAVE;
        const dim3 grid(ceil_div(seq_len + 15, 16), ceil_div(items, TILE_WAVES * per_wave), (unsigned)batch);
        switch (a.c.d) {
            case 64: hipLaunchKernelGGL(kv4_rope_tile_kernel<64>, grid, dim3(64 * TILE_WAVES), 0, as_stream(stream), a, per_wave); break;
            case 128: hipLaunchKernelGGL(kv4_rope_tile_kernel<128>, grid, dim3(64 * TILE_WAVES), 0, as_stream(stream), a, per_wave); break;
            default: hipLaunchKernelGGL(kv4_rope_tile_kernel<256>, grid, dim3(64 * TILE_WAVES), 0, as_stream(stream), a, per_wave);
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
