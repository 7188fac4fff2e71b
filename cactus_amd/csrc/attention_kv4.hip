// attention_kv4.hip -- attention over the paged 4-bit KV cache.
//
//   o = sum_j softmax_j(scale q.k_j) v_j,  k_j = s (u - 8), v_j likewise,
// u the stored code + 8 and s the group's scale.  A workgroup takes up to 16
// query vectors (row, query head) of one KV head as the columns of
// v_mfma_f32_16x16x32_f16:
//   scores  S^T = K Q^T, one product per 32-dim group g with the raw codes:
//           u read as an FP16 subnormal (u 2^-24, one AND per two codes; the
//           high nibble of a byte 16 u 2^-24), so that
//           q.k = 2^24 sum_g s_g ((u 2^-24).q_g - (8 2^-24).q_g),
//           the second product being the same for every key: it is the
//           accumulator's start
//   output  O^T = V^T P'^T_g with P'_g = fp16(p s_g): the lane's scores are
//           already the operand's lane order; the 8 of u - 8 comes off once at
//           the end through sum_j P'_g (a product with a constant)
// The running maximum and the sum are FP32, kept per column.  The weights are
// rounded to FP16 after the scale (2^-12 relative each): the matrix
// instruction takes them so, and the sum of thousands averages it out.
#include "kv4_device.h"

#include <algorithm>
#include <math.h>

namespace cactus_hip {

typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct Kv4AttnArgs {
    Kv4View c;
    const int32_t* seqs;
    const int32_t* counts;
    const uint16_t* q;
    uint16_t* o;
    size_t q_stride;
    int B, S, Hq, G;          // G query heads per KV head
    int window, sink, causal; // window 0: none
    float scale;              // times log2(e): the softmax runs in powers of two
};

// rows and keys of one request
struct Kv4Seq {
    int slot, len, rows;      // tokens; rows that stand at the last positions
    int main0, sinks, steps;  // 32-key steps: [0, sinks) and from main0 on; steps in all
};
constexpr int KV4_STEP = 32;

__device__ __forceinline__ Kv4Seq kv4_seq(const Kv4AttnArgs& a, int b) {
    Kv4Seq s;
    s.slot = kv4_slot(a.c, a.seqs, b);
    s.rows = s.slot < 0 ? 0 : kv4_count(a.counts, b, a.S);
    s.len = s.slot < 0 ? 0 : kv4_len(a.c, s.slot);
    const int p0 = s.len - s.rows;                       // first row's position: its window reaches furthest back
    int lo = a.window > 0 && p0 > a.window ? p0 - a.window : 0;
    s.main0 = lo / KV4_STEP;
    s.sinks = a.window > 0 ? min((min(a.sink, s.len) + KV4_STEP - 1) / KV4_STEP, s.main0) : 0;
    s.steps = s.sinks + (s.len + KV4_STEP - 1) / KV4_STEP - s.main0;
    return s;
}

// whether the row at position p sees key j of n
__device__ __forceinline__ bool kv4_sees(const Kv4AttnArgs& a, int p, int j, int n) {
    return j < n && (!a.causal || j <= p) && (a.window == 0 || p - j <= a.window || j < a.sink);
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ h16x8 frag(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __builtin_bit_cast(h16x8, (u32x4){a, b, c, d});
}
// The low nibbles of 8 bytes (bytes 0, 2, 1, 3 of each word) as FP16 u 2^-24,
// and the high ones as 16 u 2^-24
__device__ __forceinline__ h16x8 low_codes(uint32_t w0, uint32_t w1) {
    const uint32_t m = 0x000F000Fu;
    return frag(w0 & m, (w0 >> 8) & m, w1 & m, (w1 >> 8) & m);
}
__device__ __forceinline__ h16x8 high_codes(uint32_t w0, uint32_t w1) {
    const uint32_t m = 0x00F000F0u;
    return frag(w0 & m, (w0 >> 8) & m, w1 & m, (w1 >> 8) & m);
}
// -8 as those products see it: -8 2^-24 and -16 8 2^-24
__device__ __forceinline__ h16x8 minus8(bool high) {
    const uint32_t m = high ? 0x80808080u : 0x80088008u;
    return frag(m, m, m, m);
}
// eight consecutive values in the order of the codes' bytes 0, 2, 1, 3, 4, 6, 5, 7
__device__ __forceinline__ h16x8 code_order(uint4 u) {
    return frag(__builtin_amdgcn_perm(u.y, u.x, 0x05040100u), __builtin_amdgcn_perm(u.y, u.x, 0x07060302u),
                __builtin_amdgcn_perm(u.w, u.z, 0x05040100u), __builtin_amdgcn_perm(u.w, u.z, 0x07060302u));
}
__device__ __forceinline__ f32x4 mfma16(h16x8 a, h16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ uint32_t pack_h(float a, float b) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    const h2 v = {(_Float16)a, (_Float16)b};
    return __builtin_bit_cast(uint32_t, v);
}

// a wave's running softmax and output sums of 16 columns
template <int D>
struct Kv4State {
    float m, l;                   // column's maximum (log2 units), this lane's part of the sum
    f32x4 acc[D / 16];            // O^T 2^-24 (odd 16-dim blocks 16 times that) before the 8 comes off
    f32x4 off[D / 32];            // -8 2^-24 sum p s_g, every row the same
};

constexpr int KV4_WAVES = 4;
constexpr float LOG2E_F = 1.4426950408889634f;

template <int D>
__global__ void __launch_bounds__(64 * KV4_WAVES) attn_kv4_kernel(Kv4AttnArgs a) {
    constexpr int NG = D / 32, NB = D / 16, OS = D + 4;
    __shared__ __align__(16) float o_sh[KV4_WAVES][16][OS];
    __shared__ float m_sh[KV4_WAVES][16], l_sh[KV4_WAVES][16];
    const int lane = threadIdx.x & 63, col = lane & 15, h = lane >> 4;
    const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int cg = blockIdx.x, head = blockIdx.y, b = blockIdx.z;
    const Kv4Seq sq = kv4_seq(a, b);
    const int ncol = min(16, sq.rows * a.G - 16 * cg);
    if (ncol <= 0) return;
    const Kv4View& c = a.c;

    // this lane's column: row, query head and position
    const int vec = 16 * cg + col, row = vec / a.G;
    const bool live = col < ncol;
    const int pos = sq.len - sq.rows + row;
    h16x8 qf[NG];
    f32x4 start[NG];
#pragma unroll
    for (int g = 0; g < NG; g++) {
        uint4 u = make_uint4(0, 0, 0, 0);
        if (live)
            u = *reinterpret_cast<const uint4*>(a.q + ((size_t)b * a.S + row) * a.q_stride +
                                                (size_t)(head * a.G + vec % a.G) * D + 32 * g + 8 * h);
        qf[g] = code_order(u);
        start[g] = mfma16(minus8(g & 1), qf[g], (f32x4){0, 0, 0, 0});
    }
    Kv4State<D> st;
    st.m = -__builtin_inff();
    st.l = 0.0f;
#pragma unroll
    for (int i = 0; i < NB; i++) st.acc[i] = (f32x4){0, 0, 0, 0};
#pragma unroll
    for (int g = 0; g < NG; g++) st.off[g] = (f32x4){0, 0, 0, 0};
    const float kscale = a.scale * 16777216.0f;

    for (int i = wid; i < sq.steps; i += KV4_WAVES) {
        const int key0 = KV4_STEP * (i < sq.sinks ? i : sq.main0 + i - sq.sinks);
        float x[2][4];
        const uint8_t* tile[2];
        bool there[2];
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const int k0 = key0 + 16 * t;
            int page = -1;
            if (k0 < sq.len) page = c.table[(size_t)sq.slot * c.max_pages + (k0 >> c.ps_log2)];
            page = __builtin_amdgcn_readfirstlane(page);
            there[t] = kv4_page_ok(c, page);
            tile[t] = kv4_tile(c, there[t] ? page : 0, head, (k0 & ((1 << c.ps_log2) - 1)) >> 4);
        }
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const uint32_t* kc = reinterpret_cast<const uint32_t*>(tile[t] + lane * (D / 8));
            const uint16_t* ks = reinterpret_cast<const uint16_t*>(tile[t] + 8 * D + h * (D / 4));
            float even[4] = {0, 0, 0, 0}, odd[4] = {0, 0, 0, 0};
#pragma unroll
            for (int p = 0; p < NG / 2; p++) {
                const uint32_t w0 = kc[2 * p], w1 = kc[2 * p + 1];
                const f32x4 lo = mfma16(low_codes(w0, w1), qf[2 * p], start[2 * p]);
                const f32x4 hi = mfma16(high_codes(w0, w1), qf[2 * p + 1], start[2 * p + 1]);
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    even[r] = __builtin_fmaf(lo[r], h2f(ks[8 * p + r]), even[r]);
                    odd[r] = __builtin_fmaf(hi[r], h2f(ks[8 * p + 4 + r]), odd[r]);
                }
            }
#pragma unroll
            for (int r = 0; r < 4; r++) {
                x[t][r] = __builtin_fmaf(odd[r], kscale * 0.0625f, even[r] * kscale);
                const int j = key0 + 16 * t + 4 * h + r;
                if (!(there[t] && kv4_sees(a, pos, j, sq.len))) x[t][r] = -__builtin_inff();
            }
        }
        // the column's maximum over the step (a NaN score reaches the sum by itself)
        float mx = x[0][0];
#pragma unroll
        for (int r = 1; r < 8; r++) mx = __builtin_fmaxf(mx, x[r >> 2][r & 3]);
        mx = __builtin_fmaxf(mx, __shfl_xor(mx, 16, 64));
        mx = __builtin_fmaxf(mx, __shfl_xor(mx, 32, 64));
        const float m = __builtin_fmaxf(st.m, mx);
        const float base = m > -__builtin_inff() ? m : 0.0f;
        const float f = exp2_fast(st.m - base);       // 0 where nothing was there
        st.m = m;
        st.l *= f;
#pragma unroll
        for (int i2 = 0; i2 < NB; i2++) st.acc[i2] *= f;
#pragma unroll
        for (int g = 0; g < NG; g++) st.off[g] *= f;
        float p[2][4];
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                p[t][r] = exp2_fast(x[t][r] - base);
                st.l += p[t][r];
            }
#pragma unroll
        for (int g = 0; g < NG; g++) {
            float w[2][4];
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const uint16_t* vs = reinterpret_cast<const uint16_t*>(tile[t] + 17 * D + h * (D / 4)) + 4 * g;
#pragma unroll
                for (int r = 0; r < 4; r++)    // a key that is not seen adds nothing, whatever its scale is
                    w[t][r] = x[t][r] == -__builtin_inff() ? 0.0f : p[t][r] * h2f(vs[r]);
            }
            const h16x8 pf = frag(pack_h(w[0][0], w[0][2]), pack_h(w[0][1], w[0][3]), pack_h(w[1][0], w[1][2]),
                                  pack_h(w[1][1], w[1][3]));
            const uint32_t v0 = *reinterpret_cast<const uint32_t*>(tile[0] + 9 * D + lane * (D / 8) + 4 * g);
            const uint32_t v1 = *reinterpret_cast<const uint32_t*>(tile[1] + 9 * D + lane * (D / 8) + 4 * g);
            st.acc[2 * g] = mfma16(low_codes(v0, v1), pf, st.acc[2 * g]);
            st.acc[2 * g + 1] = mfma16(high_codes(v0, v1), pf, st.acc[2 * g + 1]);
            st.off[g] = mfma16(minus8(false), pf, st.off[g]);
        }
    }

    // the waves' shares of the keys meet
    st.l += __shfl_xor(st.l, 16, 64);
    st.l += __shfl_xor(st.l, 32, 64);
#pragma unroll
    for (int g = 0; g < NG; g++) {
        f32x4 y0 = st.acc[2 * g] + st.off[g];
        f32x4 y1 = st.acc[2 * g + 1] * 0.0625f + st.off[g];
        *reinterpret_cast<f32x4*>(&o_sh[wid][col][32 * g + 4 * h]) = y0 * 16777216.0f;
        *reinterpret_cast<f32x4*>(&o_sh[wid][col][32 * g + 16 + 4 * h]) = y1 * 16777216.0f;
    }
    if (h == 0) {
        m_sh[wid][col] = st.m;
        l_sh[wid][col] = st.l;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < ncol * D; e += 64 * KV4_WAVES) {
        const int cc = e / D, d = e % D;
        float m = -__builtin_inff();
#pragma unroll
        for (int w = 0; w < KV4_WAVES; w++) m = __builtin_fmaxf(m, m_sh[w][cc]);
        float num = 0.0f, den = 0.0f;
#pragma unroll
        for (int w = 0; w < KV4_WAVES; w++) {
            // without a maximum the wave's sums are zero, or NaN from a NaN score
            const float f = m_sh[w][cc] > -__builtin_inff() ? exp2_fast(m_sh[w][cc] - m) : 1.0f;
            num = __builtin_fmaf(f, o_sh[w][cc][d], num);
            den = __builtin_fmaf(f, l_sh[w][cc], den);
        }
        const int vv = 16 * cg + cc;
        a.o[(((size_t)b * a.S + vv / a.G) * a.Hq + (size_t)head * a.G + vv % a.G) * D + d] = f2h(den != 0.0f ? num / den : 0.0f);
    }
}

}  // namespace cactus_hip

using namespace cactus_hip;

extern "C" {

size_t cactus_hip_attention_kv4_workspace(const cactus_hip_kv4_cache* cache, size_t batch, size_t seq_len,
                                          size_t num_q_heads) {
    (void)batch; (void)seq_len; (void)num_q_heads;
    if (kv4_view(cache, 0, "attention_kv4_workspace", nullptr)) return 0;
    return 4096;
}

int cactus_hip_attention_kv4_f16(const cactus_hip_kv4_cache* cache, size_t layer, const int32_t* seqs,
                                 const int32_t* counts, const uint16_t* q, size_t q_stride, uint16_t* o, size_t batch,
                                 size_t seq_len, size_t num_q_heads, float scale, size_t window_size,
                                 size_t sink_size, int is_causal, void* workspace, size_t workspace_bytes,
                                 void* stream) {
    Kv4AttnArgs a;
    int rc = kv4_view(cache, layer, "attention_kv4", &a.c);
    if (rc) return rc;
    if (batch == 0 || seq_len == 0 || num_q_heads == 0) return CACTUS_HIP_OK;
    CH_REQUIRE(q && o, "attention_kv4: null pointer");
    CH_REQUIRE(num_q_heads % cache->kv_heads == 0 && num_q_heads <= 65536, "attention_kv4: num_q_heads is not a multiple of the cache's kv_heads");
    CH_REQUIRE(((uintptr_t)q & 15) == 0 && ((uintptr_t)o & 15) == 0 && q_stride % 8 == 0,
               "attention_kv4: rows are not 16-byte aligned");
    CH_REQUIRE(q_stride >= num_q_heads * cache->head_dim, "attention_kv4: q_stride is shorter than a row");
    CH_REQUIRE(batch <= 65535, "attention_kv4: more than 65535 requests");
    const size_t G = num_q_heads / cache->kv_heads;
    CH_REQUIRE(seq_len < (1u << 24) && seq_len * G < (1u << 30), "attention_kv4: seq_len out of range");
    CH_REQUIRE(workspace && ((uintptr_t)workspace & 255) == 0 &&
                   workspace_bytes >= cactus_hip_attention_kv4_workspace(cache, batch, seq_len, num_q_heads),
               "attention_kv4: workspace too small or not 256-byte aligned");
    const size_t top = (size_t)1 << 30;   // beyond every position
    a.seqs = seqs;
    a.counts = counts;
    a.q = q;
    a.o = o;
    a.q_stride = q_stride;
    a.B = (int)batch;
    a.S = (int)seq_len;
    a.Hq = (int)num_q_heads;
    a.G = (int)G;
    a.window = (int)std::min(window_size, top);
    a.sink = (int)std::min(sink_size, top);
    a.causal = is_causal != 0;
    a.scale = (scale == 0.0f ? 1.0f / sqrtf((float)cache->head_dim) : scale) * LOG2E_F;
    const dim3 grid(ceil_div(seq_len * G, 16), cache->kv_heads, (unsigned)batch);
    const hipStream_t st = as_stream(stream);
    switch (a.c.d) {
        case 64: hipLaunchKernelGGL(attn_kv4_kernel<64>, grid, dim3(64 * KV4_WAVES), 0, st, a); break;
        case 128: hipLaunchKernelGGL(attn_kv4_kernel<128>, grid, dim3(64 * KV4_WAVES), 0, st, a); break;
        default: hipLaunchKernelGGL(attn_kv4_kernel<256>, grid, dim3(64 * KV4_WAVES), 0, st, a);
    }
    return check_launch("attention_kv4");
}

}  // extern "C"
