// lora.hip -- low-rank adapters of many requests beside a projection that they
// share: y = base + s_a B_a (A_a x) for the rows of a request with adapter a.
#include "hip_common.h"

namespace cactus_hip {

struct LoraArgs {
    const uint16_t* x;
    const uint16_t* A;        // [adapters][r][K]
    const uint16_t* B;        // [adapters][N][r]
    const float* scales;
    const int32_t* ids;
    const int32_t* counts;
    const uint16_t* base;
    uint16_t* y;
    size_t x_stride, base_stride, y_stride;
    int adapters, r, batch, S, K, N;
    int tiles, splits, share; // row tiles of a request, workgroups that share a tile, outputs of each
};

// A workgroup takes 16 RT rows of a request and a share of the outputs.
//   shrink  h^T = A x^T on v_mfma_f32_16x16x32_f16 (A's rows the operand's rows, x's the
//           columns), the contraction over K dealt to the W waves in steps of 64 so that
//           each element of A and x is loaded once per workgroup, straight in operand
//           order (16 lanes' rows, 128 contiguous bytes of each); the partial sums meet in LDS
//   expand  y^T = B h^T, h as two FP16 operands (h 2^e = hi + lo, 22 bits of it: the
//           product's operands are FP16, and one of 11 bits would show in y); the rows of B
//           are dealt to the operand's rows so that two tiles leave a lane eight
//           neighbouring outputs of one row: 16-byte loads of base and stores of y
// Where several workgroups share a tile's rows each computes h for itself: reading x and A
// again from the L2 costs less than a second launch or a wait.
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
constexpr int LORA_MAX_RANK = 256, LORA_WGS = 512;
__device__ __forceinline__ h16x8 as_h8(uint4 u) { return __builtin_bit_cast(h16x8, u); }

// RB blocks of 16 ranks at a time, NP times; RB 1: ranks 8 and 16, hi and lo in one operand
template <int RT, int RB, int NP, int W>
__global__ void __launch_bounds__(64 * W) lora_tile_kernel(LoraArgs a) {
    constexpr int ROWS = 16 * RT, RP = 16 * RB * NP, PS = 16 * RB + 4, HS = 2 * RP + 8, TPR = 64 * W / ROWS;
    constexpr int VPT = 16 * RB / TPR > 0 ? 16 * RB / TPR : 1;       // ranks of a row that a thread sums, per pass
    constexpr int LDS_A = W * ROWS * PS * 4, LDS_B = ROWS * HS * 2;
    __shared__ __attribute__((aligned(16))) uint8_t lds[LDS_A > LDS_B ? LDS_A : LDS_B];
    __shared__ float back[ROWS];                                     // 2^-e of a row
    float* part = reinterpret_cast<float*>(lds);
    uint16_t* hs = reinterpret_cast<uint16_t*>(lds);

    // workgroups of one tile on one XCD (workgroup i runs on XCD i % 8)
    const uint32_t xcd = blockIdx.x & 7u, local = blockIdx.x >> 3;
    const uint32_t tile = xcd + 8u * (local / (uint32_t)a.splits), split = local % (uint32_t)a.splits;
    const int req = (int)(tile / (uint32_t)a.tiles);
    if (req >= a.batch) return;
    const int row0 = (int)(tile % (uint32_t)a.tiles) * ROWS;
    const int m = min(a.counts ? a.counts[req] : a.S, a.S);
    if (row0 >= m) return;
    const int id = a.ids[req];
    const size_t at = (size_t)req * a.S + row0;
    const uint16_t *x = a.x + at * a.x_stride, *base = a.base + at * a.base_stride;
    uint16_t* y = a.y + at * a.y_stride;
    const int rows = min(ROWS, m - row0);
    const int n_lo = (int)split * a.share, n_hi = min(n_lo + a.share, a.N);
    const int tid = threadIdx.x;
    if ((unsigned)id >= (unsigned)a.adapters) {
        if (y != base) {
            const int per = (n_hi - n_lo) / 8;
            for (int i = tid; i < rows * per; i += 64 * W) {
                const int r = i / per, n = n_lo + i % per * 8;
                *reinterpret_cast<uint4*>(y + r * a.y_stride + n) = *reinterpret_cast<const uint4*>(base + r * a.base_stride + n);
            }
        }
        return;
    }
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c16 = lane & 15, quad = lane >> 4;
    const uint16_t* A = a.A + (size_t)id * a.r * a.K;
    const uint16_t* B = a.B + (size_t)id * a.N * a.r;
    const float scale = a.scales ? a.scales[id] : 1.0f;

    // rows and ranks behind the last one repeat it: their results are dropped
    const uint16_t* xr[RT];
#pragma unroll
    for (int t = 0; t < RT; t++) xr[t] = x + (size_t)min(16 * t + c16, rows - 1) * a.x_stride;
    const int steps = (a.K + 63) / 64;
    const int row = tid / TPR, sub = tid % TPR;
    float h[NP][VPT];
    float most = 0.0f;
#pragma unroll
    for (int p = 0; p < NP; p++) {
        const uint16_t* ar[RB];
#pragma unroll
        for (int b = 0; b < RB; b++) ar[b] = A + (size_t)min(16 * (p * RB + b) + c16, a.r - 1) * a.K;
        f32x4 acc[RB][RT] = {};
        struct Step {
            uint4 A[RB][2], x[RT][2];
        };
        const auto load = [&](Step& s, int i) {
            const int k = 64 * i + 16 * quad;
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const int ku = min(k + 8 * u, a.K - 8);
#pragma unroll
                for (int b = 0; b < RB; b++) s.A[b][u] = *reinterpret_cast<const uint4*>(ar[b] + ku);
#pragma unroll
                for (int t = 0; t < RT; t++) s.x[t][u] = *reinterpret_cast<const uint4*>(xr[t] + ku);
            }
        };
        const auto mul = [&](Step& s, int i) {
            if (64 * i + 64 > a.K) {          // (the same for the wave) the last step of a K that is no multiple of 64
#pragma unroll
                for (int u = 0; u < 2; u++)
                    if (64 * i + 16 * quad + 8 * u >= a.K) {
#pragma unroll
                        for (int b = 0; b < RB; b++) s.A[b][u] = make_uint4(0, 0, 0, 0);
#pragma unroll
                        for (int t = 0; t < RT; t++) s.x[t][u] = make_uint4(0, 0, 0, 0);
                    }
            }
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int b = 0; b < RB; b++)
#pragma unroll
                    for (int t = 0; t < RT; t++)
                        acc[b][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_h8(s.A[b][u]), as_h8(s.x[t][u]), acc[b][t], 0, 0, 0);
        };
        Step s0, s1;
        int i = wave;
        if (i < steps) load(s0, i);
        while (i < steps) {
            if (i + W < steps) load(s1, i + W);
            mul(s0, i);
            i += W;
            if (i >= steps) break;
            if (i + W < steps) load(s0, i + W);
            mul(s1, i);
            i += W;
        }
        if (p > 0) __syncthreads();           // the sums of the pass before are read
#pragma unroll
        for (int b = 0; b < RB; b++)
#pragma unroll
            for (int t = 0; t < RT; t++)
                *reinterpret_cast<f32x4*>(part + (wave * ROWS + 16 * t + c16) * PS + 16 * b + 4 * quad) = acc[b][t];
        __syncthreads();
#pragma unroll
        for (int v = 0; v < VPT; v++) {
            const int j = sub + TPR * v;      // rank of this pass
            float s = 0.0f;
            if (TPR <= 16 * RB || j < 16 * RB) {
#pragma unroll
                for (int w = 0; w < W; w++) s += part[(w * ROWS + row) * PS + j];
            }
            h[p][v] = p * 16 * RB + j < a.r && j < 16 * RB ? s : 0.0f;
            const float u = __builtin_fabsf(h[p][v]);
            most = __builtin_fmaxf(most, u < __builtin_inff() ? u : 0.0f);      // (of the finite ones)
        }
    }
    // the row's largest to [2^14, 2^15)
#pragma unroll
    for (int o = TPR / 2; o > 0; o >>= 1) most = __builtin_fmaxf(most, __shfl_xor(most, o, 64));
    const int e = most > 0.0f ? 15 - __builtin_amdgcn_frexp_expf(most) : 0;
    __syncthreads();                          // (the halves lie where the sums did)
    if (sub == 0) back[row] = __builtin_ldexpf(1.0f, -e);
#pragma unroll
    for (int p = 0; p < NP; p++)
#pragma unroll
        for (int v = 0; v < VPT; v++) {
            const int j = sub + TPR * v;
            const float s = __builtin_ldexpf(h[p][v], e);
            const f16 hi = (f16)s;
            const bool number = __builtin_fabsf(s) < __builtin_inff();
            const f16 lo = number ? (f16)(s - (float)hi) : (f16)0.0f;
            if (TPR <= 16 * RB || j < 16 * RB) {
                hs[row * HS + p * 16 * RB + j] = bitsh(hi);
                hs[row * HS + RP + p * 16 * RB + j] = bitsh(lo);
            }
        }
    __syncthreads();

    constexpr int KS = RB == 1 ? 1 : RP / 32;
    float unlift[RT];
#pragma unroll
    for (int t = 0; t < RT; t++) unlift[t] = back[16 * t + c16];
    for (int n0 = n_lo + 32 * wave; n0 < n_hi; n0 += 32 * W) {
        const int n = n0 + 8 * quad, nc = min(n, a.N - 8);
        uint4 bs[RT];
#pragma unroll
        for (int t = 0; t < RT; t++)
            bs[t] = *reinterpret_cast<const uint4*>(base + (size_t)min(16 * t + c16, rows - 1) * a.base_stride + nc);
        f32x4 acc[RT][2] = {};
        const int nb = min(n0 + 8 * (c16 >> 2), a.N - 8) + (c16 & 3);
#pragma unroll
        for (int k = 0; k < KS; k++) {
            const int chunk = RB == 1 ? quad & 1 : 4 * k + quad;
            const bool there = 8 * chunk < a.r;
#pragma unroll
            for (int u = 0; u < 2; u++) {
                uint4 w = *reinterpret_cast<const uint4*>(B + (size_t)(nb + 4 * u) * a.r + (there ? 8 * chunk : 0));
                if (!there) w = make_uint4(0, 0, 0, 0);
#pragma unroll
                for (int t = 0; t < RT; t++) {
                    const uint16_t* at_h = hs + (16 * t + c16) * HS + 8 * chunk;
                    if constexpr (RB == 1) {
                        const h16x8 z = *reinterpret_cast<const h16x8*>(at_h + (quad >> 1) * RP);
                        acc[t][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_h8(w), z, acc[t][u], 0, 0, 0);
                    } else {
                        const h16x8 hi = *reinterpret_cast<const h16x8*>(at_h), lo = *reinterpret_cast<const h16x8*>(at_h + RP);
                        acc[t][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_h8(w), hi, acc[t][u], 0, 0, 0);
                        acc[t][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_h8(w), lo, acc[t][u], 0, 0, 0);
                    }
                }
            }
        }
        if (n >= n_hi) continue;
#pragma unroll
        for (int t = 0; t < RT; t++) {
            if (16 * t + c16 >= rows) continue;
            const uint32_t w[4] = {bs[t].x, bs[t].y, bs[t].z, bs[t].w};
            uint32_t o[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float d0 = acc[t][j >> 1][2 * (j & 1)] * unlift[t], d1 = acc[t][j >> 1][2 * (j & 1) + 1] * unlift[t];
                o[j] = f2h(__builtin_fmaf(d0, scale, h2f((uint16_t)w[j]))) |
                       (uint32_t)f2h(__builtin_fmaf(d1, scale, h2f((uint16_t)(w[j] >> 16)))) << 16;
            }
            *reinterpret_cast<uint4*>(y + (size_t)(16 * t + c16) * a.y_stride + n) = make_uint4(o[0], o[1], o[2], o[3]);
        }
    }
}

template <int RT, int RB, int NP, int W>
static void lora_launch(LoraArgs a, int target, hipStream_t st) {
    a.tiles = (a.S + 16 * RT - 1) / (16 * RT);
    const size_t tiles = (size_t)a.tiles * a.batch;
    const int units = (a.N + 31) / 32;
    int splits = (int)((target + tiles - 1) / tiles);
    splits = splits < 1 ? 1 : splits > (units + W - 1) / W ? (units + W - 1) / W : splits;
    a.share = (units + splits - 1) / splits * 32;
    a.splits = (a.N + a.share - 1) / a.share;
    hipLaunchKernelGGL((lora_tile_kernel<RT, RB, NP, W>), dim3((unsigned)((tiles + 7) / 8 * 8 * a.splits)), dim3(64 * W), 0, st, a);
}

}  // namespace cactus_hip

using namespace cactus_hip;

extern "C" int cactus_hip_lora_add_f16(const uint16_t* x, size_t x_stride, const uint16_t* A, const uint16_t* B,
                                       const float* scales, size_t num_adapters, size_t rank, const int32_t* adapters,
                                       const int32_t* counts, const uint16_t* base, size_t base_stride, uint16_t* y,
                                       size_t y_stride, size_t batch, size_t seq_len, size_t K, size_t N, void* stream) {
    CH_REQUIRE(rank >= 8 && rank <= LORA_MAX_RANK && rank % 8 == 0, "lora_add: rank is a multiple of 8 from 8 to 256");
    CH_REQUIRE(K % 8 == 0 && N % 8 == 0 && K < (1u << 24) && N < (1u << 24), "lora_add: K and N are multiples of 8 below 2^24");
    CH_REQUIRE(num_adapters < (1u << 24), "lora_add: num_adapters out of range");
    CH_REQUIRE(batch <= 65535 && seq_len < (1u << 24), "lora_add: batch or seq_len out of range");
    if (batch == 0 || seq_len == 0 || N == 0) return CACTUS_HIP_OK;
    CH_REQUIRE(adapters && base && y && (num_adapters == 0 || (A && B && x) || K == 0), "lora_add: null pointer");
    const auto aligned = [](const void* p, size_t stride) { return ((uintptr_t)p & 15) == 0 && stride % 8 == 0; };
    CH_REQUIRE(aligned(x, x_stride) && aligned(A, 0) && aligned(B, 0) && aligned(base, base_stride) && aligned(y, y_stride),
               "lora_add: rows are not 16-byte aligned");
    CH_REQUIRE(x_stride >= K && base_stride >= N && y_stride >= N, "lora_add: a stride is shorter than its row");
    CH_REQUIRE(y != base || y_stride == base_stride, "lora_add: y in place of base needs its stride");
    LoraArgs a{x,        A,           B,        scales, adapters, counts, base, y, x_stride, base_stride, y_stride, (int)num_adapters,
               (int)rank, (int)batch, (int)seq_len, (int)K, (int)N, 0, 0, 0};
    CH_REQUIRE(batch * ceil_div(seq_len, 16) < (1u << 22), "lora_add: batch times seq_len out of range");
    const hipStream_t st = as_stream(stream);
    const int rt = seq_len <= 16 ? 1 : batch * ceil_div(seq_len, 64) >= 128 && rank <= 64 ? 4 : batch * ceil_div(seq_len, 32) >= 64 ? 2 : 1;
#define LORA_RANKS(RT, W)                                                     \
    if (rank <= 16) lora_launch<RT, 1, 1, W>(a, LORA_WGS, st);                \
    else if (rank <= 32) lora_launch<RT, 2, 1, W>(a, LORA_WGS, st);           \
    else if (rank <= 64) lora_launch<RT, 4, 1, W>(a, LORA_WGS, st)
#define LORA_MORE(RT, W)                                                      \
    else if (rank <= 128) lora_launch<RT, 4, 2, W>(a, LORA_WGS, st);          \
    else lora_launch<RT, 4, 4, W>(a, LORA_WGS, st)
    if (rt == 4) {
        LORA_RANKS(4, 4);
    } else if (rt == 2) {
        LORA_RANKS(2, 4);
        LORA_MORE(2, 4);
    } else {
        LORA_RANKS(1, 8);
        LORA_MORE(1, 8);
    }
#undef LORA_RANKS
#undef LORA_MORE
    return check_launch("lora_add");
}
