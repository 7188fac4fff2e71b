// lora.hip -- low-rank adapters of many requests beside a projection that they
// share: y = base + s_a B_a (A_a x) for the rows of a request with adapter a.
//
// Bound by memory: x, base and y are 2 (K + 2 N) bytes a row for 2 r (K + N) operations.  8 x
// 1024 rows of 4096 by 4096: rank 16 46 us and rank 32 48 (4.4 and 4.3 TB/s; a copy of 2 GiB runs
// at 4.9), rank 64 56 us, where the weights that 256 workgroups read from the L2, 1 MB each, tell.
// That is 256 tiles of 32 rows on 256 CUs.  A workgroup's 91 to 156 KB of LDS leave room for one per CU, so
// that more rows come in rounds: 8224 rows 57 and 84 us (ranks 16 and 64), 16384 83 and 101.  Ranks above 64
// have four waves per workgroup and read x again in every pass: 95 us (rank 128) and 157 (256)
// for 8192 rows, 151 and 247 for 8224.
// Five prompts of up to 701 rows, 1024 by 2048, rank 32: 9.4 us (rank 64 12.3, 128 27.7,
// 256 47.9); 64 single rows with 24 adapters, 2048 by 1024, rank 16: 4.6 us; one row 3.3 (an empty
// launch 2.4).
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
//           columns), the contraction over K dealt to the W waves in steps of 32, so that
//           each element of A and x is loaded once per workgroup; the partial sums meet in LDS
//   expand  y^T = B h^T, h as two FP16 operands (h 2^e = hi + lo, 22 bits of it: the
//           product's operands are FP16, and one of 11 bits would show in y)
// A wave loads 64 or 128 bytes of a row with neighbouring lanes, and its LDS turns them into
// operands (the instruction wants 16 rows side by side: loads in that order take the L1 64
// accesses each instead of 16, which was half of the time).  A and x go there by DMA, in a
// ring of ST steps; B through registers; products of B come back the same way, so that base
// and y move in whole lines too.  All of it is the wave's own: only the sums need barriers.
// Where several workgroups share a tile's rows each computes h for itself: reading x and A
// again from the L2 costs less than a second launch or a wait, as long as the workgroups do not
// outnumber the CUs (8 x 1024 rows in 512 workgroups 97 us, in 256 59).
// y goes past the caches: 57.3 -> 55.6 us.
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
constexpr int LORA_MAX_RANK = 256;
__device__ __forceinline__ h16x8 as_h8(u32x4 u) { return __builtin_bit_cast(h16x8, u); }

__device__ __forceinline__ float wave_sum(float v) {
    v += dpp_move_keep<0xB1>(v);      // within rows of 16 lanes
    v += dpp_move_keep<0x4E>(v);
    v += dpp_move_keep<0x141>(v);
    v += dpp_move_keep<0x140>(v);
    const auto of = [&](int l) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), l)); };
    return (of(0) + of(16)) + (of(32) + of(48));
}

// RB blocks of 16 ranks at a time, NP times; RB 1: ranks 8 and 16, hi and lo in one operand
template <int RT, int RB, int NP, int W>
struct LoraShape {
    static constexpr int ROWS = 16 * RT, RP = 16 * RB * NP;
    static constexpr int PS = 16 * RB + 4, HS = 2 * RP + 8;          // pitches of the sums and of h's halves
    static constexpr int UN = RP <= 64 ? 64 : 32, DS = UN + 4;       // outputs at a time, pitch of their products
    static constexpr int ST = RB + RT <= 3 ? 4 : 3;
    static constexpr int STEP = 1024 * (RB + RT), PART = ROWS * PS * 4, BUF = UN * RP * 2, EXPAND = BUF + 16 * DS * 4;
    static constexpr int SHRINK = ST * STEP > PART ? ST * STEP : PART, WAVE = SHRINK > EXPAND ? SHRINK : EXPAND;
    static constexpr int LDS = W * WAVE + ROWS * HS * 2 + ROWS * 4;
    static_assert(LDS <= 160 * 1024, "LDS");
};

template <int RT, int RB, int NP, int W>
__global__ void __launch_bounds__(64 * W) lora_tile_kernel(LoraArgs a) {
    using Z = LoraShape<RT, RB, NP, W>;
    constexpr int ROWS = Z::ROWS, RP = Z::RP, PS = Z::PS, HS = Z::HS, UN = Z::UN, DS = Z::DS, ST = Z::ST, TPR = 64 * W / ROWS;
    constexpr int VPT = 16 * RB / TPR > 0 ? 16 * RB / TPR : 1;       // ranks of a row that a thread sums, per pass
    __shared__ __attribute__((aligned(128))) uint8_t lds[Z::LDS];
    uint16_t* hs = reinterpret_cast<uint16_t*>(lds + W * Z::WAVE);
    float* back = reinterpret_cast<float*>(lds + W * Z::WAVE + ROWS * HS * 2);      // 2^-e of a row

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
                *reinterpret_cast<u32x4*>(y + r * a.y_stride + n) = *reinterpret_cast<const u32x4*>(base + r * a.base_stride + n);
            }
        }
        return;
    }
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c16 = lane & 15, quad = lane >> 4;
    const uint16_t* A = a.A + (size_t)id * a.r * a.K;
    const uint16_t* B = a.B + (size_t)id * a.N * a.r;
    const float scale = a.scales ? a.scales[id] : 1.0f;
    uint8_t* own = lds + wave * Z::WAVE;
    const uint32_t own_at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)own;

    // rows and ranks behind the last one repeat it: their results are dropped
    const int steps = (a.K + 31) / 32;
    const int mine = steps > wave ? (steps - wave + W - 1) / W : 0;  // steps of this wave
    const uint16_t* src[RB + RT];
#pragma unroll
    for (int i = 0; i < RT; i++) src[RB + i] = x + (size_t)min(16 * i + (lane >> 2), rows - 1) * a.x_stride;
    const int row = tid / TPR, sub = tid % TPR;
    float h[NP][VPT];
    float most = 0.0f;
#pragma unroll
    for (int p = 0; p < NP; p++) {
#pragma unroll
        for (int i = 0; i < RB; i++) src[i] = A + (size_t)min(16 * (p * RB + i) + (lane >> 2), a.r - 1) * a.K;
        // 16 bytes to slot s of row r: piece s ^ (r / 4), so that 8 rows' reads of a piece meet different banks
        const auto issue = [&](int j) __attribute__((always_inline)) {
            const int k = min(32 * (wave + W * j) + 8 * ((lane & 3) ^ (lane >> 4)), a.K - 8);
            const uint32_t to = own_at + (uint32_t)(j % ST * Z::STEP);
#pragma unroll
            for (int i = 0; i < RB + RT; i++) lds_dma<16>(src[i] + k, to + 1024 * i);
        };
        if (p > 0) __syncthreads();           // the sums of the pass before are read
#pragma unroll
        for (int j = 0; j < ST - 1; j++)
            if (j < mine) issue(j);
        f32x4 acc[RB][RT] = {};
        for (int j = 0; j < mine; j++) {
            if (j + ST - 1 < mine) {
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the step before has left its place
                issue(j + ST - 1);
            }
            const int younger = min(ST - 1, mine - 1 - j);
            if (ST > 3 && younger == 3) wait_dma<3 * (RB + RT)>();
            else if (younger == 2) wait_dma<2 * (RB + RT)>();
            else if (younger == 1) wait_dma<RB + RT>();
            else wait_dma<0>();
            const uint8_t* at_s = own + j % ST * Z::STEP + c16 * 64 + 16 * (quad ^ (c16 >> 2));
            u32x4 fa[RB], fx[RT];
#pragma unroll
            for (int b = 0; b < RB; b++) fa[b] = *reinterpret_cast<const u32x4*>(at_s + 1024 * b);
#pragma unroll
            for (int t = 0; t < RT; t++) fx[t] = *reinterpret_cast<const u32x4*>(at_s + 1024 * (RB + t));
            const int k0 = 32 * (wave + W * j);
            if (k0 + 32 > a.K && k0 + 8 * quad >= a.K) {     // the last step of a K that is no multiple of 32
#pragma unroll
                for (int b = 0; b < RB; b++) fa[b] = (u32x4){0, 0, 0, 0};
#pragma unroll
                for (int t = 0; t < RT; t++) fx[t] = (u32x4){0, 0, 0, 0};
            }
#pragma unroll
            for (int b = 0; b < RB; b++)
#pragma unroll
                for (int t = 0; t < RT; t++)
                    acc[b][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_h8(fa[b]), as_h8(fx[t]), acc[b][t], 0, 0, 0);
        }
#pragma unroll
        for (int b = 0; b < RB; b++)
#pragma unroll
            for (int t = 0; t < RT; t++)
                *reinterpret_cast<f32x4*>(own + ((16 * t + c16) * PS + 16 * b + 4 * quad) * 4) = acc[b][t];
        __syncthreads();
#pragma unroll
        for (int v = 0; v < VPT; v++) {
            const int j = sub + TPR * v;      // rank of this pass
            float s = 0.0f;
            if (TPR <= 16 * RB || j < 16 * RB) {
#pragma unroll
                for (int w = 0; w < W; w++) s += *reinterpret_cast<const float*>(lds + w * Z::WAVE + (row * PS + j) * 4);
            }
            h[p][v] = p * 16 * RB + j < a.r && j < 16 * RB ? s : 0.0f;
            const float u = __builtin_fabsf(h[p][v]);
            most = __builtin_fmaxf(most, u < __builtin_inff() ? u : 0.0f);      // (of the finite ones)
        }
    }
    // what the outputs take, UN of them per step: B's rows of them, whole lines one after the other, and base
    constexpr int KS = RB == 1 ? 1 : RP / 32, BI = UN * RP / 512, LPR = UN / 8, BJ = ROWS * LPR / 64;
    const int lp = 31 - __builtin_clz(a.r / 8);
    const bool pow2 = a.r == 8 << lp;         // pieces per row
    const int swz = !pow2 || lp < 2 ? 0 : lp == 2 ? 3 : lp == 3 ? 7 : 15, swz_sh = lp == 2 ? 2 : 0;
    const auto turn = [&](int n) { return (n >> swz_sh) & swz; };
    const int all_b = a.N * (a.r / 8);        // pieces of B (below 2^24 * 32)
    u32x4 bw[BI], bb[BJ];
    const auto get = [&](int n0) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < BI; i++) {
            const int j = 64 * i + lane, n = j >> lp;
            const int piece = swz ? (n << lp) + ((j & ((1 << lp) - 1)) ^ turn(n)) : j;
            bw[i] = *reinterpret_cast<const u32x4*>(B + (size_t)min(n0 * (a.r / 8) + piece, all_b - 1) * 8);
        }
#pragma unroll
        for (int i = 0; i < BJ; i++) {
            const int j = 64 * i + lane;
            bb[i] = *reinterpret_cast<const u32x4*>(base + (size_t)min(j / LPR, rows - 1) * a.base_stride + min(n0 + j % LPR * 8, a.N - 8));
        }
    };
    int n0 = n_lo + UN * wave;
    if (n0 < n_hi) get(n0);                   // on its way before the sums have met
    // the row's largest to [2^14, 2^15)
#pragma unroll
    for (int o = TPR / 2; o > 0; o >>= 1) most = __builtin_fmaxf(most, __shfl_xor(most, o, 64));
    const int e = most > 0.0f ? 15 - __builtin_amdgcn_frexp_expf(most) : 0;
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

    uint8_t* own_b = own;      // (the sums are read)
    float* own_d = reinterpret_cast<float*>(own_b + Z::BUF);
    for (; n0 < n_hi; n0 += UN * W) {
        wave_lds_order();
#pragma unroll
        for (int i = 0; i < BI; i++) *reinterpret_cast<u32x4*>(own_b + 1024 * i + 16 * lane) = bw[i];
        u32x4 bc[BJ];
#pragma unroll
        for (int i = 0; i < BJ; i++) bc[i] = bb[i];
        if (n0 + UN * W < n_hi) get(n0 + UN * W);
        wave_lds_order();
        f32x4 acc[RT][UN / 16] = {};
#pragma unroll
        for (int k = 0; k < KS; k++) {
            const int chunk = RB == 1 ? quad & 1 : 4 * k + quad;
            const bool there = 8 * chunk < a.r;
            u32x4 z[RT][RB == 1 ? 1 : 2];
#pragma unroll
            for (int t = 0; t < RT; t++) {
                const uint16_t* at_h = hs + (16 * t + c16) * HS + 8 * chunk;
                if constexpr (RB == 1) {
                    z[t][0] = *reinterpret_cast<const u32x4*>(at_h + (quad >> 1) * RP);
                } else {
                    z[t][0] = *reinterpret_cast<const u32x4*>(at_h);
                    z[t][1] = *reinterpret_cast<const u32x4*>(at_h + RP);
                }
            }
#pragma unroll
            for (int u = 0; u < UN / 16; u++) {
                const int n = 16 * u + c16;
                u32x4 w = *reinterpret_cast<const u32x4*>(own_b + 2 * n * a.r + (there ? 16 * (chunk ^ turn(n)) : 0));
                if (!there) w = (u32x4){0, 0, 0, 0};
#pragma unroll
                for (int t = 0; t < RT; t++)
#pragma unroll
                    for (int q = 0; q < (RB == 1 ? 1 : 2); q++)
                        acc[t][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_h8(w), as_h8(z[t][q]), acc[t][u], 0, 0, 0);
            }
        }
#pragma unroll
        for (int t = 0; t < RT; t++) {
            wave_lds_order();
#pragma unroll
            for (int u = 0; u < UN / 16; u++) *reinterpret_cast<f32x4*>(own_d + c16 * DS + 16 * u + 4 * quad) = acc[t][u];
            wave_lds_order();
#pragma unroll
            for (int i = 0; i < BJ / RT; i++) {
                const int j = 64 * i + lane, r = j / LPR, n = n0 + j % LPR * 8;
                const f32x4 d0 = *reinterpret_cast<const f32x4*>(own_d + r * DS + j % LPR * 8);
                const f32x4 d1 = *reinterpret_cast<const f32x4*>(own_d + r * DS + j % LPR * 8 + 4);
                const float unlift = back[16 * t + r];
                const u32x4 w = bc[BJ / RT * t + i];
                uint32_t o[4];
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const float e0 = (q < 2 ? d0 : d1)[2 * (q & 1)] * unlift, e1 = (q < 2 ? d0 : d1)[2 * (q & 1) + 1] * unlift;
                    o[q] = f2h(__builtin_fmaf(e0, scale, h2f((uint16_t)w[q]))) |
                           (uint32_t)f2h(__builtin_fmaf(e1, scale, h2f((uint16_t)(w[q] >> 16)))) << 16;
                }
                if (16 * t + r < rows && n < n_hi)
                    __builtin_nontemporal_store((u32x4){o[0], o[1], o[2], o[3]}, reinterpret_cast<u32x4*>(y + (size_t)(16 * t + r) * a.y_stride + n));
            }
        }
    }
}

// Single rows (a decode step): nothing is shared by 16 rows, so the products are FP32 on the
// vector units, with nothing to turn round in LDS (64 rows 4.6 against 5.7 us in tiles, one 3.3
// against 4.6).  Waves take ranks, RB of them side by side,
// over the whole row; then lanes take 8 ranks of 8 neighbouring outputs.  Bound by the
// chain of loads: id, A and x, (B and base on their way meanwhile,) store.
template <int RB>
__global__ void __launch_bounds__(512) lora_row_kernel(LoraArgs a) {
    constexpr int W = 8;
    __shared__ __attribute__((aligned(16))) float h[LORA_MAX_RANK];
    const int req = blockIdx.y;
    const int m = a.counts ? a.counts[req] : 1;
    const int id = a.ids[req];
    const uint16_t *x = a.x + (size_t)req * a.x_stride, *base = a.base + (size_t)req * a.base_stride;
    uint16_t* y = a.y + (size_t)req * a.y_stride;
    const int n_lo = (int)blockIdx.x * a.share, n_hi = min(n_lo + a.share, a.N);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    if (m < 1) return;
    if ((unsigned)id >= (unsigned)a.adapters) {
        if (y != base)
            for (int n = n_lo + 8 * tid; n < n_hi; n += 512 * 8)
                *reinterpret_cast<u32x4*>(y + n) = *reinterpret_cast<const u32x4*>(base + n);
        return;
    }
    const uint16_t* A = a.A + (size_t)id * a.r * a.K;
    const uint16_t* B = a.B + (size_t)id * a.N * a.r;
    const float scale = a.scales ? a.scales[id] : 1.0f;
    // outputs: 2^lp lanes (pieces of 8 ranks of a row of B) to 8 outputs, a wave 512 >> lp of them
    const int pieces = a.r / 8, lp = pieces > 1 ? 32 - __builtin_clz(pieces - 1) : 0;
    const int piece = lane & ((1 << lp) - 1), group = lane >> lp, per_wave = 512 >> lp;
    const bool there = piece < pieces;
    u32x4 bw[8], bb;
    const auto get = [&](int n0) __attribute__((always_inline)) {
        const int n = min(n0 + 8 * group, a.N - 8);
#pragma unroll
        for (int q = 0; q < 8; q++) bw[q] = *reinterpret_cast<const u32x4*>(B + (size_t)(n + q) * a.r + 8 * (there ? piece : 0));
        bb = *reinterpret_cast<const u32x4*>(base + n);
    };
    int n0 = n_lo + per_wave * wave;

    const int ranks = a.r / W;                // of each wave
    for (int j0 = 0; j0 < ranks; j0 += RB) {
        const uint16_t* ar[RB];
#pragma unroll
        for (int b = 0; b < RB; b++) ar[b] = A + (size_t)(wave * ranks + min(j0 + b, ranks - 1)) * a.K;
        float acc[RB] = {};
        constexpr int U = RB > 4 ? 1 : 2;
        for (int k0 = 0; k0 < a.K; k0 += 512 * U) {
            u32x4 xv[U], av[U][RB];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int k = min(k0 + 512 * u + 8 * lane, a.K - 8);
                xv[u] = *reinterpret_cast<const u32x4*>(x + k);
#pragma unroll
                for (int b = 0; b < RB; b++) av[u][b] = *reinterpret_cast<const u32x4*>(ar[b] + k);
            }
            if (k0 == 0 && j0 == 0 && n0 < n_hi) get(n0);
#pragma unroll
            for (int u = 0; u < U; u++) {
                if (k0 + 512 * u + 8 * lane >= a.K) continue;
#pragma unroll
                for (int b = 0; b < RB; b++)
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        acc[b] = __builtin_fmaf(h2f((uint16_t)(av[u][b][i / 2] >> 16 * (i & 1))), h2f((uint16_t)(xv[u][i / 2] >> 16 * (i & 1))), acc[b]);
            }
        }
#pragma unroll
        for (int b = 0; b < RB; b++) acc[b] = wave_sum(acc[b]);
        if (lane == 0) {
#pragma unroll
            for (int b = 0; b < RB; b++)
                if (j0 + b < ranks) h[wave * ranks + j0 + b] = acc[b];
        }
    }
    if (a.K == 0 && n0 < n_hi) get(n0);
    __syncthreads();
    float hv[8];
#pragma unroll
    for (int i = 0; i < 8; i++) hv[i] = there ? h[8 * piece + i] : 0.0f;
    for (; n0 < n_hi; n0 += per_wave * W) {
        float s[8];
#pragma unroll
        for (int q = 0; q < 8; q++) {
            s[q] = 0.0f;
            if (there) {
#pragma unroll
                for (int i = 0; i < 8; i++) s[q] = __builtin_fmaf(h2f((uint16_t)(bw[q][i / 2] >> 16 * (i & 1))), hv[i], s[q]);
            }
        }
        const u32x4 w = bb;
        const int n = n0 + 8 * group;
        if (n0 + per_wave * W < n_hi) get(n0 + per_wave * W);
        for (int o = 1; o < 1 << lp; o <<= 1)
#pragma unroll
            for (int q = 0; q < 8; q++) s[q] += __shfl_xor(s[q], o, 64);
        if (piece == 0 && n < n_hi) {
            uint32_t o[4];
#pragma unroll
            for (int j = 0; j < 4; j++)
                o[j] = f2h(__builtin_fmaf(s[2 * j], scale, h2f((uint16_t)w[j]))) |
                       (uint32_t)f2h(__builtin_fmaf(s[2 * j + 1], scale, h2f((uint16_t)(w[j] >> 16)))) << 16;
            *reinterpret_cast<u32x4*>(y + n) = (u32x4){o[0], o[1], o[2], o[3]};
        }
    }
}

// Workgroups that a call is cut into, about: more share a tile's rows where there are fewer tiles.
// Tiles of 32 rows from LORA_TILE2 of them on: 2048 rows in 16s or 32s 7.2 and 7.2 us (1024 by 2048,
// rank 16), 13.0 and 13.2 (4096 by 4096), 20.4 and 19.8 (rank 64); 1024 rows 5.7 and 6.6, 10.0 and 11.3,
// 16.6 and 17.8; 8192 rows of rank 64 76 and 59.
constexpr size_t LORA_WGS = 256, LORA_TILE2 = 64;

static void lora_rows(LoraArgs a, hipStream_t st) {
    const int pieces = a.r / 8, lp = pieces > 1 ? 32 - __builtin_clz(pieces - 1) : 0, per_wave = 512 >> lp;
    const size_t units = ceil_div(a.N, per_wave), want = ceil_div(LORA_WGS, a.batch);
    const size_t share = ceil_div(units, want < units ? want : units);
    a.share = (int)share * per_wave;
    const dim3 grid(ceil_div(a.N, a.share), (unsigned)a.batch);
    if (a.r <= 8) hipLaunchKernelGGL(lora_row_kernel<1>, grid, dim3(512), 0, st, a);
    else if (a.r <= 16) hipLaunchKernelGGL(lora_row_kernel<2>, grid, dim3(512), 0, st, a);
    else if (a.r <= 32) hipLaunchKernelGGL(lora_row_kernel<4>, grid, dim3(512), 0, st, a);
    else hipLaunchKernelGGL(lora_row_kernel<8>, grid, dim3(512), 0, st, a);
}

template <int RT, int RB, int NP, int W>
static void lora_tiles(LoraArgs a, hipStream_t st) {
    a.tiles = (a.S + 16 * RT - 1) / (16 * RT);
    const size_t tiles = (size_t)a.tiles * a.batch;
    // outputs are shared out in whole rounds of the W waves
    const size_t rounds = ceil_div(a.N, LoraShape<RT, RB, NP, W>::UN * W), each = ceil_div(rounds * tiles, LORA_WGS);
    a.share = (int)(each < rounds ? each : rounds) * LoraShape<RT, RB, NP, W>::UN * W;
    a.splits = (a.N + a.share - 1) / a.share;
    hipLaunchKernelGGL((lora_tile_kernel<RT, RB, NP, W>), dim3((unsigned)((tiles + 7) / 8 * 8 * a.splits)), dim3(64 * W), 0, st, a);
}
template <int RT>
static void lora_ranks(const LoraArgs& a, hipStream_t st) {
    if (a.r <= 16) lora_tiles<RT, 1, 1, 8>(a, st);
    else if (a.r <= 32) lora_tiles<RT, 2, 1, 8>(a, st);
    else if (a.r <= 64) lora_tiles<RT, 4, 1, 8>(a, st);
    else if (a.r <= 128) lora_tiles<RT, 4, 2, 4>(a, st);
    else lora_tiles<RT, 4, 4, 4>(a, st);
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
    CH_REQUIRE(adapters && base && y && (num_adapters == 0 || (B && ((A && x) || K == 0))), "lora_add: null pointer");
    const auto aligned = [](const void* p, size_t stride) { return ((uintptr_t)p & 15) == 0 && stride % 8 == 0; };
    CH_REQUIRE(aligned(x, x_stride) && aligned(A, 0) && aligned(B, 0) && aligned(base, base_stride) && aligned(y, y_stride),
               "lora_add: rows are not 16-byte aligned");
    CH_REQUIRE(x_stride >= K && base_stride >= N && y_stride >= N, "lora_add: a stride is shorter than its row");
    CH_REQUIRE(y != x || num_adapters == 0 || K == 0, "lora_add: y in place of x, which other workgroups still read");
    CH_REQUIRE(y != base || y_stride == base_stride, "lora_add: y in place of base needs its stride");
    LoraArgs a{x,        A,           B,        scales, adapters, counts, base, y, x_stride, base_stride, y_stride, (int)num_adapters,
               (int)rank, (int)batch, (int)seq_len, (int)K, (int)N, 0, 0, 0};
    CH_REQUIRE(batch * ceil_div(seq_len, 16) < (1u << 22), "lora_add: batch times seq_len out of range");
    const hipStream_t st = as_stream(stream);
    if (seq_len == 1) lora_rows(a, st);
    else if (seq_len > 16 && batch * ceil_div(seq_len, 32) >= LORA_TILE2) lora_ranks<2>(a, st);
    else lora_ranks<1>(a, st);
    return check_launch("lora_add");
}
