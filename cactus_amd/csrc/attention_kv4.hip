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
    uint32_t* counters;       // [workgroups] zero between calls
    float* part;              // [workgroups][2][16 (D + 2)]: output, maxima, sums
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

constexpr float LOG2E_F = 1.4426950408889634f;
__device__ __forceinline__ float agent_load(const float* p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void agent_store(float* p, float v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// inclusive sum over the wave's lanes: row_shr 1, 2, 4, 8 within each 16-lane
// row, then row_bcast:15 and row_bcast:31 across rows
__device__ __forceinline__ uint32_t wave_scan_add(uint32_t v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
    return v;
}
__device__ __forceinline__ uint32_t lane_u(uint32_t v, int l) { return (uint32_t)__builtin_amdgcn_readlane((int)v, l); }

// N words of LDS
template <int N>
__device__ __forceinline__ void load_words(uint32_t (&w)[N], const uint8_t* p) {
    if constexpr (N == 2) {
        const uint2 u = *reinterpret_cast<const uint2*>(p);
        w[0] = u.x, w[1] = u.y;
    } else {
#pragma unroll
        for (int i = 0; i < N / 4; i++) {
            const uint4 u = reinterpret_cast<const uint4*>(p)[i];
            w[4 * i] = u.x, w[4 * i + 1] = u.y, w[4 * i + 2] = u.z, w[4 * i + 3] = u.w;
        }
    }
}
__device__ __forceinline__ float half_of(uint32_t w, int i) { return h2f((uint16_t)(i ? w >> 16 : w)); }

// ------------------------------------------------------------ few rows
// The work is a line of block steps (KV4_BLOCK keys of one unit: a request's
// KV head and up to 16 query vectors), unit after unit, request after
// request; each workgroup takes an equal stretch of it, whatever the lengths
// of the sequences are.  A unit that lies in one stretch is written at once;
// one that several workgroups share is written as partial (maximum, sum,
// output) to the workspace, and the last of them to finish joins the parts
// in their order.
constexpr int KV4_WAVES = 4;
constexpr int KV4_BLOCK = KV4_STEP * KV4_WAVES;   // a wave takes a step of 32 keys
constexpr int KV4_GRID = 512;                     // two workgroups per CU
constexpr int KV4_PARTS = 128;                    // a unit's stretches at most
constexpr size_t KV4_COUNTERS = 4096;             // bytes: one counter per workgroup

// block steps of a unit and units of a request (0: no rows)
__device__ __forceinline__ uint32_t unit_blocks(const Kv4Seq& s) {
    return (uint32_t)max(1, (s.steps + KV4_WAVES - 1) / KV4_WAVES);
}
__device__ __forceinline__ uint32_t seq_units(const Kv4AttnArgs& a, const Kv4Seq& s) {
    return (uint32_t)((s.rows * a.G + 15) / 16) * (uint32_t)a.c.Hkv;
}

// Steps of a wave's ring in LDS: as many as leave room for two workgroups per CU
template <int D>
constexpr int kv4_ring() { return 4 - D / 256; }

template <int D>
__global__ void __launch_bounds__(64 * KV4_WAVES, D == 256 ? 1 : 2) attn_kv4_kernel(Kv4AttnArgs a) {
    constexpr int NG = D / 32, NB = D / 16, OS = D + 4;
    constexpr int TB = 18 * D, SLOT = 2 * TB;                  // bytes of a tile and of a step
    constexpr int NI = 2 * ((TB + 1023) / 1024);               // LDS loads of a step
    constexpr int R = kv4_ring<D>();
    static_assert(R * SLOT >= 16 * OS * 4 && R * SLOT >= KV4_PARTS * 64 + 64, "the ring holds the wave's sums, then the parts' weights");
    __shared__ __align__(16) uint8_t ring[KV4_WAVES][R][SLOT];
    __shared__ float m_sh[KV4_WAVES][16], l_sh[KV4_WAVES][16];
    __shared__ int last_sh;
    float (*o_sh)[R * SLOT / 4] = reinterpret_cast<float (*)[R * SLOT / 4]>(&ring[0][0][0]);   // [wave][16][OS]
    float (*w_sh)[16] = reinterpret_cast<float (*)[16]>(&ring[0][0][0]);   // a part's weight in each column, then the sum
    const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, h = lane >> 4;
    const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Kv4View& c = a.c;
    const float kscale = a.scale * 16777216.0f;

    // ---- this workgroup's stretch [at, end) of the line
    uint32_t total = 0, longest = 1;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
        uint32_t cost = 0, blocks = 0;
        if (b0 + lane < a.B) {
            const Kv4Seq s = kv4_seq(a, b0 + lane);
            blocks = s.rows > 0 ? unit_blocks(s) : 0;
            cost = blocks * seq_units(a, s);
        }
        total += lane_u(wave_scan_add(cost), 63);
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) blocks = max(blocks, (uint32_t)__shfl_xor((int)blocks, o, 64));
        longest = max(longest, (uint32_t)__builtin_amdgcn_readfirstlane((int)blocks));
    }
    const uint32_t per = max((total + gridDim.x - 1) / gridDim.x, (longest + KV4_PARTS - 2) / (KV4_PARTS - 1));
    uint32_t at = blockIdx.x * per;
    const uint32_t end = min(total, at + per);

    while (at < end) {
        // ---- the unit at `at`: request, KV head, columns, its block steps
        uint32_t base = 0, blocks = 0;
        int b = 0;
        for (int b0 = 0; b0 < a.B; b0 += 64) {
            uint32_t cost = 0, mine = 0;
            if (b0 + lane < a.B) {
                const Kv4Seq s = kv4_seq(a, b0 + lane);
                mine = unit_blocks(s);
                cost = s.rows > 0 ? mine * seq_units(a, s) : 0;
            }
            const uint32_t incl = wave_scan_add(cost);
            const unsigned long long over = __ballot(base + incl > at);
            if (over) {
                const int j = __builtin_ctzll(over);
                b = b0 + j;
                base += lane_u(incl - cost, j);
                blocks = lane_u(mine, j);
                break;
            }
            base += lane_u(incl, 63);
        }
        const Kv4Seq sq = kv4_seq(a, b);
        const uint32_t rel = at - base, unit = rel / blocks, s0 = rel % blocks;
        const uint32_t nblk = min(blocks - s0, end - at);
        const int ncg = (sq.rows * a.G + 15) / 16;
        const int head = (int)unit / ncg, cg = (int)unit % ncg;
        const int ncol = min(16, sq.rows * a.G - 16 * cg);

        // ---- this lane's column: row, query head and position
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
        // keys that every column of the unit sees: below `all`, and within the last column's window
        const int first_pos = sq.len - sq.rows + 16 * cg / a.G;
        const int last_pos = sq.len - sq.rows + (16 * cg + ncol - 1) / a.G;
        const int all = a.causal ? min(first_pos + 1, sq.len) : sq.len;

        float m = -__builtin_inff(), mbase = 0.0f, l = 0.0f;
        f32x4 acc[NB], off[NG];       // O^T 2^-24 (odd blocks 2^-20) before the 8 comes off, -8 2^-24 sum p s_g
#pragma unroll
        for (int i = 0; i < NB; i++) acc[i] = (f32x4){0, 0, 0, 0};
#pragma unroll
        for (int g = 0; g < NG; g++) off[g] = (f32x4){0, 0, 0, 0};

        // ---- pages of the run, 64 table entries in the lanes at a time
        int page_first = 0, pages = -1;
        bool have_pages = false;
        auto page_of = [&](int key) -> int {
            const int j = key >> c.ps_log2;
            if (!have_pages || j < page_first || j >= page_first + 64) {
                page_first = j;
                have_pages = true;
                pages = j + lane < c.max_pages ? c.table[(size_t)sq.slot * c.max_pages + j + lane] : -1;
            }
            return __builtin_amdgcn_readlane(pages, j - page_first);
        };
        auto key_of = [&](int i) { return KV4_STEP * (i < sq.sinks ? i : sq.main0 + i - sq.sinks); };
        const uint32_t ring_lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)&ring[wid][0][0];
        // step i of the unit into slot s of the ring; whose pages are there
        auto fetch = [&](int i, int s) -> uint32_t {
            const int key0 = key_of(i);
            uint32_t there = 0;
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");     // the slot's last reads are back
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const int k0 = key0 + 16 * t;
                const int page = k0 < sq.len ? page_of(k0) : -1;
                const bool ok = kv4_page_ok(c, page);
                there |= (uint32_t)ok << t;
                const uint8_t* tile = kv4_tile(c, ok ? page : 0, head, (k0 & ((1 << c.ps_log2) - 1)) >> 4) + 16 * lane;
                const uint32_t to = ring_lds + s * SLOT + t * TB;
#pragma unroll
                for (int o = 0; o + 1024 <= TB; o += 1024) lds_dma<16>(tile + o, to + o);
                if (16 * lane < TB % 1024) lds_dma<16>(tile + TB / 1024 * 1024, to + TB / 1024 * 1024);
            }
            return there;
        };
        auto compute = [&](int key0, int s, uint32_t there) {
            const uint8_t* slot = &ring[wid][s][0];
            float x[2][4];
#pragma unroll
            for (int t = 0; t < 2; t++) {
                uint32_t k[D / 32], ks[D / 16];
                load_words(k, slot + t * TB + lane * (D / 8));
                load_words(ks, slot + t * TB + 8 * D + h * (D / 4));
                float even[4] = {0, 0, 0, 0}, odd[4] = {0, 0, 0, 0};
#pragma unroll
                for (int p = 0; p < NG / 2; p++) {
                    const uint32_t w0 = k[2 * p], w1 = k[2 * p + 1];
                    const f32x4 lo = mfma16(low_codes(w0, w1), qf[2 * p], start[2 * p]);
                    const f32x4 hi = mfma16(high_codes(w0, w1), qf[2 * p + 1], start[2 * p + 1]);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        even[i] = __builtin_fmaf(lo[i], half_of(ks[4 * p + i / 2], i & 1), even[i]);
                        odd[i] = __builtin_fmaf(hi[i], half_of(ks[4 * p + 2 + i / 2], i & 1), odd[i]);
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; i++) x[t][i] = __builtin_fmaf(odd[i], kscale * 0.0625f, even[i] * kscale);
            }
            uint32_t v[2][D / 32], vs[2][D / 16];
#pragma unroll
            for (int t = 0; t < 2; t++) {
                load_words(v[t], slot + t * TB + 9 * D + lane * (D / 8));
                load_words(vs[t], slot + t * TB + 17 * D + h * (D / 4));
            }
            const bool whole = there == 3 && key0 + KV4_STEP <= all &&
                               (a.window == 0 || last_pos - key0 <= a.window || key0 + KV4_STEP <= a.sink);
            if (!whole) {
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (!((there >> t & 1) && kv4_sees(a, pos, key0 + 16 * t + 4 * h + i, sq.len)))
                            x[t][i] = -__builtin_inff();
            }
            // the running maximum, where one of the step's scores is above it (a
            // NaN score reaches the sum by itself)
            float top = x[0][0];
#pragma unroll
            for (int i = 1; i < 8; i++) top = __builtin_fmaxf(top, x[i >> 2][i & 3]);
            if (__ballot(top > m)) {
                top = __builtin_fmaxf(top, __shfl_xor(top, 16, 64));
                top = __builtin_fmaxf(top, __shfl_xor(top, 32, 64));
                const float mn = __builtin_fmaxf(m, top);
                mbase = mn > -__builtin_inff() ? mn : 0.0f;
                const float f = exp2_fast(m - mbase);      // 0 where nothing was there
                m = mn;
                l *= f;
#pragma unroll
                for (int i = 0; i < NB; i++) acc[i] *= f;
#pragma unroll
                for (int g = 0; g < NG; g++) off[g] *= f;
            }
            float p[2][4];
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    p[t][i] = exp2_fast(x[t][i] - mbase);
                    l += p[t][i];
                }
#pragma unroll
            for (int g = 0; g < NG; g++) {
                float w[2][4];
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) w[t][i] = p[t][i] * half_of(vs[t][2 * g + i / 2], i & 1);
                if (!whole) {      // a key that is not seen adds nothing, whatever its scale is
#pragma unroll
                    for (int t = 0; t < 2; t++)
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            if (x[t][i] == -__builtin_inff()) w[t][i] = 0.0f;
                }
                const h16x8 pf = frag(pack_h(w[0][0], w[0][2]), pack_h(w[0][1], w[0][3]), pack_h(w[1][0], w[1][2]),
                                      pack_h(w[1][1], w[1][3]));
                acc[2 * g] = mfma16(low_codes(v[0][g], v[1][g]), pf, acc[2 * g]);
                acc[2 * g + 1] = mfma16(high_codes(v[0][g], v[1][g]), pf, acc[2 * g + 1]);
                off[g] = mfma16(minus8(false), pf, off[g]);
            }
        };

        // ---- this wave's steps, the next R - 1 on their way
        const int last = min(sq.steps, (int)(s0 + nblk) * KV4_WAVES), i0 = (int)s0 * KV4_WAVES + wid;
        const int n = i0 < last ? (last - i0 + KV4_WAVES - 1) / KV4_WAVES : 0;
        uint32_t there = 0;          // two bits per slot of the ring
        auto put = [&](int j) {
            const int s = j % R;
            there = (there & ~(3u << 2 * s)) | fetch(i0 + KV4_WAVES * j, s) << 2 * s;
        };
#pragma unroll
        for (int j = 0; j < R - 1; j++)
            if (j < n) put(j);
        for (int j = 0; j < n; j++) {
            if (j + R - 1 < n) {
                put(j + R - 1);
                wait_dma<NI * (R - 1)>();
            } else if (R > 2 && j + R - 2 < n) {
                wait_dma<NI * (R - 2)>();
            } else if (R > 3 && j + R - 3 < n) {
                wait_dma<NI * (R - 3)>();
            } else {
                wait_dma<0>();
            }
            compute(key_of(i0 + KV4_WAVES * j), j % R, there >> 2 * (j % R) & 3u);
        }

        // ---- the waves' shares of the keys meet
        l += __shfl_xor(l, 16, 64);
        l += __shfl_xor(l, 32, 64);
        if (live) {
#pragma unroll
            for (int g = 0; g < NG; g++) {
                *reinterpret_cast<f32x4*>(&o_sh[wid][col * OS + 32 * g + 4 * h]) = (acc[2 * g] + off[g]) * 16777216.0f;
                *reinterpret_cast<f32x4*>(&o_sh[wid][col * OS + 32 * g + 16 + 4 * h]) =
                    (acc[2 * g + 1] * 0.0625f + off[g]) * 16777216.0f;
            }
            if (h == 0) {
                m_sh[wid][col] = m;
                l_sh[wid][col] = l;
            }
        }
        __syncthreads();
        const bool alone = nblk == blocks;
        // parts of the unit: the first workgroup has it at the end of its stretch
        // (slot 1), the others at the start of theirs (slot 0)
        const uint32_t unit0 = base + unit * blocks;
        const uint32_t wg0 = unit0 / per, nparts = (unit0 + blocks - 1) / per - wg0 + 1;
        float* part = a.part + (size_t)(2 * blockIdx.x + (blockIdx.x == wg0)) * 16 * (D + 2);
        for (int e = tid; e < ncol * D; e += 64 * KV4_WAVES) {
            const int cc = e / D, d = e % D;
            float mw = -__builtin_inff();
#pragma unroll
            for (int w = 0; w < KV4_WAVES; w++) mw = __builtin_fmaxf(mw, m_sh[w][cc]);
            float num = 0.0f, den = 0.0f;
#pragma unroll
            for (int w = 0; w < KV4_WAVES; w++) {
                // without a maximum the wave's sums are zero, or NaN from a NaN score
                const float f = m_sh[w][cc] > -__builtin_inff() ? exp2_fast(m_sh[w][cc] - mw) : 1.0f;
                num = __builtin_fmaf(f, o_sh[w][cc * OS + d], num);
                den = __builtin_fmaf(f, l_sh[w][cc], den);
            }
            if (alone) {
                const int vv = 16 * cg + cc;
                a.o[(((size_t)b * a.S + vv / a.G) * a.Hq + (size_t)head * a.G + vv % a.G) * D + d] =
                    f2h(den != 0.0f ? num / den : 0.0f);
            } else {
                agent_store(part + e, num);
                if (d == 0) {
                    agent_store(part + 16 * D + cc, mw);
                    agent_store(part + 16 * D + 16 + cc, den);
                }
            }
        }
        if (!alone) {
            // every store of the workgroup is complete at the coherence point (the
            // partials are agent-scope stores) before the count goes up
            __builtin_amdgcn_s_waitcnt(0);
            __syncthreads();
            if (tid == 0)
                last_sh = __hip_atomic_fetch_add(a.counters + wg0, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == nparts - 1;
            __syncthreads();
            if (last_sh) {
                auto part_of = [&](uint32_t p) {
                    return a.part + (size_t)(2 * (wg0 + p) + (p == 0)) * 16 * (D + 2);
                };
                // 16 threads per column: the parts' maxima and sums
                if (tid < 16 * ncol) {
                    const int cc = tid >> 4;
                    float mx = -__builtin_inff();
                    for (uint32_t p = tid & 15; p < nparts; p += 16) {
                        const float v = agent_load(part_of(p) + 16 * D + cc);
                        w_sh[p][cc] = v;
                        mx = __builtin_fmaxf(mx, v);
                    }
#pragma unroll
                    for (int o = 1; o < 16; o <<= 1) mx = __builtin_fmaxf(mx, __shfl_xor(mx, o, 64));
                    float sum = 0.0f;
                    for (uint32_t p = tid & 15; p < nparts; p += 16) {
                        const float v = w_sh[p][cc];
                        const float f = v > -__builtin_inff() ? exp2_fast(v - mx) : 1.0f;
                        w_sh[p][cc] = f;
                        sum = __builtin_fmaf(f, agent_load(part_of(p) + 16 * D + 16 + cc), sum);
                    }
#pragma unroll
                    for (int o = 1; o < 16; o <<= 1) sum += __shfl_xor(sum, o, 64);
                    if ((tid & 15) == 0) w_sh[KV4_PARTS][cc] = sum;
                }
                __syncthreads();
                for (int e = tid; e < ncol * D; e += 64 * KV4_WAVES) {
                    const int cc = e / D, d = e % D;
                    float num = 0.0f;
#pragma unroll 8
                    for (uint32_t p = 0; p < nparts; p++)
                        num = __builtin_fmaf(w_sh[p][cc], agent_load(part_of(p) + e), num);
                    const float den = w_sh[KV4_PARTS][cc];
                    const int vv = 16 * cg + cc;
                    a.o[(((size_t)b * a.S + vv / a.G) * a.Hq + (size_t)head * a.G + vv % a.G) * D + d] =
                        f2h(den != 0.0f ? num / den : 0.0f);
                }
                if (tid == 0) __hip_atomic_store(a.counters + wg0, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
        }
        __syncthreads();
        at += nblk;
    }
}

}  // namespace cactus_hip

using namespace cactus_hip;

extern "C" {

size_t cactus_hip_attention_kv4_workspace(const cactus_hip_kv4_cache* cache, size_t batch, size_t seq_len,
                                          size_t num_q_heads) {
    (void)batch; (void)seq_len; (void)num_q_heads;
    if (kv4_view(cache, 0, "attention_kv4_workspace", nullptr)) return 0;
    return KV4_COUNTERS + (size_t)KV4_GRID * 2 * 16 * (cache->head_dim + 2) * 4;
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
    a.counters = static_cast<uint32_t*>(workspace);
    a.part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + KV4_COUNTERS);
    // block steps at most, by what the tables can hold
    const size_t blocks = (cache->max_pages * cache->page_size + KV4_BLOCK - 1) / KV4_BLOCK;
    const size_t units = batch * cache->kv_heads * ceil_div(seq_len * G, 16);
    if (units >= (1u << 31) / blocks)
        return fail(CACTUS_HIP_EUNSUPPORTED, "attention_kv4: batch times rows times table length is too large");
    const dim3 grid((unsigned)std::min<size_t>(KV4_GRID, units * blocks)), block(64 * KV4_WAVES);
    const hipStream_t st = as_stream(stream);
    switch (a.c.d) {
        case 64: hipLaunchKernelGGL(attn_kv4_kernel<64>, grid, block, 0, st, a); break;
        case 128: hipLaunchKernelGGL(attn_kv4_kernel<128>, grid, block, 0, st, a); break;
        default: hipLaunchKernelGGL(attn_kv4_kernel<256>, grid, block, 0, st, a);
    }
    return check_launch("attention_kv4");
}

}  // extern "C"
