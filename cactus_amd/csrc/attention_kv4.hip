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
// rounded to FP16 after the scale (2^-11 relative each, lifted by a power of two
// so that small ones keep their bits): the matrix instruction takes them so,
// and the sum of thousands averages it out.
#include "kv4_device.h"

#include <algorithm>
#include <math.h>

namespace cactus_hip {

typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

// n / d for 0 <= n < 2^31: n m / 2^(31 + s) with 2^s the power of two at or above d
// and m = 2^(31 + s) / d + 1, whose error n / 2^(31 + s) stays below 1 / d
struct FastDiv {
    uint32_t m = 0;
    int s = 0;
    void set(uint32_t d) {
        for (s = 0; (1ull << s) < d; s++) {}
        m = (uint32_t)((1ull << (31 + s)) / d + 1);
    }
    __device__ __forceinline__ int operator()(int n) const { return s == 0 ? n : (int)(__umulhi((uint32_t)n, m) >> (s - 1)); }
};

struct Kv4AttnArgs {
    Kv4View c;
    const int32_t* seqs;
    const int32_t* counts;
    const uint16_t* q;
    uint16_t* o;
    size_t q_stride;
    int B, S, Hq, G;          // G query heads per KV head
    FastDiv by_g, by_nvb;     // division by G, and by the blocks of query vectors of a request
    int window, sink, causal; // window 0: none
    int join_log2;            // parts that the few-row kernel joins at a time
    float scale;              // times log2(e): the softmax runs in powers of two
    uint32_t* counters;       // [workgroups] zero between calls
    float* part;              // [workgroups][2][vectors][D + 4]: output, maximum, sum
};

// rows and keys of one request
struct Kv4Seq {
    int slot, len, rows;      // tokens; rows that stand at the last positions
    int main0, sinks, steps;  // 32-key steps: [0, sinks) and from main0 on; steps in all
};
constexpr int KV4_STEP = 32;

__device__ __forceinline__ Kv4Seq kv4_span(const Kv4AttnArgs& a, int slot, int len, int rows) {
    Kv4Seq s;
    s.slot = slot;
    s.len = len;
    s.rows = rows;
    const int p0 = s.len - s.rows;                       // first row's position: its window reaches furthest back
    int lo = a.window > 0 && p0 > a.window ? p0 - a.window : 0;
    s.main0 = lo / KV4_STEP;
    s.sinks = a.window > 0 ? min((min(a.sink, s.len) + KV4_STEP - 1) / KV4_STEP, s.main0) : 0;
    s.steps = s.sinks + (s.len + KV4_STEP - 1) / KV4_STEP - s.main0;
    return s;
}
__device__ __forceinline__ Kv4Seq kv4_seq(const Kv4AttnArgs& a, int b) {
    const int slot = kv4_slot(a.c, a.seqs, b);
    return kv4_span(a, slot, slot < 0 ? 0 : kv4_len(a.c, slot), slot < 0 ? 0 : kv4_count(a.counts, b, a.S));
}

// whether the row at position p sees key j of n
__device__ __forceinline__ bool kv4_sees(const Kv4AttnArgs& a, int p, int j, int n) {
    return (j < n) & (!a.causal | (j <= p)) & ((a.window == 0) | (p - j <= a.window) | (j < a.sink));
}

// row of o, in heads, that query vector vv of a KV head has within its request
__device__ __forceinline__ size_t out_offset(const Kv4AttnArgs& a, int head, int vv) {
    const int row = a.by_g(vv);
    return (size_t)row * a.Hq + (size_t)(head * a.G + vv - row * a.G);
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
// pairs of values that workgroups hand to each other
__device__ __forceinline__ float2 agent_load2(const float* p) {
    const uint64_t u = __hip_atomic_load(reinterpret_cast<const uint64_t*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return make_float2(bits_f((uint32_t)u), bits_f((uint32_t)(u >> 32)));
}
__device__ __forceinline__ void agent_store2(float* p, float x, float y) {
    const uint64_t u = __builtin_bit_cast(uint32_t, x) | (uint64_t)__builtin_bit_cast(uint32_t, y) << 32;
    __hip_atomic_store(reinterpret_cast<uint64_t*>(p), u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
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

// ------------------------------------------------------------ few rows
// The work is a line of block steps (32 keys per wave of one unit: a request's
// KV head and up to 16 query vectors), unit after unit, request after
// request; each workgroup takes an equal stretch of it, whatever the lengths
// of the sequences are.  A unit that lies in one stretch is written at once;
// one that several workgroups share is written as partial (maximum, sum,
// output) to the workspace, and the last of them to finish joins the parts
// in their order.
constexpr int KV4_PARTS = 128;                    // a unit's stretches at most
constexpr size_t KV4_COUNTERS = 4096;             // bytes: one counter per workgroup

// block steps of a unit (one at least: a request without tokens gets its zeros)
template <int W>
__device__ __forceinline__ uint32_t unit_blocks(const Kv4Seq& s) {
    return (uint32_t)max(1, (s.steps + W - 1) / W);
}

// Query vectors of a unit.  PACK: a vector takes NG = d / 32 of the product's
// 16 columns, one per scale group, so that a lane multiplies by one group's
// scale and the softmax runs once per lane, not per group; the products' other
// groups' columns are computed and not used.  Otherwise a column is a vector
// and each lane scales all its groups.
template <int D, bool PACK>
constexpr int kv4_vectors() { return PACK ? 16 / (D / 32) : 16; }
// Steps of a wave's ring in LDS, workgroups per CU
template <int D, bool PACK>
constexpr int kv4_ring() { return D == 64 ? 4 : PACK || D == 256 ? 2 : 3; }
// Waves of a workgroup: with 16 vectors, twice the keys per part, whose joining
// costs as much as the keys (16 rows at 4096 keys, 16 / 8 heads of 128: 24 us with
// four waves, 14 with eight; one row 9.2 against 10.4)
template <int D, bool PACK>
constexpr int kv4_waves() { return PACK ? 4 : 8; }
template <int D, bool PACK>
constexpr int kv4_per_cu() { return PACK ? (D == 256 ? 2 : 4) : D == 64 ? 2 : 1; }

// threads that share a quad of dims, of `quads`, when parts are joined
template <int D, bool PACK>
__host__ __device__ constexpr int kv4_shares(int quads) {
    return 64 * kv4_waves<D, PACK>() > quads ? 64 * kv4_waves<D, PACK>() / quads : 1;
}

// a times half I of w plus c, one instruction (v_fma_mix_f32; as a builtin, so that
// the compiler knows what waits for the matrix and transcendental units' results)
template <int I>
__device__ __forceinline__ float fma_half(float a, uint32_t w, float c) {
    return __builtin_fmaf(a, h2f((uint16_t)(I ? w >> 16 : w)), c);
}
template <int I>
__device__ __forceinline__ float mul_half(float a, uint32_t w) { return fma_half<I>(a, w, 0.0f); }
template <int CTRL>
__device__ __forceinline__ float add_dpp(float v) {
    return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true));
}
// sum over the N lanes of a group (consecutive lanes, N = 2, 4 or 8), in each of them
template <int N>
__device__ __forceinline__ float sum_lanes(float v) {
    v = add_dpp<0xB1>(v);                        // quad_perm [1,0,3,2]
    if constexpr (N > 2) v = add_dpp<0x4E>(v);   // quad_perm [2,3,0,1]
    if constexpr (N > 4) v = add_dpp<0x141>(v);  // row_half_mirror
    return v;
}
__device__ __forceinline__ float max3(float a, float b, float c) { return __builtin_fmaxf(__builtin_fmaxf(a, b), c); }
// f over the four lanes of a column (16 apart), in each of them, by lane swaps: a step in
// which the maximum rises waits for the result twice
template <class F>
__device__ __forceinline__ float column(float v, F f) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);     // rows 0, 0, 2, 2 and 1, 1, 3, 3
    const uint32_t w = __builtin_bit_cast(uint32_t, f(bits_f(r[0]), bits_f(r[1])));
    const auto t = __builtin_amdgcn_permlane32_swap(w, w, false, false);     // the lower half twice, and the upper one
    return f(bits_f(t[0]), bits_f(t[1]));
}
__device__ __forceinline__ float column_max(float v) {
    return column(v, [](float a, float b) { return __builtin_fmaxf(a, b); });
}
__device__ __forceinline__ float column_sum(float v) {
    return column(v, [](float a, float b) { return a + b; });
}

// 16 bytes per active lane to LDS; ONCE: not to be kept in the caches
template <bool ONCE>
__device__ __forceinline__ void tile_dma(const void* src, uint32_t lds_addr) {
    if constexpr (ONCE) {
        const uint32_t lds = (uint32_t)__builtin_amdgcn_readfirstlane((int)lds_addr);
        asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off nt" ::"v"(src), "s"(lds) : "memory");
    } else {
        lds_dma<16>(src, lds_addr);
    }
}

template <int D, bool PACK>
__global__ void __launch_bounds__((64 * kv4_waves<D, PACK>()), (kv4_per_cu<D, PACK>() * kv4_waves<D, PACK>() / 4)) attn_kv4_kernel(Kv4AttnArgs a) {
    constexpr int W = kv4_waves<D, PACK>();
    constexpr int NG = D / 32, NB = D / 16, OS = D + 4, QV = kv4_vectors<D, PACK>();
    constexpr int SG = PACK ? 1 : NG;                          // scale groups of a lane
    constexpr int TB = 18 * D, SLOT = 2 * TB;                  // bytes of a tile and of a step
    constexpr int NI = 2 * ((TB + 1023) / 1024);               // LDS loads of a step
    constexpr int R = kv4_ring<D, PACK>();
    static_assert(R * SLOT >= QV * OS * 4 && W * R * SLOT >= 64 * W * 24,
                  "the ring holds a wave's sums, then the joined parts'");
    __shared__ __align__(16) uint8_t ring[W][R][SLOT];
    __shared__ float m_sh[W][QV], l_sh[W][QV];
    __shared__ int last_sh;
    float (*o_sh)[R * SLOT / 4] = reinterpret_cast<float (*)[R * SLOT / 4]>(&ring[0][0][0]);   // [wave][QV][OS]
    float* j_sh = reinterpret_cast<float*>(&ring[0][0][0]);    // [threads][6]: sums of parts
    const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, h = lane >> 4;
    const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int qi = PACK ? col / NG : col, gi = PACK ? col % NG : 0;    // the lane's query vector and group
    const Kv4View& c = a.c;
    // PACK: odd groups' codes are 16 times theirs
    const float kscale = a.scale * 16777216.0f * (PACK && (gi & 1) ? 0.0625f : 1.0f);

    // ---- 64 requests at a time, one per lane: slot, tokens, rows, block steps
    // of a unit, and how far the line reaches with this request
    int r_slot = -1, r_len = 0, r_rows = 0;
    uint32_t r_blocks = 0, r_cost = 0, r_upto = 0;
    auto look = [&](int b0) {
        r_rows = 0;
        r_blocks = r_cost = 0;
        if (b0 + lane < a.B) {
            const Kv4Seq s = kv4_seq(a, b0 + lane);
            r_slot = s.slot;
            r_len = s.len;
            r_rows = s.rows;
            r_blocks = s.rows > 0 ? unit_blocks<W>(s) : 0;
            r_cost = r_blocks * (uint32_t)((s.rows * a.G + QV - 1) / QV) * (uint32_t)c.Hkv;
        }
        r_upto = wave_scan_add(r_cost);
    };
    // ---- this workgroup's stretch [at, end) of the line
    uint32_t total = 0;
    int longest = 1;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
        look(b0);
        total += lane_u(r_upto, 63);
        longest = max(longest, __builtin_amdgcn_readlane(wave_scan_max((int)r_blocks), 63));
    }
    uint32_t per = max((total + gridDim.x - 1) / gridDim.x, ((uint32_t)longest + KV4_PARTS - 2) / (KV4_PARTS - 1));
    // The joining takes 2^join_log2 parts at a time, which costs as much as two steps:
    // longer stretches, for one or two such rounds, where that saves more (one row at
    // 9000 keys, 16 / 8 heads of 128, in stretches of 1, 2, 3 and 4 steps: 14.2, 12.8,
    // 11.3 and 12.7 us; at 4096, one round in any case: 9.1, 10.3, 11.1 and 12.0; at
    // 32000: 24.8 -> 16.8; heads of 64 and 256 were not timed).  With 16 vectors a
    // step costs more than a round.
    if constexpr (PACK) {
        const uint32_t one = ((uint32_t)longest + (1u << a.join_log2) - 1) >> a.join_log2;   // steps of a part for one round
        const uint32_t rounds = (uint32_t)((float)(one + per - 1) * __builtin_amdgcn_rcpf((float)per));
        const uint32_t q = one <= 3 ? one : (one + 1) / 2;
        if (q > per && q + (one <= 3 ? 2 : 4) < per + 2 * rounds) per = q;
    }
    // Stretches that end inside a unit cost their workgroup another unit's start (7
    // us, where a block step takes 0.5 to 3).  If units cut into whole parts of at
    // most `per` steps, or one or two more, make no more parts than there are
    // workgroups, each takes a part (up to five rows of 8 sequences 18.7 -> 16.7 us);
    // the line then counts parts.  (Of long stretches the ends matter less than
    // equal lengths.)
    bool parts = false;
    if (a.B <= 64 && per > 1 && per <= 12) {
        const uint32_t units = r_blocks ? r_cost / r_blocks : 0;
        for (uint32_t q = per; q <= per + 2 && !parts; q++) {
            const uint32_t cost = units * ((r_blocks + q - 1) / q), upto = wave_scan_add(cost);
            if (lane_u(upto, 63) <= gridDim.x) {
                parts = true;
                per = q;
                total = lane_u(upto, 63);
                r_cost = cost;
                r_upto = upto;
            }
        }
    }
    uint32_t at = parts ? blockIdx.x : blockIdx.x * per;
    const uint32_t end = min(total, parts ? at + 1 : at + per);

    while (at < end) {
        // ---- the unit at `at`: request, KV head, vectors, its block steps
        uint32_t base = 0;
        int b = 0, j = 0;
        for (int b0 = 0; b0 < a.B; b0 += 64) {
            if (a.B > 64) look(b0);
            const unsigned long long over = __ballot(base + r_upto > at);
            if (over) {
                j = __builtin_ctzll(over);
                b = b0 + j;
                base += lane_u(r_upto - r_cost, j);
                break;
            }
            base += lane_u(r_upto, 63);
        }
        const uint32_t blocks = lane_u(r_blocks, j);
        const Kv4Seq sq = kv4_span(a, __builtin_amdgcn_readlane(r_slot, j), __builtin_amdgcn_readlane(r_len, j),
                                   __builtin_amdgcn_readlane(r_rows, j));
        const uint32_t nparts = (blocks + per - 1) / per;            // (of a unit in parts)
        const uint32_t rel = at - base, unit = rel / (parts ? nparts : blocks), first = rel - unit * (parts ? nparts : blocks);
        const uint32_t s0 = parts ? first * per : first;
        const uint32_t nblk = min(blocks - s0, parts ? per : end - at);
        const int ncg = (sq.rows * a.G + QV - 1) / QV;
        const int head = ncg == 1 ? (int)unit : (int)unit / ncg, v0 = ncg == 1 ? 0 : (int)unit % ncg * QV;
        const int nvec = min(QV, sq.rows * a.G - v0);

        // ---- pages of the run, 64 table entries in the lanes at a time
        int page_first = 0, pages = -1;
        bool have_pages = false;
        auto page_of = [&](int key) -> int {
            const int e = key >> c.ps_log2;
            if (!have_pages || e < page_first || e >= page_first + 64) {
                page_first = e;
                have_pages = true;
                pages = c.table[(size_t)sq.slot * c.max_pages + min(e + lane, c.max_pages - 1)];
                // waited for here: at its use a wait would hold up the tiles under way each time
                __builtin_amdgcn_s_waitcnt(0x0F70);     // vmcnt(0)
            }
            return __builtin_amdgcn_readlane(pages, e - page_first);
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
                for (int o = 0; o + 1024 <= TB; o += 1024) tile_dma<PACK>(tile + o, to + o);
                if (16 * lane < TB % 1024) tile_dma<PACK>(tile + TB / 1024 * 1024, to + TB / 1024 * 1024);
            }
            return there;
        };
        // ---- this wave's steps, the first R - 1 on their way
        const int last = min(sq.steps, (int)(s0 + nblk) * W), i0 = (int)s0 * W + wid;
        const int n = i0 < last ? (last - i0 + W - 1) / W : 0;
        uint32_t there = 0;          // two bits per slot of the ring
        auto put = [&](int k) {
            const int s = k % R;
            there = (there & ~(3u << 2 * s)) | fetch(i0 + W * k, s) << 2 * s;
        };
#pragma unroll 1
        for (int k = 0; k < min(R - 1, n); k++) put(k);

        // ---- this lane's vector: row, query head and position
        const int vec = v0 + qi, row = a.by_g(vec);
        const bool live = qi < nvec;
        const int pos = sq.len - sq.rows + row;
        h16x8 qf[NG];
        f32x4 start[SG];
#pragma unroll
        for (int g = 0; g < NG; g++) {
            uint4 u = make_uint4(0, 0, 0, 0);
            if (live && (!PACK || g == gi))
                u = *reinterpret_cast<const uint4*>(a.q + ((size_t)b * a.S + row) * a.q_stride +
                                                    (size_t)(head * a.G + vec - row * a.G) * D + 32 * g + 8 * h);
            qf[g] = code_order(u);
        }
#pragma unroll
        for (int g = 0; g < NG; g++)
            start[PACK ? 0 : g] = mfma16(minus8(g & 1), qf[g], PACK && g > 0 ? start[0] : (f32x4){0, 0, 0, 0});
        // keys that every vector of the unit sees: below `all`, and within the last one's window
        const int first_pos = sq.len - sq.rows + a.by_g(v0);
        const int last_pos = sq.len - sq.rows + a.by_g(v0 + nvec - 1);
        const int all = a.causal ? min(first_pos + 1, sq.len) : sq.len;

        // The products p s are lifted by 2^lift_exp before they become FP16: so that a
        // step's largest is below 2^12 where it is chosen (as the maximum rises, or
        // when a product reaches 2^15; FP16 holds 2^16).  It then keeps its 11 bits
        // down to 2^-25 of that product.  (Without it the weights of small values, or of many
        // keys beside one that takes most of the weight, fell to FP16 subnormals or
        // to zero; chosen by the scales alone, one key of large values and no
        // weight did that to the others.  It costs 2% of a decode step of 32 requests,
        // 10% of five drafted rows of heads of 64.)
        int lift_exp = 26;
        float lift = 0x1p26f;
        uint32_t scale_end = 0;      // 2^15 / lift: below it no scale's products reach 2^15
        float m = -__builtin_inff(), mbase = 0.0f, l = 0.0f;
        f32x4 acc[NB], off[SG];       // O^T 2^-24 (odd blocks 2^-20) before the 8 comes off, -8 2^-24 sum p s_g
#pragma unroll
        for (int i = 0; i < NB; i++) acc[i] = (f32x4){0, 0, 0, 0};
#pragma unroll
        for (int g = 0; g < SG; g++) off[g] = (f32x4){0, 0, 0, 0};

        auto compute = [&](bool whole, int key0, int s, uint32_t there) {
            const uint8_t* slot = &ring[wid][s][0];
            float x[2][4];
#pragma unroll
            for (int t = 0; t < 2; t++) {
                uint32_t k[D / 32], ks[2 * SG];
                load_words(k, slot + t * TB + lane * (D / 8));
                load_words(ks, slot + t * TB + 8 * D + h * (D / 4) + gi * 8);
                if constexpr (PACK) {
                    f32x4 st = start[0];
#pragma unroll
                    for (int p = 0; p < NG / 2; p++) {
                        st = mfma16(low_codes(k[2 * p], k[2 * p + 1]), qf[2 * p], st);
                        st = mfma16(high_codes(k[2 * p], k[2 * p + 1]), qf[2 * p + 1], st);
                    }
                    x[t][0] = sum_lanes<NG>(mul_half<0>(st[0] * kscale, ks[0]));
                    x[t][1] = sum_lanes<NG>(mul_half<1>(st[1] * kscale, ks[0]));
                    x[t][2] = sum_lanes<NG>(mul_half<0>(st[2] * kscale, ks[1]));
                    x[t][3] = sum_lanes<NG>(mul_half<1>(st[3] * kscale, ks[1]));
                } else {
                    float even[4] = {0, 0, 0, 0}, odd[4] = {0, 0, 0, 0};
#pragma unroll
                    for (int p = 0; p < NG / 2; p++) {
                        const f32x4 lo = mfma16(low_codes(k[2 * p], k[2 * p + 1]), qf[2 * p], start[2 * p]);
                        const f32x4 hi = mfma16(high_codes(k[2 * p], k[2 * p + 1]), qf[2 * p + 1], start[2 * p + 1]);
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            even[2 * i] = fma_half<0>(lo[2 * i], ks[4 * p + i], even[2 * i]);
                            even[2 * i + 1] = fma_half<1>(lo[2 * i + 1], ks[4 * p + i], even[2 * i + 1]);
                            odd[2 * i] = fma_half<0>(hi[2 * i], ks[4 * p + 2 + i], odd[2 * i]);
                            odd[2 * i + 1] = fma_half<1>(hi[2 * i + 1], ks[4 * p + 2 + i], odd[2 * i + 1]);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 4; i++) x[t][i] = __builtin_fmaf(odd[i], kscale * 0.0625f, even[i] * kscale);
                }
            }
            uint32_t v[2][D / 32], vs[2][2 * SG];
#pragma unroll
            for (int t = 0; t < 2; t++) {
                load_words(v[t], slot + t * TB + 9 * D + lane * (D / 8));
                load_words(vs[t], slot + t * TB + 17 * D + h * (D / 4) + gi * 8);
            }
            if (!whole) {     // a key that is not seen adds nothing, whatever its scales are
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const bool sees = (there >> t & 1) & kv4_sees(a, pos, key0 + 16 * t + 4 * h + i, sq.len);
                        x[t][i] = sees ? x[t][i] : -__builtin_inff();
#pragma unroll
                        for (int g = 0; g < SG; g++)
                            vs[t][2 * g + i / 2] = sees ? vs[t][2 * g + i / 2] : vs[t][2 * g + i / 2] & (i & 1 ? 0xFFFFu : 0xFFFF0000u);
                    }
            }
            // the running maximum, where one of the step's scores is above it (a
            // NaN score reaches the sum by itself)
            float top = max3(max3(x[0][0], x[0][1], x[0][2]), max3(x[0][3], x[1][0], x[1][1]), __builtin_fmaxf(x[1][2], x[1][3]));
            const bool rises = __ballot(top > m) != 0;
            float f = 1.0f;
            if (rises) {
                top = column_max(top);
                const float mn = __builtin_fmaxf(m, top);
                mbase = mn > -__builtin_inff() ? mn : 0.0f;
                f = exp2_fast(m - mbase);                  // 0 where nothing was there
                m = mn;
                l *= f;
            }
            float p[2][4];
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    p[t][i] = exp2_fast(x[t][i] - mbase);
                    l += p[t][i];
                }
            u16x2 sc = __builtin_bit_cast(u16x2, vs[0][0]);
#pragma unroll
            for (int k = 1; k < 4 * SG; k++)
                sc = __builtin_elementwise_max(sc, __builtin_bit_cast(u16x2, vs[k / (2 * SG)][k % (2 * SG)]));
            // (no weight is above 1, and no product of the lane above that of its largest
            // weight and largest scale)
            const uint32_t top_scale = max((uint32_t)sc[0], (uint32_t)sc[1]);
            if (rises || (__ballot(top_scale >= scale_end) &&
                          __ballot(!(exp2_fast(top - mbase) * lift * h2f((uint16_t)top_scale) < 0x1p15f)))) {
                float most = 0.0f;
#pragma unroll
                for (int k = 0; k < 4 * SG; k++) {
                    const int t = k / (2 * SG), i = 2 * (k & 1);
                    uint32_t s = vs[t][k % (2 * SG)];
                    asm volatile("" : "+v"(s));      // (converted here: held until the products, the scales spilled)
                    most = max3(most, __builtin_fabsf(mul_half<0>(p[t][i], s)), __builtin_fabsf(mul_half<1>(p[t][i + 1], s)));
                }
                most = column_max(most);             // (NaNs are not counted)
                const int to = most > 0.0f ? min(12 - __builtin_amdgcn_frexp_expf(most), 26) : 26;
                const float fs = __builtin_ldexpf(f, to - lift_exp);
                lift_exp = to;
                lift = __builtin_ldexpf(1.0f, to);
                scale_end = (uint32_t)(30 - to) << 10;
#pragma unroll
                for (int i = 0; i < NB; i++) acc[i] *= fs;
#pragma unroll
                for (int g = 0; g < SG; g++) off[g] *= fs;
            }
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) p[t][i] *= lift;
            h16x8 pf[SG];
#pragma unroll
            for (int g = 0; g < SG; g++) {
                float w[2][4];
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    w[t][0] = mul_half<0>(p[t][0], vs[t][2 * g]);
                    w[t][1] = mul_half<1>(p[t][1], vs[t][2 * g]);
                    w[t][2] = mul_half<0>(p[t][2], vs[t][2 * g + 1]);
                    w[t][3] = mul_half<1>(p[t][3], vs[t][2 * g + 1]);
                }
                pf[g] = frag(pack_h(w[0][0], w[0][2]), pack_h(w[0][1], w[0][3]), pack_h(w[1][0], w[1][2]),
                             pack_h(w[1][1], w[1][3]));
                off[g] = mfma16(minus8(false), pf[g], off[g]);
            }
            // the codes of the groups that follow are not taken apart ahead of their
            // products (the registers that this holds spilled)
#pragma unroll
            for (int g = 0; g < NG; g++) {
                __builtin_amdgcn_sched_barrier(0);
                acc[2 * g] = mfma16(low_codes(v[0][g], v[1][g]), pf[PACK ? 0 : g], acc[2 * g]);
                acc[2 * g + 1] = mfma16(high_codes(v[0][g], v[1][g]), pf[PACK ? 0 : g], acc[2 * g + 1]);
            }
        };
#pragma unroll 1
        for (int k = 0; k < n; k++) {
            if (k + R - 1 < n) {
                put(k + R - 1);
                wait_dma<NI * (R - 1)>();
            } else if (R > 2 && k + R - 2 < n) {
                wait_dma<NI * (R - 2)>();
            } else if (R > 3 && k + R - 3 < n) {
                wait_dma<NI * (R - 3)>();
            } else {
                wait_dma<0>();
            }
            const int key0 = key_of(i0 + W * k), s = k % R;
            const uint32_t ok = there >> 2 * s & 3u;
            const bool whole = ok == 3 && key0 + KV4_STEP <= all &&
                               (a.window == 0 || last_pos - key0 <= a.window || key0 + KV4_STEP <= a.sink);
            compute(whole, key0, s, ok);
        }

        // ---- the waves' shares of the keys meet
        // (the thread's number hidden from the compiler, which would hold what follows
        // from it in registers over the steps: 40 of them, a workgroup per CU less)
        int et = tid;
        asm volatile("" : "+v"(et));
        const int eh = (et & 63) >> 4;
        l = column_sum(l);
        const float drop = __builtin_ldexpf(1.0f, 24 - lift_exp);      // the lift, and the codes' 2^-24
        if (live) {
#pragma unroll
            for (int g = 0; g < NG; g++) {
                if (PACK && g != gi) continue;
                const f32x4 o8 = off[PACK ? 0 : g];
                *reinterpret_cast<f32x4*>(&o_sh[wid][qi * OS + 32 * g + 4 * eh]) = (acc[2 * g] + o8) * drop;
                *reinterpret_cast<f32x4*>(&o_sh[wid][qi * OS + 32 * g + 16 + 4 * eh]) =
                    (acc[2 * g + 1] * 0.0625f + o8) * drop;
            }
            if (eh == 0 && gi == 0) {
                m_sh[wid][qi] = m;
                l_sh[wid][qi] = l;
            }
        }
        __syncthreads();
        const bool alone = nblk == blocks;
        // parts of the unit: the first workgroup has it at the end of its stretch
        // (slot 1), the others at the start of theirs (slot 0)
        const uint32_t unit0 = base + unit * blocks;
        const uint32_t wg0 = alone ? 0 : parts ? blockIdx.x - first : unit0 / per;
        const uint32_t joined = parts ? nparts : (unit0 + blocks - 1) / per - wg0 + 1;
        // rows of D sums, maximum, sum of weights
        auto part_row = [&](uint32_t wg, int cc) {
            return a.part + ((size_t)(2 * wg + (wg == wg0)) * QV + cc) * (D + 4);
        };
        auto write_row = [&](int cc, int d, f32x4 num, float den) {
            const int vv = v0 + cc;
            const float inv = den != 0.0f ? 1.0f / den : 0.0f;
            uint16_t r[4];
#pragma unroll
            for (int i = 0; i < 4; i++) r[i] = f2h(num[i] * inv);
            *reinterpret_cast<uint2*>(a.o + ((size_t)b * a.S * a.Hq + out_offset(a, head, vv)) * D + d) =
                make_uint2(r[0] | (uint32_t)r[1] << 16, r[2] | (uint32_t)r[3] << 16);
        };
        const int nquad = nvec * (D / 4);
        for (int e = et; e < nquad; e += 64 * W) {
            const int cc = e / (D / 4), d = e % (D / 4) * 4;
            float mw = m_sh[0][cc];
#pragma unroll
            for (int w = 1; w < W; w++) mw = __builtin_fmaxf(mw, m_sh[w][cc]);
            f32x4 num = {0, 0, 0, 0};
            float den = 0.0f;
#pragma unroll
            for (int w = 0; w < W; w++) {
                // without a maximum the wave's sums are zero, or NaN from a NaN score
                const float f = m_sh[w][cc] > -__builtin_inff() ? exp2_fast(m_sh[w][cc] - mw) : 1.0f;
                const f32x4 y = *reinterpret_cast<const f32x4*>(&o_sh[w][cc * OS + d]);
#pragma unroll
                for (int i = 0; i < 4; i++) num[i] = __builtin_fmaf(f, y[i], num[i]);
                den = __builtin_fmaf(f, l_sh[w][cc], den);
            }
            if (alone) {
                write_row(cc, d, num, den);
            } else {
                float* row_at = part_row(blockIdx.x, cc);
                agent_store2(row_at + d, num[0], num[1]);
                agent_store2(row_at + d + 2, num[2], num[3]);
                if (d == 0) agent_store2(row_at + D, mw, den);
            }
        }
        if (!alone) {
            // every store of the workgroup is complete at the coherence point (the
            // partials are agent-scope stores) before the count goes up
            __builtin_amdgcn_s_waitcnt(0);
            __syncthreads();
            if (et == 0)
                last_sh = __hip_atomic_fetch_add(a.counters + wg0, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == joined - 1;
            __syncthreads();
            if (last_sh) {
                // a thread takes a quad of dims and every (threads / quads)-th part,
                // eight parts' loads at a time: 4096 keys in 32 parts take one round of
                // loads (a part after the other: 4 us more)
                const int share = kv4_shares<D, PACK>(nquad);
                for (int e0 = 0; e0 < nquad; e0 += 64 * W) {
                    const int e = e0 + (share > 1 ? et % nquad : et), pl = share > 1 ? et / nquad : 0;
                    const bool in = e < nquad && pl < share;
                    const int cc = in ? e / (D / 4) : 0, d = in ? e % (D / 4) * 4 : 0;
                    f32x4 num = {0, 0, 0, 0};
                    float mx = -__builtin_inff(), den = 0.0f;
                    for (int p0 = pl; in && p0 < (int)joined; p0 += 8 * share) {
                        f32x4 y[8];
                        float2 ml[8];
#pragma unroll
                        for (int u = 0; u < 8; u++) {
                            y[u] = (f32x4){0, 0, 0, 0};
                            ml[u] = make_float2(-__builtin_inff(), 0.0f);
                            if (p0 + u * share < (int)joined) {
                                const float* row_at = part_row(wg0 + p0 + u * share, cc);
                                const float2 lo = agent_load2(row_at + d), hi = agent_load2(row_at + d + 2);
                                y[u] = (f32x4){lo.x, lo.y, hi.x, hi.y};
                                ml[u] = agent_load2(row_at + D);
                            }
                        }
                        float mn = mx;
#pragma unroll
                        for (int u = 0; u < 8; u++) mn = __builtin_fmaxf(mn, ml[u].x);
                        const float f0 = mx > -__builtin_inff() ? exp2_fast(mx - mn) : 1.0f;
                        mx = mn;
                        num *= f0;
                        den *= f0;
#pragma unroll
                        for (int u = 0; u < 8; u++) {
                            const float f = ml[u].x > -__builtin_inff() ? exp2_fast(ml[u].x - mx) : 1.0f;
#pragma unroll
                            for (int i = 0; i < 4; i++) num[i] = __builtin_fmaf(f, y[u][i], num[i]);
                            den = __builtin_fmaf(f, ml[u].y, den);
                        }
                    }
                    if (share > 1) {
                        if (in) {
                            float* s = &j_sh[(pl * nquad + e) * 6];
                            s[0] = num[0], s[1] = num[1], s[2] = num[2], s[3] = num[3], s[4] = mx, s[5] = den;
                        }
                        __syncthreads();
                        if (et < nquad) {
                            mx = j_sh[e * 6 + 4];
                            for (int u = 1; u < share; u++) mx = __builtin_fmaxf(mx, j_sh[(u * nquad + e) * 6 + 4]);
                            num = (f32x4){0, 0, 0, 0};
                            den = 0.0f;
                            for (int u = 0; u < share; u++) {
                                const float* s = &j_sh[(u * nquad + e) * 6];
                                const float f = s[4] > -__builtin_inff() ? exp2_fast(s[4] - mx) : 1.0f;
#pragma unroll
                                for (int i = 0; i < 4; i++) num[i] = __builtin_fmaf(f, s[i], num[i]);
                                den = __builtin_fmaf(f, s[5], den);
                            }
                        }
                    }
                    if (share > 1 ? et < nquad : in) write_row(cc, d, num, den);
                }
                if (et == 0) __hip_atomic_store(a.counters + wg0, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
        }
        __syncthreads();
        at += parts ? 1 : nblk;
    }
}

// ------------------------------------------------------------ many rows
// A workgroup takes 32 W query vectors of one KV head, 32 per wave in two
// column blocks of 16, and walks the keys 16 W at a time.  Each stage's codes
// become FP16 values once for all the waves: (u - 8) s is exact in FP16 (the
// scale has 8 significant bits), so nothing is rounded that the few-row kernel
// does not round, and the scores and outputs are plain products without a scale
// per group.  The waves write the values to LDS in the order of the matrix
// operands, two stages in turn: stage t + 1 is written while stage t is used, and
// stage t + 2's tiles are on their way to LDS as they are stored.
//
// A column's maximum is raised only when a score exceeds it by 2^PF_SLACK, and
// the outputs are rescaled a few times per row instead of at every new maximum.  The
// weights are 2^PF_LIFT times those of the maximum, below 2^15 (FP16 holds 2^16):
// where one key takes most of the weight, the many small ones keep their bits.  The
// sum of the weights is a product with ones, of the rounded weights that the outputs use.
constexpr int PF_SLACK = 8, PF_LIFT = 7;
//
// More query vectors of a request per KV head than PF_FROM come here.  Its 256
// columns (D = 256: 128) are dear for few vectors and its joining is a second
// launch: 40 vectors at 4096 keys, 8 heads of 128: 14.2 us there, 20.6 here; 8
// requests of 40 at 9000: 62 and 73; 16 of 64 at 2000: 41 and 46.  With more the
// codes are unpacked too often there: 4 requests of 68 at 4096: 33.5 there, 27.5
// here; one of 128 at 32000: 71 and 46 (at 8000 25 and 26, at 2000 13 and 20: the
// rule goes by vectors alone, and a single request of few keys pays for that).
constexpr size_t PF_FROM = 64;

typedef _Float16 h16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ h16x2 as_h2(uint32_t u) { return __builtin_bit_cast(h16x2, u); }
// pairs of codes (bits 0 and 16, or 4 and 20, of w on) times the scales s: as
// 1024 + u, exactly u - 8, times s
__device__ __forceinline__ uint32_t low_values(uint32_t w, h16x2 s) {
    const h16x2 x = as_h2((w & 0x000F000Fu) | 0x64006400u) - (h16x2){(_Float16)1032.0f, (_Float16)1032.0f};
    return __builtin_bit_cast(uint32_t, x * s);
}
__device__ __forceinline__ uint32_t high_values(uint32_t w, h16x2 s) {
    const h16x2 x = __builtin_elementwise_fma(as_h2((w & 0x00F000F0u) | 0x64006400u),
                                              (h16x2){(_Float16)0.0625f, (_Float16)0.0625f},
                                              (h16x2){(_Float16)-72.0f, (_Float16)-72.0f});
    return __builtin_bit_cast(uint32_t, x * s);
}
// a pair of FP16 values, none of them NaN, cut to the largest finite ones
__device__ __forceinline__ uint32_t finite(uint32_t w) {
    const h16x2 top = {(_Float16)65504.0f, (_Float16)65504.0f};
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_elementwise_min(as_h2(w), top), -top));
}

// The line of stages: units (request, block of NV vectors, KV head) in that
// order; 64 (request, block) pairs at a time, one per lane.
template <int NV, int KT>
struct PrefillLine {
    const Kv4AttnArgs& a;
    int lane, nvb, npairs;
    int slot = -1, len = 0, rows = 0;                // of the lane's pair
    uint32_t blocks = 0, cost = 0, upto = 0;         // stages of a unit, of the pair, of the pairs up to it
    uint32_t total = 0, base = 0;                    // base: stages before the pair that find() found
    bool single = false;                             // and each unit is one part
    bool parts = false;                              // the line counts parts of units: each workgroup takes one
    int pair = 0;

    struct Span { int slot, len, rows, main0, sinks, steps; };
    __device__ Span span(int slot, int len, int rows, int vb) const {
        Span s{slot, len, rows, 0, 0, 0};
        const int nv = rows * a.G, v0 = vb * NV;
        if (v0 >= nv) return s;
        const int p0 = len - rows + a.by_g(v0), p1 = len - rows + a.by_g(min(v0 + NV, nv) - 1);
        const int hi = max(0, a.causal ? min(len, p1 + 1) : len);
        const int lo = a.window > 0 && p0 > a.window ? min(p0 - a.window, hi) : 0;
        s.main0 = lo / KT;
        s.sinks = a.window > 0 ? min((min(a.sink, hi) + KT - 1) / KT, s.main0) : 0;
        s.steps = s.sinks + (hi + KT - 1) / KT - s.main0;
        return s;
    }
    __device__ PrefillLine(const Kv4AttnArgs& args, int l)
        : a(args), lane(l), nvb((args.S * args.G + NV - 1) / NV), npairs(args.B * nvb) {}
    __device__ void look(int i0) {
        rows = 0;
        blocks = cost = 0;
        const int i = i0 + lane;
        if (i < npairs) {
            const int b = a.by_nvb(i), vb = i - b * nvb;
            slot = kv4_slot(a.c, a.seqs, b);
            rows = slot < 0 ? 0 : kv4_count(a.counts, b, a.S);
            len = slot < 0 ? 0 : kv4_len(a.c, slot);
            blocks = vb * NV < rows * a.G ? (uint32_t)max(1, span(slot, len, rows, vb).steps) : 0;
            cost = blocks * (uint32_t)a.c.Hkv;
        }
        upto = wave_scan_add(cost);
    }
    // stages of a workgroup's stretch
    __device__ uint32_t stretch(uint32_t workgroups) {
        int longest = 1;
        for (int i0 = 0; i0 < npairs; i0 += 64) {
            look(i0);
            total += lane_u(upto, 63);
            longest = max(longest, __builtin_amdgcn_readlane(wave_scan_max((int)blocks), 63));
        }
        const uint32_t per = max((total + workgroups - 1) / workgroups, ((uint32_t)longest + KV4_PARTS - 2) / (KV4_PARTS - 1));
        // Units cut into whole parts, as in the few-row kernel, where they make no more
        // parts than there are workgroups (333 rows at 3333 keys, 16 / 8 heads of 128:
        // 31 -> 27 us); one part where the longest unit is hardly longer than an equal
        // share, which saves the parts' way through memory (2048 rows at 16384 keys,
        // 32 / 8 heads: 611 -> 591 us with the joining).
        if (npairs <= 64) {
            const uint32_t units = blocks ? (uint32_t)a.c.Hkv : 0;
            const uint32_t pair_cost = cost, pair_upto = upto;
            auto fits = [&](uint32_t q) {
                cost = units * ((blocks + q - 1) / q);
                upto = wave_scan_add(cost);
                if (lane_u(upto, 63) > workgroups) return false;
                parts = true;
                single = q >= (uint32_t)longest;
                total = lane_u(upto, 63);
                return true;
            };
            const uint32_t most = per <= 12 ? per + 2 : per;
            for (uint32_t q = per; q <= most; q++)
                if (fits(q)) return q;
            if ((uint32_t)longest <= per + per / 8 && fits((uint32_t)longest)) return (uint32_t)longest;
            cost = pair_cost;
            upto = pair_upto;
        }
        return per;
    }
    // the lane of the pair that stage `at` of the line belongs to
    __device__ int find(uint32_t at) {
        base = 0;
        for (int i0 = 0; i0 < npairs; i0 += 64) {
            if (npairs > 64) look(i0);
            const unsigned long long over = __ballot(base + upto > at);
            if (over) {
                const int j = __builtin_ctzll(over);
                pair = i0 + j;
                base += lane_u(upto - cost, j);
                return j;
            }
            base += lane_u(upto, 63);
        }
        return 0;   // (not reached: at < total)
    }
};

template <int D, int W>
__global__ void __launch_bounds__(64 * W, W == 8 ? 2 : 1) attn_kv4_prefill_kernel(Kv4AttnArgs a) {
    constexpr int NG = D / 32, NB = D / 16, NT = W, KT = 16 * NT, NV = 32 * W;
    constexpr int NQ = NT / 2;                       // 32-key parts of a stage
    __shared__ __align__(16) uint4 kf[2][NT][NG][64];          // K operands: [tile][group][lane]
    __shared__ __align__(16) uint4 vf[2][NT / 2][NB][64];      // V operands: [32 keys][16 dims][lane]
    constexpr int TB = 18 * D;
    __shared__ __align__(16) uint8_t raw_sh[W][TB];            // a wave's tile of the stage after the next, as it is stored
    __shared__ uint32_t nan_sh[2][KT];               // stage << 8 | value groups of a key that read as NaN
    __shared__ int any_sh[2];                        // the last stage (plus 1) that has such a key
    const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, h = lane >> 4;
    const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Kv4View& c = a.c;
    const float kscale = __builtin_fabsf(a.scale);   // (a negative one turns the sign of q)
    const uint32_t qsign = a.scale < 0.0f ? 0x80008000u : 0u;

    // no marks: here, and behind each unit
    auto clear_marks = [&]() {
        for (int e = tid; e < 2 * KT; e += 64 * W) (&nan_sh[0][0])[e] = 0;
        if (tid < 2) any_sh[tid] = 0;
    };
    clear_marks();
    PrefillLine<NV, KT> line(a, lane);
    const uint32_t per = line.stretch(gridDim.x);
    __syncthreads();
    uint32_t at = line.parts ? blockIdx.x : blockIdx.x * per;
    const uint32_t end = min(line.total, line.parts ? at + 1 : at + per);

    while (at < end) {
        const int j = line.find(at);
        const uint32_t base = line.base, blocks = lane_u(line.blocks, j);
        const int b = a.by_nvb(line.pair), vb = line.pair - b * line.nvb;
        const auto sq = line.span(__builtin_amdgcn_readlane(line.slot, j), __builtin_amdgcn_readlane(line.len, j),
                                  __builtin_amdgcn_readlane(line.rows, j), vb);
        const uint32_t rel = at - base;
        const uint32_t nparts = (blocks + per - 1) / per, span = line.parts ? nparts : blocks;
        const int head = (int)(rel / span);
        const uint32_t first = rel - (uint32_t)head * span, s0 = line.parts ? first * per : first;
        const uint32_t nblk = min(blocks - s0, line.parts ? per : end - at);
        const int nvec = min(NV, sq.rows * a.G - vb * NV);          // of the workgroup
        const int w0 = 32 * wid, wvec = max(0, min(32, nvec - w0)); // of this wave
        const int row0 = sq.len - sq.rows;

        // ---- pages, 64 table entries in the lanes at a time
        int page_first = 0, pages = -1;
        bool have_pages = false;
        auto key_of = [&](int i) { return KT * (i < sq.sinks ? i : sq.main0 + i - sq.sinks); };
        // ---- the wave's tile of a stage (tile `wid`), to LDS
        const uint32_t raw_lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)&raw_sh[wid][0];
        uint32_t there = 0;          // tiles of that stage that have a page, a bit each
        auto fetch = [&](int i) {
            const int key0 = key_of(i), e0 = key0 >> c.ps_log2, e1 = (key0 + KT - 1) >> c.ps_log2;
            if (!have_pages || e0 < page_first || e1 >= page_first + 64) {
                page_first = e0;
                have_pages = true;
                pages = c.table[(size_t)sq.slot * c.max_pages + min(e0 + lane, c.max_pages - 1)];
                __builtin_amdgcn_s_waitcnt(0x0F70);     // vmcnt(0), see the few-row kernel
            }
            const int k0 = key0 + 16 * wid;
            int page = __builtin_amdgcn_readlane(pages, (k0 >> c.ps_log2) - page_first);
            bool ok = kv4_page_ok(c, page);
            if (e0 == e1) {
                there = ok ? (1u << NT) - 1 : 0;
            } else {
                there = 0;
#pragma unroll
                for (int t = 0; t < NT; t++)
                    there |= (uint32_t)kv4_page_ok(c, __builtin_amdgcn_readlane(pages, ((key0 + 16 * t) >> c.ps_log2) - page_first)) << t;
            }
            const uint8_t* p = kv4_tile(c, ok ? page : 0, head, (k0 & ((1 << c.ps_log2) - 1)) >> 4);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");     // the last tile has been read
#pragma unroll
            for (int o = 0; o + 1024 <= TB; o += 1024) lds_dma<16>(p + 16 * lane + o, raw_lds + o);
            if (16 * lane < TB % 1024) lds_dma<16>(p + 16 * lane + TB / 1024 * 1024, raw_lds + TB / 1024 * 1024);
        };
        // Every value operand has to be finite: a weight of 0 times NaN or infinity would
        // reach the rows that do not see the key, and what a page holds behind the last
        // token, in tokens that are not written yet, or in page 0 where it stands in for
        // a missing one, is anything.  A NaN or infinite scale of a value group: the key
        // is marked and the group reads as 0.  A scale from 8192 on, whose product with a
        // code may be beyond FP16: the result says so, and the products are cut to
        // 65504 (those of written tokens stay below, 7 x 9344).
        auto mark = [&](int i, uint32_t (&vscl)[D / 16]) -> bool {
            uint32_t bad = 0;        // an exponent field from 28 on carries into bits 15 and 31
#pragma unroll
            for (int k = 0; k < D / 16; k++) bad |= (vscl[k] & 0x7C007C00u) + 0x10001000u;
            const bool large = __ballot((bad & 0x80008000u) != 0) != 0;
            if (__builtin_expect(large, 0)) {
                uint32_t groups[4] = {0, 0, 0, 0};
#pragma unroll
                for (int k = 0; k < D / 16; k++)
#pragma unroll
                    for (int half = 0; half < 2; half++) {
                        if ((vscl[k] >> 16 * half & 0x7C00u) != 0x7C00u) continue;
                        vscl[k] &= half ? 0xFFFFu : 0xFFFF0000u;
                        groups[2 * (k & 1) + half] |= 1u << (k >> 1);
                    }
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int key = 16 * wid + 4 * h + r;
                    if (groups[r] && key_of(i) + key < sq.len && (there >> wid & 1)) {
                        nan_sh[i & 1][key] = (uint32_t)i << 8 | groups[r];
                        any_sh[i & 1] = i + 1;
                    }
                }
            }
            return large;
        };
        // stage i's tile, once it has arrived, to the operands of buffer `buf`
        auto put = [&](int i, int buf) {
            wait_dma<0>();
            const uint8_t* raw = &raw_sh[wid][0];
            {
                uint32_t x[D / 32];
                load_words(x, raw + lane * (D / 8));
#pragma unroll
                for (int p = 0; p < NG / 2; p++) {
                    // scales of key `col`
                    const uint16_t* s = reinterpret_cast<const uint16_t*>(raw + 8 * D) + ((col >> 2) * NG + 2 * p) * 4 + (col & 3);
                    const h16x2 sl = as_h2(s[0] | (uint32_t)s[0] << 16), sh = as_h2(s[4] | (uint32_t)s[4] << 16);
                    const uint32_t x0 = x[2 * p], x1 = x[2 * p + 1];
                    kf[buf][wid][2 * p][lane] = make_uint4(low_values(x0, sl), low_values(x0 >> 8, sl), low_values(x1, sl),
                                                           low_values(x1 >> 8, sl));
                    kf[buf][wid][2 * p + 1][lane] = make_uint4(high_values(x0, sh), high_values(x0 >> 8, sh),
                                                               high_values(x1, sh), high_values(x1 >> 8, sh));
                }
            }
            uint32_t x[D / 32], vscl[D / 16];        // scales of keys 4 h + i
            load_words(x, raw + 9 * D + lane * (D / 8));
            load_words(vscl, raw + 17 * D + h * (D / 4));
            const bool large = mark(i, vscl);
#pragma unroll
            for (int g = 0; g < NG; g++) {
                const uint32_t s01 = vscl[2 * g], s23 = vscl[2 * g + 1], w = x[g];
                const h16x2 se = as_h2(__builtin_amdgcn_perm(s23, s01, 0x05040100u));    // keys 4 h, 4 h + 2
                const h16x2 so = as_h2(__builtin_amdgcn_perm(s23, s01, 0x07060302u));    // keys 4 h + 1, 4 h + 3
                reinterpret_cast<uint2*>(&vf[buf][wid >> 1][2 * g][lane])[wid & 1] =
                    make_uint2(low_values(w, se), low_values(w >> 8, so));
                reinterpret_cast<uint2*>(&vf[buf][wid >> 1][2 * g + 1][lane])[wid & 1] =
                    make_uint2(high_values(w, se), high_values(w >> 8, so));
            }
            if (__builtin_expect(large, 0)) {
#pragma unroll 1
                for (int n = 0; n < NB; n++) {
                    uint2* at = reinterpret_cast<uint2*>(&vf[buf][wid >> 1][n][lane]) + (wid & 1);
                    const uint2 x = *at;
                    *at = make_uint2(finite(x.x), finite(x.y));
                }
            }
        };

        // ---- this wave's vectors: lane's column in two blocks of 16
        // (their loads go ahead of the first tile's, which wait for its page number)
        uint4 qraw[2][NG];
        int pos[2];
#pragma unroll
        for (int cb = 0; cb < 2; cb++) {
            const int vec = vb * NV + w0 + 16 * cb + col, row = a.by_g(vec);
            pos[cb] = row0 + row;
#pragma unroll
            for (int g = 0; g < NG; g++) {
                uint4 u = make_uint4(0, 0, 0, 0);
                if (16 * cb + col < wvec)
                    u = *reinterpret_cast<const uint4*>(a.q + ((size_t)b * a.S + row) * a.q_stride +
                                                        (size_t)(head * a.G + vec - row * a.G) * D + 32 * g + 8 * h);
                qraw[cb][g] = u;
            }
        }
        const int i0 = (int)s0, i1 = min(sq.steps, (int)(s0 + nblk));
        if (i0 < i1) fetch(i0);
        h16x8 qf[2][NG];
#pragma unroll
        for (int cb = 0; cb < 2; cb++)
#pragma unroll
            for (int g = 0; g < NG; g++) {
                const uint4 u = qraw[cb][g];
                qf[cb][g] = code_order(make_uint4(u.x ^ qsign, u.y ^ qsign, u.z ^ qsign, u.w ^ qsign));
            }
        const int first_pos = row0 + a.by_g(vb * NV + w0);
        const int last_pos = row0 + a.by_g(vb * NV + w0 + max(wvec, 1) - 1);
        const int all = a.causal ? min(first_pos + 1, sq.len) : sq.len;      // keys that each of them sees (but for a window)

        float m[2], mbase[2];
        f32x4 acc[2][NB], lsum[2];
#pragma unroll
        for (int cb = 0; cb < 2; cb++) {
            m[cb] = -__builtin_inff();
            mbase[cb] = 0.0f;
            lsum[cb] = (f32x4){0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < NB; i++) acc[cb][i] = (f32x4){0, 0, 0, 0};
        }
        u32x4 one4 = {0x3C003C00u, 0x3C003C00u, 0x3C003C00u, 0x3C003C00u};
        asm volatile("" : "+v"(one4));               // in registers: not made anew at each stage
        const h16x8 ones = __builtin_bit_cast(h16x8, one4);

        // ---- a stage: its 32-key parts in turn, the next part's scores beside this
        // one's powers of two, then this part's outputs.  Operands are read from LDS a
        // group of products ahead; the barriers and groups keep the compiler from
        // moving them together.
        constexpr int VG = 4, NVG = NB / VG;
        auto stage = [&](int i, int buf, uint32_t there) {
            const int key0 = key_of(i);
            const bool active = wvec > 0 && (!a.causal || key0 <= last_pos);
            if (!active) return;
            f32x4 st[2][2][2];                        // [part parity][column block][tile]
            h16x8 pf[2], ka[NG], kb[NG], va[VG], vb2[VG];
            auto read_k = [&](int t, h16x8 (&to)[NG]) {
#pragma unroll
                for (int g = 0; g < NG; g++) to[g] = __builtin_bit_cast(h16x8, kf[buf][t][g][lane]);
            };
            auto read_v = [&](int q, int n, h16x8 (&to)[VG]) {
#pragma unroll
                for (int u = 0; u < VG; u++) to[u] = __builtin_bit_cast(h16x8, vf[buf][q][n * VG + u][lane]);
            };
            auto scores = [&](int q, int t, const h16x8 (&k)[NG]) {
#pragma unroll
                for (int g = 0; g < NG; g++)
#pragma unroll
                    for (int cb = 0; cb < 2; cb++)
                        st[q & 1][cb][t] = mfma16(k[g], qf[cb][g], g ? st[q & 1][cb][t] : (f32x4){0, 0, 0, 0});
            };
            // part q's scores: masked where not every vector sees every key, and the maxima
            auto check = [&](int q) {
                const int k0 = key0 + 32 * q;
                f32x4 (&s)[2][2] = st[q & 1];
                const bool whole = (there >> 2 * q & 3u) == 3u && k0 + 32 <= all &&
                                   (a.window == 0 || last_pos - k0 <= a.window || k0 + 32 <= a.sink);
                if (!whole) {
                    // a column sees keys below its upper limit and, under a window, from its
                    // lower one on or below the sink (computed here: held over the
                    // stages, the limits' registers spilled the accumulators)
                    int k4 = k0 + 4 * h;
                    asm volatile("" : "+v"(k4));
#pragma unroll
                    for (int cb = 0; cb < 2; cb++) {
                        const int hi = (a.causal ? min(pos[cb] + 1, sq.len) : sq.len) - k4;
                        const int lo = a.window > 0 ? pos[cb] - a.window - k4 : -64, sink = a.sink - k4;
#pragma unroll
                        for (int t = 0; t < 2; t++)
#pragma unroll
                            for (int r = 0; r < 4; r++) {
                                const int k = 16 * t + r;
                                s[cb][t][r] = (there >> (2 * q + t) & 1) & (k < hi) & ((k >= lo) | (k < sink)) ? s[cb][t][r] : -__builtin_inff();
                            }
                    }
                }
                float top[2];
#pragma unroll
                for (int cb = 0; cb < 2; cb++)
                    top[cb] = kscale * max3(max3(s[cb][0][0], s[cb][0][1], s[cb][0][2]), max3(s[cb][0][3], s[cb][1][0], s[cb][1][1]),
                                            __builtin_fmaxf(s[cb][1][2], s[cb][1][3]));
                if (__ballot((top[0] > m[0] + PF_SLACK) | (top[1] > m[1] + PF_SLACK))) {
#pragma unroll
                    for (int cb = 0; cb < 2; cb++) {
                        float y = top[cb];
                        y = __builtin_fmaxf(y, __shfl_xor(y, 16, 64));
                        y = __builtin_fmaxf(y, __shfl_xor(y, 32, 64));
                        const float mn = __builtin_fmaxf(m[cb], y), base = mn > -__builtin_inff() ? mn - PF_LIFT : 0.0f;
                        const float f = m[cb] > -__builtin_inff() ? exp2_fast(mbase[cb] - base) : 0.0f;
                        mbase[cb] = base;
                        m[cb] = mn;
                        lsum[cb] *= f;
#pragma unroll
                        for (int n = 0; n < NB; n++) acc[cb][n] *= f;
                    }
                }
            };
            auto weights = [&](int q) {
#pragma unroll
                for (int cb = 0; cb < 2; cb++) {
                    float p[2][4];
#pragma unroll
                    for (int t = 0; t < 2; t++)
#pragma unroll
                        for (int r = 0; r < 4; r++) p[t][r] = exp2_fast(__builtin_fmaf(st[q & 1][cb][t][r], kscale, -mbase[cb]));
                    pf[cb] = frag(pack_h(p[0][0], p[0][2]), pack_h(p[0][1], p[0][3]), pack_h(p[1][0], p[1][2]),
                                  pack_h(p[1][1], p[1][3]));
                }
            };
            auto values = [&](int n, const h16x8 (&v)[VG]) {
#pragma unroll
                for (int u = 0; u < VG; u++)
#pragma unroll
                    for (int cb = 0; cb < 2; cb++) acc[cb][n * VG + u] = mfma16(v[u], pf[cb], acc[cb][n * VG + u]);
            };
            read_k(0, ka);
            read_k(1, kb);
            __builtin_amdgcn_sched_barrier(0);
            scores(0, 0, ka);
            scores(0, 1, kb);
            if (NQ > 1) read_k(2, ka);
            __builtin_amdgcn_sched_barrier(0);
            check(0);
#pragma unroll
            for (int q = 0; q < NQ; q++) {
                // A: scores of part q + 1, weights of part q
                if (q + 1 < NQ) read_k(2 * q + 3, kb);
                __builtin_amdgcn_sched_barrier(0);
                if (q + 1 < NQ) scores(q + 1, 0, ka);
                weights(q);
                if (q + 1 < NQ) scores(q + 1, 1, kb);
                read_v(q, 0, va);
                if (q + 1 < NQ) {
#pragma unroll
                    for (int n = 0; n < 4 * NG; n++) {
                        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
                        __builtin_amdgcn_sched_group_barrier(0x402, (40 + 4 * NG - 1) / (4 * NG), 0);
                    }
                    __builtin_amdgcn_sched_group_barrier(0x100, VG, 0);
                }
                __builtin_amdgcn_sched_barrier(0);
                // B: outputs of part q
#pragma unroll
                for (int n = 0; n < NVG; n++) {
                    h16x8 (&cur)[VG] = n & 1 ? vb2 : va;
                    h16x8 (&nxt)[VG] = n & 1 ? va : vb2;
                    if (n + 1 < NVG) read_v(q, n + 1, nxt);
                    else if (q + 2 < NQ) read_k(2 * q + 4, ka);
                    __builtin_amdgcn_sched_barrier(0);
                    values(n, cur);
                    if (n + 1 == NVG) {
#pragma unroll
                        for (int cb = 0; cb < 2; cb++) lsum[cb] = mfma16(ones, pf[cb], lsum[cb]);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
                __builtin_amdgcn_sched_barrier(0);
                if (q + 1 < NQ) check(q + 1);
            }
            if (__builtin_expect(any_sh[buf] == i + 1, 0)) {
                for (int key = 0; key < KT; key++) {
                    const uint32_t w = nan_sh[buf][key];
                    if (w >> 8 != ((uint32_t)i & 0xFFFFFFu) || !(w & 0xFFu)) continue;
#pragma unroll
                    for (int cb = 0; cb < 2; cb++) {
                        const bool sees = kv4_sees(a, pos[cb], key0 + key, sq.len);
#pragma unroll
                        for (int n = 0; n < NB; n++)
                            if (sees && (w >> (n >> 1) & 1))
                                acc[cb][n] = (f32x4){__builtin_nanf(""), __builtin_nanf(""), __builtin_nanf(""), __builtin_nanf("")};
                    }
                }
            }
        };

        // ---- the stages
        // Iteration i writes stage i + 1's operands and uses stage i's (from i0 - 1 on:
        // one copy of the code).  Two waves share a SIMD's units: the first four prepare
        // the next stage before their products, the others after theirs, so that one
        // wave's vector instructions run beside the other's matrix ones.  (With four
        // waves, heads of 256, there is no other: 2048 rows by 16384 keys, 32 / 8
        // heads, at 592 TFLOP/s where heads of 128 reach 981.)
        uint32_t now = 0;
#pragma unroll 1
        for (int i = i0 - 1; i < i1; i++) {
            const uint32_t next = there;
            auto prepare = [&]() {
                if (i + 1 < i1) {
                    put(i + 1, (i + 1) & 1);
                    if (i + 2 < i1) fetch(i + 2);
                }
            };
            if (wid < 4) prepare();
            if (i >= i0) stage(i, i & 1, now);
            if (wid >= 4) prepare();
            now = next;
            __syncthreads();
        }

        clear_marks();

        // ---- outputs, or this workgroup's part of them
        const bool alone = nblk == blocks;
        const uint32_t unit0 = base + (uint32_t)head * blocks;
        const uint32_t wg0 = line.parts ? blockIdx.x - first : unit0 / per;    // the unit's first workgroup has it in slot 1
        auto out_row = [&](int v) {
            const int vv = vb * NV + v;
            return a.o + ((size_t)b * a.S * a.Hq + out_offset(a, head, vv)) * D;
        };
        auto write4 = [&](uint16_t* p, f32x4 num, float inv) {
            uint16_t r[4];
#pragma unroll
            for (int k = 0; k < 4; k++) r[k] = f2h(num[k] * inv);
            *reinterpret_cast<uint2*>(p) = make_uint2(r[0] | (uint32_t)r[1] << 16, r[2] | (uint32_t)r[3] << 16);
        };
#pragma unroll
        for (int cb = 0; cb < 2; cb++) {
            const int v = w0 + 16 * cb + col;
            if (v >= nvec) continue;
            if (alone) {
                uint16_t* o = out_row(v);
                const float inv = lsum[cb][0] != 0.0f ? 1.0f / lsum[cb][0] : 0.0f;
#pragma unroll
                for (int n = 0; n < NB; n++) write4(o + 16 * n + 4 * h, acc[cb][n], inv);
            } else {
                float* row_at = a.part + ((size_t)(2 * blockIdx.x + (blockIdx.x == wg0)) * NV + v) * (D + 4);
#pragma unroll
                for (int n = 0; n < NB; n++) *reinterpret_cast<f32x4*>(row_at + 16 * n + 4 * h) = acc[cb][n];
                if (h == 0)
                    *reinterpret_cast<float2*>(row_at + D) = make_float2(m[cb] > -__builtin_inff() ? mbase[cb] : m[cb], lsum[cb][0]);
            }
        }
        __syncthreads();
        at += line.parts ? 1 : nblk;
    }
}

// The joining of units that several workgroups shared, a quad of dims per thread,
// eight parts' loads at a time: o = sum_p 2^(m_p - m) o_p / sum_p 2^(m_p - m) l_p.  A
// launch of its own: the last workgroup of a unit, joining 256 vectors' parts
// alone, took longer than the products of a few hundred rows.  Bound by the
// latency of the lengths, then of the parts (333 rows, 16 / 8 heads of 128: 7.7
// us; 40 vectors in 32 parts 7.0, with a part after the other 12.9).  1024
// workgroups: with one for each share, 2048 rows whose units are one part each take 10.5
// us to find that there is nothing to join, 4.8 so.
template <int D>
constexpr int pj_vec() { return 1024 / D; }       // vectors of a workgroup's share
constexpr size_t PJ_WORKGROUPS = 1024;
template <int D, int W>
__global__ void __launch_bounds__(256) attn_kv4_join_kernel(Kv4AttnArgs a, uint32_t workgroups) {
    constexpr int NV = 32 * W, KT = 16 * W, VEC = pj_vec<D>(), NVJ = NV / VEC;
    const int tid = threadIdx.x, lane = tid & 63;
    PrefillLine<NV, KT> line(a, lane);
    const uint32_t per = line.stretch(workgroups);
    if (line.single) return;
    // A workgroup takes shares in turn, a unit's vectors VEC at a time.  With many
    // requests, whose lengths do not stay in the lanes, it looks for units from the main launch's
    // workgroups instead (a unit that is shared is the last of its first
    // workgroup's stretch), and takes eight times the vectors (64 requests of 600
    // vectors 112 -> 20 us; with few units these would meet in few workgroups: 100
    // rows at 4096 keys 8 -> 37).
    const bool from_units = line.npairs <= 64;
    const int steps = from_units ? 1 : 8;
    const uint32_t per_unit = NVJ / steps, shares = (from_units ? (uint32_t)(line.npairs * a.c.Hkv) : workgroups) * per_unit;
    for (uint32_t w = blockIdx.x; w < shares; w += gridDim.x) {
        const uint32_t of = w / per_unit;                        // which unit, or workgroup
        const int v0 = (int)(w - of * per_unit) * steps * VEC;
        int j, head;
        if (from_units) {
            j = (int)of / a.c.Hkv;
            head = (int)of - j * a.c.Hkv;
            line.pair = j;
            line.base = lane_u(line.upto - line.cost, j);
        } else {
            if (of * per >= line.total) return;
            const uint32_t end = min(line.total, (of + 1) * per);
            j = line.find(end - 1);
            head = (int)((end - 1 - line.base) / lane_u(line.blocks, j));
        }
        const uint32_t blocks = lane_u(line.blocks, j), span = line.parts ? (blocks + per - 1) / per : blocks;
        if (blocks == 0) continue;
        const uint32_t unit0 = line.base + (uint32_t)head * span, wg0 = line.parts ? unit0 : unit0 / per;
        const uint32_t nparts = line.parts ? span : (unit0 + span - 1) / per - wg0 + 1;
        if (nparts == 1 || (!from_units && wg0 != of)) continue;
        const int b = a.by_nvb(line.pair), vb = line.pair - b * line.nvb;
        const int nvec = min(NV, __builtin_amdgcn_readlane(line.rows, j) * a.G - vb * NV);
        for (int v = v0 + tid / (D / 4); v < min(v0 + steps * VEC, nvec); v += VEC) {
            const int d = tid % (D / 4) * 4;
            f32x4 num = {0, 0, 0, 0};
            float mx = -__builtin_inff(), den = 0.0f;
            for (int p0 = 0; p0 < (int)nparts; p0 += 8) {
                f32x4 y[8];
                float2 ml[8];
#pragma unroll
                for (int u = 0; u < 8; u++) {
                    y[u] = (f32x4){0, 0, 0, 0};
                    ml[u] = make_float2(-__builtin_inff(), 0.0f);
                    if (p0 + u < (int)nparts) {
                        const float* row_at = a.part + ((size_t)(2 * (wg0 + p0 + u) + (p0 + u == 0)) * NV + v) * (D + 4);
                        y[u] = *reinterpret_cast<const f32x4*>(row_at + d);
                        ml[u] = *reinterpret_cast<const float2*>(row_at + D);
                    }
                }
                float mn = mx;
#pragma unroll
                for (int u = 0; u < 8; u++) mn = __builtin_fmaxf(mn, ml[u].x);
                const float f0 = mx > -__builtin_inff() ? exp2_fast(mx - mn) : 1.0f;
                mx = mn;
                num *= f0;
                den *= f0;
#pragma unroll
                for (int u = 0; u < 8; u++) {
                    const float f = ml[u].x > -__builtin_inff() ? exp2_fast(ml[u].x - mx) : 1.0f;
#pragma unroll
                    for (int k = 0; k < 4; k++) num[k] = __builtin_fmaf(f, y[u][k], num[k]);
                    den = __builtin_fmaf(f, ml[u].y, den);
                }
            }
            const int vv = vb * NV + v;
            const float inv = den != 0.0f ? 1.0f / den : 0.0f;
            uint16_t r[4];
#pragma unroll
            for (int k = 0; k < 4; k++) r[k] = f2h(num[k] * inv);
            *reinterpret_cast<uint2*>(a.o + ((size_t)b * a.S * a.Hq + out_offset(a, head, vv)) * D + d) =
                make_uint2(r[0] | (uint32_t)r[1] << 16, r[2] | (uint32_t)r[3] << 16);
        }
    }
}

}  // namespace cactus_hip

using namespace cactus_hip;

extern "C" {

size_t cactus_hip_attention_kv4_workspace(const cactus_hip_kv4_cache* cache, size_t batch, size_t seq_len,
                                          size_t num_q_heads) {
    if (kv4_view(cache, 0, "attention_kv4_workspace", nullptr)) return 0;
    const size_t vectors = seq_len * (num_q_heads / cache->kv_heads);
    const size_t few = (size_t)512 * 2 * 16;                  // (packed: 1024 workgroups of 8 vectors at most)
    const size_t many = (size_t)256 * 2 * (cache->head_dim == 256 ? 128 : 256);
    (void)batch;
    return KV4_COUNTERS + (vectors > PF_FROM ? many : few) * (cache->head_dim + 4) * 4;
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
    a.by_g.set((uint32_t)G);
    a.window = (int)std::min(window_size, top);
    a.sink = (int)std::min(sink_size, top);
    a.causal = is_causal != 0;
    a.scale = (scale == 0.0f ? 1.0f / sqrtf((float)cache->head_dim) : scale) * LOG2E_F;
    a.counters = static_cast<uint32_t*>(workspace);
    a.part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + KV4_COUNTERS);
    const hipStream_t st = as_stream(stream);
    const size_t vectors = seq_len * G;
    auto launch = [&](auto kernel, int per_unit, int keys, int per_cu, int waves, unsigned* workgroups) {
        const size_t units = batch * cache->kv_heads * ceil_div(vectors, per_unit);
        // block steps of a unit at most, by what the tables can hold
        const size_t blocks = ceil_div(cache->max_pages * cache->page_size, keys);
        // the line counts steps, and requests times blocks of vectors, in 32 bits
        if (units >= (1u << 30) / blocks)
            return fail(CACTUS_HIP_EUNSUPPORTED, "attention_kv4: batch times rows times table length is too large");
        *workgroups = (unsigned)std::min<size_t>(256 * per_cu, units * blocks);
        hipLaunchKernelGGL(kernel, dim3(*workgroups), dim3(64 * waves), 0, st, a);
        return (int)CACTUS_HIP_OK;
    };
    auto many = [&](auto kernel, auto join, int waves) {
        unsigned workgroups = 0;
        a.by_nvb.set((uint32_t)ceil_div(vectors, 32 * waves));
        const int r = launch(kernel, 32 * waves, 16 * waves, 1, waves, &workgroups);
        if (r) return r;
        const size_t shares = batch * cache->kv_heads * ceil_div(vectors, 32 * waves) * (32 * waves * cache->head_dim / 1024);
        hipLaunchKernelGGL(join, dim3((unsigned)std::min(shares, PJ_WORKGROUPS)), dim3(256), 0, st, a, workgroups);
        return (int)CACTUS_HIP_OK;
    };
    unsigned n = 0;
    const int quads = (int)std::min<size_t>(vectors, 16) * a.c.d / 4;     // (of up to 8 vectors: the packed kernel's)
    const int shares = a.c.d == 64 ? kv4_shares<64, true>(quads) : a.c.d == 128 ? kv4_shares<128, true>(quads) : kv4_shares<256, true>(quads);
    a.join_log2 = 31 - __builtin_clz(8 * shares);
#define KV4_FEW(D, PACK)                                                                                  \
    launch(attn_kv4_kernel<D, PACK>, kv4_vectors<D, PACK>(), KV4_STEP * kv4_waves<D, PACK>(), kv4_per_cu<D, PACK>(), \
           kv4_waves<D, PACK>(), &n)
#define KV4_LAUNCH(D, W)                                                              \
    (vectors <= (size_t)kv4_vectors<D, true>() ? KV4_FEW(D, true)                     \
     : vectors <= PF_FROM                      ? KV4_FEW(D, false)                    \
                                               : many(attn_kv4_prefill_kernel<D, W>, attn_kv4_join_kernel<D, W>, W))
    rc = a.c.d == 64 ? KV4_LAUNCH(64, 8) : a.c.d == 128 ? KV4_LAUNCH(128, 8) : KV4_LAUNCH(256, 4);
#undef KV4_LAUNCH
#undef KV4_FEW
    if (rc) return rc;
    return check_launch("attention_kv4");
}

}  // extern "C"
