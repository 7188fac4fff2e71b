// logits.hip -- penalties for repeated tokens, biases and grammar masks on the
// logits of many sequences, and each one's best token.
//
// Bound by memory without lists (256 rows of 151936 FP16 logits 51 us, 4.6 TB/s); with histories of up
// to 8192 tokens, biases and masks 64 us, 3.7 TB/s: the counting, three barriers and the penalties'
// divisions, beyond what other workgroups' memory traffic covers.  32 rows with histories of up to
// 2000, 40 biases and grammars 12.1 us (9.5 without the best token, whose three trips to the
// workspace end the call), one row with 300 tokens 6.1 us.  The logits and the result go past the
// caches: 67 -> 64 us for 256 rows, 13.4 -> 12.1 for 32.  256 FP32 rows 65 us without lists
// (4.8 TB/s) and 73 with them.
#include "hip_common.h"

namespace cactus_hip {

struct RulesArgs {
    cactus_hip_logits_rules r;
    const int32_t* seqs;
    const void* in;
    float* out;
    uint32_t* best;
    uint32_t* work;           // [rows][4]: best key (64 bits), workgroups done, 0
    size_t in_stride, out_stride;
    int V;
};

// Larger for a larger value, and for equal values (0 and -0 are) for the lower index; 0
// for NaN and -infinity.
__device__ __forceinline__ uint64_t best_key(float x, uint32_t i) {
    if (!(x > -__builtin_inff())) return 0;
    const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);
    return (uint64_t)(b >> 31 ? ~b : b | 0x80000000u) << 32 | (0xFFFFFFFFu - i);
}
__device__ __forceinline__ void load_words(uint32_t (&n)[8], const uint32_t* p) {
    const uint4 u = reinterpret_cast<const uint4*>(p)[0], v = reinterpret_cast<const uint4*>(p)[1];
    n[0] = u.x, n[1] = u.y, n[2] = u.z, n[3] = u.w, n[4] = v.x, n[5] = v.y, n[6] = v.z, n[7] = v.w;
}
__device__ __forceinline__ float penalized(float x, int n, float rep, float freq, float pres) {
    x = x > 0.0f ? x / rep : x * rep;
    const float f = freq * (float)n;
    return (x - f) - pres;
}

// A workgroup takes 16 tokens per thread of a row, in groups of 8 that start
// where 16-byte loads of the row may (tokens before and behind the row are passed over).
// The logits are on their way while it counts, in LDS, how often the history names each of
// its tokens: every workgroup of a row reads the whole history, which the L2 holds, and
// keeps what falls among its own.  Bias entries then count themselves into the same words:
// a token that one entry names (most are) is that entry's thread's; of several the first
// takes them all, in order.
// 512 threads for every call: 256 rows with lists 67 us (256 threads 77, 1024 69; all before the loads
// and stores went past the caches), one row with a history 6.2 (6.3 and 7.1).
constexpr int RULES_THREADS = 512, RULES_MAX_BIAS = CACTUS_HIP_LOGITS_MAX_BIAS;
constexpr uint32_t COUNT_BITS = 20;      // of the history; above it the entries, bit 31: value in b_out
template <typename T>
__global__ void __launch_bounds__(RULES_THREADS) logits_rules_kernel(RulesArgs a) {
    constexpr int THREADS = RULES_THREADS, GROUPS = 2, CHUNK = 8 * GROUPS * THREADS, EPT = RULES_MAX_BIAS / THREADS, EARLY = 4;
    __shared__ __attribute__((aligned(16))) uint32_t counts[CHUNK];
    __shared__ float b_out[RULES_MAX_BIAS];
    __shared__ uint64_t w_key[THREADS / 64];
    const int tid = threadIdx.x, row = blockIdx.y;
    const int slot = a.seqs ? a.seqs[row] : row;
    if ((unsigned)slot >= (unsigned)a.r.max_seqs) return;
    const T* in = static_cast<const T*>(a.in) + (size_t)row * a.in_stride;
    float* out = a.out + (size_t)row * a.out_stride;
    // tokens before the first one that starts 16 bytes of the row, and whether it does so in out too
    const int shift = (int)(-(uintptr_t)in & 15) / (int)sizeof(T);
    const bool vec = ((uintptr_t)(out + shift) & 15) == 0;
    const int c0 = (shift ? shift - 8 : 0) + (int)blockIdx.x * CHUNK;      // (down to -7)
    const int lo = max(c0, 0), hi = max(lo, min(c0 + CHUNK, a.V));

    float x[GROUPS][8];
#pragma unroll
    for (int g = 0; g < GROUPS; g++) {
        const int t = c0 + 8 * (tid + THREADS * g);
        if (vec && t >= 0 && t + 8 <= a.V) {
            if constexpr (sizeof(T) == 2) {
                const i32x4 w = __builtin_nontemporal_load(reinterpret_cast<const i32x4*>(in + t));
#pragma unroll
                for (int j = 0; j < 8; j++) x[g][j] = h2f((uint16_t)((uint32_t)w[j / 2] >> 16 * (j & 1)));
            } else {
                const f32x4 u = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(in + t)), v = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(in + t + 4));
#pragma unroll
                for (int j = 0; j < 4; j++) x[g][j] = u[j], x[g][4 + j] = v[j];
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                x[g][j] = 0.0f;
                if (t + j >= 0 && t + j < a.V) {
                    if constexpr (sizeof(T) == 2) x[g][j] = h2f(in[t + j]);
                    else x[g][j] = in[t + j];
                }
            }
        }
    }
    // The lists' first entries are on their way before it is known how many count: a list's length
    // and then its entries, one after the other, cost more than the entries that go unused.
    const int32_t* h = a.r.history + (size_t)slot * a.r.history_stride;
    const int32_t* tokens = a.r.bias_tokens + (size_t)slot * a.r.bias_stride;
    const float* values = a.r.bias_values + (size_t)slot * a.r.bias_stride;
    int ht[EARLY], bt[EPT];
    float bv[EPT], bx[EPT];
    const int room = a.r.history ? (int)a.r.history_stride : 0, broom = a.r.bias_tokens ? (int)a.r.bias_stride : 0;
#pragma unroll
    for (int u = 0; u < EARLY; u++) ht[u] = tid + THREADS * u < room ? h[tid + THREADS * u] : -1;
#pragma unroll
    for (int e = 0; e < EPT; e++) {
        bt[e] = tid + THREADS * e < broom ? tokens[tid + THREADS * e] : -1;
        bv[e] = tid + THREADS * e < broom ? values[tid + THREADS * e] : 0.0f;
    }
    const int hist = a.r.history_lens && room ? min(max(a.r.history_lens[slot], 0), room) : room;
    const int nb = a.r.bias_counts && broom ? min(max(a.r.bias_counts[slot], 0), broom) : broom;
    const float rep = a.r.repetition ? a.r.repetition[slot] : 1.0f, freq = a.r.frequency ? a.r.frequency[slot] : 0.0f,
                pres = a.r.presence ? a.r.presence[slot] : 0.0f;
    uint32_t bits[GROUPS];                    // bit i of group g: its token i is allowed
#pragma unroll
    for (int g = 0; g < GROUPS; g++) bits[g] = 0xFFu;
    if (a.r.masks) {
        const int id = a.r.mask_ids ? a.r.mask_ids[slot] : slot;
        if (id >= 0) {
            const bool none = (size_t)id >= a.r.num_masks;
            const uint32_t* mask = a.r.masks + (none ? 0 : (size_t)id * a.r.mask_stride);
#pragma unroll
            for (int g = 0; g < GROUPS; g++) {
                const int t = c0 + 8 * (tid + THREADS * g), t0 = min(max(t, 0), a.V - 1), t1 = min(max(t + 7, 0), a.V - 1);
                const uint64_t w = none ? 0 : (uint64_t)mask[t0 >> 5] | (uint64_t)mask[t1 >> 5] << 32;
                bits[g] = t < 0 ? (uint32_t)w << -t : t0 >> 5 == t1 >> 5 ? (uint32_t)w >> (t0 & 31) : (uint32_t)(w >> (t0 & 31));
            }
        }
    }
    const bool listed = hist > 0 || nb > 0;
    if (listed) {
#pragma unroll
        for (int i = 0; i < CHUNK / 4 / THREADS; i++) reinterpret_cast<uint4*>(counts)[tid + THREADS * i] = make_uint4(0, 0, 0, 0);
        __syncthreads();
#pragma unroll
        for (int u = 0; u < EARLY; u++)
            if (tid + THREADS * u < hist && (uint32_t)ht[u] - (uint32_t)lo < (uint32_t)(hi - lo)) atomicAdd(&counts[ht[u] - c0], 1u);
        for (int i0 = EARLY * THREADS; i0 < hist; i0 += 8 * THREADS) {
            int t[8];
#pragma unroll
            for (int u = 0; u < 8; u++) t[u] = i0 + tid + THREADS * u < hist ? h[i0 + tid + THREADS * u] : -1;
#pragma unroll
            for (int u = 0; u < 8; u++)
                if ((uint32_t)t[u] - (uint32_t)lo < (uint32_t)(hi - lo)) atomicAdd(&counts[t[u] - c0], 1u);
        }
        if (nb > 0) {
#pragma unroll
            for (int e = 0; e < EPT; e++) {
                if (tid + THREADS * e >= nb || bt[e] < lo || bt[e] >= hi) {
                    bt[e] = -1;
                    continue;
                }
                atomicAdd(&counts[bt[e] - c0], 1u << COUNT_BITS);
                if constexpr (sizeof(T) == 2) bx[e] = h2f(in[bt[e]]);
                else bx[e] = in[bt[e]];
            }
        }
        __syncthreads();
        if (nb > 0) {
#pragma unroll
            for (int e = 0; e < EPT; e++) {
                const int i = tid + THREADS * e, t = bt[e];
                if (t < 0) continue;
                const uint32_t w = counts[t - c0], n = w & ((1u << COUNT_BITS) - 1);
                bool own = !(w >> 31);            // (else the token's first entry has been here)
                const bool single = w >> COUNT_BITS == 1;
                if (!single)
                    for (int j = 0; j < i && own; j++) own = tokens[j] != t;
                if (!own) continue;
                float v = bx[e];
                if (n) v = penalized(v, (int)n, rep, freq, pres);
                v = v + bv[e];
                if (!single)
                    for (int j = i + 1; j < nb; j++)
                        if (tokens[j] == t) v = v + values[j];
                b_out[i] = v;
                counts[t - c0] = 0x80000000u + i;
            }
            __syncthreads();
        }
    }
    float most = -__builtin_inff();
    int at = 0;
#pragma unroll
    for (int g = 0; g < GROUPS; g++) {
        const int l = 8 * (tid + THREADS * g), t = c0 + l;
        if (t >= a.V || t + 8 <= 0) continue;
        if (listed) {
            uint32_t n[8];
            load_words(n, counts + l);
            if (n[0] | n[1] | n[2] | n[3] | n[4] | n[5] | n[6] | n[7]) {
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    if (n[j] >> 31) x[g][j] = b_out[n[j] & 0x7FFFFFFFu];
                    else if (n[j]) x[g][j] = penalized(x[g][j], (int)n[j], rep, freq, pres);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < 8; j++) x[g][j] = bits[g] >> j & 1 ? x[g][j] : -__builtin_inff();
        if (vec && t >= 0 && t + 8 <= a.V) {
            __builtin_nontemporal_store((f32x4){x[g][0], x[g][1], x[g][2], x[g][3]}, reinterpret_cast<f32x4*>(out + t));
            __builtin_nontemporal_store((f32x4){x[g][4], x[g][5], x[g][6], x[g][7]}, reinterpret_cast<f32x4*>(out + t + 4));
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (x[g][j] > most) most = x[g][j], at = t + j;
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                if (t + j < 0 || t + j >= a.V) continue;
                out[t + j] = x[g][j];
                if (x[g][j] > most) most = x[g][j], at = t + j;
            }
        }
    }
    if (!a.best) return;
    uint64_t key = best_key(most, (uint32_t)at);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const uint64_t k = __shfl_xor((unsigned long long)key, o, 64);
        key = k > key ? k : key;
    }
    if ((tid & 63) == 0) w_key[tid >> 6] = key;
    __syncthreads();
    if (tid != 0) return;
#pragma unroll
    for (int w = 1; w < THREADS / 64; w++) key = w_key[w] > key ? w_key[w] : key;
    // The row's largest key in the workspace; whoever comes last takes it and leaves zeros.  The
    // maximum is performed where the counter is, and has been when the counter is raised.
    uint64_t* best = reinterpret_cast<uint64_t*>(a.work + 4 * (size_t)row);
    uint32_t* done = a.work + 4 * (size_t)row + 2;
    (void)__hip_atomic_fetch_max(best, key, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (__hip_atomic_fetch_add(done, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1 < gridDim.x) return;
    key = __hip_atomic_exchange(best, (uint64_t)0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __hip_atomic_store(done, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    a.best[row] = key ? 0xFFFFFFFFu - (uint32_t)key : 0u;
}

template <typename T>
static void rules_launch(const RulesArgs& a, size_t batch, hipStream_t st) {
    const dim3 grid(ceil_div((size_t)a.V + 7, 16 * RULES_THREADS), (unsigned)batch);      // (a row's groups may start up to 7 before it)
    hipLaunchKernelGGL(logits_rules_kernel<T>, grid, dim3(RULES_THREADS), 0, st, a);
}

static int rules(const cactus_hip_logits_rules* r, const int32_t* seqs, const void* logits, size_t stride, float* out,
                 size_t out_stride, uint32_t* best, size_t batch, size_t vocab, void* workspace, size_t workspace_bytes,
                 void* stream, bool half) {
    CH_REQUIRE(r, "logits_rules: null rules");
    CH_REQUIRE(r->max_seqs >= 1 && r->max_seqs < (1u << 30), "logits_rules: max_seqs out of range");
    CH_REQUIRE(r->history_stride < (1u << COUNT_BITS) && r->bias_stride <= CACTUS_HIP_LOGITS_MAX_BIAS,
               "logits_rules: history_stride or bias_stride out of range");
    CH_REQUIRE(!r->bias_tokens || r->bias_values, "logits_rules: biases without values");
    CH_REQUIRE(!r->masks || r->mask_stride >= (vocab + 31) / 32, "logits_rules: mask_stride is shorter than a mask");
    CH_REQUIRE(!r->masks || r->mask_ids || r->num_masks >= r->max_seqs, "logits_rules: a mask for each slot, or mask_ids");
    CH_REQUIRE(batch <= 65535, "logits_rules: more than 65535 rows");
    CH_REQUIRE(vocab < (1u << 28), "logits_rules: vocab out of range");
    if (batch == 0 || vocab == 0) return CACTUS_HIP_OK;
    CH_REQUIRE(logits && out, "logits_rules: null pointer");
    CH_REQUIRE(stride >= vocab && out_stride >= vocab, "logits_rules: a stride is shorter than a row");
    CH_REQUIRE(((uintptr_t)logits & (half ? 1 : 3)) == 0 && ((uintptr_t)out & 3) == 0, "logits_rules: misaligned logits");
    CH_REQUIRE((const void*)out != logits || (!half && stride == out_stride), "logits_rules: in place are FP32 rows of one stride");
    CH_REQUIRE(!best || (workspace && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= 16 * batch),
               "logits_rules: workspace too small or not 16-byte aligned");
    RulesArgs a{*r, seqs, logits, out, best, static_cast<uint32_t*>(workspace), stride, out_stride, (int)vocab};
    if (half) rules_launch<uint16_t>(a, batch, as_stream(stream));
    else rules_launch<float>(a, batch, as_stream(stream));
    return check_launch("logits_rules");
}

}  // namespace cactus_hip

using namespace cactus_hip;

extern "C" {

size_t cactus_hip_logits_rules_workspace(size_t batch) { return 16 * batch; }

int cactus_hip_logits_rules_f16(const cactus_hip_logits_rules* rules_, const int32_t* seqs, const uint16_t* logits,
                                size_t stride, float* out, size_t out_stride, uint32_t* best, size_t batch, size_t vocab,
                                void* workspace, size_t workspace_bytes, void* stream) {
    return rules(rules_, seqs, logits, stride, out, out_stride, best, batch, vocab, workspace, workspace_bytes, stream, true);
}

int cactus_hip_logits_rules_f32(const cactus_hip_logits_rules* rules_, const int32_t* seqs, const float* logits,
                                size_t stride, float* out, size_t out_stride, uint32_t* best, size_t batch, size_t vocab,
                                void* workspace, size_t workspace_bytes, void* stream) {
    return rules(rules_, seqs, logits, stride, out, out_stride, best, batch, vocab, workspace, workspace_bytes, stream, false);
}

}  // extern "C"
