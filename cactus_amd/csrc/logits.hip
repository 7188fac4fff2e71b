// logits.hip -- penalties for repeated tokens, biases and grammar masks on the
// logits of many sequences, and each one's best token.
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
__device__ __forceinline__ float penalized(float x, int n, float rep, float freq, float pres) {
    x = x > 0.0f ? x / rep : x * rep;
    const float f = freq * (float)n;
    return (x - f) - pres;
}

// A workgroup takes RULES_CHUNK tokens of a row.  It counts the history's tokens that
// fall among them in LDS, then the biases' owners: the first entry that names a token
// takes the whole chain of its entries, in order.
constexpr int RULES_CHUNK = 4096, RULES_THREADS = 256, RULES_MAX_BIAS = CACTUS_HIP_LOGITS_MAX_BIAS;
template <typename T>
__global__ void __launch_bounds__(RULES_THREADS) logits_rules_kernel(RulesArgs a) {
    // per token: occurrences; 2^31 + entry where a bias list's entry holds the value
    __shared__ uint32_t counts[RULES_CHUNK];
    __shared__ int b_tok[RULES_MAX_BIAS];
    __shared__ float b_val[RULES_MAX_BIAS], b_out[RULES_MAX_BIAS];
    __shared__ uint64_t w_key[RULES_THREADS / 64];
    const int tid = threadIdx.x, row = blockIdx.y, c0 = (int)blockIdx.x * RULES_CHUNK, c1 = min(c0 + RULES_CHUNK, a.V);
    const int slot = a.seqs ? a.seqs[row] : row;
    if ((unsigned)slot >= (unsigned)a.r.max_seqs) return;
    const T* in = static_cast<const T*>(a.in) + (size_t)row * a.in_stride;
    float* out = a.out + (size_t)row * a.out_stride;
    const auto load = [&](int t) -> float {
        if constexpr (sizeof(T) == 2) return h2f(in[t]);
        else return in[t];
    };
    const int hist = a.r.history ? (a.r.history_lens ? min(max(a.r.history_lens[slot], 0), (int)a.r.history_stride) : (int)a.r.history_stride) : 0;
    const int nb = a.r.bias_tokens ? (a.r.bias_counts ? min(max(a.r.bias_counts[slot], 0), (int)a.r.bias_stride) : (int)a.r.bias_stride) : 0;
    const float rep = a.r.repetition ? a.r.repetition[slot] : 1.0f, freq = a.r.frequency ? a.r.frequency[slot] : 0.0f,
                pres = a.r.presence ? a.r.presence[slot] : 0.0f;
    const uint32_t* mask = nullptr;
    bool none = false;
    if (a.r.masks) {
        const int id = a.r.mask_ids ? a.r.mask_ids[slot] : slot;
        if (id >= 0) {
            none = (size_t)id >= a.r.num_masks;
            mask = none ? nullptr : a.r.masks + (size_t)id * a.r.mask_stride;
        }
    }
    for (int i = tid; i < RULES_CHUNK; i += RULES_THREADS) counts[i] = 0;
    __syncthreads();
    for (int i = tid; i < hist; i += RULES_THREADS) {
        const int t = a.r.history[(size_t)slot * a.r.history_stride + i];
        if (t >= c0 && t < c1) atomicAdd(&counts[t - c0], 1u);
    }
    for (int i = tid; i < nb; i += RULES_THREADS) {
        b_tok[i] = a.r.bias_tokens[(size_t)slot * a.r.bias_stride + i];
        b_val[i] = a.r.bias_values[(size_t)slot * a.r.bias_stride + i];
    }
    __syncthreads();
    for (int i = tid; i < nb; i += RULES_THREADS) {
        const int t = b_tok[i];
        if (t < c0 || t >= c1) continue;
        bool first = true;
        for (int j = 0; j < i; j++) first = first && b_tok[j] != t;
        if (!first) continue;
        float x = load(t);
        const uint32_t n = counts[t - c0];
        if (n) x = penalized(x, (int)n, rep, freq, pres);
        for (int j = i; j < nb; j++)
            if (b_tok[j] == t) x = x + b_val[j];
        b_out[i] = x;
        counts[t - c0] = 0x80000000u + i;
    }
    __syncthreads();
    uint64_t key = 0;
    for (int t = c0 + tid; t < c1; t += RULES_THREADS) {
        const uint32_t n = counts[t - c0];
        float x;
        if (n >> 31) x = b_out[n & 0x7FFFFFFFu];
        else {
            x = load(t);
            if (n) x = penalized(x, (int)n, rep, freq, pres);
        }
        if (none || (mask && !(mask[t >> 5] >> (t & 31) & 1u))) x = -__builtin_inff();
        out[t] = x;
        const uint64_t k = best_key(x, (uint32_t)t);
        key = k > key ? k : key;
    }
    if (!a.best) return;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const uint64_t k = __shfl_xor((unsigned long long)key, o, 64);
        key = k > key ? k : key;
    }
    if ((tid & 63) == 0) w_key[tid >> 6] = key;
    __syncthreads();
    if (tid != 0) return;
    for (int w = 1; w < RULES_THREADS / 64; w++) key = w_key[w] > key ? w_key[w] : key;
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

static int rules(const cactus_hip_logits_rules* r, const int32_t* seqs, const void* logits, size_t stride, float* out,
                 size_t out_stride, uint32_t* best, size_t batch, size_t vocab, void* workspace, size_t workspace_bytes,
                 void* stream, bool half) {
    CH_REQUIRE(r, "logits_rules: null rules");
    CH_REQUIRE(r->max_seqs >= 1 && r->max_seqs < (1u << 30), "logits_rules: max_seqs out of range");
    CH_REQUIRE(r->history_stride < (1u << 31) && r->bias_stride <= CACTUS_HIP_LOGITS_MAX_BIAS,
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
    const dim3 grid(ceil_div(vocab, RULES_CHUNK), (unsigned)batch);
    if (half) hipLaunchKernelGGL(logits_rules_kernel<uint16_t>, grid, dim3(RULES_THREADS), 0, as_stream(stream), a);
    else hipLaunchKernelGGL(logits_rules_kernel<float>, grid, dim3(RULES_THREADS), 0, as_stream(stream), a);
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
