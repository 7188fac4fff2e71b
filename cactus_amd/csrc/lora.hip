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
    int adapters, r, S, K, N;
};

// A workgroup per row: the waves take the rank's products in turn, then a thread per output.
constexpr int LORA_MAX_RANK = 256;
__global__ void __launch_bounds__(256) lora_row_kernel(LoraArgs a) {
    __shared__ float h[LORA_MAX_RANK];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = blockIdx.x, req = blockIdx.y;
    const int m = a.counts ? a.counts[req] : a.S;
    if (row >= min(m, a.S)) return;
    const int id = a.ids[req];
    const bool has = (unsigned)id < (unsigned)a.adapters;
    const size_t at = (size_t)req * a.S + row;
    const uint16_t *x = a.x + at * a.x_stride, *base = a.base + at * a.base_stride;
    uint16_t* y = a.y + at * a.y_stride;
    if (!has) {
        if (y != base)
            for (int n = threadIdx.x; n < a.N; n += 256) y[n] = base[n];
        return;
    }
    for (int j = wave; j < a.r; j += 4) {
        const uint16_t* A = a.A + ((size_t)id * a.r + j) * a.K;
        float s = 0;
        for (int k = lane; k < a.K; k += 64) s = __builtin_fmaf(h2f(A[k]), h2f(x[k]), s);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
        if (lane == 0) h[j] = s;
    }
    __syncthreads();
    const float scale = a.scales ? a.scales[id] : 1.0f;
    for (int n = threadIdx.x; n < a.N; n += 256) {
        const uint16_t* B = a.B + ((size_t)id * a.N + n) * a.r;
        float s = 0;
        for (int j = 0; j < a.r; j++) s = __builtin_fmaf(h2f(B[j]), h[j], s);
        y[n] = f2h(__builtin_fmaf(s, scale, h2f(base[n])));
    }
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
               (int)rank, (int)seq_len, (int)K, (int)N};
    hipLaunchKernelGGL(lora_row_kernel, dim3((unsigned)seq_len, (unsigned)batch), dim3(256), 0, as_stream(stream), a);
    return check_launch("lora_add");
}
