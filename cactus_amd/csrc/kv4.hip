// kv4.hip -- the paged 4-bit KV cache: quantizing new rows into pages,
// reading them back, and the bookkeeping of pages (extend, fork, free,
// compact, copy) on the device.
#include "kv4_device.h"

#include <algorithm>

namespace cactus_hip {

typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));

// ------------------------------------------------------------ append
// Scale of a 32-dim group from the largest magnitude: a / 7 rounded to 8
// significant bits (bf16) and then to fp16, which only rounds again where the
// scale is an fp16 subnormal.  NaN for a group with a NaN or an infinity.
__device__ __forceinline__ uint16_t kv4_scale(float amax, bool bad) {
    const float q = amax / 7.0f;
    uint32_t b = __builtin_bit_cast(uint32_t, q);
    b = (b + 0x7FFFu + ((b >> 16) & 1u)) & 0xFFFF0000u;   // finite: to nearest, ties to even
    return bad ? (uint16_t)0x7E00u : f2h(bits_f(b));
}
// code + 8 of x under scale s
__device__ __forceinline__ uint32_t kv4_code(float x, float s) {
    const float c = __builtin_rintf(x / s);
    const float t = __builtin_fminf(__builtin_fmaxf(c, -7.0f), 7.0f);
    return (s > 0.0f) ? (uint32_t)((int)t + 8) : 8u;   // s NaN or 0: code 0
}

// One wave per (request, KV head, 16-key tile): lane 16 h + key takes dims 8 h
// to 8 h + 7 of each 32-dim group of its key, which are the K codes of the
// lane of that number in the page; a group's maximum meets over the four
// lanes of the key.
template <int D>
__global__ void __launch_bounds__(64) kv4_append_kernel(Kv4View c, const int32_t* seqs, const int32_t* counts,
                                                        const uint16_t* k, const uint16_t* v, int seq_len, size_t stride) {
    constexpr int NG = D / 32;
    const int lane = threadIdx.x, key = lane & 15, h = lane >> 4;
    const int head = blockIdx.y, req = blockIdx.z;
    if (c.state[KV4_STATUS] != 0) return;
    const int slot = kv4_slot(c, seqs, req);
    if (slot < 0) return;
    const int len = kv4_len(c, slot), first = len - kv4_count(counts, req, seq_len);   // (negative: rows without a token)
    const int lo = max(first, 0);
    const int pos0 = (lo & ~15) + 16 * (int)blockIdx.x;      // first position of this wave's tile
    if (pos0 >= len) return;
    const int page = c.table[(size_t)slot * c.max_pages + (pos0 >> c.ps_log2)];
    if (!kv4_page_ok(c, page)) return;
    uint8_t* tile = kv4_tile(c, page, head, (pos0 & ((1 << c.ps_log2) - 1)) >> 4);
    const int pos = pos0 + key;
    const bool mine = pos >= lo && pos < len;
    const size_t row = ((size_t)req * seq_len + (mine ? pos - first : 0)) * stride + (size_t)head * D;
    uint8_t codes[NG][8];
#pragma unroll
    for (int kv = 0; kv < 2; kv++) {
        const uint16_t* src = (kv ? v : k) + row;
        uint8_t* out = tile + kv * 9 * D;
        uint16_t* scales = reinterpret_cast<uint16_t*>(out + 8 * D);
#pragma unroll
        for (int g = 0; g < NG; g++) {
            const h16x8 x = *reinterpret_cast<const h16x8*>(src + 32 * g + 8 * h);
            float amax = 0.0f;
            int bad = 0;
#pragma unroll
            for (int t = 0; t < 8; t++) {
                const float a = __builtin_fabsf((float)x[t]);
                bad |= !(a <= 65504.0f);
                amax = __builtin_fmaxf(amax, a);
            }
            amax = __builtin_fmaxf(amax, __shfl_xor(amax, 16, 64));
            amax = __builtin_fmaxf(amax, __shfl_xor(amax, 32, 64));
            bad |= __shfl_xor(bad, 16, 64);
            bad |= __shfl_xor(bad, 32, 64);
            const uint16_t sb = kv4_scale(amax, bad != 0);
            const float s = h2f(sb);
#pragma unroll
            for (int t = 0; t < 8; t++) codes[g][t] = (uint8_t)kv4_code((float)x[t], s);
            if (mine && h == (g & 3)) scales[((key >> 2) * NG + g) * 4 + (key & 3)] = sb;
        }
        if (kv == 0) {
            // byte 8 p + t: groups 2 p and 2 p + 1
#pragma unroll
            for (int p = 0; p < NG / 2; p++) {
                uint64_t w = 0;
#pragma unroll
                for (int t = 0; t < 8; t++)
                    w |= (uint64_t)(codes[2 * p][t] | codes[2 * p + 1][t] << 4) << (8 * t);
                if (mine) *reinterpret_cast<uint64_t*>(out + lane * (D / 8) + 8 * p) = w;
            }
        } else {
            // lane h < 2 holds dims x = 8 h + t of each group, its partner h + 2 dims x + 16
#pragma unroll
            for (int g = 0; g < NG; g++)
#pragma unroll
                for (int t = 0; t < 8; t++) {
                    const int hi = __shfl_xor((int)codes[g][t], 32, 64);
                    if (mine && h < 2)
                        out[(key >> 2) * 2 * D + (8 * h + t) * (D / 8) + 4 * g + (key & 3)] =
                            (uint8_t)(codes[g][t] | hi << 4);
                }
        }
    }
}

// ------------------------------------------------------------ read
// One wave per (request, KV head, 16-key tile), lane = 16 h + key as above.
// code * scale is an exact fp16 value.
template <int D>
__global__ void __launch_bounds__(64) kv4_read_kernel(Kv4View c, const int32_t* seqs, const int32_t* starts,
                                                      const int32_t* counts, uint16_t* k, uint16_t* v, int seq_len) {
    constexpr int NG = D / 32;
    const int lane = threadIdx.x, key = lane & 15, h = lane >> 4;
    const int head = blockIdx.y, req = blockIdx.z;
    const int slot = kv4_slot(c, seqs, req);
    if (slot < 0) return;
    const int len = kv4_len(c, slot), m = kv4_count(counts, req, seq_len);
    const int first = starts ? starts[req] : len - m;   // may lie outside the slot's tokens
    const int64_t end64 = (int64_t)first + m;
    const int end = end64 < len ? (int)end64 : len;
    const int lo = max(first, 0);
    const int pos0 = (lo & ~15) + 16 * (int)blockIdx.x;
    if (pos0 >= end) return;
    const int page = c.table[(size_t)slot * c.max_pages + (pos0 >> c.ps_log2)];
    if (!kv4_page_ok(c, page)) return;
    const uint8_t* tile = kv4_tile(c, page, head, (pos0 & ((1 << c.ps_log2) - 1)) >> 4);
    const int pos = pos0 + key;
    if (pos < lo || pos >= end) return;
    const size_t row = (((size_t)req * seq_len + (size_t)(pos - first)) * c.Hkv + head) * D;
#pragma unroll
    for (int kv = 0; kv < 2; kv++) {
        uint16_t* dst = kv ? v : k;
        if (!dst) continue;
        const uint8_t* in = tile + kv * 9 * D;
        const uint16_t* scales = reinterpret_cast<const uint16_t*>(in + 8 * D);
#pragma unroll
        for (int g = 0; g < NG; g++) {
            const float s = h2f(scales[((key >> 2) * NG + g) * 4 + (key & 3)]);
            h16x8 y;
#pragma unroll
            for (int t = 0; t < 8; t++) {
                // dim 32 g + 8 h + t
                const int x = 8 * (h & 1) + t;
                const int byte = kv == 0 ? in[lane * (D / 8) + 8 * (g >> 1) + t]
                                         : in[(key >> 2) * 2 * D + x * (D / 8) + 4 * g + (key & 3)];
                const int up = kv == 0 ? (g & 1) : (h >> 1);
                y[t] = (_Float16)((float)(((byte >> (4 * up)) & 15) - 8) * s);
            }
            *reinterpret_cast<h16x8*>(dst + row + 32 * g + 8 * h) = y;
        }
    }
}

// ------------------------------------------------------------ bookkeeping
constexpr int BK_THREADS = 1024;      // the one workgroup that allocates
constexpr int BK_IDS = 8192;          // free pages collected at a time

__global__ void kv4_reset_kernel(Kv4View c) {
    const size_t i0 = (size_t)blockIdx.x * blockDim.x + threadIdx.x, step = (size_t)gridDim.x * blockDim.x;
    for (size_t i = i0; i < (size_t)c.max_seqs * c.max_pages; i += step) c.table[i] = -1;
    for (size_t i = i0; i < (size_t)c.max_seqs; i += step) c.lens[i] = 0;
    for (size_t i = i0; i < (size_t)c.num_pages; i += step) c.refs[i] = 0;
    if (i0 == 0) {
        c.state[KV4_FREE] = c.num_pages;
        c.state[KV4_HINT] = 0;
        c.state[KV4_STATUS] = 0;
        c.state[3] = 0;
    }
}
__global__ void kv4_clear_status_kernel(int32_t* state) { state[KV4_STATUS] = 0; }

// exclusive prefix sum of v over the workgroup's threads; *total: the sum
__device__ __forceinline__ int block_scan(int v, int* wave_sums, int* total) {
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, waves = blockDim.x >> 6;
    int incl = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(incl, o, 64);
        if (lane >= o) incl += u;
    }
    __syncthreads();                      // the sums of an earlier call are read
    if (lane == 63) wave_sums[wid] = incl;
    __syncthreads();
    int before = 0, all = 0;
    for (int w = 0; w < waves; w++) {
        if (w < wid) before += wave_sums[w];
        all += wave_sums[w];
    }
    *total = all;
    return before + incl - v;
}

// Collects free pages, ascending from *at on, until `want` or BK_IDS of them
// are in ids; returns how many, *at: where to go on.  Whole workgroup.
__device__ int collect_free(const Kv4View& c, int* at, int want, int* ids, int* wave_sums) {
    int have = 0, pos = *at;
    want = min(want, BK_IDS);
    while (have < want && pos < c.num_pages) {
        const int i = pos + (int)threadIdx.x * 4;
        int z = 0;
#pragma unroll
        for (int u = 0; u < 4; u++) z |= (i + u < c.num_pages && c.refs[i + u] == 0) << u;
        int got;
        int rank = have + block_scan(__popc(z), wave_sums, &got);
#pragma unroll
        for (int u = 0; u < 4; u++)
            if (z >> u & 1) {
                if (rank < want) ids[rank] = i + u;
                rank++;
            }
        __syncthreads();
        if (have + got > want) {
            pos = ids[want - 1] + 1;      // the rest is taken up from here
            have = want;
        } else {
            have += got;
            pos += BK_THREADS * 4;
        }
    }
    *at = min(pos, c.num_pages);
    __syncthreads();
    return have;
}

__device__ __forceinline__ bool mark_twice(uint32_t* bits, int slot) {
    return (atomicOr(&bits[slot >> 5], 1u << (slot & 31)) >> (slot & 31)) & 1u;
}

__global__ void __launch_bounds__(BK_THREADS) kv4_extend_kernel(Kv4View c, const int32_t* seqs, const int32_t* counts,
                                                                int batch, int count) {
    __shared__ uint32_t bits[KV4_MAX_SEQS / 32];
    __shared__ int ids[BK_IDS], off[BK_THREADS], wave_sums[16];
    __shared__ int bad, total_s;
    const int tid = threadIdx.x, cap = c.max_pages << c.ps_log2;
    for (int i = tid; i < (c.max_seqs + 31) / 32; i += BK_THREADS) bits[i] = 0;
    if (tid == 0) {
        bad = 0;
        total_s = 0;
    }
    __syncthreads();
    // every request is right, and how many pages they need together (at most
    // max_seqs * max_pages, which the host bounds)
    for (int i = tid; i < batch; i += BK_THREADS) {
        const int s = kv4_slot(c, seqs, i), n = counts ? counts[i] : count;
        if (s < 0 || n < 0 || mark_twice(bits, s)) {
            bad = 1;
            continue;
        }
        const int len = kv4_len(c, s);
        if (n > cap - len) {
            bad = 1;
            continue;
        }
        const int need = kv4_pages_of(c, len + n) - kv4_pages_of(c, len);
        if (need) atomicAdd(&total_s, need);
    }
    __syncthreads();
    const int total = total_s;
    if (bad || total > c.state[KV4_FREE]) {
        if (tid == 0) atomicOr((uint32_t*)c.state + KV4_STATUS, bad ? CACTUS_HIP_KV4_BAD_REQUEST : CACTUS_HIP_KV4_NO_PAGES);
        return;
    }
    // free pages in rounds of BK_IDS, each handed to the requests whose share
    // of the sequence of new pages falls into the round
    int at = c.state[KV4_HINT], done = 0;
    at = at < 0 ? 0 : at;
    while (done < total) {
        const int got = collect_free(c, &at, total - done, ids, wave_sums);
        if (got == 0) {                    // the free count was wrong: no page is handed out twice
            if (tid == 0) atomicOr((uint32_t*)c.state + KV4_STATUS, CACTUS_HIP_KV4_NO_PAGES);
            break;
        }
        int base = 0;
        for (int i0 = 0; i0 < batch; i0 += BK_THREADS) {
            const int i = i0 + tid;
            int need = 0;
            if (i < batch) {
                const int s = kv4_slot(c, seqs, i), n = counts ? counts[i] : count, len = kv4_len(c, s);
                need = kv4_pages_of(c, len + n) - kv4_pages_of(c, len);
            }
            int chunk;
            const int o = block_scan(need, wave_sums, &chunk);
            off[tid] = base + o;
            __syncthreads();
            // a wave per request
            for (int r = tid >> 6; r < min(BK_THREADS, batch - i0); r += BK_THREADS / 64) {
                const int s = kv4_slot(c, seqs, i0 + r), n = counts ? counts[i0 + r] : count, len = kv4_len(c, s);
                const int p0 = kv4_pages_of(c, len), np = kv4_pages_of(c, len + n) - p0;
                for (int j = max(0, done - off[r]) + (tid & 63); j < min(np, done + got - off[r]); j += 64) {
                    const int id = ids[off[r] + j - done];
                    c.table[(size_t)s * c.max_pages + p0 + j] = id;
                    c.refs[id] = 1;
                }
            }
            base += chunk;
            __syncthreads();
        }
        done += got;
    }
    __syncthreads();
    if (done < total) return;
    for (int i = tid; i < batch; i += BK_THREADS) c.lens[kv4_slot(c, seqs, i)] += counts ? counts[i] : count;
    if (tid == 0 && total > 0) {
        c.state[KV4_FREE] -= total;
        c.state[KV4_HINT] = at;
    }
}

// Lists of a fork in the workspace, behind the attention's counters.
struct ForkPlan {
    int32_t* ok;         // [1]
    int32_t* tail;       // [n] new page of the partly filled last one, -1
    int32_t* len;        // [n] the source's tokens before the call
    int32_t* rows;       // [n][max_pages] the source's pages before the call
};
constexpr size_t KV4_WORK_SKIP = 4096;

// Requests checked and the copies' pages allocated, before anything changes
// that a wrong call would have to undo.
__global__ void __launch_bounds__(BK_THREADS) kv4_fork_plan_kernel(Kv4View c, ForkPlan p, const int32_t* src,
                                                                   const int32_t* dst, int n) {
    __shared__ uint32_t bits[KV4_MAX_SEQS / 32];
    __shared__ int ids[BK_IDS], wave_sums[16];
    __shared__ int bad, total_s;
    const int tid = threadIdx.x, ps1 = (1 << c.ps_log2) - 1;
    for (int i = tid; i < (c.max_seqs + 31) / 32; i += BK_THREADS) bits[i] = 0;
    if (tid == 0) {
        bad = 0;
        total_s = 0;
    }
    __syncthreads();
    for (int i = tid; i < n; i += BK_THREADS) {
        const int s = kv4_slot(c, src, i), d = kv4_slot(c, dst, i);
        if (s < 0 || d < 0 || mark_twice(bits, d)) {
            bad = 1;
            continue;
        }
        if (s != d && (kv4_len(c, s) & ps1)) atomicAdd(&total_s, 1);
    }
    __syncthreads();
    const int total = total_s;
    if (bad || total > c.state[KV4_FREE]) {
        if (tid == 0) {
            atomicOr((uint32_t*)c.state + KV4_STATUS, bad ? CACTUS_HIP_KV4_BAD_REQUEST : CACTUS_HIP_KV4_NO_PAGES);
            *p.ok = 0;
        }
        return;
    }
    // at most max_seqs pages: dst slots differ
    int at = c.state[KV4_HINT], done = 0;
    at = at < 0 ? 0 : at;
    do {
        const int got = done < total ? collect_free(c, &at, total - done, ids, wave_sums) : 0;
        if (got == 0 && done < total) {
            if (tid == 0) {
                atomicOr((uint32_t*)c.state + KV4_STATUS, CACTUS_HIP_KV4_NO_PAGES);
                *p.ok = 0;
            }
            return;
        }
        int base = 0;
        for (int i0 = 0; i0 < n; i0 += BK_THREADS) {
            const int i = i0 + tid;
            bool part = false;
            if (i < n) {
                const int s = kv4_slot(c, src, i);
                part = s != kv4_slot(c, dst, i) && (kv4_len(c, s) & ps1);
            }
            int chunk;
            const int o = base + block_scan(part, wave_sums, &chunk) - done;
            if (i < n) {
                if (!part) p.tail[i] = -1;
                else if (o >= 0 && o < got) p.tail[i] = ids[o];
            }
            base += chunk;
        }
        done += got;
        __syncthreads();
    } while (done < total);
    if (tid == 0) {
        *p.ok = 1;
        if (total > 0) {
            c.state[KV4_FREE] -= total;
            c.state[KV4_HINT] = at;
        }
    }
}
// the sources' rows and lengths set aside, their full pages' counts raised
__global__ void kv4_fork_share_kernel(Kv4View c, ForkPlan p, const int32_t* src, const int32_t* dst) {
    if (!*p.ok) return;
    const int i = blockIdx.x, s = kv4_slot(c, src, i);
    if (s == kv4_slot(c, dst, i)) return;
    const int len = kv4_len(c, s), full = len >> c.ps_log2, np = kv4_pages_of(c, len);
    if (threadIdx.x == 0) {
        p.len[i] = len;
        if (p.tail[i] >= 0) c.refs[p.tail[i]] = 1;
    }
    for (int j = threadIdx.x; j < np; j += blockDim.x) {
        const int id = c.table[(size_t)s * c.max_pages + j];
        p.rows[(size_t)i * c.max_pages + j] = id;
        if (j < full && kv4_page_ok(c, id)) atomicAdd(&c.refs[id], 1);
    }
}
// a slot's pages given up (its row as it stands)
__device__ __forceinline__ void release_row(const Kv4View& c, int slot, int len) {
    const int np = kv4_pages_of(c, len);
    for (int j = threadIdx.x; j < np; j += blockDim.x) {
        const int id = c.table[(size_t)slot * c.max_pages + j];
        if (kv4_page_ok(c, id) && atomicSub(&c.refs[id], 1) == 1) {
            atomicAdd(&c.state[KV4_FREE], 1);
            atomicMin(&c.state[KV4_HINT], id);
        }
    }
}
__device__ __forceinline__ void copy_bytes16(uint8_t* dst, const uint8_t* src, size_t bytes, size_t first, size_t step) {
    for (size_t o = first * 16; o < bytes; o += step * 16)
        *reinterpret_cast<uint4*>(dst + o) = *reinterpret_cast<const uint4*>(src + o);
}
// block y 0: the destination's table row; blocks from 1 on: the last page, a layer each
__global__ void kv4_fork_apply_kernel(Kv4View c, ForkPlan p, const int32_t* src, const int32_t* dst) {
    if (!*p.ok) return;
    const int i = blockIdx.x, d = kv4_slot(c, dst, i);
    if (kv4_slot(c, src, i) == d) return;
    const int32_t* row = p.rows + (size_t)i * c.max_pages;
    const int len = p.len[i], full = len >> c.ps_log2, tail = p.tail[i];
    if (blockIdx.y > 0) {
        if (tail < 0 || !kv4_page_ok(c, row[full])) return;
        const size_t layer = (size_t)(blockIdx.y - 1) * c.layer_bytes;
        copy_bytes16(c.pages + layer + (size_t)tail * c.page_bytes, c.pages + layer + (size_t)row[full] * c.page_bytes,
                     c.page_bytes, threadIdx.x, blockDim.x);
        return;
    }
    release_row(c, d, kv4_len(c, d));
    __syncthreads();
    for (int j = threadIdx.x; j < c.max_pages; j += blockDim.x)
        c.table[(size_t)d * c.max_pages + j] = j < full ? row[j] : (j == full && tail >= 0 ? tail : -1);
    if (threadIdx.x == 0) c.lens[d] = len;
}

__global__ void kv4_free_kernel(Kv4View c, const int32_t* seqs) {
    __shared__ int len_s;
    const int s = kv4_slot(c, seqs, blockIdx.x);
    if (s < 0) {
        if (threadIdx.x == 0) atomicOr((uint32_t*)c.state + KV4_STATUS, CACTUS_HIP_KV4_BAD_REQUEST);
        return;
    }
    // of several requests for a slot, one finds its tokens
    if (threadIdx.x == 0) len_s = atomicExch(&c.lens[s], 0);
    __syncthreads();
    const int cap = c.max_pages << c.ps_log2, len = min(len_s, cap);
    if (len <= 0) return;
    release_row(c, s, len);
    __syncthreads();
    for (int j = threadIdx.x; j < c.max_pages; j += blockDim.x) c.table[(size_t)s * c.max_pages + j] = -1;
}

// ------------------------------------------------------------ compact
constexpr int CP_THREADS = 256, CP_PER = 16, CP_BLOCK = CP_THREADS * CP_PER;   // pages per workgroup
struct CompactPlan {
    int32_t* moves;      // [1]
    int32_t* live;       // [1] pages in use
    int32_t* used;       // [blocks] pages in use among a workgroup's
    int32_t* rank;       // [num_pages] of a page that moves: which of them it is
    int32_t* from;       // [num_pages] pages that move, ascending
    int32_t* to;         // [num_pages] free pages below `live`, ascending
};
__global__ void __launch_bounds__(CP_THREADS) kv4_compact_count_kernel(Kv4View c, CompactPlan p) {
    __shared__ int sums[4];
    int n = 0;
    for (int u = 0; u < CP_PER; u++) {
        const int i = blockIdx.x * CP_BLOCK + u * CP_THREADS + threadIdx.x;
        n += i < c.num_pages && c.refs[i] > 0;
    }
    int total;
    block_scan(n, sums, &total);
    if (threadIdx.x == 0) p.used[blockIdx.x] = total;
}
__global__ void __launch_bounds__(CP_THREADS) kv4_compact_list_kernel(Kv4View c, CompactPlan p) {
    __shared__ int sums[4];
    const int tid = threadIdx.x, blocks = gridDim.x, me = blockIdx.x;
    int before_me = 0, all = 0, t;
    for (int b0 = 0; b0 < blocks; b0 += CP_THREADS) {
        const int b = b0 + tid, v = b < blocks ? p.used[b] : 0;
        block_scan(b < me ? v : 0, sums, &t);
        before_me += t;
        block_scan(v, sums, &t);
        all += t;
    }
    const int live = all;
    // pages in use below `live`
    const int edge = live / CP_BLOCK;
    int below = 0;
    for (int b0 = 0; b0 < edge; b0 += CP_THREADS) {
        block_scan(b0 + tid < edge ? p.used[b0 + tid] : 0, sums, &t);
        below += t;
    }
    int n = 0;
    for (int u = 0; u < CP_PER; u++) {
        const int i = edge * CP_BLOCK + u * CP_THREADS + tid;
        n += i < live && c.refs[i] > 0;
    }
    block_scan(n, sums, &t);
    below += t;
    // this workgroup's pages, CP_PER consecutive ones per thread
    const int i0 = me * CP_BLOCK + tid * CP_PER;
    uint32_t in_use = 0;
    for (int u = 0; u < CP_PER; u++) in_use |= (uint32_t)(i0 + u < c.num_pages && c.refs[i0 + u] > 0) << u;
    int r = before_me + block_scan(__popc(in_use), sums, &t);   // pages in use before page i0
    for (int u = 0; u < CP_PER; u++) {
        const int i = i0 + u;
        if (i >= c.num_pages) break;
        const bool used = in_use >> u & 1;
        if (i < live) {
            if (!used) p.to[i - r] = i;
        } else if (used) {
            p.rank[i] = r - below;
            p.from[r - below] = i;
        }
        r += used;
    }
    if (me == 0 && tid == 0) {
        *p.moves = live - below;
        *p.live = live;
    }
}
// grid x: page copies first (one workgroup per move and layer in turn), the
// last CP_TABLE workgroups tables and counts
constexpr int CP_TABLE = 64;
__global__ void __launch_bounds__(CP_THREADS) kv4_compact_apply_kernel(Kv4View c, CompactPlan p) {
    const int moves = *p.moves, live = *p.live;
    const int ncopy = gridDim.x - CP_TABLE;
    if ((int)blockIdx.x < ncopy) {
        for (int64_t w = blockIdx.x; w < (int64_t)moves * c.layers; w += ncopy) {
            const int m = (int)(w % moves);
            const size_t layer = (size_t)(w / moves) * c.layer_bytes;
            copy_bytes16(c.pages + layer + (size_t)p.to[m] * c.page_bytes, c.pages + layer + (size_t)p.from[m] * c.page_bytes,
                         c.page_bytes, threadIdx.x, blockDim.x);
        }
        return;
    }
    const int me = (blockIdx.x - ncopy) * CP_THREADS + threadIdx.x, step = CP_TABLE * CP_THREADS;
    for (int m = me; m < moves; m += step) {
        c.refs[p.to[m]] = c.refs[p.from[m]];
        c.refs[p.from[m]] = 0;
    }
    for (int64_t e = me; e < (int64_t)c.max_seqs * c.max_pages; e += step) {
        const int s = (int)(e / c.max_pages), j = (int)(e % c.max_pages);
        if (j >= kv4_pages_of(c, kv4_len(c, s))) continue;
        const int id = c.table[e];
        if (kv4_page_ok(c, id) && id >= live) c.table[e] = p.to[p.rank[id]];
    }
    if (me == 0) {
        c.state[KV4_FREE] = c.num_pages - live;
        c.state[KV4_HINT] = live;
    }
}

__global__ void kv4_copy_kernel(Kv4View c, const int32_t* src, const int32_t* dst) {
    const int s = src[blockIdx.x], d = dst[blockIdx.x];
    if (!kv4_page_ok(c, s) || !kv4_page_ok(c, d)) {
        if (threadIdx.x == 0 && blockIdx.y == 0) atomicOr((uint32_t*)c.state + KV4_STATUS, CACTUS_HIP_KV4_BAD_REQUEST);
        return;
    }
    const size_t layer = (size_t)blockIdx.y * c.layer_bytes;
    copy_bytes16(c.pages + layer + (size_t)d * c.page_bytes, c.pages + layer + (size_t)s * c.page_bytes, c.page_bytes,
                 threadIdx.x, blockDim.x);
}

// ------------------------------------------------------------ host side
int kv4_view(const cactus_hip_kv4_cache* c, size_t layer, const char* what, Kv4View* out) {
    const std::string w(what);
    CH_REQUIRE(c, w + ": null cache");
    CH_REQUIRE(c->head_dim == 64 || c->head_dim == 128 || c->head_dim == 256, w + ": head_dim is 64, 128 or 256");
    CH_REQUIRE(c->page_size >= 16 && c->page_size <= 4096 && (c->page_size & (c->page_size - 1)) == 0,
               w + ": page_size is a power of two from 16 to 4096");
    CH_REQUIRE(c->layers >= 1 && c->layers < 65535 && c->kv_heads >= 1 && c->kv_heads <= 4096, w + ": layers or kv_heads out of range");
    CH_REQUIRE(c->num_pages >= 1 && c->num_pages < (1u << 30) && c->max_seqs >= 1 && c->max_seqs <= KV4_MAX_SEQS &&
                   c->max_pages >= 1 && c->max_pages < (1u << 30) / c->page_size &&
                   c->max_seqs * c->max_pages < (1u << 31),
               w + ": num_pages, max_seqs or max_pages out of range");
    if (!out) return CACTUS_HIP_OK;
    CH_REQUIRE(c->pages && c->table && c->lens && c->refs && c->state, w + ": null buffer");
    CH_REQUIRE(((uintptr_t)c->pages & 127) == 0, w + ": pages is not 128-byte aligned");
    CH_REQUIRE(layer < c->layers, w + ": no such layer");
    Kv4View v;
    v.table = c->table;
    v.lens = c->lens;
    v.refs = c->refs;
    v.state = c->state;
    v.Hkv = (int)c->kv_heads;
    v.d = (int)c->head_dim;
    v.ps_log2 = __builtin_ctzll(c->page_size);
    v.num_pages = (int)c->num_pages;
    v.max_seqs = (int)c->max_seqs;
    v.max_pages = (int)c->max_pages;
    v.layers = (int)c->layers;
    v.page_bytes = c->kv_heads * (c->page_size / 16) * (18 * c->head_dim);
    v.layer_bytes = v.page_bytes * c->num_pages;
    v.pages = static_cast<uint8_t*>(c->pages) + layer * v.layer_bytes;
    *out = v;
    return CACTUS_HIP_OK;
}

// bytes of the lists behind the first 4096 of the workspace
static size_t fork_bytes(const cactus_hip_kv4_cache* c, size_t n) { return 4 * (64 + n * (c->max_pages + 2)); }
static size_t compact_bytes(const cactus_hip_kv4_cache* c) {
    return 4 * (64 + (c->num_pages + CP_BLOCK - 1) / CP_BLOCK + 3 * c->num_pages);
}

}  // namespace cactus_hip

using namespace cactus_hip;

extern "C" {

int cactus_hip_kv4_bytes(const cactus_hip_kv4_cache* cache, size_t* bytes) {
    CH_REQUIRE(bytes, "kv4_bytes: null");
    int rc = kv4_view(cache, 0, "kv4_bytes", nullptr);
    if (rc) return rc;
    *bytes = cache->layers * cache->num_pages * cache->kv_heads * (cache->page_size / 16) * (18 * cache->head_dim);
    return CACTUS_HIP_OK;
}

int cactus_hip_kv4_reset(const cactus_hip_kv4_cache* cache, void* stream) {
    Kv4View c;
    int rc = kv4_view(cache, 0, "kv4_reset", &c);
    if (rc) return rc;
    hipLaunchKernelGGL(kv4_reset_kernel, dim3(256), dim3(256), 0, as_stream(stream), c);
    return check_launch("kv4_reset");
}

int cactus_hip_kv4_status(const cactus_hip_kv4_cache* cache, int* status, void* stream) {
    Kv4View c;
    CH_REQUIRE(status, "kv4_status: null");
    int rc = kv4_view(cache, 0, "kv4_status", &c);
    if (rc) return rc;
    int32_t s = 0;
    rc = cactus_hip_memcpy_d2h(&s, c.state + KV4_STATUS, 4, stream);
    if (rc) return rc;
    *status = s;
    if (s) {
        hipLaunchKernelGGL(kv4_clear_status_kernel, dim3(1), dim3(1), 0, as_stream(stream), c.state);
        return check_launch("kv4_status");
    }
    return CACTUS_HIP_OK;
}

int cactus_hip_kv4_extend(const cactus_hip_kv4_cache* cache, const int32_t* seqs, const int32_t* counts, size_t batch,
                          size_t count, void* stream) {
    Kv4View c;
    int rc = kv4_view(cache, 0, "kv4_extend", &c);
    if (rc) return rc;
    CH_REQUIRE(batch <= cache->max_seqs, "kv4_extend: more requests than slots");
    CH_REQUIRE(counts || count < (1u << 30), "kv4_extend: count out of range");
    if (batch == 0) return CACTUS_HIP_OK;
    hipLaunchKernelGGL(kv4_extend_kernel, dim3(1), dim3(BK_THREADS), 0, as_stream(stream), c, seqs, counts, (int)batch,
                       (int)count);
    return check_launch("kv4_extend");
}

int cactus_hip_kv4_append_f16(const cactus_hip_kv4_cache* cache, size_t layer, const int32_t* seqs,
                              const int32_t* counts, const uint16_t* k, const uint16_t* v, size_t batch,
                              size_t seq_len, size_t kv_stride, void* stream) {
    Kv4View c;
    int rc = kv4_view(cache, layer, "kv4_append", &c);
    if (rc) return rc;
    if (batch == 0 || seq_len == 0) return CACTUS_HIP_OK;
    CH_REQUIRE(k && v, "kv4_append: null pointer");
    CH_REQUIRE(((uintptr_t)k & 15) == 0 && ((uintptr_t)v & 15) == 0 && kv_stride % 8 == 0,
               "kv4_append: rows are not 16-byte aligned");
    CH_REQUIRE(kv_stride >= cache->kv_heads * cache->head_dim, "kv4_append: kv_stride is shorter than a row");
    CH_REQUIRE(batch <= cache->max_seqs, "kv4_append: more requests than slots");
    CH_REQUIRE(seq_len < (1u << 30), "kv4_append: seq_len out of range");
    const dim3 grid(ceil_div(seq_len + 15, 16), c.Hkv, (unsigned)batch);
    switch (c.d) {
        case 64: hipLaunchKernelGGL(kv4_append_kernel<64>, grid, dim3(64), 0, as_stream(stream), c, seqs, counts, k, v, (int)seq_len, kv_stride); break;
        case 128: hipLaunchKernelGGL(kv4_append_kernel<128>, grid, dim3(64), 0, as_stream(stream), c, seqs, counts, k, v, (int)seq_len, kv_stride); break;
        default: hipLaunchKernelGGL(kv4_append_kernel<256>, grid, dim3(64), 0, as_stream(stream), c, seqs, counts, k, v, (int)seq_len, kv_stride);
    }
    return check_launch("kv4_append");
}

int cactus_hip_kv4_read_f16(const cactus_hip_kv4_cache* cache, size_t layer, const int32_t* seqs, const int32_t* starts,
                            const int32_t* counts, uint16_t* k, uint16_t* v, size_t batch, size_t seq_len,
                            void* stream) {
    Kv4View c;
    int rc = kv4_view(cache, layer, "kv4_read", &c);
    if (rc) return rc;
    if (batch == 0 || seq_len == 0 || (!k && !v)) return CACTUS_HIP_OK;
    CH_REQUIRE(((uintptr_t)k & 15) == 0 && ((uintptr_t)v & 15) == 0, "kv4_read: rows are not 16-byte aligned");
    CH_REQUIRE(batch <= 65535, "kv4_read: more than 65535 requests");
    CH_REQUIRE(seq_len < (1u << 30), "kv4_read: seq_len out of range");
    const dim3 grid(ceil_div(seq_len + 15, 16), c.Hkv, (unsigned)batch);
    switch (c.d) {
        case 64: hipLaunchKernelGGL(kv4_read_kernel<64>, grid, dim3(64), 0, as_stream(stream), c, seqs, starts, counts, k, v, (int)seq_len); break;
        case 128: hipLaunchKernelGGL(kv4_read_kernel<128>, grid, dim3(64), 0, as_stream(stream), c, seqs, starts, counts, k, v, (int)seq_len); break;
        default: hipLaunchKernelGGL(kv4_read_kernel<256>, grid, dim3(64), 0, as_stream(stream), c, seqs, starts, counts, k, v, (int)seq_len);
    }
    return check_launch("kv4_read");
}

size_t cactus_hip_kv4_pages_workspace(const cactus_hip_kv4_cache* cache, size_t n) {
    if (kv4_view(cache, 0, "kv4_pages_workspace", nullptr)) return 0;
    n = std::min(n, cache->max_seqs);
    return KV4_WORK_SKIP + std::max(fork_bytes(cache, n), compact_bytes(cache));
}

int cactus_hip_kv4_fork(const cactus_hip_kv4_cache* cache, const int32_t* src, const int32_t* dst, size_t n,
                        void* workspace, size_t workspace_bytes, void* stream) {
    Kv4View c;
    int rc = kv4_view(cache, 0, "kv4_fork", &c);
    if (rc) return rc;
    if (n == 0) return CACTUS_HIP_OK;
    CH_REQUIRE(src && dst, "kv4_fork: null pointer");
    CH_REQUIRE(n <= cache->max_seqs, "kv4_fork: more pairs than slots");
    CH_REQUIRE(workspace && ((uintptr_t)workspace & 255) == 0 && workspace_bytes >= KV4_WORK_SKIP + fork_bytes(cache, n),
               "kv4_fork: workspace too small or not 256-byte aligned");
    int32_t* w = reinterpret_cast<int32_t*>(static_cast<uint8_t*>(workspace) + KV4_WORK_SKIP);
    ForkPlan p{w, w + 64, w + 64 + n, w + 64 + 2 * n};
    const hipStream_t st = as_stream(stream);
    hipLaunchKernelGGL(kv4_fork_plan_kernel, dim3(1), dim3(BK_THREADS), 0, st, c, p, src, dst, (int)n);
    hipLaunchKernelGGL(kv4_fork_share_kernel, dim3((unsigned)n), dim3(256), 0, st, c, p, src, dst);
    hipLaunchKernelGGL(kv4_fork_apply_kernel, dim3((unsigned)n, c.layers + 1), dim3(256), 0, st, c, p, src, dst);
    return check_launch("kv4_fork");
}

int cactus_hip_kv4_free(const cactus_hip_kv4_cache* cache, const int32_t* seqs, size_t n, void* stream) {
    Kv4View c;
    int rc = kv4_view(cache, 0, "kv4_free", &c);
    if (rc) return rc;
    if (n == 0) return CACTUS_HIP_OK;
    CH_REQUIRE(n < (1u << 31), "kv4_free: too many requests");
    hipLaunchKernelGGL(kv4_free_kernel, dim3((unsigned)n), dim3(256), 0, as_stream(stream), c, seqs);
    return check_launch("kv4_free");
}

int cactus_hip_kv4_compact(const cactus_hip_kv4_cache* cache, void* workspace, size_t workspace_bytes, void* stream) {
    Kv4View c;
    int rc = kv4_view(cache, 0, "kv4_compact", &c);
    if (rc) return rc;
    CH_REQUIRE(workspace && ((uintptr_t)workspace & 255) == 0 && workspace_bytes >= KV4_WORK_SKIP + compact_bytes(cache),
               "kv4_compact: workspace too small or not 256-byte aligned");
    const unsigned blocks = ceil_div(cache->num_pages, CP_BLOCK);
    int32_t* w = reinterpret_cast<int32_t*>(static_cast<uint8_t*>(workspace) + KV4_WORK_SKIP);
    const size_t np = cache->num_pages;
    CompactPlan p{w, w + 1, w + 64, w + 64 + blocks, w + 64 + blocks + np, w + 64 + blocks + 2 * np};
    const hipStream_t st = as_stream(stream);
    hipLaunchKernelGGL(kv4_compact_count_kernel, dim3(blocks), dim3(CP_THREADS), 0, st, c, p);
    hipLaunchKernelGGL(kv4_compact_list_kernel, dim3(blocks), dim3(CP_THREADS), 0, st, c, p);
    hipLaunchKernelGGL(kv4_compact_apply_kernel, dim3(2048 + CP_TABLE), dim3(CP_THREADS), 0, st, c, p);
    return check_launch("kv4_compact");
}

int cactus_hip_kv4_copy_pages(const cactus_hip_kv4_cache* cache, const int32_t* src, const int32_t* dst, size_t n,
                              void* stream) {
    Kv4View c;
    int rc = kv4_view(cache, 0, "kv4_copy_pages", &c);
    if (rc) return rc;
    if (n == 0) return CACTUS_HIP_OK;
    CH_REQUIRE(src && dst, "kv4_copy_pages: null pointer");
    CH_REQUIRE(n <= cache->num_pages, "kv4_copy_pages: more pairs than pages");
    hipLaunchKernelGGL(kv4_copy_kernel, dim3((unsigned)n, c.layers), dim3(256), 0, as_stream(stream), c, src, dst);
    return check_launch("kv4_copy_pages");
}

}  // extern "C"
