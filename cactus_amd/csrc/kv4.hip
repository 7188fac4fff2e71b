// kv4.hip -- the paged 4-bit KV cache: quantizing new rows into pages,
// reading them back, and the bookkeeping of pages (extend, fork, free,
// compact, copy) on the device.
#include "kv4_device.h"

#include <algorithm>

namespace cactus_hip {

// ------------------------------------------------------------ append and read
// A wave takes the keys or the values of one 16-token tile of a KV head, lane 16 h +
// token with dims 8 h to 8 h + 7 of each 32-dim group.  For the keys that is the lane
// order of the page.  For the values the page holds, per dim, the four tokens of a
// quad of lanes: the quads transpose 4 x 4 bytes in registers, so that pages are
// read and written 4 bytes per group and lane, contiguous over the groups.
//
// Bound by memory for prompts, by the chain of loads (slot, length, page, row) for
// single tokens.

// grid (tile, KV head, request), two waves: keys and values
template <int D>
__global__ void __launch_bounds__(128) kv4_append_kernel(Kv4View c, const int32_t* seqs, const int32_t* counts,
                                                         const uint16_t* k, const uint16_t* v, int seq_len, size_t stride) {
    constexpr int NG = D / 32;
    const int lane = threadIdx.x & 63, key = lane & 15, h = lane >> 4;
    const bool vals = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6) != 0;
    const int head = blockIdx.y, req = blockIdx.z;
    const int status = c.state[KV4_STATUS];
    const int slot = kv4_slot(c, seqs, req);
    if (slot < 0 || status != 0) return;
    const int len = kv4_len(c, slot), first = len - kv4_count(counts, req, seq_len);   // (negative: rows without a token)
    const int lo = max(first, 0);
    const int pos0 = (lo & ~15) + 16 * (int)blockIdx.x;      // first position of this tile
    if (pos0 >= len) return;
    const int pos = pos0 + key;
    const bool mine = pos >= lo && pos < len;
    const uint16_t* src = (vals ? v : k) + ((size_t)req * seq_len + (mine ? pos - first : lo - first)) * stride +
                          (size_t)head * D + 8 * h;
    uint4 x[NG];
#pragma unroll
    for (int g = 0; g < NG; g++) x[g] = *reinterpret_cast<const uint4*>(src + 32 * g);
    const int page = c.table[(size_t)slot * c.max_pages + (pos0 >> c.ps_log2)];
    if (!kv4_page_ok(c, page)) return;
    uint8_t* out = kv4_tile(c, page, head, (pos0 & ((1 << c.ps_log2) - 1)) >> 4) + (vals ? 9 * D : 0);

    kv4_write_tile<D>(x, out, vals, mine, pos0 >= lo && pos0 + 16 <= len);
}

// four codes (a byte each, low nibble: code + 8) times s, an exact fp16 value
__device__ __forceinline__ uint2 kv4_values(uint32_t b, h16x2 s) {
    const h16x2 bias = {(_Float16)1032.0f, (_Float16)1032.0f};
    const h16x2 y0 = __builtin_bit_cast(h16x2, __builtin_amdgcn_perm(0x64646464u, b, 0x04010400u)) - bias;
    const h16x2 y1 = __builtin_bit_cast(h16x2, __builtin_amdgcn_perm(0x64646464u, b, 0x04030402u)) - bias;
    return make_uint2(__builtin_bit_cast(uint32_t, y0 * s), __builtin_bit_cast(uint32_t, y1 * s));
}

template <int D>
__global__ void __launch_bounds__(128) kv4_read_kernel(Kv4View c, const int32_t* seqs, const int32_t* starts,
                                                       const int32_t* counts, uint16_t* k, uint16_t* v, int seq_len) {
    constexpr int NG = D / 32;
    const int lane = threadIdx.x & 63, key = lane & 15, h = lane >> 4, i = lane & 3;
    const bool vals = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6) != 0;
    const int head = blockIdx.y, req = blockIdx.z;
    uint16_t* dst = vals ? v : k;
    const int slot = kv4_slot(c, seqs, req);
    if (slot < 0 || !dst) return;
    const int len = kv4_len(c, slot), m = kv4_count(counts, req, seq_len);
    const int first = starts ? starts[req] : len - m;   // may lie outside the slot's tokens
    const int64_t end64 = (int64_t)first + m;
    const int end = end64 < len ? (int)end64 : len;
    const int lo = max(first, 0);
    const int64_t pos64 = (int64_t)(lo & ~15) + 16 * (int64_t)blockIdx.x;
    if (pos64 >= end) return;
    const int pos0 = (int)pos64;
    const int page = c.table[(size_t)slot * c.max_pages + (pos0 >> c.ps_log2)];
    if (!kv4_page_ok(c, page)) return;
    const uint8_t* in = kv4_tile(c, page, head, (pos0 & ((1 << c.ps_log2) - 1)) >> 4) + (vals ? 9 * D : 0);
    uint16_t s[NG];
#pragma unroll
    for (int g = 0; g < NG; g++) s[g] = reinterpret_cast<const uint16_t*>(in + 8 * D)[((key >> 2) * NG + g) * 4 + (key & 3)];
    uint32_t c0[NG], c1[NG];                                 // codes of dims 0-3 and 4-7, low nibbles
    if (!vals) {
        uint32_t b[NG];
        load_dwords(b, in + lane * (D / 8));
#pragma unroll
        for (int p = 0; p < NG / 2; p++) {
            c0[2 * p] = b[2 * p] & 0x0F0F0F0Fu;
            c1[2 * p] = b[2 * p + 1] & 0x0F0F0F0Fu;
            c0[2 * p + 1] = (b[2 * p] >> 4) & 0x0F0F0F0Fu;
            c1[2 * p + 1] = (b[2 * p + 1] >> 4) & 0x0F0F0F0Fu;
        }
    } else {
        const uint8_t* at = in + (key >> 2) * 2 * D + (8 * (h & 1) + i) * (D / 8);
        load_dwords(c0, at);
        load_dwords(c1, at + 4 * (D / 8));
#pragma unroll
        for (int g = 0; g < NG; g++) {
            c0[g] = (quad_transpose(c0[g], i) >> (h & 2 ? 4 : 0)) & 0x0F0F0F0Fu;
            c1[g] = (quad_transpose(c1[g], i) >> (h & 2 ? 4 : 0)) & 0x0F0F0F0Fu;
        }
    }
    const int pos = pos0 + key;
    if (pos < lo || pos >= end) return;
    uint16_t* row = dst + (((size_t)req * seq_len + (size_t)(pos - first)) * c.Hkv + head) * D + 8 * h;
#pragma unroll
    for (int g = 0; g < NG; g++) {
        const h16x2 ss = {hbits(s[g]), hbits(s[g])};
        const uint2 y0 = kv4_values(c0[g], ss), y1 = kv4_values(c1[g], ss);
        *reinterpret_cast<uint4*>(row + 32 * g) = make_uint4(y0.x, y0.y, y1.x, y1.y);
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
        if (i + 4 <= c.num_pages) {
            const int r0 = c.refs[i], r1 = c.refs[i + 1], r2 = c.refs[i + 2], r3 = c.refs[i + 3];
            z = (r0 == 0) | (r1 == 0) << 1 | (r2 == 0) << 2 | (r3 == 0) << 3;
        } else {
            for (int u = 0; i + u < c.num_pages; u++) z |= (c.refs[i + u] == 0) << u;
        }
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
    const int free_pages = c.state[KV4_FREE], hint = c.state[KV4_HINT];   // (before anything is waited for)
    if (c.state[KV4_STATUS] != 0) return;     // the appends to come write nothing: no tokens for them
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
    if (bad || total > free_pages) {
        if (tid == 0) atomicOr((uint32_t*)c.state + KV4_STATUS, bad ? CACTUS_HIP_KV4_BAD_REQUEST : CACTUS_HIP_KV4_NO_PAGES);
        return;
    }
    // free pages in rounds of BK_IDS, each handed to the requests whose share
    // of the sequence of new pages falls into the round
    int at = max(hint, 0), done = 0;
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
    int32_t* ok;         // [3] whether the call is carried out, pages it takes, status bits
    int32_t* tail;       // [n] new page of the partly filled last one, -1
    int32_t* len;        // [n] the source's tokens before the call
    int32_t* rows;       // [n][max_pages] the source's pages before the call
};
constexpr size_t KV4_WORK_SKIP = 4096;

// The whole workgroup: whether the pairs are right, and how many pages they need.
__device__ bool fork_checked(const Kv4View& c, const int32_t* src, const int32_t* dst, int n, uint32_t* bits, int* counts,
                             int* total) {
    const int tid = threadIdx.x, ps1 = (1 << c.ps_log2) - 1;
    for (int i = tid; i < (c.max_seqs + 31) / 32; i += blockDim.x) bits[i] = 0;
    if (tid < 2) counts[tid] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += blockDim.x) {
        const int s = kv4_slot(c, src, i), d = kv4_slot(c, dst, i);
        if (s < 0 || d < 0 || mark_twice(bits, d)) {
            counts[0] = 1;
            continue;
        }
        if (s != d && (kv4_len(c, s) & ps1)) atomicAdd(&counts[1], 1);
    }
    __syncthreads();
    *total = counts[1];
    return counts[0] == 0;
}

// Workgroup 0 allocates the copies' pages; workgroup 1 + i sets pair i's source
// aside (row and length) and raises its full pages' counts.  Each checks the call
// by itself, so that one launch does both: the counts of pages in use are raised
// while workgroup 0 looks for pages whose count is 0, and the number of free
// pages and the status, which all of them read, change in the second launch.
__global__ void __launch_bounds__(BK_THREADS) kv4_fork_plan_kernel(Kv4View c, ForkPlan p, const int32_t* src,
                                                                   const int32_t* dst, int n) {
    __shared__ uint32_t bits[KV4_MAX_SEQS / 32];
    __shared__ int ids[BK_IDS], wave_sums[16], counts[2];
    const int tid = threadIdx.x, ps1 = (1 << c.ps_log2) - 1;
    const int free_pages = c.state[KV4_FREE], hint = c.state[KV4_HINT];   // (before anything is waited for)
    const int status = c.state[KV4_STATUS];
    int total;
    const bool right = fork_checked(c, src, dst, n, bits, counts, &total);
    const bool ok = right && total <= free_pages && status == 0;
    if (blockIdx.x > 0) {
        const int i = blockIdx.x - 1;
        if (!ok) return;
        const int s = kv4_slot(c, src, i);
        if (s == kv4_slot(c, dst, i)) return;
        const int len = kv4_len(c, s), full = len >> c.ps_log2, np = kv4_pages_of(c, len);
        if (tid == 0) p.len[i] = len;
        for (int j = tid; j < np; j += BK_THREADS) {
            const int id = c.table[(size_t)s * c.max_pages + j];
            p.rows[(size_t)i * c.max_pages + j] = id;
            if (j < full && kv4_page_ok(c, id)) atomicAdd(&c.refs[id], 1);
        }
        return;
    }
    if (tid == 0) {
        p.ok[0] = ok;
        p.ok[1] = total;
        p.ok[2] = ok || status ? 0 : right ? CACTUS_HIP_KV4_NO_PAGES : CACTUS_HIP_KV4_BAD_REQUEST;
    }
    if (!ok) return;
    // at most max_seqs pages: dst slots differ
    int at = max(hint, 0), done = 0;
    do {
        const int got = done < total ? collect_free(c, &at, total - done, ids, wave_sums) : 0;
        if (got == 0 && done < total) {
            // the free count was wrong: the pairs behind are left without a last page
            if (tid == 0) p.ok[2] = CACTUS_HIP_KV4_NO_PAGES;
            for (int i = tid; i < n; i += BK_THREADS) p.tail[i] = done ? p.tail[i] : -1;
            break;
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
                if (!part || o >= got) {
                    if (done == 0) p.tail[i] = -1;
                } else if (o >= 0) {
                    p.tail[i] = ids[o];
                    c.refs[ids[o]] = 1;
                }
            }
            base += chunk;
        }
        done += got;
        __syncthreads();
    } while (done < total);
    if (tid == 0 && total > 0) c.state[KV4_HINT] = at;
}
// a slot's pages given up (its row as it stands); whole waves
__device__ __forceinline__ void release_row(const Kv4View& c, int slot, int len) {
    const int np = kv4_pages_of(c, len), lane = threadIdx.x & 63;
    int freed = 0, lowest = 0x7FFFFFFF;
    for (int j = threadIdx.x; j < np; j += blockDim.x) {
        const int id = c.table[(size_t)slot * c.max_pages + j];
        if (kv4_page_ok(c, id) && atomicSub(&c.refs[id], 1) == 1) {
            freed++;
            lowest = min(lowest, id);
        }
    }
    // one update of the shared words per wave
    freed = wave_sum_i32(freed);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) lowest = min(lowest, __shfl_xor(lowest, o, 64));
    if (lane == 0 && freed) {
        atomicAdd(&c.state[KV4_FREE], freed);
        atomicMin(&c.state[KV4_HINT], lowest);
    }
}
// Pages are copied in pieces of COPY_PIECE bytes, a workgroup of 256 each, every
// load of a piece before its stores (a whole page per workgroup, load by load:
// 15 pages of 28 layers 17 us, 62 MB).
// Stores pass the caches (15 pages 13.8 -> 12.1 us); with ONCE the loads do too: a
// compaction's pages are not read again soon (784 MB moved 161 -> 150 us), a
// fork's source is (12.1 -> 16.3).
constexpr int COPY_PIECE = 16384;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
template <bool ONCE>
__device__ __forceinline__ void copy_piece(uint8_t* dst, const uint8_t* src, size_t bytes, int piece) {
    const uint32_t at = (uint32_t)piece * COPY_PIECE + 16 * threadIdx.x;
    const uint32_t end = min((uint32_t)bytes, (uint32_t)(piece + 1) * COPY_PIECE);
    if (end - (uint32_t)piece * COPY_PIECE == COPY_PIECE) {
        // (an array of four was moved to LDS, for which the kernel read its launch
        // packet in host memory: 13 us)
        const u32x4* s = reinterpret_cast<const u32x4*>(src + at);
        u32x4* d = reinterpret_cast<u32x4*>(dst + at);
        u32x4 w0, w1, w2, w3;
        if constexpr (ONCE) {
            w0 = __builtin_nontemporal_load(s), w1 = __builtin_nontemporal_load(s + 256);
            w2 = __builtin_nontemporal_load(s + 512), w3 = __builtin_nontemporal_load(s + 768);
        } else {
            w0 = s[0], w1 = s[256], w2 = s[512], w3 = s[768];
        }
        __builtin_nontemporal_store(w0, d);
        __builtin_nontemporal_store(w1, d + 256);
        __builtin_nontemporal_store(w2, d + 512);
        __builtin_nontemporal_store(w3, d + 768);
    } else {
        for (uint32_t o = at; o < end; o += 4096) *reinterpret_cast<uint4*>(dst + o) = *reinterpret_cast<const uint4*>(src + o);
    }
}

// block y 0: the destination's table row; from 1 on: a piece of the last page, a layer
__global__ void __launch_bounds__(256) kv4_fork_apply_kernel(Kv4View c, ForkPlan p, const int32_t* src, const int32_t* dst,
                                                             int pieces) {
    const int i = blockIdx.x;
    const bool first = blockIdx.y == 0 && i == 0 && threadIdx.x == 0;
    if (first && p.ok[2]) atomicOr((uint32_t*)c.state + KV4_STATUS, (uint32_t)p.ok[2]);
    if (!p.ok[0]) return;
    const int d = kv4_slot(c, dst, i);
    if (first) atomicSub(&c.state[KV4_FREE], p.ok[1]);
    if (kv4_slot(c, src, i) == d) return;
    const int32_t* row = p.rows + (size_t)i * c.max_pages;
    const int len = p.len[i], full = len >> c.ps_log2, tail = p.tail[i];
    if (blockIdx.y > 0) {
        if (tail < 0 || !kv4_page_ok(c, row[full])) return;
        const size_t layer = (size_t)((blockIdx.y - 1) / pieces) * c.layer_bytes;
        copy_piece<false>(c.pages + layer + (size_t)tail * c.page_bytes, c.pages + layer + (size_t)row[full] * c.page_bytes,
                   c.page_bytes, (blockIdx.y - 1) % pieces);
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
constexpr int CP_THREADS = 1024, CP_PER = 4, CP_BLOCK = CP_THREADS * CP_PER;   // pages per workgroup
struct CompactPlan {
    int32_t* moves;      // [1]
    int32_t* live;       // [1] pages in use
    int32_t* used;       // [blocks] pages in use among a workgroup's
    int32_t* rank;       // [num_pages] of a page that moves: which of them it is
    int32_t* from;       // [num_pages] pages that move, ascending
    int32_t* to;         // [num_pages] free pages below `live`, ascending
};
// bit u: page i0 + u is in use
__device__ __forceinline__ uint32_t pages_in_use(const Kv4View& c, int i0) {
    uint32_t bits = 0;
#pragma unroll
    for (int u = 0; u < CP_PER; u++) bits |= (uint32_t)(i0 + u < c.num_pages && c.refs[i0 + u] > 0) << u;
    return bits;
}
__device__ __forceinline__ uint32_t bits_below(int i0, int top) {   // of pages i0 on, those below `top`
    return top <= i0 ? 0 : top - i0 >= CP_PER ? (1u << CP_PER) - 1 : (1u << (top - i0)) - 1;
}
// (pools of more than CP_BLOCK pages)
__global__ void __launch_bounds__(CP_THREADS) kv4_compact_count_kernel(Kv4View c, CompactPlan p) {
    __shared__ int sums[16];
    int total;
    block_scan(__popc(pages_in_use(c, (blockIdx.x * CP_THREADS + threadIdx.x) * CP_PER)), sums, &total);
    if (threadIdx.x == 0) p.used[blockIdx.x] = total;
}
__global__ void __launch_bounds__(CP_THREADS) kv4_compact_list_kernel(Kv4View c, CompactPlan p) {
    __shared__ int sums[16];
    const int tid = threadIdx.x, blocks = gridDim.x, me = blockIdx.x;
    const int i0 = (me * CP_THREADS + tid) * CP_PER;
    const uint32_t in_use = pages_in_use(c, i0);
    int mine, t, before_me = 0, live, below = 0;
    const int inside = block_scan(__popc(in_use), sums, &mine);
    if (blocks == 1) {
        live = mine;
        block_scan(__popc(in_use & bits_below(i0, live)), sums, &below);
    } else {
        live = 0;
        for (int b0 = 0; b0 < blocks; b0 += CP_THREADS) {
            const int b = b0 + tid, v = b < blocks ? p.used[b] : 0;
            block_scan(b < me ? v : 0, sums, &t);
            before_me += t;
            block_scan(v, sums, &t);
            live += t;
        }
        // pages in use below `live`: whole workgroups' shares and a part of one
        const int edge = live / CP_BLOCK;
        for (int b0 = 0; b0 < edge; b0 += CP_THREADS) {
            block_scan(b0 + tid < edge ? p.used[b0 + tid] : 0, sums, &t);
            below += t;
        }
        const int e0 = (edge * CP_THREADS + tid) * CP_PER;
        block_scan(__popc(pages_in_use(c, e0) & bits_below(e0, live)), sums, &t);
        below += t;
    }
    int r = before_me + inside;                   // pages in use before page i0
#pragma unroll
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
// the first CP_TABLE workgroups tables and counts, the others pieces of pages in turn
constexpr int CP_TABLE = 64;
__global__ void __launch_bounds__(256) kv4_compact_apply_kernel(Kv4View c, CompactPlan p, int pieces) {
    const int moves = *p.moves, live = *p.live;
    if (blockIdx.x >= CP_TABLE) {
        const uint64_t per_page = (uint64_t)pieces * c.layers;
        for (uint64_t w = blockIdx.x - CP_TABLE; w < moves * per_page; w += gridDim.x - CP_TABLE) {
            const int m = (int)(w / per_page), r = (int)(w % per_page);
            const size_t layer = (size_t)(r / pieces) * c.layer_bytes;
            copy_piece<true>(c.pages + layer + (size_t)p.to[m] * c.page_bytes, c.pages + layer + (size_t)p.from[m] * c.page_bytes,
                       c.page_bytes, r % pieces);
        }
        return;
    }
    const int me = blockIdx.x * 256 + threadIdx.x, step = CP_TABLE * 256;
    for (int m = me; m < moves; m += step) {
        c.refs[p.to[m]] = c.refs[p.from[m]];
        c.refs[p.from[m]] = 0;
    }
    for (uint32_t e = me; e < (uint32_t)c.max_seqs * (uint32_t)c.max_pages; e += step) {
        const int id = c.table[e];
        if (!kv4_page_ok(c, id) || id < live) continue;
        const int s = (int)(e / (uint32_t)c.max_pages), j = (int)(e % (uint32_t)c.max_pages);
        const uint32_t r = (uint32_t)p.rank[id];
        if (j < kv4_pages_of(c, kv4_len(c, s)) && r < (uint32_t)moves) c.table[e] = p.to[r];
    }
    if (me == 0) {
        c.state[KV4_FREE] = c.num_pages - live;
        c.state[KV4_HINT] = live;
    }
}

__global__ void __launch_bounds__(256) kv4_copy_kernel(Kv4View c, const int32_t* src, const int32_t* dst, int pieces) {
    const int s = src[blockIdx.x], d = dst[blockIdx.x];
    if (!kv4_page_ok(c, s) || !kv4_page_ok(c, d)) {
        if (threadIdx.x == 0 && blockIdx.y == 0) atomicOr((uint32_t*)c.state + KV4_STATUS, CACTUS_HIP_KV4_BAD_REQUEST);
        return;
    }
    const size_t layer = (size_t)(blockIdx.y / pieces) * c.layer_bytes;
    copy_piece<false>(c.pages + layer + (size_t)d * c.page_bytes, c.pages + layer + (size_t)s * c.page_bytes, c.page_bytes,
               blockIdx.y % pieces);
}

// ------------------------------------------------------------ host side
int kv4_view(const cactus_hip_kv4_cache* c, size_t layer, const char* what, Kv4View* out) {
    using std::string;
    CH_REQUIRE(c, string(what) + ": null cache");
    CH_REQUIRE(c->head_dim == 64 || c->head_dim == 128 || c->head_dim == 256, string(what) + ": head_dim is 64, 128 or 256");
    CH_REQUIRE(c->page_size >= 16 && c->page_size <= 4096 && (c->page_size & (c->page_size - 1)) == 0,
               string(what) + ": page_size is a power of two from 16 to 4096");
    CH_REQUIRE(c->layers >= 1 && c->layers <= 4096 && c->kv_heads >= 1 && c->kv_heads <= 4096,
               string(what) + ": layers or kv_heads out of range");
    // a page in pieces, all layers, is a launch dimension
    CH_REQUIRE(c->layers * ceil_div(c->kv_heads * (c->page_size / 16) * (18 * c->head_dim), 16384) < 65535,
               string(what) + ": layers times page bytes out of range");
    CH_REQUIRE(c->num_pages >= 1 && c->num_pages < (1u << 30) && c->max_seqs >= 1 && c->max_seqs <= KV4_MAX_SEQS &&
                   c->max_pages >= 1 && c->max_pages < (1u << 30) / c->page_size &&
                   c->max_seqs * c->max_pages < (1u << 31),
               string(what) + ": num_pages, max_seqs or max_pages out of range");
    if (!out) return CACTUS_HIP_OK;
    CH_REQUIRE(c->pages && c->table && c->lens && c->refs && c->state, string(what) + ": null buffer");
    CH_REQUIRE(((uintptr_t)c->pages & 127) == 0, string(what) + ": pages is not 128-byte aligned");
    CH_REQUIRE(layer < c->layers, string(what) + ": no such layer");
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
    CH_REQUIRE(batch <= cache->max_seqs && batch <= 65535, "kv4_append: more requests than slots, or than 65535");
    CH_REQUIRE(seq_len <= (1u << 28), "kv4_append: seq_len out of range");
    const dim3 grid(ceil_div(seq_len + 15, 16), c.Hkv, (unsigned)batch);
    switch (c.d) {
        case 64: hipLaunchKernelGGL(kv4_append_kernel<64>, grid, dim3(128), 0, as_stream(stream), c, seqs, counts, k, v, (int)seq_len, kv_stride); break;
        case 128: hipLaunchKernelGGL(kv4_append_kernel<128>, grid, dim3(128), 0, as_stream(stream), c, seqs, counts, k, v, (int)seq_len, kv_stride); break;
        default: hipLaunchKernelGGL(kv4_append_kernel<256>, grid, dim3(128), 0, as_stream(stream), c, seqs, counts, k, v, (int)seq_len, kv_stride);
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
    CH_REQUIRE(seq_len <= (1u << 28), "kv4_read: seq_len out of range");
    const dim3 grid(ceil_div(seq_len + 15, 16), c.Hkv, (unsigned)batch);
    switch (c.d) {
        case 64: hipLaunchKernelGGL(kv4_read_kernel<64>, grid, dim3(128), 0, as_stream(stream), c, seqs, starts, counts, k, v, (int)seq_len); break;
        case 128: hipLaunchKernelGGL(kv4_read_kernel<128>, grid, dim3(128), 0, as_stream(stream), c, seqs, starts, counts, k, v, (int)seq_len); break;
        default: hipLaunchKernelGGL(kv4_read_kernel<256>, grid, dim3(128), 0, as_stream(stream), c, seqs, starts, counts, k, v, (int)seq_len);
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
    const int pieces = (int)ceil_div(c.page_bytes, COPY_PIECE);
    hipLaunchKernelGGL(kv4_fork_plan_kernel, dim3((unsigned)n + 1), dim3(BK_THREADS), 0, st, c, p, src, dst, (int)n);
    hipLaunchKernelGGL(kv4_fork_apply_kernel, dim3((unsigned)n, c.layers * pieces + 1), dim3(256), 0, st, c, p, src, dst, pieces);
    return check_launch("kv4_fork");
}

int cactus_hip_kv4_free(const cactus_hip_kv4_cache* cache, const int32_t* seqs, size_t n, void* stream) {
    Kv4View c;
    int rc = kv4_view(cache, 0, "kv4_free", &c);
    if (rc) return rc;
    if (n == 0) return CACTUS_HIP_OK;
    CH_REQUIRE(n < (1u << 24), "kv4_free: too many requests");
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
    const int pieces = (int)ceil_div(c.page_bytes, COPY_PIECE);
    if (blocks > 1) hipLaunchKernelGGL(kv4_compact_count_kernel, dim3(blocks), dim3(CP_THREADS), 0, st, c, p);
    hipLaunchKernelGGL(kv4_compact_list_kernel, dim3(blocks), dim3(CP_THREADS), 0, st, c, p);
    hipLaunchKernelGGL(kv4_compact_apply_kernel, dim3(2048 + CP_TABLE), dim3(256), 0, st, c, p, pieces);
    return check_launch("kv4_compact");
}

int cactus_hip_kv4_copy_pages(const cactus_hip_kv4_cache* cache, const int32_t* src, const int32_t* dst, size_t n,
                              void* stream) {
    Kv4View c;
    int rc = kv4_view(cache, 0, "kv4_copy_pages", &c);
    if (rc) return rc;
    if (n == 0) return CACTUS_HIP_OK;
    CH_REQUIRE(src && dst, "kv4_copy_pages: null pointer");
    CH_REQUIRE(n <= cache->num_pages && n < (1u << 24), "kv4_copy_pages: more pairs than pages, or than 2^24");
    const int pieces = (int)ceil_div(c.page_bytes, COPY_PIECE);
    hipLaunchKernelGGL(kv4_copy_kernel, dim3((unsigned)n, c.layers * pieces), dim3(256), 0, as_stream(stream), c, src, dst, pieces);
    return check_launch("kv4_copy_pages");
}

}  // extern "C"
