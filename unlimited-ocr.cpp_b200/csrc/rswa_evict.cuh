// Eviction from the fixed region of the paged cache by accumulated attention weight: choose the tokens to
// keep, move their K and V rows together, publish the shorter region.
#pragma once

#include "rswa_paged.cuh"

namespace uocr_b200 {

// -------------------------------------------------------------------------------------------------
// choose: the `keep` tokens of the largest mass, ties to the lowest index, as an ascending list.
// One CTA per slot.  The masses become 32-bit keys of the same order (protected tokens the key of
// +infinity, so that more of them than `keep` are kept from the front like any tie; NaN below everything); four passes of 8 bits narrow the keep-th largest key down by a
// histogram in shared memory, and a last ordered pass writes the tokens above it and the first of those
// equal to it.  The keys of up to kSelectSharedTokens tokens stay in shared memory.
// Bound by latency: 10 us for 1024 of 4096 tokens of 8 slots, 6.5 us for 128 of 273.
// -------------------------------------------------------------------------------------------------
constexpr int kSelectThreads = 1024;
constexpr int kSelectCopies = 8;
constexpr int kSelectSharedTokens = 49152;

struct SelectParams {
    const float* mass;
    int mass_stride;
    const int* d_prefill_len;
    const int* d_slots;
    int n, keep, sinks, recent;
    int* d_keep;  // [n][keep]
    int* d_keep_len;
    int* status;
};

__device__ __forceinline__ uint32_t mass_key(float m) {
    if (m != m) return 0u;
    const uint32_t u = __float_as_uint(m + 0.f);  // -0 counts as 0
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

__global__ void __launch_bounds__(kSelectThreads) rswa_evict_select_kernel(const SelectParams p, int shared_tokens) {
    extern __shared__ uint32_t keys[];
    __shared__ int hist[kSelectCopies][256];  // masses crowd into few bins: every fourth warp has its own counts
    __shared__ int warp_gt[32], warp_eq[32];
    __shared__ uint32_t s_prefix;
    __shared__ int s_need;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the compaction may be set up meanwhile (it waits for this launch)
    const int slot = __ldg(p.d_slots + blockIdx.x);
    const int pfx = max(__ldg(p.d_prefill_len + slot), 0);
    const int n = min(pfx, p.mass_stride);
    if (pfx > p.mass_stride && tid == 0 && p.status) atomicOr(p.status, kStatusBadSlot);
    int* out = p.d_keep + (size_t)blockIdx.x * p.keep;
    const int take = min(n, p.keep);
    const float* mass = p.mass + (size_t)slot * p.mass_stride;
    auto key_of = [&](int s) -> uint32_t {
        if (s < p.sinks || s >= n - p.recent) return 0xff800000u;
        return mass_key(__ldg(mass + s));
    };
    const bool cached = n <= shared_tokens;
    if (cached)
        for (int s = tid; s < n; s += kSelectThreads) keys[s] = key_of(s);
    if (tid == 0) {
        s_prefix = 0;
        s_need = take;
        p.d_keep_len[blockIdx.x] = take;
    }
    auto key = [&](int s) { return cached ? keys[s] : key_of(s); };
    uint32_t threshold = 0;
    int need_eq = n;  // everything is kept: no threshold to look for
    if (take < n && take > 0) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (int i = tid; i < kSelectCopies * 256; i += kSelectThreads) (&hist[0][0])[i] = 0;
            __syncthreads();
            const uint32_t prefix = s_prefix, mask = shift == 24 ? 0u : ~0u << (shift + 8);
            for (int s0 = 0; s0 < n; s0 += kSelectThreads) {
                const int s = s0 + tid;
                const uint32_t k = s < n ? key(s) : 0u;
                if (s < n && (k & mask) == prefix) atomicAdd(&hist[warp % kSelectCopies][(k >> shift) & 255u], 1);
            }
            __syncthreads();
            if (tid < 256) {
                int sum = 0;
#pragma unroll
                for (int i = 0; i < kSelectCopies; ++i) sum += hist[i][tid];
                hist[0][tid] = sum;
            }
            __syncthreads();
            if (warp == 0) {  // the bin, from the top, in which the running count reaches what is still needed
                const int need = s_need;
                int mine = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) mine += hist[0][255 - lane * 8 - i];
                int incl = mine;
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) {
                    const int t = __shfl_up_sync(0xffffffffu, incl, d);
                    if (lane >= d) incl += t;
                }
                const unsigned reach = __ballot_sync(0xffffffffu, incl >= need);
                if (lane == __ffs(reach) - 1) {
                    int above = incl - mine;
                    for (int i = 0; i < 8; ++i) {
                        const int bin = 255 - lane * 8 - i;
                        if (above + hist[0][bin] >= need) {
                            s_prefix = prefix | ((uint32_t)bin << shift);
                            s_need = need - above;
                            break;
                        }
                        above += hist[0][bin];
                    }
                }
            }
            __syncthreads();
        }
        threshold = s_prefix;
        need_eq = s_need;
    }
    __syncthreads();
    // ordered output: every warp owns a run of tokens
    const int run = ((n + 32 * 32 - 1) / (32 * 32)) * 32;
    const int begin = min(n, warp * run), end = min(n, begin + run);
    const bool all = take == n;
    int gt = 0, eq = 0;
    for (int s0 = begin; s0 < end; s0 += 32) {
        const int s = s0 + lane;
        const uint32_t k = s < end ? key(s) : 0u;
        gt += __popc(__ballot_sync(0xffffffffu, s < end && (all || k > threshold)));
        eq += __popc(__ballot_sync(0xffffffffu, s < end && !all && k == threshold));
    }
    if (lane == 0) {
        warp_gt[warp] = gt;
        warp_eq[warp] = eq;
    }
    __syncthreads();
    int at_gt = 0, at_eq = 0;
    for (int w = 0; w < warp; ++w) {
        at_gt += warp_gt[w];
        at_eq += warp_eq[w];
    }
    if (take > 0)
        for (int s0 = begin; s0 < end; s0 += 32) {
            const int s = s0 + lane;
            const uint32_t k = s < end ? key(s) : 0u;
            const bool is_gt = s < end && (all || k > threshold), is_eq = s < end && !all && k == threshold;
            const unsigned b_gt = __ballot_sync(0xffffffffu, is_gt), b_eq = __ballot_sync(0xffffffffu, is_eq);
            const unsigned below = (1u << lane) - 1;
            const int eq_rank = at_eq + __popc(b_eq & below);
            if (is_gt || (is_eq && eq_rank < need_eq))
                out[at_gt + __popc(b_gt & below) + min(eq_rank, need_eq)] = s;
            at_gt += __popc(b_gt);
            at_eq += __popc(b_eq);
        }
    for (int j = take + tid; j < p.keep; j += kSelectThreads) out[j] = -1;
}

// -------------------------------------------------------------------------------------------------
// move: token keep[i][j] of the fixed region of slot d_slots[i] becomes token j of the new region, in every layer.
// Bytes in, bytes out, bound by HBM: 16 bytes a thread, one CTA per new block (a contiguous 16-token block of all
// KV heads) of K or V of a layer.
// 8 slots x 1024 tokens x 6 layers (503 MB moved): 82 us, 6.1 TB/s, 0.93 of the copy rate.
// -------------------------------------------------------------------------------------------------
struct CompactParams {
    LayerPools pools;
    const int32_t* table;
    int table_stride, num_blocks;
    int kv_heads, row_chunks;  // 16-byte chunks of a head row
    const int* d_prefill_len;
    const int* d_slots;
    const int* d_keep;
    int keep_stride;
    const int* d_keep_len;
    const int32_t* d_new_blocks;  // [n][new_stride]; null: in place
    int new_stride;
    int* status;
};

constexpr int kCompactThreads = 256;

// An earlier entry of the list names the same slot: it alone counts.  Block-wide.
__device__ __forceinline__ bool slot_seen_before(const int* d_slots, int i, int slot) {
    bool seen = false;
    for (int j = threadIdx.x; j < i; j += blockDim.x) seen |= __ldg(d_slots + j) == slot;
    return __syncthreads_or(seen) != 0;
}

// Chunk index of token `at` (head 0, chunk 0) of the old region, or -1.
__device__ __forceinline__ long long old_token(const CompactParams& p, int slot, int at, int pfx) {
    if (at < 0 || at >= pfx || at / kBlockTokens >= p.table_stride) {
        if (p.status) atomicOr(p.status, kStatusBadSlot);
        return -1;
    }
    const int blk = __ldg(p.table + (size_t)slot * p.table_stride + at / kBlockTokens);
    if (blk < 0 || blk >= p.num_blocks) {
        if (p.status) atomicOr(p.status, kStatusBadBlock);
        return -1;
    }
    return ((long long)blk * p.kv_heads * kBlockTokens + (at & (kBlockTokens - 1))) * p.row_chunks;
}

__global__ void __launch_bounds__(kCompactThreads) rswa_evict_compact_kernel(const __grid_constant__ CompactParams p) {
    __shared__ long long s_src[kBlockTokens];
    asm volatile("griddepcontrol.wait;" ::: "memory");  // (launched so that its set-up overlaps the launch before it)
    const int i = blockIdx.z, nb = blockIdx.x, tid = threadIdx.x;
    const int layer = blockIdx.y >> 1;
    uint4* pool = reinterpret_cast<uint4*>((blockIdx.y & 1) ? p.pools.v[layer] : p.pools.k[layer]);
    const int count = min(__ldcg(p.d_keep_len + i), p.keep_stride);
    if (nb * kBlockTokens >= count) return;
    const int dst = nb < p.new_stride ? __ldg(p.d_new_blocks + (size_t)i * p.new_stride + nb) : -1;
    if (dst < 0 || dst >= p.num_blocks) {
        if (tid == 0 && p.status) atomicOr(p.status, kStatusBadBlock);
        return;
    }
    if (tid < kBlockTokens) {
        const int slot = __ldg(p.d_slots + i);
        const int j = nb * kBlockTokens + tid;
        s_src[tid] = j < count ? old_token(p, slot, __ldcg(p.d_keep + (size_t)i * p.keep_stride + j), __ldg(p.d_prefill_len + slot)) : -1;
    }
    __syncthreads();
    uint4* out = pool + (long long)dst * p.kv_heads * kBlockTokens * p.row_chunks;
    const int chunks = p.kv_heads * kBlockTokens * p.row_chunks;
    // Four to five loads in flight: 8 slots x 1024 tokens x 6 layers move in 82 us with either (10 heads of 128), 66 (8 heads; 4 of 256),
    // 129 (16 heads), 38 (8 heads of 64); with eight loads in 86, 67, 128, 47.
    constexpr int kUnroll = 5;
    for (int c0 = tid; c0 < chunks; c0 += kUnroll * kCompactThreads) {
        uint4 w[kUnroll];
        bool live[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int c = c0 + u * kCompactThreads;
            const int row = c / p.row_chunks;  // head * 16 + token
            const int head = row / kBlockTokens;
            const long long src = c < chunks ? s_src[row & (kBlockTokens - 1)] : -1;
            live[u] = src >= 0;
            if (live[u]) w[u] = __ldg(pool + src + (long long)head * kBlockTokens * p.row_chunks + (c - row * p.row_chunks));
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
            if (live[u]) out[c0 + u * kCompactThreads] = w[u];
    }
}

// In place: the new region takes the first blocks of the old one.  The list ascends, so token j comes from a token at
// or behind j; one CTA walks a head of a layer in order and reads a batch of rows before it writes it, so nothing is
// overwritten before it has been read.
__global__ void __launch_bounds__(kCompactThreads) rswa_evict_compact_in_place_kernel(const __grid_constant__ CompactParams p) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int i = blockIdx.z, head = blockIdx.x, tid = threadIdx.x;
    const int layer = blockIdx.y >> 1;
    uint4* pool = reinterpret_cast<uint4*>((blockIdx.y & 1) ? p.pools.v[layer] : p.pools.k[layer]);
    const int slot = __ldg(p.d_slots + i);
    if (slot_seen_before(p.d_slots, i, slot)) return;
    const int count = min(__ldcg(p.d_keep_len + i), p.keep_stride), pfx = __ldg(p.d_prefill_len + slot);
    const int* keep = p.d_keep + (size_t)i * p.keep_stride;
    const int rows = kCompactThreads / p.row_chunks;  // head rows of at most 64 chunks
    const int my_row = tid / p.row_chunks, c = tid - my_row * p.row_chunks;
    const long long head_at = (long long)head * kBlockTokens * p.row_chunks + c;
    for (int j0 = 0; j0 < count; j0 += 4 * rows) {
        uint4 w[4];
        long long dst[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int j = j0 + u * rows + my_row;
            dst[u] = -1;
            if (my_row < rows && j < count) {
                const int at = __ldcg(keep + j);
                const long long src = at >= j ? old_token(p, slot, at, pfx) : -1;
                if (src >= 0 && at != j) {
                    dst[u] = old_token(p, slot, j, pfx);
                    w[u] = pool[src + head_at];
                }
            }
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (dst[u] >= 0) pool[dst[u] + head_at] = w[u];
        __syncthreads();
    }
}

// -------------------------------------------------------------------------------------------------
// publish: block-table row, lengths, and the per-token arrays that go with the region.  One CTA per slot.
// -------------------------------------------------------------------------------------------------
struct EvictPublishParams {
    int32_t* table;
    int table_stride;
    const int* d_slots;
    const int* d_keep;
    int keep_stride;
    const int* d_keep_len;
    const int32_t* d_new_blocks;
    int new_stride;
    int* d_len;
    long long cursor_layer_stride;
    int layers;
    int* d_prefill_len;
    int window;
    float* mass;
    int mass_stride;
    int* key_pos;
    int key_pos_stride;
    int* status;
};

constexpr int kPublishThreads = 256;

// x[j] <- x[keep[j]] for j < count (the list ascends), `fill` from there up to `old`.
template <typename T>
__device__ __forceinline__ void compact_tokens(T* x, int stride, const int* keep, int count, int old, T fill, int* status) {
    const int tid = threadIdx.x;
    if (old > stride && tid == 0 && status) atomicOr(status, kStatusBadSlot);
    const int end = min(old, stride);
    for (int j0 = 0; j0 < end; j0 += kPublishThreads) {
        const int j = j0 + tid;
        T t = fill;
        if (j < count) {
            const int at = __ldcg(keep + j);
            if (at >= j && at < end) t = x[at];
        }
        __syncthreads();
        if (j < end) x[j] = t;
        __syncthreads();
    }
}

__global__ void __launch_bounds__(kPublishThreads) rswa_evict_publish_kernel(const __grid_constant__ EvictPublishParams p) {
    const int i = blockIdx.x, tid = threadIdx.x;
    const int slot = __ldg(p.d_slots + i);
    if (slot_seen_before(p.d_slots, i, slot)) return;
    const int old = p.d_prefill_len[slot];
    const int count = min(min(__ldcg(p.d_keep_len + i), p.keep_stride), old);
    if (count < 0) return;
    const int* keep = p.d_keep + (size_t)i * p.keep_stride;
    const int old_blocks = (old + kBlockTokens - 1) / kBlockTokens, new_blocks = (count + kBlockTokens - 1) / kBlockTokens;
    const int ring_blocks = (p.window + kBlockTokens - 1) / kBlockTokens;
    int32_t* row = p.table + (size_t)slot * p.table_stride;
    if (p.d_new_blocks && new_blocks > p.new_stride && tid == 0 && p.status) atomicOr(p.status, kStatusBadBlock);
    // the row moves left: the ring's blocks follow the new region's, what is left over is cleared
    for (int e0 = 0; e0 < p.table_stride; e0 += kPublishThreads) {
        const int e = e0 + tid;
        int32_t blk = -1;
        if (e < new_blocks) {
            blk = !p.d_new_blocks ? (e < p.table_stride ? row[e] : -1) : (e < p.new_stride ? __ldg(p.d_new_blocks + (size_t)i * p.new_stride + e) : -1);
        } else if (e < new_blocks + ring_blocks) {
            const int from = old_blocks + e - new_blocks;
            if (from < p.table_stride) blk = row[from];
        }
        __syncthreads();
        if (e < p.table_stride) row[e] = blk;
        __syncthreads();
    }
    if (p.mass) compact_tokens(p.mass + (size_t)slot * p.mass_stride, p.mass_stride, keep, count, old, 0.f, p.status);
    if (p.key_pos) compact_tokens(p.key_pos + (size_t)slot * p.key_pos_stride, p.key_pos_stride, keep, count, old, 0, p.status);
    for (int l = tid; l < p.layers; l += kPublishThreads) {
        int* len = p.d_len + l * p.cursor_layer_stride + slot;
        *len = max(*len - old, 0) + count;
    }
    if (tid == 0) p.d_prefill_len[slot] = count;
}

}  // namespace uocr_b200
