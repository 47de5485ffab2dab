// The paged pool as the kernels see it, and the ring state machine of the append.
#pragma once

#include "rswa_device.cuh"

namespace uocr_b200 {

// The ring state machine of RSWACache::append_decode (src/scheduler/kv_cache.cpp:54-82) on device
// cursors, as in rswa_append_batch_kernel (src/kernels/cuda/rswa_attention.cu:309-338) -- except
// that exactly one thread reads and updates the cursors (the reference lets every thread of the
// CTA do both without a barrier in between).  Returns the logical slot to write.
__device__ __forceinline__ int ring_advance(int* len_p, int* ring_p, int prefill_len, int window) {
    const int len = *len_p;
    int row;
    if (len < prefill_len + window) {
        row = len;
        *len_p = len + 1;
        if (len + 1 >= prefill_len + window) *ring_p = 0;
    } else {
        const int rp = *ring_p;
        row = prefill_len + rp;
        *ring_p = (rp + 1) % window;
    }
    return row;
}

// ---- paged pool: [block][kv_head][16][head_dim] ---------------------------------------------------
struct PagedView {
    uint8_t* k_pool;
    uint8_t* v_pool;
    const int32_t* table;
    int table_stride, num_blocks, kv_heads, head_dim;
};

// Pools of several layers for the kernels that serve all layers of a step in one launch (blockIdx.z = layer).
constexpr int kMaxLayersPerLaunch = 32;
struct LayerPools {
    uint8_t* k[kMaxLayersPerLaunch];
    uint8_t* v[kMaxLayersPerLaunch];
};

}  // namespace uocr_b200
