// extern "C" entry points of the eviction from the fixed region.
#include "rswa_evict.cuh"
#include "rswa_workspace.cuh"

using namespace uocr_b200;

extern "C" {

int uocr_b200_rswa_evict_select(const float* mass, int mass_stride, const int* d_prefill_len, const int* d_slots, int n, int keep, int sinks,
                                int recent, int* d_keep, int* d_keep_len, uocr_b200_workspace* ws, uocr_b200_stream_t stream) {
    if (n <= 0) return UOCR_B200_OK;
    if (!mass || !d_prefill_len || !d_slots || !d_keep || !d_keep_len) return fail(UOCR_B200_ERR_INVALID, "evict_select: null pointer");
    if (mass_stride <= 0 || keep <= 0 || sinks < 0 || recent < 0) return fail(UOCR_B200_ERR_INVALID, "evict_select: mass_stride and keep must be positive, sinks and recent not negative");
    const DeviceInfo* di = nullptr;
    if (int rc = device_info(&di)) return rc;
    if (int rc = check_workspace_device(ws, "evict_select")) return rc;
    int dev = 0;
    CHECK_CUDA(cudaGetDevice(&dev), "cudaGetDevice");
    const int tokens = mass_stride < kSelectSharedTokens ? mass_stride : kSelectSharedTokens;
    static SmemLimit limit;
    CHECK_CUDA(limit.allow(rswa_evict_select_kernel, dev, kSelectSharedTokens * (int)sizeof(uint32_t)), "smem attribute");
    SelectParams p{};
    p.mass = mass;
    p.mass_stride = mass_stride;
    p.d_prefill_len = d_prefill_len;
    p.d_slots = d_slots;
    p.n = n;
    p.keep = keep;
    p.sinks = sinks;
    p.recent = recent;
    p.d_keep = d_keep;
    p.d_keep_len = d_keep_len;
    p.status = ws ? ws->status : nullptr;
    rswa_evict_select_kernel<<<n, kSelectThreads, tokens * sizeof(uint32_t), reinterpret_cast<cudaStream_t>(stream)>>>(p, tokens);
    return after_launch("evict: select");
}

int uocr_b200_rswa_evict_compact_paged_layers(const uocr_b200_paged_kv* kv_layers, int layers, const int* d_prefill_len, const int* d_slots,
                                              int n, const int* d_keep, int keep_stride, const int* d_keep_len, const int32_t* d_new_blocks,
                                              int new_stride, uocr_b200_workspace* ws, uocr_b200_stream_t stream) {
    if (n <= 0) return UOCR_B200_OK;
    PagedView pv;
    CompactParams p{};
    if (int rc = collect_layers(kv_layers, layers, &pv, &p.pools, "evict_compact_paged_layers")) return rc;
    if (!d_prefill_len || !d_slots || !d_keep || !d_keep_len) return fail(UOCR_B200_ERR_INVALID, "evict_compact_paged_layers: null pointer");
    if (keep_stride <= 0 || (d_new_blocks && new_stride <= 0)) return fail(UOCR_B200_ERR_INVALID, "evict_compact_paged_layers: strides must be positive");
    if (n > 65535) return fail(UOCR_B200_ERR_UNSUPPORTED, "evict_compact_paged_layers: at most 65535 slots per call");
    const DeviceInfo* di = nullptr;
    if (int rc = device_info(&di)) return rc;
    if (int rc = check_workspace_device(ws, "evict_compact_paged_layers")) return rc;
    p.table = pv.table;
    p.table_stride = pv.table_stride;
    p.num_blocks = pv.num_blocks;
    p.kv_heads = pv.kv_heads;
    p.row_chunks = pv.head_dim * (kv_layers[0].dtype == UOCR_B200_BF16 ? 2 : 4) / 16;
    p.d_prefill_len = d_prefill_len;
    p.d_slots = d_slots;
    p.d_keep = d_keep;
    p.keep_stride = keep_stride;
    p.d_keep_len = d_keep_len;
    p.d_new_blocks = d_new_blocks;
    p.new_stride = new_stride;
    p.status = ws ? ws->status : nullptr;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const dim3 grid = d_new_blocks ? dim3((keep_stride + kBlockTokens - 1) / kBlockTokens, 2 * layers, n) : dim3(pv.kv_heads, 2 * layers, n);
    CHECK_CUDA(launch_after(d_new_blocks ? rswa_evict_compact_kernel : rswa_evict_compact_in_place_kernel, grid, kCompactThreads, 0, st, p), "evict: compact");
    return after_launch("evict: compact");
}

int uocr_b200_rswa_evict_publish(int32_t* block_table, int table_stride, const int* d_slots, int n, const int* d_keep, int keep_stride,
                                 const int* d_keep_len, const int32_t* d_new_blocks, int new_stride, int* d_len,
                                 long long cursor_layer_stride, int layers, int* d_prefill_len, int window, float* mass, int mass_stride,
                                 int* d_key_pos, int key_pos_stride, uocr_b200_workspace* ws, uocr_b200_stream_t stream) {
    if (n <= 0) return UOCR_B200_OK;
    if (!block_table || !d_slots || !d_keep || !d_keep_len || !d_len || !d_prefill_len) return fail(UOCR_B200_ERR_INVALID, "evict_publish: null pointer");
    if (table_stride <= 0 || keep_stride <= 0 || layers <= 0 || window <= 0 || (d_new_blocks && new_stride <= 0) || (mass && mass_stride <= 0) ||
        (d_key_pos && key_pos_stride <= 0))
        return fail(UOCR_B200_ERR_INVALID, "evict_publish: bad geometry");
    const DeviceInfo* di = nullptr;
    if (int rc = device_info(&di)) return rc;
    if (int rc = check_workspace_device(ws, "evict_publish")) return rc;
    EvictPublishParams p{};
    p.table = block_table;
    p.table_stride = table_stride;
    p.d_slots = d_slots;
    p.d_keep = d_keep;
    p.keep_stride = keep_stride;
    p.d_keep_len = d_keep_len;
    p.d_new_blocks = d_new_blocks;
    p.new_stride = new_stride;
    p.d_len = d_len;
    p.cursor_layer_stride = cursor_layer_stride;
    p.layers = layers;
    p.d_prefill_len = d_prefill_len;
    p.window = window;
    p.mass = mass;
    p.mass_stride = mass_stride;
    p.key_pos = d_key_pos;
    p.key_pos_stride = key_pos_stride;
    p.status = ws ? ws->status : nullptr;
    rswa_evict_publish_kernel<<<n, kPublishThreads, 0, reinterpret_cast<cudaStream_t>(stream)>>>(p);
    return after_launch("evict: publish");
}

}  // extern "C"
