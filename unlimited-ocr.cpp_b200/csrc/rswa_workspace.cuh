// Host side shared by the translation units of the C ABI: the workspace, error reporting and launch
// accounting.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <string>

#include "rswa_device.cuh"
#include "uocr_rswa_b200.h"

namespace uocr_b200 {

struct RowInfo;
struct ScoreRow;
struct PrefillTile;
struct TcWork;

// Records `msg` as the calling thread's last error and returns `code`.
int fail(int code, const std::string& msg);
int cuda_fail(cudaError_t e, const char* what);
// Counts a launch and turns its launch error, if any, into a status.
int after_launch(const char* what);

#define CHECK_CUDA(expr, what)                             \
    do {                                                   \
        cudaError_t e_ = (expr);                           \
        if (e_ != cudaSuccess) return cuda_fail(e_, what); \
    } while (0)

struct DeviceInfo {
    bool known = false;
    int sms = 0;
    int smem_optin = 0;
    int cc_major = 0;
};
// The current device, refused unless it is an sm_100 part.
int device_info(const DeviceInfo** out);

// Dynamic shared memory of a kernel (one object per instantiation), allowed once per device.  `bytes` is the most that any call
// asks for, not what this one does: threads that raised the limit to sizes of their own could lower one another's.
struct SmemLimit {
    std::atomic<bool> set[64] = {};
    template <typename Kernel>
    cudaError_t allow(Kernel kernel, int device, int bytes) {
        if (set[device & 63].load(std::memory_order_acquire)) return cudaSuccess;
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e == cudaSuccess) set[device & 63].store(true, std::memory_order_release);
        return e;
    }
};

// Launches a kernel that opens with griddepcontrol.wait: its set-up may overlap the launch before it in the stream.
template <typename P>
cudaError_t launch_after(void (*kernel)(P), dim3 grid, int threads, int smem, cudaStream_t st, const P& params) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, params);
}

constexpr int kMaxHeadDim = 256;
constexpr int kPartElems = 512;  // accumulator elements of one partial: a head, or the heads of a group that share a KV tile

constexpr int kScoreMaxGroup = 4;  // query heads of a group that share one pass over a KV tile
constexpr size_t kScoreRowBytes = 32;
constexpr int kScoreJoinWidth = 8, kScoreJoinLevels = 4;  // partials are joined 8 at a time: 4 levels cover 4096 pieces

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

inline bool head_dim_ok(int hd, int dtype) {
    if (hd < (dtype == UOCR_B200_BF16 ? 8 : 4) || hd > kMaxHeadDim) return false;
    return (hd & (hd - 1)) == 0;
}

// The cap and the scale of modified scores.
int check_score(const uocr_b200_score* score, int head_dim, const char* who);

struct PagedView;
struct LayerPools;
// Checked views of one layer, and of several layers of one geometry behind one block table.
int paged_view(const uocr_b200_paged_kv* kv, PagedView* pv);
int collect_layers(const uocr_b200_paged_kv* kv, int layers, PagedView* pv, LayerPools* pools, const char* who);

}  // namespace uocr_b200

struct uocr_b200_workspace {
    int device = 0;
    int max_rows = 0;
    int total_warps_max = 0;
    uint8_t* base = nullptr;
    size_t bytes = 0;
    int* status = nullptr;
    int* rs = nullptr;
    uocr_b200::RowInfo* info = nullptr;
    uocr_b200::ScoreRow* score_rows = nullptr;  // [max_rows] plan of the attention with modified scores, when it is made in global memory
    long long* score_rs = nullptr;              // [max_rows + 1]
    int* score_counters = nullptr;              // [2 kScoreJoinLevels][pieces_max], zero between launches
    float* part_acc = nullptr;
    float* part_ml = nullptr;
    int* counters = nullptr;   // [pieces_max] arrival counters, zero between launches
    int* planned_ctas = nullptr;  // fused step: ticket counter of CTAs that have planned; wraps to zero by itself
    int pieces_max = 0;
    uint32_t wait_limit = uocr_b200::kWaitLimit;  // polls a tile wait may take (uocr_b200_workspace_set_wait_limit)
    uocr_b200::PrefillTile* tiles = nullptr;  // [max_rows] query-tile descriptors of the tensor-core prefill
    uocr_b200::TcWork* tile_work = nullptr;   // [max_rows] the same tiles, most key tiles first, with their key-tile counts
    int* item_counter = nullptr;   // items the persistent prefill grid has handed out beyond every CTA's first
    int plan_tiles = 0;            // tiles of the plan in tile_work (0: none)
    int plan_window = 0;
    bool plan_any_text = false;
    bool plan_scored = false;      // made for visible ranges (the call with modified scores)
    unsigned plan_serial = 0;      // plans made on this workspace so far
    int tiles_cap = 0;
    bool out_bf16 = false;  // attention results are written as bf16 instead of fp32
    bool timing = false;
    bool overlap = false;  // fused decode step may start its prologue before the preceding kernel ends
    cudaEvent_t ev0 = nullptr, ev1 = nullptr;
};

namespace uocr_b200 {

// A workspace (null: none) serves the device that it was made on; kernels of another one must not get its memory.
inline int check_workspace_device(const uocr_b200_workspace* ws, const char* who) {
    int dev = 0;
    CHECK_CUDA(cudaGetDevice(&dev), "cudaGetDevice");
    return ws && ws->device != dev ? fail(UOCR_B200_ERR_INVALID, std::string(who) + ": the workspace belongs to another device") : UOCR_B200_OK;
}

}  // namespace uocr_b200
