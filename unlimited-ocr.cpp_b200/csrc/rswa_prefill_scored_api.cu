// extern "C" entry points of the tensor-core prefill with modified scores.
#include <algorithm>
#include <cmath>

#include "rswa_paged.cuh"
#include "rswa_prefill_tc.cuh"
#include "rswa_workspace.cuh"

using namespace uocr_b200;

namespace {

template <bool CAP, bool BIAS, bool PAIR_Q, bool FINE_CAP>
int launch(const PrefillParams& pp, const PrefillMaps& maps, int grid, int device, cudaStream_t st) {
    auto kern = rswa_prefill_tc_kernel<TcMode<true, CAP, BIAS, PAIR_Q, FINE_CAP>>;
    static SmemLimit limit;  // one per instantiation
    CHECK_CUDA(limit.allow(kern, device, kTcSmemBytes), "prefill smem attribute");
    kern<<<grid, kTcThreads, kTcSmemBytes, st>>>(pp, maps);
    return after_launch("tensor-core prefill attention (modified scores)");
}

template <bool CAP, bool BIAS>
int launch_types(bool pair_q, bool fine_cap, const PrefillParams& pp, const PrefillMaps& maps, int grid, int device, cudaStream_t st) {
    if (!CAP || fine_cap)  // (without a cap the last argument says nothing)
        return pair_q ? launch<CAP, BIAS, true, true>(pp, maps, grid, device, st) : launch<CAP, BIAS, false, true>(pp, maps, grid, device, st);
    return pair_q ? launch<CAP, BIAS, true, !CAP>(pp, maps, grid, device, st) : launch<CAP, BIAS, false, !CAP>(pp, maps, grid, device, st);
}

// What this call takes of the modified scores.
int check_tc_score(const uocr_b200_score* score, const char* who) {
    if (int rc = check_score(score, kTcTile, who)) return rc;
    // the kernel's tanh is off by 2^-20 of the cap (2^-19 for bf16 results): a cap far above the scores would drown them
    if (score->softcap > 256.f) return fail(UOCR_B200_ERR_UNSUPPORTED, std::string(who) + ": softcap above 256 (use the calls for any geometry)");
    if (score->d_key_pos) return fail(UOCR_B200_ERR_UNSUPPORTED, std::string(who) + ": keys stand at their own index here (d_key_pos: use the calls for any geometry)");
    return UOCR_B200_OK;
}

}  // namespace

extern "C" {

int uocr_b200_rswa_prefill_plan_scored_tc(const uocr_b200_score* score, const uocr_b200_prefill_tile* h_tiles, int n_tiles,
                                          const int* d_prefill_len, int window, uocr_b200_workspace* ws, uocr_b200_stream_t stream) {
    if (int rc = check_tc_score(score, "prefill_plan_scored_tc")) return rc;
    const DeviceInfo* di = nullptr;
    if (ws) {
        if (int rc = device_info(&di)) return rc;
        if (int rc = check_workspace_device(ws, "prefill_plan_scored_tc")) return rc;
    }
    return prefill_plan(h_tiles, n_tiles, d_prefill_len, window, score, ws, reinterpret_cast<cudaStream_t>(stream), "prefill_plan_scored_tc");
}

int uocr_b200_rswa_prefill_attention_scored_tc(const uocr_b200_paged_kv* kv, const void* text_k_pool, const void* text_v_pool, int text_blocks,
                                               const uocr_b200_score* score, const void* q, int q_dtype, const int* d_prefill_len,
                                               const uocr_b200_prefill_tile* h_tiles, int n_tiles, int window, int heads, void* out,
                                               uocr_b200_workspace* ws, uocr_b200_stream_t stream) {
    const char* who = "prefill_attention_scored_tc";
    auto bad = [&](const char* what) { return fail(UOCR_B200_ERR_INVALID, std::string(who) + ": " + what); };
    if (n_tiles <= 0) return UOCR_B200_OK;
    PagedView pv;
    if (int rc = paged_view(kv, &pv)) return rc;
    if (kv->dtype != UOCR_B200_BF16 || kv->head_dim != kTcTile) return fail(UOCR_B200_ERR_UNSUPPORTED, std::string(who) + ": needs bf16 KV and head_dim 128");
    if (int rc = check_tc_score(score, who)) return rc;
    if (!q || !out || !d_prefill_len || !ws) return bad("null pointer");
    if (q_dtype != UOCR_B200_F32 && q_dtype != UOCR_B200_BF16) return fail(UOCR_B200_ERR_UNSUPPORTED, std::string(who) + ": q must be fp32 or bf16");
    if (!aligned16(q) || !aligned16(out)) return bad("q/out must be 16-byte aligned");
    if (heads <= 0 || heads % kv->kv_heads != 0) return bad("heads must be a multiple of kv_heads");
    if (window <= 0) return bad("window must be positive");
    if (text_k_pool && (!aligned16(text_k_pool) || !aligned16(text_v_pool))) return bad("the text pools must be 16-byte aligned");
    const DeviceInfo* di = nullptr;
    if (int rc = device_info(&di)) return rc;
    if (int rc = check_workspace_device(ws, who)) return rc;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (h_tiles) {
        if (int rc = prefill_plan(h_tiles, n_tiles, d_prefill_len, window, score, ws, st, who)) return rc;
    } else if (ws->plan_tiles != n_tiles || ws->plan_window != window || !ws->plan_scored) {
        return bad("no tiles given and the workspace holds no plan of this size and window made for modified scores");
    }
    const bool any_text = ws->plan_any_text;
    if (any_text && (!text_k_pool || !text_v_pool || text_blocks <= 0)) return bad("text tiles need the text pool");
    if (any_text && score->slopes && !score->d_q_pos) return bad("a distance bias on text rows needs d_q_pos");
    if ((long long)n_tiles * heads >= (1ll << 31)) return fail(UOCR_B200_ERR_UNSUPPORTED, std::string(who) + ": too many tiles");
    PrefillParams pp{};
    pp.q = static_cast<const float*>(q);
    pp.out = static_cast<float*>(out);
    pp.out_bf16 = ws->out_bf16 ? 1 : 0;
    pp.k_pool = pv.k_pool;
    pp.v_pool = pv.v_pool;
    pp.k_text = static_cast<const uint8_t*>(text_k_pool);
    pp.v_text = static_cast<const uint8_t*>(text_v_pool);
    pp.table = pv.table;
    pp.d_prefill_len = d_prefill_len;
    pp.tiles = ws->tiles;
    pp.work = ws->tile_work;
    pp.counter = ws->item_counter + 1;  // (the plain call has its own)
    pp.n_tiles = n_tiles;
    pp.table_stride = pv.table_stride;
    pp.num_blocks = pv.num_blocks;
    pp.text_blocks = text_blocks;
    pp.heads = heads;
    pp.kv_heads = kv->kv_heads;
    pp.group = heads / kv->kv_heads;
    pp.window = window;
    pp.status = ws->status;
    pp.wait_limit = ws->wait_limit;
    pp.d_lo = score->d_lo;
    pp.d_hi = score->d_hi;
    pp.d_q_pos = score->d_q_pos;
    pp.slopes = score->slopes;
    const double scale = score->scale != 0.f ? (double)score->scale : 1.0 / std::sqrt(128.0);
    const double log2e = 1.4426950408889634;
    pp.score_mul = (float)(score->softcap > 0.f ? 2.0 * log2e * scale / score->softcap : log2e * scale);
    pp.cap_log2 = (float)(score->softcap * log2e);
    PrefillMaps maps;
    if (int rc = make_kv_map(&maps.k, pv.k_pool, (long)kv->num_blocks * kv->kv_heads * kBlockTokens)) return rc;
    if (int rc = make_kv_map(&maps.v, pv.v_pool, (long)kv->num_blocks * kv->kv_heads * kBlockTokens)) return rc;
    if (any_text) {
        if (int rc = make_kv_map(&maps.tk, text_k_pool, (long)text_blocks * kv->kv_heads * kBlockTokens)) return rc;
        if (int rc = make_kv_map(&maps.tv, text_v_pool, (long)text_blocks * kv->kv_heads * kBlockTokens)) return rc;
    } else {  // never read: no text tile in this launch
        maps.tk = maps.k;
        maps.tv = maps.v;
    }
    const int grid = (int)std::min<long long>((long long)n_tiles * heads, di->sms);
    const bool pair_q = q_dtype == UOCR_B200_F32, fine_cap = !ws->out_bf16;
    const bool cap = score->softcap > 0.f, bias = score->slopes != nullptr;
    if (cap && bias) return launch_types<true, true>(pair_q, fine_cap, pp, maps, grid, ws->device, st);
    if (cap) return launch_types<true, false>(pair_q, fine_cap, pp, maps, grid, ws->device, st);
    if (bias) return launch_types<false, true>(pair_q, fine_cap, pp, maps, grid, ws->device, st);
    return launch_types<false, false>(pair_q, fine_cap, pp, maps, grid, ws->device, st);
}

}  // extern "C"
