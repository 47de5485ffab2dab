// extern "C" entry points of the attention with modified scores (any geometry): argument checks, dispatch, launches.
#include <cmath>

#include "rswa_scored.cuh"
#include "rswa_workspace.cuh"

using namespace uocr_b200;

namespace {

template <typename C, int HD>
int launch_scored(ScoreParams& p, const DeviceInfo& di, const uocr_b200_workspace* ws, cudaStream_t st) {
    constexpr int per_warp = kScoreRing * C::kTile;
    const int plan_bytes = p.rows <= kScoreSharedRows ? (int)(sizeof(ScoreRow) * p.rows + sizeof(long long) * (p.rows + 1 + 32)) : 0;
    const int budget = di.smem_optin < 200 * 1024 ? di.smem_optin : 200 * 1024;
    int warps = (budget - 1024 - plan_bytes) / per_warp;
    if (warps > C::kThreads / 32) warps = C::kThreads / 32;
    if (warps < 1) return fail(UOCR_B200_ERR_UNSUPPORTED, "attention_scored: tile does not fit in shared memory");
    p.total_warps = di.sms * warps;
    if (p.total_warps > ws->total_warps_max) return fail(UOCR_B200_ERR_WORKSPACE, "attention_scored: workspace built for a smaller device");
    const int smem = ((warps * kScoreRing * 8 + 127) & ~127) + warps * per_warp + plan_bytes;
    auto kern = rswa_scored_kernel<C, HD>;
    static SmemLimit limit;  // one per instantiation
    CHECK_CUDA(limit.allow(kern, ws->device, budget), "smem attribute");
    kern<<<di.sms, warps * 32, smem, st>>>(p);
    return after_launch("attention with modified scores");
}

template <typename KV, int HD>
int dispatch_group(int g, ScoreParams& p, const DeviceInfo& di, const uocr_b200_workspace* ws, cudaStream_t st) {
    // Four heads of a bf16 cache go to the tensor cores: 24 sequences, 4 KV heads, 300 MB of cache take 70 us (head_dim 128) and 83 (64),
    // 90 and 109 on the CUDA cores; 16 + 4 heads of 128 over 144 000 tokens with a bias 72 and 155.  Two heads do not fill the
    // columns and stay on the CUDA cores: 66 and 71 us, on the tensor cores 70 and 87.
    if constexpr (KV::kBytes == 2 && (HD == 64 || HD == 128)) {
        if (g == 4) return launch_scored<ScoreMma<HD>, HD>(p, di, ws, st);
    } else if constexpr (4 * HD <= kPartElems) {
        if (g == 4) return launch_scored<ScoreFma<KV, HD, 4>, HD>(p, di, ws, st);
    }
    if (g == 2) return launch_scored<ScoreFma<KV, HD, 2>, HD>(p, di, ws, st);
    return launch_scored<ScoreFma<KV, HD, 1>, HD>(p, di, ws, st);
}

template <typename KV>
int dispatch_head_dim(int hd, int g, ScoreParams& p, const DeviceInfo& di, const uocr_b200_workspace* ws, cudaStream_t st) {
    switch (hd) {
        case 4:
            if constexpr (KV::kBytes == 4) return dispatch_group<KV, 4>(g, p, di, ws, st);
            break;
        case 8: return dispatch_group<KV, 8>(g, p, di, ws, st);
        case 16: return dispatch_group<KV, 16>(g, p, di, ws, st);
        case 32: return dispatch_group<KV, 32>(g, p, di, ws, st);
        case 64: return dispatch_group<KV, 64>(g, p, di, ws, st);
        case 128: return dispatch_group<KV, 128>(g, p, di, ws, st);
        case 256: return dispatch_group<KV, 256>(g, p, di, ws, st);
        default: break;
    }
    return fail(UOCR_B200_ERR_UNSUPPORTED, "attention_scored: head_dim must be a power of two in [8,256] (bf16) or [4,256] (fp32)");
}

struct TextPool {
    const void* k = nullptr;
    const void* v = nullptr;
    int blocks = 0;
};

int run_scored(const uocr_b200_paged_kv* kv, const uocr_b200_score* score, const void* q, int q_dtype, ScorePlan& plan, const TextPool& text,
               int heads, void* out, const uocr_b200_mass* mass, uocr_b200_workspace* ws, cudaStream_t st, const char* who) {
    auto bad = [&](const char* what) { return fail(UOCR_B200_ERR_INVALID, std::string(who) + ": " + what); };
    PagedView pv;
    if (int rc = paged_view(kv, &pv)) return rc;
    if (int rc = check_score(score, kv->head_dim, who)) return rc;
    if (!q || !out || !ws || !plan.d_slots || !plan.d_prefill_len) return bad("null pointer");
    if (q_dtype != UOCR_B200_F32 && q_dtype != UOCR_B200_BF16) return fail(UOCR_B200_ERR_UNSUPPORTED, std::string(who) + ": q must be fp32 or bf16");
    if (heads <= 0 || heads % kv->kv_heads != 0) return bad("heads must be a positive multiple of kv_heads");
    if (!aligned16(q) || !aligned16(out)) return bad("q/out must be 16-byte aligned");
    if (score->d_key_pos && score->key_pos_stride <= 0) return bad("key_pos_stride must be positive");
    if (score->slopes && plan.mode != kScoreRagged && !score->d_q_pos) return bad("a distance bias needs d_q_pos");
    if (plan.rows > ws->max_rows) return fail(UOCR_B200_ERR_WORKSPACE, std::string(who) + ": more rows than the workspace was created for");
    if ((long long)plan.rows * heads >= (1ll << 31) || (long long)kv->num_blocks * kv->kv_heads >= (1ll << 32) ||
        (long long)text.blocks * kv->kv_heads >= (1ll << 32) || text.blocks > kScoreTextBlocks)
        return fail(UOCR_B200_ERR_UNSUPPORTED, std::string(who) + ": rows * heads or a pool is too large");
    size_t score_bytes = 0;
    if (mass) {
        if (!mass->mass_out || !mass->scratch) return bad("null pointer in the mass");
        if (mass->stride <= 0 || !(mass->decay >= 0.f) || !std::isfinite(mass->decay)) return bad("the mass needs a positive stride and a finite decay >= 0");
        if (!aligned16(mass->scratch)) return bad("the mass scratch must be 16-byte aligned");
        if (plan.rows > 65535) return fail(UOCR_B200_ERR_UNSUPPORTED, std::string(who) + ": at most 65535 rows with attention weights");
        score_bytes = (sizeof(float) * (size_t)plan.rows * heads * mass->stride + 15) & ~size_t(15);
        if (mass->scratch_bytes < uocr_b200_rswa_mass_scratch_bytes(plan.rows, heads, mass->stride))
            return fail(UOCR_B200_ERR_WORKSPACE, std::string(who) + ": the mass scratch is too small");
    }
    const DeviceInfo* di = nullptr;
    if (int rc = device_info(&di)) return rc;
    if (int rc = check_workspace_device(ws, who)) return rc;

    const int group = heads / kv->kv_heads;
    // Heads of a group that share a pass over its tiles: as many of 4, 2, 1 as divide the group and fit a partial.  (Also where the
    // wider ones spill registers: 24 sequences, 300 MB of cache, a group of four by 4 / 2 / 1: fp32 x 128 86, 95, 169 us; fp32 x 64
    // 68, 108, 183; fp32 x 32 82, 106, 156; bf16 x 32 160, 195, 297; bf16 x 16 252, 321, 519.)
    int g = group % 4 == 0 ? 4 : group % 2 == 0 ? 2 : 1;
    while (g > 1 && g * kv->head_dim > kPartElems) g /= 2;

    plan.items_per_row = heads / g;
    plan.d_lo = score->d_lo;
    plan.d_hi = score->d_hi;
    plan.d_q_pos = score->slopes ? score->d_q_pos : nullptr;
    plan.out = static_cast<uint32_t*>(out);
    plan.out_row_words = heads * kv->head_dim / (ws->out_bf16 ? 2 : 1);

    ScoreParams p{};
    p.plan = plan;
    p.q = q;
    p.q_bf16 = q_dtype == UOCR_B200_BF16 ? 1 : 0;
    p.out = out;
    p.out_bf16 = ws->out_bf16 ? 1 : 0;
    p.k_base = pv.k_pool;
    p.v_base = pv.v_pool;
    p.k_text = static_cast<const uint8_t*>(text.k);
    p.v_text = static_cast<const uint8_t*>(text.v);
    p.text_blocks = text.blocks;
    p.table = pv.table;
    p.table_stride = pv.table_stride;
    p.num_blocks = pv.num_blocks;
    p.rows = plan.rows;
    p.heads = heads;
    p.kv_heads = kv->kv_heads;
    p.group = group;
    const double scale = score->scale != 0.f ? (double)score->scale : 1.0 / std::sqrt((double)kv->head_dim);
    const double log2e = 1.4426950408889634;
    p.q_scale = (float)(score->softcap > 0.f ? scale / score->softcap : scale * log2e);
    p.cap_log2 = (float)(score->softcap * log2e);
    p.slopes = score->slopes;
    p.d_key_pos = score->d_key_pos;
    p.key_pos_stride = score->key_pos_stride;
    if (mass) {
        p.scores = static_cast<float*>(mass->scratch);
        p.score_ml = reinterpret_cast<float*>(static_cast<uint8_t*>(mass->scratch) + score_bytes);
        p.score_stride = mass->stride;
    }
    p.info = ws->score_rows;
    p.rs = ws->score_rs;
    p.part_acc = ws->part_acc;
    p.part_ml = ws->part_ml;
    static_assert(kScoreJoin == kScoreJoinWidth, "the workspace holds the counters of this tree");
    p.counters = ws->score_counters;
    p.pieces = ws->pieces_max;
    p.status = ws->status;
    p.wait_limit = ws->wait_limit;

    if (p.rows > kScoreSharedRows) {
        rswa_scored_plan_kernel<<<1, 1024, 0, st>>>(plan, ws->score_rows, ws->score_rs);
        if (int rc = after_launch("plan (modified scores)")) return rc;
    }
    if (int rc = kv->dtype == UOCR_B200_BF16 ? dispatch_head_dim<BF16>(kv->head_dim, g, p, *di, ws, st)
                                             : dispatch_head_dim<F32>(kv->head_dim, g, p, *di, ws, st))
        return rc;
    if (mass) {
        MassParams mp{};
        mp.plan = plan;
        mp.heads = heads;
        mp.scores = p.scores;
        mp.score_ml = p.score_ml;
        mp.mass_in = mass->mass_in;
        mp.mass_out = mass->mass_out;
        mp.stride = mass->stride;
        mp.decay = mass->decay;
        mp.status = ws->status;
        CHECK_CUDA(launch_after(rswa_mass_kernel, dim3((mass->stride + kMassThreads - 1) / kMassThreads, plan.rows), kMassThreads, 0, st, mp), "attention weights");
        return after_launch("attention weights");
    }
    return UOCR_B200_OK;
}

}  // namespace

namespace uocr_b200 {

int check_score(const uocr_b200_score* score, int head_dim, const char* who) {
    auto bad = [&](const char* what) { return fail(UOCR_B200_ERR_INVALID, std::string(who) + ": " + what); };
    if (!score) return bad("null pointer");
    if (!(score->softcap == 0.f || (score->softcap >= 1e-6f && score->softcap <= 1e30f))) return bad("softcap must be 0 (none) or in [1e-6, 1e30]");
    if (!std::isfinite(score->scale)) return bad("scale must be finite (0: 1/sqrt(head_dim))");
    // what q is multiplied by on the way into the log2 domain, twice of it at most
    const double scale = score->scale != 0.f ? (double)score->scale : 1.0 / std::sqrt((double)head_dim);
    if (!std::isfinite((float)(2 * 1.4426950408889634 * scale / (score->softcap > 0.f ? std::fmin(score->softcap, 1.f) : 1.f)))) return bad("scale (over softcap) overflows fp32");
    return UOCR_B200_OK;
}

}  // namespace uocr_b200

extern "C" {

size_t uocr_b200_rswa_mass_scratch_bytes(int batch, int heads, int stride) {
    if (batch <= 0 || heads <= 0 || stride <= 0) return 0;
    const size_t rows = (size_t)batch * heads;
    return ((sizeof(float) * rows * stride + 15) & ~size_t(15)) + 2 * sizeof(float) * rows;
}

int uocr_b200_rswa_attention_scored_batch_paged(const uocr_b200_paged_kv* kv, const uocr_b200_score* score, const void* q, int q_dtype,
                                                const int* d_len, const int* d_ring_pos, const int* d_prefill_len, const int* d_slots,
                                                int batch, int window, int heads, void* out, const uocr_b200_mass* mass,
                                                uocr_b200_workspace* ws, uocr_b200_stream_t stream) {
    if (batch <= 0) return UOCR_B200_OK;
    if (!d_len || !d_ring_pos) return fail(UOCR_B200_ERR_INVALID, "attention_scored_batch_paged: null pointer");
    if (window <= 0) return fail(UOCR_B200_ERR_INVALID, "attention_scored_batch_paged: window must be positive");
    ScorePlan plan{};
    plan.mode = kScoreDecode;
    plan.rows = batch;
    plan.window = window;
    plan.d_slots = d_slots;
    plan.d_len = d_len;
    plan.d_ring_pos = d_ring_pos;
    plan.d_prefill_len = d_prefill_len;
    return run_scored(kv, score, q, q_dtype, plan, TextPool{}, heads, out, mass, ws, reinterpret_cast<cudaStream_t>(stream), "attention_scored_batch_paged");
}

int uocr_b200_rswa_attention_scored_ragged_paged(const uocr_b200_paged_kv* kv, const uocr_b200_score* score, const void* q, int q_dtype,
                                                 const int* d_prefill_len, const int* d_slots, const int* d_pos, int total, int heads,
                                                 void* out, uocr_b200_workspace* ws, uocr_b200_stream_t stream) {
    if (total <= 0) return UOCR_B200_OK;
    if (!d_pos) return fail(UOCR_B200_ERR_INVALID, "attention_scored_ragged_paged: null pointer");
    ScorePlan plan{};
    plan.mode = kScoreRagged;
    plan.rows = total;
    plan.window = 1;
    plan.d_slots = d_slots;
    plan.d_pos = d_pos;
    plan.d_prefill_len = d_prefill_len;
    return run_scored(kv, score, q, q_dtype, plan, TextPool{}, heads, out, nullptr, ws, reinterpret_cast<cudaStream_t>(stream), "attention_scored_ragged_paged");
}

int uocr_b200_rswa_prefill_text_scored_paged(const uocr_b200_paged_kv* kv, const void* text_k_pool, const void* text_v_pool, int text_blocks,
                                               const uocr_b200_score* score, const void* q, int q_dtype, const int* d_prefill_len,
                                               const int* d_slots, const int* d_pos, const int* d_text_block0, int total, int window, int heads,
                                               void* out, uocr_b200_workspace* ws, uocr_b200_stream_t stream) {
    if (total <= 0) return UOCR_B200_OK;
    if (!text_k_pool || !text_v_pool || text_blocks <= 0 || !d_pos || !d_text_block0) return fail(UOCR_B200_ERR_INVALID, "prefill_text_scored_paged: null pointer");
    if (!aligned16(text_k_pool) || !aligned16(text_v_pool)) return fail(UOCR_B200_ERR_INVALID, "prefill_text_scored_paged: the text pools must be 16-byte aligned");
    if (window <= 0) return fail(UOCR_B200_ERR_INVALID, "prefill_text_scored_paged: window must be positive");
    ScorePlan plan{};
    plan.mode = kScoreText;
    plan.rows = total;
    plan.window = window;
    plan.d_slots = d_slots;
    plan.d_pos = d_pos;
    plan.d_prefill_len = d_prefill_len;
    plan.d_text_block0 = d_text_block0;
    return run_scored(kv, score, q, q_dtype, plan, TextPool{text_k_pool, text_v_pool, text_blocks}, heads, out, nullptr, ws,
                      reinterpret_cast<cudaStream_t>(stream), "prefill_text_scored_paged");
}

}  // extern "C"
