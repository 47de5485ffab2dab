// extern "C" entry points of the rotary positions.
#include <cmath>
#include <new>

#include "rswa_rope.cuh"
#include "rswa_workspace.cuh"

using namespace uocr_b200;

struct uocr_b200_rope {
    unsigned long long turn[kRopeMaxPairs];
    float amplitude;
    int interleaved, rotary_dim;
};

namespace {

// Angle per position of every rotary pair, scaled for long contexts.
void rope_frequencies(const uocr_b200_rope_desc& d, long double* f) {
    const int r = d.rotary_dim;
    const long double pi = acosl(-1.0L), s = d.factor, L = d.orig_context;
    long double theta = d.theta;
    if (d.scaling == UOCR_B200_ROPE_BASE && r > 2) theta *= powl(s, (long double)r / (r - 2));
    long double first = 0, last = 0;
    if (d.scaling == UOCR_B200_ROPE_RAMP) {
        // the pair index at which a pair makes the given number of turns over the original context
        auto index = [&](long double turns) { return r * logl(L / (turns * 2 * pi)) / (2 * logl(theta)); };
        first = fmaxl(floorl(index(d.high)), 0.0L);
        last = fminl(ceill(index(d.low)), (long double)(r - 1));
        if (last == first) last += 0.001L;
    }
    for (int i = 0; i < r / 2; ++i) {
        f[i] = powl(theta, -2.0L * i / r);
        if (d.scaling == UOCR_B200_ROPE_LINEAR) {
            f[i] /= s;
        } else if (d.scaling == UOCR_B200_ROPE_RAMP) {
            const long double mix = fminl(fmaxl((i - first) / (last - first), 0.0L), 1.0L);
            f[i] = f[i] / s * mix + f[i] * (1 - mix);
        } else if (d.scaling == UOCR_B200_ROPE_BANDS) {
            const long double turns = L * f[i] / (2 * pi);
            const long double mix = fminl(fmaxl((turns - d.low) / ((long double)d.high - d.low), 0.0L), 1.0L);
            f[i] = f[i] / s * (1 - mix) + f[i] * mix;
        }
    }
}

template <typename ROW, typename KV, int MODE>
void launch_rope(RopeParams& p, bool interleaved, bool vec, int sms, cudaStream_t st) {
    const int half = p.rotary_dim / 2, hd = p.head_dim;
    if (!vec) {
        p.per_head = hd - half;
        p.items = (p.heads + p.kv_heads) * (hd - half) + (MODE == kRopeRows ? 0 : p.kv_heads * hd);
        const int grid = MODE == kRopeAppend || p.rows < sms * 64 ? p.rows : sms * 64;
        rswa_rope_elements_kernel<ROW, KV, MODE><<<grid, kRopeThreads, 0, st>>>(p, interleaved);
        return;
    }
    p.per_head = interleaved ? hd / 8 : (hd - half) / 8;
    // A warp takes a whole row while that still gives every SM 16 warps; fewer rows are cut finer, to one head (or 32 chunks) a lane.
    constexpr int warps = kRopeThreads / 32;
    static_assert(warps == 8, "append: the 8 warps of a CTA share its row");
    int log2 = MODE == kRopeAppend ? 3 : 0;
    const long long lanes = (long long)(p.heads + p.kv_heads) * p.per_head;
    if (MODE != kRopeAppend)
        while (((long long)p.rows << log2) < 2ll * sms * warps && (lanes >> log2) > 32) ++log2;
    p.parts_log2 = log2;
    const long long want = (((long long)p.rows << log2) + warps - 1) / warps;
    const int grid = MODE == kRopeAppend ? p.rows : (int)(want < (1 << 30) ? want : 1 << 30);
    if (interleaved) rswa_rope_kernel<ROW, KV, MODE, true><<<grid, kRopeThreads, 0, st>>>(p);
    else rswa_rope_kernel<ROW, KV, MODE, false><<<grid, kRopeThreads, 0, st>>>(p);
}

// Checks the rows, fills what every mode shares and launches.
template <int MODE>
int run_rope(RopeParams& p, const uocr_b200_rope* rope, const uocr_b200_qkv_rows* rows, int kv_dtype, const uocr_b200_workspace* ws, cudaStream_t st, const char* who) {
    auto bad = [&](const char* what) { return fail(UOCR_B200_ERR_INVALID, std::string(who) + ": " + what); };
    if (!rope || !rows || !p.d_positions) return bad("null pointer");
    if (rows->dtype != UOCR_B200_F32 && rows->dtype != UOCR_B200_BF16) return fail(UOCR_B200_ERR_UNSUPPORTED, std::string(who) + ": rows must be fp32 or bf16");
    if (rows->heads < 0 || p.kv_heads < 0 || rows->heads + p.kv_heads == 0 || rows->heads > 4096 || p.kv_heads > 4096) return bad("head counts must be in [0, 4096] and not both 0");
    if (p.head_dim < 2 || p.head_dim > 1024 || rope->rotary_dim > p.head_dim) return bad("head_dim must be in [2, 1024] and hold the rotated dims");
    if (rows->heads > 0 && (!rows->q || !rows->q_out)) return bad("null pointer");
    if (p.kv_heads > 0 && (!rows->k || (MODE == kRopeRows ? !p.k_out : !rows->v))) return bad("null pointer");
    const long long q_row = (long long)rows->heads * p.head_dim, kv_row = (long long)p.kv_heads * p.head_dim;
    if (rows->heads > 0 && (rows->q_stride < q_row || rows->q_out_stride < q_row)) return bad("a row stride is smaller than the row");
    if (p.kv_heads > 0 && (rows->k_stride < kv_row || (MODE == kRopeRows ? p.k_out_stride : rows->v_stride) < kv_row)) return bad("a row stride is smaller than the row");
    if (rows->heads > 0 && rows->q == rows->q_out && rows->q_stride != rows->q_out_stride) return bad("in place, the strides must be equal");
    if (MODE == kRopeRows && p.kv_heads > 0 && rows->k == p.k_out && rows->k_stride != p.k_out_stride) return bad("in place, the strides must be equal");
    const DeviceInfo* di = nullptr;
    if (int rc = device_info(&di)) return rc;
    if (int rc = check_workspace_device(ws, who)) return rc;
    p.status = ws ? ws->status : nullptr;

    for (int i = 0; i < kRopeMaxPairs; ++i) p.turn[i] = rope->turn[i];
    p.amplitude = rope->amplitude;
    const bool il = rope->interleaved != 0;
    p.rotary_dim = rope->rotary_dim;
    p.heads = rows->heads;
    p.q = rows->q;
    p.k = rows->k;
    p.v = rows->v;
    p.q_out = rows->q_out;
    p.q_stride = rows->q_stride;
    p.k_stride = rows->k_stride;
    p.v_stride = rows->v_stride;
    p.q_out_stride = rows->q_out_stride;

    // chunks of 8 elements: 16-byte aligned, and in the half layout wholly inside one half of the rotated dims
    const int elem = rows->dtype == UOCR_B200_BF16 ? 2 : 4;
    auto ok = [&](const void* ptr, long long stride) { return !ptr || (aligned16(ptr) && stride * elem % 16 == 0); };
    bool vec = p.head_dim % 8 == 0 && (il || p.rotary_dim % 16 == 0);
    if (rows->heads > 0) vec = vec && ok(p.q, p.q_stride) && ok(p.q_out, p.q_out_stride);
    if (p.kv_heads > 0) vec = vec && ok(p.k, p.k_stride) && (MODE == kRopeRows ? ok(p.k_out, p.k_out_stride) : ok(p.v, p.v_stride));
    const bool rb = rows->dtype == UOCR_B200_BF16, kb = kv_dtype == UOCR_B200_BF16;
    if constexpr (MODE == kRopeRows) {
        if (rb) launch_rope<BF16, BF16, MODE>(p, il, vec, di->sms, st);
        else launch_rope<F32, F32, MODE>(p, il, vec, di->sms, st);
    } else {
        if (rb && kb) launch_rope<BF16, BF16, MODE>(p, il, vec, di->sms, st);
        else if (rb) launch_rope<BF16, F32, MODE>(p, il, vec, di->sms, st);
        else if (kb) launch_rope<F32, BF16, MODE>(p, il, vec, di->sms, st);
        else launch_rope<F32, F32, MODE>(p, il, vec, di->sms, st);
    }
    return after_launch(who);
}

}  // namespace

extern "C" {

int uocr_b200_rope_create(const uocr_b200_rope_desc* d, uocr_b200_rope** out) {
    if (!d || !out) return fail(UOCR_B200_ERR_INVALID, "rope_create: null argument");
    if (d->layout != UOCR_B200_ROPE_HALF && d->layout != UOCR_B200_ROPE_INTERLEAVED) return fail(UOCR_B200_ERR_INVALID, "rope_create: unknown layout");
    if (d->rotary_dim < 2 || d->rotary_dim > 2 * kRopeMaxPairs || (d->rotary_dim & 1)) return fail(UOCR_B200_ERR_UNSUPPORTED, "rope_create: rotary_dim must be even and in [2, 256]");
    if (d->scaling < UOCR_B200_ROPE_NONE || d->scaling > UOCR_B200_ROPE_BANDS) return fail(UOCR_B200_ERR_INVALID, "rope_create: unknown scaling");
    if (!(d->theta > 0.f) || !std::isfinite(d->theta)) return fail(UOCR_B200_ERR_INVALID, "rope_create: theta must be positive");
    if (!(d->amplitude > 0.f) || !std::isfinite(d->amplitude)) return fail(UOCR_B200_ERR_INVALID, "rope_create: amplitude must be positive");
    if (d->scaling != UOCR_B200_ROPE_NONE && (!(d->factor > 0.f) || !std::isfinite(d->factor))) return fail(UOCR_B200_ERR_INVALID, "rope_create: factor must be positive");
    if (d->scaling == UOCR_B200_ROPE_RAMP || d->scaling == UOCR_B200_ROPE_BANDS) {
        if (!(d->orig_context > 0.f) || !std::isfinite(d->orig_context) || !(d->low > 0.f) || !(d->high > d->low) || !std::isfinite(d->high))
            return fail(UOCR_B200_ERR_INVALID, "rope_create: orig_context must be positive and 0 < low < high");
        if (d->scaling == UOCR_B200_ROPE_RAMP && !(d->theta > 1.f)) return fail(UOCR_B200_ERR_INVALID, "rope_create: the ramp needs theta > 1");
    }
    auto* r = new (std::nothrow) uocr_b200_rope;
    if (!r) return fail(UOCR_B200_ERR_EXHAUSTED, "rope_create: out of host memory");
    long double f[kRopeMaxPairs] = {};
    rope_frequencies(*d, f);
    const long double two_pi = 2 * acosl(-1.0L);
    for (int i = 0; i < kRopeMaxPairs; ++i) {
        r->turn[i] = 0;
        if (i >= d->rotary_dim / 2) continue;
        if (!std::isfinite(f[i])) {
            delete r;
            return fail(UOCR_B200_ERR_INVALID, "rope_create: a frequency is not finite");
        }
        const long double turns = f[i] / two_pi;
        const long double part = ldexpl(turns - floorl(turns), 64);
        r->turn[i] = part >= 18446744073709551615.0L ? 0ull : (unsigned long long)llrintl(part - 9223372036854775808.0L) + 9223372036854775808ull;
    }
    r->amplitude = d->amplitude;
    r->interleaved = d->layout == UOCR_B200_ROPE_INTERLEAVED ? 1 : 0;
    r->rotary_dim = d->rotary_dim;
    *out = r;
    return UOCR_B200_OK;
}

int uocr_b200_rope_destroy(uocr_b200_rope* rope) {
    delete rope;
    return UOCR_B200_OK;
}

int uocr_b200_rswa_rope_rows(const uocr_b200_rope* rope, const uocr_b200_qkv_rows* rows, void* k_out, int64_t k_out_stride,
                             const int* d_positions, int total, int kv_heads, int head_dim, uocr_b200_stream_t stream) {
    if (total <= 0) return UOCR_B200_OK;
    RopeParams p{};
    p.rows = total;
    p.kv_heads = kv_heads;
    p.head_dim = head_dim;
    p.k_out = k_out;
    p.k_out_stride = k_out_stride;
    p.d_positions = d_positions;
    return run_rope<kRopeRows>(p, rope, rows, UOCR_B200_F32, nullptr, reinterpret_cast<cudaStream_t>(stream), "rope_rows");
}

int uocr_b200_rswa_rope_write_prefill_paged(const uocr_b200_paged_kv* kv, const uocr_b200_rope* rope, const uocr_b200_qkv_rows* rows,
                                            const int* d_positions, const int* d_slots, const int* d_pos, int total,
                                            uocr_b200_workspace* ws, uocr_b200_stream_t stream) {
    if (total <= 0) return UOCR_B200_OK;
    RopeParams p{};
    if (int rc = paged_view(kv, &p.pv)) return rc;
    if (!d_slots || !d_pos) return fail(UOCR_B200_ERR_INVALID, "rope_write_prefill_paged: null pointer");
    p.rows = total;
    p.kv_heads = kv->kv_heads;
    p.head_dim = kv->head_dim;
    p.d_positions = d_positions;
    p.d_slots = d_slots;
    p.d_pos = d_pos;
    return run_rope<kRopeWrite>(p, rope, rows, kv->dtype, ws, reinterpret_cast<cudaStream_t>(stream), "rope_write_prefill_paged");
}

int uocr_b200_rswa_rope_append_decode_batch_paged(const uocr_b200_paged_kv* kv, const uocr_b200_rope* rope, const uocr_b200_qkv_rows* rows,
                                                  const int* d_positions, int* d_len, int* d_ring_pos, const int* d_prefill_len,
                                                  const int* d_slots, int batch, int window, uocr_b200_workspace* ws,
                                                  uocr_b200_stream_t stream) {
    if (batch <= 0) return UOCR_B200_OK;
    RopeParams p{};
    if (int rc = paged_view(kv, &p.pv)) return rc;
    if (!d_len || !d_ring_pos || !d_prefill_len || !d_slots) return fail(UOCR_B200_ERR_INVALID, "rope_append_decode_batch_paged: null pointer");
    if (window <= 0) return fail(UOCR_B200_ERR_INVALID, "rope_append_decode_batch_paged: window must be positive");
    p.rows = batch;
    p.kv_heads = kv->kv_heads;
    p.head_dim = kv->head_dim;
    p.d_positions = d_positions;
    p.d_slots = d_slots;
    p.d_len = d_len;
    p.d_ring_pos = d_ring_pos;
    p.d_prefill_len = d_prefill_len;
    p.window = window;
    return run_rope<kRopeAppend>(p, rope, rows, kv->dtype, ws, reinterpret_cast<cudaStream_t>(stream), "rope_append_decode_batch_paged");
}

}  // extern "C"
