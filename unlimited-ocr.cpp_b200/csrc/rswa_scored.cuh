// Split-KV attention with modified scores over the paged R-SWA cache: a tanh cap, a bias that grows with
// the distance, and a visible range of the fixed region per row (pages, documents, prefixes).
//
//   x = scale * q.k;   x <- cap * tanh(x / cap);   x <- x - slope_h * |pos_q - pos_k|;   softmax over the
//   visible keys;   out = sum of the weights times v, 0 for a row that sees nothing.
//
// The work model is that of the plain attention kernel: the 16-token tiles a row's heads can see are laid
// out on one line and cut into equal pieces, one per warp of a persistent grid, so a batch of one long
// sequence and a batch of many short ones load the SMs alike; a warp streams its piece's K and V tiles
// through a private ring of shared memory with bulk copies, and the partial results (maximum, sum,
// accumulator) of an item that straddles pieces are joined by the warps that finish last.  What differs:
//   - an item is a row and up to four query heads of one KV head (G): a group of two or four reads a tile once, one of eight twice
//     (115 us where one of four takes 70), an odd one as often as it has heads; four heads of a bf16 cache of head_dim 64 or 128 run
//     their products on the tensor cores;
//   - only tiles that hold a visible token are on the line: the cost of a page is the page;
//   - the line is planned by every CTA in its own shared memory when the rows fit (one launch), else by
//     rswa_scored_plan_kernel;
//   - scores are modified one token per lane pair, after the reduction of the dot products, so the cap's
//     tanh costs one call per token and head, not per element;
//   - with attention weights asked for, the modified scores of the fixed region go to scratch (4 bytes per
//     token and head, against 2 * head_dim * 2 bytes of K and V) and rswa_mass_kernel turns them into
//     weights once the row's maximum and sum are known -- in a fixed order, without atomics.
// Statistics, scores and accumulators are fp32; keys and values outside the visible range are never
// multiplied, whatever they hold.  Bound by HBM for batches: 64 sequences on the pages of a shared document (10 heads of 128,
// bf16, 307 MB) take 54 us, 5.7 TB/s; by the latency of planning, one tile and two joins for one short sequence (273 + 128
// tokens: 10.5 us).
#pragma once

#include "rswa_paged.cuh"
#include "rswa_split.cuh"

namespace uocr_b200 {

enum ScoreMode : int { kScoreDecode = 0, kScoreRagged = 1, kScoreText = 2 };

// What one row attends: tokens [lo, hi) of the fixed region, then `ring` tokens of its ring (table entries
// from ring_entry) or of the text pool (from block text >> 4, the first text & 15 tokens of it skipped).
struct ScoreRow {
    int slot, lo, hi;
    int ring_entry;
    int ring;
    int text;  // -1: ring
    int age0;  // distance of token 0 of the first ring / text block; the distance of token t is age0 - t (+ window if negative)
    int q_pos;
};
static_assert(sizeof(ScoreRow) == 32, "the workspace reserves 32 bytes a row");

struct ScorePlan {
    int mode, rows, items_per_row, window;
    const int* d_slots;
    const int* d_len;
    const int* d_ring_pos;
    const int* d_prefill_len;
    const int* d_pos;
    const int* d_text_block0;
    const int* d_lo;
    const int* d_hi;
    const int* d_q_pos;
    uint32_t* out;  // rows without a visible key are zero-filled here
    int out_row_words;
};

struct ScoreParams {
    ScorePlan plan;
    const void* q;
    int q_bf16;
    void* out;
    int out_bf16;
    const uint8_t* k_base;
    const uint8_t* v_base;
    const uint8_t* k_text;
    const uint8_t* v_text;
    int text_blocks;
    const int32_t* table;
    int table_stride, num_blocks;
    int rows, heads, kv_heads, group;
    float q_scale;   // what q is multiplied by: scale / cap with a cap, scale * log2(e) without
    float cap_log2;  // cap * log2(e); 0: none
    const float* slopes;
    const int* d_key_pos;
    int key_pos_stride;
    float* scores;  // attention weights asked for: [rows * heads][score_stride] modified scores (log2 domain), then [rows * heads][2] (max, 1 / sum)
    float* score_ml;
    int score_stride;
    ScoreRow* info;  // plan in global memory (rows beyond kScoreSharedRows)
    long long* rs;
    float* part_acc;  // [2 * pieces][G * head_dim]
    float* part_ml;   // [2 * pieces][2 G]
    int* counters;  // [2 kScoreJoinLevels][pieces] arrival counters of the joins, zero between launches
    int pieces;
    int* status;
    uint32_t wait_limit;
    int total_warps;
};

constexpr int kScoreJoin = 8;  // partials joined at a time
constexpr int kScoreTextBlocks = (1 << 27) - 1;  // more blocks than a text pool may have

constexpr int kScoreSharedRows = 512;  // rows a CTA plans in its own shared memory

// Clamped visible range of row r in a fixed region whose first `fixed` tokens are in the cache.
__device__ __forceinline__ void score_range(const int* d_lo, const int* d_hi, int r, int fixed, int def_hi, int& lo, int& hi) {
    hi = min(d_hi ? __ldg(d_hi + r) : def_hi, fixed);
    lo = max(d_lo ? __ldg(d_lo + r) : 0, 0);
    if (hi <= lo) lo = hi = 0;
}

__device__ __forceinline__ int score_ring_tiles(const ScoreRow& o) {
    const int skip = o.text >= 0 ? o.text & 15 : 0;
    return o.ring > 0 ? (skip + o.ring + kBlockTokens - 1) / kBlockTokens : 0;
}

__device__ __forceinline__ int score_plan_row(const ScorePlan& p, int r, ScoreRow& o) {
    const int slot = __ldg(p.d_slots + r);
    const int pfx = max(__ldg(p.d_prefill_len + slot), 0);
    o.slot = slot;
    o.ring_entry = (pfx + kBlockTokens - 1) / kBlockTokens;
    o.ring = 0;
    o.text = -1;
    o.age0 = 0;
    o.q_pos = 0;
    int skip = 0;
    if (p.mode == kScoreDecode) {
        const int len = max(__ldg(p.d_len + slot), 0);
        score_range(p.d_lo, p.d_hi, r, min(len, pfx), pfx, o.lo, o.hi);
        o.ring = min(max(len - pfx, 0), p.window);
        if (p.d_q_pos) o.q_pos = __ldg(p.d_q_pos + r);
        // the newest ring token: the last one written before the window filled, the one behind the cursor after
        const int cursor = __ldg(p.d_ring_pos + slot);
        o.age0 = o.ring < p.window ? o.ring - 1 : (cursor > 0 ? cursor : p.window) - 1;
    } else if (p.mode == kScoreRagged) {
        const int pos = __ldg(p.d_pos + r);
        score_range(p.d_lo, p.d_hi, r, pfx, pos + 1, o.lo, o.hi);
        o.q_pos = p.d_q_pos ? __ldg(p.d_q_pos + r) : pos;
    } else {
        const int pos = __ldg(p.d_pos + r);
        score_range(p.d_lo, p.d_hi, r, pfx, pfx, o.lo, o.hi);
        const int first = max(0, pos - p.window + 1);
        skip = first & (kBlockTokens - 1);
        o.ring = max(pos - first + 1, 0);
        const long long blk = (long long)__ldg(p.d_text_block0 + r) + first / kBlockTokens;
        o.text = (int)(blk < 0 || blk >= kScoreTextBlocks ? kScoreTextBlocks : blk) << 4 | skip;  // (a block outside the pool is reported when it is read)
        o.age0 = pos - (first - skip);
        if (p.d_q_pos) o.q_pos = __ldg(p.d_q_pos + r);
    }
    const int fixed_tiles = o.hi > o.lo ? (o.hi + kBlockTokens - 1) / kBlockTokens - o.lo / kBlockTokens : 0;
    return fixed_tiles + score_ring_tiles(o);
}

__device__ __forceinline__ void score_zero_row(const ScorePlan& p, int r) {
    for (int i = 0; i < p.out_row_words; ++i) p.out[(size_t)r * p.out_row_words + i] = 0u;
}

__device__ __forceinline__ long long warp_inclusive_sum(long long v, int lane) {
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const long long t = __shfl_up_sync(0xffffffffu, v, d);
        if (lane >= d) v += t;
    }
    return v;
}

// info[0..rows) and the prefix sum of the rows' units (rs[0..rows]), by one warp for up to 32 rows.
__device__ __forceinline__ void score_plan_warp(const ScorePlan& p, ScoreRow* info, long long* rs, bool zero_rows, int lane) {
    long long units = 0;
    if (lane < p.rows) {
        ScoreRow o;
        units = (long long)score_plan_row(p, lane, o) * p.items_per_row;
        info[lane] = o;
        if (units == 0 && zero_rows) score_zero_row(p, lane);
    }
    const long long incl = warp_inclusive_sum(units, lane);
    if (lane < p.rows) rs[lane + 1] = incl;
    if (lane == 0) rs[0] = 0;
}

// The same for any number of rows, block-wide.  `scratch`: 32 long longs of shared memory.
__device__ __forceinline__ void score_plan_rows(const ScorePlan& p, ScoreRow* info, long long* rs, long long* scratch, bool zero_rows) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nthreads = blockDim.x;
    long long carry = 0;
    for (int base = 0; base < p.rows; base += nthreads) {
        const int r = base + tid;
        long long units = 0;
        if (r < p.rows) {
            ScoreRow o;
            units = (long long)score_plan_row(p, r, o) * p.items_per_row;
            info[r] = o;
            if (units == 0 && zero_rows) score_zero_row(p, r);
        }
        const long long incl = warp_inclusive_sum(units, lane);
        if (lane == 31) scratch[warp] = incl;
        __syncthreads();
        const long long sums = warp_inclusive_sum(lane < (nthreads >> 5) ? scratch[lane] : 0, lane);
        const long long before = warp > 0 ? __shfl_sync(0xffffffffu, sums, warp - 1) : 0;
        if (r < p.rows) rs[r] = carry + before + incl - units;
        carry += __shfl_sync(0xffffffffu, sums, 31);
        __syncthreads();
    }
    if (tid == 0) rs[p.rows] = carry;
}

// 64-bit divisions cost hundreds of cycles and are taken only where 32 bits do not hold the operands.
__device__ __forceinline__ long long div_units(long long a, long long b) {
    return ((unsigned long long)a | (unsigned long long)b) >> 32 ? a / b : (long long)((uint32_t)a / (uint32_t)b);
}
// The unit line [0, total) cut into ns pieces of equal length, but for one unit: piece k begins at floor(k total / ns).
struct ScorePieces {
    long long total, each;
    int ns, rest;  // total = each * ns + rest
    __device__ __forceinline__ ScorePieces(long long n, int total_warps) {
        total = n;
        ns = (int)min((long long)total_warps, total);
        each = div_units(total, ns);
        rest = (int)(total - each * ns);
    }
    __device__ __forceinline__ long long start(int k) const { return k * each + (uint32_t)(k * rest) / (uint32_t)ns; }  // (at most 4096 pieces)
    __device__ __forceinline__ int of(long long u) const { return (int)div_units((u + 1) * ns - 1, total); }
};

__global__ void __launch_bounds__(1024) rswa_scored_plan_kernel(ScorePlan p, ScoreRow* info, long long* rs) {
    __shared__ long long scratch[32];
    score_plan_rows(p, info, rs, scratch, true);
}

// Descriptor bits of a unit (one 16-token tile of an item).
constexpr uint32_t kSuValid = 0x1f;        // bits 0-4: tokens [skip, valid) are visible
constexpr int kSuSkipShift = 5;            // bits 5-8
constexpr uint32_t kSuLast = 1u << 9;
constexpr uint32_t kSuFirst = 1u << 10;
constexpr uint32_t kSuFixed = 1u << 11;    // tile of the fixed region
constexpr uint32_t kSuText = 1u << 12;     // tile of the text pool

constexpr int kScoreRing = 2;              // tile slots per warp
constexpr int kScoreThreads = 512;

// The item (row, head group) a warp is working on, as both consumers below need it.
struct ScoreItem {
    uint32_t index;  // row * items_per_row + group
    int slot, q_pos;
};

__device__ __forceinline__ float score_distance(const ScoreParams& p, const ScoreItem& it, uint32_t meta, int tok0, int t, bool visible) {
    if (meta & kSuFixed) {
        int at = tok0 + t;
        if (p.d_key_pos && visible && at < p.key_pos_stride) at = __ldg(p.d_key_pos + (size_t)it.slot * p.key_pos_stride + at);
        return __uint2float_rn((uint32_t)max(it.q_pos, at) - (uint32_t)min(it.q_pos, at));
    }
    const int a = tok0 - t;
    return (float)(a < 0 ? a + p.plan.window : a);
}

// x = q.k times q_scale -> the modified score in the log2 domain
__device__ __forceinline__ float score_modify(const ScoreParams& p, float x, float slope, float dist) {
    if (p.cap_log2 > 0.f) x = p.cap_log2 * tanhf(x);
    if (p.slopes) x = fmaf(-slope, dist, x);
    return x;
}

__device__ __forceinline__ void score_record(const ScoreParams& p, size_t head_row, int at, float x) {
    if (at < p.score_stride) __stcs(p.scores + head_row * p.score_stride + at, x);
}

__device__ __forceinline__ void score_store8(const ScoreParams& p, size_t at, const float (&v)[8]) {
    if (p.out_bf16) {
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + at) =
            make_uint4(rn_bf16x2(v[0], v[1]), rn_bf16x2(v[2], v[3]), rn_bf16x2(v[4], v[5]), rn_bf16x2(v[6], v[7]));
    } else {
        float4* o = reinterpret_cast<float4*>(static_cast<float*>(p.out) + at);
        o[0] = make_float4(v[0], v[1], v[2], v[3]);
        o[1] = make_float4(v[4], v[5], v[6], v[7]);
    }
}

// -------------------------------------------------------------------------------------------------
// consumer on the CUDA cores: LPR lanes share a cache row, every lane keeps its chunk of q and of the accumulator
// -------------------------------------------------------------------------------------------------
template <typename KV, int HD, int G>
struct ScoreFma {
    using M = TileMap<KV, HD>;
    static constexpr int kGroup = G, kTile = M::kTileBytes, kThreads = kScoreThreads;
    static constexpr int LPR = M::kLanesPerRow, CPL = M::kChunksPerLane, RPW = M::kRowsPerLoad;
    static constexpr int ITER = M::kIters, EPC = KV::kPerChunk, EPL = M::kElemsPerLane;
    static constexpr int PPC = EPC / 2, PPL = EPL / 2, ROWB = M::kRowBytes;

    float2 q2[G][PPL], acc2[G][PPL];
    float m_run[G], l_run[G], slope[G], pr[G];
    int g, rg, my_tok;
    bool one_of_pair;

    __device__ __forceinline__ void init(int lane) {
        g = lane % LPR;   // chunk position inside the row
        rg = lane / LPR;  // which of the RPW rows of a warp-wide load
        my_tok = (LPR >= 2 ? (g >> 1) * RPW : 0) + rg;  // the token whose score this lane ends up with
        one_of_pair = LPR < 2 || (g & 1) == 0;
    }
    __device__ __forceinline__ void load(const ScoreParams& p, const ScoreItem& it) {
        const size_t at = (size_t)it.index * (G * HD);  // items_per_row * G == heads
        const int h0 = (int)(it.index % (uint32_t)p.plan.items_per_row) * G;
#pragma unroll
        for (int i = 0; i < G; ++i) {
#pragma unroll
            for (int cp = 0; cp < CPL; ++cp) {
                const int d0 = (g + 32 * cp) * EPC;
#pragma unroll
                for (int e = 0; e < EPC; e += 4) {
                    float4 t;
                    if (p.q_bf16) {
                        const uint2 w = __ldg(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p.q) + at + i * HD + d0 + e));
                        t = make_float4(bf16_lo(w.x), bf16_hi(w.x), bf16_lo(w.y), bf16_hi(w.y));
                    } else {
                        t = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(p.q) + at + i * HD + d0 + e));
                    }
                    q2[i][(cp * EPC + e) / 2] = make_float2(t.x * p.q_scale, t.y * p.q_scale);
                    q2[i][(cp * EPC + e) / 2 + 1] = make_float2(t.z * p.q_scale, t.w * p.q_scale);
                }
            }
#pragma unroll
            for (int e = 0; e < PPL; ++e) acc2[i][e] = make_float2(0.f, 0.f);
            m_run[i] = -INFINITY;
            l_run[i] = 0.f;
            slope[i] = p.slopes ? __ldg(p.slopes + h0 + i) * 1.4426950408889634f : 0.f;
        }
    }
    // dot products of the tile's 16 tokens; `released` is called once the tile has been read
    template <typename F>
    __device__ __forceinline__ void scores(const ScoreParams& p, const ScoreItem& it, const uint8_t* ktile, uint32_t meta, int tok0, int nskip, int nvalid,
                                           int lane, F released) {
        float sc[G][ITER];
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            const int t = (i * RPW + rg) & (kBlockTokens - 1);
            float2 d2[G];
#pragma unroll
            for (int h = 0; h < G; ++h) d2[h] = make_float2(0.f, 0.f);
#pragma unroll
            for (int cp = 0; cp < CPL; ++cp) {
                const uint4 w = *reinterpret_cast<const uint4*>(ktile + t * ROWB + (g + 32 * cp) * 16);
                float2 f[PPC];
                unpack2<KV>(w, f);
#pragma unroll
                for (int h = 0; h < G; ++h)
#pragma unroll
                    for (int e = 0; e < PPC; ++e) d2[h] = fma2(q2[h][cp * PPC + e], f[e], d2[h]);
            }
#pragma unroll
            for (int h = 0; h < G; ++h) sc[h][i] = d2[h].x + d2[h].y;
        }
        released();
        const bool visible = my_tok >= nskip && my_tok < nvalid;
        const float dist = p.slopes ? score_distance(p, it, meta, tok0, my_tok, visible) : 0.f;
#pragma unroll
        for (int h = 0; h < G; ++h) {
            RowReduce<ITER, LPR / 2>::run(sc[h], lane);
            float x = score_modify(p, sc[h][0], slope[h], dist);
            if (p.scores && (meta & kSuFixed) && visible && one_of_pair) score_record(p, (size_t)it.index * G + h, tok0 + my_tok, x);
            x = visible ? x : -INFINITY;
            // online softmax, one running maximum per row group
            float mt = x;
#pragma unroll
            for (int d = LPR / 2; d >= 2; d >>= 1) mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, d));
            const float m_new = fmaxf(m_run[h], mt);
            const float m_safe = (m_new == -INFINITY) ? 0.f : m_new;
            const float alpha = fast_exp2(m_run[h] - m_safe);
            pr[h] = fast_exp2(x - m_safe);
            l_run[h] = l_run[h] * alpha + pr[h];
            m_run[h] = m_new;
            const float2 alpha2 = make_float2(alpha, alpha);
#pragma unroll
            for (int e = 0; e < PPL; ++e) acc2[h][e] = mul2(acc2[h][e], alpha2);
        }
    }
    template <bool ALL>
    __device__ __forceinline__ void add_values(const uint8_t* vtile, int nskip, int nvalid) {
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            const int t = i * RPW + rg;
            float2 pi2[G];
#pragma unroll
            for (int h = 0; h < G; ++h) {
                float pi = (LPR >= 2) ? __shfl_sync(0xffffffffu, pr[h], rg * LPR + 2 * i) : pr[h];
                if (ALL && RPW > kBlockTokens && rg >= kBlockTokens) pi = 0.f;
                pi2[h] = make_float2(pi, pi);
            }
            if (ALL || (t >= nskip && t < nvalid)) {  // rows outside may hold anything
#pragma unroll
                for (int cp = 0; cp < CPL; ++cp) {
                    const uint4 w = *reinterpret_cast<const uint4*>(vtile + (ALL ? t & (kBlockTokens - 1) : t) * ROWB + (g + 32 * cp) * 16);
                    float2 f[PPC];
                    unpack2<KV>(w, f);
#pragma unroll
                    for (int h = 0; h < G; ++h)
#pragma unroll
                        for (int e = 0; e < PPC; ++e) acc2[h][cp * PPC + e] = fma2(pi2[h], f[e], acc2[h][cp * PPC + e]);
                }
            }
        }
    }
    __device__ __forceinline__ void values(const uint8_t* vtile, int nskip, int nvalid, int) {
        // (two loops: a condition inside the loop keeps the loads of its iterations apart)
        if (nvalid == kBlockTokens && nskip == 0) add_values<true>(vtile, nskip, nvalid);
        else add_values<false>(vtile, nskip, nvalid);
    }
    // the item's result, or this segment's partial into slot my_slot
    __device__ __forceinline__ void emit(const ScoreParams& p, const ScoreItem& it, bool whole, int my_slot, int lane) {
#pragma unroll
        for (int h = 0; h < G; ++h) {
            float mx = m_run[h];
#pragma unroll
            for (int d = LPR; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
            const float mx_safe = (mx == -INFINITY) ? 0.f : mx;
            const float wgt = fast_exp2(m_run[h] - mx_safe);
            float lsum = l_run[h] * wgt;
#pragma unroll
            for (int d = 16; d >= 1; d >>= 1) lsum += __shfl_xor_sync(0xffffffffu, lsum, d);
            if (LPR >= 2) lsum *= 0.5f;  // the two lanes of a pair carry the same token
            float acc[EPL];
#pragma unroll
            for (int e = 0; e < PPL; ++e) {
                acc[2 * e] = acc2[h][e].x * wgt;
                acc[2 * e + 1] = acc2[h][e].y * wgt;
            }
#pragma unroll
            for (int e = 0; e < EPL; ++e)
#pragma unroll
                for (int d = LPR; d < 32; d <<= 1) acc[e] += __shfl_xor_sync(0xffffffffu, acc[e], d);
            const float inv = 1.f / lsum;  // (0 only where every score is -inf: 0/0, NaN)
            if (lane < LPR) {
                float* dst = p.part_acc + (size_t)my_slot * (G * HD) + h * HD;
                const size_t at = ((size_t)it.index * G + h) * HD;
#pragma unroll
                for (int cp = 0; cp < CPL; ++cp)
#pragma unroll
                    for (int e = 0; e < EPC; e += 4) {
                        const int d0 = (g + 32 * cp) * EPC + e;
                        const float* a = acc + cp * EPC + e;
                        if (!whole)
                            __stcg(reinterpret_cast<float4*>(dst + d0), make_float4(a[0], a[1], a[2], a[3]));
                        else if (p.out_bf16)
                            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + at + d0) = make_uint2(rn_bf16x2(a[0] * inv, a[1] * inv), rn_bf16x2(a[2] * inv, a[3] * inv));
                        else
                            *reinterpret_cast<float4*>(static_cast<float*>(p.out) + at + d0) = make_float4(a[0] * inv, a[1] * inv, a[2] * inv, a[3] * inv);
                    }
            }
            if (lane == 0) {
                if (!whole) __stcg(reinterpret_cast<float2*>(p.part_ml + (size_t)my_slot * (2 * G) + 2 * h), make_float2(mx, lsum));
                else if (p.scores) *reinterpret_cast<float2*>(p.score_ml + 2 * ((size_t)it.index * G + h)) = make_float2(mx_safe, inv);
            }
        }
    }
};

// -------------------------------------------------------------------------------------------------
// consumer on the tensor cores (mma.sync m16n8k16), for four query heads of a bf16 KV head: a product per head on the CUDA
// cores costs as many instructions as the memory leaves time for, and here the heads are columns that cost nothing.  fp32 operands
// (queries, weights) go in as three bf16 whose sum is exact to 24 bits, as columns of their own:
//   scores   S[16 tokens][8 columns] = K[16 x HD] Q^T: A is the tile's rows, lane (g, c) = (lane / 4, lane % 4) reads chunks
//            c + 4 i of rows g and g + 8 -- the order of the dims is the same permutation for Q, so no element is moved;
//   values   out^T[HD][8] = V^T[HD x 16 tokens] P: lane (g, c) reads chunk(s) g of tokens 2c, 2c + 1, 2c + 8, 2c + 9 and pairs
//            the tokens' elements with byte permutes; P comes from the lanes that hold the scores by four shuffles.
// Column n of a product is part n % 2 of head n / 2; the third parts are a second product into the same
// accumulators (the columns of a head are summed in the end, whatever they hold).  Measured: 16 + 4 heads of 128 over six caches
// of 24096 tokens (282 MB) 72 us, 155 us on the CUDA cores; bound by the instructions and latency of a tile's chain.  The
// two-way (K) and four-way (V) bank conflicts of the unswizzled tiles are left: rows fetched one by one into padded slots have none,
// but sixteen copies a tile cost more (84 us), and 16 warps with the Q fragments in shared memory were slower too (77 us).
// -------------------------------------------------------------------------------------------------
__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Part 0, 1 or 2 of the split of two values into three bf16 each, packed.
__device__ __forceinline__ uint32_t split3(float a, float b, int part) {
    const uint32_t hi = rn_bf16x2(a, b);
    if (part == 0) return hi;
    const float ra = a - bf16_lo(hi), rb = b - bf16_hi(hi);
    const uint32_t mid = rn_bf16x2(ra, rb);
    if (part == 1) return mid;
    return part == 2 ? rn_bf16x2(ra - bf16_lo(mid), rb - bf16_hi(mid)) : 0u;
}

template <int HD>
struct ScoreMma {
    static_assert(HD == 64 || HD == 128, "what the fragments below are laid out for");
    static constexpr int G = 4, kGroup = G, kTile = kBlockTokens * HD * 2, kThreads = 384;  // 12 warps: 168 registers a thread
    static constexpr int NT = 2;                // products per K / V fragment
    static constexpr int CH = HD / 32;          // chunks of a K row per lane
    static constexpr int MT = HD / 16;          // 16-dim tiles of the accumulator
    static constexpr int VC = HD / 64;          // chunks of a V row per lane
    static constexpr int ROWB = HD * 2;

    uint4 qf[NT][CH];
    float acc[MT][4];
    float p0, p1;  // weights of tokens g and g + 8, of this lane's head
    float m_run, l_run, slope;
    int g, c, head;

    __device__ __forceinline__ void init(int lane) {
        g = lane >> 2;
        c = lane & 3;
        head = c;  // whose scores and accumulator columns (2c, 2c + 1) this lane holds
    }
    __device__ __forceinline__ int part_of(int column, int nt) const {
        return nt == 0 ? column & 1 : (column & 1) ? 3 : 2;  // 3: nothing
    }
    __device__ __forceinline__ void load(const ScoreParams& p, const ScoreItem& it) {
        const int col_head = g >> 1;  // column g of the B operand
        const size_t at = ((size_t)it.index * G + col_head) * HD;
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int d0 = (c + 4 * i) * 8;
            float f[8];
            if (p.q_bf16) {
                BF16::unpack(__ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.q) + at + d0)), f);
            } else {
                const float4 a = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(p.q) + at + d0));
                const float4 b = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(p.q) + at + d0 + 4));
                f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
                f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const int part = part_of(g, nt);
                qf[nt][i] = make_uint4(split3(f[0], f[1], part), split3(f[2], f[3], part), split3(f[4], f[5], part), split3(f[6], f[7], part));
            }
        }
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[m][e] = 0.f;
        m_run = -INFINITY;
        l_run = 0.f;
        slope = p.slopes ? __ldg(p.slopes + (int)(it.index % (uint32_t)p.plan.items_per_row) * G + head) * 1.4426950408889634f : 0.f;
    }
    template <typename F>
    __device__ __forceinline__ void scores(const ScoreParams& p, const ScoreItem& it, const uint8_t* ktile, uint32_t meta, int tok0, int nskip, int nvalid,
                                           int, F released) {
        uint4 lo[CH], hi[CH];  // rows g and g + 8
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            lo[i] = *reinterpret_cast<const uint4*>(ktile + g * ROWB + (c + 4 * i) * 16);
            hi[i] = *reinterpret_cast<const uint4*>(ktile + (g + 8) * ROWB + (c + 4 * i) * 16);
        }
        released();
        float s[2 * NT][4];  // chains of products that do not wait for one another
#pragma unroll
        for (int k = 0; k < 2 * NT; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[k][e] = 0.f;
#pragma unroll
        for (int i = 0; i < CH; ++i)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                mma_16816(s[2 * nt], lo[i].x, hi[i].x, lo[i].y, hi[i].y, qf[nt][i].x, qf[nt][i].y);
                mma_16816(s[2 * nt + 1], lo[i].z, hi[i].z, lo[i].w, hi[i].w, qf[nt][i].z, qf[nt][i].w);
            }
        float x0 = (s[0][0] + s[1][0]) + (s[0][1] + s[1][1]), x1 = (s[0][2] + s[1][2]) + (s[0][3] + s[1][3]);
        x0 += (s[2][0] + s[3][0]) + (s[2][1] + s[3][1]);
        x1 += (s[2][2] + s[3][2]) + (s[2][3] + s[3][3]);
        const bool v0 = g >= nskip && g < nvalid, v1 = g + 8 >= nskip && g + 8 < nvalid;
        float d0 = 0.f, d1 = 0.f;
        if (p.slopes) {
            d0 = score_distance(p, it, meta, tok0, g, v0);
            d1 = score_distance(p, it, meta, tok0, g + 8, v1);
        }
        x0 = score_modify(p, x0 * p.q_scale, slope, d0);
        x1 = score_modify(p, x1 * p.q_scale, slope, d1);
        if (p.scores && (meta & kSuFixed)) {
            if (v0) score_record(p, (size_t)it.index * G + head, tok0 + g, x0);
            if (v1) score_record(p, (size_t)it.index * G + head, tok0 + g + 8, x1);
        }
        x0 = v0 ? x0 : -INFINITY;
        x1 = v1 ? x1 : -INFINITY;
        float mt = fmaxf(x0, x1);
#pragma unroll
        for (int d = 4; d <= 16; d <<= 1) mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, d));
        const float m_new = fmaxf(m_run, mt);
        const float m_safe = (m_new == -INFINITY) ? 0.f : m_new;
        const float alpha = fast_exp2(m_run - m_safe);
        p0 = fast_exp2(x0 - m_safe);
        p1 = fast_exp2(x1 - m_safe);
        l_run = l_run * alpha + (p0 + p1);
        const bool moved = m_new != m_run;
        m_run = m_new;
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[m][e] *= alpha;
        }
    }
    __device__ __forceinline__ void values(const uint8_t* vtile, int nskip, int nvalid, int) {
        // weights of tokens 2c, 2c + 1, 2c + 8, 2c + 9 for column g
        const int col_head = g >> 1;
        const float w0 = __shfl_sync(0xffffffffu, p0, 8 * c + col_head), w1 = __shfl_sync(0xffffffffu, p0, 8 * c + 4 + col_head);
        const float w2 = __shfl_sync(0xffffffffu, p1, 8 * c + col_head), w3 = __shfl_sync(0xffffffffu, p1, 8 * c + 4 + col_head);
        uint32_t b[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            b[nt][0] = split3(w0, w1, part_of(g, nt));
            b[nt][1] = split3(w2, w3, part_of(g, nt));
        }
        uint4 v[VC][4];
#pragma unroll
        for (int k = 0; k < VC; ++k)
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const int tok = 2 * c + (t & 1) + (t >> 1) * 8;
                v[k][t] = *reinterpret_cast<const uint4*>(vtile + tok * ROWB + (g + 8 * k) * 16);
                if ((nskip > 0 || nvalid < kBlockTokens) && !(tok >= nskip && tok < nvalid)) v[k][t] = make_uint4(0u, 0u, 0u, 0u);  // may hold anything
            }
        // element e of chunk k, as (token 2c, token 2c + 1) and (2c + 8, 2c + 9) pairs
        auto word = [](const uint4& w, int e) { return e < 2 ? w.x : e < 4 ? w.y : e < 6 ? w.z : w.w; };
        auto pair = [&](int k, int e, int t) { return __byte_perm(word(v[k][t], e), word(v[k][t + 1], e), (e & 1) ? 0x7632 : 0x5410); };
        // four 16-dim tiles at a time, so that a tile's second product does not wait for its first
#pragma unroll
        for (int m0 = 0; m0 < MT; m0 += 4) {
            uint32_t a[4][4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                // rows g and g + 8 of the tile: with 128 dims element m of chunks g and g + 8, with 64 elements m and m + 4 of chunk g
                constexpr bool kTwo = VC == 2;
                const int m = m0 + i, k1 = kTwo ? 1 : 0, e1 = kTwo ? m : m + 4;
                a[i][0] = pair(0, m, 0);
                a[i][1] = pair(k1, e1, 0);
                a[i][2] = pair(0, m, 2);
                a[i][3] = pair(k1, e1, 2);
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < 4; ++i) mma_16816(acc[m0 + i], a[i][0], a[i][1], a[i][2], a[i][3], b[nt][0], b[nt][1]);
        }
    }
    __device__ __forceinline__ void emit(const ScoreParams& p, const ScoreItem& it, bool whole, int my_slot, int) {
        const float m_safe = (m_run == -INFINITY) ? 0.f : m_run;
        float lsum = l_run;
#pragma unroll
        for (int d = 4; d <= 16; d <<= 1) lsum += __shfl_xor_sync(0xffffffffu, lsum, d);
        const float inv = 1.f / lsum;
        float lo[MT], hi[MT];  // rows g, g + 8 of the tiles
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            lo[m] = acc[m][0] + acc[m][1];
            hi[m] = acc[m][2] + acc[m][3];
        }
        const size_t at = ((size_t)it.index * G + head) * HD;
        float* part = p.part_acc + (size_t)my_slot * (G * HD) + head * HD;
        auto put = [&](int chunk, float (&f)[8]) {
            if (whole) {
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] *= inv;
                score_store8(p, at + chunk * 8, f);
            } else {
                __stcg(reinterpret_cast<float4*>(part + chunk * 8), make_float4(f[0], f[1], f[2], f[3]));
                __stcg(reinterpret_cast<float4*>(part + chunk * 8 + 4), make_float4(f[4], f[5], f[6], f[7]));
            }
        };
        float f[8];
        if constexpr (VC == 2) {
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = lo[e];
            put(g, f);
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = hi[e];
            put(g + 8, f);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                f[e] = lo[e];
                f[4 + e] = hi[e];
            }
            put(g, f);
        }
        if (g == 0) {
            if (!whole) __stcg(reinterpret_cast<float2*>(p.part_ml + (size_t)my_slot * (2 * G) + 2 * head), make_float2(m_run, lsum));
            else if (p.scores) *reinterpret_cast<float2*>(p.score_ml + 2 * ((size_t)it.index * G + head)) = make_float2(m_safe, inv);
        }
    }
};

template <typename C, int HD>
__global__ void __launch_bounds__(C::kThreads, 1) rswa_scored_kernel(const __grid_constant__ ScoreParams p) {
    constexpr int G = C::kGroup, TILE = C::kTile;
    constexpr unsigned FULL = 0xffffffffu;

    extern __shared__ __align__(128) uint8_t smem[];
    const int warps = blockDim.x >> 5;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int bar_bytes = (warps * kScoreRing * 8 + 127) & ~127;
    uint8_t* my_tiles = smem + bar_bytes + (size_t)warp * (kScoreRing * TILE);
    const uint32_t bar0 = smem_addr(smem) + warp * (kScoreRing * 8);
    const uint32_t tile0 = smem_addr(my_tiles);
    auto init_barriers = [&]() {
        if (lane == 0) {
#pragma unroll
            for (int s = 0; s < kScoreRing; ++s) mbar_init(bar0 + 8 * s, 1);
            mbar_init_fence();
        }
        __syncwarp();
    };

    // ---- the plan: up to 32 rows by warp 0 while the others set up their barriers, more by the whole CTA, many in global memory ----
    const ScoreRow* info = p.info;
    const long long* rs = p.rs;
    if (p.rows <= kScoreSharedRows) {
        uint8_t* plan_base = smem + bar_bytes + (size_t)warps * (kScoreRing * TILE);
        ScoreRow* info_s = reinterpret_cast<ScoreRow*>(plan_base);
        long long* rs_s = reinterpret_cast<long long*>(plan_base + sizeof(ScoreRow) * p.rows);
        if (p.rows > 32) score_plan_rows(p.plan, info_s, rs_s, rs_s + p.rows + 1, blockIdx.x == 0);
        else if (warp == 0) score_plan_warp(p.plan, info_s, rs_s, blockIdx.x == 0, lane);
        init_barriers();
        __syncthreads();
        info = info_s;
        rs = rs_s;
    } else {
        init_barriers();
    }
    const int items_per_row = p.plan.items_per_row;
    const long long total = rs[p.rows];
    if (total == 0) return;
    const ScorePieces pm(total, p.total_warps);
    // fewer pieces than warps are spread over the SMs
    const int piece = pm.ns == p.total_warps ? (int)blockIdx.x * warps + warp : warp * (int)gridDim.x + (int)blockIdx.x;
    if (piece >= pm.ns) return;
    const long long u0 = pm.start(piece);
    const int n_units = (int)(pm.start(piece + 1) - u0);

    if (p.scores) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the kernel that turns scores into weights
    C work;
    work.init(lane);

    // ---- unit descriptors: lane l describes unit desc_base + l of this piece ----------------------------
    uint32_t d_tile = 0, d_meta = 0, d_item = 0;
    int d_tok = 0;  // fixed region: index of the tile's token 0; ring / text: its distance from the query
    int desc_base = 0;
    auto build_desc = [&](int base) {
        desc_base = base;
        d_tile = d_meta = d_item = 0;
        d_tok = 0;
        if (base + lane < n_units) {
            const long long u = u0 + base + lane;
            int lo = 0, hi = p.rows;  // rs[lo] <= u < rs[hi]
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (rs[mid] <= u) lo = mid; else hi = mid;
            }
            const ScoreRow o = info[lo];
            const int first = o.lo / kBlockTokens;
            const int fixed_tiles = o.hi > o.lo ? (o.hi + kBlockTokens - 1) / kBlockTokens - first : 0;
            const int per_item = fixed_tiles + score_ring_tiles(o);
            const long long rem = u - rs[lo];
            const int it = (int)div_units(rem, per_item), j = (int)(rem - (long long)it * per_item);
            const int kvh = (int)((uint32_t)(it * G) / (uint32_t)p.group);
            uint32_t m = 0;
            int valid, skip = 0, blk = -1;
            if (j < fixed_tiles) {
                const int s0 = (first + j) * kBlockTokens;
                valid = min(kBlockTokens, o.hi - s0);
                skip = max(o.lo - s0, 0);
                d_tok = s0;
                m |= kSuFixed;
                if (first + j < p.table_stride) blk = __ldg(p.table + (size_t)o.slot * p.table_stride + first + j);
                else atomicOr(p.status, kStatusBadSlot);
            } else {
                const int jr = j - fixed_tiles;
                const int lead = o.text >= 0 ? o.text & 15 : 0;
                valid = min(kBlockTokens, lead + o.ring - jr * kBlockTokens);
                skip = jr == 0 ? lead : 0;
                d_tok = o.age0 - jr * kBlockTokens;
                if (o.text >= 0) {
                    blk = (o.text >> 4) + jr;
                    m |= kSuText;
                } else if (o.ring_entry + jr < p.table_stride) {
                    blk = __ldg(p.table + (size_t)o.slot * p.table_stride + o.ring_entry + jr);
                } else {
                    atomicOr(p.status, kStatusBadSlot);
                }
            }
            if (blk < 0 || blk >= ((m & kSuText) ? p.text_blocks : p.num_blocks)) {
                atomicOr(p.status, kStatusBadBlock);
                blk = 0;
            }
            d_tile = (uint32_t)blk * p.kv_heads + kvh;
            if (j == per_item - 1) m |= kSuLast;
            if (j == 0) m |= kSuFirst;
            d_meta = m | (uint32_t)valid | ((uint32_t)skip << kSuSkipShift);
            d_item = (uint32_t)lo * (uint32_t)items_per_row + (uint32_t)it;
        }
    };

    // ---- producer: tiles K(0) V(0) K(1) V(1) ... rotate through the slots ------------------------------
    const uint64_t pol_stream = l2_policy_evict_first(), pol_keep = l2_policy_evict_last();
    int issue_slot = 0, use_slot = 0;
    int issue_seq = 0, consumed = 0;
    uint32_t phases = 0;
    auto issue_next = [&]() {
        if (issue_seq >= 2 * n_units) return;
        const int src = (issue_seq >> 1) - desc_base;
        const bool is_v = (issue_seq & 1) != 0;
        const uint32_t tile = __shfl_sync(FULL, d_tile, src);
        const uint32_t meta = __shfl_sync(FULL, d_meta, src);
        if (lane == 0) {
            const uint32_t bar = bar0 + 8 * issue_slot;
            const uint8_t* base = (meta & kSuText) ? (is_v ? p.v_text : p.k_text) : (is_v ? p.v_base : p.k_base);
            mbar_arrive_expect_tx(bar, TILE);
            // ring tiles are read once per launch; tiles of the fixed region again by whoever shares the prefix
            bulk_copy_g2s_hint(tile0 + issue_slot * TILE, base + (size_t)tile * TILE, TILE, bar, (meta & kSuFixed) ? pol_keep : pol_stream);
        }
        issue_slot = issue_slot == kScoreRing - 1 ? 0 : issue_slot + 1;
        ++issue_seq;
    };
    auto wait_tile = [&]() -> uint8_t* {
        if (!mbar_wait_bounded(bar0 + 8 * use_slot, (phases >> use_slot) & 1u, p.status, p.wait_limit)) return nullptr;
        uint8_t* t = my_tiles + use_slot * TILE;
        phases ^= 1u << use_slot;
        use_slot = use_slot == kScoreRing - 1 ? 0 : use_slot + 1;
        ++consumed;
        return t;
    };

    ScoreItem item{};
    auto start_item = [&](uint32_t index) {
        item.index = index;
        if (p.slopes) {
            const ScoreRow& o = info[index / (uint32_t)items_per_row];
            item.slot = o.slot;
            item.q_pos = o.q_pos;
        }
        work.load(p, item);
    };

    uint32_t pend[2];  // items this piece left a partial of: the first and the last
    int pend_n = 0;

    build_desc(0);
#pragma unroll
    for (int s = 0; s < kScoreRing; ++s) issue_next();
    start_item(__shfl_sync(FULL, d_item, 0));
    bool first_segment = true, gave_up = false;
    bool from_start = (__shfl_sync(FULL, d_meta, 0) & kSuFirst) != 0;

    for (int it = 0; it < n_units; ++it) {
        if (it - desc_base >= 32 - 2) build_desc(it);  // the producer looks two units ahead
        const uint32_t meta = __shfl_sync(FULL, d_meta, it - desc_base);
        const int tok0 = __shfl_sync(FULL, d_tok, it - desc_base);
        const int nvalid = (int)(meta & kSuValid), nskip = (int)((meta >> kSuSkipShift) & 15);

        const uint8_t* ktile = wait_tile();
        if (!ktile) { gave_up = true; break; }
        work.scores(p, item, ktile, meta, tok0, nskip, nvalid, lane, [&]() {
            __syncwarp();
            issue_next();  // the K slot is free
        });
        const uint8_t* vtile = wait_tile();
        if (!vtile) { gave_up = true; break; }
        work.values(vtile, nskip, nvalid, lane);
        __syncwarp();
        issue_next();  // the V slot is free

        // ---- end of an item or of the piece ---------------------------------------------------------------
        const bool item_done = (meta & kSuLast) != 0, piece_done = it == n_units - 1;
        if (item_done || piece_done) {
            const bool whole = item_done && from_start;
            work.emit(p, item, whole, 2 * piece + (first_segment ? 0 : 1), lane);
            if (!whole) pend[pend_n++ & 1] = item.index;
            first_segment = false;
            if (!piece_done) {
                start_item(__shfl_sync(FULL, d_item, it + 1 - desc_base));
                from_start = true;
            }
        }
    }
    if (gave_up) {
        // A wait ran out (the status word says so and the launch's results are void).  Tiles issued and not yet consumed
        // may still be on their way into this warp's slots: see them land before the CTA exits.  Full limit.
        for (; consumed < issue_seq; ++consumed) {
            mbar_wait_bounded(bar0 + 8 * use_slot, (phases >> use_slot) & 1u, nullptr);
            phases ^= 1u << use_slot;
            use_slot = use_slot == kScoreRing - 1 ? 0 : use_slot + 1;
        }
        return;
    }

    // ---- partials are joined in a tree: eight at a time, by the warp that arrives last at the eight ------------------------
    // (One warp that joins everything is the tail of the launch when a long row is cut into many pieces: 74 partials of four heads
    // took 40 of 100 us.)  Level l joins entries of kScoreJoin^l consecutive pieces of the item into the first one's slot; the last
    // level writes the result.  A group's counter is that of its first piece, in an array of its own per level and for the groups
    // that start the item (a piece can end one item and begin the next).
    for (int k = 0; k < pend_n; ++k) {
        const uint32_t done = pend[k];
        const int r = (int)(done / (uint32_t)items_per_row);
        const int n = (int)div_units(rs[r + 1] - rs[r], items_per_row);
        const long long s0 = rs[r] + (long long)(done - (uint32_t)r * (uint32_t)items_per_row) * n;
        const int wf = pm.of(s0), n_part = pm.of(s0 + n - 1) - wf + 1;
        const bool wf_second = pm.start(wf) < s0;  // the item is piece wf's second segment
        auto slot_of = [&](int i) { return (size_t)(2 * (wf + i) + ((i == 0 && wf_second) ? 1 : 0)); };
        int i = piece - wf;
        for (int span = 1, level = 0;; span *= kScoreJoin, ++level) {
            const int entries = (n_part + span - 1) / span, group = i / (span * kScoreJoin);
            const int members = min(kScoreJoin, entries - group * kScoreJoin);
            i = group * span * kScoreJoin;
            if (members == 1) continue;  // the odd one out goes up as it is
            __syncwarp();  // the stores of every lane come before the arriving lane's release
            int* counter = p.counters + (size_t)(2 * level + (group > 0 ? 1 : 0)) * p.pieces + wf + i;
            int old = 0;
            if (lane == 0)  // release: this warp's partial (ordered before by the barrier above); acquire: the others'
                asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(old) : "l"(counter) : "memory");
            old = __shfl_sync(FULL, old, 0);
            if (old != members - 1) break;
            __syncwarp();  // the arriving lane's acquire covers the loads the whole warp issues next
            if (lane == 0) *counter = 0;  // for the next launch
            const bool last = entries <= kScoreJoin;
            // lane 4 m + h holds (max, sum) of member m, head h; the accumulators follow in 16-byte columns, 128 floats a round
            const int m_lane = lane >> 2, h_lane = lane & 3;
            const bool on = m_lane < members && h_lane < G;
            const float2 ml = on ? __ldcg(reinterpret_cast<const float2*>(p.part_ml + slot_of(i + m_lane * span) * (2 * G) + 2 * h_lane)) : make_float2(-INFINITY, 0.f);
            constexpr int kRounds = (G * HD + 127) / 128;
            float4 o[kRounds];
            float mx = ml.x;
#pragma unroll
            for (int d = 4; d <= 16; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(FULL, mx, d));
            const float m_safe = (mx == -INFINITY) ? 0.f : mx;
            const float wgt = on ? fast_exp2(ml.x - m_safe) : 0.f;
            float lsum = on ? ml.y * wgt : 0.f;
#pragma unroll
            for (int d = 4; d <= 16; d <<= 1) lsum += __shfl_xor_sync(FULL, lsum, d);
#pragma unroll
            for (int c = 0; c < kRounds; ++c) {
                const int col = c * 128 + lane * 4;
                float4 t[kScoreJoin];
#pragma unroll
                for (int m = 0; m < kScoreJoin; ++m)
                    t[m] = m < members && col < G * HD ? __ldcg(reinterpret_cast<const float4*>(p.part_acc + slot_of(i + m * span) * (G * HD) + col)) : make_float4(0.f, 0.f, 0.f, 0.f);
                const int head = min(col / HD, G - 1);
                o[c] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int m = 0; m < kScoreJoin; ++m) {
                    const float w = __shfl_sync(FULL, wgt, 4 * m + head);
                    o[c].x = fmaf(t[m].x, w, o[c].x);
                    o[c].y = fmaf(t[m].y, w, o[c].y);
                    o[c].z = fmaf(t[m].z, w, o[c].z);
                    o[c].w = fmaf(t[m].w, w, o[c].w);
                }
            }
            const float inv_lane = 1.f / lsum;
#pragma unroll
            for (int c = 0; c < kRounds; ++c) {
                const int col = c * 128 + lane * 4;
                const float inv = __shfl_sync(FULL, inv_lane, min(col / HD, G - 1));
                if (col >= G * HD) continue;
                if (!last) {
                    __stcg(reinterpret_cast<float4*>(p.part_acc + slot_of(i) * (G * HD) + col), o[c]);
                } else if (p.out_bf16) {
                    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + (size_t)done * (G * HD) + col) =
                        make_uint2(rn_bf16x2(o[c].x * inv, o[c].y * inv), rn_bf16x2(o[c].z * inv, o[c].w * inv));
                } else {
                    *reinterpret_cast<float4*>(static_cast<float*>(p.out) + (size_t)done * (G * HD) + col) = make_float4(o[c].x * inv, o[c].y * inv, o[c].z * inv, o[c].w * inv);
                }
            }
            if (lane < G) {  // member 0's lanes
                if (!last) __stcg(reinterpret_cast<float2*>(p.part_ml + slot_of(i) * (2 * G) + 2 * lane), make_float2(mx, lsum));
                else if (p.scores) *reinterpret_cast<float2*>(p.score_ml + 2 * ((size_t)done * G + lane)) = make_float2(m_safe, inv_lane);
            }
            if (last) break;
        }
    }
}

// -------------------------------------------------------------------------------------------------
// attention weights: mass_out[slot][s] = decay * mass_in[slot][s] + sum over the slot's rows and heads of the weight of
// token s of the fixed region.  One thread per token adds its rows and heads in order; a slot named by several rows is
// handled by its first row's CTAs.
// -------------------------------------------------------------------------------------------------
struct MassParams {
    ScorePlan plan;
    int heads;
    const float* scores;
    const float* score_ml;
    const float* mass_in;
    float* mass_out;
    int stride;
    float decay;
    int* status;
};

constexpr int kMassThreads = 256;

__global__ void __launch_bounds__(kMassThreads) rswa_mass_kernel(const __grid_constant__ MassParams p) {
    asm volatile("griddepcontrol.wait;" ::: "memory");  // (launched so that its set-up overlaps the attention)
    const int b = blockIdx.y, tid = threadIdx.x;
    const int slot = __ldg(p.plan.d_slots + b);
    const int pfx = max(__ldg(p.plan.d_prefill_len + slot), 0);  // (on their way while the batch is looked through)
    const int len = __ldg(p.plan.d_len + slot);
    int others = 0;  // rows that name the slot too: 1 earlier, 2 later ones
    for (int j = tid; j < p.plan.rows; j += kMassThreads)
        if (j != b && __ldg(p.plan.d_slots + j) == slot) others |= j < b ? 1 : 2;
    if (__syncthreads_or(others & 1)) return;
    const int last = __syncthreads_or(others & 2) ? p.plan.rows : b + 1;
    const int n = min(pfx, p.stride);
    if (pfx > p.stride && tid == 0 && blockIdx.x == 0) atomicOr(p.status, kStatusBadSlot);
    const int s = blockIdx.x * kMassThreads + tid;
    if ((int)blockIdx.x * kMassThreads >= n) return;
    const size_t at = (size_t)slot * p.stride + s;
    float sum = (s < n && p.mass_in && p.decay != 0.f) ? p.decay * p.mass_in[at] : 0.f;
    const int fixed = min(max(len, 0), pfx);
    for (int r = b; r < last; ++r) {
        if (__ldg(p.plan.d_slots + r) != slot) continue;
        int lo, hi;
        score_range(p.plan.d_lo, p.plan.d_hi, r, fixed, pfx, lo, hi);
        if (s < lo || s >= hi || s >= n) continue;
        const float* sc = p.scores + (size_t)r * p.heads * p.stride + s;
        const float2* ml = reinterpret_cast<const float2*>(p.score_ml) + (size_t)r * p.heads;
        // (eight heads' loads in flight.  48 rows of 2048 tokens, 10 / 16 / 32 heads: 7.7, 10.8 and 18 us; by ten 8.5, 13 and 22;
        // by sixteen 9.1, 9.5 and 16; by four 9.3, 13.6 and 24)
#pragma unroll 8
        for (int h = 0; h < p.heads; ++h) {
            const float2 w = __ldcg(ml + h);
            sum += fast_exp2(__ldcs(sc + (size_t)h * p.stride) - w.x) * w.y;
        }
    }
    if (s < n) p.mass_out[at] = sum;
}

}  // namespace uocr_b200
