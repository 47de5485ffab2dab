// Rotary positions for packed query / key rows, on their own or fused with the write of K and V into the
// paged cache (fixed region, or the ring append of single tokens).
//
// A pair (x0, x1) of a head turns by angle = position * freq_i:  (x0 c - x1 s, x0 s + x1 c), times an
// amplitude.  Angles of far positions lose everything in fp32 (position 10^6 times freq 1 is only known to
// 0.06 rad), so they are kept as 64-bit fixed-point fractions of a turn: freq_i / 2 pi is rounded once to
// 2^-64 turns on the host and position * that, modulo 2^64, is the exact fraction of the product -- one
// integer multiply.  Rounded to 2^-32 turns that is good to 2^-33, and the frequency's own rounding adds up to 2^-34 at the last
// 32-bit positions (frequencies above 1, of theta or factor below 1, add more in proportion).  What is left after the quadrant is
// taken off is at most an eighth of a turn and goes to sincospi in fp32, whose own step of up to 2^-28 turns is the larger error.
//
// The kernel moves bytes (q, k, v in; q and the pool rows out) and is bound by HBM, which takes few instructions a chunk and
// loads in flight with nothing to wait on.  A warp takes a row, or a share of its heads.  A lane keeps one 16-byte chunk position
// of a head and walks over the heads: the position's cosines and sines stay in registers, the loads of a batch of heads start
// before anything else, the warp's table of the row's angles (one entry per pair of one head) is filled meanwhile.  In the half
// layout a lane owns a chunk and its partner rotary_dim / 2 further on, in the interleaved layout a chunk holds whole pairs; every
// element is read and written by one lane, so a call may work in place.
// Measured: 16384 rows of 10 + 10 + 10 heads of 128, bf16 (252 MB) in 51 us, 4.9 TB/s, where a plain copy of the bytes takes 40;
// four rows around one table and a CTA barrier took 61-64 us, chunks dealt out one by one (twice the instructions) 74.
#pragma once

#include "rswa_paged.cuh"

namespace uocr_b200 {

constexpr int kRopeMaxPairs = 128;  // rotary_dim <= 256
constexpr int kRopeThreads = 256;

enum RopeMode : int { kRopeRows = 0, kRopeWrite = 1, kRopeAppend = 2 };

struct RopeParams {
    unsigned long long turn[kRopeMaxPairs];  // freq_i / 2 pi in units of 2^-64 turns
    float amplitude;
    int rotary_dim;
    const void* q;
    const void* k;
    const void* v;
    void* q_out;
    void* k_out;
    long long q_stride, k_stride, v_stride, q_out_stride, k_out_stride;  // elements between rows
    int rows, heads, kv_heads, head_dim;
    const int* d_positions;
    const int* d_slots;
    const int* d_pos;
    int* d_len;
    int* d_ring_pos;
    const int* d_prefill_len;
    int window;
    PagedView pv;
    int* status;
    int parts_log2;  // 2^x warps share a row
    int per_head;    // chunks of a rotated head a lane each (half layout: a chunk and its partner are one), or elements / pairs
    int items;       // element by element: items of a row
};

__device__ __forceinline__ void rope_sincos(unsigned long long turn, int position, float& sn, float& cs) {
    const unsigned long long t64 = (unsigned long long)(long long)position * turn + 0x80000000ull;
    const uint32_t t = (uint32_t)(t64 >> 32);
    const uint32_t quad = (t + 0x20000000u) >> 30;
    const float r = (float)(int)(t - (quad << 30)) * 4.656612873077393e-10f;  // half turns, |r| <= 1/4
    float s, c;
    sincospif(r, &s, &c);
    const float a = (quad & 1u) ? s : c, b = (quad & 1u) ? c : s;
    cs = (quad == 1u || quad == 2u) ? -a : a;
    sn = (quad & 2u) ? -b : b;
}

// The rotation, with its roundings fixed: every variant of the kernel gives the same bits.
__device__ __forceinline__ void rope_turn(float& x0, float& x1, float2 t) {
    const float y = __fmaf_rn(x0, t.x, -__fmul_rn(x1, t.y));
    x1 = __fmaf_rn(x0, t.y, __fmul_rn(x1, t.x));
    x0 = y;
}

template <typename T>
__device__ __forceinline__ void store8(void* base, long long at, const float (&f)[8]) {
    if constexpr (T::kBytes == 2) {
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(base) + at) =
            make_uint4(rn_bf16x2(f[0], f[1]), rn_bf16x2(f[2], f[3]), rn_bf16x2(f[4], f[5]), rn_bf16x2(f[6], f[7]));
    } else {
        *reinterpret_cast<float4*>(static_cast<float*>(base) + at) = make_float4(f[0], f[1], f[2], f[3]);
        *reinterpret_cast<float4*>(static_cast<float*>(base) + at + 4) = make_float4(f[4], f[5], f[6], f[7]);
    }
}

template <typename T>
__device__ __forceinline__ float load1(const void* base, long long at) {
    if constexpr (T::kBytes == 2) return __uint_as_float((uint32_t) static_cast<const uint16_t*>(base)[at] << 16);
    else return static_cast<const float*>(base)[at];
}
template <typename T>
__device__ __forceinline__ void store1(void* base, long long at, float f) {
    if constexpr (T::kBytes == 2) static_cast<__nv_bfloat16*>(base)[at] = __float2bfloat16_rn(f);
    else static_cast<float*>(base)[at] = f;
}

// Where row `row` goes in the pool: block (-1: nowhere) and token of the block.
template <int MODE>
__device__ __forceinline__ void rope_write_place(const RopeParams& p, int row, int& blk, int& off) {
    const int slot = __ldg(p.d_slots + row), at = __ldg(p.d_pos + row);
    blk = -1;
    off = at & (kBlockTokens - 1);
    if (at >= 0 && at / kBlockTokens < p.pv.table_stride) {
        blk = __ldg(p.pv.table + (size_t)slot * p.pv.table_stride + at / kBlockTokens);
        if (blk < 0 || blk >= p.pv.num_blocks) {
            if (p.status) atomicOr(p.status, kStatusBadBlock);
            blk = -1;
        }
    } else if (p.status) {
        atomicOr(p.status, kStatusBadSlot);
    }
}

// The append of row `row`, block-wide: one token per slot and call, for the first row that names the slot.  Thread 0 gets the place.
__device__ __forceinline__ void rope_append_place(const RopeParams& p, int row, int& blk, int& off) {
    const int slot = __ldg(p.d_slots + row);
    bool again = false;
    for (int j = threadIdx.x; j < row; j += blockDim.x) again |= __ldg(p.d_slots + j) == slot;
    again = __syncthreads_or(again);
    blk = -1;
    off = 0;
    if (threadIdx.x != 0) return;
    if (again) {
        if (p.status) atomicOr(p.status, kStatusBadSlot);
        return;
    }
    const int pfx = __ldg(p.d_prefill_len + slot);
    const int ring = ring_advance(p.d_len + slot, p.d_ring_pos + slot, pfx, p.window) - pfx;
    const int entry = (pfx + kBlockTokens - 1) / kBlockTokens + ring / kBlockTokens;
    off = ring & (kBlockTokens - 1);
    if (ring >= 0 && entry < p.pv.table_stride) blk = __ldg(p.pv.table + (size_t)slot * p.pv.table_stride + entry);
    else if (p.status) atomicOr(p.status, kStatusBadSlot);
    if (blk < 0 || blk >= p.pv.num_blocks) {
        if (p.status) atomicOr(p.status, kStatusBadBlock);
        blk = -1;
    }
}

// ROW: type of the q / k / v rows, KV: of the pool (ROW again where nothing goes to the pool).  Every chunk of 8 elements is
// 16-byte aligned and, in the half layout, lies in one half of the rotated dims.  Append: one row per CTA, 8 warps to a row.
// CTAs of an SM: the half layout takes 3, whose registers let the loads of a batch stay in flight (against 4: 8192 bf16 rows of
// 20 heads of 128 rotated in 19.0 us, not 21.5; 16384 / 8192 / 1537 bf16 rows of 10 + 10 + 10 heads written in 60.5 / 34.8 / 8.2,
// not 67.3 / 37.1 / 10.0, to an fp32 pool 77 for 88, although that one spills 100 bytes and the bf16 one 72; 1537 fp32 rows of 16 + 4
// heads of 64 written in 6.9, not 7.6; the one loss is 8192 fp32 rows of 20 heads of 128 rotated, 35.6, not 33.4).  Interleaved, 3
// would gain on small calls (1537 bf16 rows of 10 + 10 heads of 128 written in 6.7, not 7.4) and lose on large ones (8192 rows 30.4,
// not 28.1; 16384 rows 52.2, not 50.8): 4.
template <typename ROW, typename KV, int MODE, bool INTERLEAVED>
__global__ void __launch_bounds__(kRopeThreads, INTERLEAVED ? 4 : 3) rswa_rope_kernel(const __grid_constant__ RopeParams p) {
    constexpr int W = ROW::kBytes / 2;               // 16-byte words of a chunk
    constexpr int U = INTERLEAVED ? 4 / W : 2 / W;   // heads of a batch: 64 bytes of loads a lane
    constexpr int T = INTERLEAVED ? 4 : 8;           // pairs a lane's chunk takes part in
    __shared__ float2 tables[kRopeThreads / 32][kRopeMaxPairs];
    __shared__ int s_place[2];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int half = p.rotary_dim >> 1, hd = p.head_dim, per_head = p.per_head;
    const int parts = 1 << p.parts_log2, n_rot = p.heads + p.kv_heads;
    float2* tab = tables[warp];
    // This lane's chunk of a head and its first head: 32 / per_head heads side by side, wider heads in rounds of 32 chunks.
    const int abreast = per_head < 32 ? 32 / per_head : 1;
    const int my_head = per_head < 32 ? lane / per_head : 0;
    const int my_chunk = per_head < 32 ? lane - my_head * per_head : lane;

    const long long units = (long long)p.rows << p.parts_log2;
    for (long long unit = (long long)blockIdx.x * (kRopeThreads / 32) + warp; unit < units; unit += (long long)gridDim.x * (kRopeThreads / 32)) {
        const int row = (int)(unit >> p.parts_log2), part = (int)(unit & (parts - 1));
        const uint8_t* q_row = static_cast<const uint8_t*>(p.q) + row * p.q_stride * ROW::kBytes;
        const uint8_t* k_row = static_cast<const uint8_t*>(p.k) + (row * p.k_stride - (long long)p.heads * hd) * ROW::kBytes;  // (head h - heads)
        int blk = 0, off = 0;
        long long pool_row = 0;  // element of the row's token in head 0 of its block
        for (int j0 = 0; j0 == 0 || j0 < per_head; j0 += 32) {
            const int j = j0 + my_chunk;
            const int first = 8 * j;
            const bool pair = !INTERLEAVED && first < half;             // this chunk and the one `half` further on
            const int d = INTERLEAVED || pair ? first : half + first;   // half layout, beyond the rotated dims: 2 half + 8 (j - half / 8)
            const bool lane_on = j < per_head && my_head < abreast;
            uint4 a[U][W], z[U][INTERLEAVED ? 1 : W];
            auto load = [&](int h0) {
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int h = h0 + u * abreast * parts;
                    if (lane_on && h < n_rot) {
                        const uint4* s4 = reinterpret_cast<const uint4*>((h < p.heads ? q_row : k_row) + (h * hd + d) * ROW::kBytes);
#pragma unroll
                        for (int w = 0; w < W; ++w) a[u][w] = s4[w];
                        if constexpr (!INTERLEAVED)
                            if (pair) {
                                const uint4* g4 = reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(s4) + half * ROW::kBytes);
#pragma unroll
                                for (int w = 0; w < W; ++w) z[u][w] = g4[w];
                            }
                    }
                }
            };
            const int begin = part * abreast + my_head;
            load(begin);  // on their way while the table is filled
            if (j0 == 0) {
                const int position = __ldg(p.d_positions + row);
                if constexpr (MODE == kRopeWrite) rope_write_place<MODE>(p, row, blk, off);
                for (int i = lane; i < half; i += 32) {
                    float sn, c;
                    rope_sincos(p.turn[i], position, sn, c);
                    tab[i] = make_float2(c * p.amplitude, sn * p.amplitude);
                }
                if constexpr (MODE == kRopeAppend) {
                    rope_append_place(p, row, blk, off);
                    if (threadIdx.x == 0) {
                        s_place[0] = blk;
                        s_place[1] = off;
                    }
                    __syncthreads();
                    blk = s_place[0];
                    off = s_place[1];
                } else {
                    __syncwarp();
                }
                pool_row = ((long long)blk * p.kv_heads * kBlockTokens + off) * hd;
            }
            float2 turn[T];
#pragma unroll
            for (int e = 0; e < T; ++e) {
                const int i = INTERLEAVED ? first / 2 + e : first + e;
                turn[e] = i < half ? tab[i] : make_float2(1.f, 0.f);
            }
            for (int h0 = begin; __any_sync(0xffffffffu, lane_on && h0 < n_rot); h0 += U * abreast * parts) {
                if (h0 != begin) load(h0);
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int h = h0 + u * abreast * parts;
                    if (!lane_on || h >= n_rot) continue;
                    float x[8], y[8];
                    auto widen = [](const uint4 (&w)[W], float (&f)[8]) {
                        if constexpr (W == 1) {
                            ROW::unpack(w[0], f);
                        } else {
                            f[0] = __uint_as_float(w[0].x); f[1] = __uint_as_float(w[0].y); f[2] = __uint_as_float(w[0].z); f[3] = __uint_as_float(w[0].w);
                            f[4] = __uint_as_float(w[W - 1].x); f[5] = __uint_as_float(w[W - 1].y); f[6] = __uint_as_float(w[W - 1].z); f[7] = __uint_as_float(w[W - 1].w);
                        }
                    };
                    widen(a[u], x);
                    if constexpr (INTERLEAVED) {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (first / 2 + e < half) rope_turn(x[2 * e], x[2 * e + 1], turn[e]);
                    } else if (pair) {
                        widen(z[u], y);
#pragma unroll
                        for (int e = 0; e < 8; ++e) rope_turn(x[e], y[e], turn[e]);
                    }
                    auto put = [&](auto type, void* dst, long long at) {
                        using D = decltype(type);
                        store8<D>(dst, at, x);
                        if constexpr (!INTERLEAVED)
                            if (pair) store8<D>(dst, at + half, y);
                    };
                    if (h < p.heads) put(ROW{}, p.q_out, row * p.q_out_stride + h * hd + d);
                    else if constexpr (MODE == kRopeRows) put(ROW{}, p.k_out, row * p.k_out_stride + (h - p.heads) * hd + d);
                    else if (blk >= 0) put(KV{}, p.pv.k_pool, pool_row + (long long)(h - p.heads) * kBlockTokens * hd + d);
                }
            }
        }
        if constexpr (MODE != kRopeRows) {  // v: chunks of the row, not rotated (head_dim is a power of two here)
            if (blk >= 0) {
                constexpr int V = 4 / W;
                const int chunks = p.kv_heads * hd / 8, shift = 31 - __clz(hd / 8);
                const uint4* v_row = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(p.v) + row * p.v_stride * ROW::kBytes);
                for (int c0 = part * 32 + lane; c0 < chunks; c0 += V * 32 * parts) {
                    uint4 a[V][W];
#pragma unroll
                    for (int u = 0; u < V; ++u)
                        if (c0 + u * 32 * parts < chunks) {
#pragma unroll
                            for (int w = 0; w < W; ++w) a[u][w] = v_row[(c0 + u * 32 * parts) * W + w];
                        }
#pragma unroll
                    for (int u = 0; u < V; ++u) {
                        const int c = c0 + u * 32 * parts;
                        if (c >= chunks) continue;
                        const int head = c >> shift;
                        const long long at = pool_row + (long long)head * kBlockTokens * hd + (c - (head << shift)) * 8;
                        if constexpr (ROW::kBytes == KV::kBytes) {  // the bits as they are
#pragma unroll
                            for (int w = 0; w < W; ++w) reinterpret_cast<uint4*>(p.pv.v_pool + at * KV::kBytes)[w] = a[u][w];
                        } else if constexpr (W == 1) {
                            float x[8];
                            ROW::unpack(a[u][0], x);
                            store8<KV>(p.pv.v_pool, at, x);
                        } else {
                            const float x[8] = {__uint_as_float(a[u][0].x), __uint_as_float(a[u][0].y), __uint_as_float(a[u][0].z), __uint_as_float(a[u][0].w),
                                                __uint_as_float(a[u][W - 1].x), __uint_as_float(a[u][W - 1].y), __uint_as_float(a[u][W - 1].z), __uint_as_float(a[u][W - 1].w)};
                            store8<KV>(p.pv.v_pool, at, x);
                        }
                    }
                }
            }
        }
        __syncwarp();  // the table is free for the next row
    }
}

// Rows that are not made of aligned chunks: element by element, one row per CTA.
template <typename ROW, typename KV, int MODE>
__global__ void __launch_bounds__(kRopeThreads) rswa_rope_elements_kernel(const __grid_constant__ RopeParams p, bool interleaved) {
    __shared__ float2 tab[kRopeMaxPairs];
    __shared__ int s_place[2];
    const int tid = threadIdx.x;
    const int half = p.rotary_dim >> 1, hd = p.head_dim, per_head = p.per_head;
    const int rotated = (p.heads + p.kv_heads) * per_head;
    for (int row = blockIdx.x; row < p.rows; row += gridDim.x) {
        int blk = 0, off = 0;
        if constexpr (MODE == kRopeAppend) rope_append_place(p, row, blk, off);
        if constexpr (MODE == kRopeWrite)
            if (tid == 0) rope_write_place<MODE>(p, row, blk, off);
        if (tid == 0) {
            s_place[0] = blk;
            s_place[1] = off;
        }
        for (int i = tid; i < half; i += kRopeThreads) {
            float sn, c;
            rope_sincos(p.turn[i], __ldg(p.d_positions + row), sn, c);
            tab[i] = make_float2(c * p.amplitude, sn * p.amplitude);
        }
        __syncthreads();
        blk = s_place[0];
        off = s_place[1];
        auto pool_at = [&](int head, int d) { return (((long long)blk * p.kv_heads + head) * kBlockTokens + off) * hd + d; };
        for (int it = tid; it < p.items; it += kRopeThreads) {
            if (it >= rotated) {  // v: no rotation
                if constexpr (MODE != kRopeRows) {
                    const int head = (it - rotated) / hd, d = it - rotated - head * hd;
                    if (blk >= 0) store1<KV>(p.pv.v_pool, pool_at(head, d), load1<ROW>(p.v, row * p.v_stride + head * hd + d));
                }
                continue;
            }
            const int h = it / per_head, j = it - h * per_head;
            const bool is_k = h >= p.heads;
            const int head = is_k ? h - p.heads : h;
            const void* src = is_k ? p.k : p.q;
            const long long at = row * (is_k ? p.k_stride : p.q_stride) + head * hd;
            auto put = [&](int d, float f) {
                if (!is_k) store1<ROW>(p.q_out, row * p.q_out_stride + head * hd + d, f);
                else if constexpr (MODE == kRopeRows) store1<ROW>(p.k_out, row * p.k_out_stride + head * hd + d, f);
                else if (blk >= 0) store1<KV>(p.pv.k_pool, pool_at(head, d), f);
            };
            if (j < half) {
                const int d0 = interleaved ? 2 * j : j, d1 = interleaved ? 2 * j + 1 : j + half;
                float x0 = load1<ROW>(src, at + d0), x1 = load1<ROW>(src, at + d1);
                rope_turn(x0, x1, tab[j]);
                put(d0, x0);
                put(d1, x1);
            } else {
                put(half + j, load1<ROW>(src, at + half + j));
            }
        }
        __syncthreads();  // the table is free for the next row
    }
}

}  // namespace uocr_b200
