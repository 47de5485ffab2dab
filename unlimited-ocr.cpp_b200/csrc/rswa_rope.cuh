// Rotary positions for packed query / key rows, on their own or fused with the write of K and V into the
// paged cache (fixed region, or the ring append of single tokens).
//
// A pair (x0, x1) of a head turns by angle = position * freq_i:  (x0 c - x1 s, x0 s + x1 c), times an
// amplitude.  Angles of far positions lose everything in fp32 (position 10^6 times freq 1 is only known to
// 0.06 rad), so they are kept as 64-bit fixed-point fractions of a turn: freq_i / 2 pi is rounded once to
// 2^-64 turns on the host and position * that, modulo 2^64, is the exact fraction of the product -- one
// integer multiply, good to 2^-33 turns for any 32-bit position.  What is left after the quadrant is taken
// off is at most an eighth of a turn and goes to sincospi in fp32.
//
// The kernel moves bytes (q, k, v in; q and the pool rows out) and is bound by HBM.  A CTA takes four rows
// at a time: 256 threads first fill the rows' cosine / sine table in shared memory (one entry per pair of
// one head, used by all heads), then run over the rows' 16-byte chunks.  In the half layout a thread owns
// a chunk and its partner rotary_dim / 2 further on, in the interleaved layout a chunk holds whole pairs;
// every element is read and written by one thread, so a call may work in place.
#pragma once

#include "rswa_paged.cuh"

namespace uocr_b200 {

constexpr int kRopeMaxPairs = 128;  // rotary_dim <= 256
constexpr int kRopeThreads = 256;

enum RopeMode : int { kRopeRows = 0, kRopeWrite = 1, kRopeAppend = 2 };

// n / d for n * d < 2^32, as a multiply
struct FastDiv {
    uint32_t d, m;
};
__device__ __forceinline__ uint32_t fast_div(uint32_t n, const FastDiv& f) { return f.d == 1 ? n : __umulhi(n, f.m); }

struct RopeParams {
    unsigned long long turn[kRopeMaxPairs];  // freq_i / 2 pi in units of 2^-64 turns
    float amplitude;
    int interleaved, rotary_dim;
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
    int rows_per_cta;
    FastDiv per_row, per_head, per_v;  // work items of a row, of a rotated head, of a head of v
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
__device__ __forceinline__ void load8(const void* base, long long at, float (&f)[8]) {
    if constexpr (T::kBytes == 2) {
        const uint4 w = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + at);
        T::unpack(w, f);
    } else {
        const float4 a = *reinterpret_cast<const float4*>(static_cast<const float*>(base) + at);
        const float4 b = *reinterpret_cast<const float4*>(static_cast<const float*>(base) + at + 4);
        f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
        f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
    }
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

// ROW: type of the q / k / v rows, KV: of the pool (ROW again where nothing goes to the pool).
// VEC: every chunk of 8 elements is 16-byte aligned and lies in one half of the rotated dims; otherwise element by element.
template <typename ROW, typename KV, int MODE, bool VEC>
__global__ void __launch_bounds__(kRopeThreads) rswa_rope_kernel(const __grid_constant__ RopeParams p) {
    constexpr int kMaxRows = 4;
    __shared__ float2 cs[kMaxRows * kRopeMaxPairs];
    __shared__ int s_blk[kMaxRows], s_off[kMaxRows];
    const int tid = threadIdx.x;
    const int half = p.rotary_dim >> 1, hd = p.head_dim;
    const int rotated = (p.heads + p.kv_heads) * (int)p.per_head.d;

    for (int row0 = blockIdx.x * p.rows_per_cta; row0 < p.rows; row0 += gridDim.x * p.rows_per_cta) {
        const int nrows = min(p.rows_per_cta, p.rows - row0);
        if constexpr (MODE == kRopeAppend) {  // one row per CTA
            const int slot = __ldg(p.d_slots + row0);
            bool again = false;  // an earlier row of the batch appends to this slot: one token per slot and call
            for (int j = tid; j < row0; j += kRopeThreads) again |= __ldg(p.d_slots + j) == slot;
            again = __syncthreads_or(again);
            if (tid == 0) {
                int blk = -1, off = 0;
                if (again) {
                    if (p.status) atomicOr(p.status, kStatusBadSlot);
                } else {
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
                s_blk[0] = blk;
                s_off[0] = off;
            }
        }
        if constexpr (MODE == kRopeWrite) {
            if (tid < nrows) {
                const int slot = __ldg(p.d_slots + row0 + tid), at = __ldg(p.d_pos + row0 + tid);
                int blk = -1;
                if (at >= 0 && at / kBlockTokens < p.pv.table_stride) {
                    blk = __ldg(p.pv.table + (size_t)slot * p.pv.table_stride + at / kBlockTokens);
                    if (blk < 0 || blk >= p.pv.num_blocks) {
                        if (p.status) atomicOr(p.status, kStatusBadBlock);
                        blk = -1;
                    }
                } else if (p.status) {
                    atomicOr(p.status, kStatusBadSlot);
                }
                s_blk[tid] = blk;
                s_off[tid] = at & (kBlockTokens - 1);
            }
        }
        for (int i = tid; i < nrows * half; i += kRopeThreads) {
            const int r = i / half, j = i - r * half;
            float sn, c;
            rope_sincos(p.turn[j], __ldg(p.d_positions + row0 + r), sn, c);
            cs[r * kRopeMaxPairs + j] = make_float2(c * p.amplitude, sn * p.amplitude);
        }
        __syncthreads();

        const int items = nrows * (int)p.per_row.d;
        for (int it = tid; it < items; it += kRopeThreads) {
            const int r = nrows == 1 ? 0 : (int)fast_div(it, p.per_row);
            const int rem = it - r * (int)p.per_row.d;
            const long long row = row0 + r;
            int blk = 0, off = 0;
            if constexpr (MODE != kRopeRows) {
                blk = s_blk[r];
                off = s_off[r];
            }
            auto pool_at = [&](int head, int d) {
                return (((long long)blk * p.kv_heads + head) * kBlockTokens + off) * hd + d;
            };
            if (rem >= rotated) {  // v: no rotation
                if constexpr (MODE != kRopeRows) {
                    const int x = rem - rotated;
                    const int head = (int)fast_div(x, p.per_v), j = x - head * (int)p.per_v.d;
                    if (blk < 0) continue;
                    if constexpr (VEC) {
                        float f[8];
                        load8<ROW>(p.v, row * p.v_stride + head * hd + 8 * j, f);
                        store8<KV>(p.pv.v_pool, pool_at(head, 8 * j), f);
                    } else {
                        store1<KV>(p.pv.v_pool, pool_at(head, j), load1<ROW>(p.v, row * p.v_stride + head * hd + j));
                    }
                }
                continue;
            }
            const int h = (int)fast_div(rem, p.per_head), j = rem - h * (int)p.per_head.d;
            const bool is_k = h >= p.heads;
            const int head = is_k ? h - p.heads : h;
            const void* src = is_k ? p.k : p.q;
            const long long at = row * (is_k ? p.k_stride : p.q_stride) + head * hd;
            const float2* tab = cs + r * kRopeMaxPairs;
            auto put8 = [&](int d, const float (&f)[8]) {
                if (!is_k) store8<ROW>(p.q_out, row * p.q_out_stride + head * hd + d, f);
                else if constexpr (MODE == kRopeRows) store8<ROW>(p.k_out, row * p.k_out_stride + head * hd + d, f);
                else if (blk >= 0) store8<KV>(p.pv.k_pool, pool_at(head, d), f);
            };
            auto put1 = [&](int d, float f) {
                if (!is_k) store1<ROW>(p.q_out, row * p.q_out_stride + head * hd + d, f);
                else if constexpr (MODE == kRopeRows) store1<ROW>(p.k_out, row * p.k_out_stride + head * hd + d, f);
                else if (blk >= 0) store1<KV>(p.pv.k_pool, pool_at(head, d), f);
            };
            if constexpr (VEC) {
                float a[8];
                if (p.interleaved) {
                    load8<ROW>(src, at + 8 * j, a);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int i = 4 * j + e;
                        if (i < half) rope_turn(a[2 * e], a[2 * e + 1], tab[i]);
                    }
                    put8(8 * j, a);
                } else if (8 * j < half) {
                    float b[8];
                    load8<ROW>(src, at + 8 * j, a);
                    load8<ROW>(src, at + half + 8 * j, b);
#pragma unroll
                    for (int e = 0; e < 8; ++e) rope_turn(a[e], b[e], tab[8 * j + e]);
                    put8(8 * j, a);
                    put8(half + 8 * j, b);
                } else {
                    load8<ROW>(src, at + half + 8 * j, a);  // beyond the rotated dims: 2 * half + 8 * (j - half / 8)
                    put8(half + 8 * j, a);
                }
            } else {
                if (j < half) {
                    const int d0 = p.interleaved ? 2 * j : j, d1 = p.interleaved ? 2 * j + 1 : j + half;
                    float x0 = load1<ROW>(src, at + d0), x1 = load1<ROW>(src, at + d1);
                    rope_turn(x0, x1, tab[j]);
                    put1(d0, x0);
                    put1(d1, x1);
                } else {
                    put1(half + j, load1<ROW>(src, at + half + j));
                }
            }
        }
        __syncthreads();  // the table is free for the next rows
    }
}

}  // namespace uocr_b200
