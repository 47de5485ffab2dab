// Building blocks of the split-KV kernels: how a line of work units is cut into pieces, the warp-level
// reduction of dot products, and packed fp32 arithmetic.
#pragma once

#include "rswa_device.cuh"

namespace uocr_b200 {

// How the unit line [0, total) is cut into pieces: one piece per warp of the persistent grid, consecutive
// and non-empty, so an item spans pieces of(first unit) .. of(last unit).
struct PieceMap {
    long long total;
    int ns;           // number of pieces: min(total warps, total units)
    int wpc;          // warps per CTA
    // Even split under launch overlap: the warps of the last CTA carry (16 - late) / 16 of a share.  CTAs of
    // an overlapped launch move in as their predecessor's CTAs leave, in block order, so the last block starts
    // several microseconds after the others (it cannot hide its prologue) and would finish last by as much.
    int late;
    long long wtot;   // sum of the piece weights (16 each, 16 - late for the last CTA's)
    __device__ __forceinline__ long long weight_before(int k) const {
        const int n1 = ns - wpc;
        return k <= n1 ? 16LL * k : 16LL * n1 + (long long)(16 - late) * (k - n1);
    }
    __device__ __forceinline__ long long start(int k) const {
        return late ? (total * weight_before(k)) / wtot : ((long long)k * total) / ns;
    }
    __device__ __forceinline__ long long end(int k) const { return k + 1 < ns ? start(k + 1) : total; }
    __device__ __forceinline__ int of(long long u) const {
        if (!late) return (int)(((u + 1) * ns - 1) / total);
        // the last piece whose weight prefix w satisfies floor(total * w / wtot) <= u
        const long long a = ((u + 1) * wtot - 1) / total;
        const int n1 = ns - wpc;
        if (a < 16LL * n1) return (int)(a / 16);
        const int k = n1 + (int)((a - 16LL * n1) / (16 - late));
        return k < ns ? k : ns - 1;
    }
};

constexpr int kPendMax = 4;  // per-warp list of partial segments awaiting their arrival (a piece leaves at most two)

// Whether the uneven (late-CTA) split applies to a launch: enough units that no piece can be empty and few
// enough that the bounds fit the arithmetic.
__device__ __forceinline__ bool uneven_split_ok(long long total, int total_warps) {
    return total >= 8LL * total_warps && total < (1LL << 26);
}

__device__ __forceinline__ PieceMap make_piece_map(long long total, int total_warps, int wpc, int late = 0) {
    PieceMap m;
    m.total = total;
    m.wpc = wpc;
    m.late = 0;
    m.wtot = 0;
    m.ns = (int)min((long long)total_warps, total);
    if (late > 0 && m.ns == total_warps && m.ns > wpc && uneven_split_ok(total, total_warps)) {
        m.late = min(late, 12);
        m.wtot = 16LL * m.ns - (long long)m.late * wpc;
    }
    return m;
}

// -------------------------------------------------------------------------------------------------
// reduce-scatter of N per-lane partial sums across the D*2 lanes that share a cache row:
// afterwards every lane holds one complete sum in v[0]
// -------------------------------------------------------------------------------------------------
template <int N, int D>
struct RowReduce {
    template <int ITER>
    __device__ static __forceinline__ void run(float (&v)[ITER], int lane) {
        if constexpr (D >= 1) {
            if constexpr (N > 1) {
                const bool upper = (lane & D) != 0;
#pragma unroll
                for (int k = 0; k < N / 2; ++k) {
                    const float send = upper ? v[k] : v[k + N / 2];
                    const float keep = upper ? v[k + N / 2] : v[k];
                    v[k] = keep + __shfl_xor_sync(0xffffffffu, send, D);
                }
                RowReduce<N / 2, D / 2>::run(v, lane);
            } else {
                v[0] += __shfl_xor_sync(0xffffffffu, v[0], D);
                RowReduce<1, D / 2>::run(v, lane);
            }
        }
    }
};

__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// packed fp32x2 arithmetic: one instruction per two lanes of the dot products and accumulators
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }

template <typename KV>
__device__ __forceinline__ void unpack2(const uint4& w, float2 (&f)[KV::kPerChunk / 2]) {
    if constexpr (KV::kBytes == 2) {
        f[0] = make_float2(bf16_lo(w.x), bf16_hi(w.x));
        f[1] = make_float2(bf16_lo(w.y), bf16_hi(w.y));
        f[2] = make_float2(bf16_lo(w.z), bf16_hi(w.z));
        f[3] = make_float2(bf16_lo(w.w), bf16_hi(w.w));
    } else {
        f[0] = make_float2(__uint_as_float(w.x), __uint_as_float(w.y));
        f[1] = make_float2(__uint_as_float(w.z), __uint_as_float(w.w));
    }
}

}  // namespace uocr_b200
