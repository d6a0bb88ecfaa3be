// gradclip.hpp -- the global norm of many gradient tensors, and clipping by it:
//   norm = sqrt(sum of all squares),  out = g min(1, max_norm / (norm + 1e-6))
//
// Two launches for up to kClipTensors tensors, whose addresses travel as kernel
// arguments: the first sums squares into one float64 part a block, the second has every
// block add the parts in the same order and scale its share.  Squares are summed in
// float64: they cannot overflow, and HBM is the bound either way (one fused
// multiply-add for 2 or 4 bytes read).  770 M bfloat16 values, not in place: 878 us, the sums
// 274 (5.6 TB/s), the scaling 594 (5.2); 3.0 M float32 values in 26 tensors: 13.5 us of launches.
#pragma once

#include "lmvec.hpp"

namespace katsu {

constexpr int kClipTensors = 128;  // 3.7 KB of kernel arguments
constexpr int kClipBlocks = 1024, kClipChunk = 16384;  // blocks at most; values a step

struct ClipTable {
    const void *in[kClipTensors];
    void *out[kClipTensors];
    int64_t count[kClipTensors];
    uint32_t first[kClipTensors + 1];  // chunks before each tensor
    uint8_t half[kClipTensors];        // bfloat16
    int n;
};

// Calls f(tensor, first value, values) for this block's chunks; BACK: the last ones first.
template <bool BACK, class F>
__device__ __forceinline__ void each_chunk(const ClipTable &t, F f) {
    const uint32_t total = t.first[t.n];
    int k = BACK ? t.n - 1 : 0;
    for (uint32_t i = blockIdx.x; i < total; i += gridDim.x) {
        const uint32_t c = BACK ? total - 1 - i : i;
        while (BACK ? t.first[k] > c : t.first[k + 1] <= c) k += BACK ? -1 : 1;
        const int64_t at = (int64_t)(c - t.first[k]) * kClipChunk;
        const int64_t left = t.count[k] - at;
        f(k, at, left < kClipChunk ? (int)left : kClipChunk);
    }
}

// Eight pieces are read before the first is squared; whole chunks need no bounds.
template <typename T>
__device__ __forceinline__ double squares(const T *p, int n) {
    constexpr int E = Piece<T>::E, U = 8;
    static_assert(kClipChunk % (256 * E * U) == 0, "whole steps");
    double s[2] = {0., 0.};
    for (int i = threadIdx.x * E; i < n; i += 256 * E * U) {
        float x[U][E];
        if (n == kClipChunk) {
#pragma unroll
            for (int u = 0; u < U; ++u) load_piece(p, i + u * 256 * E, INT64_MAX, x[u]);
        } else {
#pragma unroll
            for (int u = 0; u < U; ++u) load_piece(p, i + u * 256 * E, n, x[u]);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < E; ++e)
                s[e & 1] = __builtin_fma((double)x[u][e], (double)x[u][e], s[e & 1]);
    }
    return s[0] + s[1];
}
// Four pieces are read before the first is written: p and q may be the same memory, so the
// compiler would wait for each in turn (770 M bfloat16 values: 903 us against 573).
template <typename T>
__device__ __forceinline__ void scale_chunk(const T *p, T *q, int n, float by) {
    constexpr int E = Piece<T>::E, U = 4;
    for (int i = threadIdx.x * E; i < n; i += 256 * E * U) {
        float x[U][E];
#pragma unroll
        for (int u = 0; u < U; ++u) load_piece(p, i + u * 256 * E, n, x[u]);
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int e = 0; e < E; ++e) x[u][e] *= by;
            store_piece(q, i + u * 256 * E, n, x[u]);
        }
    }
}
__device__ __forceinline__ double block_sum_f64(double v, double *part) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    return ((part[0] + part[1]) + part[2]) + part[3];
}

__global__ void __launch_bounds__(256) clip_squares_kernel(const ClipTable t, double *parts) {
    __shared__ double part[4];
    double s = 0.;
    each_chunk<false>(t, [&](int k, int64_t at, int n) {
        s += t.half[k] ? squares((const __bf16 *)t.in[k] + at, n)
                       : squares((const float *)t.in[k] + at, n);
    });
    s = block_sum_f64(s, part);
    if (threadIdx.x == 0) parts[blockIdx.x] = s;
}

__global__ void __launch_bounds__(256) clip_scale_kernel(const ClipTable t, const double *parts,
                                                         int nparts, float max_norm, float *norm) {
    __shared__ double part[4];
    double s = 0.;
    for (int i = threadIdx.x; i < nparts; i += 256) s += parts[i];
    s = sqrt(block_sum_f64(s, part));
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)s;
    const double q = (double)max_norm / (s + 1e-6);
    const float by = q >= 1. ? 1.f : (float)q;  // a norm that is NaN gives NaN
    // Backwards: what the sums read last is in the 256 MB cache still.
    each_chunk<true>(t, [&](int k, int64_t at, int n) {
        if (by == 1.f && t.in[k] == t.out[k]) return;  // in place, nothing to do
        if (t.half[k])
            scale_chunk((const __bf16 *)t.in[k] + at, (__bf16 *)t.out[k] + at, n, by);
        else
            scale_chunk((const float *)t.in[k] + at, (float *)t.out[k] + at, n, by);
    });
}

}  // namespace katsu
