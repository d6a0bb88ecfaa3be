// lmvec.hpp -- 16-byte pieces of float32 or bfloat16 rows at any alignment, and the
// sums over a row's threads, for the HBM-bound language-model kernels.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace katsu {

typedef uint32_t lm_u4 __attribute__((ext_vector_type(4)));

// E neighbouring values as float32.
template <typename T>
struct Piece {
    static constexpr int E = 16 / (int)sizeof(T);
};
// Values [i, i + E) of a row of n; those past its end are zero.  Global memory takes
// 16-byte accesses at any address (rows of an odd number of bfloat16 too).
template <typename T>
__device__ __forceinline__ void load_piece(const T *p, int64_t i, int64_t n, float *x) {
    constexpr int E = Piece<T>::E;
    T e[E];
    if (i + E <= n) {
        __builtin_memcpy(e, p + i, 16);
    } else {
#pragma unroll
        for (int j = 0; j < E; ++j) e[j] = i + j < n ? p[i + j] : (T)0.f;
    }
#pragma unroll
    for (int j = 0; j < E; ++j) x[j] = (float)e[j];
}
template <typename T>
__device__ __forceinline__ void store_piece(T *p, int64_t i, int64_t n, const float *x) {
    constexpr int E = Piece<T>::E;
    T e[E];
#pragma unroll
    for (int j = 0; j < E; ++j) e[j] = (T)x[j];
    if (i + E <= n) {
        __builtin_memcpy(p + i, e, 16);
    } else {
#pragma unroll
        for (int j = 0; j < E; ++j)
            if (i + j < n) p[i + j] = e[j];
    }
}

// The sum over a row's TPR threads (a wave, or a whole block), the same in each: a
// fixed tree.  Each call of a block uses its own slot of `part`.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float *part) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    if constexpr (TPR > 64) {
        constexpr int W = TPR / 64;
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) part[wave] = v;
        __syncthreads();
        v = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) v += part[w];
    }
    return v;
}

}  // namespace katsu
