// lmvec.hpp -- 16-byte pieces of float32 or bfloat16 rows at any alignment, and the
// sums over a row's threads, for the HBM-bound language-model kernels.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace katsu {

typedef uint32_t lm_u4 __attribute__((ext_vector_type(4)));
typedef float lm_f2 __attribute__((ext_vector_type(2)));
typedef __bf16 lm_b2 __attribute__((ext_vector_type(2)));

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
// The same as it is in memory, in four registers.  From an array of values, as above, the compiler
// makes three accesses, one of which the one at a row's end, value by value, shares, and holds a
// register for each value of bfloat16.  Whole accesses are faster where the memory is all
// (130000 rows of 2 KB set to zero: 67 and 51 us; 16384 rows of 8 KB looked up: 53 and 40), not in
// the norms' gradient, which has no registers for what is then loaded early (114 and 136 us).
template <typename T>
struct RawPiece {
    static constexpr int E = Piece<T>::E;
    lm_u4 v;
    // Those outside the row's [first, n) are `none`, and not written.
    __device__ __forceinline__ void load(const T *p, int64_t i, int64_t n, float none = 0.f,
                                         int64_t first = INT64_MIN) {
        if (i >= first && i + E <= n) {
            __builtin_memcpy(&v, p + i, 16);
        } else {
            T e[E];
#pragma unroll
            for (int j = 0; j < E; ++j)
                e[j] = i + j >= first && i + j < n ? p[i + j] : (T)none;
            __builtin_memcpy(&v, e, 16);
        }
    }
    __device__ __forceinline__ void store(T *p, int64_t i, int64_t n,
                                          int64_t first = INT64_MIN) const {
        if (i >= first && i + E <= n) {
            __builtin_memcpy(p + i, &v, 16);
        } else {
#pragma unroll
            for (int j = 0; j < E; ++j)
                if (i + j >= first && i + j < n) p[i + j] = (T)at(j);
        }
    }
    // Its values are converted again after this: held as float32 they take twice the registers.
    __device__ __forceinline__ void packed() { asm volatile("" : "+v"(v)); }
    __device__ __forceinline__ float at(int j) const {
        const uint32_t u = v[j * (int)sizeof(T) / 4];
        return __builtin_bit_cast(float, sizeof(T) == 4 ? u : j & 1 ? u & 0xffff0000u : u << 16);
    }
    __device__ __forceinline__ void fill(float x) {
        float y[E];
#pragma unroll
        for (int j = 0; j < E; ++j) y[j] = x;
        set(y);
    }
    __device__ __forceinline__ void set(const float *x) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            uint32_t u;
            if constexpr (sizeof(T) == 4) {
                const float f = x[k];
                u = __builtin_bit_cast(uint32_t, f);
            } else {
                u = __builtin_bit_cast(
                    uint32_t, __builtin_convertvector(lm_f2{x[2 * k], x[2 * k + 1]}, lm_b2));
            }
            v[k] = u;
        }
    }
};
template <typename T>
__device__ __forceinline__ void load_whole(const T *p, int64_t i, int64_t n, float *x) {
    RawPiece<T> r;
    r.load(p, i, n);
#pragma unroll
    for (int j = 0; j < Piece<T>::E; ++j) x[j] = r.at(j);
}
template <typename T>
__device__ __forceinline__ void store_whole(T *p, int64_t i, int64_t n, const float *x) {
    RawPiece<T> r;
    r.set(x);
    r.store(p, i, n);
}

// N neighbouring values, of any alignment.
template <typename T, int N>
__device__ __forceinline__ void rotary_load(const T *p, float *x) {
    T e[N];
    __builtin_memcpy(e, p, sizeof e);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = (float)e[i];
}
template <typename T, int N>
__device__ __forceinline__ void rotary_store(T *p, const float *x) {
    T e[N];
#pragma unroll
    for (int i = 0; i < N; ++i) e[i] = (T)x[i];
    __builtin_memcpy(p, e, sizeof e);
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
