// blocknorm.hpp -- what lies between two blocks of a model: the norm after a block, its
// gate and residual scale, the residual sum, and the norm before the next block.
//
//   n = o r_o w_post,  r_o = 1/sqrt(mean(o^2) + eps)       (n = o without w_post)
//   y = x + alpha gate n
//   h = y r_y w_pre,   r_y = 1/sqrt(mean(y^2) + eps)       (none without w_pre)
//
// HBM-bound: a row stays in the registers of its threads between the two sums, so each
// operand is read once and each result written once (4096 x 2048 float32, a gate for each
// channel: 25.8 us, 5.2 TB/s; a copy reaches 4.7).  h is of the y before it is rounded.
#pragma once

#include "lmvec.hpp"

namespace katsu {

struct NormArgs {
    const void *x, *o, *gate, *w_post, *w_pre;
    void *y, *h;
    float *stats;  // [2][rows]: r_o (0 without w_post), r_y (0 without w_pre)
    int64_t rows, cols, gate_row;  // gate_row: 0 (one gate a channel) or cols
    float alpha, eps, inv_cols;
};

template <typename T, int TPR, int NV>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR) block_norm_kernel(const NormArgs a) {
    constexpr int E = Piece<T>::E, RPB = TPR < 256 ? 256 / TPR : 1;
    __shared__ float part[2][16];
    const int64_t block = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
    const int64_t row = block * RPB + (RPB > 1 ? threadIdx.x / TPR : 0);
    const int lane = threadIdx.x % TPR;
    if (row >= a.rows) return;  // a whole wave, or (one row a block) all of it
    const T *x = (const T *)a.x + row * a.cols, *o = (const T *)a.o + row * a.cols;
    const T *gate = a.gate ? (const T *)a.gate + row * a.gate_row : nullptr;
    float u[NV][E], v[NV][E];
    float ss = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int64_t i = ((int64_t)k * TPR + lane) * E;
        load_piece(o, i, a.cols, u[k]);
        load_piece(x, i, a.cols, v[k]);
#pragma unroll
        for (int e = 0; e < E; ++e) ss += u[k][e] * u[k][e];
    }
    float r_o = 0.f;
    if (a.w_post) r_o = rsqrtf(row_sum<TPR>(ss, part[0]) * a.inv_cols + a.eps);
    ss = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int64_t i = ((int64_t)k * TPR + lane) * E;
        float w[E];
        if (a.w_post) {
            load_piece((const T *)a.w_post, i, a.cols, w);
#pragma unroll
            for (int e = 0; e < E; ++e) u[k][e] = u[k][e] * r_o * w[e];
        }
        if (gate) {
            load_piece(gate, i, a.cols, w);
#pragma unroll
            for (int e = 0; e < E; ++e) u[k][e] *= w[e];
        }
#pragma unroll
        for (int e = 0; e < E; ++e) {
            v[k][e] += a.alpha * u[k][e];
            ss += v[k][e] * v[k][e];
        }
        store_piece((T *)a.y + row * a.cols, i, a.cols, v[k]);
    }
    float r_y = 0.f;
    if (a.w_pre) {
        r_y = rsqrtf(row_sum<TPR>(ss, part[1]) * a.inv_cols + a.eps);
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int64_t i = ((int64_t)k * TPR + lane) * E;
            float w[E];
            load_piece((const T *)a.w_pre, i, a.cols, w);
#pragma unroll
            for (int e = 0; e < E; ++e) v[k][e] = v[k][e] * r_y * w[e];
            store_piece((T *)a.h + row * a.cols, i, a.cols, v[k]);
        }
    }
    if (lane == 0 && a.stats) {
        a.stats[row] = r_o;
        a.stats[a.rows + row] = r_y;
    }
}

// Backward, from dy, dh and what the forward call left (y, o, stats):
//   yn = y r_y, g' = dh w_pre:   dx = dy + r_y (g' - yn mean(g' yn))
//   on = o r_o, g' = alpha gate dx w_post:   do = r_o (g' - on mean(g' on))
//   dgate = alpha dx n,  dw_post = sum alpha gate dx on,  dw_pre = sum dh yn
// A thread's columns are the same in every row it takes, so the sums over rows stay in
// its registers, one part for each set of rows; block_norm_sum_kernel adds the parts.
// 8192 x 4096 bfloat16, a gate for each element: 113.5 us, 4.7 TB/s (188 with two pieces a
// thread: half as many waves to a CU).
struct NormBwdArgs {
    const void *dy, *dh, *y, *o, *gate, *w_post, *w_pre;
    const float *stats;
    void *dx, *d_o, *dgate;
    float *part;  // [sets][sums][cols]: dw_pre, dw_post, dgate of one gate a channel
    int64_t rows, cols, gate_row;
    int sets, sums, at_post, at_gate;
    float alpha, inv_cols;
};

template <typename T, int TPR, int NV>
__global__ void __launch_bounds__(TPR == 64 ? 256 : TPR) block_norm_bwd_kernel(
    const NormBwdArgs a) {
    constexpr int E = Piece<T>::E, RPB = TPR == 64 ? 4 : 1;
    __shared__ float part[2][2][16];
    const int set = blockIdx.x * RPB + (RPB > 1 ? threadIdx.x / TPR : 0);
    const int lane = threadIdx.x % TPR;
    if (set >= a.sets) return;  // a whole wave, or never (one set a block)
    float wpre[NV][E] = {}, wpost[NV][E] = {}, gch[NV][E] = {};
    float s_pre[NV][E] = {}, s_post[NV][E] = {}, s_gate[NV][E] = {};
    const bool channel = a.gate && a.gate_row == 0;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int64_t i = ((int64_t)k * TPR + lane) * E;
        if (a.w_pre) load_piece((const T *)a.w_pre, i, a.cols, wpre[k]);
        if (a.w_post) load_piece((const T *)a.w_post, i, a.cols, wpost[k]);
        if (channel) load_piece((const T *)a.gate, i, a.cols, gch[k]);
    }
    int turn = 0;
    for (int64_t row = set; row < a.rows; row += a.sets, turn ^= 1) {
        const int64_t at = row * a.cols;
        const float r_o = a.w_post ? a.stats[row] : 1.f, r_y = a.stats[a.rows + row];
        float gx[NV][E], yn[NV][E], dh[NV][E], on[NV][E], g[NV][E];
        float ss = 0.f;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int64_t i = ((int64_t)k * TPR + lane) * E;
            load_piece((const T *)a.dy + at, i, a.cols, gx[k]);
            load_piece((const T *)a.o + at, i, a.cols, on[k]);
            if (a.w_pre) {
                load_piece((const T *)a.dh + at, i, a.cols, dh[k]);
                load_piece((const T *)a.y + at, i, a.cols, yn[k]);
            }
            if (a.gate && !channel) load_piece((const T *)a.gate + at, i, a.cols, g[k]);
        }
        if (a.w_pre) {
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    yn[k][e] *= r_y;
                    s_pre[k][e] += dh[k][e] * yn[k][e];
                    dh[k][e] *= wpre[k][e];
                    ss += dh[k][e] * yn[k][e];
                }
            const float c = row_sum<TPR>(ss, part[turn][0]) * a.inv_cols;
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int e = 0; e < E; ++e) gx[k][e] += r_y * (dh[k][e] - yn[k][e] * c);
        }
        ss = 0.f;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int64_t i = ((int64_t)k * TPR + lane) * E;
            store_piece((T *)a.dx + at, i, a.cols, gx[k]);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                on[k][e] *= r_o;
                const float ag = a.alpha * gx[k][e];
                const float gt = channel ? gch[k][e] : a.gate ? g[k][e] : 1.f;
                const float n = a.w_post ? on[k][e] * wpost[k][e] : on[k][e];
                g[k][e] = ag * n;                        // dgate
                s_gate[k][e] += ag * n;
                gx[k][e] = ag * gt;                      // of n
                s_post[k][e] += gx[k][e] * on[k][e];
                if (a.w_post) gx[k][e] *= wpost[k][e];
                ss += gx[k][e] * on[k][e];
            }
            if (a.gate && !channel) store_piece((T *)a.dgate + at, i, a.cols, g[k]);
        }
        const float c = a.w_post ? row_sum<TPR>(ss, part[turn][1]) * a.inv_cols : 0.f;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int64_t i = ((int64_t)k * TPR + lane) * E;
            if (a.w_post) {
#pragma unroll
                for (int e = 0; e < E; ++e) gx[k][e] = r_o * (gx[k][e] - on[k][e] * c);
            }
            store_piece((T *)a.d_o + at, i, a.cols, gx[k]);
        }
    }
    float *p = a.part + (int64_t)set * a.sums * a.cols;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int64_t i = ((int64_t)k * TPR + lane) * E;
#pragma unroll
        for (int e = 0; e < E; e += 4) {
            if (a.w_pre) store_piece<float>(p, i + e, a.cols, s_pre[k] + e);
            if (a.w_post) store_piece<float>(p + a.at_post * a.cols, i + e, a.cols, s_post[k] + e);
            if (channel) store_piece<float>(p + a.at_gate * a.cols, i + e, a.cols, s_gate[k] + e);
        }
    }
}

// Column sums of the parts, in order within each of a block's 16 waves, then the waves'.
// `sums` of w_pre, w_post (null if there is none) and, if it is one more, gate.
template <typename T>
__global__ void __launch_bounds__(1024) block_norm_sum_kernel(const float *part, int sets,
                                                             int64_t cols, int sums, T *w_pre,
                                                             T *w_post, T *gate) {
    __shared__ float s[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, which = blockIdx.y;
    const int64_t c = (int64_t)blockIdx.x * 64 + lane;
    float v = 0.f;
    if (c < cols) {
#pragma unroll 8
        for (int i = wave; i < sets; i += 16) v += part[((int64_t)i * sums + which) * cols + c];
    }
    s[wave][lane] = v;
    __syncthreads();
    if (wave != 0 || c >= cols) return;
    v = s[0][lane];
#pragma unroll
    for (int w = 1; w < 16; ++w) v += s[w][lane];
    const int n = (w_pre != nullptr) + (w_post != nullptr);
    T *out = which == 0 && w_pre ? w_pre : which < n ? w_post : gate;
    out[c] = (T)v;
}

}  // namespace katsu
