// headnorm.hpp -- each query and key head divided by its root mean square, times a weight
// for each channel, and its first R channels turned by the token's position, in one pass:
//
//   r = 1/sqrt(mean(x^2) + eps),  n = x r w,  y = turn(n)       (the turn as in rotary.hpp)
//
// and its gradient, with g = the gradient of y turned back:
//   dw = sum over tokens and heads of g x r,  dx = r g w - x r^3 mean(g w x)
// where both of a head's sums are taken at once.  Squares are float32: a head with values beyond
// 1.8e19 becomes 0, and without eps one of values below 1e-19 is inexact or infinite.
//
// A head stays in its lanes' registers, so each operand is read once and each result written once:
// HBM-bound where heads are many (the gradient of 16384 tokens, 32 + 8 heads of 128, bfloat16: 110
// us, 4.6 TB/s).  8192 tokens, 16 + 4 heads: 24.4 us, 3.7 TB/s (a copy of as much takes 19.1), vector
// instructions 62% of the time; 18.4 where the caches hold the outputs.  The gradient of 6000
// tokens, 16 + 4: 24.4 us, vector instructions 68% of the time, and 4 for the sums of dw.
#pragma once

#include "lmvec.hpp"

namespace katsu {

constexpr int kHeadThreads = 256;  // of a block of the gradient

// One of q and k.
struct HeadTensor {
    const void *x, *w, *dy;  // dy: the gradient of the output (backward)
    void *out;               // output, or the gradient of x
    int64_t x_token, x_head, dy_token, dy_head, out_token, out_head;
    int heads;
};
struct HeadArgs {
    HeadTensor t[2];  // q and k
    const float *table;
    const int32_t *positions;  // NULL: 0, 1, ..
    int64_t tokens, length;
    int D, R, units;           // units of 2E channels of a head
    uint64_t inv[3];           // head_inv of q's heads, k's, both
    float eps, inv_d;
    float *part;               // backward, [blocks][D]: sums of dw, q's blocks first
    int blocks[2];             // backward: blocks of q, of k
};

// E neighbouring values as they are in memory.
template <typename T, int E>
struct HeadPacked {
    uint32_t w[(E * sizeof(T) + 3) / 4] = {};
    __device__ __forceinline__ void load(const T *p) { __builtin_memcpy(w, p, E * sizeof(T)); }
    __device__ __forceinline__ float at(int e) const {
        const uint32_t u = w[e * (int)sizeof(T) / 4];
        return __builtin_bit_cast(float, sizeof(T) == 4 ? u : e & 1 ? u & 0xffff0000u : u << 16);
    }
};

// A head is units of 2E channels: E pairs (R/2 apart, or 2E neighbours with INTER) for the
// part that turns, then two pieces of E neighbours of the rest.  E divides R/2 and the rest,
// whose last unit may have one piece only.
template <typename T, bool INTER, int E>
struct HeadUnit {
    int c[2];      // its pieces' first channels
    bool has[2];
    bool turns;
    int angle;     // its first pair

    __device__ __forceinline__ void init(const HeadArgs &a, int u) {
        const int half = a.R / 2, turning = half / E;
        turns = u < turning;
        angle = u * E;
        if (turns) {
            c[0] = INTER ? 2 * u * E : u * E;
            c[1] = INTER ? c[0] + E : half + u * E;
        } else {
            c[0] = a.R + (u - turning) * 2 * E;
            c[1] = c[0] + E;
        }
        has[0] = u < a.units;
        has[1] = has[0] && c[1] < a.D;
    }
    __device__ __forceinline__ void load(const void *p, int64_t at, float (&x)[2][E]) const {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (has[i])
                rotary_load<T, E>((const T *)p + at + c[i], x[i]);
            else
#pragma unroll
                for (int e = 0; e < E; ++e) x[i][e] = 0.f;
    }
    // As it is in memory, for heads that wait.
    __device__ __forceinline__ void load(const void *p, int64_t at, HeadPacked<T, E> (&x)[2]) const {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (has[i]) x[i].load((const T *)p + at + c[i]);
    }
    __device__ __forceinline__ void store(void *p, int64_t at, const float (&x)[2][E]) const {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (has[i]) rotary_store<T, E>((T *)p + at + c[i], x[i]);
    }
    __device__ __forceinline__ void angles(const float *row, int R, float (&cs)[2][E]) const {
        if (!turns) return;
        rotary_load<float, E>(row + angle, cs[0]);
        rotary_load<float, E>(row + R / 2 + angle, cs[1]);
    }
    // sign: -1 turns back.
    __device__ __forceinline__ void turn(float (&x)[2][E], const float (&cs)[2][E],
                                         float sign) const {
        if (!turns) return;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            // INTER: pair e is the unit's channels 2e and 2e + 1.
            const int i0 = INTER ? (2 * e) / E : 0, e0 = INTER ? (2 * e) % E : e;
            const int i1 = INTER ? (2 * e + 1) / E : 1, e1 = INTER ? (2 * e + 1) % E : e;
            const float u = x[i0][e0], v = x[i1][e1], c = cs[0][e], s = sign * cs[1][e];
            x[i0][e0] = u * c - v * s;
            x[i1][e1] = u * s + v * c;
        }
    }
};

// A token's position as it is given; 0 beyond the last token.
__device__ __forceinline__ int64_t head_position(const HeadArgs &a, int64_t token) {
    return !a.positions ? token : token < a.tokens ? a.positions[token] : 0;
}
// Where its angles begin: inside the table.
__device__ __forceinline__ int64_t head_row(const HeadArgs &a, int64_t pos) {
    return (pos < 0 ? 0 : pos < a.length ? pos : a.length - 1) * a.R;
}
template <int G>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
    for (int off = G / 2; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
}
// floor(i / n) for i n below 2^64: a product's upper half, as a division of 64 bits takes as many
// instructions as the rest of a head.
struct HeadPlace {
    int64_t token;
    int head;
};
__device__ __forceinline__ HeadPlace head_place(int64_t base, int local, int n, uint64_t inv) {
    const int64_t t = inv ? (int64_t)__umul64hi((uint64_t)base, inv) : base;
    // `local` after the base-th: below 2^20, so that the quotient is exact.
    local += (int)(base - t * n);
    const int q = (int)(((float)local + 0.5f) * (1.f / (float)n));
    return {t + q, local - q * n};
}

// G lanes a head, NU units a lane.
template <typename T, bool INTER, int E, int G, int NU>
__global__ void __launch_bounds__(256) head_norm_kernel(const HeadArgs a) {
    constexpr int PER = 256 / G;
    const int n = a.t[0].heads + a.t[1].heads, lane = threadIdx.x % G;
    const int64_t base = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * PER;
    const HeadPlace at = head_place(base, threadIdx.x / G, n, a.inv[2]);
    const int64_t token = at.token;
    int head = at.head;
    if (token >= a.tokens) return;  // a whole group
    const bool second = head >= a.t[0].heads;
    const HeadTensor &t = a.t[second];
    if (second) head -= a.t[0].heads;
    const int64_t in = token * t.x_token + head * t.x_head;
    HeadUnit<T, INTER, E> u[NU];
    float x[NU][2][E], cs[NU][2][E], w[NU][2][E];
    float ss = 0.f;
#pragma unroll
    for (int k = 0; k < NU; ++k) {
        u[k].init(a, k * G + lane);
        u[k].load(t.x, in, x[k]);
    }
    if (a.R) {
        const float *row = a.table + head_row(a, head_position(a, token));
#pragma unroll
        for (int k = 0; k < NU; ++k) u[k].angles(row, a.R, cs[k]);
    }
    if (t.w) {
#pragma unroll
        for (int k = 0; k < NU; ++k) u[k].load(t.w, 0, w[k]);
    }
#pragma unroll
    for (int k = 0; k < NU; ++k)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < E; ++e) ss += x[k][i][e] * x[k][i][e];
    const float r = rsqrtf(group_sum<G>(ss) * a.inv_d + a.eps);
#pragma unroll
    for (int k = 0; k < NU; ++k) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < E; ++e) x[k][i][e] *= t.w ? r * w[k][i][e] : r;
        u[k].turn(x[k], cs[k], 1.f);
        u[k].store(t.out, token * t.out_token + head * t.out_head, x[k]);
    }
}

// The gradient.  A block takes heads of q or of k, so that a lane's channels, and with them
// its sums of dw, stay the same; the blocks' sums are added by head_norm_sum_kernel.
template <typename T, bool INTER, int E, int G, int NU>
__global__ void __launch_bounds__(kHeadThreads) head_norm_bwd_kernel(const HeadArgs a) {
    constexpr int PER = kHeadThreads / G, W = kHeadThreads / 64;
    __shared__ float part[W][G * NU * 2 * E];
    const bool second = (int)blockIdx.x >= a.blocks[0];
    const HeadTensor &t = a.t[second];
    const int block = (int)blockIdx.x - (second ? a.blocks[0] : 0);
    const int lane = threadIdx.x % G, group = threadIdx.x / G;
    const int64_t step = (int64_t)a.blocks[second] * PER;
    HeadUnit<T, INTER, E> u[NU];
    float w[NU][2][E], dw[NU][2][E] = {};
#pragma unroll
    for (int k = 0; k < NU; ++k) {
        u[k].init(a, k * G + lane);
        if (t.w) u[k].load(t.w, 0, w[k]);
    }
    HeadPacked<T, E> px[NU][2], pg[NU][2];  // zeros where the lane has no piece
    float pcs[NU][2][E];
    int64_t out = 0;
    // A head's angles lie where its token's position says, which is read a head earlier still.
    auto place = [&](int64_t base) { return head_place(base, group, t.heads, a.inv[second]); };
    int64_t pos = head_position(a, place((int64_t)block * PER).token);
    auto fetch = [&](int64_t base) {  // whether this group has a head there
        const HeadPlace p = place(base);
        if (p.token >= a.tokens) return false;
        const float *row = a.table + head_row(a, pos);
#pragma unroll
        for (int k = 0; k < NU; ++k) {
            u[k].load(t.x, p.token * t.x_token + p.head * t.x_head, px[k]);
            u[k].load(t.dy, p.token * t.dy_token + p.head * t.dy_head, pg[k]);
            if (a.R) u[k].angles(row, a.R, pcs[k]);
        }
        pos = head_position(a, place(base + step).token);
        out = p.token * t.out_token + p.head * t.out_head;
        return true;
    };
    int64_t base = (int64_t)block * PER;
    for (bool has = fetch(base); has;) {  // the same for all of a group's lanes
        float x[NU][2][E], g[NU][2][E], cs[NU][2][E];
#pragma unroll
        for (int k = 0; k < NU; ++k)
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int e = 0; e < E; ++e) cs[k][i][e] = pcs[k][i][e];
#pragma unroll
        for (int k = 0; k < NU; ++k)
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    x[k][i][e] = px[k][i].at(e);
                    g[k][i][e] = pg[k][i].at(e);
                }
        const int64_t to = out;
        base += step;
        has = fetch(base);
        float ss = 0.f, sg = 0.f;
#pragma unroll
        for (int k = 0; k < NU; ++k) {
            u[k].turn(g[k], cs[k], -1.f);
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    ss += x[k][i][e] * x[k][i][e];
                    sg += (t.w ? g[k][i][e] * w[k][i][e] : g[k][i][e]) * x[k][i][e];
                }
        }
        ss = group_sum<G>(ss);
        sg = group_sum<G>(sg);
        const float r = rsqrtf(ss * a.inv_d + a.eps), c = r * r * (sg * a.inv_d);
#pragma unroll
        for (int k = 0; k < NU; ++k) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    dw[k][i][e] += g[k][i][e] * (x[k][i][e] * r);
                    const float gw = t.w ? g[k][i][e] * w[k][i][e] : g[k][i][e];
                    x[k][i][e] = r * (gw - x[k][i][e] * c);
                }
            u[k].store(t.out, to, x[k]);
        }
    }
    if (!t.w) return;
    // The wave's groups, then the waves.
#pragma unroll
    for (int k = 0; k < NU; ++k)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                float v = dw[k][i][e];
#pragma unroll
                for (int off = 32; off >= G; off >>= 1) v += __shfl_xor(v, off, 64);
                if ((threadIdx.x & 63) < G && u[k].has[i])
                    part[threadIdx.x >> 6][u[k].c[i] + e] = v;
            }
    __syncthreads();
    for (int d = threadIdx.x; d < a.D; d += kHeadThreads) {
        float v = part[0][d];
#pragma unroll
        for (int i = 1; i < W; ++i) v += part[i][d];
        a.part[(int64_t)blockIdx.x * a.D + d] = v;
    }
}

// dw: the blocks' sums, in order within each of 32 rows of threads, then the rows' in pairs (one
// after the other they were off by 1.3 times as much).  blockIdx.y: q or k.
template <typename T>
__global__ void __launch_bounds__(1024) head_norm_sum_kernel(const float *part, int n_q, int n_k,
                                                            int D, T *dw_q, T *dw_k) {
    __shared__ float s[32][33];
    const bool second = blockIdx.y != 0;
    T *out = second ? dw_k : dw_q;
    if (!out) return;
    const float *p = part + (second ? (int64_t)n_q * D : 0);
    const int n = second ? n_k : n_q, col = threadIdx.x & 31, row = threadIdx.x >> 5;
    const int d = blockIdx.x * 32 + col;
    float v = 0.f;
    for (int i = row; d < D && i < n; i += 32 * 16) {  // 16 in flight
        float x[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) x[j] = i + 32 * j < n ? p[(int64_t)(i + 32 * j) * D + d] : 0.f;
#pragma unroll
        for (int j = 0; j < 16; ++j) v += x[j];
    }
    s[row][col] = v;
    __syncthreads();
    if (row != 0 || d >= D) return;
    float x[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) x[i] = s[i][col];
#pragma unroll
    for (int n = 16; n > 0; n >>= 1)
#pragma unroll
        for (int i = 0; i < n; ++i) x[i] += x[i + n];
    out[d] = (T)x[0];
}

}  // namespace katsu
