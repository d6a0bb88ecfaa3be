// rotary.hpp -- rotary positions: each pair (a, b) of a head's first R channels turns by
// its position's angle, (a cos - b sin, a sin + b cos); the rest of the head stays.
//
// The angles' cosines and sines are a table [length][R], cosines first, in float32,
// computed in float64 once (an angle of 32768 radians has an error of 0.002 in float32).
// HBM-bound: q and k are read and written once, in one launch (16384 tokens, 16 + 4 heads of
// 128, half of each turning, float32: 66 us, 5.1 TB/s; a copy reaches 4.7).
#pragma once

#include "lmvec.hpp"

namespace katsu {

struct RotaryTensor {
    const void *in;
    void *out;
    int64_t in_token, in_head, out_token, out_head;
    int heads;
};
struct RotaryArgs {
    RotaryTensor t[2];  // q and k
    const float *table;
    const int32_t *positions;  // NULL: 0, 1, ..
    int64_t tokens, length;
    int D, R, items, per_head;  // items of a token, of a head
    float inv_per_head, sign;
};

// One block a token (grid-stride), a thread an item: E pairs in the half layout (two
// pieces R/2 apart), E/2 pairs in the interleaved one, or a piece of the rest.  VEC: all
// these are whole pieces; else an item is one pair or one channel.
template <typename T, bool INTER, bool VEC>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryArgs a) {
    constexpr int E = VEC ? Piece<T>::E : 1;
    const int half = a.R / 2;
    const int turning = INTER ? (VEC ? a.R / E : half) : half / E;  // items that turn
    for (int64_t token = blockIdx.x; token < a.tokens; token += gridDim.x) {
        int64_t pos = a.positions ? a.positions[token] : token;
        pos = pos < 0 ? 0 : pos < a.length ? pos : a.length - 1;  // stays inside the table
        const float *cs = a.table + pos * a.R;
        for (int it = threadIdx.x; it < a.items; it += 256) {
            // Exact for items below 2^20: the quotient is at least half an item off a step.
            int head = (int)(((float)it + 0.5f) * a.inv_per_head);
            const int j = it - head * a.per_head;
            const bool second = head >= a.t[0].heads;
            const RotaryTensor &t = a.t[second];
            if (second) head -= a.t[0].heads;
            const T *in = (const T *)t.in + token * t.in_token + head * t.in_head;
            T *out = (T *)t.out + token * t.out_token + head * t.out_head;
            if (j >= turning) {
                const int d = a.R + (j - turning) * E;
                if constexpr (VEC) {
                    lm_u4 u;
                    __builtin_memcpy(&u, in + d, 16);
                    __builtin_memcpy(out + d, &u, 16);
                } else {
                    out[d] = in[d];
                }
                continue;
            }
            if constexpr (INTER) {
                constexpr int P = VEC ? E / 2 : 1;  // pairs
                const int i = j * P;
                float c[P], s[P], x[2 * P];
                if constexpr (VEC) {
                    __builtin_memcpy(c, cs + i, sizeof c);
                    __builtin_memcpy(s, cs + half + i, sizeof s);
                    load_piece(in, 2 * i, a.D, x);
                } else {
                    c[0] = cs[i];
                    s[0] = cs[half + i];
                    x[0] = (float)in[2 * i];
                    x[1] = (float)in[2 * i + 1];
                }
#pragma unroll
                for (int p = 0; p < P; ++p) {
                    const float u = x[2 * p], v = x[2 * p + 1], w = a.sign * s[p];
                    x[2 * p] = u * c[p] - v * w;
                    x[2 * p + 1] = u * w + v * c[p];
                }
                if constexpr (VEC) {
                    store_piece(out, 2 * i, a.D, x);
                } else {
                    out[2 * i] = (T)x[0];
                    out[2 * i + 1] = (T)x[1];
                }
            } else {
                const int i = j * E;
                float c[E], s[E], u[E], v[E];
                if constexpr (VEC) {
                    __builtin_memcpy(c, cs + i, sizeof c);
                    __builtin_memcpy(s, cs + half + i, sizeof s);
                    load_piece(in, i, a.D, u);
                    load_piece(in, half + i, a.D, v);
                } else {
                    c[0] = cs[i];
                    s[0] = cs[half + i];
                    u[0] = (float)in[i];
                    v[0] = (float)in[half + i];
                }
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float x = u[e], y = v[e], w = a.sign * s[e];
                    u[e] = x * c[e] - y * w;
                    v[e] = x * w + y * c[e];
                }
                if constexpr (VEC) {
                    store_piece(out, i, a.D, u);
                    store_piece(out, half + i, a.D, v);
                } else {
                    out[i] = (T)u[0];
                    out[half + i] = (T)v[0];
                }
            }
        }
    }
}

// table[p][i] = amp cos(p f_i), table[p][R/2 + i] = amp sin(p f_i), f_i the frequency
// base^(-2i/R) scaled (katsu_hip.h): linear, f / factor; by wavelength, between f / factor
// and f by how often it turns within the original length.
__global__ void __launch_bounds__(256) rotary_table_kernel(float *table, int64_t length, int R,
                                                           double base, double factor,
                                                           int by_wavelength) {
    const int half = R / 2;
    const int64_t n = length * half, step = (int64_t)gridDim.x * 256;
    for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < n; t += step) {
        const int64_t p = t / half;
        const int i = (int)(t % half);
        double f = pow(base, -2.0 * i / R), amp = 1.0;
        if (by_wavelength) {
            const double turns = (double)length / factor * f / 6.283185307179586;
            const double keep = fmin(fmax((turns - 1.0) / 31.0, 0.0), 1.0);
            f = f * (keep + (1.0 - keep) / factor);
            amp = 0.1 * log(factor) + 1.0;
        } else {
            f = f / factor;
        }
        double s, c;
        sincos((double)p * f, &s, &c);
        table[p * R + i] = (float)(amp * c);
        table[p * R + half + i] = (float)(amp * s);
    }
}

}  // namespace katsu
