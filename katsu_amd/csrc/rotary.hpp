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

// One block a token (grid-stride), a thread an item: E pairs in the half layout (two pieces
// of E channels R/2 apart), E/2 pairs (one at least) in the interleaved one, or E channels
// of the rest.
template <typename T, bool INTER, int E>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryArgs a) {
    constexpr int P = !INTER ? E : E > 1 ? E / 2 : 1;  // pairs
    const int half = a.R / 2, turning = half / P;      // items that turn
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
                T e[E];
                __builtin_memcpy(e, in + d, sizeof e);
                __builtin_memcpy(out + d, e, sizeof e);
                continue;
            }
            const int i = j * P;
            float c[P], s[P], u[P], v[P];
            rotary_load<float, P>(cs + i, c);
            rotary_load<float, P>(cs + half + i, s);
            if constexpr (INTER) {
                float x[2 * P];
                rotary_load<T, 2 * P>(in + 2 * i, x);
#pragma unroll
                for (int e = 0; e < P; ++e) {
                    u[e] = x[2 * e];
                    v[e] = x[2 * e + 1];
                }
            } else {
                rotary_load<T, P>(in + i, u);
                rotary_load<T, P>(in + half + i, v);
            }
#pragma unroll
            for (int e = 0; e < P; ++e) {
                const float x = u[e], y = v[e], w = a.sign * s[e];
                u[e] = x * c[e] - y * w;
                v[e] = x * w + y * c[e];
            }
            if constexpr (INTER) {
                float x[2 * P];
#pragma unroll
                for (int e = 0; e < P; ++e) {
                    x[2 * e] = u[e];
                    x[2 * e + 1] = v[e];
                }
                rotary_store<T, 2 * P>(out + 2 * i, x);
            } else {
                rotary_store<T, P>(out + i, u);
                rotary_store<T, P>(out + half + i, v);
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
