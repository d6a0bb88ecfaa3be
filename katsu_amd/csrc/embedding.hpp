// embedding.hpp -- rows of a table by token, times a scale, and the table's gradient.
//
//   out[t] = scale table[ids[t]]                       (zeros where ids[t] is no row)
//   dtable[v] = (dtable[v] +) scale sum over t with ids[t] = v of dout[t], t rising
//
// HBM-bound: each row is read and written once.
#pragma once

#include "lmvec.hpp"

namespace katsu {

struct EmbedArgs {
    const int32_t *ids;
    const void *in;   // table or dout
    void *out;        // out or dtable
    int64_t tokens, vocab, cols, in_row, out_row;
    float scale;
    int chunks, add;  // pieces of a row, 64 * kEmbedPieces of 16 bytes; whether dtable is added to
};

constexpr int kEmbedPieces = 4;

// A wave a row's chunk: 4 KB in flight.
template <typename T>
__global__ void __launch_bounds__(256) embed_kernel(const EmbedArgs a) {
    constexpr int E = Piece<T>::E, N = kEmbedPieces;
    const int lane = threadIdx.x & 63;
    const int64_t step = (int64_t)gridDim.x * 4, items = a.tokens * a.chunks;
    for (int64_t it = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); it < items; it += step) {
        const int64_t t = it / a.chunks, c0 = (it - t * a.chunks) * (64 * N * E);
        const int64_t id = a.ids[t];
        const T *in = (const T *)a.in + id * a.in_row;
        T *out = (T *)a.out + t * a.out_row;
        const bool has = id >= 0 && id < a.vocab;
        float x[N][E];
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int64_t i = c0 + (k * 64 + lane) * E;
            if (has && i < a.cols) load_piece(in, i, a.cols, x[k]);
        }
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int64_t i = c0 + (k * 64 + lane) * E;
#pragma unroll
            for (int e = 0; e < E; ++e) x[k][e] = has ? x[k][e] * a.scale : 0.f;
            if (i < a.cols) store_piece(out, i, a.cols, x[k]);
        }
    }
}

// The gradient of few tokens: a wave a row of the table, which looks through all ids.
template <typename T>
__global__ void __launch_bounds__(256) embed_grad_few_kernel(const EmbedArgs a) {
    constexpr int E = Piece<T>::E;
    const int lane = threadIdx.x & 63;
    const int64_t step = (int64_t)gridDim.x * 4;
    for (int64_t v = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); v < a.vocab; v += step) {
        T *out = (T *)a.out + v * a.out_row;
        for (int64_t c = 0; c < a.cols; c += 64 * E) {
            const int64_t i = c + lane * E;
            float x[E] = {};
            bool some = false;
            for (int64_t t0 = 0; t0 < a.tokens; t0 += 64) {
                const int64_t t = t0 + lane;
                uint64_t m = __ballot(t < a.tokens && a.ids[t] == v);
                some |= m != 0;
                for (; m; m &= m - 1) {
                    const T *in = (const T *)a.in + (t0 + __builtin_ctzll(m)) * a.in_row;
                    float y[E];
                    if (i < a.cols) {
                        load_piece(in, i, a.cols, y);
#pragma unroll
                        for (int e = 0; e < E; ++e) x[e] += y[e];
                    }
                }
            }
            if (i >= a.cols || (a.add && !some)) continue;
            float old[E] = {};
            if (a.add) load_piece(out, i, a.cols, old);
#pragma unroll
            for (int e = 0; e < E; ++e) x[e] = x[e] * a.scale + old[e];
            store_piece(out, i, a.cols, x);
        }
    }
}

}  // namespace katsu
