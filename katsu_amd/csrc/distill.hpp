// distill.hpp -- the loss of a row's logits z against a teacher's top logits t_k at ids
// id_k, and its gradient.  Over the entries whose id is one of the V columns:
//
//   p = softmax(t / tau),  P = softmax(z / tau) over all V,
//   loss = tau^2 sum_k p_k (log p_k - log P[id_k])
//        = tau sum_k p_k ((t_k - max t) - (z[id_k] - M) + tau (log L - log T))
//   dz_v = dloss tau (P_v - sum of the p_k with id_k = v)
//
// A row without such an entry, or with none above -inf, has loss and gradient 0, and its
// logits are not read.  M = max z, L = sum exp((z - M)/tau), T the teacher's.  Differences of
// logits are taken first, so that large ones lose nothing, and stay logits: over a tau below 1 the
// type's lowest value would be infinite, and tau^2 is 0 or infinite before tau is.  They are summed
// as fourths, which are as exact: the sum of the whole ones may be infinite where tau times it is not.
//
// An exponential is exp2 of a difference times log2(e)/tau in float32, whose rounding (1.3e-8 of it at
// a tau of 1) grows with the distance: totals are 5.5e-8 too large for normal logits of deviation
// 2.5.  Results below 2^-126 are 0.
//
// The loss in one pass with each thread's running maximum and sum: 4096 x 32000 bfloat16 51-53 us,
// 4.7-4.8 TB/s, where the vector unit is busy 83% of the time as well.  The gradient 1000 x 32001 float32
// 62 us, 4.3 TB/s; both in a pass, 8192 x 32000 bfloat16, 203 us, 5.0 TB/s: HBM (a copy of as much
// reaches 5.1 to 5.3).
#pragma once

#include <type_traits>

#include "lmvec.hpp"

namespace katsu {

struct DistillArgs {
    const void *z, *teacher;
    const int32_t *ids;
    const float *dloss;
    float *stats;       // [2][rows]: M, 1/L (0, 0 without an entry)
    float *loss;
    void *dz;
    int64_t rows, vocab, z_row, dz_row, dloss_step, run;  // run: columns of a block's gradient
    int top, teacher_bf16;
    float tau, scale2;  // scale2: log2(e) / tau
};

constexpr int kDistillTop = 1024, kDistillBits = 1 << 16;

struct DistillIds {
    int id[kDistillTop];
    float p[kDistillTop];
    uint32_t bits[kDistillBits / 32];
};

__device__ __forceinline__ float distill_exp(float x, float by) {  // exp((x)/tau)
    return __builtin_amdgcn_exp2f(x * by);
}

// A block's sum or maximum; each call uses its own slot of `part`.
template <int NT, class F>
__device__ __forceinline__ float block_join(float v, float *part, F f) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v = f(v, __shfl_xor(v, off, 64));
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = part[0];
#pragma unroll
    for (int w = 1; w < NT / 64; ++w) v = f(v, part[w]);
    return v;
}
struct JoinSum {
    __device__ __forceinline__ float operator()(float a, float b) const { return a + b; }
};
struct JoinMax {
    __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
};

// A thread's entries of a row: entry tid + NT i.
template <int NT>
struct DistillRow {
    static constexpr int N = kDistillTop / NT;
    int id[N];        // -1 where there is none
    float t[N], p[N];
    float largest, total;
    bool some;

    __device__ __forceinline__ void load(const DistillArgs &a, int64_t row) {
        float m = -INFINITY;
        bool any = false;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int k = threadIdx.x + NT * i;
            id[i] = -1;
            t[i] = -INFINITY;
            if (k < a.top) {
                const int v = a.ids[row * a.top + k];
                const float x = a.teacher_bf16
                                    ? (float)((const __bf16 *)a.teacher)[row * a.top + k]
                                    : ((const float *)a.teacher)[row * a.top + k];
                if (v >= 0 && v < a.vocab) {
                    id[i] = v;
                    t[i] = x;
                    any |= t[i] != -INFINITY;
                    m = fmaxf(m, t[i]);
                }
            }
        }
        some = __syncthreads_or(any);
        largest = m;
    }
    __device__ __forceinline__ void softmax(const DistillArgs &a, float *part_m, float *part_l) {
        largest = block_join<NT>(largest, part_m, JoinMax());
        float l = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            p[i] = t[i] == -INFINITY ? 0.f : distill_exp(t[i] - largest, a.scale2);
            l += p[i];
        }
        total = block_join<NT>(l, part_l, JoinSum());
#pragma unroll
        for (int i = 0; i < N; ++i) p[i] /= total;
    }
};

// A running maximum and sum.
struct DistillSum {
    float m = -INFINITY, l = 0.f;
    __device__ __forceinline__ static float ref(float m) { return m == -INFINITY ? 0.f : m; }
    template <int N>
    __device__ __forceinline__ void add(const float (&x)[N], float by) {
        float top = x[0];
#pragma unroll
        for (int i = 1; i < N; ++i) top = fmaxf(top, x[i]);
        const float mn = fmaxf(m, top), r = ref(mn);
        l *= distill_exp(m - r, by);
#pragma unroll
        for (int i = 0; i < N; ++i) l += distill_exp(x[i] - r, by);
        m = mn;
    }
    __device__ __forceinline__ void join(float m2, float l2, float by) {
        const float mn = fmaxf(m, m2), r = ref(mn);
        l = l * distill_exp(m - r, by) + l2 * distill_exp(m2 - r, by);
        m = mn;
    }
    __device__ __forceinline__ void wave(float by) {  // of all lanes, in each
#pragma unroll
        for (int off = 32; off > 0; off >>= 1)
            join(__shfl_xor(m, off, 64), __shfl_xor(l, off, 64), by);
    }
};

// How many values a row begins after a 16-byte boundary.  Its pieces begin that much before it, so
// that they lie on such boundaries: accesses of 16 bytes that begin in the middle of 4 take longer
// (2000 rows of 32001 bfloat16: the loss 34 us so, 30 with the shift, the gradient 67 and 62).
template <typename T>
__device__ __forceinline__ int row_shift(const T *p) {
    return (int)((uintptr_t)p / sizeof(T) % Piece<T>::E);
}

// M and L of a thread's pieces of a row, U of them in flight.
template <typename T, int NT, int U>
__device__ __forceinline__ DistillSum distill_pieces(const T *z, int64_t n, float by) {
    constexpr int E = Piece<T>::E;
    DistillSum s;
    for (int64_t i = (int)threadIdx.x * E - row_shift(z); i < n; i += U * NT * E) {
        RawPiece<T> r[U];
        float x[U * E];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (u == 0 || i + u * NT * E < n)
                r[u].load(z, i + u * NT * E, n, -INFINITY, 0);
            else
                r[u].fill(-INFINITY);
#pragma unroll
        for (int e = 0; e < U * E; ++e) x[e] = r[e / E].at(e % E);
        s.add(x, by);
    }
    return s;
}
// M and L of a row, the same in every thread.
template <typename T, int NT, int U>
__device__ __forceinline__ DistillSum distill_row(const T *z, int64_t n, float by, float *part) {
    DistillSum s = distill_pieces<T, NT, U>(z, n, by);
    s.wave(by);
    if ((threadIdx.x & 63) == 0) {
        part[2 * (threadIdx.x >> 6)] = s.m;
        part[2 * (threadIdx.x >> 6) + 1] = s.l;
    }
    __syncthreads();
    DistillSum all;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) all.join(part[2 * w], part[2 * w + 1], by);
    return all;
}

template <typename T, int NT>
__device__ __forceinline__ void distill_loss(const DistillArgs &a, int64_t row,
                                             const DistillRow<NT> &d, const DistillSum &s,
                                             float *part) {
    const T *z = (const T *)a.z + row * a.z_row;
    const float rest = 0.25f * (a.tau * (logf(s.l) - logf(d.total)));
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < DistillRow<NT>::N; ++i)
        if (d.id[i] >= 0 && d.p[i] != 0.f)
            v += d.p[i] * ((0.25f * d.t[i] - 0.25f * d.largest) -
                           (0.25f * (float)z[d.id[i]] - 0.25f * s.m) + rest);
    v = block_join<NT>(v, part, JoinSum());
    if (threadIdx.x == 0) a.loss[row] = 4.f * (a.tau * v);
}

// The teacher's columns among [c0, c1): an entry's value, of which the first of equal ids takes the
// sum, and whether the thread writes it.  A set of bits tells whether any id occurs twice (ids that
// share the last 16 bits count as well): only then they are compared with each other.
template <int NT>
struct DistillFix {
    static constexpr int N = DistillRow<NT>::N;
    float v[N];
    bool own[N];

    template <typename T>
    __device__ __forceinline__ void find(const DistillArgs &a, const T *z, int64_t c0, int64_t c1,
                                         const DistillRow<NT> &d, float m, float inv, float g,
                                         DistillIds &s) {
        for (int i = threadIdx.x; i < kDistillBits / 32; i += NT) s.bits[i] = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            s.id[threadIdx.x + NT * i] = d.id[i];
            s.p[threadIdx.x + NT * i] = d.p[i];
        }
        __syncthreads();
        bool twice = false;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            own[i] = d.id[i] >= c0 && d.id[i] < c1;
            if (!own[i]) continue;
            const uint32_t bit = 1u << (d.id[i] & 31);
            twice |= atomicOr(s.bits + (d.id[i] % kDistillBits >> 5), bit) & bit;
        }
        twice = __syncthreads_or(twice);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (!own[i]) continue;
            const int k = threadIdx.x + NT * i;
            float p = d.p[i];
            if (twice) {
                p = 0.f;
                for (int j = 0; j < a.top; ++j) {
                    if (s.id[j] != d.id[i]) continue;
                    p += s.p[j];
                    if (j < k) own[i] = false;
                }
            }
            if (own[i]) v[i] = (distill_exp((float)z[d.id[i]] - m, a.scale2) * inv - p) * g;
        }
    }
    template <typename T>
    __device__ __forceinline__ void write(const DistillRow<NT> &d, T *dz) const {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (own[i]) dz[d.id[i]] = (T)v[i];
    }
};

// A thread's pieces of columns [c0, c1) as if there were no teacher, U of them in flight.
template <typename T, int NT, int U>
__device__ __forceinline__ void grad_pieces(const T *z, T *dz, int64_t c0, int64_t c1, float m,
                                            float scale2, float by) {
    constexpr int E = Piece<T>::E;
    for (int64_t i = c0 + (int)threadIdx.x * E - (c0 == 0 ? row_shift(z) : 0); i < c1;
         i += U * NT * E) {
        RawPiece<T> r[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (u == 0 || i + u * NT * E < c1) r[u].load(z, i + u * NT * E, c1, 0.f, 0);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (u > 0 && i + u * NT * E >= c1) break;
            float x[E];
#pragma unroll
            for (int e = 0; e < E; ++e) x[e] = distill_exp(r[u].at(e) - m, scale2) * by;
            r[u].set(x);
            r[u].store(dz, i + u * NT * E, c1, 0);
        }
    }
}

// The gradient of columns [c0, c1): all of them as if there were no teacher, then the
// teacher's.
template <typename T, int NT, int U>
__device__ __forceinline__ void distill_grad(const DistillArgs &a, int64_t row, int64_t c0,
                                             int64_t c1, const DistillRow<NT> &d, float m,
                                             float inv, DistillIds &s) {
    const T *z = (const T *)a.z + row * a.z_row;
    T *dz = (T *)a.dz + row * a.dz_row;
    const float g = a.dloss[row * a.dloss_step] * a.tau, by = inv * g;
    DistillFix<NT> fix;
    fix.find(a, z, c0, c1, d, m, inv, g, s);
    __syncthreads();  // dz may be z: all of the teacher's logits are read
    grad_pieces<T, NT, U>(z, dz, c0, c1, m, a.scale2, by);
    __syncthreads();  // and all others written
    fix.write(d, dz);
}

template <typename T, int NT>
__device__ __forceinline__ void distill_zero(const DistillArgs &a, int64_t row, int64_t c0,
                                             int64_t c1) {
    constexpr int E = Piece<T>::E;
    T *dz = (T *)a.dz + row * a.dz_row;
    const RawPiece<T> zero = {};
    for (int64_t i = c0 + (int)threadIdx.x * E - (c0 == 0 ? row_shift(dz) : 0); i < c1;
         i += NT * E)
        zero.store(dz, i, c1, 0);
}

// Loss, gradient or both of whole rows: a block a row, U of a thread's pieces in flight.
template <typename T, int NT, bool LOSS, bool GRAD, int U>
__global__ void __launch_bounds__(NT) distill_kernel(const DistillArgs a) {
    __shared__ float part[5][2 * NT / 64];
    __shared__ std::conditional_t<GRAD, DistillIds, int> ids;
    const int64_t row = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
    if (row >= a.rows) return;
    int64_t c0 = 0, c1 = a.vocab;
    if (!LOSS) {  // runs of pieces
        const int shift = row_shift((const T *)a.z + row * a.z_row);
        if (blockIdx.z > 0) c0 = blockIdx.z * a.run - shift;
        if (blockIdx.z + 1 < gridDim.z) c1 = (blockIdx.z + 1) * a.run - shift;
    }
    DistillRow<NT> d;
    d.load(a, row);
    if (!d.some) {
        if (LOSS && threadIdx.x == 0) {
            a.loss[row] = 0.f;
            if (a.stats) a.stats[row] = a.stats[a.rows + row] = 0.f;
        }
        if (GRAD) distill_zero<T, NT>(a, row, c0, c1);
        return;
    }
    d.softmax(a, part[0], part[1]);
    float m, inv;
    if constexpr (LOSS) {
        const DistillSum s =
            distill_row<T, NT, U>((const T *)a.z + row * a.z_row, a.vocab, a.scale2, part[2]);
        distill_loss<T, NT>(a, row, d, s, part[3]);
        m = s.m;
        inv = 1.f / s.l;
        if (a.stats && threadIdx.x == 0) {
            a.stats[row] = m;
            a.stats[a.rows + row] = inv;
        }
    } else {
        m = a.stats[row];
        inv = a.stats[a.rows + row];
    }
    if constexpr (GRAD) distill_grad<T, NT, U>(a, row, c0, c1, d, m, inv, ids);
}

// Loss and gradient of rows of up to NT * NP pieces, which stay in the block's registers between
// the two: the logits are read once.
template <typename T, int NT, int NP>
__global__ void __launch_bounds__(NT) distill_step_kernel(const DistillArgs a) {
    constexpr int E = Piece<T>::E;
    __shared__ float part[5][NT / 64];
    __shared__ DistillIds ids;
    const int64_t row = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
    if (row >= a.rows) return;
    const T *z = (const T *)a.z + row * a.z_row;
    T *dz = (T *)a.dz + row * a.dz_row;
    const int V = (int)a.vocab;
    DistillRow<NT> d;
    d.load(a, row);
    if (!d.some) {
        if (threadIdx.x == 0) a.loss[row] = 0.f;
        distill_zero<T, NT>(a, row, 0, V);
        return;
    }
    const int shift = V + E <= NT * NP * E ? row_shift(z) : 0;
    RawPiece<T> x[NP];
#pragma unroll
    for (int k = 0; k < NP; ++k) {
        const int first = k * NT * E - shift;  // of the block's pieces
        const T *at = z + first;
        if (first >= 0 && first + NT * E <= V)
            __builtin_memcpy(&x[k].v, at + threadIdx.x * E, 16);
        else
            x[k].load(at, threadIdx.x * E, V - first, -INFINITY, -first);
    }
    d.softmax(a, part[0], part[1]);
    float m = -INFINITY;
#pragma unroll
    for (int k = 0; k < NP; ++k)
#pragma unroll
        for (int e = 0; e < E; ++e) m = fmaxf(m, x[k].at(e));
    m = block_join<NT>(m, part[2], JoinMax());
    float l = 0.f;
#pragma unroll
    for (int k = 0; k < NP; ++k) x[k].packed();
#pragma unroll
    for (int k = 0; k < NP; ++k)
#pragma unroll
        for (int e = 0; e < E; ++e) l += distill_exp(x[k].at(e) - m, a.scale2);
    DistillSum s;
    s.m = m;
    s.l = block_join<NT>(l, part[3], JoinSum());
    distill_loss<T, NT>(a, row, d, s, part[4]);
    const float inv = 1.f / s.l, g = a.dloss[row * a.dloss_step] * a.tau, by = inv * g;
    DistillFix<NT> fix;
    fix.find(a, z, 0, V, d, m, inv, g, ids);
#pragma unroll
    for (int k = 0; k < NP; ++k) x[k].packed();
    __syncthreads();  // dz may be z: all of the teacher's logits are read
#pragma unroll
    for (int k = 0; k < NP; ++k) {
        const int i = (k * NT + (int)threadIdx.x) * E - shift;
        if (i >= V) break;
        float y[E];
#pragma unroll
        for (int e = 0; e < E; ++e) y[e] = distill_exp(x[k].at(e) - m, a.scale2) * by;
        x[k].set(y);
        x[k].store(dz, i, V, 0);
    }
    __syncthreads();  // and all others written
    fix.write(d, dz);
}

}  // namespace katsu
