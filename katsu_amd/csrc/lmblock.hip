// lmblock.hip -- launches of the HBM-bound language-model kernels: rotary positions,
// the norms around a block, gradient clipping.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "blocknorm.hpp"
#include "gradclip.hpp"
#include "lm.hpp"
#include "rotary.hpp"

namespace katsu {
namespace {

constexpr int64_t kI32Max = 0x7fffffff;

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

int status_of(hipError_t e) {
    if (e == hipSuccess) return KATSU_OK;
    return e == hipErrorNoDevice || e == hipErrorInvalidDevice ? KATSU_E_NODEVICE : KATSU_E_LAUNCH;
}

bool dtype_ok(int t) { return t == KATSU_F32 || t == KATSU_BF16; }

template <typename T, bool INTER, int E>
int launch_rotary(RotaryArgs a, hipStream_t st) {
    constexpr int P = !INTER ? E : E > 1 ? E / 2 : 1;
    a.per_head = a.R / 2 / P;
    const bool in_place = a.t[0].in == a.t[0].out && (!a.t[1].heads || a.t[1].in == a.t[1].out);
    if (!in_place) a.per_head += (a.D - a.R) / E;  // else the rest of each head is in its place
    a.items = a.per_head * (a.t[0].heads + a.t[1].heads);
    a.inv_per_head = 1.f / (float)a.per_head;
    rotary_kernel<T, INTER, E>
        <<<dim3((unsigned)std::min<int64_t>(a.tokens, 1 << 20)), 256, 0, st>>>(a);
    return status_of(hipGetLastError());
}
// The widest accesses that the turning part, its halves and the rest are multiples of.
template <typename T, bool INTER>
int launch_rotary(const RotaryArgs &a, hipStream_t st) {
    auto fits = [&](int e) { return (INTER ? a.R : a.R / 2) % e == 0 && (a.D - a.R) % e == 0; };
    if constexpr (sizeof(T) == 2)
        if (fits(8)) return launch_rotary<T, INTER, 8>(a, st);
    if (fits(4)) return launch_rotary<T, INTER, 4>(a, st);
    if (fits(2)) return launch_rotary<T, INTER, 2>(a, st);
    return launch_rotary<T, INTER, 1>(a, st);
}

// Threads a row and 16-byte pieces a thread: a wave for rows of up to 128 pieces, so that
// its sums need no barrier, else a block.
template <typename T, class F>
int by_row_size(int64_t cols, F f) {
    const int64_t pieces = cdiv(cols, Piece<T>::E);
    if (pieces <= 64) return f(std::integral_constant<int, 64>(), std::integral_constant<int, 1>());
    if (pieces <= 128) return f(std::integral_constant<int, 64>(), std::integral_constant<int, 2>());
    if (pieces <= 256)
        return f(std::integral_constant<int, 256>(), std::integral_constant<int, 1>());
    if (pieces <= 512)
        return f(std::integral_constant<int, 256>(), std::integral_constant<int, 2>());
    if (pieces <= 1024)
        return f(std::integral_constant<int, 1024>(), std::integral_constant<int, 1>());
    if (pieces <= 2048)
        return f(std::integral_constant<int, 1024>(), std::integral_constant<int, 2>());
    if constexpr (sizeof(T) == 4)  // 16384 columns are 2048 pieces of bfloat16
        return f(std::integral_constant<int, 1024>(), std::integral_constant<int, 4>());
    return KATSU_E_INVALID;
}

// A launch has fewer than 2^32 threads along x: rows beyond that go along y.
dim3 grid_of(int64_t blocks) {
    const int64_t x = std::min<int64_t>(blocks, 1 << 20);
    return dim3((unsigned)x, (unsigned)cdiv(blocks, x));
}

template <typename T>
int launch_norm(const NormArgs &a, hipStream_t st) {
    return by_row_size<T>(a.cols, [&](auto tpr, auto nv) {
        constexpr int TPR = decltype(tpr)::value, NV = decltype(nv)::value;
        constexpr int RPB = TPR < 256 ? 256 / TPR : 1;
        block_norm_kernel<T, TPR, NV>
            <<<grid_of(cdiv(a.rows, RPB)), dim3(TPR < 256 ? 256 : TPR), 0, st>>>(a);
        return status_of(hipGetLastError());
    });
}

// The gradient holds five values and three sums of each of a thread's elements: one piece a
// thread while a block can have that many.
int bwd_threads(int64_t pieces) {
    return pieces <= 64 ? 64 : pieces <= 128 ? 128 : pieces <= 256 ? 256 : pieces <= 512 ? 512 : 1024;
}
template <typename T, class F>
int by_row_size_bwd(int64_t cols, F f) {
    const int64_t pieces = cdiv(cols, Piece<T>::E);
    std::integral_constant<int, 1> one;
    switch (bwd_threads(pieces)) {
        case 64: return f(std::integral_constant<int, 64>(), one);
        case 128: return f(std::integral_constant<int, 128>(), one);
        case 256: return f(std::integral_constant<int, 256>(), one);
        case 512: return f(std::integral_constant<int, 512>(), one);
        default: break;
    }
    if (pieces <= 1024) return f(std::integral_constant<int, 1024>(), one);
    if (pieces <= 2048)
        return f(std::integral_constant<int, 1024>(), std::integral_constant<int, 2>());
    if constexpr (sizeof(T) == 4)
        return f(std::integral_constant<int, 1024>(), std::integral_constant<int, 4>());
    return KATSU_E_INVALID;
}

// Sets of rows, each one part of the column sums: 16 waves a CU, but no more parts than an
// eighth of the rows, whose bytes they then stay well below.
int norm_sets(int dtype, int64_t rows, int64_t cols) {
    const int threads = bwd_threads(cdiv(cols, dtype == KATSU_F32 ? 4 : 8));
    const int64_t most = std::min<int64_t>(2048, 256 * 1024 / threads);
    return (int)std::min(rows, std::min(most, std::max<int64_t>(256, rows / 8)));
}

template <typename T>
int launch_norm_bwd(const NormBwdArgs &a, void *dw_pre, void *dw_post, void *dgate,
                    hipStream_t st) {
    const int rc = a.sets == 0 ? KATSU_OK : by_row_size_bwd<T>(a.cols, [&](auto tpr, auto nv) {
        constexpr int TPR = decltype(tpr)::value, NV = decltype(nv)::value;
        constexpr int RPB = TPR == 64 ? 4 : 1;
        block_norm_bwd_kernel<T, TPR, NV>
            <<<dim3((unsigned)cdiv(a.sets, RPB)), dim3(RPB * TPR), 0, st>>>(a);
        return status_of(hipGetLastError());
    });
    if (rc != KATSU_OK || a.sums == 0) return rc;
    block_norm_sum_kernel<T><<<dim3((unsigned)cdiv(a.cols, 64), a.sums), 1024, 0, st>>>(
        a.part, a.sets, a.cols, a.sums, a.w_pre ? (T *)dw_pre : nullptr,
        a.w_post ? (T *)dw_post : nullptr, (T *)dgate);
    return status_of(hipGetLastError());
}

}  // namespace

// An output's places are its own, and if it is its input it is so value by value: a thread
// may write before another has read.
bool rotary_out_ok(const int64_t (&in)[2], const int64_t (&out)[2], bool same, uint64_t tokens,
                   uint64_t heads, uint64_t dim) {
    const uint64_t n[2] = {tokens, heads};
    for (int i = 0; i < 2; ++i) {
        if (in[i] < 0 || out[i] < 0) return false;
        if (n[i] > 1 && (out[i] < (int64_t)dim || (same && in[i] != out[i]))) return false;
    }
    if (tokens < 2 || heads < 2) return true;
    // One of the two within a step of the other, as almost always;
    const int inner = out[0] < out[1] ? 0 : 1;
    const int64_t step = out[1 - inner];
    if ((__int128)(n[inner] - 1) * out[inner] + (int64_t)dim <= step) return true;
    // else no number of heads' steps may come closer than `dim` to one of tokens' steps.
    for (uint64_t j = 1; j < heads; ++j) {
        const __int128 at = (__int128)j * out[1];
        const __int128 i = at / out[0], left = at - i * out[0];
        if (i < (__int128)tokens && left < (__int128)dim) return false;
        if (i + 1 < (__int128)tokens && out[0] - left < (__int128)dim) return false;
    }
    return true;
}

bool rotary_ok(const katsu_rotary &d) {
    if (!dtype_ok(d.dtype) || d.heads > 65535 || d.k_heads > 65535) return false;
    if (d.head_dim == 0 || d.head_dim > 65536 || d.rotary_dim == 0 || d.rotary_dim % 2 != 0 ||
        d.rotary_dim > d.head_dim)
        return false;
    // Items of a token are counted exactly in float32.
    if ((d.heads + d.k_heads) * d.head_dim >= 1 << 20) return false;
    return d.tokens <= (uint64_t)kI32Max && d.length > 0 && d.length <= (uint64_t)kI32Max;
}

int rotary(const katsu_rotary &d, const void *q, const void *k, const float *table,
           const int32_t *positions, void *q_out, void *k_out, hipStream_t st) {
    if (d.heads && !rotary_out_ok(d.q_stride, d.q_out_stride, q == q_out, d.tokens, d.heads,
                                  d.head_dim))
        return KATSU_E_INVALID;
    if (d.k_heads && !rotary_out_ok(d.k_stride, d.k_out_stride, k == k_out, d.tokens, d.k_heads,
                                    d.head_dim))
        return KATSU_E_INVALID;
    RotaryArgs a{};
    a.t[0] = {q, q_out, d.q_stride[0], d.q_stride[1], d.q_out_stride[0], d.q_out_stride[1],
              (int)d.heads};
    a.t[1] = {k, k_out, d.k_stride[0], d.k_stride[1], d.k_out_stride[0], d.k_out_stride[1],
              (int)d.k_heads};
    a.table = table;
    a.positions = positions;
    a.tokens = (int64_t)d.tokens;
    a.length = (int64_t)d.length;
    a.D = (int)d.head_dim;
    a.R = (int)d.rotary_dim;
    a.sign = d.inverse ? -1.f : 1.f;
    if (d.interleaved)
        return d.dtype == KATSU_F32 ? launch_rotary<float, true>(a, st)
                                    : launch_rotary<__bf16, true>(a, st);
    return d.dtype == KATSU_F32 ? launch_rotary<float, false>(a, st)
                                : launch_rotary<__bf16, false>(a, st);
}

int rotary_table(float *table, int64_t length, int dim, double base, double factor,
                 int by_wavelength, hipStream_t st) {
    const int64_t blocks = std::min<int64_t>(cdiv(length * (dim / 2), 256), 4096);
    rotary_table_kernel<<<dim3((unsigned)blocks), 256, 0, st>>>(table, length, dim, base, factor,
                                                                by_wavelength);
    return status_of(hipGetLastError());
}

bool block_norm_ok(const katsu_block_norm &d) {
    return dtype_ok(d.dtype) && d.gate_rows >= 0 && d.gate_rows <= 2 && d.rows <= (uint64_t)kI32Max && d.cols > 0 &&
           d.cols <= 16384 && std::isfinite(d.alpha) && d.eps >= 0.f && std::isfinite(d.eps);
}

int block_norm(const katsu_block_norm &d, const void *x, const void *o, const void *gate,
               const void *w_post, const void *w_pre, void *y, void *h, float *stats,
               hipStream_t st) {
    NormArgs a{};
    a.x = x;
    a.o = o;
    a.gate = d.gate_rows ? gate : nullptr;
    a.w_post = w_post;
    a.w_pre = w_pre;
    a.y = y;
    a.h = h;
    a.stats = stats;
    a.rows = (int64_t)d.rows;
    a.cols = (int64_t)d.cols;
    a.gate_row = d.gate_rows == KATSU_GATE_ELEMENT ? a.cols : 0;
    a.alpha = d.alpha;
    a.eps = d.eps;
    a.inv_cols = 1.f / (float)d.cols;
    return d.dtype == KATSU_F32 ? launch_norm<float>(a, st) : launch_norm<__bf16>(a, st);
}

size_t block_norm_bwd_bytes(const katsu_block_norm &d) {
    return (size_t)norm_sets(d.dtype, (int64_t)d.rows, (int64_t)d.cols) * 3 * d.cols *
           sizeof(float);
}

int block_norm_bwd(const katsu_block_norm &d, const void *dy, const void *dh, const void *y,
                   const void *o, const float *stats, const void *gate, const void *w_post,
                   const void *w_pre, void *dx, void *d_o, void *dgate, void *dw_post,
                   void *dw_pre, void *ws, hipStream_t st) {
    NormBwdArgs a{};
    a.dy = dy;
    a.dh = dh;
    a.y = y;
    a.o = o;
    a.gate = d.gate_rows ? gate : nullptr;
    a.w_post = w_post;
    a.w_pre = w_pre;
    a.stats = stats;
    a.dx = dx;
    a.d_o = d_o;
    a.dgate = dgate;
    a.part = (float *)ws;
    a.rows = (int64_t)d.rows;
    a.cols = (int64_t)d.cols;
    a.gate_row = d.gate_rows == KATSU_GATE_ELEMENT ? a.cols : 0;
    a.sets = norm_sets(d.dtype, a.rows, a.cols);
    a.at_post = w_pre ? 1 : 0;
    a.at_gate = a.at_post + (w_post ? 1 : 0);
    a.sums = a.at_gate + (d.gate_rows == KATSU_GATE_CHANNEL ? 1 : 0);
    a.alpha = d.alpha;
    a.inv_cols = 1.f / (float)d.cols;
    return d.dtype == KATSU_F32 ? launch_norm_bwd<float>(a, dw_pre, dw_post, dgate, st)
                                : launch_norm_bwd<__bf16>(a, dw_pre, dw_post, dgate, st);
}

size_t clip_bytes(size_t n) {
    return (n + kClipTensors - 1) / kClipTensors * kClipBlocks * sizeof(double);
}

int clip_grad_norm(const int32_t *dtypes, const void *const *in, void *const *out,
                   const size_t *counts, size_t n, float max_norm, float *norm, void *ws,
                   hipStream_t st) {
    // Both launches of a table have the same blocks; all tables' parts follow each other.
    auto table = [&](size_t at, ClipTable &t) {
        t.n = 0;
        t.first[0] = 0;
        for (; at < n && t.n < kClipTensors; ++at) {
            if (counts[at] == 0) continue;
            t.in[t.n] = in[at];
            t.out[t.n] = out[at];
            t.count[t.n] = (int64_t)counts[at];
            t.half[t.n] = dtypes[at] == KATSU_BF16;
            t.first[t.n + 1] = t.first[t.n] + (uint32_t)cdiv((int64_t)counts[at], kClipChunk);
            ++t.n;
        }
        return at;
    };
    ClipTable t;
    double *parts = (double *)ws;
    int nparts = 0;
    for (size_t at = 0; at < n;) {
        at = table(at, t);
        if (t.n == 0) continue;
        const int blocks = (int)std::min<uint32_t>(t.first[t.n], kClipBlocks);
        clip_squares_kernel<<<blocks, 256, 0, st>>>(t, parts + nparts);
        nparts += blocks;
    }
    for (size_t at = 0, first = 1; at < n || first; first = 0) {
        at = table(at, t);
        if (t.n == 0 && !first) continue;
        const int blocks = (int)std::max<uint32_t>(std::min<uint32_t>(t.first[t.n], kClipBlocks), 1);
        clip_scale_kernel<<<blocks, 256, 0, st>>>(t, parts, nparts, max_norm,
                                                  first ? norm : nullptr);
    }
    return status_of(hipGetLastError());
}

}  // namespace katsu
