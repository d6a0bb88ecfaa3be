// attention_bwd.hpp -- the backward pass.  With P = 2^(s - lse2), s = scale log2(e) q.k,
// recomputed tile by tile from the forward pass's lse (lse2 = log2(e) lse):
//
//   delta_i = do_i . o_i          dP = do v^T          dS = P (dP - delta)
//   dq = scale dS k               dk = scale dS^T q    dv = P^T do
//
// Rows of 128 channels have no registers for hard fences around the row products (4096
// tokens, 16/4 heads of 128, bfloat16: 508 us with, 485 without; heads of 64: 258 and 263).
//
// Two kernels and no atomics: the sums over keys (dq) and over queries (dk, dv) each stay
// in the registers of the wave that owns the row.  That computes the scores and dP twice,
// seven products for five, and gives the same bits on every call.
//
// Bound by the matrix cores: 4096 tokens, 16/4 heads of 128, bfloat16, all keys 447-474 us (1.0-1.1
// PFLOP/s of the seven products), 16384 tokens, 8 heads 3400 us (1.13); float32, 16/16 heads of
// 64: 1744 us, 138 TFLOP/s, of the 154 that a large product on the float32 instruction reaches.
// 2711 + 1024 + 1777 + 488 tokens packed, 16/4 heads, bfloat16: dq 97 us, dk and dv 138 and their
// sum 18.
#pragma once

#include "attention.hpp"

namespace katsu {

// dS of rows of up to 32 channels takes part with 16 bits: its rounding to bfloat16 would be
// the larger part of the error there (300 tokens, heads of 16: dq 2.5e-3 off against 1.7e-3
// of its own rounding), and the products are the smaller part of the time.
template <typename T, int ND>
constexpr bool kFine = sizeof(T) == 2 && ND == 1;

// ---- dq, and what dk and dv take of a row ----------------------------------------
// As the forward pass: a wave owns 32 rows (a row's scores in one lane and its partner),
// the block's waves share the key tiles.
template <typename T, int ND, int BN, bool VEC>
struct AttnDq {
    using R = Rows<T, ND>;
    static constexpr int BM = 128, THREADS = 256;
    static constexpr int NS = R::NS, NB = BN / 32;
    static constexpr int kTile = BN * R::RB, kLds = 4 * kTile;
    using Copy = TileCopy<T, ND, BN, 4, VEC>;

    // P and dP of 32 keys.
    __device__ static __forceinline__ void probs(lds_at row, const uintx4 (&qf)[NS],
                                                 const uintx4 (&gf)[NS], floatx16 &p, floatx16 &g,
                                                 float lse2, float scale2, int b) {
        floatx16 s[1] = {}, x[1] = {};
        row_product<T, ND, 1, 2, R::W == 64>(s, row, 32 * b, [&](int st) { return qf[st]; }, [] {});
        row_product<T, ND, 1, 2, R::W == 64>(x, row + kTile, 32 * b, [&](int st) { return gf[st]; }, [] {});
        g = x[0];
#pragma unroll
        for (int v = 0; v < 16; ++v)
            p[v] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[0][v], scale2, -lse2));
    }
    __device__ static __forceinline__ void tile(lds_at row, lds_at col, const uintx4 (&qf)[NS],
                                                const uintx4 (&gf)[NS], floatx16 (&dq)[ND],
                                                float lse2, float delta, float scale2, bool mask,
                                                int jmax, int h) {
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            floatx16 p, g;
            probs(row, qf, gf, p, g, lse2, scale2, b);
#pragma unroll
            for (int v = 0; v < 16; ++v) g[v] = p[v] * (g[v] - delta);
            if (mask) {
#pragma unroll
                for (int v = 0; v < 16; ++v)
                    if (32 * b + reg_row(v, h) > jmax) g[v] = 0.f;
            }
            col_product<T, ND, true, kFine<T, ND>>(dq, col, 32 * b, col_frags<T, ND>(col, 32 * b, 0), g, [] {});
        }
    }

    __device__ static void run(const AttnArgs &a, char *lds) {
        const int tid = threadIdx.x, lane = tid & 63, wave = uni(tid >> 6);
        const int l31 = lane & 31, h = lane >> 5;
        const unsigned id = block_id();
        const int kvh = id % a.Hkv, split = id / a.Hkv % a.splits;
        AttnTile tl;
        if (!tile_by_work(a, a.cu_q, a.Tq, a.G, BM, (int)(id / a.Hkv / a.splits), lane, tl))
            return;
        const AttnSeq sq = tl.seq;
        const int64_t rows = (int64_t)sq.lq * a.G, row0 = (int64_t)tl.at * BM;
        if (row0 >= rows) return;
        const int64_t r = row0 + wave * 32 + l31;
        const bool valid = r < rows;
        const int tok = (int)(r / a.G), head = kvh * a.G + (int)(r % a.G);
        const int shift = sq.lk - sq.lq;
        auto sees = [&](int64_t row) {  // how many keys
            return !a.causal ? sq.lk : min(max((int)(row / a.G) + shift + 1, 0), sq.lk);
        };
        const int seen = sees(min(r, rows - 1)), jmax = seen - 1;
        const int wend = sees(min(row0 + wave * 32 + 31, rows - 1));
        const int wall = sees(row0 + wave * 32);
        const int tiles = (sees(min(row0 + BM - 1, rows - 1)) + BN - 1) / BN;
        const int per = (tiles + a.splits - 1) / a.splits;
        const int t0 = split * per, t1 = min(tiles, t0 + per);

        Copy ck, cv;
        ck.init(wave, lane, a.k.token, a.D);
        cv.init(wave, lane, a.v.token, a.D);
        const char *kp = (const char *)a.k.p + (sq.k0 * a.k.token + kvh * a.k.head) * sizeof(T);
        const char *vp = (const char *)a.v.p + (sq.k0 * a.v.token + kvh * a.v.head) * sizeof(T);
        auto fetch = [&](int t, int buf) {
            char *d = lds + buf * (2 * kTile);
            const int64_t j = (int64_t)t * BN;
            ck.load(kp + j * ck.stride, sq.lk - t * BN, d);
            cv.load(vp + j * cv.stride, sq.lk - t * BN, d + kTile);
        };
        if (t0 < t1) fetch(t0, 0);

        const int64_t token = sq.q0 + tok, at = head * a.Tq + token;
        uintx4 qf[NS], gf[NS];
        load_row<T, ND, VEC>(a.out, token, head, valid, a.D, h, qf);
        load_row<T, ND, VEC>(a.dout, token, head, valid, a.D, h, gf);
        float delta = 0.f;
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t x = qf[s][e], y = gf[s][e];
                if constexpr (sizeof(T) == 2) {
                    delta += as_float(x << 16) * as_float(y << 16);
                    delta += as_float(x & 0xffff0000u) * as_float(y & 0xffff0000u);
                } else {
                    delta += as_float(x) * as_float(y);
                }
            }
        delta = half_sum(delta);
        const float lse2 = valid ? a.lse[at] * kLog2e : 0.f;
        load_row<T, ND, VEC>(a.q, token, head, valid, a.D, h, qf);
        loaded(qf);
        loaded(gf);
        asm volatile("" ::"v"(lse2));

        floatx16 dq[ND] = {};
        bool bad = false;
        const lds_at row = row_lane<T, ND>(lane), col = col_lane<T, ND>(lane);
        const lds_at base = lds_addr(lds);
        for (int t = t0, buf = 0; t < t1; ++t, buf ^= 1) {
            attn_wait_dma();
            __syncthreads();  // the tile is there, the other buffer read
            if (t + 1 < t1) fetch(t + 1, buf ^ 1);
            const lds_at b = base + buf * (2 * kTile);
            if (sizeof(T) == 2 && wend <= BN && t == 0) {
                // Rows whose keys are one tile: dP is near delta there, and out's rounding to
                // bfloat16 as large as what dS is to be; delta is sum P dP as well.
                delta = 0.f;
#pragma unroll 1
                for (int q = 0; q < NB; ++q) {
                    floatx16 p, g;
                    probs(b + row, qf, gf, p, g, lse2, a.scale2, q);
#pragma unroll
                    for (int v = 0; v < 16; ++v)
                        if (32 * q + reg_row(v, h) <= jmax) delta += p[v] * g[v];
                }
                delta = half_sum(delta);
            }
            if (t * BN < wend) {
                const bool mask = t * BN + BN > wall;
                if (mask) bad |= tile_nonfinite<T, ND, BN>(b, lane);
                tile(b + row, b + col, qf, gf, dq, lse2, delta, a.scale2, mask, jmax - t * BN, h);
            }
        }
        if (valid && h == 0 && split == 0) {
            a.start[at] = -lse2;
            a.start[a.H * a.Tq + at] = -delta;
        }
        float *part = a.part + ((split * a.Tq + token) * a.H + head) * R::W;
        if (bad) {
            constexpr int N = ND * 16;
            const int c0 = h * N, n = min(max(a.D - c0, 0), N);
            const T *q = plain_at<T>(a.q, valid ? token : 0, head, c0);
            const T *g = plain_at<T>(a.dout, valid ? token : 0, head, c0);
            float acc[N] = {};
            for (int j = t0 * BN; j < min(t1 * BN, seen); ++j) {
                const T *k = plain_at<T>(a.k, sq.k0 + j, kvh, c0);
                const float s = plain_dot(q, k, n);
                const float dp = plain_dot(g, plain_at<T>(a.v, sq.k0 + j, kvh, c0), n);
                plain_add(acc,
                          __builtin_amdgcn_exp2f(__builtin_fmaf(s, a.scale2, -lse2)) * (dp - delta),
                          k, n);
            }
            if (!valid) return;
            if (a.splits > 1)
                plain_store(part + c0, acc, a.scale, n);
            else
                plain_store(plain_at<T>(a.dq, token, head, c0), acc, a.scale, n);
            return;
        }
        if (!valid) return;
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            if (a.splits > 1)
                store_row<float, true>(part, dq[d], a.scale, d, h, R::W);
            else
                store_row<T, VEC>(plain_at<T>(a.dq, token, head, 0), dq[d], a.scale, d, h, a.D);
        }
    }
};

// ---- dk and dv -------------------------------------------------------------------
// A wave owns 32 keys: their k rows in registers as B operands, their v rows there or
// (VLDS: bfloat16 rows of 128, whose sums need the registers) in LDS, the sums of dk and
// dv transposed (a lane holds its key's channels).  The block's four waves share tiles of
// QT queries, q and do, of the group's heads in turn, or of one head, or of a run of
// these: then the sums go to `part` in float32 and attention_sum_kernel adds them in order.
template <typename T, int ND, int QT, bool VEC>
struct AttnDkv {
    using R = Rows<T, ND>;
    static constexpr int BK = 128, THREADS = 256;
    static constexpr int NS = R::NS, NQ = QT / 32, W = R::W;
    static constexpr bool VLDS = sizeof(T) == 2 && ND > 2;
    static constexpr int kTile = QT * R::RB, kStage = 2 * kTile + 512;
    static constexpr int kKeys = VLDS ? BK * R::RB : 0, kLds = kKeys + 2 * kStage;
    using Copy = TileCopy<T, ND, QT, 4, VEC>;
    static_assert(QT <= 64, "a wave copies what there is of each row");

    // 32 queries (rows r0 .. of the tile) against the wave's keys.  row, col: this lane's
    // places in q's tile, followed by do's; vrow: in the block's v rows; stats: -lse2 and
    // -delta.  mask: only the tile's rows [ifirst, iend) take part.
    //
    // lse2 enters with the exponential's multiply-add: score sums that start from lse / scale
    // are rounded to its size at each step (1047 tokens, heads of 80, float32: dk 1.0e-6 off
    // so, 4.9e-7 from zero).  The sums of dP start from -delta, which is of their own size.
    __device__ static __forceinline__ void block(lds_at row, lds_at col, lds_at stats, lds_at vrow,
                                                 const uintx4 (&kf)[NS], const uintx4 *vf,
                                                 floatx16 (&dk)[ND], floatx16 (&dv)[ND],
                                                 float scale2, int r0, bool mask, int ifirst,
                                                 int iend, int h) {
        floatx16 sa[1] = {}, ga[1];
        floatx16 &s = sa[0], &g = ga[0];
#pragma unroll
        for (int q = 0; q < 4; ++q) {  // sums of dP that start from -delta
            const floatx4 y = lds_read<floatx4>(stats + 256 + (r0 + 8 * q + 4 * h) * 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) g[4 * q + e] = y[e];
        }
        ColFrags<ND> c;
        row_product<T, ND, 1, 2, R::W == 64>(sa, row, r0, [&](int st) { return kf[st]; }, [] {});
        row_product<T, ND, 1, 2, R::W == 64>(
            ga, row + kTile, r0,
            [&](int st) {
                if constexpr (VLDS)
                    return row_frag<T, ND>(vrow, 0, st);
                else
                    return vf[st];
            },
            [&] { c = col_frags<T, ND>(col + kTile, r0, 0); });
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const floatx4 x = lds_read<floatx4>(stats + (r0 + 8 * q + 4 * h) * 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int v = 4 * q + e;
                s[v] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[v], scale2, x[e]));
                g[v] *= s[v];
            }
        }
        if (mask) {  // one comparison for both ends: below the first, the difference is large
            asm volatile("" : "+v"(ifirst));  // computed here: no register for it in the loop
            const uint32_t n = iend > ifirst ? iend - ifirst : 0;
#pragma unroll
            for (int v = 0; v < 16; ++v)
                if ((uint32_t)(r0 + reg_row(v, h) - ifirst) >= n) s[v] = g[v] = 0.f;
        }
        col_product<T, ND, true, false>(dv, col + kTile, r0, c, s,
                           [&] { c = col_frags<T, ND>(col, r0, 0); });
        col_product<T, ND, true, kFine<T, ND>>(dk, col, r0, c, g, [] {});
    }

    __device__ static void run(const AttnArgs &a, char *lds) {
        const int tid = threadIdx.x, lane = tid & 63, wave = uni(tid >> 6);
        const int l31 = lane & 31, h = lane >> 5;
        // A key head's queries are `parts` blocks' work: every head's tiles in `splits` runs,
        // or (!each) all heads' together.
        const unsigned id = block_id();
        const int kvh = id % a.Hkv, p = id / a.Hkv % a.parts;
        const int split = p % a.splits;
        const int head0 = kvh * a.G + (a.each ? p / a.splits : 0), heads = a.each ? 1 : a.G;
        AttnTile tl;
        if (!tile_by_work(a, a.cu_k, a.Tk, 1, BK, (int)(id / a.Hkv / a.parts), lane, tl))
            return;
        const AttnSeq sq = tl.seq;
        // The first keys have the most queries: the work of the tiles from the end.
        const int key0 = ((sq.lk + BK - 1) / BK - 1 - tl.at) * BK;
        if (key0 < 0) return;
        const int wkey = key0 + wave * 32, key = wkey + l31;
        const bool valid = key < sq.lk;
        const int shift = sq.lk - sq.lq;
        // The first query that sees this key; the block's first; the wave's first and the
        // first that sees all of the wave's keys.
        const int ifirst = a.causal ? key - shift : 0;
        const int bfirst = a.causal ? max(key0 - shift, 0) : 0;
        const int wfirst = a.causal ? wkey - shift : 0, wall = a.causal ? wkey + 31 - shift : 0;
        const int t0 = bfirst / QT, tiles = max((sq.lq + QT - 1) / QT - t0, 0);

        Copy cq, cg;
        cq.init(wave, lane, a.q.token, a.D);
        cg.init(wave, lane, a.dout.token, a.D);
        const char *qp = (const char *)a.q.p + (sq.q0 * a.q.token + head0 * a.q.head) * sizeof(T);
        const char *gp =
            (const char *)a.dout.p + (sq.q0 * a.dout.token + head0 * a.dout.head) * sizeof(T);
        // The rows' -lse2 and -delta are copied too, by the first wave, as zeros past the
        // end.  Rows past the end are masked: their P would be 1 (or NaN, of a key with Inf).
        auto fetch = [&](int g, int t, int buf) {
            char *d = lds + kKeys + buf * kStage;
            const int64_t i = (int64_t)(t0 + t) * QT;
            const int left = sq.lq - (int)i;
            cq.load(qp + i * cq.stride + g * a.q.head * (int64_t)sizeof(T), left, d);
            cg.load(gp + i * cg.stride + g * a.dout.head * (int64_t)sizeof(T), left, d + kTile);
            if (wave == 0) {
                const int64_t at = (head0 + g) * a.Tq + sq.q0 + i;
                const int bytes = min(left, QT) * 4;
#pragma unroll
                for (int w = 0; w < 2; ++w)
                    dma_b32(attn_buffer(a.start + w * (a.H * a.Tq) + at, bytes), lane * 4,
                            lds_addr(d + 2 * kTile + w * 256));
            }
        };
        const int per = (tiles * heads + a.splits - 1) / a.splits;
        const int n0 = split * per, n1 = min(tiles * heads, n0 + per);
        int g = n0 < n1 ? n0 / tiles : 0, t = n0 - g * tiles;
        if (n0 < n1) fetch(g, t, 0);

        const int64_t token = sq.k0 + key;
        uintx4 kf[NS], vf[VLDS ? 1 : NS];
        load_row<T, ND, VEC>(a.k, token, kvh, valid, a.D, h, kf);
        if constexpr (VLDS) {
            TileCopy<T, ND, 32, 1, VEC> cv;  // each wave its own rows
            cv.init(0, lane, a.v.token, a.D);
            cv.load((const char *)a.v.p +
                        ((int64_t)(sq.k0 + wkey) * a.v.token + kvh * a.v.head) * sizeof(T),
                    sq.lk - wkey, lds + wave * 32 * R::RB);
        } else {
            load_row<T, ND, VEC>(a.v, token, kvh, valid, a.D, h, vf);
            loaded(vf);
        }
        loaded(kf);
        floatx16 dk[ND] = {}, dv[ND] = {};
        bool bad = false;
        const lds_at row = row_lane<T, ND>(lane), col = col_lane<T, ND>(lane);
        const lds_at base = lds_addr(lds) + kKeys;
        lds_at vrow = row + lds_addr(lds) + wave * 32 * R::RB;
        for (int n = n0, buf = 0; n < n1; ++n, buf ^= 1) {
            attn_wait_dma();
            __syncthreads();  // the tile is there, the other buffer read
            const int i0 = (t0 + t) * QT;
            if (++t == tiles) {
                t = 0;
                ++g;
            }
            if (n + 1 < n1) fetch(g, t, buf ^ 1);
            const lds_at b = base + buf * kStage, stats = b + 2 * kTile;
            asm("" : "+v"(vrow));  // no register for each of its places
#pragma unroll
            for (int q = 0; q < NQ; ++q) {
                if (i0 + 32 * q + 31 < wfirst || i0 + 32 * q >= sq.lq) continue;
                const bool cut = i0 + 32 * q < wall;  // by the causal mask
                if (cut)
                    bad |= tile_nonfinite<T, ND, 32>(b + 32 * q * R::RB, lane) ||
                           tile_nonfinite<T, ND, 32>(b + kTile + 32 * q * R::RB, lane);
                block(b + row, b + col, stats, vrow, kf, vf, dk, dv, a.scale2, 32 * q,
                      cut || i0 + 32 * q + 32 > sq.lq, ifirst - i0, sq.lq - i0, h);
            }
        }
        float *pk = a.part + ((int64_t)(kvh * a.parts + p) * a.Tk + token) * W;
        float *pv = pk + (int64_t)a.Hkv * a.parts * a.Tk * W;
        if (bad) {
            constexpr int N = ND * 16;
            const int c0 = h * N, n = min(max(a.D - c0, 0), N);
            const T *k = plain_at<T>(a.k, valid ? token : 0, kvh, c0);
            const T *v = plain_at<T>(a.v, valid ? token : 0, kvh, c0);
            float ak[N] = {}, av[N] = {};
            for (int m = n0; m < n1; ++m) {  // the tiles' rows that see the key
                const int gg = head0 + m / tiles, i0 = (t0 + m % tiles) * QT;
                for (int i = max(ifirst, i0); i < min(sq.lq, i0 + QT); ++i) {
                    const int64_t at = gg * a.Tq + sq.q0 + i;
                    const T *q = plain_at<T>(a.q, sq.q0 + i, gg, c0);
                    const T *d = plain_at<T>(a.dout, sq.q0 + i, gg, c0);
                    const float s = plain_dot(q, k, n), dp = plain_dot(d, v, n);
                    const float w =
                        __builtin_amdgcn_exp2f(__builtin_fmaf(s, a.scale2, a.start[at]));
                    plain_add(av, w, d, n);
                    plain_add(ak, w * (dp + a.start[a.H * a.Tq + at]), q, n);
                }
            }
            if (!valid) return;
            if (a.parts > 1) {
                plain_store(pk + c0, ak, a.scale, n);
                plain_store(pv + c0, av, 1.f, n);
            } else {
                plain_store(plain_at<T>(a.dk, token, kvh, c0), ak, a.scale, n);
                plain_store(plain_at<T>(a.dv, token, kvh, c0), av, 1.f, n);
            }
            return;
        }
        if (!valid) return;
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            if (a.parts > 1) {
                store_row<float, true>(pk, dk[d], a.scale, d, h, W);
                store_row<float, true>(pv, dv[d], 1.f, d, h, W);
            } else {
                store_row<T, VEC>(plain_at<T>(a.dk, token, kvh, 0), dk[d], a.scale, d, h, a.D);
                store_row<T, VEC>(plain_at<T>(a.dv, token, kvh, 0), dv[d], 1.f, d, h, a.D);
            }
        }
    }
};

template <typename T, int ND, int BN, bool VEC, int OCC>
__global__ void __launch_bounds__(256, OCC) attention_dq_kernel(const AttnArgs a) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    AttnDq<T, ND, BN, VEC>::run(a, lds);
}
template <typename T, int ND, int QT, bool VEC, int OCC>
__global__ void __launch_bounds__(256, OCC) attention_dkv_kernel(const AttnArgs a) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    AttnDkv<T, ND, QT, VEC>::run(a, lds);
}

// Gradients from their parts, in order.  A thread: four channels of one token and head of
// each of the launch's gradients (blockIdx.y: dk and dv, or dq).  Part i of a token's head
// lies at part + head*head_step + i*part_step + token*token_step.
struct AttnSum {
    AttnTensor out[2];
    const float *part[2];
    int64_t tokens, head_step, part_step, token_step;
    int heads, parts, D, W;
};
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) attention_sum_kernel(const AttnSum a) {
    const int per = a.W / 4;
    const int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int d = (int)(n % per) * 4, head = (int)(n / per % a.heads);
    const int64_t token = n / per / a.heads;
    if (token >= a.tokens || d >= a.D) return;
    const AttnTensor &t = a.out[blockIdx.y];
    const float *p = a.part[blockIdx.y] + head * a.head_step + token * a.token_step + d;
    floatx4 x = {0.f, 0.f, 0.f, 0.f};
    for (int i = 0; i < a.parts; ++i) x += *reinterpret_cast<const floatx4 *>(p + i * a.part_step);
    T *o = plain_at<T>(t, token, head, d);
    T e[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) e[i] = (T)x[i];
    if constexpr (VEC) {
        __builtin_memcpy(__builtin_assume_aligned(o, 4 * sizeof(T)), e, sizeof e);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (d + i < a.D) o[i] = e[i];
    }
}

}  // namespace katsu
