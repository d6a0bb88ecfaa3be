// attention_bwd.hpp -- the backward pass.  With P = 2^(s - lse2), s = scale log2(e) q.k,
// recomputed tile by tile from the forward pass's lse (lse2 = log2(e) lse):
//
//   delta_i = do_i . o_i          dP = do v^T          dS = P (dP - delta)
//   dq = scale dS k               dk = scale dS^T q    dv = P^T do
//
// Two kernels and no atomics: the sums over keys (dq) and over queries (dk, dv) each stay
// in the registers of the wave that owns the row.  That computes the scores and dP twice,
// seven products for five, and gives the same bits on every call.
#pragma once

#include "attention.hpp"

namespace katsu {

// ---- dq, delta and lse2 --------------------------------------------------------
// As the forward pass: a wave owns 32 rows (a row's scores in one lane and its partner),
// the block's waves share the key tiles.
template <typename T, int DP, int BN, bool VEC>
struct AttnDq {
    using R = Rows<T, DP>;
    static constexpr int BM = 128, THREADS = 256;
    static constexpr int NS = R::CH / 2, ND = DP / 32, NB = BN / 32, NF = 16 / R::E;
    static constexpr int kTile = BN * R::RB, kLds = 4 * kTile;
    using Copy = TileCopy<T, DP, BN, 4, VEC>;

    template <bool MASK>
    __device__ static __forceinline__ void tile(const char *kl, const char *vl,
                                                const uintx4 (&qf)[NS], const uintx4 (&gf)[NS],
                                                floatx16 (&dq)[ND], float lse2, float delta,
                                                float scale2, int key0, int jmax, int lane) {
        const int l31 = lane & 31, h = lane >> 5;
        const bool bad = MASK && tile_nonfinite<T, DP, BN>(kl, lane);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            floatx16 s = {}, g = {};
#pragma unroll
            for (int st = 0; st < NS; ++st)
                s = attn_mma<T>(row_frag<T, DP>(kl, 32 * b, st, l31, h), qf[st], s);
#pragma unroll
            for (int st = 0; st < NS; ++st)
                g = attn_mma<T>(row_frag<T, DP>(vl, 32 * b, st, l31, h), gf[st], g);
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[v], scale2, -lse2));
                g[v] = p * (g[v] - delta);
                if (MASK && key0 + 32 * b + reg_row(v, h) > jmax) g[v] = 0.f;
            }
#pragma unroll
            for (int f = 0; f < NF; ++f) {
                const uintx4 p = reg_frag<T>(g, f);
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    uintx4 k = col_frag<T, DP>(kl, 32 * b, f, d, lane);
                    if (MASK && bad) k = clear_nonfinite<T>(k);
                    dq[d] = attn_mma<T>(k, p, dq[d]);
                }
            }
        }
        if (MASK && bad) {
            const int seen = min(max(jmax + 1 - key0, 0), BN);
#pragma unroll
            for (int d = 0; d < ND; ++d) add_nonfinite<T, DP, true>(kl, 0, seen, d, h, dq[d]);
        }
    }

    __device__ static void run(const AttnArgs &a, char *lds) {
        const int tid = threadIdx.x, lane = tid & 63, wave = uni(tid >> 6);
        const int l31 = lane & 31, h = lane >> 5;
        const unsigned id = blockIdx.x;
        const int kvh = id % a.Hkv, slot = a.slots - 1 - (int)(id / a.Hkv);
        const AttnSeq sq = find_seq(a, a.cu_q, a.Tq, a.G, BM, slot, lane);
        const int64_t rows = (int64_t)sq.lq * a.G;
        const int64_t row0 =
            (int64_t)(slot - uni(first_slot(a.cu_q, sq.s, a.Tq, a.G, BM))) * BM;
        if (row0 >= rows) return;
        const int64_t r = row0 + wave * 32 + l31;
        const bool valid = r < rows;
        const int tok = (int)(r / a.G), head = kvh * a.G + (int)(r % a.G);
        const int shift = sq.lk - sq.lq;
        const int jmax = !valid ? -1 : a.causal ? min(tok + shift, sq.lk - 1) : sq.lk - 1;
        const int wtop = (int)(min(row0 + wave * 32 + 31, rows - 1) / a.G);
        const int wend = row0 + wave * 32 >= rows ? 0
                         : a.causal ? min(max(wtop + shift + 1, 0), sq.lk) : sq.lk;
        const int wall = row0 + wave * 32 + 31 >= rows ? 0
                         : a.causal
                             ? min(max((int)((row0 + wave * 32) / a.G) + shift + 1, 0), sq.lk)
                             : sq.lk;
        const int btop = (int)(min(row0 + BM - 1, rows - 1) / a.G);
        const int end = a.causal ? min(max(btop + shift + 1, 0), sq.lk) : sq.lk;
        const int tiles = (end + BN - 1) / BN;

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
        if (tiles > 0) fetch(0, 0);

        const int64_t token = sq.q0 + tok, at = head * a.Tq + token;
        uintx4 qf[NS], gf[NS];
        load_row<T, DP, VEC>(a.out, token, head, valid, a.D, h, qf);
        load_row<T, DP, VEC>(a.dout, token, head, valid, a.D, h, gf);
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
        if (valid && h == 0) {
            a.lse2[at] = lse2;
            a.delta[at] = delta;
        }
        load_row<T, DP, VEC>(a.q, token, head, valid, a.D, h, qf);

        floatx16 dq[ND] = {};
        for (int t = 0, buf = 0; t < tiles; ++t, buf ^= 1) {
            attn_wait_dma();
            __syncthreads();  // the tile is there, the other buffer read
            if (t + 1 < tiles) fetch(t + 1, buf ^ 1);
            const char *kl = lds + buf * (2 * kTile), *vl = kl + kTile;
            if (t * BN + BN <= wall)
                tile<false>(kl, vl, qf, gf, dq, lse2, delta, a.scale2, t * BN, jmax, lane);
            else if (t * BN < wend)
                tile<true>(kl, vl, qf, gf, dq, lse2, delta, a.scale2, t * BN, jmax, lane);
        }
        if (!valid) return;
        T *p = (T *)const_cast<void *>(a.dq.p) + token * a.dq.token + head * a.dq.head;
#pragma unroll
        for (int d = 0; d < ND; ++d) store_row<T, VEC>(p, dq[d], a.scale, d, h, a.D);
    }
};

// ---- dk and dv -------------------------------------------------------------------
// A wave owns 32 keys: their k and v rows in registers as B operands, the sums of dk and
// dv transposed (a lane holds its key's channels).  The block's four waves share tiles of
// QT queries, q and do, of the group's heads in turn, or of one head: then the heads' sums
// go to `part` in float32 and attention_group_kernel adds them in the heads' order.
template <typename T, int DP, int QT, bool VEC>
struct AttnDkv {
    using R = Rows<T, DP>;
    static constexpr int BK = 128, THREADS = 256;
    static constexpr int NS = R::CH / 2, ND = DP / 32, NQ = QT / 32, NF = 16 / R::E;
    static constexpr int kTile = QT * R::RB, kStage = 2 * kTile + 512, kLds = 2 * kStage;
    using Copy = TileCopy<T, DP, QT, 4, VEC>;
    static_assert(QT <= 64, "a wave copies the rows' lse2 and delta");

    // 32 queries (rows r0.. of the tile, query i0 + r0 first) against the wave's keys.
    template <bool MASK>
    __device__ static __forceinline__ void block(const char *ql, const char *gl,
                                                 const float *stats, const uintx4 (&kf)[NS],
                                                 const uintx4 (&vf)[NS], floatx16 (&dk)[ND],
                                                 floatx16 (&dv)[ND], float scale2, int r0,
                                                 int ifirst, int lane) {
        const int l31 = lane & 31, h = lane >> 5;
        floatx16 s = {}, g = {};
#pragma unroll
        for (int st = 0; st < NS; ++st)
            s = attn_mma<T>(row_frag<T, DP>(ql, r0, st, l31, h), kf[st], s);
#pragma unroll
        for (int st = 0; st < NS; ++st)
            g = attn_mma<T>(row_frag<T, DP>(gl, r0, st, l31, h), vf[st], g);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const floatx4 lse2 = *reinterpret_cast<const floatx4 *>(stats + r0 + 8 * q + 4 * h);
            const floatx4 delta =
                *reinterpret_cast<const floatx4 *>(stats + 64 + r0 + 8 * q + 4 * h);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int v = 4 * q + e;
                const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[v], scale2, -lse2[e]));
                s[v] = p;
                g[v] = p * (g[v] - delta[e]);
                if (MASK && r0 + reg_row(v, h) < ifirst) s[v] = g[v] = 0.f;
            }
        }
        const bool badg = MASK && tile_nonfinite<T, DP, 32>(gl + r0 * R::RB, lane);
        const bool badq = MASK && tile_nonfinite<T, DP, 32>(ql + r0 * R::RB, lane);
#pragma unroll
        for (int f = 0; f < NF; ++f) {
            const uintx4 p = reg_frag<T>(s, f);
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                uintx4 x = col_frag<T, DP>(gl, r0, f, d, lane);
                if (MASK && badg) x = clear_nonfinite<T>(x);
                dv[d] = attn_mma<T>(x, p, dv[d]);
            }
        }
#pragma unroll
        for (int f = 0; f < NF; ++f) {
            const uintx4 p = reg_frag<T>(g, f);
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                uintx4 x = col_frag<T, DP>(ql, r0, f, d, lane);
                if (MASK && badq) x = clear_nonfinite<T>(x);
                dk[d] = attn_mma<T>(x, p, dk[d]);
            }
        }
        if (MASK && (badg || badq)) {
            const int lo = r0 + min(max(ifirst - r0, 0), 32);
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                if (badg) add_nonfinite<T, DP, false>(gl, lo, r0 + 32, d, h, dv[d]);
                if (badq) add_nonfinite<T, DP, true>(ql, lo, r0 + 32, d, h, dk[d]);
            }
        }
    }

    __device__ static void run(const AttnArgs &a, char *lds) {
        const int tid = threadIdx.x, lane = tid & 63, wave = uni(tid >> 6);
        const int l31 = lane & 31, h = lane >> 5;
        // Heads innermost; with a causal mask the keys that most queries see first.
        const bool each = a.part != nullptr;  // one head a block
        const unsigned id = blockIdx.x, hs = each ? a.H : a.Hkv;
        const int hd = id % hs, slot = (int)(id / hs);
        const int kvh = each ? hd / a.G : hd;
        const int head0 = each ? hd : hd * a.G, heads = each ? 1 : a.G;
        const AttnSeq sq = find_seq(a, a.cu_k, a.Tk, 1, BK, slot, lane);
        const int key0 = (slot - uni(first_slot(a.cu_k, sq.s, a.Tk, 1, BK))) * BK;
        if (key0 >= sq.lk) return;
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
        // Tile n of the heads' tiles: head n / tiles, rows (t0 + n % tiles) * QT ..; the four
        // waves copy it, the first also the rows' lse2 and delta, as zeros past the end: such
        // rows have P = 1 and q, do, delta = 0, and add nothing.
        auto fetch = [&](int g, int t, int buf) {
            char *d = lds + buf * kStage;
            const int64_t i = (int64_t)(t0 + t) * QT;
            const int left = sq.lq - (int)i;
            cq.load(qp + i * cq.stride + g * a.q.head * (int64_t)sizeof(T), left, d);
            cg.load(gp + i * cg.stride + g * a.dout.head * (int64_t)sizeof(T), left, d + kTile);
            if (wave == 0) {
                const int64_t at = (head0 + g) * a.Tq + sq.q0 + i;
                const int bytes = min(left, QT) * 4;
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
                        (w ? a.delta : a.lse2) + at, (short)0, bytes, 0x00020000);
                    __builtin_amdgcn_raw_ptr_buffer_load_lds(
                        rs, (attn_lds_void *)(d + 2 * kTile + w * 256), 4, lane * 4, 0, 0, 0);
                }
            }
        };
        const int total = tiles * heads;
        if (total > 0) fetch(0, 0, 0);

        const int64_t token = sq.k0 + key;
        uintx4 kf[NS], vf[NS];
        load_row<T, DP, VEC>(a.k, token, kvh, valid, a.D, h, kf);
        load_row<T, DP, VEC>(a.v, token, kvh, valid, a.D, h, vf);
        floatx16 dk[ND] = {}, dv[ND] = {};
        int g = 0, t = 0;
        for (int n = 0, buf = 0; n < total; ++n, buf ^= 1) {
            attn_wait_dma();
            __syncthreads();  // the tile is there, the other buffer read
            const int i0 = (t0 + t) * QT;
            if (++t == tiles) {
                t = 0;
                ++g;
            }
            if (n + 1 < total) fetch(g, t, buf ^ 1);
            const char *ql = lds + buf * kStage, *gl = ql + kTile;
            const float *stats = reinterpret_cast<const float *>(gl + kTile);
#pragma unroll
            for (int q = 0; q < NQ; ++q) {
                if (i0 + 32 * q >= wall)
                    block<false>(ql, gl, stats, kf, vf, dk, dv, a.scale2, 32 * q, 0, lane);
                else if (i0 + 32 * q + 31 >= wfirst)
                    block<true>(ql, gl, stats, kf, vf, dk, dv, a.scale2, 32 * q, ifirst - i0,
                                lane);
            }
        }
        if (!valid) return;
        if (each) {
            float *pk = a.part + (hd * a.Tk + token) * DP, *pv = pk + a.H * a.Tk * DP;
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                store_row<float, true>(pk, dk[d], a.scale, d, h, DP);
                store_row<float, true>(pv, dv[d], 1.f, d, h, DP);
            }
            return;
        }
        T *pk = (T *)const_cast<void *>(a.dk.p) + token * a.dk.token + kvh * a.dk.head;
        T *pv = (T *)const_cast<void *>(a.dv.p) + token * a.dv.token + kvh * a.dv.head;
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            store_row<T, VEC>(pk, dk[d], a.scale, d, h, a.D);
            store_row<T, VEC>(pv, dv[d], 1.f, d, h, a.D);
        }
    }
};

template <typename T, int DP, int BN, bool VEC, int OCC>
__global__ void __launch_bounds__(256, OCC) attention_dq_kernel(const AttnArgs a) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    AttnDq<T, DP, BN, VEC>::run(a, lds);
}
template <typename T, int DP, int QT, bool VEC, int OCC>
__global__ void __launch_bounds__(256, OCC) attention_dkv_kernel(const AttnArgs a) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    AttnDkv<T, DP, QT, VEC>::run(a, lds);
}

// dk and dv of a key head: the sums of its group's heads, in their order.  A thread: four
// channels of one token and key head, of dk (blockIdx.y 0) or dv.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) attention_group_kernel(const AttnArgs a, int DP) {
    const int per = DP / 4;
    const int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int d = (int)(n % per) * 4, kvh = (int)(n / per % a.Hkv);
    const int64_t token = n / per / a.Hkv;
    if (token >= a.Tk || d >= a.D) return;
    const AttnTensor &t = blockIdx.y ? a.dv : a.dk;
    const float *p = a.part + ((blockIdx.y ? a.H : 0) + kvh * a.G) * a.Tk * DP + token * DP + d;
    floatx4 x = {0.f, 0.f, 0.f, 0.f};
    for (int g = 0; g < a.G; ++g) x += *reinterpret_cast<const floatx4 *>(p + g * a.Tk * DP);
    T *o = (T *)const_cast<void *>(t.p) + token * t.token + kvh * t.head + d;
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
