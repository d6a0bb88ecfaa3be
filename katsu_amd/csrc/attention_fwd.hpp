// attention_fwd.hpp -- the forward pass: one pass over the keys with each row's
// running maximum and total.
//
//   m' = max(m, max_j s_j),  l' = 2^(m-m') l + sum_j 2^(s_j-m'),
//   o' = 2^(m-m') o + sum_j 2^(s_j-m') v_j,   out = o / l,  lse = ln2 (m + log2 l)
//
// with s = scale log2(e) q.k, so that the exponential is the hardware's 2^x.
//
// A tile is BM = 32*WM rows of one key head: row r is token r / G, head r % G of
// the group, so the group shares the keys in LDS, and a single token's heads fill
// a tile's rows.  WM waves take 32 rows each; WK waves share the key tiles between
// them (each its own LDS, no barrier) and join at the end, for tiles of few rows.
//
// Bound: long prompts in bfloat16 by the matrix cores and, beside them, the exponentials
// and conversions (8192 tokens, 16/4 heads of 128, causal: 283-298 us, 0.92-0.97 PFLOP/s, matrix
// cores 55% busy, where a large library product reaches 1.33; 16384 tokens, 8 heads, all keys:
// 1.07); in float32 by the float32 instruction's rate (4096 tokens, 16/4 heads of 128, all keys:
// 1000 us, 137 TFLOP/s, of 154); single tokens in bfloat16 by reading the cache (32 of 1500-7650
// keys, 8 key heads of 128: 127-130 us, 4.6-4.7 TB/s, where a copy reaches 4.75), in float32 by
// the two waves that a CU has of 512-byte rows (532 us, 2.26 TB/s; heads of 64 3.8).  32 rows a wave, two waves a SIMD: the
// sums, q and one tile's scores fit 256 registers, and the one wave's exponentials run under
// the other's products; tiles of 64 keys (32 of 512-byte rows), two of each in LDS, let two
// blocks share a CU.
#pragma once

#include "attention.hpp"

namespace katsu {

// Until a row's maximum has grown by 2^8, its sums stay on the old one: any reference
// gives the same quotient, and sums 2^8 larger lose nothing in float32.
constexpr float kAttnSlack = 8.f;

template <typename T, int ND, int WM, int WK, int BN, bool VEC>
struct AttnFwd {
    using R = Rows<T, ND>;
    static constexpr int BM = 32 * WM, NW = WM * WK, THREADS = 64 * NW;
    static constexpr int NS = R::NS, NB = BN / 32, W = R::W;
    static constexpr int kTile = BN * R::RB;               // K or V
    static constexpr int kStages = 4 * kTile * WK;         // two of both, per key wave
    static constexpr int kMerge = WK > 1 ? WK * (ND * 4096 + 256) + 16 : 0;
    static constexpr int kLds = kStages > kMerge ? kStages : kMerge;
    using Copy = TileCopy<T, ND, BN, (WK > 1 ? 1 : WM), VEC>;

    // One key tile: scores, the running softmax, the values.  row, col: this lane's places
    // in the tile of keys and in that of values.
    __device__ static __forceinline__ void tile(lds_at row, lds_at col, const uintx4 (&qf)[NS],
                                                floatx16 (&o)[ND], float &m, float &l,
                                                float scale2, bool mask, int jmax, int h) {
        floatx16 s[NB] = {};
        ColFrags<ND> c;
        row_product<T, ND, NB, 4, true>(s, row, 0, [&](int st) { return qf[st]; },
                                  [&] { c = col_frags<T, ND>(col, 0, 0); });
        if (mask) {
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int v = 0; v < 16; ++v)
                    if (32 * b + reg_row(v, h) > jmax) s[b][v] = -INFINITY;
        }
        float mx = -INFINITY;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int v = 0; v < 16; ++v) mx = fmaxf(mx, s[b][v]);
        mx = half_max(mx) * scale2;
        if (__ballot(mx > m + kAttnSlack)) {  // the first keys: m is -inf
            const float mn = fmaxf(m, mx);
            const float by = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= by;
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int v = 0; v < 16; ++v) o[d][v] *= by;
        }
        const float ref = m == -INFINITY ? 0.f : m;
        float sum = 0.f;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                s[b][v] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][v], scale2, -ref));
                sum += s[b][v];
            }
        l += sum;
#pragma unroll
        for (int b = 0; b < NB; ++b)
            col_product<T, ND, true, false>(o, col, 32 * b, c, s[b], [&] {
                if (b + 1 < NB) c = col_frags<T, ND>(col, 32 * (b + 1), 0);
            });
    }

    // A row's result, of keys [j0, j1) of the sequence: parts of a split key axis as they are.
    struct Row {
        int64_t token;
        int head, split;
        bool valid;
    };
    __device__ static __forceinline__ float *part_of(const AttnArgs &a, const Row &r) {
        return a.part + (r.split * (a.Tq * a.H) + r.token * a.H + r.head) * W;
    }
    // The row's maximum and total; a total of -1 says that it saw no key.
    __device__ static __forceinline__ void finish_row(const AttnArgs &a, const Row &r, float m,
                                                      float l) {
        if (a.splits > 1) {
            float *ml = a.part_ml + (r.split * (a.Tq * a.H) + r.token * a.H + r.head) * 2;
            ml[0] = m;
            ml[1] = l;
        } else if (a.lse) {
            a.lse[r.head * a.Tq + r.token] =
                l < 0.f ? -INFINITY : kLn2 * (m + __builtin_amdgcn_logf(l));
        }
    }
    __device__ static __forceinline__ void finish(const AttnArgs &a, const Row &r,
                                                  const floatx16 &x, int db, int h, float m,
                                                  float l) {
        if (!r.valid) return;
        if (db == 0 && h == 0) finish_row(a, r, m, l);
        if (a.splits > 1)
            store_row<float, true>(part_of(a, r), x, 1.f, db, h, W);
        else
            store_row<T, VEC>(plain_at<T>(a.out, r.token, r.head, 0), x, l < 0.f ? 0.f : 1.f / l,
                              db, h, a.D);
    }
    __device__ static __forceinline__ void careful(const AttnArgs &a, const Row &r, int64_t k0,
                                                   int kvh, int j0, int j1, int h) {
        constexpr int N = ND * 16;
        const int c0 = h * N, n = min(max(a.D - c0, 0), N);
        const T *q = plain_at<T>(a.q, r.valid ? r.token : 0, r.head, c0);
        float m = -INFINITY, l = j0 < j1 ? 0.f : -1.f, acc[N] = {};
        for (int j = j0; j < j1; ++j) {
            const float s =
                plain_dot(q, plain_at<T>(a.k, k0 + j, kvh, c0), n) * a.scale2;
            const float mn = fmaxf(m, s), ref = mn == -INFINITY ? 0.f : mn;
            const float by = __builtin_amdgcn_exp2f(m - ref), p = __builtin_amdgcn_exp2f(s - ref);
            m = mn;
            l = l * by + p;
#pragma unroll
            for (int i = 0; i < N; ++i) acc[i] *= by;
            plain_add(acc, p, plain_at<T>(a.v, k0 + j, kvh, c0), n);
        }
        if (!r.valid) return;
        if (h == 0) finish_row(a, r, m, l);
        if (a.splits > 1)
            plain_store(part_of(a, r) + c0, acc, 1.f, n);
        else
            plain_store(plain_at<T>(a.out, r.token, r.head, c0), acc, l < 0.f ? 0.f : 1.f / l, n);
    }

    __device__ static void run(const AttnArgs &a, char *lds) {
        const int tid = threadIdx.x, lane = tid & 63, wave = uni(tid >> 6);
        const int l31 = lane & 31, h = lane >> 5;
        const int wm = WK > 1 ? 0 : wave, wk = WK > 1 ? wave : 0;
        // Key heads innermost (blocks go round-robin over the 8 XCDs, so an XCD's L2
        // holds few heads' keys).
        const unsigned id = block_id();
        const int kvh = id % a.Hkv, split = id / a.Hkv % a.splits;
        const int rank = (int)(id / a.Hkv / a.splits);
        AttnTile tl;
        if (!(WK > 1 ? tile_by_place(a, a.cu_q, a.Tq, a.G, BM, rank, lane, tl)
                     : tile_by_work(a, a.cu_q, a.Tq, a.G, BM, rank, lane, tl)))
            return;
        const AttnSeq sq = tl.seq;
        const int64_t rows = (int64_t)sq.lq * a.G, row0 = (int64_t)tl.at * BM;
        if (row0 >= rows) return;
        const int64_t r = row0 + wm * 32 + l31;
        const int tok = (int)(r / a.G);
        const Row me = {sq.q0 + tok, kvh * a.G + (int)(r % a.G), split, r < rows};
        const int shift = sq.lk - sq.lq;  // query i sees keys up to i + shift
        auto sees = [&](int64_t row) {    // how many keys
            return !a.causal ? sq.lk : min(max((int)(row / a.G) + shift + 1, 0), sq.lk);
        };
        // Rows past the sequence's end are computed with whatever they give, and not stored.
        const int seen = sees(min(r, rows - 1)), jmax = seen - 1;
        const int wend = sees(min(row0 + wm * 32 + 31, rows - 1)), wall = sees(row0 + wm * 32);
        const int tiles = (sees(min(row0 + BM - 1, rows - 1)) + BN - 1) / BN;
        const int per = (tiles + a.splits - 1) / a.splits;
        const int f0 = split * per, t0 = f0 + wk, t1 = min(tiles, f0 + per);

        Copy ck, cv;
        ck.init(WK > 1 ? 0 : wave, lane, a.k.token, a.D);
        cv.init(WK > 1 ? 0 : wave, lane, a.v.token, a.D);
        const char *kp = (const char *)a.k.p + (sq.k0 * a.k.token + kvh * a.k.head) * sizeof(T);
        const char *vp = (const char *)a.v.p + (sq.k0 * a.v.token + kvh * a.v.head) * sizeof(T);
        char *mine = lds + wk * (4 * kTile);
        auto fetch = [&](int t, int buf) {
            char *d = mine + buf * (2 * kTile);
            const int64_t j = (int64_t)t * BN;
            ck.load(kp + j * ck.stride, sq.lk - t * BN, d);
            cv.load(vp + j * cv.stride, sq.lk - t * BN, d + kTile);
        };
        if (t0 < t1) fetch(t0, 0);
        uintx4 qf[NS];
        load_row<T, ND, VEC>(a.q, me.token, me.head, me.valid, a.D, h, qf);
        loaded(qf);
        floatx16 o[ND] = {};
        float m = -INFINITY, l = 0.f;
        bool bad = false;
        const lds_at row = row_lane<T, ND>(lane), col = col_lane<T, ND>(lane) + kTile;
        lds_at at = lds_addr(mine);
        for (int t = t0, buf = 0; t < t1; t += WK, buf ^= 1) {
            attn_wait_dma();
            if constexpr (WK == 1) __syncthreads();  // the tile is there, the other buffer read
            if (t + WK < t1) fetch(t + WK, buf ^ 1);
            const lds_at b = at + buf * (2 * kTile);
            if (t * BN < wend) {
                const bool mask = t * BN + BN > wall;
                if (mask) bad |= tile_nonfinite<T, ND, BN>(b + kTile, lane);
                tile(b + row, b + col, qf, o, m, l, a.scale2, mask, jmax - t * BN, h);
            }
        }
        l = half_sum(l);
        if (!(t0 < t1 && t0 * BN < seen)) l = -1.f;  // this row saw no key here
        const int j0 = f0 * BN, j1 = min(t1 * BN, seen);
        if constexpr (WK == 1) {
            if (bad) {
                careful(a, me, sq.k0, kvh, j0, j1, h);
                return;
            }
#pragma unroll
            for (int d = 0; d < ND; ++d) finish(a, me, o[d], d, h, m, l);
        } else {
            float *om = reinterpret_cast<float *>(lds);
            float *ml = om + WK * ND * 1024;
            int *flag = reinterpret_cast<int *>(ml + WK * 64);
            __syncthreads();
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int v = 0; v < 16; ++v) om[((wave * ND + d) * 16 + v) * 64 + lane] = o[d][v];
            if (h == 0) {
                ml[wave * 64 + l31] = m;
                ml[wave * 64 + 32 + l31] = l;
            }
            if (lane == 0) flag[wave] = bad;
            __syncthreads();
            int any = 0;
#pragma unroll
            for (int w = 0; w < WK; ++w) any |= flag[w];
            if (uni(any)) {
                if (wave == 0) careful(a, me, sq.k0, kvh, j0, j1, h);
                return;
            }
            float M = -INFINITY, L = -1.f;
#pragma unroll
            for (int w = 0; w < WK; ++w) M = fmaxf(M, ml[w * 64 + l31]);
            const float ref = M == -INFINITY ? 0.f : M;
            float by[WK];
#pragma unroll
            for (int w = 0; w < WK; ++w) {
                const float lw = ml[w * 64 + 32 + l31];
                const bool has = !(lw < 0.f);
                by[w] = has ? __builtin_amdgcn_exp2f(ml[w * 64 + l31] - ref) : 0.f;
                if (has) L = (L < 0.f ? 0.f : L) + by[w] * lw;
            }
            for (int d = wave; d < ND; d += WK) {
                floatx16 x = {};
#pragma unroll
                for (int w = 0; w < WK; ++w)
#pragma unroll
                    for (int v = 0; v < 16; ++v)
                        x[v] += by[w] * om[((w * ND + d) * 16 + v) * 64 + lane];
                finish(a, me, x, d, h, M, L);
            }
        }
    }
};

template <typename T, int ND, int WM, int WK, int BN, bool VEC, int OCC>
__global__ void __launch_bounds__(64 * WM * WK, OCC) attention_fwd_kernel(const AttnArgs a) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    AttnFwd<T, ND, WM, WK, BN, VEC>::run(a, lds);
}

// Joins the parts of the key axis.  WPR waves a row, lane l channels l and l + 64: the lanes
// hold the parts' weights, 64 of them at a time; each wave takes every WPR-th part, and the
// waves' sums are added in order.
template <typename T, int WPR>
__global__ void __launch_bounds__(256) attention_join_kernel(const AttnArgs a, int W) {
    __shared__ float sums[4][128];
    const int lane = threadIdx.x & 63, wave = uni(threadIdx.x >> 6);
    const int64_t rows = a.Tq * a.H;
    const int64_t row = WPR == 1 ? (int64_t)blockIdx.x * 4 + wave : (int64_t)blockIdx.x;
    if (row >= rows) return;  // a whole wave, or (one row a block) never
    const int first = WPR == 1 ? 0 : wave;
    const float *ml = a.part_ml + row * 2;
    float M = -INFINITY;
    bool some = false;
    for (int s = lane; s < a.splits; s += 64)
        if (!(ml[s * rows * 2 + 1] < 0.f)) {  // no total is negative
            M = fmaxf(M, ml[s * rows * 2]);
            some = true;
        }
    some = __ballot(some) != 0;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) M = fmaxf(M, __shfl_xor(M, off, 64));
    const float ref = M == -INFINITY ? 0.f : M;
    float L = 0.f, x[2] = {0.f, 0.f};
    for (int s0 = 0; s0 < a.splits; s0 += 64) {
        const int s = s0 + lane, n = min(a.splits - s0, 64);
        float w = 0.f;
        if (s < a.splits && !(ml[s * rows * 2 + 1] < 0.f)) {
            w = __builtin_amdgcn_exp2f(ml[s * rows * 2] - ref);
            L += w * ml[s * rows * 2 + 1];
        }
        const bool has = s < a.splits && !(ml[s * rows * 2 + 1] < 0.f);
        const uint64_t there = __ballot(has);  // parts without a key hold nothing
#pragma unroll 8
        for (int i = first; i < n; i += WPR) {
            if (!(there >> i & 1)) continue;
            const float by = as_float(__builtin_amdgcn_readlane(as_bits(w), i));
            const float *p = a.part + ((s0 + i) * rows + row) * W + lane;
            if (lane < a.D) x[0] += by * p[0];
            if (lane + 64 < a.D) x[1] += by * p[64];
        }
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) L += __shfl_xor(L, off, 64);
    if constexpr (WPR > 1) {
        sums[wave][lane] = x[0];
        sums[wave][lane + 64] = x[1];
        __syncthreads();
        if (wave != 0) return;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            x[i] = sums[0][lane + 64 * i];
#pragma unroll
            for (int w = 1; w < WPR; ++w) x[i] += sums[w][lane + 64 * i];
        }
    }
    const int64_t token = row / a.H;
    const int head = (int)(row % a.H);
    T *p = plain_at<T>(a.out, token, head, 0);
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if (lane + 64 * i < a.D) p[lane + 64 * i] = (T)(some ? x[i] / L : 0.f);
    if (lane == 0 && a.lse)
        a.lse[head * a.Tq + token] = some ? kLn2 * (M + __builtin_amdgcn_logf(L)) : -INFINITY;
}

}  // namespace katsu
