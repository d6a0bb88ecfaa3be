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
#pragma once

#include "attention.hpp"

namespace katsu {

// 2^3: until a row's maximum has grown by more, its sums stay on the old one.
// Any reference gives the same quotient; 2^8 times 2^-24 sums lose nothing.
constexpr float kAttnSlack = 8.f;

template <typename T, int DP, int WM, int WK, int BN, bool VEC>
struct AttnFwd {
    using R = Rows<T, DP>;
    static constexpr int BM = 32 * WM, NW = WM * WK, THREADS = 64 * NW;
    static constexpr int NS = R::CH / 2, ND = DP / 32, NB = BN / 32, NF = 16 / R::E;
    static constexpr int kTile = BN * R::RB;               // K or V
    static constexpr int kStages = 4 * kTile * WK;         // two of both, per key wave
    static constexpr int kMerge = WK > 1 ? WK * (ND * 4096 + 256) : 0;
    static constexpr int kLds = kStages > kMerge ? kStages : kMerge;
    using Copy = TileCopy<T, DP, BN, (WK > 1 ? 1 : WM), VEC>;

    // One key tile: scores, the running softmax, the values.
    template <bool MASK>
    __device__ static __forceinline__ void tile(const char *kl, const char *vl,
                                                const uintx4 (&qf)[NS], floatx16 (&o)[ND], float &m,
                                                float &l, float scale2, int key0, int jmax,
                                                int lane) {
        const int l31 = lane & 31, h = lane >> 5;
        floatx16 s[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            floatx16 c = {};
#pragma unroll
            for (int st = 0; st < NS; ++st)
                c = attn_mma<T>(row_frag<T, DP>(kl, 32 * b, st, l31, h), qf[st], c);
            s[b] = c;
        }
        float mx = -INFINITY;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                if (MASK && key0 + 32 * b + reg_row(v, h) > jmax) s[b][v] = -INFINITY;
                mx = fmaxf(mx, s[b][v]);
            }
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
        bool bad = false;
        if constexpr (MASK) bad = tile_nonfinite<T, DP, BN>(vl, lane);
        if (MASK && bad) {
#pragma unroll 1
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int f = 0; f < NF; ++f) {
                    uintx4 p = reg_frag<T>(s[0], f);
                    if (NB > 1 && b == 1) p = reg_frag<T>(s[NB - 1], f);
#pragma unroll
                    for (int d = 0; d < ND; ++d)
                        o[d] = attn_mma<T>(
                            clear_nonfinite<T>(col_frag<T, DP>(vl, 32 * b, f, d, lane)), p, o[d]);
                }
            const int seen = min(max(jmax + 1 - key0, 0), BN);
#pragma unroll
            for (int d = 0; d < ND; ++d) add_nonfinite<T, DP, false>(vl, 0, seen, d, h, o[d]);
        } else {
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int f = 0; f < NF; ++f) {
                    const uintx4 p = reg_frag<T>(s[b], f);
#pragma unroll
                    for (int d = 0; d < ND; ++d)
                        o[d] = attn_mma<T>(col_frag<T, DP>(vl, 32 * b, f, d, lane), p, o[d]);
                }
        }
    }

    __device__ static void run(const AttnArgs &a, char *lds) {
        const int tid = threadIdx.x, lane = tid & 63, wave = uni(tid >> 6);
        const int l31 = lane & 31, h = lane >> 5;
        const int wm = WK > 1 ? 0 : wave, wk = WK > 1 ? wave : 0;
        // Key heads innermost (blocks go round-robin over the 8 XCDs, so an XCD's L2
        // holds few heads' keys); with a causal mask the longest rows first.
        const unsigned id = blockIdx.x;
        const int kvh = id % a.Hkv, split = id / a.Hkv % a.splits;
        const int slot = a.slots - 1 - (int)(id / a.Hkv / a.splits);
        const AttnSeq sq = find_seq(a, a.cu_q, a.Tq, a.G, BM, slot, lane);
        const int64_t rows = (int64_t)sq.lq * a.G;
        const int64_t row0 =
            (int64_t)(slot - uni(first_slot(a.cu_q, sq.s, a.Tq, a.G, BM))) * BM;
        if (row0 >= rows) return;
        const int64_t r = row0 + wm * 32 + l31;
        const bool valid = r < rows;
        const int tok = (int)(r / a.G), head = kvh * a.G + (int)(r % a.G);
        const int shift = sq.lk - sq.lq;  // query i sees keys up to i + shift
        const int jmax = !valid ? -1 : a.causal ? min(tok + shift, sq.lk - 1) : sq.lk - 1;
        // Keys that this wave's rows see at most, and those that all of them see.
        const int wtop = (int)(min(row0 + wm * 32 + 31, rows - 1) / a.G);
        const int wend = row0 + wm * 32 >= rows ? 0
                         : a.causal ? min(max(wtop + shift + 1, 0), sq.lk) : sq.lk;
        const int wall = row0 + wm * 32 + 31 >= rows ? 0
                         : a.causal
                             ? min(max((int)((row0 + wm * 32) / a.G) + shift + 1, 0), sq.lk)
                             : sq.lk;
        const int btop = (int)(min(row0 + BM - 1, rows - 1) / a.G);
        const int end = a.causal ? min(max(btop + shift + 1, 0), sq.lk) : sq.lk;
        const int tiles = (end + BN - 1) / BN, per = (tiles + a.splits - 1) / a.splits;
        const int t0 = split * per + wk, t1 = min(tiles, (split + 1) * per);

        uintx4 qf[NS];
        load_row<T, DP, VEC>(a.q, sq.q0 + tok, head, valid, a.D, h, qf);
        floatx16 o[ND] = {};
        float m = -INFINITY, l = 0.f;

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
        int buf = 0;
        for (int t = t0; t < t1; t += WK, buf ^= 1) {
            attn_wait_dma();
            if constexpr (WK == 1) __syncthreads();  // the tile is there, the other buffer read
            if (t + WK < t1) fetch(t + WK, buf ^ 1);
            const char *kl = mine + buf * (2 * kTile), *vl = kl + kTile;
            if (t * BN + BN <= wall)
                tile<false>(kl, vl, qf, o, m, l, a.scale2, t * BN, jmax, lane);
            else if (t * BN < wend)
                tile<true>(kl, vl, qf, o, m, l, a.scale2, t * BN, jmax, lane);
        }
        l = half_sum(l);

        const int64_t token = sq.q0 + tok, grow = token * a.H + head;
        // Whether this row saw a key here: one that saw none is zero, whatever keys hold.
        const bool saw = t0 < t1 && t0 * BN <= jmax;
        auto finish = [&](const floatx16 &x, int db, float M, float L) {
            if (!valid) return;
            const bool some = !(L < 0.f);
            if (a.splits > 1) {
                float *p = a.part + (split * (a.Tq * a.H) + grow) * DP;
                store_row<float, true>(p, x, 1.f, db, h, DP);
                if (db == 0 && h == 0) {
                    float *ml = a.part_ml + (split * (a.Tq * a.H) + grow) * 2;
                    ml[0] = M;
                    ml[1] = L;
                }
                return;
            }
            T *p = (T *)const_cast<void *>(a.out.p) + token * a.out.token + head * a.out.head;
            store_row<T, VEC>(p, x, some ? 1.f / L : 0.f, db, h, a.D);
            if (db == 0 && h == 0 && a.lse)
                a.lse[head * a.Tq + token] =
                    some ? kLn2 * (M + __builtin_amdgcn_logf(L)) : -INFINITY;
        };
        if (!saw) l = -1.f;  // no total is negative
        if constexpr (WK == 1) {
#pragma unroll
            for (int d = 0; d < ND; ++d) finish(o[d], d, m, l);
        } else {
            float *om = reinterpret_cast<float *>(lds);
            float *ml = om + WK * ND * 1024;
            __syncthreads();
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int v = 0; v < 16; ++v) om[((wave * ND + d) * 16 + v) * 64 + lane] = o[d][v];
            if (h == 0) {
                ml[wave * 64 + l31] = m;
                ml[wave * 64 + 32 + l31] = l;
            }
            __syncthreads();
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
                        if (by[w] != 0.f) x[v] += by[w] * om[((w * ND + d) * 16 + v) * 64 + lane];
                finish(x, d, M, L);
            }
        }
    }
};

template <typename T, int DP, int WM, int WK, int BN, bool VEC, int OCC>
__global__ void __launch_bounds__(64 * WM * WK, OCC) attention_fwd_kernel(const AttnArgs a) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    AttnFwd<T, DP, WM, WK, BN, VEC>::run(a, lds);
}

// Joins the parts of the key axis: one wave a row, lane l channels l and l + 64.
template <typename T>
__global__ void __launch_bounds__(256) attention_join_kernel(const AttnArgs a, int DP) {
    const int lane = threadIdx.x & 63;
    const int64_t rows = a.Tq * a.H, row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= rows) return;
    float M = -INFINITY, L = -1.f, x[2] = {0.f, 0.f};
    for (int s = 0; s < a.splits; ++s)
        if (!(a.part_ml[(s * rows + row) * 2 + 1] < 0.f))
            M = fmaxf(M, a.part_ml[(s * rows + row) * 2]);
    const float ref = M == -INFINITY ? 0.f : M;
    for (int s = 0; s < a.splits; ++s) {
        const float l = a.part_ml[(s * rows + row) * 2 + 1];
        if (l < 0.f) continue;
        const float by = __builtin_amdgcn_exp2f(a.part_ml[(s * rows + row) * 2] - ref);
        L = (L < 0.f ? 0.f : L) + by * l;
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (lane + 64 * i < DP) x[i] += by * a.part[(s * rows + row) * DP + lane + 64 * i];
    }
    const bool some = !(L < 0.f);
    const int64_t token = row / a.H;
    const int head = (int)(row % a.H);
    T *p = (T *)const_cast<void *>(a.out.p) + token * a.out.token + head * a.out.head;
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if (lane + 64 * i < a.D) p[lane + 64 * i] = (T)(some ? x[i] / L : 0.f);
    if (lane == 0 && a.lse)
        a.lse[head * a.Tq + token] = some ? kLn2 * (M + __builtin_amdgcn_logf(L)) : -INFINITY;
}

}  // namespace katsu
