// attention.hpp -- attention over packed sequences, in float32 and bfloat16:
// what the forward and the two backward kernels share.
//
// Sequence s has queries cu_q[s] .. cu_q[s+1] and keys cu_k[s] .. + Lk.  Query i
// sees key j if j < Lk and, with causal set, j <= i + Lk - Lq (the last query
// sees the last key).  H query heads share Hkv key heads, G = H/Hkv neighbours
// each.
//
// The matrix instruction computes D[32 x 32] += A[32 x k] B[k x 32]; lane l holds
// column l % 32 of D, rows 8*(v/4) + 4*(l/32) + v%4 in its 16 registers v, and a
// 16-byte piece of row (column) l % 32 of A (B), that of the k's of its half l/32.
// Scores are computed with the keys along the rows, S^T = K Q^T: a lane then
// holds 16 keys' scores of one query, so a row's maximum and sum stay in the lane
// and its partner in the other half.  The keys a register holds and the k's that
// a half of the next product's B operand takes are matched by choosing that
// product's A rows accordingly, so the probabilities go from one matrix
// instruction to the next without leaving the registers.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "split3.hpp"

namespace katsu {

typedef short shortx4 __attribute__((ext_vector_type(4)));
typedef uint32_t uintx2 __attribute__((ext_vector_type(2)));

// By value: __builtin_bit_cast of a vector's element takes element 0 with this compiler.
__device__ __forceinline__ float as_float(uint32_t x) { return __builtin_bit_cast(float, x); }
__device__ __forceinline__ uint32_t as_bits(float x) { return __builtin_bit_cast(uint32_t, x); }

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.693147180559945309417f;

// One operand: elements between tokens and between heads; channels are adjacent.
struct AttnTensor {
    const void *p;
    int64_t token, head;
};
enum AttnOrder { kByPlace, kByWork, kInPairs };
struct AttnArgs {
    AttnTensor q, k, v, out, dout, dq, dk, dv;
    float *lse;                       // [H][Tq]
    float *start;                     // backward, [2][H][Tq]: -log2(e) lse, -do.o
    const int32_t *cu_q, *cu_k, *k_lens;
    int64_t Tq, Tk;
    int B, H, Hkv, G, D, causal;
    float scale, scale2;              // of the scores; times log2(e)
    int slots, splits;                // tiles of all sequences; runs of the other axis's tiles
    int parts, each;                  // dk, dv: blocks a key tile and head; one head a block
    int order;                        // AttnOrder
    float *part, *part_ml;            // the runs' sums; their rows' maxima and totals
};

// ---- the sequence a tile belongs to -----------------------------------------
// Tiles of `unit` rows, `mult` rows a token, are numbered so that sequence s
// begins at cu[s]*mult/unit + s: it has at most that many tiles until the next
// one begins, so a launch can be sized, and a tile placed, without the lengths
// being known on the host.

__device__ __forceinline__ int64_t cu_at(const int32_t *cu, int i, int64_t total) {
    const int64_t c = cu[i];
    return c < 0 ? 0 : c < total ? c : total;  // whatever the array holds, accesses stay inside
}
__device__ __forceinline__ int first_slot(const int32_t *cu, int i, int64_t total, int mult,
                                          int unit) {
    return cu ? (int)(cu_at(cu, i, total) * mult / unit) + i : 0;
}

struct AttnSeq {
    int s, q0, lq, k0, lk;
};
__device__ __forceinline__ int uni(int x) { return __builtin_amdgcn_readfirstlane(x); }
// This block's number in a launch of rows of gridDim.x of them; those past the last have no tile.
__device__ __forceinline__ unsigned block_id() { return blockIdx.y * gridDim.x + blockIdx.x; }

__device__ __forceinline__ AttnSeq seq_at(const AttnArgs &a, int s) {
    AttnSeq r;
    r.s = s;
    const int64_t qa = a.cu_q ? cu_at(a.cu_q, s, a.Tq) : 0;
    const int64_t qb = a.cu_q ? cu_at(a.cu_q, s + 1, a.Tq) : a.Tq;
    const int64_t ka = a.cu_k ? cu_at(a.cu_k, s, a.Tk) : 0;
    const int64_t kb = a.cu_k ? cu_at(a.cu_k, s + 1, a.Tk) : a.Tk;
    int64_t lk = kb > ka ? kb - ka : 0;
    if (a.k_lens) {
        const int64_t c = a.k_lens[s];
        lk = c < 0 ? 0 : c < lk ? c : lk;
    }
    r.q0 = uni((int)qa);
    r.lq = uni((int)(qb > qa ? qb - qa : 0));
    r.k0 = uni((int)ka);
    r.lk = uni((int)lk);
    return r;
}

// The sequence and the tile in it that the rank-th of a launch's `slots` places works on:
// false if none.
struct AttnTile {
    AttnSeq seq;
    int at;
};
// By place, from the last: the last sequence whose first slot is not beyond it, 64
// candidates a step, of which the first always counts: slots before the first sequence's
// (starts that begin after 0) find that one, and are no tile's.
__device__ __forceinline__ bool tile_by_place(const AttnArgs &a, const int32_t *cu, int64_t total,
                                              int mult, int unit, int rank, int lane,
                                              AttnTile &t) {
    const int slot = a.slots - 1 - rank;
    int lo = 0, n = a.B;
    if (cu) {
        while (n > 1) {
            const int step = (n + 63) >> 6, i = lane * step;
            const bool ok =
                lane == 0 || (i < n && first_slot(cu, lo + i, total, mult, unit) <= slot);
            const int at = ((int)__popcll(__ballot(ok)) - 1) * step;
            lo += at;
            n = min(step, n - at);
        }
    }
    t.seq = seq_at(a, uni(lo));
    t.at = slot - uni(first_slot(cu, t.seq.s, total, mult, unit));
    return t.at >= 0;
}
// By work, the longest first: with a causal mask tile j of a sequence has j + 1 tiles' work,
// so the ranks go down the levels j, and at each through the sequences that have a tile
// there.  Up to 64 sequences (a lane each); 64 levels a step, one a lane.  In order of place
// a launch ends on its longest tiles (2711, 1024, 1777 and 488 tokens packed: 83 us; 78 so).
// In pairs: where all blocks are on the card at once, two a CU, the second half goes up the
// levels, so that a CU's two together have the same work as any other's.
__device__ __forceinline__ bool tile_by_work(const AttnArgs &a, const int32_t *cu, int64_t total,
                                             int mult, int unit, int rank, int lane,
                                             AttnTile &t) {
    if (a.order == kByPlace || a.B > 64) return tile_by_place(a, cu, total, mult, unit, rank, lane, t);
    int n = 0;  // this lane's sequence's tiles
    if (lane < a.B) {
        const int64_t len = cu ? cu_at(cu, lane + 1, total) - cu_at(cu, lane, total) : total;
        n = len > 0 ? (int)((len * mult + unit - 1) / unit) : 0;
    }
    int most = n, all = n;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        most = max(most, __shfl_xor(most, off, 64));
        all += __shfl_xor(all, off, 64);
    }
    most = uni(most);
    all = uni(all);
    if (rank >= all) return false;
    const int half = (all + 1) / 2;
    if (a.order == kInPairs && rank >= half) rank = all - 1 - (rank - half);
    int before = 0, level = 0;
    for (int top = most; top > 0; top -= 64) {
        const int l = top - 1 - lane;
        int c = 0;
        for (int s = 0; s < a.B; ++s) c += l >= 0 && __builtin_amdgcn_readlane(n, s) > l;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int up = __shfl_up(c, off, 64);
            c += lane >= off ? up : 0;
        }
        const uint64_t over = __ballot(before + c > rank);
        if (over) {
            const int f = __builtin_ctzll(over);
            level = top - 1 - f;
            if (f > 0) before += __builtin_amdgcn_readlane(c, f - 1);
            break;
        }
        before += __builtin_amdgcn_readlane(c, 63);
    }
    const bool has = n > level;
    const uint64_t ones = __ballot(has);
    const int mine = __popcll(ones & (((uint64_t)1 << lane) - 1));
    const uint64_t which = __ballot(has && mine == rank - before);
    t.seq = seq_at(a, uni(which ? __builtin_ctzll(which) : 0));
    t.at = uni(level);
    return which != 0;
}

// ---- tiles in LDS -------------------------------------------------------------
// ND blocks of 32 channels are computed with; a tile's rows are RB bytes, of 64 or 128
// channels, those that the operand does not have zero, in 16-byte chunks.  Row r's chunk c
// lies at place c ^ swz(r): the 32 rows that a fragment reads at one chunk, and the 4 rows
// by 64 bytes that a transposing read takes, then spread over all banks (measured in a
// loop: 240 and 200 bytes a cycle and CU, the transposing read 63 with c ^ (r & 15)).
template <typename T, int ND>
struct Rows {
    static constexpr int W = ND <= 2 ? 64 : 128;                  // channels of a row in LDS
    static constexpr int E = 16 / (int)sizeof(T), RB = W * (int)sizeof(T), CH = RB / 16;
    static constexpr int NS = ND * 32 / (2 * E);                  // fragments of a row
    static constexpr int NF = 16 / E;                             // of a 32 x 32 result
    __device__ static __forceinline__ int swz(int r) {
        return CH == 8 ? (((r >> 1) & 1) << 2) | ((r >> 2) & 3) : ((r & 3) << 2) | ((r >> 2) & 3);
    }
    __device__ static __forceinline__ int at(int r, int c) { return r * RB + ((c ^ swz(r)) << 4); }
};

typedef __attribute__((address_space(3))) char *lds_char;
typedef uint32_t lds_at;  // a byte address in LDS
__device__ __forceinline__ lds_at lds_addr(const char *p) {
    return (lds_at)(uintptr_t)(lds_char)const_cast<char *>(p);
}
template <typename V>
__device__ __forceinline__ V lds_read(lds_at a) {
    return *(const __attribute__((address_space(3))) V *)(uintptr_t)a;
}

constexpr int kAttnOOB = (int)0x80000000;  // beyond any tile: such a load returns zero

// A buffer of `bytes` from base: what lies past its end reads as zero.
__device__ __forceinline__ uintx4 attn_buffer(const void *base, int bytes) {
    const uint64_t p = (uint64_t)(uintptr_t)base;
    return uintx4{(uint32_t)uni((int)(uint32_t)p), (uint32_t)uni((int)(uint32_t)(p >> 32)) & 0xffffu,
                  (uint32_t)uni(bytes), 0x00020000u};
}
// Loads to LDS directly: lane l's 16 (or 4) bytes go to `to` + 16 l (4 l).  Written out, as
// the compiler has a transposing LDS read wait for every load of the builtin's that is in
// flight, also into another tile; nothing waits for these but attn_wait_dma.  They have no
// output register.  M0 is reserved, and nothing else here uses it; the wait state is what it
// needs between its write and its use.
__device__ __forceinline__ void dma_b128(uintx4 rs, int off, lds_at to) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds"
                 :
                 : "v"(off), "s"(rs), "s"(uni((int)to))
                 : "memory");
}
__device__ __forceinline__ void dma_b32(uintx4 rs, int off, lds_at to) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dword %0, %1, 0 offen lds"
                 :
                 : "v"(off), "s"(rs), "s"(uni((int)to))
                 : "memory");
}

// Copies a tile of ROWS rows to LDS, spread over NW waves, of which this is
// wave w.  DMA: by loads that go to LDS directly, 16 bytes a lane, not waited
// for here; rows and chunks that do not exist are out of the buffer's range and
// arrive as zeros, but where all tokens share one row (a token stride of zero) the
// rows past the last hold it too, so whoever reads a tile masks them.  Else (rows
// that are not a multiple of 16 bytes, not aligned so, or overlap otherwise)
// element by element.
template <typename T, int ND, int ROWS, int NW, bool DMA>
struct TileCopy {
    using R = Rows<T, ND>;
    static constexpr int N = ROWS * R::RB / 1024 / NW;
    static_assert(N >= 1, "tile too small for the waves");
    int off[DMA ? N : 1];
    int64_t stride;  // bytes between rows
    int row_bytes, D, lane, w;

    __device__ __forceinline__ void init(int wave, int ln, int64_t token_stride, int d) {
        stride = token_stride * (int64_t)sizeof(T);
        D = d;
        row_bytes = d * (int)sizeof(T);
        lane = ln;
        w = wave;
        if constexpr (DMA) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int b = (w * N + i) * 1024 + lane * 16;
                const int r = b / R::RB, c = (b % R::RB / 16) ^ R::swz(r);
                off[i] = c * 16 < row_bytes ? r * (int)stride + c * 16 : kAttnOOB;
            }
        }
    }
    // The tile whose first row is at base; `valid` rows exist (any number).
    __device__ __forceinline__ void load(const char *base, int valid, char *lds) const {
        valid = min(valid, ROWS);
        if constexpr (DMA) {
            const int bytes = valid > 0 ? (valid - 1) * (int)stride + row_bytes : 0;
            const uintx4 rs = attn_buffer(base, bytes);
            const lds_at to = lds_addr(lds) + w * N * 1024;
#pragma unroll
            for (int i = 0; i < N; ++i) dma_b128(rs, off[i], to + i * 1024);
        } else {
            for (int c = w * 64 + lane; c < ROWS * R::CH; c += NW * 64) {
                const int r = c / R::CH, ch = c % R::CH;
                T e[R::E];
#pragma unroll
                for (int i = 0; i < R::E; ++i) {
                    const int d = ch * R::E + i;
                    e[i] = r < valid && d < D
                               ? reinterpret_cast<const T *>(base + r * stride)[d]
                               : (T)0.f;
                }
                uintx4 u;
                __builtin_memcpy(&u, e, 16);
                *reinterpret_cast<uintx4 *>(lds + R::at(r, ch)) = u;
            }
        }
    }
};
// Also for this wave's reads of LDS: the next loads go where the last tile was read.
__device__ __forceinline__ void attn_wait_dma() {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
}

// ---- fragments and products ---------------------------------------------------

// A fragment: 16 bytes a lane, k's [E*h, E*h + E) of the 2E that it covers.
template <typename T>
__device__ __forceinline__ floatx16 attn_mma(uintx4 a, uintx4 b, floatx16 c) {
    if constexpr (sizeof(T) == 2) {
        return mfma32(a, b, c);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            c = __builtin_amdgcn_mfma_f32_32x32x2f32(as_float(a[e]), as_float(b[e]), c, 0, 0, 0);
        return c;
    }
}
// Places in a tile are a lane's own part, which the tile's address is added to, changed by
// constants: an exclusive or of bits below a row's size, and an offset.  The tile's address
// changes from step to step, so the compiler cannot keep one register for each place.
//
// Rows r0 + l%32 of a tile at step's chunks: the operand of a product over channels.
template <typename T, int ND>
__device__ __forceinline__ lds_at row_lane(int lane) {
    return Rows<T, ND>::at(lane & 31, lane >> 5);
}
template <typename T, int ND>
__device__ __forceinline__ uintx4 row_frag(lds_at row, int r0, int step) {
    return lds_read<uintx4>((row ^ (step << 5)) + r0 * Rows<T, ND>::RB);
}
// Channel 32*db + l%32 of a tile's rows r0 ..: the operand of a product over rows, for the
// rows whose values registers E*f .. E*f + E - 1 of a 32 x 32 result hold.
//
// bfloat16: in each 16 lanes, lanes 4e .. 4e+3 read 16 channels of row e, and lane i
// receives channel i of the four rows; the two reads are rows 16f + 8p + 4h + 0..3.
// float32: rows 8f + 4h + e, one read each.
template <typename T, int ND>
__device__ __forceinline__ lds_at col_lane(int lane) {
    using R = Rows<T, ND>;
    const int h = lane >> 5;
    if (sizeof(T) == 2)
        return R::at(4 * h + ((lane & 15) >> 2), 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) +
               (lane & 1) * 8;
    return R::at(4 * h, (lane & 31) >> 2) + (lane & 3) * 4;
}
template <typename T, int ND>
__device__ __forceinline__ uintx4 col_frag(lds_at col, int r0, int f, int db) {
    using R = Rows<T, ND>;
    uintx4 u;
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            const lds_at a = (col ^ (((db << 2) ^ (2 * p)) << 4)) + (r0 + 16 * f + 8 * p) * R::RB;
            const uintx2 t = __builtin_bit_cast(
                uintx2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                            (__attribute__((address_space(3))) shortx4 *)(uintptr_t)a));
            u[2 * p] = t[0];
            u[2 * p + 1] = t[1];
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            u[e] = lds_read<uint32_t>((col ^ (((db << 3) ^ (e << 2) ^ (2 * (f & 1))) << 4)) +
                                      (r0 + 8 * f + e) * R::RB);
    }
    return u;
}
// Registers E*f .. of a result as the operand of a product over its rows.  In
// bfloat16 they are rounded here: 2^-9 of each probability, no more than its
// row's rounding of the output; the row's total is summed before.
template <typename T>
__device__ __forceinline__ uintx4 reg_frag(const floatx16 &x, int f) {
    uintx4 u;
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            u[i] = __builtin_bit_cast(
                uint32_t, __builtin_convertvector(floatx2{x[8 * f + 2 * i], x[8 * f + 2 * i + 1]},
                                                  bf16x2));
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = as_bits(x[4 * f + i]);
    }
    return u;
}
// What reg_frag leaves of x in bfloat16, rounded in turn: the two together hold 16 bits.
__device__ __forceinline__ uintx4 reg_frag_rest(const floatx16 &x, int f, uintx4 hi) {
    uintx4 u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t h = hi[i];
        u[i] = __builtin_bit_cast(
            uint32_t, __builtin_convertvector(floatx2{x[8 * f + 2 * i] - as_float(h << 16),
                                                      x[8 * f + 2 * i + 1] -
                                                          as_float(h & 0xffff0000u)},
                                              bf16x2));
    }
    return u;
}
// The row of a result that register v of half h holds.
__device__ __forceinline__ int reg_row(int v, int h) { return 8 * (v >> 2) + 4 * h + (v & 3); }

// The LDS reads of a product are kept one step ahead of its matrix instructions, and no
// further: the compiler would put all of them in front, and has no registers for them.  The
// fence keeps reads (HARD: and matrix instructions) in their steps; vector instructions may
// cross it.
template <bool HARD>
__device__ __forceinline__ void step_fence() {
    __builtin_amdgcn_sched_barrier(HARD ? 0x676 : 0x277);
}

template <int ND>
struct ColFrags {
    uintx4 x[ND];
};
template <typename T, int ND>
__device__ __forceinline__ ColFrags<ND> col_frags(lds_at col, int r0, int f) {
    ColFrags<ND> c;
#pragma unroll
    for (int d = 0; d < ND; ++d) c.x[d] = col_frag<T, ND>(col, r0, f, d);
    return c;
}
// acc[d] += (channels 32*d .. of the tile's rows r0 .. r0 + 31)^T x; `c` is the first step's
// operand, read already.  `ahead` reads what follows the product during its last step.
// FINE: x in bfloat16 takes part with what the rounding leaves as well.
template <typename T, int ND, bool HARD, bool FINE, class F>
__device__ __forceinline__ void col_product(floatx16 (&acc)[ND], lds_at col, int r0,
                                            ColFrags<ND> c, const floatx16 &x, F ahead) {
    constexpr int NF = Rows<T, ND>::NF;
#pragma unroll
    for (int f = 0; f < NF; ++f) {
        ColFrags<ND> n;
        if (f + 1 < NF)
            n = col_frags<T, ND>(col, r0, f + 1);
        else
            ahead();
        const uintx4 p = reg_frag<T>(x, f);
#pragma unroll
        for (int d = 0; d < ND; ++d) acc[d] = attn_mma<T>(c.x[d], p, acc[d]);
        if constexpr (FINE) {
            const uintx4 rest = reg_frag_rest(x, f, p);
#pragma unroll
            for (int d = 0; d < ND; ++d) acc[d] = attn_mma<T>(c.x[d], rest, acc[d]);
        }
        step_fence<HARD>();
        if (f + 1 < NF) c = n;
    }
}
// acc[i] += (rows r0 + 32 i .. of the tile at row) . b(step), over the channels, for NB
// blocks of 32 rows; a step is S fragments.
template <typename T, int ND, int NB, int S, bool HARD, class B, class F>
__device__ __forceinline__ void row_product(floatx16 (&acc)[NB], lds_at row, int r0, B b, F ahead) {
    constexpr int NS = Rows<T, ND>::NS, N = NB * NS;
    uintx4 c[S], n[S], y[S], z[S];
#pragma unroll
    for (int i = 0; i < S; ++i)
        if (i < N) {
            c[i] = row_frag<T, ND>(row, r0 + 32 * (i / NS), i % NS);
            y[i] = b(i % NS);
        }
    if (HARD) step_fence<true>();
#pragma unroll
    for (int st = 0; st < N; st += S) {
#pragma unroll
        for (int i = 0; i < S; ++i)
            if (st + S + i < N) {
                n[i] = row_frag<T, ND>(row, r0 + 32 * ((st + S + i) / NS), (st + S + i) % NS);
                z[i] = b((st + S + i) % NS);
            }
        if (st + S >= N) ahead();
        if (HARD) step_fence<true>();
#pragma unroll
        for (int i = 0; i < S; ++i)
            if (st + i < N) acc[(st + i) / NS] = attn_mma<T>(c[i], y[i], acc[(st + i) / NS]);
        step_fence<HARD>();
#pragma unroll
        for (int i = 0; i < S; ++i) {
            c[i] = n[i];
            y[i] = z[i];
        }
    }
}

// x of the lower half's lane and of the upper one's, in both.
__device__ __forceinline__ void halves(float x, float &lo, float &hi) {
    const uint32_t u = as_bits(x);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    lo = as_float(r[0]);
    hi = as_float(r[1]);
}
__device__ __forceinline__ float half_max(float x) {
    float a, b;
    halves(x, a, b);
    return fmaxf(a, b);
}
__device__ __forceinline__ float half_sum(float x) {
    float a, b;
    halves(x, a, b);
    return a + b;
}

// Row r's fragments of a [token][head][D] operand, straight from memory: NS of
// them, zero where the row or the channels do not exist.
template <typename T, int ND, bool VEC>
__device__ __forceinline__ void load_row(const AttnTensor &t, int64_t token, int head, bool valid,
                                         int D, int h, uintx4 *f) {
    using R = Rows<T, ND>;
    const T *p = reinterpret_cast<const T *>(t.p) + token * t.token + head * t.head;
#pragma unroll
    for (int s = 0; s < R::NS; ++s) {
        const int d = (2 * s + h) * R::E;
        uintx4 u = {0, 0, 0, 0};
        if constexpr (VEC) {
            if (valid && d < D) u = *reinterpret_cast<const uintx4 *>(p + d);
        } else {
            T e[R::E];
#pragma unroll
            for (int i = 0; i < R::E; ++i) e[i] = valid && d + i < D ? p[d + i] : (T)0.f;
            __builtin_memcpy(&u, e, 16);
        }
        f[s] = u;
    }
}
// Waits here for loads to registers: where their first use lies in a loop, the compiler has
// every turn of it wait for all loads in flight.
template <int N>
__device__ __forceinline__ void loaded(uintx4 (&f)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+v"(f[i]));
}
// Channels 32*db + 8g + 4h .. + 3 (registers 4g .. 4g+3 of x) of a row, times `by`.
template <typename T, bool VEC>
__device__ __forceinline__ void store_row(T *p, const floatx16 &x, float by, int db, int h, int D) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const int d = db * 32 + 8 * g + 4 * h;
        T e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) e[i] = (T)(x[4 * g + i] * by);
        if constexpr (VEC) {
            if (d < D) __builtin_memcpy(__builtin_assume_aligned(p + d, 4 * sizeof(T)), e, sizeof e);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (d + i < D) p[d + i] = e[i];
        }
    }
}

// ---- non-finite values in masked places -----------------------------------------
// A masked key's probability is zero, but a matrix product still multiplies it by what the
// masked row holds, and 0 * Inf is NaN.  In the tiles that the mask cuts a wave looks for
// such values; if there are any, it computes its rows again at the end, over the keys that
// they see and no others, in the plain way (`careful`: a lane a row and half of the
// channels).

// Whether rows [r0, r0 + ROWS) of the tile at `a` hold one; the same answer in every lane.
template <typename T, int ND, int ROWS>
__device__ __forceinline__ bool tile_nonfinite(lds_at a, int lane) {
    typedef unsigned short us2 __attribute__((ext_vector_type(2)));
    us2 m2 = {0, 0};
    uint32_t m1 = 0;
#pragma unroll 4
    for (int i = 0; i < ROWS * Rows<T, ND>::RB / 1024; ++i) {
        const uintx4 u = lds_read<uintx4>(a + i * 1024 + lane * 16);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t x = u[e];
            if constexpr (sizeof(T) == 2)
                m2 = __builtin_elementwise_max(m2, __builtin_bit_cast(us2, x & 0x7f807f80u));
            else
                m1 = max(m1, x & 0x7f800000u);
        }
    }
    const bool bad = sizeof(T) == 2 ? (m2[0] == 0x7f80 || m2[1] == 0x7f80) : m1 == 0x7f800000u;
    return __ballot(bad) != 0;
}
// Channels c0 .. of a row: the first n of them exist.
template <typename T>
__device__ __forceinline__ T *plain_at(const AttnTensor &t, int64_t token, int head, int c0) {
    return (T *)const_cast<void *>(t.p) + token * t.token + head * t.head + c0;
}
// x . y over n channels of this lane and its partner's.
template <typename T>
__device__ __forceinline__ float plain_dot(const T *x, const T *y, int n) {
    float s = 0.f;
    for (int i = 0; i < n; ++i) s += (float)x[i] * (float)y[i];
    return half_sum(s);
}
// acc += by x, acc's N channels in registers.
template <typename T, int N>
__device__ __forceinline__ void plain_add(float (&acc)[N], float by, const T *x, int n) {
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (i < n) acc[i] += by * (float)x[i];
}
template <typename T, int N>
__device__ __forceinline__ void plain_store(T *p, const float (&acc)[N], float by, int n) {
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (i < n) p[i] = (T)(acc[i] * by);
}

}  // namespace katsu
