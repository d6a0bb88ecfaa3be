// embedding.hpp -- rows of a table by token, times a scale, and the table's gradient.
//
//   out[t] = scale table[ids[t]]                       (zeros where ids[t] is no row)
//   dtable[v] = (dtable[v] +) scale sum over t with ids[t] = v of dout[t]
//
// A row's sum is float32, its order the tokens' inside a tile (below) and fixed by ids and sizes.
//
// HBM-bound: each row is read and written once (16384 tokens of 32000 x 2048 float32: 40 us, 212 MB
// moved, 5.3 TB/s; the gradient in bfloat16, 200 MB: 64 us, of which adding and writing zeros 47,
// 4.3 TB/s, the sort before it 11, the join behind it 6; a copy of as much reaches 5.1).  A wave a
// token whatever its width: rows of 256 bfloat16 use half of its lanes (262144 tokens: 84 us, 32
// by the bytes; their gradient 100, 28 by the bytes), rows of 32 four (72 us, 4 by the bytes).
#pragma once

#include "lmvec.hpp"

namespace katsu {

struct EmbedArgs {
    const int32_t *ids;
    const void *in;   // table or dout
    void *out;        // out or dtable
    int64_t tokens, vocab, cols, in_row, out_row;
    float scale;
    int add;          // whether dtable is added to
};

constexpr int kEmbedPieces = 4;

// A wave a token's chunk of 4 KB, all of it in flight.
template <typename T>
__global__ void __launch_bounds__(256) embed_kernel(const EmbedArgs a) {
    constexpr int E = Piece<T>::E, N = kEmbedPieces;
    const int lane = threadIdx.x & 63;
    const int64_t c0 = (int64_t)blockIdx.y * (64 * N * E);
    for (int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); t < a.tokens;
         t += (int64_t)gridDim.x * 4) {
        const int64_t id = a.ids[t];
        const T *in = (const T *)a.in + id * a.in_row;
        T *out = (T *)a.out + t * a.out_row;
        const bool has = id >= 0 && id < a.vocab;
        float x[N][E];
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int64_t i = c0 + (k * 64 + lane) * E;
            if (has && i < a.cols) load_whole(in, i, a.cols, x[k]);
        }
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int64_t i = c0 + (k * 64 + lane) * E;
#pragma unroll
            for (int e = 0; e < E; ++e) x[k][e] = has ? x[k][e] * a.scale : 0.f;
            if (i < a.cols) store_whole(out, i, a.cols, x[k]);
        }
    }
}

template <typename T>
__device__ __forceinline__ void embed_zero_row(const EmbedArgs &a, int64_t v, int lane) {
    constexpr int E = Piece<T>::E;
    const float x[E] = {};
    for (int64_t i = (int64_t)lane * E; i < a.cols; i += 64 * E)
        store_whole((T *)a.out + v * a.out_row, i, a.cols, x);
}
// dtable[v] = (dtable[v] +) scale x, of a lane's piece.
template <typename T>
__device__ __forceinline__ void embed_write(const EmbedArgs &a, int64_t v, int64_t i, float *x) {
    constexpr int E = Piece<T>::E;
    T *out = (T *)a.out + v * a.out_row;
    float old[E] = {};
    if (a.add) load_whole(out, i, a.cols, old);
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = x[e] * a.scale + old[e];
    store_whole(out, i, a.cols, x);
}

// The gradient of up to kEmbedFew tokens: a wave a row of the table, which it compares with all
// ids, and `rows` times so; the rows that all blocks take in a turn are neighbours.
constexpr int kEmbedFew = 256;
template <typename T>
__global__ void __launch_bounds__(256) embed_grad_few_kernel(const EmbedArgs a, int rows) {
    constexpr int E = Piece<T>::E, U = 8, N = kEmbedFew / 64;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int id[N];
#pragma unroll
    for (int j = 0; j < N; ++j) id[j] = j * 64 + lane < a.tokens ? a.ids[j * 64 + lane] : -1;
    for (int r = 0; r < rows; ++r) {
        const int64_t v = ((int64_t)r * gridDim.x + blockIdx.x) * 4 + wave;
        if (v >= a.vocab) return;
        uint64_t m[N], any = 0;
#pragma unroll
        for (int j = 0; j < N; ++j) any |= m[j] = __ballot(id[j] == (int)v);
        if (!any) {
            if (!a.add) embed_zero_row<T>(a, v, lane);
            continue;
        }
        for (int64_t i = lane * E; i < a.cols + lane * E; i += 64 * E) {  // all lanes
            float x[E] = {};
#pragma unroll
            for (int j = 0; j < N; ++j)
                for (uint64_t rest = m[j]; rest;) {
                    RawPiece<T> y[U];
                    int n = 0;
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        if (!rest) break;
                        const int t = j * 64 + __builtin_ctzll(rest);
                        rest &= rest - 1;
                        if (i < a.cols) y[u].load((const T *)a.in + t * a.in_row, i, a.cols);
                        n = u + 1;
                    }
#pragma unroll
                    for (int u = 0; u < U; ++u)
                        if (u < n)
#pragma unroll
                            for (int e = 0; e < E; ++e) x[e] += y[u].at(e);
                }
            if (i < a.cols) embed_write<T>(a, v, i, x);
        }
    }
}

// ---- the gradient of more tokens: sorted by id, then summed ----------------------
// Sorting is stable, so that a row's tokens stay in order, and ids that are no row go last
// as `vocab`.  The sorted tokens are cut into tiles of `tile`, whatever rows they belong to,
// so that a frequent token is the work of many waves: a run of equal ids inside a tile is a
// row's sum, what a tile's ends cut off goes to `part` and is joined.

struct EmbedSort {
    const int32_t *ids;
    int32_t *key, *at;        // sorted ids, and their tokens
    const int32_t *key_in, *at_in;  // NULL: ids themselves
    int32_t *counts;          // [blocks][1 << bits]
    uint32_t *there;          // a bit for each row of the table
    int64_t tokens, vocab;
    int shift, bits, blocks;
    int per;                  // tokens of a block, a multiple of 1024; rows of a slab
};
struct EmbedTiles {
    EmbedArgs a;
    const int32_t *key, *at;
    const uint32_t *there;    // NULL: rows without a token stay as they are
    float *part;              // [tiles][2][cols]: what belongs to the tile before, after
    int64_t tiles;
    int tile, chunks;         // chunks: of 64 pieces
    int64_t tile_blocks, zero_blocks;  // blocks that add tokens; that set rows to zero
};

constexpr int kEmbedSlab = 512, kEmbedSlabTokens = 1 << 16, kEmbedBits = 10;
constexpr int kEmbedAhead = 16;  // rows in flight

__device__ __forceinline__ int embed_key(const int32_t *ids, int64_t t, int64_t vocab) {
    const int v = ids[t];
    return v >= 0 && v < vocab ? v : (int)vocab;
}
// Which lanes have the same digit, among those of `live`: few of them one digit after the other,
// else bit by bit.
__device__ __forceinline__ uint64_t same_digit(int d, int bits, uint64_t live) {
    uint64_t m = live;
    if (__popcll(live) <= 8) {
        for (uint64_t rest = live; rest;) {
            const int v = __builtin_amdgcn_readlane(d, __builtin_ctzll(rest));
            const uint64_t same = __ballot(d == v) & live;
            if (d == v) m = same;
            rest &= ~same;
        }
        return m;
    }
    for (int b = 0; b < bits; ++b) {
        const bool bit = d >> b & 1;
        const uint64_t on = __ballot(bit);
        m &= bit ? on : ~on;
    }
    return m;
}
// What a wave's lanes have read and written before is before what they do after.
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}
// This lane's place among its wave's equal digits so far; count[d] is the wave's.
__device__ __forceinline__ int digit_rank(int *count, int d, int bits, bool live, int lane) {
    const uint64_t m = same_digit(d, bits, __ballot(live));
    const int before = __popcll(m & (((uint64_t)1 << lane) - 1));
    int at = 0;
    if (live) at = count[d] + before;
    wave_sync();
    if (live && before == 0) count[d] += __popcll(m);
    wave_sync();
    return at;
}
// The exclusive sum over a block of 1024 threads; part: 16 values.
__device__ __forceinline__ int block_scan(int v, int *part) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int s = v;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int up = __shfl_up(s, off, 64);
        if (lane >= off) s += up;
    }
    if (lane == 63) part[wave] = s;
    __syncthreads();
    int before = 0;
    for (int w = 0; w < wave; ++w) before += part[w];
    return before + s - v;
}
// A block sorts the tokens of a slab of rows: all blocks look through all ids, count those of
// smaller rows, which are before the slab's, and each wave's of every row of the slab; then each
// wave places its tokens, of which it looks only at the batches that had some.  Bound by latency and,
// where a frequent token makes one block's waves place most of theirs, by that block's
// instructions (16384 tokens: 11 us; 23 with every match by bits, one at a time where they are few).
__global__ void __launch_bounds__(1024) embed_slab_kernel(const EmbedSort s) {
    __shared__ int count[16][kEmbedSlab], part[16], below[16], end;
    constexpr int U = 8;  // rounds of 64 tokens in a batch, of which a wave has 64 at most
    static_assert(kEmbedSlabTokens <= 16 * 64 * 64 * U, "a bit a batch");
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = (int)s.tokens;
    const int per = (n + 1023) / 1024 * 64;  // tokens of a wave
    const int t0 = min(wave * per, n), t1 = min(t0 + per, n);
    const int64_t slabs = (s.vocab + s.per - 1) / s.per;
    int *mine = count[wave];
    for (int64_t slab = blockIdx.x; slab < slabs; slab += gridDim.x) {
        const uint32_t v0 = (uint32_t)(slab * s.per);
        const uint32_t rows = (uint32_t)min((int64_t)s.per, s.vocab - v0);
        auto batch = [&](int r, uint32_t (&id)[U]) {
            const int32_t *p = s.ids + r;
            if (r + 64 * U <= t1) {
#pragma unroll
                for (int u = 0; u < U; ++u) id[u] = (uint32_t)p[u * 64 + lane];
            } else {
#pragma unroll
                for (int u = 0; u < U; ++u)
                    id[u] = r + u * 64 + lane < t1 ? (uint32_t)p[u * 64 + lane] : 0xffffffffu;
            }
        };
        for (uint32_t i = lane; i < rows; i += 64) mine[i] = 0;
        wave_sync();
        int less = 0;
        uint64_t some = 0;
        for (int r = t0, b = 0; r < t1; r += 64 * U, ++b) {
            uint32_t id[U];
            batch(r, id);
            bool any = false;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                less += id[u] < v0;
                any |= id[u] - v0 < rows;
            }
            if (!__ballot(any)) continue;
            some |= (uint64_t)1 << b;
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (id[u] - v0 < rows) atomicAdd(mine + (id[u] - v0), 1);
        }
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) less += __shfl_xor(less, off, 64);
        if (lane == 0) below[wave] = less;
        __syncthreads();
        int sum = 0;
        if (threadIdx.x < rows) {
#pragma unroll
            for (int w = 0; w < 16; ++w) sum += count[w][threadIdx.x];
        }
        // The slab's rows are whole words of bits.
        const uint64_t there = __ballot(sum > 0);
        if ((lane & 31) == 0 && threadIdx.x < rows)
            s.there[(v0 + threadIdx.x) >> 5] = (uint32_t)(there >> lane);
        int first = block_scan(sum, part);
#pragma unroll
        for (int w = 0; w < 16; ++w) first += below[w];
        if (threadIdx.x < rows) {
            int at = first;
#pragma unroll
            for (int w = 0; w < 16; ++w) {
                const int c = count[w][threadIdx.x];
                count[w][threadIdx.x] = at;
                at += c;
            }
            if (threadIdx.x + 1 == rows) end = at;
        }
        __syncthreads();
        for (; some; some &= some - 1) {
            const int r = t0 + __builtin_ctzll(some) * (64 * U);
            uint32_t id[U];
            batch(r, id);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const bool has = id[u] - v0 < rows;
                if (!__ballot(has)) continue;
                const int to = digit_rank(mine, has ? (int)(id[u] - v0) : 0, s.bits, has, lane);
                if (has) {
                    s.key[to] = (int)id[u];
                    s.at[to] = r + u * 64 + lane;
                }
            }
        }
        if (slab + 1 == slabs)  // behind the last row's tokens
            for (int t = end + (int)threadIdx.x; t < n; t += 1024) s.key[t] = (int)s.vocab;
        __syncthreads();
    }
}

// More tokens: a pass for each digit of `bits` from `shift` on, in two launches.  How many of
// each digit every block has;
__global__ void __launch_bounds__(1024) embed_count_kernel(const EmbedSort s) {
    __shared__ int count[1 << kEmbedBits];
    const int mask = (1 << s.bits) - 1;
    if (!s.key_in)  // the first launch: no row has a token yet
        for (int64_t i = (int64_t)blockIdx.x * 1024 + threadIdx.x; i < (s.vocab + 31) / 32;
             i += (int64_t)gridDim.x * 1024)
            s.there[i] = 0;
    if ((int)threadIdx.x <= mask) count[threadIdx.x] = 0;
    __syncthreads();
    const int64_t t0 = (int64_t)blockIdx.x * s.per, t1 = min(t0 + s.per, s.tokens);
    for (int64_t t = t0 + threadIdx.x; t < t1; t += 1024) {
        const int k = s.key_in ? s.key_in[t] : embed_key(s.ids, t, s.vocab);
        atomicAdd(count + (k >> s.shift & mask), 1);
    }
    __syncthreads();
    if ((int)threadIdx.x <= mask)
        s.counts[((int64_t)blockIdx.x << s.bits) + threadIdx.x] = count[threadIdx.x];
}
// then each block's places, after those of all smaller digits and of the blocks before it.
__global__ void __launch_bounds__(1024) embed_scatter_kernel(const EmbedSort s) {
    constexpr int D = 1 << kEmbedBits;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    int *count = (int *)lds, *part = count + 16 * D;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, mask = (1 << s.bits) - 1;
    int *mine = count + wave * D;
    int total = 0, before = 0;
    if ((int)threadIdx.x <= mask) {
#pragma unroll 8
        for (int b = 0; b < s.blocks; ++b) {
            const int c = s.counts[((int64_t)b << s.bits) + threadIdx.x];
            total += c;
            before += b < (int)blockIdx.x ? c : 0;
        }
    }
    const int first = block_scan(total, part) + before;
    for (int i = lane; i <= mask; i += 64) mine[i] = 0;
    wave_sync();
    // Each wave's tokens follow those of the wave before.
    const int64_t per = s.per / 16, t0 = (int64_t)blockIdx.x * s.per + wave * per;
    const int64_t t1 = min(t0 + per, s.tokens);
    for (int64_t t = t0 + lane; t < t1; t += 64) {
        const int k = s.key_in ? s.key_in[t] : embed_key(s.ids, t, s.vocab);
        atomicAdd(mine + (k >> s.shift & mask), 1);
    }
    __syncthreads();
    if ((int)threadIdx.x <= mask) {
        int at = first;
        for (int w = 0; w < 16; ++w) {
            const int c = count[w * D + threadIdx.x];
            count[w * D + threadIdx.x] = at;
            at += c;
        }
    }
    __syncthreads();
    for (int64_t r = t0; r < t1; r += 64) {
        const int64_t t = r + lane;
        const bool live = t < t1;
        int k = 0, at = 0;
        if (live) {
            k = s.key_in ? s.key_in[t] : embed_key(s.ids, t, s.vocab);
            at = s.at_in ? s.at_in[t] : (int)t;
        }
        const int to = digit_rank(mine, k >> s.shift & mask, s.bits, live, lane);
        if (!live) continue;
        s.key[to] = k;
        s.at[to] = at;
    }
}
// Which rows have a token: the first of each run of the sorted ids says so (a bit set for every
// token took 80 us of 262144 tokens' 165).
__global__ void __launch_bounds__(256) embed_there_kernel(const EmbedSort s) {
    const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (t >= s.tokens) return;
    const int k = s.key_in[t], before = t > 0 ? s.key_in[t - 1] : -1;
    if (k < s.vocab && k != before) atomicOr(s.there + (k >> 5), 1u << (k & 31));
}

// A wave a tile's chunk of 64 pieces, kEmbedAhead tokens' rows in flight (16384 tokens, 32000 x 2048
// bfloat16, all launches: 64.4 us with 16, 65.1 with 8, 67.7 with 32; 65536 tokens of 256 columns
// 57, 57 and 64).
template <typename T>
__global__ void __launch_bounds__(256) embed_tile_kernel(const EmbedTiles t) {
    constexpr int E = Piece<T>::E, U = kEmbedAhead;
    const EmbedArgs &a = t.a;
    const int lane = threadIdx.x & 63;
    const int64_t id = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
    // One of each kind by turns (16384 tokens, 32000 x 2048 bfloat16: 63 us, all tiles first 61, all
    // zeros first 65; 8192 tokens of 4096 columns 81, 82 and 80).
    const int64_t both = min(t.tile_blocks, t.zero_blocks);
    if (id >= t.tile_blocks + t.zero_blocks) return;
    const int64_t block = id < 2 * both ? (id & 1 ? t.tile_blocks : 0) + id / 2
                          : id - both + (t.zero_blocks > both ? t.tile_blocks : 0);
    if (block >= t.tile_blocks) {
        // Eight rows a wave, whose bits are read before the first store.
        const int64_t v = (block - t.tile_blocks) * 4 + (threadIdx.x >> 6);
        const int64_t mine = v + (lane & 7) * (t.zero_blocks * 4);
        if (!t.there) return;
        const uint64_t none = __ballot(mine < a.vocab && !(t.there[mine >> 5] >> (mine & 31) & 1));
        for (int i = 0; i < 8; ++i)
            if (none >> i & 1) embed_zero_row<T>(a, v + i * (t.zero_blocks * 4), lane);
        return;
    }
    const int64_t item = block * 4 + (threadIdx.x >> 6), j = item / t.chunks;
    if (j >= t.tiles) return;
    const int64_t i = (item - j * t.chunks) * (64 * E) + lane * E;
    const int64_t t0 = j * t.tile, t1 = min(t0 + t.tile, a.tokens);
    int cur = t.key[t0];
    if (cur >= a.vocab) return;
    bool before = t0 > 0 && t.key[t0 - 1] == cur;
    float x[E] = {};
    auto flush = [&](bool after) {
        if (i >= a.cols) return;
        if (!before && !after) {
            embed_write<T>(a, cur, i, x);
        } else {
            float *p = t.part + (2 * j + (before ? 0 : 1)) * a.cols;
#pragma unroll
            for (int e = 0; e < E; e += 4) store_whole<float>(p, i + e, a.cols, x + e);
        }
    };
    for (int64_t b = t0; b < t1; b += 64) {
        const bool in = b + lane < t1;
        const int key = in ? t.key[b + lane] : (int)a.vocab, at = in ? t.at[b + lane] : 0;
        const int n = __popcll(__ballot(key < a.vocab));  // the rest is no row's
        for (int r = 0; r < n; r += U) {
            RawPiece<T> y[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (r + u < n && i < a.cols)
                    y[u].load((const T *)a.in + __builtin_amdgcn_readlane(at, r + u) * a.in_row,
                              i, a.cols);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (r + u >= n) break;
                const int k = __builtin_amdgcn_readlane(key, r + u);
                if (k != cur) {
                    flush(false);
                    before = false;
                    cur = k;
#pragma unroll
                    for (int e = 0; e < E; ++e) x[e] = 0.f;
                }
#pragma unroll
                for (int e = 0; e < E; ++e) x[e] += y[u].at(e);
            }
        }
        if (n < 64) break;
    }
    flush(t1 < a.tokens && t.key[t1] == cur);
}

// A block a tile and 256 columns: the run that begins in the tile and does not end there, with
// what the next tiles have of it, each wave every fourth of them.
template <typename T>
__global__ void __launch_bounds__(256) embed_join_kernel(const EmbedTiles t) {
    __shared__ float sums[3][64][4];
    const EmbedArgs &a = t.a;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t j = blockIdx.x, t0 = j * t.tile, t1 = t0 + t.tile;
    if (t1 >= a.tokens) return;
    // Read together; most blocks end here.
    const int cur = t.key[t1], last = t.key[t1 - 1], head = t.key[t0];
    const int before = t.key[max(t0, (int64_t)1) - 1];
    if (cur >= a.vocab || last != cur) return;
    if (head == cur && t0 > 0 && before == cur) return;  // began before the tile
    const int64_t i = (int64_t)blockIdx.y * 256 + lane * 4;
    // The tiles that begin with it.
    int64_t n = 0;
    for (;;) {
        const int64_t b = (j + 1 + n + lane) * t.tile;
        const uint64_t other = __ballot(!(b < a.tokens && t.key[b] == cur));
        n += other ? __builtin_ctzll(other) : 64;
        if (other) break;
    }
    float x[4] = {};
    if (i < a.cols) {
        if (wave == 0) load_whole<float>(t.part + (2 * j + 1) * a.cols, i, a.cols, x);
#pragma unroll 8
        for (int64_t k = wave; k < n; k += 4) {
            float y[4];
            load_whole<float>(t.part + 2 * (j + 1 + k) * a.cols, i, a.cols, y);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] += y[e];
        }
    }
    if (wave > 0) {
#pragma unroll
        for (int e = 0; e < 4; ++e) sums[wave - 1][lane][e] = x[e];
    }
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int w = 0; w < 3; ++w)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] += sums[w][lane][e];
    if (i >= a.cols) return;
    T *out = (T *)a.out + cur * a.out_row;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (i + e < a.cols)
            out[i + e] = (T)(x[e] * a.scale + (a.add ? (float)out[i + e] : 0.f));
}

}  // namespace katsu
