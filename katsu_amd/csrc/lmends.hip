// lmends.hip -- launches of the kernels at the ends of a language model and before its
// attention: embedding, the norms of query and key heads with their turn, distillation.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "distill.hpp"
#include "embedding.hpp"
#include "headnorm.hpp"
#include "lm.hpp"

namespace katsu {
namespace {

constexpr int64_t kI32Max = 0x7fffffff, kStrideMax = (int64_t)1 << 40;
constexpr int kCUs = 256;

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

int status_of(hipError_t e) {
    if (e == hipSuccess) return KATSU_OK;
    return e == hipErrorNoDevice || e == hipErrorInvalidDevice ? KATSU_E_NODEVICE : KATSU_E_LAUNCH;
}

bool dtype_ok(int t) { return t == KATSU_F32 || t == KATSU_BF16; }
bool stride_ok(int64_t s) { return s >= 0 && s <= kStrideMax; }

// Dynamic LDS above 64 KiB must be opted into, once per kernel function.
template <auto Kern>
int lds_optin(size_t bytes) {
    if (bytes <= 65536) return KATSU_OK;
    static const hipError_t e = hipFuncSetAttribute(
        (const void *)Kern, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
    return status_of(e);
}

// A launch has fewer than 2^32 threads along x: blocks beyond that go along y.
dim3 grid_of(int64_t blocks, int z = 1) {
    const int64_t x = std::min<int64_t>(blocks, 1 << 20);
    return dim3((unsigned)x, (unsigned)cdiv(blocks, x), (unsigned)z);
}

// ---- embedding ----

constexpr uint64_t kEmbedCols = 1 << 20;

EmbedArgs embed_args(const katsu_embedding &d, const int32_t *ids) {
    EmbedArgs a{};
    a.ids = ids;
    a.tokens = (int64_t)d.tokens;
    a.vocab = (int64_t)d.vocab;
    a.cols = (int64_t)d.cols;
    a.scale = d.scale;
    return a;
}

// The gradient's shape.
enum EmbedPath { kByRows, kBySlabs, kByPasses };
struct EmbedPlan {
    EmbedPath path;
    int bits, passes, blocks, per, tile;
    int64_t tiles;
    size_t keys, counts, there, part, bytes;  // bytes of each, of all
};
size_t up16(size_t n) { return (n + 15) / 16 * 16; }
EmbedPlan embed_plan(const katsu_embedding &d) {
    EmbedPlan p{};
    const int64_t T = (int64_t)d.tokens;
    const int64_t V = (int64_t)d.vocab;
    auto bits = [](int64_t n) {  // of numbers up to n
        int b = 1;
        while (n >> b) ++b;
        return b;
    };
    // By rows: 256 tokens 13 us, 21 by slabs (32000 x 256 float32); 500 tokens would take 18 and 21, but
    // with eight ids a lane instead of four 256 tokens 14.  Slabs: one a CU, more where a block's LDS
    // does not hold its rows' counts.  Their blocks all read all ids, so with more tokens or rows the
    // passes: 16384 tokens 28 us, 46 in passes, 65536 tokens 57 and 59, 131072 tokens 94 and 74 (32000
    // x 256 bfloat16); 20000 tokens, 10^6 rows of 128 115 and 100; where one pass is enough, 32768
    // tokens 38 and 38, 65536 tokens 60 and 44 (1001 rows).
    p.per = (int)std::min<int64_t>(cdiv(V, kCUs * 32) * 32, kEmbedSlab);
    const int64_t slabs = cdiv(V, p.per);
    p.passes = (int)cdiv(bits(V), kEmbedBits);
    const bool few = T <= (p.passes == 1 ? kEmbedSlabTokens / 2 : kEmbedSlabTokens) &&
                     T * std::max<int64_t>(slabs, kCUs) <= kEmbedSlabTokens * kCUs;
    p.path = T <= kEmbedFew ? kByRows : few ? kBySlabs : kByPasses;
    if (p.path == kByRows) return p;
    if (p.path == kBySlabs) {
        p.blocks = (int)slabs;
        p.bits = bits(p.per - 1);
    } else {
        p.bits = (int)cdiv(bits(V), p.passes);
    }
    const int chunks = (int)cdiv((int64_t)d.cols, 64 * (d.dtype == KATSU_F32 ? 4 : 8));
    // Tiles of 8 tokens, more where that makes enough waves: longer tiles leave fewer parts (8192 tokens,
    // 32000 x 4096 bfloat16: 83 us in tiles of 32, 86 of 64, 91 of 16; 65536 tokens of 256 columns 57,
    // 60 and 64; 16384 of 2048 64.3, 64.5 and 64.9).
    p.tile = 8;
    while (cdiv(T, p.tile) * chunks > 2048 && p.tile < 1024) p.tile *= 2;
    p.tiles = cdiv(T, p.tile);
    p.keys = up16((size_t)T * 4);
    p.part = p.tiles > 1 ? up16((size_t)p.tiles * 2 * d.cols * 4) : 0;
    p.there = up16((size_t)cdiv(V, 32) * 4);
    p.bytes = 2 * p.keys + p.part + p.there;
    if (p.path == kByPasses) {
        p.per = (int)(cdiv(T, 256 * 1024) * 1024);
        p.per = std::max(p.per, 4096);
        p.blocks = (int)cdiv(T, p.per);
        p.counts = up16(((size_t)p.blocks << p.bits) * 4);
        p.bytes += 2 * p.keys + p.counts;
    }
    return p;
}
template <typename T>
int embed_grad(const katsu_embedding &d, const EmbedArgs &a, char *ws, hipStream_t st) {
    const EmbedPlan p = embed_plan(d);
    if (p.path == kByRows) {
        const int rows = (int)std::min<int64_t>(std::max<int64_t>(a.vocab / 8192, 1), 1 << 12);
        embed_grad_few_kernel<T><<<(unsigned)cdiv(a.vocab, 4 * rows), 256, 0, st>>>(a, rows);
        return status_of(hipGetLastError());
    }
    auto take = [&](size_t n) {
        char *at = ws;
        ws += n;
        return at;
    };
    EmbedTiles t{};
    t.a = a;
    t.part = (float *)take(p.part);
    EmbedSort s{};
    s.ids = a.ids;
    s.tokens = a.tokens;
    s.vocab = a.vocab;
    s.bits = p.bits;
    s.key = (int32_t *)take(p.keys);
    s.at = (int32_t *)take(p.keys);
    s.there = (uint32_t *)take(p.there);
    if (p.path == kBySlabs) {
        s.per = p.per;
        embed_slab_kernel<<<(unsigned)p.blocks, 1024, 0, st>>>(s);
    } else {
        constexpr size_t lds = (16 * 4 << kEmbedBits) + 64;
        const int rc = lds_optin<embed_scatter_kernel>(lds);
        if (rc != KATSU_OK) return rc;
        int32_t *key[2] = {(int32_t *)take(p.keys), s.key}, *at[2] = {(int32_t *)take(p.keys), s.at};
        s.counts = (int32_t *)take(p.counts);
        s.blocks = p.blocks;
        s.per = p.per;
        for (int i = 0; i < p.passes; ++i) {
            s.shift = i * p.bits;
            s.key = key[i & 1];
            s.at = at[i & 1];
            embed_count_kernel<<<(unsigned)p.blocks, 1024, 0, st>>>(s);
            embed_scatter_kernel<<<(unsigned)p.blocks, 1024, lds, st>>>(s);
            s.key_in = s.key;
            s.at_in = s.at;
        }
        if (!a.add) embed_there_kernel<<<(unsigned)cdiv(s.tokens, 256), 256, 0, st>>>(s);
    }
    if (!a.add) t.there = s.there;
    t.key = s.key;
    t.at = s.at;
    t.tile = p.tile;
    t.tiles = p.tiles;
    t.chunks = (int)cdiv(a.cols, 64 * Piece<T>::E);
    t.tile_blocks = cdiv(t.tiles * t.chunks, 4);
    t.zero_blocks = t.there ? cdiv(a.vocab, 8 * 4) : 0;  // eight rows a wave
    embed_tile_kernel<T><<<grid_of(t.tile_blocks + t.zero_blocks), 256, 0, st>>>(t);
    if (t.tiles > 1)
        embed_join_kernel<T><<<dim3((unsigned)t.tiles, (unsigned)cdiv(a.cols, 256)), 256, 0,
                               st>>>(t);
    return status_of(hipGetLastError());
}

// ---- heads ----

// The widest accesses that half of the turning part and the rest are multiples of, up to
// MAX elements (the gradient holds two heads at once, for which 16 bytes of bfloat16 a lane
// spill: 38 us at 6000 tokens of 20 heads of 128, 8 bytes 29), the lanes of a head, and the
// units of a lane.
template <typename T, bool INTER, int MAX, class F>
int by_head(const HeadArgs &a, F f) {
    auto with = [&](auto e) {
        constexpr int E = decltype(e)::value;
        const int units = a.R / 2 / E + (int)cdiv(a.D - a.R, 2 * E);
        auto lanes = [&](auto g, auto nu) { return f(e, g, nu, units); };
        std::integral_constant<int, 1> one;
        if constexpr (E >= 4) {
            if (units <= 4) return lanes(std::integral_constant<int, 4>(), one);
            if (units <= 8) return lanes(std::integral_constant<int, 8>(), one);
        }
        if (units <= 16) return lanes(std::integral_constant<int, 16>(), one);
        if (units <= 32) return lanes(std::integral_constant<int, 32>(), one);
        if constexpr (E <= 4)
            if (units <= 64) return lanes(std::integral_constant<int, 64>(), one);
        if constexpr (E <= 2)
            if (units <= 128)
                return lanes(std::integral_constant<int, 64>(), std::integral_constant<int, 2>());
        if constexpr (E == 1)
            if (units <= 256)
                return lanes(std::integral_constant<int, 64>(), std::integral_constant<int, 4>());
        return (int)KATSU_E_INVALID;
    };
    auto fits = [&](int e) { return a.R / 2 % e == 0 && (a.D - a.R) % e == 0; };
    if constexpr (MAX == 8)
        if (fits(8)) return with(std::integral_constant<int, 8>());
    if (fits(4)) return with(std::integral_constant<int, 4>());
    if (fits(2)) return with(std::integral_constant<int, 2>());
    return with(std::integral_constant<int, 1>());
}
template <class F>
int by_head_type(const katsu_qk_norm_rotary &d, F f) {
    auto with = [&](auto t) {
        return d.interleaved ? f(t, std::true_type()) : f(t, std::false_type());
    };
    return d.dtype == KATSU_F32 ? with(float()) : with(__bf16());
}

HeadArgs head_args(const katsu_qk_norm_rotary &d, const float *table, const int32_t *positions) {
    HeadArgs a{};
    for (int i = 0; i < 2; ++i) {
        HeadTensor &t = a.t[i];
        const int64_t(&in)[2] = i ? d.k_stride : d.q_stride;
        const int64_t(&out)[2] = i ? d.k_out_stride : d.q_out_stride;
        t.x_token = in[0];
        t.x_head = in[1];
        t.out_token = out[0];
        t.out_head = out[1];
        t.heads = (int)(i ? d.k_heads : d.heads);
    }
    auto inverse = [](uint64_t n) { return n > 1 ? ~(uint64_t)0 / n + 1 : 0; };
    a.inv[0] = inverse(d.heads);
    a.inv[1] = inverse(d.k_heads);
    a.inv[2] = inverse(d.heads + d.k_heads);
    a.table = table;
    a.positions = positions;
    a.tokens = (int64_t)d.tokens;
    a.length = (int64_t)d.length;
    a.D = (int)d.head_dim;
    a.R = (int)d.rotary_dim;
    a.eps = d.eps;
    a.inv_d = 1.f / (float)d.head_dim;
    return a;
}

// Blocks of the gradient's launch: of q, of k; each block's sums of dw are a part. Five a CU
// (20 waves) over the whole, shared by the numbers of heads: with the next head on its way
// 16 waves a CU took 34 us, 20 29.5, 24 30.5 (6000 tokens of 20 heads of 128, bfloat16); few
// heads get no block with fewer than 16 of them.
void head_blocks(const katsu_qk_norm_rotary &d, int (&blocks)[2]) {
    const int64_t most = 5 * kCUs, n = (int64_t)(d.heads + d.k_heads);
    const int64_t heads[2] = {(int64_t)d.heads, (int64_t)d.k_heads};
    for (int i = 0; i < 2; ++i) {
        const int64_t items = heads[i] * (int64_t)d.tokens;
        blocks[i] = items == 0 ? 0
                               : (int)std::min(cdiv(items, 16),
                                               std::max<int64_t>(1, most * heads[i] / n));
    }
}

// ---- distillation ----

// log2(e) / tau: what the kernels multiply differences of logits with.
float exponent_scale(float tau) { return (float)(1.4426950408889634 / (double)tau); }

DistillArgs distill_args(const katsu_distillation &d, const void *logits, const int32_t *ids,
                         const void *teacher) {
    DistillArgs a{};
    a.z = logits;
    a.teacher = teacher;
    a.ids = ids;
    a.rows = (int64_t)d.rows;
    a.vocab = (int64_t)d.vocab;
    a.z_row = d.stride;
    a.dz_row = d.out_stride;
    a.dloss_step = d.dloss_stride;
    a.run = a.vocab;
    a.top = (int)d.top;
    a.teacher_bf16 = d.teacher_dtype == KATSU_BF16;
    a.tau = d.temperature;
    a.scale2 = exponent_scale(d.temperature);
    return a;
}
// Four of a thread's pieces in flight where it has as many; where it has not, the look at each
// costs more than it gives (the loss of 8000 x 1000 bfloat16: 16 us with one, 20 with four; of
// 8000 x 8000: 34 and 32).
template <typename T, int NT, class F>
int by_pieces(int64_t cols, F f) {
    if (cols < 4 * NT * Piece<T>::E) return f(std::integral_constant<int, 1>());
    return f(std::integral_constant<int, 4>());
}
// A block a row.  16 waves where there are few rows and long ones (250 x 130000 float32: 31 us, 40
// with 4); else 4 (1000 x 32000 bfloat16: 16 us, 32 with 16), or 2 for short rows, whose time is
// the block's joins (8000 x 1000: 16 us, 22 with 4; 8000 x 16000 54 and 57; 4096 x 32000 54 and
// 52).  Rows that are read twice, for the gradient as well, fill the card with fewer (400 x
// 100000 float32: 115 us with 16 waves, 128 with 4).
template <typename T, int NT, bool GRAD>
int launch_loss(const DistillArgs &a, hipStream_t st) {
    return by_pieces<T, NT>(a.vocab, [&](auto u) {
        distill_kernel<T, NT, true, GRAD, decltype(u)::value><<<grid_of(a.rows), NT, 0, st>>>(a);
        return status_of(hipGetLastError());
    });
}
template <typename T, bool GRAD>
int launch_loss(const DistillArgs &a, hipStream_t st) {
    if (GRAD ? a.rows < 4 * kCUs : a.rows < kCUs && a.vocab > 8192)
        return launch_loss<T, 1024, GRAD>(a, st);
    if constexpr (!GRAD)
        if (a.vocab <= 16384) return launch_loss<T, 128, GRAD>(a, st);
    return launch_loss<T, 256, GRAD>(a, st);
}
// Loss and gradient with the rows in registers: threads of a row, and its pieces a thread.  Two
// waves up to 512 pieces (8000 x 3000 bfloat16: 36 us, 40 with four; 8000 x 8000 59 and 54), then
// four as long as 16 pieces a thread hold the row (8192 x 32000 bfloat16: 201 us, 226 with
// eight waves, 337 with 16).
template <typename T, class F>
bool by_row_pieces(const DistillArgs &a, F f) {
    const int64_t pieces = cdiv(a.vocab, Piece<T>::E);
    std::integral_constant<int, 128> two;
    std::integral_constant<int, 256> four;
    if (pieces <= 128) return f(two, std::integral_constant<int, 1>());
    if (pieces <= 512) return f(two, std::integral_constant<int, 4>());
    if (pieces <= 1024) return f(four, std::integral_constant<int, 4>());
    if (pieces <= 2048) return f(four, std::integral_constant<int, 8>());
    if (pieces <= 4096) return f(four, std::integral_constant<int, 16>());
    if (pieces <= 8192)
        return f(std::integral_constant<int, 512>(), std::integral_constant<int, 16>());
    if (pieces <= 16384)
        return f(std::integral_constant<int, 1024>(), std::integral_constant<int, 16>());
    return false;
}

}  // namespace

bool embedding_ok(const katsu_embedding &d) {
    return dtype_ok(d.dtype) && (d.accumulate == 0 || d.accumulate == 1) &&
           d.tokens <= (uint64_t)kI32Max && d.vocab <= (uint64_t)kI32Max && d.cols > 0 &&
           d.cols <= kEmbedCols && stride_ok(d.table_stride) && stride_ok(d.out_stride) &&
           std::isfinite(d.scale);
}
bool embedding_out_ok(uint64_t rows, uint64_t cols, int64_t stride) {
    return rows < 2 || stride >= (int64_t)cols;
}

bool rows_share(const void *a, uint64_t n_a, int64_t stride_a, uint64_t cols_a, const void *b,
                uint64_t n_b, int64_t stride_b, uint64_t cols_b, int dtype) {
    if (n_a == 0 || n_b == 0 || cols_a == 0 || cols_b == 0) return false;
    struct Rows {
        __int128 at, step, len;
        uint64_t n;
        __int128 end() const { return at + (__int128)(n - 1) * step + len; }
    };
    const int size = dtype == KATSU_F32 ? 4 : 2;
    auto rows = [&](const void *p, uint64_t n, int64_t stride, uint64_t cols) {
        Rows r{(__int128)(uintptr_t)p, (__int128)stride * size, (__int128)cols * size, n};
        if (n == 1 || r.step <= r.len) r = {r.at, 0, r.end() - r.at, 1};  // no gaps
        return r;
    };
    Rows x = rows(a, n_a, stride_a, cols_a), y = rows(b, n_b, stride_b, cols_b);
    if (x.end() <= y.at || y.end() <= x.at) return false;
    if (x.n > 1 && x.step == y.step) {  // parts of the same wider rows
        if (y.at < x.at) std::swap(x, y);
        const __int128 d = (y.at - x.at) % x.step;
        return d < x.len || d + y.len > x.step;
    }
    if (x.n > y.n) std::swap(x, y);
    for (uint64_t i = 0; i < x.n; ++i) {
        const __int128 at = x.at + (__int128)i * x.step, before = at - y.at - y.len;
        // y's first row that ends behind this one's beginning
        const __int128 j = before < 0 ? 0 : y.n > 1 ? before / y.step + 1 : 1;
        if (j < (__int128)y.n && y.at + j * y.step < at + x.len) return true;
    }
    return false;
}

int embedding(const katsu_embedding &d, const int32_t *ids, const void *table, void *out,
              hipStream_t st) {
    EmbedArgs a = embed_args(d, ids);
    a.in = table;
    a.out = out;
    a.in_row = d.table_stride;
    a.out_row = d.out_stride;
    const int64_t wide = 64 * kEmbedPieces * (d.dtype == KATSU_F32 ? 4 : 8);
    const dim3 blocks((unsigned)std::min<int64_t>(cdiv(a.tokens, 4), 1 << 20),
                      (unsigned)cdiv(a.cols, wide));
    if (d.dtype == KATSU_F32)
        embed_kernel<float><<<blocks, 256, 0, st>>>(a);
    else
        embed_kernel<__bf16><<<blocks, 256, 0, st>>>(a);
    return status_of(hipGetLastError());
}

size_t embedding_bwd_bytes(const katsu_embedding &d) { return embed_plan(d).bytes; }

int embedding_bwd(const katsu_embedding &d, const void *dout, const int32_t *ids, void *dtable,
                  void *ws, hipStream_t st) {
    EmbedArgs a = embed_args(d, ids);
    a.in = dout;
    a.out = dtable;
    a.in_row = d.out_stride;
    a.out_row = d.table_stride;
    a.add = d.accumulate;
    return d.dtype == KATSU_F32 ? embed_grad<float>(d, a, (char *)ws, st)
                                : embed_grad<__bf16>(d, a, (char *)ws, st);
}

bool heads_share(const katsu_qk_norm_rotary &d, const void *a, uint64_t heads_a,
                 const int64_t (&stride_a)[2], const void *b, uint64_t heads_b,
                 const int64_t (&stride_b)[2]) {
    if (d.tokens == 0 || heads_a == 0 || heads_b == 0) return false;
    if (a == b) return true;
    struct Rows {
        uint64_t n, cols;
        int64_t stride;
    };
    const int64_t D = (int64_t)d.head_dim;
    auto rows = [&](uint64_t heads, const int64_t(&s)[2], Rows &r) {
        if (heads == 1 || s[1] == D)  // a token's heads side by side
            r = {d.tokens, heads * d.head_dim, s[0]};
        else if (d.tokens == 1 || s[0] == D)  // a head's tokens
            r = {heads, d.tokens * d.head_dim, s[1]};
        else
            return false;
        return true;
    };
    Rows x, y;
    return rows(heads_a, stride_a, x) && rows(heads_b, stride_b, y) &&
           rows_share(a, x.n, x.stride, x.cols, b, y.n, y.stride, y.cols, d.dtype);
}

bool qk_norm_rotary_ok(const katsu_qk_norm_rotary &d) {
    if (!dtype_ok(d.dtype) || d.heads > 65535 || d.k_heads > 65535) return false;
    if (d.head_dim == 0 || d.head_dim > 512 || d.rotary_dim % 2 != 0 ||
        d.rotary_dim > d.head_dim)
        return false;
    if (d.tokens > (uint64_t)kI32Max || d.length > (uint64_t)kI32Max) return false;
    if (d.rotary_dim > 0 && d.length == 0) return false;
    // Items are divided by the heads with a product of 64 bits (head_place).
    if (d.tokens * (d.heads + d.k_heads) > (uint64_t)1 << 46) return false;
    for (const auto &s : {d.q_stride, d.k_stride, d.q_out_stride, d.k_out_stride})
        if (!stride_ok(s[0]) || !stride_ok(s[1])) return false;
    return d.eps >= 0.f && std::isfinite(d.eps);
}

int qk_norm_rotary(const katsu_qk_norm_rotary &d, const void *q, const void *k, const void *w_q,
                   const void *w_k, const float *table, const int32_t *positions, void *q_out,
                   void *k_out, hipStream_t st) {
    HeadArgs a = head_args(d, table, positions);
    a.t[0].x = q;
    a.t[0].w = w_q;
    a.t[0].out = q_out;
    a.t[1].x = k;
    a.t[1].w = w_k;
    a.t[1].out = k_out;
    return by_head_type(d, [&](auto t, auto inter) {
        using T = decltype(t);
        constexpr bool INTER = decltype(inter)::value;
        return by_head<T, INTER, 16 / sizeof(T)>(a, [&](auto e, auto g, auto nu, int units) {
            constexpr int G = decltype(g)::value;
            a.units = units;
            const int64_t items = a.tokens * (a.t[0].heads + a.t[1].heads);
            head_norm_kernel<T, INTER, decltype(e)::value, G, decltype(nu)::value>
                <<<grid_of(cdiv(items, 256 / G)), 256, 0, st>>>(a);
            return status_of(hipGetLastError());
        });
    });
}

size_t qk_norm_rotary_bwd_bytes(const katsu_qk_norm_rotary &d) {
    int blocks[2];
    head_blocks(d, blocks);
    return (size_t)(blocks[0] + blocks[1]) * d.head_dim * sizeof(float);
}

int qk_norm_rotary_bwd(const katsu_qk_norm_rotary &d, const katsu_qk_norm_rotary_grads &g,
                       const void *dq, const void *dk, const void *q, const void *k,
                       const void *w_q, const void *w_k, const float *table,
                       const int32_t *positions, void *dq_out, void *dk_out, void *dw_q,
                       void *dw_k, void *ws, hipStream_t st) {
    HeadArgs a = head_args(d, table, positions);
    head_blocks(d, a.blocks);
    a.part = (float *)ws;
    a.t[0].x = q;
    a.t[0].w = w_q;
    a.t[0].dy = dq;
    a.t[0].out = dq_out;
    a.t[0].dy_token = g.dq_stride[0];
    a.t[0].dy_head = g.dq_stride[1];
    a.t[1].x = k;
    a.t[1].w = w_k;
    a.t[1].dy = dk;
    a.t[1].out = dk_out;
    a.t[1].dy_token = g.dk_stride[0];
    a.t[1].dy_head = g.dk_stride[1];
    const int blocks = a.blocks[0] + a.blocks[1];
    int rc = KATSU_OK;
    if (blocks > 0)
        rc = by_head_type(d, [&](auto t, auto inter) {
            using T = decltype(t);
            constexpr bool INTER = decltype(inter)::value;
            return by_head<T, INTER, 4>(a, [&](auto e, auto g, auto nu, int units) {
                a.units = units;
                head_norm_bwd_kernel<T, INTER, decltype(e)::value, decltype(g)::value,
                                     decltype(nu)::value>
                    <<<dim3((unsigned)blocks), kHeadThreads, 0, st>>>(a);
                return status_of(hipGetLastError());
            });
        });
    if (rc != KATSU_OK || (!w_q && !w_k)) return rc;
    const dim3 grid((unsigned)cdiv(a.D, 32), 2);
    if (!w_q) dw_q = nullptr;
    if (!w_k) dw_k = nullptr;
    if (d.dtype == KATSU_F32)
        head_norm_sum_kernel<float><<<grid, 1024, 0, st>>>(a.part, a.blocks[0], a.blocks[1], a.D,
                                                           (float *)dw_q, (float *)dw_k);
    else
        head_norm_sum_kernel<__bf16><<<grid, 1024, 0, st>>>(a.part, a.blocks[0], a.blocks[1],
                                                            a.D, (__bf16 *)dw_q, (__bf16 *)dw_k);
    return status_of(hipGetLastError());
}

bool distillation_ok(const katsu_distillation &d) {
    return dtype_ok(d.dtype) && dtype_ok(d.teacher_dtype) && d.rows <= (uint64_t)kI32Max &&
           d.vocab <= (uint64_t)kI32Max && d.top <= kDistillTop && stride_ok(d.stride) &&
           stride_ok(d.out_stride) && stride_ok(d.dloss_stride) && d.temperature > 0.f &&
           std::isfinite(d.temperature) && std::isfinite(exponent_scale(d.temperature));
}

int distillation(const katsu_distillation &d, const void *logits, const int32_t *ids,
                 const void *teacher, float *loss, float *stats, hipStream_t st) {
    DistillArgs a = distill_args(d, logits, ids, teacher);
    a.loss = loss;
    a.stats = stats;
    return d.dtype == KATSU_F32 ? launch_loss<float, false>(a, st)
                                : launch_loss<__bf16, false>(a, st);
}

int distillation_bwd(const katsu_distillation &d, const float *dloss, const void *logits,
                     const int32_t *ids, const void *teacher, const float *stats, void *dlogits,
                     hipStream_t st) {
    DistillArgs a = distill_args(d, logits, ids, teacher);
    a.dloss = dloss;
    a.stats = const_cast<float *>(stats);
    a.dz = dlogits;
    // Few rows: runs of columns, four blocks a CU.
    const int64_t want = std::min(cdiv(4 * kCUs, a.rows), cdiv(a.vocab, 4096));
    a.run = cdiv(cdiv(a.vocab, want), 2048) * 2048;
    const dim3 grid = grid_of(a.rows, (int)cdiv(a.vocab, a.run));
    auto run = [&](auto t) {
        using T = decltype(t);
        return by_pieces<T, 256>(a.run, [&](auto u) {
            distill_kernel<T, 256, false, true, decltype(u)::value><<<grid, 256, 0, st>>>(a);
            return status_of(hipGetLastError());
        });
    };
    return d.dtype == KATSU_F32 ? run(float()) : run(__bf16());
}

int distillation_step(const katsu_distillation &d, const void *logits, const int32_t *ids,
                      const void *teacher, const float *dloss, float *loss, void *dlogits,
                      hipStream_t st) {
    DistillArgs a = distill_args(d, logits, ids, teacher);
    a.loss = loss;
    a.dloss = dloss;
    a.dz = dlogits;
    auto run = [&](auto t) {
        using T = decltype(t);
        if (by_row_pieces<T>(a, [&](auto nt, auto np) {
                constexpr int NT = decltype(nt)::value, NP = decltype(np)::value;
                distill_step_kernel<T, NT, NP><<<grid_of(a.rows), NT, 0, st>>>(a);
                return true;
            }))
            return status_of(hipGetLastError());
        return launch_loss<T, true>(a, st);  // rows that the registers do not hold
    };
    return d.dtype == KATSU_F32 ? run(float()) : run(__bf16());
}

}  // namespace katsu
