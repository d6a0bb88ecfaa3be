// attention.hip -- launches of the attention kernels: which variant, how many
// blocks, how many parts of the key axis.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "attention_bwd.hpp"
#include "attention_fwd.hpp"
#include "lm.hpp"

namespace katsu {
namespace {

constexpr int64_t kI32Max = 0x7fffffff;
constexpr int kCUs = 256;

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

int status_of(hipError_t e) {
    if (e == hipSuccess) return KATSU_OK;
    return e == hipErrorNoDevice || e == hipErrorInvalidDevice ? KATSU_E_NODEVICE : KATSU_E_LAUNCH;
}

// Dynamic LDS above 64 KiB must be opted into, once per kernel function.
template <auto Kern>
int lds_optin(size_t bytes) {
    if (bytes <= 65536) return KATSU_OK;
    static const hipError_t e = hipFuncSetAttribute(
        (const void *)Kern, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
    return status_of(e);
}

// Any in memory: places are computed in 64 bits.
bool strides_ok(const int64_t (&s)[2]) {
    const int64_t most = (int64_t)1 << 40;
    return s[0] >= 0 && s[1] >= 0 && s[0] <= most && s[1] <= most;
}

int elem(const katsu_attention &d) { return d.dtype == KATSU_F32 ? 4 : 2; }

// 16-byte accesses: rows of whole 16-byte chunks at aligned places, a tile's rows (64 at
// most) within the 32-bit offsets of a buffer load, and rows that do not overlap unless all
// are one: a buffer's end does not tell those past the last one.
bool vec_ok(const katsu_attention &d, const void *p, const int64_t (&stride)[2]) {
    const int e = elem(d);
    return ((uintptr_t)p & 15) == 0 && d.head_dim * e % 16 == 0 && stride[0] * e % 16 == 0 &&
           stride[1] * e % 16 == 0 && stride[0] * e < (1 << 23) &&
           (stride[0] == 0 || stride[0] >= (int64_t)d.head_dim);
}

AttnArgs base_args(const katsu_attention &d, const int32_t *cu_q, const int32_t *cu_k,
                   const int32_t *k_lens) {
    AttnArgs a{};
    a.cu_q = cu_q;
    a.cu_k = cu_k;
    a.k_lens = k_lens;
    a.Tq = (int64_t)d.tokens_q;
    a.Tk = (int64_t)d.tokens_k;
    a.B = (int)d.seqs;
    a.H = (int)d.heads;
    a.Hkv = (int)d.kv_heads;
    a.G = a.H / a.Hkv;
    a.D = (int)d.head_dim;
    a.causal = d.causal;
    a.scale = d.scale;
    a.scale2 = d.scale * kLog2e;
    a.splits = 1;
    return a;
}

AttnTensor tensor(const void *p, const int64_t (&stride)[2]) {
    return {p, stride[0], stride[1]};
}

// Channels of a row in LDS and in the parts.
int width_of(const katsu_attention &d) { return d.head_dim <= 64 ? 64 : 128; }

// Runs that an axis of `len` is split into: `want` blocks in all, a run at least `least` long.
int runs(int64_t want, int64_t blocks, int64_t len, int64_t least) {
    return (int)std::max<int64_t>(
        1, std::min(want / std::max<int64_t>(blocks, 1), cdiv(len, least)));
}

// The forward call's shape: tiles of 32 rows whose waves share the keys, or of 128.  Of 32 where
// a sequence has no more rows than that in the mean (32 single tokens over 1500-7650 keys, 32/8
// heads of 128, bfloat16: 130 us, 161 in tiles of 128; 8 tokens of these over 2000 keys: 53 and
// 63); beyond, a second tile reads the keys again (16 tokens: 69 and 66; 300 sequences of 40
// over themselves, 8/4 heads of 64: 45 and 18; 31 single tokens and one prompt of 2000: 154 and
// 103; only float32 still gains, 16 tokens over 2000 keys, 16/4 heads of 64: 90 and 142).
struct FwdPlan {
    bool few;
    int bm, slots, splits;
};
FwdPlan fwd_plan(const katsu_attention &d) {
    FwdPlan p;
    const int64_t group = (int64_t)(d.heads / d.kv_heads);
    const int64_t rows = (int64_t)d.tokens_q * group, B = (int64_t)d.seqs;
    p.few = rows <= 32 * B;
    p.bm = p.few ? 32 : 128;
    p.slots = (int)(rows / p.bm + B);
    const int64_t blocks = (int64_t)p.slots * (int64_t)d.kv_heads;
    // A block a CU; a run's keys have to be worth the launch that joins the runs: single
    // tokens 256 of them (32000 keys, 32/8 heads of 128: 34 us in 32 runs, 45 in 64; 4000: 15 in
    // 16, 19 in 4), tiles of 128 rows 1024 in bfloat16 (1000 tokens, 16/4 heads of 128: 25 us in
    // one run, 32 in four) and two tiles, 3.4 us each, in float32.
    const int64_t keys = cdiv((int64_t)d.tokens_k, B);
    if (d.dtype == KATSU_F32 && !p.few)
        p.splits = runs(2 * kCUs, blocks, keys, d.head_dim > 64 ? 64 : 128);
    else
        p.splits = runs(kCUs, blocks, keys, p.few ? 256 : 1024);
    return p;
}
size_t part_floats(const katsu_attention &d, const FwdPlan &p) {
    if (p.splits <= 1) return 0;
    return (size_t)p.splits * d.tokens_q * d.heads * (size_t)(width_of(d) + 2);
}

// Calls f with the operand type, the blocks of 32 channels and whether rows are whole
// 16-byte chunks, as constants (rows that are not take the next of 64 or 128 channels).
template <class F>
int by_shape(const katsu_attention &d, bool vec, F f) {
    const int nd = (int)cdiv((int64_t)d.head_dim, 32);
    auto with = [&](auto t) {
        auto with_nd = [&](auto n) {
            constexpr int ND = decltype(n)::value;
            if constexpr (ND % 2 == 0)
                if (!vec) return f(t, n, std::false_type());
            return f(t, n, std::true_type());
        };
        const int m = vec ? nd : (nd + 1) / 2 * 2;
        if (m == 1) return with_nd(std::integral_constant<int, 1>());
        if (m == 2) return with_nd(std::integral_constant<int, 2>());
        if (m == 3) return with_nd(std::integral_constant<int, 3>());
        return with_nd(std::integral_constant<int, 4>());
    };
    return d.dtype == KATSU_F32 ? with(float()) : with(__bf16());
}

template <auto Kern>
int launch(int64_t blocks, int threads, int lds, const AttnArgs &a, hipStream_t st) {
    const int rc = lds_optin<Kern>(lds);
    if (rc != KATSU_OK || blocks == 0) return rc;
    // A launch has fewer than 2^32 threads along x: blocks beyond that go along y.
    const int64_t x = std::min<int64_t>(blocks, 1 << 20);
    Kern<<<dim3((unsigned)x, (unsigned)cdiv(blocks, x)), dim3(threads), lds, st>>>(a);
    return status_of(hipGetLastError());
}

// The order of a causal call's tiles: by work where blocks wait for others to end, in pairs
// where all are on the card at once, two a CU (4096 tokens, 16/16 heads of 64, float32: 381 us
// in order of place, 295 in pairs).  Otherwise, or where the other axis is split and all
// blocks are short, finding a tile by its place costs less.
int tile_order(const AttnArgs &a, int64_t blocks, int runs) {
    const int64_t used = blocks - (int64_t)a.B * a.Hkv * runs;  // at most a tile a sequence more
    if (!a.causal || used <= kCUs) return kByPlace;
    return used > 2 * kCUs ? kByWork : runs > 1 ? kByPlace : kInPairs;
}

template <typename T, int ND, int WM, int WK, int BN, bool VEC, int OCC>
int launch_fwd(AttnArgs a, hipStream_t st) {
    using K = AttnFwd<T, ND, WM, WK, BN, VEC>;
    static_assert(K::kLds <= 160 * 1024, "LDS");
    const int64_t blocks = (int64_t)a.slots * a.Hkv * a.splits;
    a.order = tile_order(a, blocks, a.splits);
    return launch<attention_fwd_kernel<T, ND, WM, WK, BN, VEC, OCC>>(blocks, K::THREADS, K::kLds, a,
                                                                     st);
}
template <typename T, int ND, bool VEC>
int launch_fwd(const AttnArgs &a, bool few, hipStream_t st) {
    // float32 rows of 128 channels: half the keys a tile, so that two blocks share a CU;
    // with few rows two waves instead of four.
    constexpr bool wide = Rows<T, ND>::RB == 512;
    if (few) return launch_fwd<T, ND, 1, wide ? 2 : 4, 32, VEC, 1>(a, st);
    return launch_fwd<T, ND, 4, 1, wide ? 32 : 64, VEC, 2>(a, st);
}

// The backward call's shape.  dk and dv: blocks of one query head each, unless the key heads
// alone give the card enough to do; in float32 always, and in runs of 2048 queries (up to
// four runs, whose sums are memory), as a long sum in one accumulator loses more (5110
// tokens, 8/4 heads of 16: dk 9.8e-7 off in three runs, 1.7e-6 in one, and 567 us against 717;
// 4096, 16/16 heads of 64, all keys: 1.2e-6 in two, 1.4e-6 in one, and 1749 us against 1733).
// That goes by the mean length, as the lengths are on the card: a sequence of 6000 among five
// short ones is one run (8/8 heads of 64: 1.6e-6; plain float32 products 1.5e-6).  Both kernels:
// the other axis in runs where there are few blocks.
struct BwdPlan {
    int dq_slots, dq_splits, dkv_slots, dkv_splits, parts;
    bool each;
};
BwdPlan bwd_plan(const katsu_attention &d) {
    BwdPlan p;
    const int64_t kv = (int64_t)d.kv_heads, group = (int64_t)d.heads / kv, B = (int64_t)d.seqs;
    p.dq_slots = (int)((int64_t)d.tokens_q * group / 128 + B);
    p.dkv_slots = (int)((int64_t)d.tokens_k / 128 + B);
    p.each = group > 1 && (d.dtype == KATSU_F32 || p.dkv_slots * kv < 4 * kCUs);
    // Keys of a run of dq, queries of one of dk and dv: two tiles in float32, 256 in bfloat16
    // (1500 tokens, 8/8 heads of 64: 48 us; 51 with 512; 54 with one block a CU).
    const int64_t least = d.dtype == KATSU_F32 ? d.head_dim > 64 ? 64 : 128 : 256;
    p.dq_splits = runs(2 * kCUs, p.dq_slots * kv, cdiv((int64_t)d.tokens_k, B), least);
    p.dkv_splits = runs(2 * kCUs, p.dkv_slots * kv * (p.each ? group : 1),
                        cdiv((int64_t)d.tokens_q, B) * (p.each ? 1 : group), least);
    if (d.dtype == KATSU_F32)
        p.dkv_splits = std::max<int>(
            p.dkv_splits, (int)std::min<int64_t>(cdiv((int64_t)d.tokens_q, B * 2048), 4));
    p.parts = (p.each ? (int)group : 1) * p.dkv_splits;
    return p;
}
size_t start_floats(const katsu_attention &d) {
    return (2 * d.tokens_q * d.heads + 63) / 64 * 64;
}

template <typename T, int ND, bool VEC>
int launch_bwd(AttnArgs a, const BwdPlan &p, hipStream_t st) {
    // Rows of 512 bytes: tiles of half the rows, one wave a SIMD for dk and dv.
    constexpr int RB = Rows<T, ND>::RB;
    constexpr int BN = RB == 512 ? 32 : 64, QT = ND > 2 ? 32 : 64;
    using Dq = AttnDq<T, ND, BN, VEC>;
    using Dkv = AttnDkv<T, ND, QT, VEC>;
    a.slots = p.dq_slots;
    a.splits = p.dq_splits;
    const int64_t dq_blocks = a.Tq > 0 ? (int64_t)p.dq_slots * a.Hkv * a.splits : 0;
    a.order = tile_order(a, dq_blocks, a.splits);
    int rc = launch<attention_dq_kernel<T, ND, BN, VEC, 2>>(dq_blocks, Dq::THREADS, Dq::kLds, a,
                                                            st);
    if (rc != KATSU_OK) return rc;
    // Sums of parts: dq's are [run][token][head], dk's and dv's [key head][part][token].
    AttnSum s{};
    s.D = a.D;
    s.W = Dkv::W;
    auto sum = [&](int outs) {
        const int64_t blocks = cdiv(s.tokens * s.heads * (s.W / 4), 256);
        attention_sum_kernel<T, VEC><<<dim3((unsigned)blocks, outs), 256, 0, st>>>(s);
        return status_of(hipGetLastError());
    };
    if (a.splits > 1 && a.Tq > 0) {
        s.out[0] = a.dq;
        s.part[0] = a.part;
        s.tokens = a.Tq;
        s.heads = a.H;
        s.parts = a.splits;
        s.head_step = s.W;
        s.token_step = (int64_t)a.H * s.W;
        s.part_step = a.Tq * s.token_step;
        rc = sum(1);
        if (rc != KATSU_OK) return rc;
    }
    if (a.Tk == 0) return KATSU_OK;
    a.slots = p.dkv_slots;
    a.splits = p.dkv_splits;
    a.parts = p.parts;
    a.each = p.each;
    const int64_t dkv_blocks = (int64_t)p.dkv_slots * a.Hkv * p.parts;
    a.order = tile_order(a, dkv_blocks, a.parts);
    if (RB == 512 && a.order == kInPairs) a.order = kByWork;  // one block a CU
    rc = launch<attention_dkv_kernel<T, ND, QT, VEC, RB == 512 ? 1 : 2>>(dkv_blocks, Dkv::THREADS,
                                                                         Dkv::kLds, a, st);
    if (rc != KATSU_OK || p.parts == 1) return rc;
    s.out[0] = a.dk;
    s.out[1] = a.dv;
    s.tokens = a.Tk;
    s.heads = a.Hkv;
    s.parts = p.parts;
    s.token_step = s.W;
    s.part_step = a.Tk * s.W;
    s.head_step = s.parts * s.part_step;
    s.part[0] = a.part;
    s.part[1] = a.part + a.Hkv * s.head_step;
    return sum(2);
}

}  // namespace

// An output's places are its own: no broadcast strides.
bool attention_out_ok(const int64_t (&s)[2], uint64_t tokens, uint64_t heads) {
    return strides_ok(s) && (tokens < 2 || s[0] > 0) && (heads < 2 || s[1] > 0);
}
bool attention_grads_ok(const katsu_attention &d, const katsu_attention_grads &g) {
    return strides_ok(g.dout_stride) && attention_out_ok(g.dq_stride, d.tokens_q, d.heads) &&
           attention_out_ok(g.dk_stride, d.tokens_k, d.kv_heads) &&
           attention_out_ok(g.dv_stride, d.tokens_k, d.kv_heads);
}

bool attention_ok(const katsu_attention &d) {
    if (d.dtype != KATSU_F32 && d.dtype != KATSU_BF16) return false;
    if (d.heads == 0 || d.kv_heads == 0 || d.heads % d.kv_heads != 0 || d.heads > 65535)
        return false;
    if (d.head_dim == 0 || d.head_dim > 128) return false;
    if (!(d.scale > 0.f) || !std::isfinite(d.scale)) return false;
    // Tokens are counted in 32 bits, a tile beyond the last included.
    const uint64_t most = (uint64_t)kI32Max - 65535;
    if (d.tokens_q > most || d.tokens_k > most || d.seqs > most) return false;
    if (!strides_ok(d.q_stride) || !strides_ok(d.k_stride) || !strides_ok(d.v_stride) ||
        !strides_ok(d.out_stride))
        return false;
    // Tiles and blocks are counted in 32 bits.
    const uint64_t group = d.heads / d.kv_heads;
    const uint64_t rows = std::max(d.tokens_q * group, d.tokens_k * group);
    return (rows / 32 + d.seqs * group) * d.kv_heads < (uint64_t)kI32Max / 4 &&
           std::max(d.tokens_q, d.tokens_k) * d.heads < (uint64_t)kI32Max * 4;
}

size_t attention_fwd_bytes(const katsu_attention &d) {
    if (d.tokens_q == 0 || d.seqs == 0) return 0;
    return part_floats(d, fwd_plan(d)) * sizeof(float);
}

int attention_fwd(const katsu_attention &d, const void *q, const void *k, const void *v,
                  const int32_t *cu_q, const int32_t *cu_k, const int32_t *k_lens, void *out,
                  float *lse, void *ws, hipStream_t st) {
    const FwdPlan p = fwd_plan(d);
    AttnArgs a = base_args(d, cu_q, cu_k, k_lens);
    a.q = tensor(q, d.q_stride);
    a.k = tensor(k, d.k_stride);
    a.v = tensor(v, d.v_stride);
    a.out = tensor(out, d.out_stride);
    a.lse = lse;
    a.slots = p.slots;
    a.splits = p.splits;
    const int width = width_of(d);
    a.part = (float *)ws;
    a.part_ml = a.part + (size_t)a.splits * d.tokens_q * d.heads * width;
    const bool vec = vec_ok(d, q, d.q_stride) && vec_ok(d, k, d.k_stride) &&
                     vec_ok(d, v, d.v_stride) && vec_ok(d, out, d.out_stride);
    const int rc = by_shape(d, vec, [&](auto t, auto nd, auto v) {
        return launch_fwd<decltype(t), decltype(nd)::value, decltype(v)::value>(a, p.few, st);
    });
    if (rc != KATSU_OK || a.splits == 1) return rc;
    // A wave a row, a block where there are parts enough for its waves.
    const int64_t rows = a.Tq * a.H;
    const bool many = a.splits >= 8;
    auto join = [&](auto t) {
        using T = decltype(t);
        if (many)
            attention_join_kernel<T, 4><<<dim3((unsigned)rows), 256, 0, st>>>(a, width);
        else
            attention_join_kernel<T, 1><<<dim3((unsigned)cdiv(rows, 4)), 256, 0, st>>>(a, width);
        return status_of(hipGetLastError());
    };
    return d.dtype == KATSU_F32 ? join(float()) : join(__bf16());
}

size_t attention_bwd_bytes(const katsu_attention &d) {
    if (d.seqs == 0) return 0;
    // The parts of dq and those of dk and dv take turns.
    const BwdPlan p = bwd_plan(d);
    const size_t dq = p.dq_splits > 1 ? p.dq_splits * d.tokens_q * d.heads : 0;
    const size_t dkv = p.parts > 1 ? 2 * (size_t)p.parts * d.kv_heads * d.tokens_k : 0;
    return (start_floats(d) + std::max(dq, dkv) * width_of(d)) * sizeof(float);
}

int attention_bwd(const katsu_attention &d, const katsu_attention_grads &g, const void *dout,
                  const void *q, const void *k, const void *v, const void *out, const float *lse,
                  const int32_t *cu_q, const int32_t *cu_k, void *dq, void *dk, void *dv, void *ws,
                  hipStream_t st) {
    const BwdPlan p = bwd_plan(d);
    AttnArgs a = base_args(d, cu_q, cu_k, nullptr);
    bool vec = true;
    auto take = [&](AttnTensor &t, const void *ptr, const int64_t (&stride)[2]) {
        t = tensor(ptr, stride);
        vec = vec && vec_ok(d, ptr, stride);
    };
    take(a.q, q, d.q_stride);
    take(a.k, k, d.k_stride);
    take(a.v, v, d.v_stride);
    take(a.out, out, d.out_stride);
    take(a.dout, dout, g.dout_stride);
    take(a.dq, dq, g.dq_stride);
    take(a.dk, dk, g.dk_stride);
    take(a.dv, dv, g.dv_stride);
    a.lse = const_cast<float *>(lse);
    a.start = (float *)ws;
    a.part = a.start + start_floats(d);
    return by_shape(d, vec, [&](auto t, auto nd, auto v) {
        return launch_bwd<decltype(t), decltype(nd)::value, decltype(v)::value>(a, p, st);
    });
}

}  // namespace katsu
