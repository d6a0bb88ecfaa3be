// attention.hip -- launches of the attention kernels: which variant, how many
// blocks, how many parts of the key axis.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

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

bool strides_ok(const int64_t (&s)[2]) {
    return s[0] >= 0 && s[1] >= 0 && s[0] <= kI32Max && s[1] <= (int64_t)1 << 40;
}

int elem(const katsu_attention &d) { return d.dtype == KATSU_F32 ? 4 : 2; }

// 16-byte accesses: rows of whole 16-byte chunks at aligned places, and a tile's
// 128 rows within the 32-bit offsets of a buffer load.
bool vec_ok(const katsu_attention &d, const void *p, const int64_t (&stride)[2]) {
    const int e = elem(d);
    return ((uintptr_t)p & 15) == 0 && d.head_dim * e % 16 == 0 && stride[0] * e % 16 == 0 &&
           stride[1] * e % 16 == 0 && stride[0] * e < (1 << 23);
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

int dp_of(const katsu_attention &d) { return d.head_dim <= 64 ? 64 : 128; }

// The forward call's shape: tiles of 32 rows whose waves share the keys, or of 128.
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
    const int64_t keys = cdiv((int64_t)d.tokens_k, B);
    p.splits = (int)std::max<int64_t>(1, std::min(2 * kCUs / std::max<int64_t>(blocks, 1),
                                                  cdiv(keys, 256)));
    return p;
}
size_t part_floats(const katsu_attention &d, const FwdPlan &p) {
    if (p.splits <= 1) return 0;
    return (size_t)p.splits * d.tokens_q * d.heads * (size_t)(dp_of(d) + 2);
}

template <typename T, int DP, int WM, int WK, int BN, bool VEC, int OCC>
int launch_fwd(const AttnArgs &a, hipStream_t st) {
    using K = AttnFwd<T, DP, WM, WK, BN, VEC>;
    constexpr auto kern = attention_fwd_kernel<T, DP, WM, WK, BN, VEC, OCC>;
    static_assert(K::kLds <= 160 * 1024, "LDS");
    const int rc = lds_optin<kern>(K::kLds);
    if (rc != KATSU_OK) return rc;
    const int64_t blocks = (int64_t)a.slots * a.Hkv * a.splits;
    kern<<<dim3((unsigned)blocks), dim3(K::THREADS), K::kLds, st>>>(a);
    return status_of(hipGetLastError());
}
template <typename T, int DP, bool VEC>
int launch_fwd(const AttnArgs &a, bool few, hipStream_t st) {
    // float32 rows of 128 channels: half the keys a tile, so that two blocks share a CU;
    // with few rows two waves instead of four.
    constexpr bool wide = DP * sizeof(T) == 512;
    if (few) return launch_fwd<T, DP, 1, wide ? 2 : 4, 32, VEC, 1>(a, st);
    return launch_fwd<T, DP, 4, 1, wide ? 32 : 64, VEC, 2>(a, st);
}
template <typename T>
int launch_fwd(const AttnArgs &a, int dp, bool vec, bool few, hipStream_t st) {
    if (dp == 64)
        return vec ? launch_fwd<T, 64, true>(a, few, st) : launch_fwd<T, 64, false>(a, few, st);
    return vec ? launch_fwd<T, 128, true>(a, few, st) : launch_fwd<T, 128, false>(a, few, st);
}

// The backward call's shape.  Blocks of one query head each, and their sums joined
// afterwards, unless the key heads alone give the card enough to do.
struct BwdPlan {
    int dq_slots, dkv_slots;
    bool each;
};
BwdPlan bwd_plan(const katsu_attention &d) {
    BwdPlan p;
    const int64_t group = (int64_t)(d.heads / d.kv_heads), B = (int64_t)d.seqs;
    p.dq_slots = (int)((int64_t)d.tokens_q * group / 128 + B);
    p.dkv_slots = (int)((int64_t)d.tokens_k / 128 + B);
    p.each = group > 1 && (int64_t)p.dkv_slots * (int64_t)d.kv_heads < 4 * kCUs;
    return p;
}
size_t stat_floats(const katsu_attention &d) {
    return (2 * d.tokens_q * d.heads + 63) / 64 * 64;
}

template <auto Kern>
int launch(int64_t blocks, int lds, const AttnArgs &a, hipStream_t st) {
    const int rc = lds_optin<Kern>(lds);
    if (rc != KATSU_OK || blocks == 0) return rc;
    Kern<<<dim3((unsigned)blocks), dim3(256), lds, st>>>(a);
    return status_of(hipGetLastError());
}
template <typename T, int DP, bool VEC>
int launch_bwd(AttnArgs a, const BwdPlan &p, hipStream_t st) {
    // float32 rows of 128 channels: tiles of half the rows, one wave a SIMD for dk and dv.
    constexpr bool wide = DP * sizeof(T) == 512;
    constexpr int BN = wide ? 32 : 64, QT = wide ? 32 : 64;
    a.slots = p.dq_slots;
    const int64_t dq_blocks = a.Tq > 0 ? (int64_t)p.dq_slots * a.Hkv : 0;
    int rc = launch<attention_dq_kernel<T, DP, BN, VEC, 2>>(dq_blocks, AttnDq<T, DP, BN, VEC>::kLds,
                                                            a, st);
    if (rc != KATSU_OK || a.Tk == 0) return rc;
    a.slots = p.dkv_slots;
    rc = launch<attention_dkv_kernel<T, DP, QT, VEC, wide ? 1 : 2>>(
        (int64_t)p.dkv_slots * (p.each ? a.H : a.Hkv), AttnDkv<T, DP, QT, VEC>::kLds, a, st);
    if (rc != KATSU_OK || !p.each) return rc;
    const int64_t blocks = cdiv(a.Tk * a.Hkv * (DP / 4), 256);
    attention_group_kernel<T, VEC><<<dim3((unsigned)blocks, 2), 256, 0, st>>>(a, DP);
    return status_of(hipGetLastError());
}
template <typename T>
int launch_bwd(const AttnArgs &a, const BwdPlan &p, int dp, bool vec, hipStream_t st) {
    if (dp == 64)
        return vec ? launch_bwd<T, 64, true>(a, p, st) : launch_bwd<T, 64, false>(a, p, st);
    return vec ? launch_bwd<T, 128, true>(a, p, st) : launch_bwd<T, 128, false>(a, p, st);
}

}  // namespace

bool attention_grads_ok(const katsu_attention_grads &g) {
    return strides_ok(g.dout_stride) && strides_ok(g.dq_stride) && strides_ok(g.dk_stride) &&
           strides_ok(g.dv_stride);
}

bool attention_ok(const katsu_attention &d) {
    if (d.dtype != KATSU_F32 && d.dtype != KATSU_BF16) return false;
    if (d.heads == 0 || d.kv_heads == 0 || d.heads % d.kv_heads != 0 || d.heads > 65535)
        return false;
    if (d.head_dim == 0 || d.head_dim > 128) return false;
    if (!(d.scale > 0.f) || !std::isfinite(d.scale)) return false;
    if (d.tokens_q > (uint64_t)kI32Max || d.tokens_k > (uint64_t)kI32Max ||
        d.seqs > (uint64_t)kI32Max)
        return false;
    if (!strides_ok(d.q_stride) || !strides_ok(d.k_stride) || !strides_ok(d.v_stride) ||
        !strides_ok(d.out_stride))
        return false;
    // Tiles and blocks are counted in 32 bits.
    const uint64_t group = d.heads / d.kv_heads;
    const uint64_t rows = std::max(d.tokens_q * group, d.tokens_k * group);
    return (rows / 32 + d.seqs) * d.kv_heads < (uint64_t)kI32Max / 4 &&
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
    const int dp = dp_of(d);
    a.part = (float *)ws;
    a.part_ml = a.part + (size_t)a.splits * d.tokens_q * d.heads * dp;
    const bool vec = vec_ok(d, q, d.q_stride) && vec_ok(d, k, d.k_stride) &&
                     vec_ok(d, v, d.v_stride) && vec_ok(d, out, d.out_stride);
    const int rc = d.dtype == KATSU_F32 ? launch_fwd<float>(a, dp, vec, p.few, st)
                                        : launch_fwd<__bf16>(a, dp, vec, p.few, st);
    if (rc != KATSU_OK || a.splits == 1) return rc;
    const unsigned blocks = (unsigned)cdiv(a.Tq * a.H, 4);
    if (d.dtype == KATSU_F32)
        attention_join_kernel<float><<<blocks, 256, 0, st>>>(a, dp);
    else
        attention_join_kernel<__bf16><<<blocks, 256, 0, st>>>(a, dp);
    return status_of(hipGetLastError());
}

size_t attention_bwd_bytes(const katsu_attention &d) {
    if (d.seqs == 0) return 0;
    const size_t part = bwd_plan(d).each ? 2 * d.heads * d.tokens_k * (size_t)dp_of(d) : 0;
    return (stat_floats(d) + part) * sizeof(float);
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
    a.lse2 = (float *)ws;
    a.delta = a.lse2 + d.tokens_q * d.heads;
    if (p.each) a.part = a.lse2 + stat_floats(d);
    const int dp = dp_of(d);
    return d.dtype == KATSU_F32 ? launch_bwd<float>(a, p, dp, vec, st)
                                : launch_bwd<__bf16>(a, p, dp, vec, st);
}

}  // namespace katsu
