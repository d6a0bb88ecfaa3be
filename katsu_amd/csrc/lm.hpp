// lm.hpp -- what the C ABI (katsu_hip.hip) calls of the language-model operators,
// which are compiled apart from it (attention.hip, lmblock.hip).  Each returns a katsu_status;
// argument checks are done here too, before any launch.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "../../include/katsu_hip.h"

namespace katsu {

// Whether d describes a problem these kernels take.
bool attention_ok(const katsu_attention &d);
// Scratch bytes of a forward call, of a backward one.
size_t attention_fwd_bytes(const katsu_attention &d);
int attention_fwd(const katsu_attention &d, const void *q, const void *k, const void *v,
                  const int32_t *cu_q, const int32_t *cu_k, const int32_t *k_lens, void *out,
                  float *lse, void *ws, hipStream_t st);

// Whether a tensor of these strides can be written; whether the gradients can.
bool attention_out_ok(const int64_t (&stride)[2], uint64_t tokens, uint64_t heads);
bool attention_grads_ok(const katsu_attention &d, const katsu_attention_grads &g);
size_t attention_bwd_bytes(const katsu_attention &d);
int attention_bwd(const katsu_attention &d, const katsu_attention_grads &g, const void *dout,
                  const void *q, const void *k, const void *v, const void *out, const float *lse,
                  const int32_t *cu_q, const int32_t *cu_k, void *dq, void *dk, void *dv, void *ws,
                  hipStream_t st);

bool rotary_ok(const katsu_rotary &d);
int rotary(const katsu_rotary &d, const void *q, const void *k, const float *table,
           const int32_t *positions, void *q_out, void *k_out, hipStream_t st);
int rotary_table(float *table, int64_t length, int dim, double base, double factor,
                 int by_wavelength, hipStream_t st);

bool block_norm_ok(const katsu_block_norm &d);
int block_norm(const katsu_block_norm &d, const void *x, const void *o, const void *gate,
               const void *w_post, const void *w_pre, void *y, void *h, float *stats,
               hipStream_t st);
size_t block_norm_bwd_bytes(const katsu_block_norm &d);
int block_norm_bwd(const katsu_block_norm &d, const void *dy, const void *dh, const void *y,
                   const void *o, const float *stats, const void *gate, const void *w_post,
                   const void *w_pre, void *dx, void *d_o, void *dgate, void *dw_post,
                   void *dw_pre, void *ws, hipStream_t st);

// Scratch bytes for n tensors.
size_t clip_bytes(size_t n);
int clip_grad_norm(const int32_t *dtypes, const void *const *in, void *const *out,
                   const size_t *counts, size_t n, float max_norm, float *norm, void *ws,
                   hipStream_t st);

}  // namespace katsu
