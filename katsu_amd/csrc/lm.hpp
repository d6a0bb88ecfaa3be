// lm.hpp -- what the C ABI (katsu_hip.hip) calls of the language-model operators,
// which are compiled apart from it (attention.hip, lmblock.hip, lmends.hip).  Each returns a katsu_status;
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

// Whether a tensor of these strides can be written: no two of its heads share memory, and where it
// is the input (`same`), each is in its place.
bool rotary_out_ok(const int64_t (&in)[2], const int64_t (&out)[2], bool same, uint64_t tokens,
                   uint64_t heads, uint64_t dim);
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

bool embedding_ok(const katsu_embedding &d);
// Whether rows of these columns can be written with this stride.
bool embedding_out_ok(uint64_t rows, uint64_t cols, int64_t stride);
// Whether any of n_a rows of a and n_b rows of b share memory.
bool rows_share(const void *a, uint64_t n_a, int64_t stride_a, uint64_t cols_a, const void *b,
                uint64_t n_b, int64_t stride_b, uint64_t cols_b, int dtype);
int embedding(const katsu_embedding &d, const int32_t *ids, const void *table, void *out,
              hipStream_t st);
size_t embedding_bwd_bytes(const katsu_embedding &d);
int embedding_bwd(const katsu_embedding &d, const void *dout, const int32_t *ids, void *dtable,
                  void *ws, hipStream_t st);

// Whether heads of a and heads of b share memory: begin at one place, or, where heads or tokens lie
// side by side in both, share any.
bool heads_share(const katsu_qk_norm_rotary &d, const void *a, uint64_t heads_a,
                 const int64_t (&stride_a)[2], const void *b, uint64_t heads_b,
                 const int64_t (&stride_b)[2]);
bool qk_norm_rotary_ok(const katsu_qk_norm_rotary &d);
int qk_norm_rotary(const katsu_qk_norm_rotary &d, const void *q, const void *k, const void *w_q,
                   const void *w_k, const float *table, const int32_t *positions, void *q_out,
                   void *k_out, hipStream_t st);
size_t qk_norm_rotary_bwd_bytes(const katsu_qk_norm_rotary &d);
int qk_norm_rotary_bwd(const katsu_qk_norm_rotary &d, const katsu_qk_norm_rotary_grads &g,
                       const void *dq, const void *dk, const void *q, const void *k,
                       const void *w_q, const void *w_k, const float *table,
                       const int32_t *positions, void *dq_out, void *dk_out, void *dw_q,
                       void *dw_k, void *ws, hipStream_t st);

bool distillation_ok(const katsu_distillation &d);
int distillation(const katsu_distillation &d, const void *logits, const int32_t *ids,
                 const void *teacher, float *loss, float *stats, hipStream_t st);
int distillation_bwd(const katsu_distillation &d, const float *dloss, const void *logits,
                     const int32_t *ids, const void *teacher, const float *stats, void *dlogits,
                     hipStream_t st);
int distillation_step(const katsu_distillation &d, const void *logits, const int32_t *ids,
                      const void *teacher, const float *dloss, float *loss, void *dlogits,
                      hipStream_t st);

}  // namespace katsu
