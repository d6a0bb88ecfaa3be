// lm.hpp -- what the C ABI (katsu_hip.hip) calls of the language-model operators,
// which are compiled apart from it (attention.hip).  Each returns a katsu_status;
// argument checks are done here too, before any launch.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>

#include "../../include/katsu_hip.h"

namespace katsu {

// Whether d describes a problem these kernels take.
bool attention_ok(const katsu_attention &d);
// Scratch bytes of a forward call, of a backward one.
size_t attention_fwd_bytes(const katsu_attention &d);
int attention_fwd(const katsu_attention &d, const void *q, const void *k, const void *v,
                  const int32_t *cu_q, const int32_t *cu_k, const int32_t *k_lens, void *out,
                  float *lse, void *ws, hipStream_t st);


bool attention_grads_ok(const katsu_attention_grads &g);
size_t attention_bwd_bytes(const katsu_attention &d);
int attention_bwd(const katsu_attention &d, const katsu_attention_grads &g, const void *dout,
                  const void *q, const void *k, const void *v, const void *out, const float *lse,
                  const int32_t *cu_q, const int32_t *cu_k, void *dq, void *dk, void *dv, void *ws,
                  hipStream_t st);

}  // namespace katsu
