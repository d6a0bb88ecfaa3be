/*
 * katsu_hip.h -- C ABI of the MI355X (gfx950) dense-contraction path.
 *
 * This library replaces the four crate-internal kernel seams of Katsu's
 * katsu-core (paths relative to the reference repository root):
 *
 *   S1  matmul forward     crates/katsu-core/src/tensor.rs:264-273
 *   S2  matmul VJPs        crates/katsu-core/src/tensor.rs:424-444
 *   S3  conv forward       crates/katsu-core/src/conv2d.rs:98-103
 *   S4  conv backward      crates/katsu-core/src/conv2d.rs:284-290
 *                          (reached from conv2d.rs:127 and tensor.rs:375)
 *
 * Layouts are the reference's: row-major matrices, NCHW activations, OIHW
 * weights, all contiguous f32.  Every entry point returns a katsu_status;
 * nothing aborts or throws across the ABI.
 *
 * Two families of entry points:
 *   - host-pointer ("drop-in") entry points take the caller's host buffers,
 *     as the reference's slices are, copy them to the device, run on the
 *     library's stream and return once the outputs are written back.  Copies
 *     of 1 MiB or more go through a ring of four pinned 8 MiB host chunks
 *     (allocated on first use, freed by katsu_hip_shutdown), the CPU side of
 *     each chunk split over four threads (environment: KATSU_COPY_THREADS,
 *     KATSU_COPY_CHUNK_MB); the caller's buffers stay pageable;
 *   - *_dev entry points take device pointers and a hipStream_t (passed as
 *     void*, 0 = the null stream) and return right after the launch.
 *
 * Threading: the reference engine is single-threaded (Rc handles,
 * tensor.rs:95-99).  The library's host-side state is guarded by mutexes, so
 * it is safe to call from several threads; the host-pointer entry points
 * share one stream and one staging pool.
 *
 * Library scratch: the *_dev entry points that need device scratch (the dW
 * split partials when no workspace is passed, the GEMM's split-K partials,
 * the sum's chunk partials, Grad-CAM's channel weights, the language-model
 * operators' partials) take it from one
 * buffer per purpose that the library keeps and shares across all streams
 * and graphs: an eager call sizes it, and a later capture of the same call
 * on any stream uses it without allocating.  Calls (or graph replays) that
 * overlap in time on different streams race on it; callers that run such
 * calls concurrently order them, or pass their own workspace where the
 * entry point takes one.  A buffer that must grow is replaced and the old
 * block is kept (not freed) until katsu_hip_shutdown, so a graph captured
 * earlier keeps valid addresses.
 *
 * Size limits: empty problems (an output with no elements, or an empty
 * reduction) return KATSU_OK whatever their other dimensions.  Otherwise the
 * kernels index in 32 bits and these entry points return KATSU_E_INVALID
 * (launching nothing) when a bound is exceeded:
 *   matmul:       m, n, k <= 2^31 - 1;
 *   convolutions: C*H*W, K*OH*OW, K*C*R*S, N*H*W, N*OH*OW, pad, stride,
 *                 H + 2*pad and W + 2*pad <= 2^31 - 1.
 */
#ifndef KATSU_HIP_H
#define KATSU_HIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef enum katsu_status {
    KATSU_OK = 0,
    KATSU_E_INVALID = 1,  /* bad argument or shape; nothing was launched */
    KATSU_E_NODEVICE = 2, /* no HIP device, or device/runtime init failed */
    KATSU_E_OOM = 3,      /* device allocation failed */
    KATSU_E_LAUNCH = 4,   /* kernel launch, copy or synchronisation failed */
    KATSU_E_SCRATCH = 5,  /* more scratch than the allocation-free entry point holds */
} katsu_status;

/* Convolution geometry, the fields of the reference's `struct Geometry`
 * (conv2d.rs:168-180).  n: batch, c: in channels, h/w: input size,
 * k: out channels, r/s: kernel height/width, stride/pad: equal on both axes
 * (conv2d.rs:11-12), oh/ow: output size.  Callers fill n..pad and either
 * fill oh/ow or call katsu_hip_conv2d_geometry. */
typedef struct katsu_conv_geom {
    uint64_t n, c, h, w, k, r, s, stride, pad, oh, ow;
} katsu_conv_geom;

/* Version string of this library. */
const char *katsu_hip_version(void);

/* Human-readable text for a katsu_status. */
const char *katsu_hip_strerror(int status);

/* Selects the first HIP device and creates the library stream.  Called
 * implicitly by every entry point that needs the device; idempotent. */
int katsu_hip_init(void);

/* Frees the staging pool and workspace and destroys the stream. */
void katsu_hip_shutdown(void);

/* Completes *g: checks it the way Geometry::new does (conv2d.rs:183-224:
 * positive OIHW dims and stride, positive H and W, kernel within the padded
 * input, no size overflow) and writes oh = (h + 2*pad - r)/stride + 1 and
 * ow likewise.  Batch 0 is accepted.  Returns KATSU_E_INVALID otherwise. */
int katsu_hip_conv2d_geometry(katsu_conv_geom *g);

/* ---- S1/S2: matmul ------------------------------------------------------
 * C[m,n] = beta*C + op(A)[m,k] . op(B)[k,n], beta in {0, 1}.
 *   op(A) = A   (A stored [m,k]) when trans_a == 0,
 *           A^T (A stored [k,m]) when trans_a == 1; likewise B.
 * Tensor::matmul (tensor.rs:264-273) is trans_a=0, trans_b=0, beta=0.
 * The Matmul VJP (tensor.rs:424-444) is dA += G.B^T (trans_b=1, beta=1)
 * followed by dB += A^T.G (trans_a=1, beta=1), in that order, because the
 * two pending buffers are the same buffer when A and B are the same node.
 * With beta == 0, C is not read.  k == 0 writes beta*C (tensor.rs:265,421).
 */
int katsu_hip_gemm_f32(const float *a, const float *b, float *c, size_t m, size_t n,
                       size_t k, int trans_a, int trans_b, float beta);
int katsu_hip_gemm_f32_dev(const float *a, const float *b, float *c, size_t m, size_t n,
                           size_t k, int trans_a, int trans_b, float beta, void *stream);

/* The whole Matmul VJP on device buffers (Op::backward Matmul arm,
 * tensor.rs:418-445), for C[m,n] = A[m,k] . B[k,n] with upstream gradient
 * G[m,n]:
 *   da[m,k] = beta_a*da + G . B^T     then     db[k,n] = beta_b*db + A^T . G
 * A NULL da or db skips that product (the parent needs no gradient).  When
 * da and db overlap (A and B the same node) this is exactly
 * katsu_hip_gemm_f32_dev(G, B, da, m, k, n, 0, 1, beta_a) followed by
 * katsu_hip_gemm_f32_dev(A, G, db, k, n, m, 1, 0, beta_b).  Otherwise the
 * two products may run as one launch, whose k-sums can be added in another
 * (fixed) order than those two calls': within the same f32 bound, and the
 * same bits on every call. */
int katsu_hip_matmul_vjp_f32_dev(const float *a, const float *b, const float *g, float *da,
                                 float *db, size_t m, size_t k, size_t n, float beta_a,
                                 float beta_b, void *stream);

/* ---- S3: convolution forward --------------------------------------------
 * y[n,k,oh,ow] = sum over valid (c,r,s) of x[n,c,oy*stride+r-pad,
 * ox*stride+s-pad] * w[k,c,r,s]  (Conv2D::forward, conv2d.rs:95-115;
 * cross-correlation, padded taps contribute nothing).  y is overwritten. */
int katsu_hip_conv2d_fwd_f32(const float *x, const float *w, float *y,
                             const katsu_conv_geom *g);
int katsu_hip_conv2d_fwd_f32_dev(const float *x, const float *w, float *y,
                                 const katsu_conv_geom *g, void *stream);

/* ---- S4: convolution backward (backward_buffers, conv2d.rs:269-292) -----
 * dx = beta*dx + d(sum(gy*y))/dx:   dx[x] += gy[y] * w[w] over the visit.
 * beta = 0 reproduces the fresh buffer of conv2d.rs:284; beta = 1 adds into
 * an engine's pending buffer (tensor.rs:383-390). */
int katsu_hip_conv2d_bwd_data_f32(const float *gy, const float *w, float *dx,
                                  const katsu_conv_geom *g, float beta);
int katsu_hip_conv2d_bwd_data_f32_dev(const float *gy, const float *w, float *dx,
                                      const katsu_conv_geom *g, float beta, void *stream);

/* dw = beta*dw + sum over the visit of gy[y] * x[x]  (conv2d.rs:289).
 * The reduction over n*oh*ow is split across workgroups and reduced in a
 * fixed order, so results are deterministic run to run.
 * The _dev form needs `workspace` of katsu_hip_conv2d_bwd_filter_workspace
 * bytes (device memory, 256-byte aligned); pass NULL to use a library-owned
 * buffer, which is allocated (hipMalloc) on first need and kept. */
int katsu_hip_conv2d_bwd_filter_workspace(const katsu_conv_geom *g, size_t *bytes);
int katsu_hip_conv2d_bwd_filter_f32(const float *x, const float *gy, float *dw,
                                    const katsu_conv_geom *g, float beta);
int katsu_hip_conv2d_bwd_filter_f32_dev(const float *x, const float *gy, float *dw,
                                        const katsu_conv_geom *g, float beta,
                                        void *workspace, size_t workspace_bytes,
                                        void *stream);

/* Both passes of backward_buffers (conv2d.rs:265-292) in one call:
 * dx = beta*dx + dX and dw = beta*dw + dW, as the two calls above make them
 * (same results, same determinism).  When both passes take their direct
 * gfx950 kernels they share one launch, so dW work fills the GPU while the
 * last dX tiles finish.  dx and dw may be the same buffer (an engine's
 * pending buffer when input and weights are one node, so equal sizes): it
 * then receives beta*buf + dX + dW, dX added first, as the reference's adds
 * are ordered (tensor.rs:383-390).  Buffers that overlap without being the
 * same are rejected with KATSU_E_INVALID.  The _dev form takes the
 * workspace of katsu_hip_conv2d_bwd_filter_workspace (or NULL, as above),
 * which covers this call as well as the filter gradient alone. */
int katsu_hip_conv2d_bwd_f32(const float *x, const float *w, const float *gy, float *dx,
                             float *dw, const katsu_conv_geom *g, float beta);
int katsu_hip_conv2d_bwd_f32_dev(const float *x, const float *w, const float *gy, float *dx,
                                 float *dw, const katsu_conv_geom *g, float beta,
                                 void *workspace, size_t workspace_bytes, void *stream);

/* The one-call backward above with no allocation of any kind: no hipMalloc,
 * hipFree or allocating library routine, on any call.  No counterpart in the
 * reference: it is for callers that cannot allocate (code under HIP graph
 * capture, tight serving loops, harnesses that forbid allocation).  The dW
 * split partials live in a static device array of
 * katsu_hip_noalloc_scratch_bytes() bytes (40 MiB), one copy per GPU, held
 * until the process ends; its address on a device is looked up on the first
 * call there.  Same kernels, plans and results as
 * katsu_hip_conv2d_bwd_f32_dev; a geometry whose partials would not fit
 * returns KATSU_E_SCRATCH before any launch (no plan of this library needs
 * more than 37.7 MB).  Every call on a GPU shares that GPU's array, so calls
 * that overlap in time on one GPU (two streams, or two threads) race: the
 * caller orders them. */
int katsu_hip_conv2d_bwd_f32_dev_noalloc(const float *x, const float *w, const float *gy,
                                         float *dx, float *dw, const katsu_conv_geom *g,
                                         float beta, void *stream);
size_t katsu_hip_noalloc_scratch_bytes(void);

/* Number of device allocations (hipMalloc) this library has made since it
 * was loaded: its scratch and staging buffers and the katsu_hip_malloc pool.
 * No counterpart in the reference; it lets a caller that cannot allocate
 * check that a code path allocated nothing (the count does not change). */
uint64_t katsu_hip_device_allocations(void);

/* ---- Device residency and the engine's elementwise work -----------------
 * For callers that keep tensor data on the GPU between calls (a device
 * mirror per immutable node, tensor.rs:96-107), accumulate adjoints in
 * device pending buffers (tensor.rs:327-360) and run the elementwise ops,
 * sum and their VJPs there (tensor.rs:217-247, 392-417).  No reference
 * function corresponds to the buffer calls: the reference has no device.
 *
 * katsu_hip_stream: the library's stream (initialising the library).
 * katsu_hip_malloc/free: device memory from a caching pool; a freed block is
 * reused by later allocations in stream order, so callers that use other
 * streams synchronise before freeing.  All blocks are released by
 * katsu_hip_shutdown.
 * katsu_hip_upload/download: count floats host->device / device->host;
 * both return after the copy completes. */
void *katsu_hip_stream(void);
int katsu_hip_malloc(void **ptr, size_t bytes);
int katsu_hip_free(void *ptr);
int katsu_hip_upload(void *dst, const float *src, size_t count, void *stream);
int katsu_hip_download(float *dst, const void *src, size_t count, void *stream);
int katsu_hip_sync(void *stream);

/* c = beta*c + (a + b) and c = beta*c + a*b over n floats, beta in {0, 1}:
 * Tensor::add / Tensor::mul (tensor.rs:217-240) with beta 0; Mul's VJP
 * pending[a] += g*b (tensor.rs:398-409) with beta 1.  Bit-identical to the
 * reference's loops. */
int katsu_hip_add_f32_dev(const float *a, const float *b, float *c, size_t n, float beta,
                          void *stream);
int katsu_hip_mul_f32_dev(const float *a, const float *b, float *c, size_t n, float beta,
                          void *stream);
/* y = beta*y + x (Add's VJP, tensor.rs:392-397; publishing pending into an
 * existing gradient, tensor.rs:349-357; beta = 0 copies into a buffer the
 * caller knows is still zero).  Bit-identical. */
int katsu_hip_accumulate_f32_dev(const float *x, float *y, size_t n, float beta, void *stream);
/* x = value (fresh zero buffers, tensor.rs:120-125 and 328-331). */
int katsu_hip_fill_f32_dev(float *x, size_t n, float value, void *stream);
/* y = beta*y + s[0] with s on the device (Sum's VJP, tensor.rs:410-417). */
int katsu_hip_add_scalar_f32_dev(const float *s, float *y, size_t n, float beta, void *stream);
/* out[0] = beta*out[0] + sum(x) (Tensor::sum, tensor.rs:242-247).  A fixed
 * tree, identical run to run; it differs from the reference's sequential
 * fold within the f32 summation bound. */
int katsu_hip_sum_f32_dev(const float *x, size_t n, float *out, float beta, void *stream);
/* The stem workload's pooling chain (config 5): out[r] = sum_c y[r][c] / cols,
 * and its VJP dy[r][c] = beta*dy[r][c] + scale*g[r]. */
int katsu_hip_mean_rows_f32_dev(const float *y, size_t rows, size_t cols, float *out,
                                void *stream);
int katsu_hip_broadcast_rows_f32_dev(const float *g, size_t rows, size_t cols, float scale,
                                     float *dy, float beta, void *stream);

/* Grad-CAM over an activation map and its gradient (the raw material
 * get_activation_map provides, conv2d.rs:140-148; the method the reference
 * outlines in docs/conv2d.md, "O que falta para Grad-CAM"), NCHW [n][c][hw]:
 *   alpha[n][c] = mean over hw of grad[n][c][.]
 *   cam[n][p]   = max(0, sum_c alpha[n][c] * act[n][c][p])
 *   then each image's map divided by its maximum (all-zero maps stay zero).
 * cam holds n*hw floats.  No counterpart in the reference's code. */
int katsu_hip_gradcam_f32_dev(const float *act, const float *grad, size_t n, size_t c,
                              size_t hw, float *cam, void *stream);

/* Grad-CAM's last step, resizing each map to the original image
 * (docs/conv2d.md, "O que falta para Grad-CAM": "redimensionar para a imagem
 * original"): n maps [ih][iw] -> dst [n][oh][ow], bilinear with half-pixel
 * centres.  Output row oy samples source row
 * sy = max(0, (oy + 0.5) * ih/oh - 0.5) and blends rows floor(sy) and
 * floor(sy) + 1 (clamped to ih - 1) with weights 1 - f and f,
 * f = sy - floor(sy); columns likewise.  Each blend is rounded as
 * (1 - f)*a + f*b (no fused multiply-add); a neighbour of weight exactly 0 is
 * left out, so NaN or Inf reaches only the outputs that use that pixel.
 * Equal sizes copy every value as it is, non-finite ones included.
 * ih*iw and oh*ow must each be <= 2^31 - 1.  No counterpart in the
 * reference's code. */
int katsu_hip_resize_bilinear_f32_dev(const float *src, size_t n, size_t ih, size_t iw,
                                      size_t oh, size_t ow, float *dst, void *stream);

/* ---- Language-model operators ---------------------------------------------
 * What a block of a language model computes between its matrix products.  No
 * counterpart in the reference's code.  All take device pointers and a stream,
 * in float32 or bfloat16; sums, softmax statistics and norms are float32 or
 * wider.  Results do not depend on the order of atomics: the same call gives
 * the same bits. */
typedef enum katsu_dtype { KATSU_F32 = 0, KATSU_BF16 = 1 } katsu_dtype;

/* Attention over packed sequences.  q and out hold tokens_q tokens of `heads`
 * heads, k and v tokens_k tokens of kv_heads (which divides heads; query head
 * h reads key head h / (heads/kv_heads)), all of head_dim channels (1..128).
 * Strides are in elements, [0] between tokens and [1] between heads; channels
 * are adjacent.  Sequence s has queries cu_q[s] .. cu_q[s+1] and keys cu_k[s]
 * .. cu_k[s+1], or with k_lens the first k_lens[s] of those (slots of a cache);
 * cu_q and cu_k are device arrays of seqs + 1 int32 that do not fall, both NULL
 * for one sequence of all tokens; they may begin after 0 and end before the last
 * token (a slice of a batch's starts); values outside the tensors are taken as
 * their ends; what outputs hold for tokens that no sequence holds is undefined.
 *   S = scale q.k over the visible keys, P = softmax(S), out = P v,
 *   lse[head][token] = log sum exp S       (natural logarithm)
 * With causal set query i of Lq sees key j of Lk if j <= i + Lk - Lq: the last
 * query sees every key.  A query that sees none gives out 0 and lse -inf.
 * What masked places hold changes nothing, Inf and NaN included.
 * scale must be positive and finite; heads at most 65535; an output's strides
 * must not be zero, nor its memory an operand's.  In bfloat16 the products take
 * P rounded to bfloat16, and the backward ones dS too (with 16 bits up to 32
 * channels); sums are float32.  Float32 operands are not rounded. */
typedef struct katsu_attention {
    int32_t dtype;  /* katsu_dtype of q, k, v, out */
    int32_t causal;
    uint64_t heads, kv_heads, head_dim;
    uint64_t seqs, tokens_q, tokens_k;
    int64_t q_stride[2], k_stride[2], v_stride[2], out_stride[2];
    float scale;
} katsu_attention;

/* The forward pass; lse may be NULL.  `workspace` of
 * katsu_hip_attention_fwd_workspace bytes (device memory, 16-byte aligned)
 * holds the parts of a key axis split over workgroups; NULL uses a
 * library-owned buffer, allocated on first need and kept. */
int katsu_hip_attention_fwd_workspace(const katsu_attention *d, size_t *bytes);
int katsu_hip_attention_fwd_dev(const katsu_attention *d, const void *q, const void *k,
                                const void *v, const int32_t *cu_q, const int32_t *cu_k,
                                const int32_t *k_lens, void *out, float *lse, void *workspace,
                                size_t workspace_bytes, void *stream);

/* The backward pass, from dout, the gradient of out, and the forward call's
 * operands, out and lse (same cu_q and cu_k; no k_lens):
 *   P = exp(S - lse),  dS = P (dout v^T - dout.out),
 *   dq = scale dS k,  dk = scale dS^T q and dv = P^T dout summed over the
 * query heads of a key head.  Outputs are overwritten.  A query that sees no
 * key gives no gradient, a key that no query sees gets zeros.
 * Workspace as above, of katsu_hip_attention_bwd_workspace bytes: in float32 dk
 * and dv once more for each query head of a group and up to four runs (65536
 * tokens, 32/8 heads of 128: 8.6 GB). */
typedef struct katsu_attention_grads {
    int64_t dout_stride[2], dq_stride[2], dk_stride[2], dv_stride[2];
} katsu_attention_grads;
int katsu_hip_attention_bwd_workspace(const katsu_attention *d, size_t *bytes);
int katsu_hip_attention_bwd_dev(const katsu_attention *d, const katsu_attention_grads *g,
                                const void *dout, const void *q, const void *k, const void *v,
                                const void *out, const float *lse, const int32_t *cu_q,
                                const int32_t *cu_k, void *dq, void *dk, void *dv,
                                void *workspace, size_t workspace_bytes, void *stream);

/* Rotary positions.  Of each head's head_dim channels the first rotary_dim (R,
 * even) turn in pairs, (a, b) -> (a cos - b sin, a sin + b cos): pair i is
 * channels i and i + R/2, or 2i and 2i + 1 with interleaved set; the rest is
 * copied.  Token t turns by row positions[t] of table ([length][R] float32:
 * R/2 cosines, then R/2 sines; rows outside it are taken as its ends), or by
 * row t if positions is NULL.  inverse turns back: the gradient of a turn.
 * q and k ([tokens][heads][head_dim], strides in elements as above) go in one
 * launch; k may be NULL with k_heads 0.  Outputs may be the inputs, with the
 * same strides; an output's strides must not be zero, none may be negative.
 * At most 65535 heads each, fewer than 2^20 channels of a token in all. */
typedef struct katsu_rotary {
    int32_t dtype, interleaved, inverse;
    uint64_t tokens, heads, k_heads, head_dim, rotary_dim, length;
    int64_t q_stride[2], k_stride[2], q_out_stride[2], k_out_stride[2];
} katsu_rotary;
int katsu_hip_rotary_dev(const katsu_rotary *d, const void *q, const void *k, const float *table,
                         const int32_t *positions, void *q_out, void *k_out, void *stream);

/* Fills such a table: position p's pair i turns by p f_i, computed in float64,
 * f_i = base^(-2i/R).  factor >= 1 scales for a context longer than the model
 * was trained on, length = factor times that: f_i / factor, or with
 * by_wavelength f_i kept where it turns 32 times or more within the original
 * length, divided where it turns once or less, mixed linearly between, and
 * cosines and sines times 0.1 ln(factor) + 1 (the scheme published as YaRN). */
int katsu_hip_rotary_table_f32_dev(float *table, size_t length, size_t rotary_dim, double base,
                                   double factor, int by_wavelength, void *stream);

/* Between two blocks of a model, rows x cols, cols <= 16384, all tensors of
 * one type and contiguous:
 *   n = o / sqrt(mean(o^2) + eps) * w_post     (n = o if w_post is NULL)
 *   y = x + alpha * gate * n
 *   h = y / sqrt(mean(y^2) + eps) * w_pre      (no h if w_pre is NULL)
 * with a gate of cols values, of rows x cols, or none (gate_rows).  h is of y
 * before its rounding.  stats [2][rows] (or NULL) receives 1/sqrt(..) of o
 * and y, 0 for a norm that is not taken: what the backward call reads.
 * y may be x, h may be o. */
typedef enum katsu_gate { KATSU_GATE_NONE = 0, KATSU_GATE_CHANNEL = 1,
                          KATSU_GATE_ELEMENT = 2 } katsu_gate;
typedef struct katsu_block_norm {
    int32_t dtype, gate_rows;  /* katsu_dtype, katsu_gate */
    uint64_t rows, cols;
    float alpha, eps;          /* eps: of the forward call only */
} katsu_block_norm;
int katsu_hip_block_norm_dev(const katsu_block_norm *d, const void *x, const void *o,
                             const void *gate, const void *w_post, const void *w_pre, void *y,
                             void *h, float *stats, void *stream);

/* Its gradient: from dy (gradient that reaches y otherwise) and dh, with the
 * forward call's y, o and stats: dx (all of y's gradient), d_o, dgate (shaped
 * as gate), dw_post and dw_pre; outputs are overwritten.  Sums over rows are
 * in float32, in a fixed order, through a workspace as above. */
int katsu_hip_block_norm_bwd_workspace(const katsu_block_norm *d, size_t *bytes);
int katsu_hip_block_norm_bwd_dev(const katsu_block_norm *d, const void *dy, const void *dh,
                                 const void *y, const void *o, const float *stats,
                                 const void *gate, const void *w_post, const void *w_pre,
                                 void *dx, void *d_o, void *dgate, void *dw_post, void *dw_pre,
                                 void *workspace, size_t workspace_bytes, void *stream);

/* norm[0] = sqrt(sum over the n tensors of all squares), squares summed in
 * float64; out = in * min(1, max_norm / (norm + 1e-6)), tensor by tensor (out
 * may be in; no two tensors that are written may share memory).  dtypes, in,
 * out and counts are host arrays; the tensors are contiguous device memory of
 * katsu_dtype dtypes[i].  A norm that is NaN
 * makes all outputs NaN, an infinite one zero (NaN where in is infinite).
 * max_norm must not be negative.  Partial sums go through a workspace as above,
 * of katsu_hip_clip_grad_norm_workspace bytes for n tensors; the form without
 * one takes the library's. */
int katsu_hip_clip_grad_norm_workspace(size_t n, size_t *bytes);
int katsu_hip_clip_grad_norm_dev(const int32_t *dtypes, const void *const *in, void *const *out,
                                 const size_t *counts, size_t n, float max_norm, float *norm,
                                 void *stream);
int katsu_hip_clip_grad_norm_ws_dev(const int32_t *dtypes, const void *const *in,
                                    void *const *out, const size_t *counts, size_t n,
                                    float max_norm, float *norm, void *workspace,
                                    size_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* KATSU_HIP_H */
