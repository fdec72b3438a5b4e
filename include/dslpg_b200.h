/*
 * dslpg_b200.h — C ABI of the B200 (sm_100a) row-wise reduction backend.
 *
 * One entry point per ViperBench kernel of the row-reduction family. Each takes
 * plain device pointers, sizes and a dtype code, launches on the given stream
 * and returns 0 on success, a positive cudaError_t when a CUDA call failed, or
 * a negative DSLPG_ERR_* code when the arguments were rejected before any
 * launch. No entry point allocates memory, synchronises, or keeps state other
 * than a per-device cache of SM counts and occupancy figures (lock-protected),
 * the per-thread kernel-shape selection below, and the per-device copy streams
 * of the host-buffer entry points.
 *
 * Layout: every row-wise operand is a dense row-major [M, N] matrix (the
 * reference flattens x[..., D] to [M, D] the same way). The caller owns every
 * buffer; inputs are never written.
 *
 * Reference interfaces (paths inside tingxi-li/DSLPerfGap):
 *   layer_norm      ViperBench/layer_norm/pytorch_impl.py:5-12
 *   rms_norm        ViperBench/rms_norm/pytorch_impl.py:3-10
 *   softmax         ViperBench/softmax/pytorch_impl.py:4-6
 *   log_softmax     ViperBench/log_softmax/pytorch_impl.py:4-8
 *   logsumexp       ViperBench/logsumexp/pytorch_impl.py:3-5
 *   cross_entropy   ViperBench/cross_entropy/pytorch_impl.py:4-90 and the
 *                   kernel layout of ViperBench/cross_entropy/triton_impl.py:13-75,123-140
 */
#ifndef DSLPG_B200_H
#define DSLPG_B200_H

#include <stdint.h>
#include <cuda_runtime_api.h>

#if defined(__GNUC__)
#define DSLPG_API __attribute__((visibility("default")))
#else
#define DSLPG_API
#endif

#ifdef __cplusplus
extern "C" {
#endif

/* Element type codes (storage types; arithmetic is always fp32). */
enum {
  DSLPG_F32 = 0,
  DSLPG_F16 = 1,
  DSLPG_BF16 = 2,
  DSLPG_I32 = 3, /* labels only */
  DSLPG_I64 = 4  /* labels only */
};

/* Argument errors (returned before anything is launched). */
enum {
  DSLPG_OK = 0,
  DSLPG_ERR_NULL_POINTER = -1,
  DSLPG_ERR_BAD_SHAPE = -2,
  DSLPG_ERR_BAD_DTYPE = -3,
  DSLPG_ERR_BAD_EPS = -4,
  DSLPG_ERR_BAD_ARGUMENT = -5,
  DSLPG_ERR_TOO_LARGE = -6 /* dslpg_kernel_ff_static: the problem does not fit its static scratch */
};

/* Kernel-shape selection (normally DSLPG_PATH_AUTO; the others exist so tests
 * and benchmarks can exercise one implementation on purpose). */
enum {
  DSLPG_PATH_AUTO = 0,     /* pick per shape */
  DSLPG_PATH_RESIDENT = 1, /* rows read straight into registers; kernel_ff: one CTA per 128x128 tile */
  DSLPG_PATH_TMA = 2,      /* rows / row chunks staged by TMA bulk copies */
  DSLPG_PATH_STREAM = 3,   /* two-pass streaming (any length or alignment); kernel_ff: the weight-streaming
                              kernel for M <= 8 (chosen by default for M <= 3) */
  DSLPG_PATH_CLUSTER = 4   /* a row split over a thread-block cluster (DSMEM exchange);
                              kernel_ff: CTA pairs (tcgen05 cta_group::2) on 256x128 tiles */
};

/* Select the kernel shape for the calling host thread's subsequent calls
 * (a per-thread setting: other threads keep their own, DSLPG_PATH_AUTO unless
 * they set one). A path that cannot handle a given shape falls back to one
 * that can. Returns 0 or DSLPG_ERR_BAD_ARGUMENT. No reference counterpart: a
 * testing aid. */
DSLPG_API int dslpg_set_kernel_path(int path);

/* The calling thread's kernel-shape selection. No reference counterpart. */
DSLPG_API int dslpg_get_kernel_path(void);

/* Number of bounded device-side waits (TMA pipeline barriers) that ran out of
 * time since the last call, and reset the count. Synchronises the device.
 * A non-zero value means some outputs of the affected launches were not
 * written. No reference counterpart. */
DSLPG_API unsigned int dslpg_take_wait_timeouts(void);

/* Library version, (major << 16) | minor. */
DSLPG_API int dslpg_version(void);

/* Human-readable text for a return code (negative: ours; positive: CUDA's). */
DSLPG_API const char* dslpg_error_string(int code);

/*
 * LayerNorm forward over the last dimension:
 *   y = (x - mean) / sqrt(var + eps) * weight + bias      (var biased)
 * x, y: [M, N] of x_dtype; weight, bias: [N] of w_dtype (bias may be NULL).
 * Replaces layer_norm(x, weight, bias, eps) of
 * ViperBench/layer_norm/pytorch_impl.py:5-12 (F.layer_norm). The eps == 1e-5
 * restriction of that file is enforced by the Python wrapper, not here.
 */
DSLPG_API int dslpg_layer_norm_fwd(const void* x, const void* weight, const void* bias, void* y,
                         int64_t M, int64_t N, int x_dtype, int w_dtype, float eps,
                         cudaStream_t stream);

/*
 * RMSNorm forward over the trailing N elements of each row:
 *   y = (x / sqrt(mean(x^2) + eps) * weight)  computed in fp32, stored as x_dtype
 * Replaces rms_norm(x, normalized_shape, weight, eps) of
 * ViperBench/rms_norm/pytorch_impl.py:3-10.
 */
DSLPG_API int dslpg_rms_norm_fwd(const void* x, const void* weight, void* y, int64_t M, int64_t N,
                       int x_dtype, int w_dtype, float eps, cudaStream_t stream);

/*
 * Softmax along the last dimension: y = exp(x - max) / sum(exp(x - max)).
 * Replaces softmax(x) of ViperBench/softmax/pytorch_impl.py:4-6.
 */
DSLPG_API int dslpg_softmax_fwd(const void* x, void* y, int64_t M, int64_t N, int dtype,
                      cudaStream_t stream);

/*
 * Log-softmax over the middle axis of a dense [M, N, K] tensor
 * (K == 1 is the last-dimension case): y = x - max - log(sum(exp(x - max))).
 * x is in_dtype, y is out_dtype; when they differ, x is first rounded to
 * out_dtype, as F.log_softmax(x, dim, dtype=out_dtype) does.
 * Replaces log_softmax(x, dim, dtype) of ViperBench/log_softmax/pytorch_impl.py:4-8.
 */
DSLPG_API int dslpg_log_softmax_fwd(const void* x, void* y, int64_t M, int64_t N, int64_t K,
                          int in_dtype, int out_dtype, cudaStream_t stream);

/*
 * logsumexp along the last dimension, with torch.logsumexp's treatment of
 * infinite maxima (a +inf entry gives +inf, an all -inf row gives -inf):
 * y[M] of dtype.  Replaces logsumexp(x) of ViperBench/logsumexp/pytorch_impl.py:3-5.
 */
DSLPG_API int dslpg_logsumexp_fwd(const void* x, void* y, int64_t M, int64_t N, int dtype,
                        cudaStream_t stream);

/*
 * Blockwise cross-entropy forward. For every row r and column block
 * cb < ceil(n_cols / block_size) it writes, at flat index cb * n_rows + r of
 * the three fp32 outputs, the block's log-sum-exp of logits * logit_scale, the
 * loss term and the z-loss term, exactly as
 * ViperBench/cross_entropy/pytorch_impl.py:4-90 (and the Triton kernel at
 * ViperBench/cross_entropy/triton_impl.py:13-75) define them. Flat entries at or
 * beyond ceil(n_cols / block_size) * n_rows are not written. Under split != 0
 * the z-loss entries are written as 0.
 * logits: [n_rows, n_cols] rows `logits_row_stride` elements apart;
 * labels: [n_rows] of labels_dtype (DSLPG_I32 or DSLPG_I64).
 * Replaces cross_entropy_fwd(...) of ViperBench/cross_entropy/pytorch_impl.py:4-90.
 */
DSLPG_API int dslpg_cross_entropy_fwd(const void* logits, const void* labels, float* loss, float* lse,
                            float* z_loss, int64_t n_rows, int64_t n_cols,
                            int64_t logits_row_stride, int logits_dtype, int labels_dtype,
                            float smoothing, float logit_scale, float lse_square_scale,
                            int64_t ignored_index, float total_classes, int64_t class_start_idx,
                            int64_t block_size, int has_smoothing, int split,
                            cudaStream_t stream);

/*
 * Blockwise cross-entropy backward: for every row r and column c < n_cols,
 *   p = exp(logits[r,c] * logit_scale - lse[r]);  p += 2 * lse_square_scale * lse[r] * p;
 *   p -= (has_smoothing ? 1 - smoothing : 1) at c == labels[r] - class_start_idx;
 *   p -= smoothing / total_classes                  (has_smoothing only);
 *   dlogits[r,c] = (dloss[r] * logit_scale) * p, with dloss[r] = 0 where
 *   labels[r] == ignored_index,
 * stored in logits_dtype. lse holds one fp32 value per row (the forward's lse
 * for a single column block); dloss[r] is read at r * dloss_stride.
 * Replaces cross_entropy_bwd(...) of ViperBench/cross_entropy/pytorch_impl.py:93-141
 * (kernel: ViperBench/cross_entropy/triton_impl.py:79-120, wrapper :143-158).
 */
DSLPG_API int dslpg_cross_entropy_bwd(const void* dloss, int dloss_dtype, int64_t dloss_stride,
                            const void* logits, const float* lse, const void* labels, void* dlogits,
                            int64_t n_rows, int64_t n_cols, int64_t logits_row_stride,
                            int64_t dlogits_row_stride, int logits_dtype, int labels_dtype,
                            float smoothing, float logit_scale, float lse_square_scale,
                            int64_t ignored_index, float total_classes, int64_t class_start_idx,
                            int has_smoothing, cudaStream_t stream);

/*
 * Cross-entropy forward and backward in one pass over the logits, for one
 * column block per row (the reference's BLOCK_SIZE >= n_cols) without SPLIT,
 * when dloss is known before the forward (the gradient of a mean or sum of
 * the per-row losses). loss / lse / z_loss: [n_rows] fp32, the values
 * dslpg_cross_entropy_fwd stores at flat index r; dlogits as
 * dslpg_cross_entropy_bwd computes them from that lse. The logits are read
 * from HBM once (the second pass over a row hits L2) instead of twice.
 * Serves cross_entropy_fwd followed by cross_entropy_bwd of
 * ViperBench/cross_entropy/triton_impl.py:123-140 and :79-120
 * (pytorch_impl.py:4-90 and :93-141).
 */
DSLPG_API int dslpg_cross_entropy_fwd_bwd(const void* logits, const void* labels, const void* dloss, int dloss_dtype,
                                          int64_t dloss_stride, float* loss, float* lse, float* z_loss, void* dlogits,
                                          int64_t n_rows, int64_t n_cols, int64_t logits_row_stride,
                                          int64_t dlogits_row_stride, int logits_dtype, int labels_dtype,
                                          float smoothing, float logit_scale, float lse_square_scale,
                                          int64_t ignored_index, float total_classes, int64_t class_start_idx,
                                          int has_smoothing, cudaStream_t stream);

/*
 * Reductions over the middle axis of a dense [M, N, K] tensor (a reduced run
 * of adjacent axes is one N; K == 1 reduces rows). Index outputs are int64 and
 * follow torch: the first NaN is the maximum; equal maxima give the smallest
 * index.
 *
 * mean: y[M*K] of out_dtype = sum / N, accumulated in fp32 after converting x
 * to out_dtype (torch.mean(x, dim, dtype=out_dtype)).
 * Replaces mean_reduction(input_tensor, dim, keepdim, dtype) of
 * ViperBench/mean_reduction/pytorch_impl.py:4-8.
 */
DSLPG_API int dslpg_mean_reduction(const void* x, void* y, int64_t M, int64_t N, int64_t K, int in_dtype,
                                   int out_dtype, cudaStream_t stream);

/* values[M*K] (x's dtype) and indices[M*K] of the maximum along N.
 * Replaces max_reduction(input, dim, keepdim) of ViperBench/max_reduction/pytorch_impl.py:4-11. */
DSLPG_API int dslpg_max_reduction(const void* x, void* values, int64_t* indices, int64_t M, int64_t N,
                                  int64_t K, int dtype, cudaStream_t stream);

/* indices[M*K] of the maximum along N.
 * Replaces argmax(input_tensor, dim, keepdim) of ViperBench/argmax/pytorch_impl.py:4-8. */
DSLPG_API int dslpg_argmax(const void* x, int64_t* indices, int64_t M, int64_t N, int64_t K, int dtype,
                           cudaStream_t stream);

/*
 * dslpg_rms_norm_fwd on HOST buffers: x_host [M, N] (x_dtype) in, y_host
 * [M, N] out; weight is a device pointer. The rows stream through the GPU in
 * chunks of about 16 MiB, the upload of one chunk, the kernel on the previous
 * one and the download of the one before overlapping (two copy streams of
 * this library plus `stream`; one cudaMemcpyAsync per chunk and direction).
 * With pinned host memory the copies run asynchronously in both directions at
 * once; pageable memory works but the copies do not overlap. `workspace`
 * (device, 256-byte aligned) holds the chunk buffers: at least
 * dslpg_rms_norm_fwd_host_workspace_bytes(M, N, x_dtype) bytes. The call
 * returns once the work is enqueued; everything is ordered on `stream`, so
 * synchronise it before reading y_host. Calls on one device are serialised by
 * a lock while they enqueue. Same result as dslpg_rms_norm_fwd row by row.
 * Serves the reference's rms_norm (ViperBench/rms_norm/pytorch_impl.py:3-10)
 * for inputs that live in host memory.
 */
DSLPG_API int dslpg_rms_norm_fwd_host_workspace_bytes(int64_t M, int64_t N, int x_dtype, int64_t* bytes);
DSLPG_API int dslpg_rms_norm_fwd_host(const void* x_host, const void* weight, void* y_host, int64_t M, int64_t N,
                                      int x_dtype, int w_dtype, float eps, void* workspace, int64_t workspace_bytes,
                                      cudaStream_t stream);

/*
 * dslpg_layer_norm_fwd on HOST buffers, with the same chunked pipeline,
 * workspace rule and ordering as dslpg_rms_norm_fwd_host above; weight and
 * bias (bias may be NULL) are device pointers. Same result as
 * dslpg_layer_norm_fwd row by row. Serves the reference's layer_norm
 * (ViperBench/layer_norm/pytorch_impl.py:5-12) for inputs that live in host
 * memory, e.g. one row block per GPU of a batch held by the host.
 */
DSLPG_API int dslpg_layer_norm_fwd_host_workspace_bytes(int64_t M, int64_t N, int x_dtype, int64_t* bytes);
DSLPG_API int dslpg_layer_norm_fwd_host(const void* x_host, const void* weight, const void* bias, void* y_host,
                                        int64_t M, int64_t N, int x_dtype, int w_dtype, float eps, void* workspace,
                                        int64_t workspace_bytes, cudaStream_t stream);

/*
 * Llama feed-forward with the RMSNorm fused around a dual GEMM (tcgen05 tensor
 * cores; for M <= 3 rows a kernel that streams the weight rows instead):
 *   a_norm[m] = rsqrt(sum_k x[m,k]^2 / K + 1e-6);  xs = x * rms_w (fp16);
 *   out[m,n] = silu(a_norm[m] * (xs @ w1^T)[m,n]) * (a_norm[m] * (xs @ w3^T)[m,n])   (fp16)
 * x [M, K], w1 and w3 [N, K], rms_w [K], out [M, N]: all fp16, row-major,
 * 16-byte aligned; K % 8 == 0. `workspace` (256-byte aligned) holds xs and
 * a_norm: at least dslpg_kernel_ff_workspace_bytes(M, K) bytes.
 * Replaces kernel_ff(x, w1, w3, rms_w) of ViperBench/linear_activation/pytorch_impl.py:5-54.
 */
DSLPG_API int dslpg_kernel_ff_workspace_bytes(int64_t M, int64_t K, int64_t* bytes);
DSLPG_API int dslpg_kernel_ff(const void* x, const void* w1, const void* w3, const void* rms_w, void* out,
                              int64_t M, int64_t N, int64_t K, void* workspace, int64_t workspace_bytes,
                              cudaStream_t stream);

/*
 * dslpg_kernel_ff without a caller-provided workspace and without any device
 * allocation: xs and a_norm live in a file-scope static __device__ scratch of
 * DSLPG_KERNEL_FF_STATIC_SCRATCH_BYTES (16 MiB + 64 KiB), enough for
 * M * K <= 8,388,608 fp16 elements (e.g. 2048 x 4096) as measured by
 * dslpg_kernel_ff_workspace_bytes; larger problems return DSLPG_ERR_TOO_LARGE
 * before anything is launched. It is meant for callers that cannot allocate
 * device memory per call: a C / FFI host that owns no device allocator (the
 * memory belongs to another framework's pool), or a loop where the device-wide
 * synchronisation of cudaMalloc / cudaFree is not acceptable.
 * Set-up: the first call on each device (the device current at the call) looks
 * up the scratch address with cudaGetSymbolAddress, which may load this
 * library's device code; make that first call before any stream capture. The
 * address is kept per device together with the id of the CUDA context it
 * belongs to, so after a cudaDeviceReset (or any replacement of the device's
 * context) the next call repeats the set-up instead of using a stale address.
 * The scratch is part of this library's device code: once any kernel_ff entry
 * point has loaded that code on a device, its 16 MiB + 64 KiB stay allocated
 * there until the context ends, also for callers that only use dslpg_kernel_ff.
 * No part of the scratch has to start at zero (every call writes all of xs and
 * a_norm before reading them). There is ONE scratch per device: calls that
 * overlap on the same device (different streams, or different host threads
 * without ordering) race on it and give wrong results; order them on one stream.
 * No reference counterpart: the reference's kernel_ff always allocates its
 * temporaries through torch.
 */
#define DSLPG_KERNEL_FF_STATIC_SCRATCH_BYTES ((int64_t)(16 * 1024 * 1024 + 64 * 1024))
DSLPG_API int dslpg_kernel_ff_static(const void* x, const void* w1, const void* w3, const void* rms_w, void* out,
                                     int64_t M, int64_t N, int64_t K, cudaStream_t stream);

/*
 * Per-head RMSNorm with the rotary position rotation, and the rotation alone,
 * forward and backward.
 *
 * q is [batch, seq, q_heads, head_dim] and k [batch, seq, k_heads, head_dim],
 * each with its own batch, seq and head strides (in elements; the last axis is
 * dense), so both may be views into one projection output. Outputs are dense
 * in that order. With n = rotary_dim / 2 frequencies inv_freq[i] (float32),
 * phi_i = position * inv_freq[i], and pairs (i, i + n) (or (2i, 2i + 1) when
 * `interleaved`) of the first rotary_dim features:
 *   u = x / sqrt(mean(x^2) + eps) * weight            (rope: u = x)
 *   y_i = u_i cos phi_i - u_j sin phi_i;   y_j = u_j cos phi_i + u_i sin phi_i
 * and the features past rotary_dim are u. Arithmetic is fp32 with one rounding
 * at the store. The angles are formed in 64-bit fixed point, off by
 * |position| 2^-64 turns for |inv_freq| up to 2^18 (which have to be finite):
 * positions up to 2^38 in size keep the cosine to fp32 accuracy, those up to
 * 2^50 to 4e-4.
 *
 * `positions` (int32 or int64) has `axes` (1 to 4) values for each token, with
 * axis, batch and seq strides (0: broadcast). Frequency i turns by axis a where
 * sections[0] + ... + sections[a - 1] <= i < sections[0] + ... + sections[a];
 * the sections add up to n.
 *
 * head_dim is at most 1024, and batch * seq * (q_heads + k_heads) at most 2^30.
 * q's pointers may be NULL when q_heads is 0, and k's when k_heads is 0.
 * No reference counterpart: the suite has the norm (rms_norm), not this form.
 */
typedef struct dslpg_heads {
  int64_t batch, seq, q_heads, k_heads, head_dim, rotary_dim;
  int64_t q_strides[3], k_strides[3];    /* batch, seq, head; rope_bwd: of dq_out and dk_out */
  int64_t dq_strides[3], dk_strides[3];  /* qk_norm_rope_bwd: of dq_out and dk_out */
  int64_t position_strides[3];           /* axis, batch, seq */
  int64_t sections[4];                   /* the first `axes` of them */
  int32_t axes, interleaved;
  int32_t dtype, weight_dtype, positions_dtype; /* q and k; both weights; I32 or I64 */
  int32_t reserved;
} dslpg_heads;

DSLPG_API int dslpg_rope_fwd(const void* q, const void* k, const void* positions, const float* inv_freq, void* q_out,
                             void* k_out, const dslpg_heads* heads, cudaStream_t stream);

/* The rotation by -phi: the gradients of rope_fwd's inputs. */
DSLPG_API int dslpg_rope_bwd(const void* dq_out, const void* dk_out, const void* positions, const float* inv_freq,
                             void* dq, void* dk, const dslpg_heads* heads, cudaStream_t stream);

DSLPG_API int dslpg_qk_norm_rope_fwd(const void* q, const void* k, const void* q_weight, const void* k_weight,
                                     const void* positions, const float* inv_freq, void* q_out, void* k_out,
                                     const dslpg_heads* heads, float eps, cudaStream_t stream);

/* dq, dk (dense, q's type) and the weights' gradients (float32, [head_dim],
 * summed over all tokens and heads in a fixed order). `workspace` (16-byte
 * aligned): dslpg_qk_norm_rope_bwd_workspace_bytes(head_dim) bytes. */
DSLPG_API int dslpg_qk_norm_rope_bwd_workspace_bytes(int64_t head_dim, int64_t* bytes);
DSLPG_API int dslpg_qk_norm_rope_bwd(const void* dq_out, const void* dk_out, const void* q, const void* k,
                                     const void* q_weight, const void* k_weight, const void* positions,
                                     const float* inv_freq, void* dq, void* dk, float* dq_weight, float* dk_weight,
                                     const dslpg_heads* heads, float eps, void* workspace, int64_t workspace_bytes,
                                     cudaStream_t stream);

/*
 * Losses of post-training on rows of logits, with their gradients: the clipped
 * policy loss with a KL term, and the preference loss on paired sequences.
 *
 * logits [n_rows, n_cols] of logits_dtype, rows row_stride elements apart;
 * labels [n_rows] (int32 or int64), dense. With z = logit_scale * logits:
 * lse = log sum exp z, logp = z[label] - lse (both float32 outputs [n_rows]).
 * A row whose label is ignored_index, or no column, is left out: its logits are
 * not read, and its loss, logp, lse, kl and gradient are 0. n_cols <= 2^30;
 * logit_scale is 0, or 1e-30 to 1e30 in size.
 * No reference counterpart: the suite has the cross-entropy of such rows.
 */
typedef struct dslpg_logit_rows {
  const void* logits;
  const void* labels;
  int64_t n_rows, n_cols, row_stride, ignored_index;
  double logit_scale;
  int32_t logits_dtype, labels_dtype;
} dslpg_logit_rows;

/*
 * Per row, with old = old_logp, A = advantages, ref = ref_logp (float32, each
 * with its own stride; 0: one value for all rows):
 *   r = exp(logp - old);  d = ref - logp;  kl = exp(d) - d - 1  (0 when ref_logp is NULL)
 *   loss = -min(r A, clip(r, 1 - clip_low, 1 + clip_high) A) + kl_coef kl
 *   g = dloss/dlogp = (0 where the clipped term alone counts, else -r A) + kl_coef (1 - exp(d))
 *   dlogits = dloss g logit_scale (onehot(label) - softmax(z))
 * 0 <= clip_low <= 1, clip_high >= 0. With kl_coef 0 the KL term is only reported.
 * Where A is 0 there is no policy term, however large r is.
 */
typedef struct dslpg_policy_terms {
  const float* old_logp;
  const float* advantages;
  const float* ref_logp;
  int64_t old_stride, advantages_stride, ref_stride;
  float clip_low, clip_high, kl_coef;
  float reserved;
} dslpg_policy_terms;

DSLPG_API int dslpg_policy_loss_fwd(const dslpg_logit_rows* rows, const dslpg_policy_terms* terms, float* loss,
                                    float* logp, float* lse, float* kl, cudaStream_t stream);

/* dlogits (logits_dtype, rows dlogits_row_stride apart) from the forward's lse
 * and the losses' gradients dloss (float32 [n_rows], stride dloss_stride). */
DSLPG_API int dslpg_policy_loss_bwd(const dslpg_logit_rows* rows, const dslpg_policy_terms* terms, const float* dloss,
                                    int64_t dloss_stride, const float* lse, void* dlogits, int64_t dlogits_row_stride,
                                    cudaStream_t stream);

/* Both in one call, for a dloss known beforehand: the logits are read from HBM
 * once where their length allows it. */
DSLPG_API int dslpg_policy_loss_fwd_bwd(const dslpg_logit_rows* rows, const dslpg_policy_terms* terms,
                                        const float* dloss, int64_t dloss_stride, float* loss, float* logp, float* lse,
                                        float* kl, void* dlogits, int64_t dlogits_row_stride, cudaStream_t stream);

/*
 * 2 n_pairs sequences of rows: sequence s is rows seq_starts[s] to
 * seq_starts[s + 1] (2 n_pairs + 1 ascending bounds, int32 or int64); the
 * chosen ones come first, pair k is sequences k and n_pairs + k. Rows before
 * the first bound or from the last one on are left out.
 *   log_ratio[s] = sum of logp - ref_logp over the rows of s that are not left out
 *   m = beta (log_ratio[k] - log_ratio[n_pairs + k])
 *   loss[k] = (1 - smoothing) softplus(-m) + smoothing softplus(m)
 * The sums are held in 64 bits, in a fixed order. 0 <= smoothing <= 1.
 */
typedef struct dslpg_pair_terms {
  const void* seq_starts;
  const float* ref_logp; /* not read by the backward */
  int64_t n_pairs, ref_stride;
  float beta, smoothing;
  int32_t starts_dtype, reserved;
} dslpg_pair_terms;

DSLPG_API int dslpg_preference_loss_fwd(const dslpg_logit_rows* rows, const dslpg_pair_terms* terms, float* loss,
                                        float* log_ratio, float* logp, float* lse, cudaStream_t stream);

/* dlogits from the forward's lse and log_ratio and the pairs' dloss (float32 [n_pairs]). */
DSLPG_API int dslpg_preference_loss_bwd(const dslpg_logit_rows* rows, const dslpg_pair_terms* terms,
                                        const float* dloss, int64_t dloss_stride, const float* lse,
                                        const float* log_ratio, void* dlogits, int64_t dlogits_row_stride,
                                        cudaStream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* DSLPG_B200_H */
