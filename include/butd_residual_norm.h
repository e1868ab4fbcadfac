/*
 * butd_residual_norm.h -- C ABI of what stands between two blocks of a pre-norm / sandwich-norm layer stack (gfx950), one
 * kernel forward and one (plus the fold of its column sums) backward:
 *     t      = post_norm(x)                              (x: a block's output; LayerNorm, RMSNorm or none)
 *     stream = residual_scale * residual + gate * t      (gate: per channel, per sample and channel, per element, or none)
 *     normed = pre_norm(stream)                          (the next block's input; LayerNorm, RMSNorm or none)
 * The reference's layers are post-norm only, LayerNorm(residual + Dropout(block)) (models/encoder_decoder_layers.py:87-122):
 * include/butd_attention.h has that one.  Everything is computed in 32 bits from the tensors' values and rounded once at each
 * output; `normed` and the backward pass use the UNROUNDED stream (the backward pass rebuilds it from x, residual and gate,
 * which it has to read anyway, so the stream is not kept).  Column sums go through per-workgroup partial sums, no atomics:
 * bit-reproducible.
 *
 * Dense row-major tensors (rows, cols), 1 <= cols <= 8192; device pointers; asynchronous launches on `stream` that neither
 * allocate nor synchronise (hipGraph-capturable); 0 or a hipError_t.
 */
#ifndef BUTD_RESIDUAL_NORM_H
#define BUTD_RESIDUAL_NORM_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef void *butd_stream_t;

enum { BUTD_NORM_F32 = 0, BUTD_NORM_BF16 = 1, BUTD_NORM_F16 = 2 };
enum { BUTD_NORM_NONE = 0, BUTD_NORM_RMS = 1, BUTD_NORM_LAYER = 2 };
enum { BUTD_GATE_NONE = 0, BUTD_GATE_CHANNEL = 1, BUTD_GATE_SAMPLE = 2, BUTD_GATE_ELEMENT = 3 };
#define BUTD_NORM_MAX_COLS 8192

typedef struct {
  int x_dtype;                      /* of x, normed and their gradients */
  int stream_dtype;                 /* of residual, stream and their gradients: x_dtype or BUTD_NORM_F32 */
  int post_kind, pre_kind, gate_kind;
  int post_dtype, pre_dtype, gate_dtype;   /* of the norms' weight and bias, of gate: x_dtype or BUTD_NORM_F32 */
  long rows, rows_per_sample;       /* 0 .. 2^31 - 1; rows = samples * rows_per_sample (read for BUTD_GATE_SAMPLE only) */
  int cols;
  float residual_scale, post_eps, pre_eps;
  const void *x, *residual;         /* residual may be NULL (taken as 0) */
  const void *gate;                 /* (cols), (samples, cols) or (rows, cols) */
  const void *post_weight, *post_bias, *pre_weight, *pre_bias;   /* (cols); NULL = 1 / 0 */
  void *stream, *normed;            /* forward; normed with pre_kind only; stream may be NULL where it is x (no residual, gate,
                                     * post norm) */
  float *stats;                     /* (4, rows): mean and 1 / deviation of the post norm, of the pre norm; forward writes it
                                     * (NULL at inference), backward reads it */
  /* backward.  d_stream and d_normed may be NULL (no gradient arrives there), every output may be NULL (not wanted). */
  const void *d_stream, *d_normed;
  void *d_x, *d_residual, *d_gate, *d_post_weight, *d_post_bias, *d_pre_weight, *d_pre_bias;
} butd_residual_norm_args;

/* sizeof(butd_residual_norm_args) in the library: a caller that was compiled against another header finds out */
long butd_residual_norm_args_size(void);

/* Outputs share no memory with inputs or each other, here and in the backward call. */
int butd_residual_norm_fwd(const butd_residual_norm_args *args, butd_stream_t stream);

/* Bytes of device scratch (16-byte aligned) that the backward call with these arguments needs: a function of sizes, kinds
 * and of which outputs are NULL; negative: the arguments are refused (-hipErrorInvalidValue). */
long butd_residual_norm_bwd_workspace(const butd_residual_norm_args *args);
int butd_residual_norm_bwd(const butd_residual_norm_args *args, void *workspace, long workspace_bytes, butd_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* BUTD_RESIDUAL_NORM_H */
