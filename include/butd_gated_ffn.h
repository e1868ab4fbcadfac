/*
 * butd_gated_ffn.h -- C ABI of the gated feed-forward block (gfx950 matrix cores; fp32, bf16, fp16 tensors).
 *
 * The gated variant of the position-wise FFN that the encoder / decoder layers use (models/encoder_decoder_layers.py:
 * 110-122,315-323,401-404 build the ungated one):
 *     a = x W_gate^T + b_gate      b = x W_up^T + b_up      h = act(a) * b      y = h W_down^T + b_down
 * and its gradients
 *     dh = dy W_down     da = dh * b * act'(a)     db = dh * act(a)     dx = da W_gate + db W_up
 *     dW_gate = da^T x   dW_up = db^T x            dW_down = dy^T h     bias gradients = column sums of da, db, dy
 * Both projections, the activation and the product are ONE kernel; so are dh with the activation's derivative, the two
 * products of dx, and the three weight gradients.  16-bit tensors: operands as they are, accumulation, biases, activation and
 * its derivative in 32 bits, h / da / db rounded once to the tensors' type where they are operands of the next product (fp16:
 * an h beyond 65504 is infinite, of da and db nothing below 2^-25 is left, as between the linear layers of an fp16 model);
 * the bias gradients are sums of the unrounded da and db.
 * No atomics: results are bit-reproducible.
 *
 * Row-major, last dimension contiguous, leading strides (ld_*) in ELEMENTS; device pointers; asynchronous launches on
 * `stream` that neither allocate nor synchronise (hipGraph-capturable); 0 or a hipError_t.
 */
#ifndef BUTD_GATED_FFN_H
#define BUTD_GATED_FFN_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef void *butd_stream_t;

enum { BUTD_FFN_F32 = 0, BUTD_FFN_BF16 = 1, BUTD_FFN_F16 = 2 };
enum { BUTD_FFN_SILU = 0, BUTD_FFN_GELU = 1, BUTD_FFN_GELU_TANH = 2, BUTD_FFN_RELU = 3, BUTD_FFN_SIGMOID = 4 };

typedef struct {
  int dtype, activation;
  long rows;                        /* tokens, 0 .. 2^27 */
  int width, hidden;                /* E, F: 1 .. 2^20 */
  const void *x;                    /* (rows, E) */
  const void *w_gate, *w_up;        /* (F, E) */
  const void *w_down;               /* (E, F) */
  long ld_x, ld_gate, ld_up, ld_down;
  const void *b_gate, *b_up;        /* (F), each may be NULL (forward only) */
  const void *b_down;               /* (E), may be NULL (forward only) */
  /* h (rows, ld_h) of the tensors' type; a, b (rows, ld_h) fp32, the pre-activations that the backward pass needs (both
   * NULL at inference).  Written by the forward, read by the backward call.  16-byte aligned, ld_h =
   * butd_gated_ffn_ld_hidden(dtype, F). */
  void *h;
  float *a, *b;
  long ld_h;
  void *y;                          /* (rows, E), forward */
  long ld_y;                        /* ld_y, ld_dx: up to 2^20 */
  /* backward: dy in; every other pointer may be NULL (that gradient is not computed).  Weight gradients are dense. */
  const void *dy;                   /* (rows, E) */
  long ld_dy;
  void *dx;                         /* (rows, E) */
  long ld_dx;
  void *dw_gate, *dw_up, *dw_down;
  void *db_gate, *db_up, *db_down;
} butd_gated_ffn_args;

/* sizeof(butd_gated_ffn_args) in the library: a caller that was compiled against another header finds out */
long butd_gated_ffn_args_size(void);

/* elements between the rows of h, a and b */
long butd_gated_ffn_ld_hidden(int dtype, int hidden);

/* Tuning hook: the tile (64, 128 or 256 rows and columns of a product; 256 is 128 for fp32) and the slices of the
 * contraction (1 .. 64, where a product can be split) of every following call of the process; (0, 0) returns to the built-in
 * rule.  A call reads it once.  The workspace functions follow it too: a call whose workspace was counted under another setting
 * that needs less refuses it.  Returns 0 or hipErrorInvalidValue. */
int butd_gated_ffn_set_tile(int tile, int split);

/* Bytes of device scratch (16-byte aligned) that the call with these arguments needs: a function of dtype, sizes, strides,
 * of the pointers' alignment and of which of them are NULL.  Negative: the arguments are refused (-hipErrorInvalidValue), by the
 * call too and before it launches anything -- also where a launch would have 2^32 threads or more: copies of operands (of above
 * 2^32 16-byte pieces), tiles that the hook forces. */
long butd_gated_ffn_fwd_workspace(const butd_gated_ffn_args *args);
long butd_gated_ffn_bwd_workspace(const butd_gated_ffn_args *args);

int butd_gated_ffn_fwd(const butd_gated_ffn_args *args, void *workspace, long workspace_bytes, butd_stream_t stream);
int butd_gated_ffn_bwd(const butd_gated_ffn_args *args, void *workspace, long workspace_bytes, butd_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* BUTD_GATED_FFN_H */
