// gated_ffn_ops.hip -- entry points of include/butd_gated_ffn.h: checks of the arguments, dispatch on the tensors' type.
#include "gated_ffn_impl.h"

#include <atomic>

#define BUTD_FFN_DECLARE(T)                                                                            \
  hipError_t butd_ffn_forward_##T(const butd_gated_ffn_args &, ffn::Arena &, bool, hipStream_t);       \
  hipError_t butd_ffn_backward_##T(const butd_gated_ffn_args &, ffn::Arena &, bool, hipStream_t);
BUTD_FFN_DECLARE(f32)
BUTD_FFN_DECLARE(bf16)
BUTD_FFN_DECLARE(f16)

namespace {

std::atomic<int> tuned{0};               // butd_gated_ffn_set_tile: tile + 1024 split as one value
ffn::Forced forced() {
  const int v = tuned.load(std::memory_order_relaxed);
  return ffn::Forced{v & 1023, v >> 10};
}

constexpr long kMostRows = 1L << 27;     // (rows and products of them by 16 bytes a row fit the plan's integers)

bool valid(const butd_gated_ffn_args *a, bool backward) {
  if (!a || a->dtype < BUTD_FFN_F32 || a->dtype > BUTD_FFN_F16) return false;
  if (a->activation < BUTD_FFN_SILU || a->activation > BUTD_FFN_SIGMOID) return false;
  if (a->rows < 0 || a->rows > kMostRows || a->width < 1 || a->hidden < 1) return false;
  // (offsets inside a tile's 256 rows have to fit 31 bits)
  constexpr long kMost = 1L << 20;
  if (a->width > kMost || a->hidden > kMost) return false;
  if (a->ld_gate < a->width || a->ld_up < a->width || a->ld_down < a->hidden) return false;
  if (a->ld_h != butd_gated_ffn_ld_hidden(a->dtype, a->hidden)) return false;
  if (a->rows == 0) return true;
  const uintptr_t size = a->dtype == BUTD_FFN_F32 ? 4 : 2;
  const void *const elements[] = {a->x, a->w_gate, a->w_up, a->w_down, a->b_gate, a->b_up, a->b_down, a->y, a->dy, a->dx,
                                  a->dw_gate, a->dw_up, a->dw_down, a->db_gate, a->db_up, a->db_down};
  for (const void *p : elements)
    if ((uintptr_t)p % size) return false;
  if (!a->x || a->ld_x < a->width || !a->w_gate || !a->w_up || !a->w_down) return false;
  if (!a->h || ((uintptr_t)a->h | (uintptr_t)a->a | (uintptr_t)a->b) & 15) return false;
  if ((a->a == nullptr) != (a->b == nullptr)) return false;
  if (!backward) return a->y && a->ld_y >= a->width && a->ld_y <= kMost;
  return a->a && a->dy && a->ld_dy >= a->width && (!a->dx || (a->ld_dx >= a->width && a->ld_dx <= kMost));
}

hipError_t dispatch(const butd_gated_ffn_args &a, ffn::Arena &ws, bool run, hipStream_t stream, bool backward) {
  switch (a.dtype) {
    case BUTD_FFN_F32: return backward ? butd_ffn_backward_f32(a, ws, run, stream) : butd_ffn_forward_f32(a, ws, run, stream);
    case BUTD_FFN_BF16: return backward ? butd_ffn_backward_bf16(a, ws, run, stream) : butd_ffn_forward_bf16(a, ws, run, stream);
    default: return backward ? butd_ffn_backward_f16(a, ws, run, stream) : butd_ffn_forward_f16(a, ws, run, stream);
  }
}

long workspace(const butd_gated_ffn_args *a, bool backward, ffn::Forced setting) {
  if (!valid(a, backward)) return -(long)hipErrorInvalidValue;
  ffn::Arena ws{nullptr, setting};
  const hipError_t err = dispatch(*a, ws, false, nullptr, backward);
  return err == hipSuccess ? ws.used : -(long)err;
}

int execute(const butd_gated_ffn_args *a, void *ws_ptr, long ws_bytes, butd_stream_t stream, bool backward) {
  const ffn::Forced setting = forced();
  const long need = workspace(a, backward, setting);
  if (need < 0) return (int)-need;
  if (need > 0 && (!ws_ptr || ws_bytes < need || ((uintptr_t)ws_ptr & 15))) return (int)hipErrorInvalidValue;
  ffn::Arena ws{(char *)ws_ptr, setting};
  return (int)dispatch(*a, ws, true, (hipStream_t)stream, backward);
}

}  // namespace

extern "C" {

long butd_gated_ffn_args_size(void) { return (long)sizeof(butd_gated_ffn_args); }
long butd_gated_ffn_ld_hidden(int dtype, int hidden) {
  const long vec = dtype == BUTD_FFN_F32 ? 4 : 8;
  return ((long)hidden + vec - 1) / vec * vec;
}
int butd_gated_ffn_set_tile(int tile, int split) {
  if (tile == 0 && split == 0) {
    tuned.store(0, std::memory_order_relaxed);
    return 0;
  }
  if ((tile != 64 && tile != 128 && tile != 256) || split < 1 || split > 64) return (int)hipErrorInvalidValue;
  tuned.store(tile + 1024 * split, std::memory_order_relaxed);
  return 0;
}
long butd_gated_ffn_fwd_workspace(const butd_gated_ffn_args *args) { return workspace(args, false, forced()); }
long butd_gated_ffn_bwd_workspace(const butd_gated_ffn_args *args) { return workspace(args, true, forced()); }
int butd_gated_ffn_fwd(const butd_gated_ffn_args *args, void *ws, long ws_bytes, butd_stream_t stream) {
  return execute(args, ws, ws_bytes, stream, false);
}
int butd_gated_ffn_bwd(const butd_gated_ffn_args *args, void *ws, long ws_bytes, butd_stream_t stream) {
  return execute(args, ws, ws_bytes, stream, true);
}

}  // extern "C"
