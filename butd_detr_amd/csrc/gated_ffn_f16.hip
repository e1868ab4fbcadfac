// gated_ffn_f16.hip -- the gated feed-forward block for _Float16 tensors (a unit of its own: the kernels compile side by side)
#include "gated_ffn_impl.h"

namespace ffn {
BUTD_FFN_TILES(_Float16, 256, 2, 4, 2, 4)
BUTD_FFN_TILES(_Float16, 128, 2, 2, 2, 2)
BUTD_FFN_TILES(_Float16, 64, 2, 2, 4, 1)
}  // namespace ffn

hipError_t butd_ffn_forward_f16(const butd_gated_ffn_args &a, ffn::Arena &ws, bool run, hipStream_t stream) {
  return ffn::Block<_Float16>::forward(a, ws, run, stream);
}
hipError_t butd_ffn_backward_f16(const butd_gated_ffn_args &a, ffn::Arena &ws, bool run, hipStream_t stream) {
  return ffn::Block<_Float16>::backward(a, ws, run, stream);
}
