// gated_ffn_f32.hip -- the gated feed-forward block for float tensors (a unit of its own: the kernels compile side by side)
#include "gated_ffn_impl.h"

namespace ffn {
BUTD_FFN_TILES(float, 128, 2, 2, 2, 2)
BUTD_FFN_TILES(float, 64, 2, 2, 4, 1)
}  // namespace ffn

hipError_t butd_ffn_forward_f32(const butd_gated_ffn_args &a, ffn::Arena &ws, bool run, hipStream_t stream) {
  return ffn::Block<float>::forward(a, ws, run, stream);
}
hipError_t butd_ffn_backward_f32(const butd_gated_ffn_args &a, ffn::Arena &ws, bool run, hipStream_t stream) {
  return ffn::Block<float>::backward(a, ws, run, stream);
}
