// gated_ffn_bf16.hip -- the gated feed-forward block for __bf16 tensors (a unit of its own: the kernels compile side by side)
#include "gated_ffn_impl.h"

namespace ffn {
BUTD_FFN_TILES(__bf16, 256, 2, 4, 2, 4)
BUTD_FFN_TILES(__bf16, 128, 2, 2, 2, 2)
BUTD_FFN_TILES(__bf16, 64, 2, 2, 4, 1)
}  // namespace ffn

hipError_t butd_ffn_forward_bf16(const butd_gated_ffn_args &a, ffn::Arena &ws, bool run, hipStream_t stream) {
  return ffn::Block<__bf16>::forward(a, ws, run, stream);
}
hipError_t butd_ffn_backward_bf16(const butd_gated_ffn_args &a, ffn::Arena &ws, bool run, hipStream_t stream) {
  return ffn::Block<__bf16>::backward(a, ws, run, stream);
}
