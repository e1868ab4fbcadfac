"""Norms before and after a block with its gate and residual scale, on the gfx950 kernels of include/butd_residual_norm.h:

    stream = residual_scale * residual + gate * post_norm(x)          normed = pre_norm(stream)

-- everything between two blocks of a pre-norm or sandwich-norm stack as one launch forward and two backward.  The
reference's layers are post-norm, LayerNorm(residual + Dropout(block)) (models/encoder_decoder_layers.py:87-122); those are
``fused_attention``'s.  Checks, allocation and the autograd node are C++ (binding/blocks_aten.cpp).
"""
import torch
from torch import nn

from .binding import build as _binding

_NONE, _RMS, _LAYER = 0, 1, 2      # BUTD_NORM_*
# nn.RMSNorm(eps=None): the epsilon of the type its statistics are computed in, 32 bits for 16-bit tensors too
_DEFAULT_EPS = torch.finfo(torch.float32).eps


def _norm(name, module, cols):
    """(weight, bias, kind, eps) of an nn.LayerNorm / nn.RMSNorm / None"""
    if module is None:
        return None, None, _NONE, 0.0
    if isinstance(module, nn.LayerNorm):
        kind, bias = _LAYER, module.bias
    elif isinstance(module, nn.RMSNorm):
        kind, bias = _RMS, None
    else:
        raise RuntimeError(f"residual_norm: {name} must be an nn.LayerNorm or nn.RMSNorm, is {type(module).__name__}")
    if tuple(module.normalized_shape) != (cols,):
        raise RuntimeError(f"residual_norm: {name} must normalise ({cols},), normalises {tuple(module.normalized_shape)}")
    return module.weight, bias, kind, _DEFAULT_EPS if module.eps is None else module.eps


def residual_norm(x, residual=None, *, post_norm=None, gate=None, residual_scale=1.0, pre_norm=None):
    """-> (stream, normed):  stream = residual_scale * residual + gate * post_norm(x),  normed = pre_norm(stream) or None.

    x (..., cols): a block's output, float32 / bfloat16 / float16, cols <= 8192; ``residual``: of x's shape and of x's dtype or
    float32 (the stream has its dtype; None counts as zeros, and without gate and post_norm too the stream IS x); ``post_norm``,
    ``pre_norm``: nn.LayerNorm / nn.RMSNorm over the last dimension (an ``eps`` of None is float32's, as the module takes it), or
    None; ``gate``: (cols,), (batch, cols) for x (batch, length, cols), or of x's shape.  Parameters of the norms and the gate
    have x's dtype or float32.  Computed in 32 bits, each output rounded once; ``normed`` is the norm of the unrounded stream.
    Runs on the current stream, also under graph capture; first derivatives only.  RuntimeError on CPU tensors, on shapes or types that do not fit, under tracers (torch.jit.trace,
    make_fx), vmap and forward mode."""
    cols = x.shape[-1] if x.dim() else 0
    w1, b1, post, post_eps = _norm("post_norm", post_norm, cols)
    w2, b2, pre, pre_eps = _norm("pre_norm", pre_norm, cols)
    stream, normed = _binding.blocks().residual_norm(x, residual, gate, w1, b1, w2, b2, post, pre, post_eps, pre_eps, residual_scale)
    return (x if stream is None else stream), normed
