"""The gated feed-forward block on the gfx950 kernels of include/butd_gated_ffn.h.

    y = W_down (act(W_gate x + b_gate) * (W_up x + b_up)) + b_down

-- the gated variant of the FFN of the encoder / decoder layers (models/encoder_decoder_layers.py:110-122,315-323 build
Linear-ReLU-Linear), for fp32, bf16 and fp16 tensors.  Forward is two launches (both projections, the activation and the
product are one kernel), with copies of odd rows and a split contraction's fold four; backward up to six.  Up to 16 rows -- a
token each of a few sequences; up to 64 where the weights are small -- take kernels that do nothing but stream the weights.
The precision is the tensors' own (``fused_attention.set_compute_dtype`` does not apply): 16-bit tensors are multiplied as they
are and accumulated in 32 bits, with biases, activation and its derivative; h and the gradients of its two factors are operands
of the next product and rounded to the tensors' type for it (fp16: an h beyond 65504 is infinite, as behind an fp16 linear
layer).  Checks, allocation and the autograd node are C++ (binding/blocks_aten.cpp): a small layer is bound by the host.
"""
from torch import nn

from .binding import build as _binding

ACTIVATIONS = {"silu": 0, "gelu": 1, "gelu_tanh": 2, "relu": 3, "sigmoid": 4}      # BUTD_FFN_*


def gated_ffn(x, w_gate, w_up, w_down, b_gate=None, b_up=None, b_down=None, activation="silu"):
    """``F.linear(act(F.linear(x, w_gate, b_gate)) * F.linear(x, w_up, b_up), w_down, b_down)``.

    x (..., width); w_gate, w_up (hidden, width); w_down (width, hidden); biases (hidden), (hidden), (width) or None; all of
    one dtype (float32, bfloat16, float16) on one GPU.  ``activation``: silu, gelu (erf), gelu_tanh, relu or sigmoid.  Any
    sizes from 1 on and any number of rows, none included; rows of a matrix may be strided (a slice of a wider buffer; of more
    dimensions such a slice is copied).  Widths or strides that are no multiple of 16 bytes cost a copy of that operand into
    padded rows, except for up to 64 rows in the forward pass.
    Under autocast all tensors are cast to its type first, as for ``F.linear``.
    Runs on the current stream, also under graph capture; first derivatives only.  RuntimeError on CPU tensors, on shapes or
    types that do not fit, under tracers (torch.jit.trace, make_fx), vmap and forward mode."""
    kind = ACTIVATIONS.get(activation)
    if kind is None:
        raise ValueError(f"gated_ffn: unknown activation {activation!r} (known: {', '.join(ACTIVATIONS)})")
    return _binding.blocks().gated_ffn(x, w_gate, w_up, w_down, b_gate, b_up, b_down, kind)


class GatedFeedForward(nn.Module):
    """The parameters of ``gated_ffn`` as three ``nn.Linear`` (``gate``, ``up``, ``down``): the gated counterpart of the layers'
    ``ffn`` Sequential.  forward(x (..., d_model)) -> (..., d_model), on the backend ``attention_blocks`` selects."""

    def __init__(self, d_model, dim_feedforward, activation="silu", bias=False, device=None, dtype=None):
        super().__init__()
        if activation not in ACTIVATIONS:
            raise ValueError(f"GatedFeedForward: unknown activation {activation!r} (known: {', '.join(ACTIVATIONS)})")
        kw = dict(bias=bias, device=device, dtype=dtype)
        self.gate, self.up = nn.Linear(d_model, dim_feedforward, **kw), nn.Linear(d_model, dim_feedforward, **kw)
        self.down = nn.Linear(dim_feedforward, d_model, **kw)
        self.activation = activation

    def forward(self, x):
        from . import attention_blocks
        return attention_blocks.gated_ffn(self, x)
