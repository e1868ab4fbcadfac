"""The gated feed-forward block on the gfx950 kernels of include/butd_gated_ffn.h.

    y = W_down (act(W_gate x + b_gate) * (W_up x + b_up)) + b_down

-- the gated variant of the FFN of the encoder / decoder layers (models/encoder_decoder_layers.py:110-122,315-323 build
Linear-ReLU-Linear), for fp32, bf16 and fp16 tensors.  Forward is two launches (both projections, the activation and the
product are one kernel), backward three to six.  Without gradients, up to 64 rows -- a token each of a few sequences -- take
kernels that do nothing but stream the weights.  The precision is the tensors' own (``fused_attention.set_compute_dtype`` does
not apply): 16-bit operands, everything between two products in 32 bits.
"""
import ctypes

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import _hiplib
from ._hiplib import GatedFfnArgs

ACTIVATIONS = {"silu": 0, "gelu": 1, "gelu_tanh": 2, "relu": 3, "sigmoid": 4}
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _stream(t):
    return torch.cuda.current_stream(t.device).cuda_stream


def _ptr(t):
    return None if t is None else t.data_ptr()


def _rows(t):
    """(..., C) as rows: a (rows, C) view with a contiguous last dimension, or a contiguous copy where there is none."""
    cols = t.shape[-1]
    if t.dim() == 2 and t.shape[0] > 1 and t.stride(1) == 1 and t.stride(0) >= cols:
        return t
    return t.contiguous().view(-1, cols)


def _ld(rows):
    return rows.stride(0) if rows.shape[0] > 1 else rows.shape[1]


def _check(x, w_gate, w_up, w_down, b_gate, b_up, b_down, activation):
    if activation not in ACTIVATIONS:
        raise ValueError(f"gated_ffn: unknown activation {activation!r} (known: {', '.join(ACTIVATIONS)})")
    if x.dim() < 1 or w_gate.dim() != 2:
        raise RuntimeError("gated_ffn: x must be (..., width) and w_gate (hidden, width)")
    hidden, width = w_gate.shape
    if width < 1 or hidden < 1:
        raise RuntimeError("gated_ffn: width and hidden must be at least 1")
    want = {"x": (x, tuple(x.shape[:-1]) + (width,)), "w_up": (w_up, (hidden, width)), "w_down": (w_down, (width, hidden)),
            "b_gate": (b_gate, (hidden,)), "b_up": (b_up, (hidden,)), "b_down": (b_down, (width,)),
            "w_gate": (w_gate, (hidden, width))}
    if x.dtype not in _DTYPES:
        raise RuntimeError(f"gated_ffn: {x.dtype} is not served (float32, bfloat16, float16)")
    for name, (t, shape) in want.items():
        if t is None:
            continue
        if tuple(t.shape) != shape:
            raise RuntimeError(f"gated_ffn: {name} must be {shape}, is {tuple(t.shape)}")
        if t.dtype != x.dtype:
            raise RuntimeError(f"gated_ffn: {name} must be {x.dtype} as x is, is {t.dtype}")
        if t.device != x.device:
            raise RuntimeError(f"gated_ffn: {name} must be on {x.device}")
    if not x.is_cuda:
        raise RuntimeError("CPU not supported")
    if x.numel() // width > 0x7fffffff:
        raise RuntimeError("gated_ffn: at most 2^31 - 1 rows")


def _args(rows, x, w_gate, w_up, w_down, activation):
    a = GatedFfnArgs()
    a.dtype, a.activation = _DTYPES[x.dtype], activation
    a.rows, a.width, a.hidden = rows, w_gate.shape[1], w_gate.shape[0]
    a.x, a.ld_x = x.data_ptr(), _ld(x)
    a.w_gate, a.ld_gate = w_gate.data_ptr(), _ld(w_gate)
    a.w_up, a.ld_up = w_up.data_ptr(), _ld(w_up)
    a.w_down, a.ld_down = w_down.data_ptr(), _ld(w_down)
    return a


def _call(name, args, ref):
    lib = _hiplib.load()
    with torch.cuda.device(ref.device):
        need = getattr(lib, name + "_workspace")(ctypes.byref(args))
        _hiplib.check(-need if need < 0 else 0, name + "_workspace")
        ws = torch.empty(need, dtype=torch.uint8, device=ref.device) if need else None
        _hiplib.check(getattr(lib, name)(ctypes.byref(args), _ptr(ws), need, _stream(ref)), name)


def _forward(x, w_gate, w_up, w_down, b_gate, b_up, b_down, activation, keep):
    """-> y (rows, width), and with ``keep`` what the backward pass reads: h (rows, ld), a | b (2, rows, ld) in fp32"""
    rows, width = x.shape
    a = _args(rows, x, w_gate, w_up, w_down, activation)
    a.b_gate, a.b_up, a.b_down = _ptr(b_gate), _ptr(b_up), _ptr(b_down)
    a.ld_h = _hiplib.load().butd_gated_ffn_ld_hidden(a.dtype, a.hidden)
    h = torch.empty((rows, a.ld_h), dtype=x.dtype, device=x.device)
    ab = torch.empty((2, rows, a.ld_h), dtype=torch.float32, device=x.device) if keep else None
    y = torch.empty((rows, width), dtype=x.dtype, device=x.device)
    a.h, a.y, a.ld_y = h.data_ptr(), y.data_ptr(), width
    if keep and rows:
        a.a, a.b = ab[0].data_ptr(), ab[1].data_ptr()
    _call("butd_gated_ffn_fwd", a, x)
    return y, h, ab


class _GatedFfn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, b_gate, b_up, b_down, activation):
        xr, wg, wu, wd = _rows(x), _rows(w_gate), _rows(w_up), _rows(w_down)
        bg, bu, bd = (None if b is None else b.contiguous() for b in (b_gate, b_up, b_down))
        y, h, ab = _forward(xr, wg, wu, wd, bg, bu, bd, activation, True)
        ctx.save_for_backward(xr, wg, wu, wd, h, ab)
        ctx.activation, ctx.shape = activation, x.shape
        return y.view(x.shape)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w_gate, w_up, w_down, h, ab = ctx.saved_tensors
        dy = _rows(dy)
        rows, width = x.shape
        hidden = w_gate.shape[0]
        a = _args(rows, x, w_gate, w_up, w_down, ctx.activation)
        a.h, a.ld_h, a.dy, a.ld_dy = h.data_ptr(), h.shape[1], dy.data_ptr(), _ld(dy)
        if rows:
            a.a, a.b = ab[0].data_ptr(), ab[1].data_ptr()
        shapes = [(rows, width), (hidden, width), (hidden, width), (width, hidden), (hidden,), (hidden,), (width,)]
        grads = [torch.empty(s, dtype=x.dtype, device=x.device) if need else None
                 for s, need in zip(shapes, ctx.needs_input_grad)]
        a.dx, a.dw_gate, a.dw_up, a.dw_down, a.db_gate, a.db_up, a.db_down = (_ptr(g) for g in grads)
        a.ld_dx = width
        _call("butd_gated_ffn_bwd", a, x)
        if grads[0] is not None:
            grads[0] = grads[0].view(ctx.shape)
        return (*grads, None)


def gated_ffn(x, w_gate, w_up, w_down, b_gate=None, b_up=None, b_down=None, activation="silu"):
    """``F.linear(act(F.linear(x, w_gate, b_gate)) * F.linear(x, w_up, b_up), w_down, b_down)``.

    x (..., width); w_gate, w_up (hidden, width); w_down (width, hidden); biases (hidden), (hidden), (width) or None; all of
    one dtype (float32, bfloat16, float16) on one GPU.  ``activation``: silu, gelu (erf), gelu_tanh, relu or sigmoid.  Any
    sizes from 1 on and any number of rows, none included; rows may be strided (a slice of a wider buffer).  Widths or strides
    that are no multiple of 16 bytes cost a copy of that operand into padded rows, except for up to 64 rows in the forward pass.
    Runs on the current stream, also under graph capture; first derivatives only.  Raises on CPU tensors."""
    _check(x, w_gate, w_up, w_down, b_gate, b_up, b_down, activation)
    tensors = (x, w_gate, w_up, w_down, b_gate, b_up, b_down)
    kind = ACTIVATIONS[activation]
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        return _GatedFfn.apply(*tensors, kind)
    bias = [None if b is None else b.contiguous() for b in (b_gate, b_up, b_down)]
    return _forward(_rows(x), _rows(w_gate), _rows(w_up), _rows(w_down), *bias, kind, False)[0].view(x.shape)


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
