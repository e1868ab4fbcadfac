"""Norms before and after a block with its gate and residual scale, on the gfx950 kernels of include/butd_residual_norm.h:

    stream = residual_scale * residual + gate * post_norm(x)          normed = pre_norm(stream)

-- everything between two blocks of a pre-norm or sandwich-norm stack as one launch forward and two backward.  The
reference's layers are post-norm, LayerNorm(residual + Dropout(block)) (models/encoder_decoder_layers.py:87-122); those are
``fused_attention``'s.
"""
import ctypes

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import _hiplib
from ._hiplib import ResidualNormArgs

MAX_COLS = 8192                    # BUTD_NORM_MAX_COLS
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_NONE, _RMS, _LAYER = 0, 1, 2
_GATE_NONE, _GATE_CHANNEL, _GATE_SAMPLE, _GATE_ELEMENT = 0, 1, 2, 3


def _stream(t):
    return torch.cuda.current_stream(t.device).cuda_stream


def _ptr(t):
    return None if t is None else t.data_ptr()


def _norm(name, module, x, input_dtype):
    """(kind, weight, bias, eps) of an nn.LayerNorm / nn.RMSNorm / None"""
    if module is None:
        return _NONE, None, None, 0.0
    if isinstance(module, nn.LayerNorm):
        kind, bias = _LAYER, module.bias
    elif isinstance(module, nn.RMSNorm):
        kind, bias = _RMS, None
    else:
        raise RuntimeError(f"residual_norm: {name} must be an nn.LayerNorm or nn.RMSNorm, is {type(module).__name__}")
    if tuple(module.normalized_shape) != (x.shape[-1],):
        raise RuntimeError(f"residual_norm: {name} must normalise ({x.shape[-1]},), normalises {tuple(module.normalized_shape)}")
    eps = module.eps if module.eps is not None else torch.finfo(input_dtype).eps       # (nn.RMSNorm's default)
    for what, t in (("weight", module.weight), ("bias", bias)):
        if t is None:
            continue
        if t.dtype not in (x.dtype, torch.float32):
            raise RuntimeError(f"residual_norm: {name}.{what} must be {x.dtype} or float32, is {t.dtype}")
        if t.device != x.device:
            raise RuntimeError(f"residual_norm: {name}.{what} must be on {x.device}")
    if module.weight is not None and bias is not None and module.weight.dtype != bias.dtype:
        raise RuntimeError(f"residual_norm: {name}'s weight and bias must have one dtype")
    return kind, module.weight, bias, float(eps)


def _gate_kind(gate, x):
    if gate is None:
        return _GATE_NONE
    cols = x.shape[-1]
    if tuple(gate.shape) == (cols,):
        return _GATE_CHANNEL
    if gate.shape == x.shape:
        return _GATE_ELEMENT
    if x.dim() == 3 and tuple(gate.shape) in ((x.shape[0], cols), (x.shape[0], 1, cols)):
        return _GATE_SAMPLE
    raise RuntimeError(f"residual_norm: gate must be ({cols},), of x's shape, or (batch, {cols}) with x (batch, length, {cols}); "
                       f"is {tuple(gate.shape)} with x {tuple(x.shape)}")


class _Config:
    """What the two passes need besides tensors."""

    def __init__(self, x, residual, gate, post, pre, scale):
        self.shape, self.cols = x.shape, x.shape[-1]
        self.rows = x.numel() // self.cols
        self.dtype, self.stream_dtype = x.dtype, x.dtype if residual is None else residual.dtype
        self.gate_kind, self.scale = _gate_kind(gate, x), float(scale)
        self.plain = residual is None and gate is None and not post[0]      # the stream is x itself: not written again
        self.post_kind, self.post_eps, self.pre_kind, self.pre_eps = post[0], post[3], pre[0], pre[3]

    def args(self, x, residual, gate, w1, b1, w2, b2, stats):
        a = ResidualNormArgs()
        dtype = lambda *ts: _DTYPES[next((t.dtype for t in ts if t is not None), self.dtype)]      # noqa: E731
        a.x_dtype, a.stream_dtype = _DTYPES[self.dtype], _DTYPES[self.stream_dtype]
        a.post_kind, a.pre_kind, a.gate_kind = self.post_kind, self.pre_kind, self.gate_kind
        a.post_dtype, a.pre_dtype, a.gate_dtype = dtype(w1, b1), dtype(w2, b2), dtype(gate)
        a.rows, a.cols = self.rows, self.cols
        a.rows_per_sample = self.shape[1] if self.gate_kind == _GATE_SAMPLE else 1
        a.residual_scale, a.post_eps, a.pre_eps = self.scale, self.post_eps, self.pre_eps
        a.x, a.residual, a.gate = _ptr(x), _ptr(residual), _ptr(gate)
        a.post_weight, a.post_bias, a.pre_weight, a.pre_bias = _ptr(w1), _ptr(b1), _ptr(w2), _ptr(b2)
        a.stats = _ptr(stats)
        return a


def _forward(cfg, x, residual, gate, w1, b1, w2, b2, keep):
    stream = None if cfg.plain else torch.empty(cfg.shape, dtype=cfg.stream_dtype, device=x.device)
    normed = torch.empty(cfg.shape, dtype=cfg.dtype, device=x.device) if cfg.pre_kind else None
    stats = torch.empty((4, cfg.rows), dtype=torch.float32, device=x.device) if keep else None
    a = cfg.args(x, residual, gate, w1, b1, w2, b2, stats)
    a.stream, a.normed = _ptr(stream), _ptr(normed)
    with torch.cuda.device(x.device):
        _hiplib.check(_hiplib.load().butd_residual_norm_fwd(ctypes.byref(a), _stream(x)), "butd_residual_norm_fwd")
    return stream, normed, stats


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, cfg, x, residual, gate, w1, b1, w2, b2):
        ctx.set_materialize_grads(False)
        stream, normed, stats = _forward(cfg, x, residual, gate, w1, b1, w2, b2, True)
        ctx.save_for_backward(x, residual, gate, w1, b1, w2, b2, stats)
        ctx.cfg = cfg
        return (normed,) if cfg.plain else (stream,) if normed is None else (stream, normed)

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        cfg = ctx.cfg
        d_stream, d_normed = (None, grads[0]) if cfg.plain else (*grads, None)[:2]
        if d_stream is None and d_normed is None:
            return (None,) * 8
        *tensors, stats = ctx.saved_tensors
        x = tensors[0]
        d_stream, d_normed = (None if d is None else d.contiguous() for d in (d_stream, d_normed))
        new = torch.empty if cfg.rows else torch.zeros       # (no rows: the sums are zeros, a gate per sample's among them)
        grads = [new(t.shape, dtype=t.dtype, device=t.device) if t is not None and need else None
                 for t, need in zip(tensors, ctx.needs_input_grad[1:])]
        a = cfg.args(*tensors, stats)
        a.d_stream, a.d_normed = _ptr(d_stream), _ptr(d_normed)
        a.d_x, a.d_residual, a.d_gate, a.d_post_weight, a.d_post_bias, a.d_pre_weight, a.d_pre_bias = (_ptr(g) for g in grads)
        lib = _hiplib.load()
        with torch.cuda.device(x.device):
            need = lib.butd_residual_norm_bwd_workspace(ctypes.byref(a))
            _hiplib.check(-need if need < 0 else 0, "butd_residual_norm_bwd_workspace")
            ws = torch.empty(need, dtype=torch.uint8, device=x.device) if need else None
            _hiplib.check(lib.butd_residual_norm_bwd(ctypes.byref(a), _ptr(ws), need, _stream(x)), "butd_residual_norm_bwd")
        return (None, *grads)


def residual_norm(x, residual=None, *, post_norm=None, gate=None, residual_scale=1.0, pre_norm=None):
    """-> (stream, normed):  stream = residual_scale * residual + gate * post_norm(x),  normed = pre_norm(stream) or None.

    x (..., cols): a block's output, float32 / bfloat16 / float16, cols <= 8192; ``residual``: of x's shape and of x's dtype or
    float32 (the stream has its dtype; None counts as zeros, and without gate and post_norm too the stream IS x); ``post_norm``, ``pre_norm``: nn.LayerNorm / nn.RMSNorm over the
    last dimension, or None; ``gate``: (cols,), (batch, cols) for x (batch, length, cols), or of x's shape.  Parameters of the
    norms and the gate have x's dtype or float32.  Computed in 32 bits, each output rounded once; ``normed`` is the norm of
    the unrounded stream.  Runs on the current stream, also under graph capture; first derivatives only.  Raises on CPU tensors."""
    if x.dim() < 1 or x.shape[-1] < 1:
        raise RuntimeError("residual_norm: x must be (..., cols) with cols >= 1")
    if x.dtype not in _DTYPES:
        raise RuntimeError(f"residual_norm: {x.dtype} is not served (float32, bfloat16, float16)")
    if x.shape[-1] > MAX_COLS:
        raise RuntimeError(f"residual_norm: rows of up to {MAX_COLS} elements, x has {x.shape[-1]}")
    if x.numel() // x.shape[-1] > 0x7fffffff:
        raise RuntimeError("residual_norm: at most 2^31 - 1 rows")
    if residual is not None:
        if residual.shape != x.shape:
            raise RuntimeError(f"residual_norm: residual must be {tuple(x.shape)}, is {tuple(residual.shape)}")
        if residual.dtype not in (x.dtype, torch.float32):
            raise RuntimeError(f"residual_norm: residual must be {x.dtype} or float32, is {residual.dtype}")
    post = _norm("post_norm", post_norm, x, x.dtype)
    pre = _norm("pre_norm", pre_norm, x, x.dtype if residual is None else residual.dtype)
    if gate is not None and gate.dtype not in (x.dtype, torch.float32):
        raise RuntimeError(f"residual_norm: gate must be {x.dtype} or float32, is {gate.dtype}")
    for name, t in (("residual", residual), ("gate", gate)):
        if t is not None and t.device != x.device:
            raise RuntimeError(f"residual_norm: {name} must be on {x.device}")
    cfg = _Config(x, residual, gate, post, pre, residual_scale)
    if not x.is_cuda:
        raise RuntimeError("CPU not supported")
    if cfg.plain and not cfg.pre_kind:
        return x, None
    tensors = [None if t is None else t.contiguous() for t in (x, residual, gate, post[1], post[2], pre[1], pre[2])]
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        out = _ResidualNorm.apply(cfg, *tensors)
    else:
        stream, normed, _ = _forward(cfg, *tensors, False)
        out = (normed,) if cfg.plain else (stream, normed)
    return (x, out[0]) if cfg.plain else (*out, None)[:2]
