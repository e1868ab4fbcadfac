"""Norms around a block without a GPU: refusals, the stock-torch backend, the C entry points' checks."""
import ctypes

import pytest
import torch
from torch import nn


def test_cpu_tensors_are_refused():
    from butd_detr_amd.residual_norm import residual_norm
    with pytest.raises(RuntimeError, match="CPU not supported"):
        residual_norm(torch.randn(2, 3, 8), torch.randn(2, 3, 8), pre_norm=nn.LayerNorm(8))


@pytest.mark.parametrize("change, message", [
    (dict(x=torch.randn(2, 3, 8).double()), "not served"),
    (dict(x=torch.tensor(1.0)), "cols"),
    (dict(x=torch.randn(2, 3, 0)), "cols"),
    (dict(x=torch.randn(1, 8193)), "rows of up to 8192"),
    (dict(residual=torch.randn(2, 1, 8)), "residual must be"),
    (dict(residual=torch.randn(2, 3, 8).half()), "residual must be"),
    (dict(post_norm=nn.LayerNorm(4)), "must normalise"),
    (dict(pre_norm=nn.LayerNorm((3, 8))), "must normalise"),
    (dict(pre_norm=nn.BatchNorm1d(8)), "nn.LayerNorm or nn.RMSNorm"),
    (dict(post_norm=nn.RMSNorm(8).half()), "must be torch.float32 or float32"),
    (dict(gate=torch.randn(3, 8)), "gate must be"),
    (dict(gate=torch.randn(2, 3, 1)), "gate must be"),
    (dict(gate=torch.randn(8).half()), "gate must be"),
])
def test_refusals(change, message):
    from butd_detr_amd.residual_norm import residual_norm
    args = dict(x=torch.randn(2, 3, 8))
    args.update(change)
    with pytest.raises(RuntimeError, match=message):
        residual_norm(**args)


def test_torch_backend():
    from butd_detr_amd import attention_blocks as ab
    from butd_detr_amd.gated_ffn import GatedFeedForward
    torch.manual_seed(0)
    x, r = torch.randn(2, 3, 8), torch.randn(2, 3, 8)
    post, pre, ffn = nn.RMSNorm(8), nn.LayerNorm(8), GatedFeedForward(8, 12)
    prev = ab.get_backend()
    try:
        ab.set_backend("torch")
        for gate in (None, torch.randn(8), torch.randn(2, 8), torch.randn(2, 3, 8)):
            g = 1.0 if gate is None else gate[:, None] if gate.dim() == 2 else gate
            stream, normed = ab.residual_norm(x, r, post_norm=post, gate=gate, residual_scale=0.5, pre_norm=pre)
            torch.testing.assert_close(stream, 0.5 * r + g * post(x))
            torch.testing.assert_close(normed, pre(stream))
        assert ab.residual_norm(x)[1] is None
        stream, normed = ab.gated_ffn_block(ffn, x, pre_norm=pre, post_norm=post, next_norm=pre)
        torch.testing.assert_close(stream, x + post(ffn(pre(x))))
        again, none = ab.gated_ffn_block(ffn, stream, normed=normed)
        torch.testing.assert_close(again, stream + ffn(pre(stream)))
        assert none is None
        with pytest.raises(ValueError, match="one of"):
            ab.gated_ffn_block(ffn, x)
        with pytest.raises(ValueError, match="one of"):
            ab.gated_ffn_block(ffn, x, pre_norm=pre, normed=x)
    finally:
        ab.set_backend(prev)


def _filled():
    from butd_detr_amd._hiplib import ResidualNormArgs
    a = ResidualNormArgs()
    a.x_dtype, a.stream_dtype, a.post_dtype, a.pre_dtype, a.gate_dtype = 1, 0, 1, 0, 1
    a.post_kind, a.pre_kind, a.gate_kind = 1, 2, 2
    a.rows, a.rows_per_sample, a.cols = 12, 4, 24
    a.residual_scale, a.post_eps, a.pre_eps = 1.0, 1e-6, 1e-5
    a.x, a.residual, a.gate, a.stream, a.normed, a.stats = (4096 * (i + 1) for i in range(6))     # never dereferenced
    return a


def test_entry_points_check_their_arguments():
    from butd_detr_amd import _hiplib
    lib = _hiplib.load()
    need = lambda a: lib.butd_residual_norm_bwd_workspace(ctypes.byref(a))      # noqa: E731
    a = _filled()
    assert need(a) == 0
    a.post_weight, a.d_post_weight, a.d_gate = 4096, 4096, 4096
    assert need(a) > 0
    assert lib.butd_residual_norm_bwd(ctypes.byref(a), None, 0, None) != 0
    assert lib.butd_residual_norm_bwd(ctypes.byref(a), 4096, need(a) - 1, None) != 0
    assert lib.butd_residual_norm_bwd(ctypes.byref(a), 4104, need(a), None) != 0
    for field, value in [("x_dtype", 3), ("stream_dtype", 2), ("post_dtype", 2), ("gate_dtype", 2), ("post_kind", 3),
                         ("pre_kind", -1), ("gate_kind", 4), ("rows", -1), ("rows", 1 << 31), ("rows_per_sample", 0),
                         ("rows_per_sample", 5), ("cols", 0), ("cols", 8193), ("x", 0), ("x", 4097), ("gate", 0),
                         ("residual", 4098), ("stream", 0), ("normed", 0)]:
        a = _filled()
        setattr(a, field, value)
        assert lib.butd_residual_norm_fwd(ctypes.byref(a), None) != 0, field
    for field, value in [("x", 0), ("cols", 0), ("rows_per_sample", 5), ("d_gate", 4097)]:
        a = _filled()
        setattr(a, field, value)
        assert need(a) < 0, field
    a = _filled()
    a.stats = 0
    assert need(a) < 0                                                          # the post norm's statistics are missing


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("params", [None, torch.float32])
def test_default_epsilon_is_the_module_s_own(dtype, params):
    """What nn.RMSNorm(eps=None) adds to the mean square of its input, solved from its own output: rows of 2^-12, where an
    epsilon of the 16-bit types' would be thousands of mean squares."""
    from butd_detr_amd.residual_norm import _norm
    m = nn.RMSNorm(64, dtype=params or dtype)
    x = torch.full((1, 64), 2.0 ** -12, dtype=dtype)
    y = float(m(x)[0, 0])                                    # x / sqrt(x^2 + eps), rounded to at most 2^-9 of itself
    eps = _norm("pre_norm", m, 64)[3]
    want = 2.0 ** -12 / (2.0 ** -24 + eps) ** 0.5
    assert abs(y - want) <= want * (torch.finfo(dtype).eps / 2 + 2.0 ** -20), (y, want, eps)
    assert _norm("pre_norm", nn.RMSNorm(64, eps=0.5), 64)[3] == 0.5


@pytest.mark.parametrize("x_type, stream_type", [(torch.bfloat16, torch.float32), (torch.bfloat16, torch.bfloat16),
                                                 (torch.float16, torch.float32), (torch.float32, torch.float32)])
@pytest.mark.parametrize("params", [None, torch.float32])
@pytest.mark.parametrize("kind", [nn.LayerNorm, nn.RMSNorm])
def test_torch_backend_takes_and_rounds_what_the_kernels_do(kind, params, x_type, stream_type):
    """Parameters of x's type or float32 beside a stream of either type; one rounding an output, normed from the unrounded
    stream.  Inside 32 bits: 2^-18 of the largest term covers the row's sums."""
    from butd_detr_amd import attention_blocks as ab
    torch.manual_seed(2)
    cols = 48
    x, r = torch.randn(3, 4, cols).to(x_type), (4 * torch.randn(3, 4, cols)).to(stream_type)
    post, pre = kind(cols).to(params or x_type), kind(cols).to(params or x_type)
    gate = torch.rand(3, cols).to(x_type)
    prev = ab.get_backend()
    try:
        ab.set_backend("torch")
        stream, normed = ab.residual_norm(x, r, post_norm=post, gate=gate, residual_scale=0.75, pre_norm=pre)
        alone = ab.residual_norm(x, post_norm=post)
        assert ab.residual_norm(x, pre_norm=pre)[0] is x
    finally:
        ab.set_backend(prev)
    n1, n2 = (kind(cols, eps=m.eps if m.eps is not None else 2.0 ** -23).double() for m in (post, pre))
    s = 0.75 * r.double() + gate.double()[:, None] * n1(x.double())
    assert stream.dtype == stream_type and normed.dtype == x_type and alone[0].dtype == x_type and alone[1] is None
    for got, want in ((stream, s), (normed, n2(s)), (alone[0], n1(x.double()))):
        u = torch.finfo(got.dtype).eps / 2
        assert float(((got.double() - want).abs() - u * want.abs() - 2.0 ** -18 * (1 + u) * 16).max()) <= 0


def test_a_block_begins_a_stack_of_16_bit_blocks_on_a_32_bit_stream():
    from butd_detr_amd import attention_blocks as ab
    from butd_detr_amd.gated_ffn import GatedFeedForward
    torch.manual_seed(5)
    ffn, norm = GatedFeedForward(16, 24, "silu").bfloat16(), nn.RMSNorm(16)
    x = torch.randn(2, 3, 16)
    prev = ab.get_backend()
    try:
        ab.set_backend("torch")
        stream, normed = ab.gated_ffn_block(ffn, x, pre_norm=norm, next_norm=norm)
        by_hand = ab.gated_ffn_block(ffn, x, normed=norm(x).bfloat16(), next_norm=norm)
    finally:
        ab.set_backend(prev)
    assert stream.dtype == torch.float32 and normed.dtype == torch.bfloat16
    assert torch.equal(stream, by_hand[0]) and torch.equal(normed, by_hand[1])


def test_torch_backend_calls_other_modules_on_the_tensors_own_type():
    from butd_detr_amd import attention_blocks as ab

    class Scale(nn.Module):
        def __init__(self):
            super().__init__()
            self.w = nn.Linear(8, 8, bias=False, dtype=torch.bfloat16)

        def forward(self, v):
            return self.w(v)                                 # (raises on another type)

    torch.manual_seed(3)
    m, hooked, calls = Scale(), nn.LayerNorm(8), []
    hooked.register_forward_hook(lambda *a: calls.append(1))
    x, r = torch.randn(2, 3, 8).bfloat16(), torch.randn(2, 3, 8).bfloat16()
    prev = ab.get_backend()
    try:
        ab.set_backend("torch")
        stream, normed = ab.residual_norm(x, r, post_norm=m, pre_norm=m)
        assert stream.dtype == normed.dtype == torch.bfloat16
        assert torch.equal(stream, (r.float() + m(x).float()).bfloat16()) and torch.equal(normed, m(stream))
        ab.residual_norm(x.float(), r.float(), pre_norm=hooked)
        assert calls == [1]
    finally:
        ab.set_backend(prev)
