"""The gated feed-forward block without a GPU: refusals, the module on the stock-torch backend, the C entry points' checks
(they return an error before anything is launched)."""
import ctypes

import pytest
import torch
import torch.nn.functional as F


def _weights(width=8, hidden=12, dtype=torch.float32, biases=False):
    torch.manual_seed(0)
    w = [torch.randn(hidden, width, dtype=dtype), torch.randn(hidden, width, dtype=dtype),
         torch.randn(width, hidden, dtype=dtype)]
    if biases:
        w += [torch.randn(hidden, dtype=dtype), torch.randn(hidden, dtype=dtype), torch.randn(width, dtype=dtype)]
    return w


def test_cpu_tensors_are_refused():
    from butd_detr_amd.gated_ffn import gated_ffn
    with pytest.raises(RuntimeError, match="CPU not supported"):
        gated_ffn(torch.randn(3, 8), *_weights())


@pytest.mark.parametrize("change, message", [
    (dict(activation="swish"), "unknown activation"),
    (dict(x=torch.randn(3, 9)), "x must be"),
    (dict(w_up=torch.randn(8, 12)), "w_up must be"),
    (dict(w_down=torch.randn(12, 8)), "w_down must be"),
    (dict(w_gate=torch.randn(12)), "w_gate"),
    (dict(w_gate=torch.randn(0, 8)), "at least 1"),
    (dict(b_gate=torch.randn(8)), "b_gate must be"),
    (dict(b_down=torch.randn(12)), "b_down must be"),
    (dict(x=torch.randn(3, 8).double()), "not served"),
    (dict(x=torch.randn(3, 8).bfloat16()), "must be torch.bfloat16"),
    (dict(b_up=torch.randn(12).half()), "must be torch.float32"),
])
def test_refusals(change, message):
    from butd_detr_amd.gated_ffn import gated_ffn
    g, u, d = _weights()
    args = dict(x=torch.randn(3, 8), w_gate=g, w_up=u, w_down=d)
    args.update(change)
    with pytest.raises((RuntimeError, ValueError), match=message):
        gated_ffn(**args)


@pytest.mark.parametrize("activation", ["silu", "gelu", "gelu_tanh", "relu", "sigmoid"])
@pytest.mark.parametrize("bias", [False, True])
def test_module_on_the_torch_backend(activation, bias):
    from butd_detr_amd import attention_blocks as ab
    from butd_detr_amd.gated_ffn import GatedFeedForward
    torch.manual_seed(1)
    ffn = GatedFeedForward(8, 12, activation, bias=bias)
    assert [n for n, _ in ffn.named_parameters()] == [f"{m}.{p}" for m in ("gate", "up", "down")
                                                      for p in (("weight", "bias") if bias else ("weight",))]
    x = torch.randn(2, 3, 8)
    act = {"silu": F.silu, "gelu": F.gelu, "gelu_tanh": lambda a: F.gelu(a, approximate="tanh"), "relu": torch.relu,
           "sigmoid": torch.sigmoid}[activation]
    want = F.linear(act(F.linear(x, ffn.gate.weight, ffn.gate.bias)) * F.linear(x, ffn.up.weight, ffn.up.bias),
                    ffn.down.weight, ffn.down.bias)
    prev = ab.get_backend()
    try:
        ab.set_backend("torch")
        assert torch.equal(ffn(x), want)
    finally:
        ab.set_backend(prev)
    with pytest.raises(ValueError, match="unknown activation"):
        GatedFeedForward(8, 12, "swish")


def _filled(lib, dtype=1, rows=4, width=16, hidden=24):
    from butd_detr_amd._hiplib import GatedFfnArgs
    a = GatedFfnArgs()
    a.dtype, a.activation, a.rows, a.width, a.hidden = dtype, 0, rows, width, hidden
    a.x, a.w_gate, a.w_up, a.w_down, a.h, a.y = (4096 * (i + 1) for i in range(6))     # never dereferenced
    a.ld_x = a.ld_gate = a.ld_up = a.ld_y = width
    a.ld_down, a.ld_h = hidden, lib.butd_gated_ffn_ld_hidden(dtype, hidden)
    return a


def test_entry_points_check_their_arguments():
    from butd_detr_amd import _hiplib
    lib = _hiplib.load()
    assert lib.butd_gated_ffn_ld_hidden(0, 5) == 8 and lib.butd_gated_ffn_ld_hidden(1, 5) == 8
    assert lib.butd_gated_ffn_ld_hidden(2, 2051) == 2056
    fwd = lambda a: lib.butd_gated_ffn_fwd_workspace(ctypes.byref(a))      # noqa: E731
    bwd = lambda a: lib.butd_gated_ffn_bwd_workspace(ctypes.byref(a))      # noqa: E731
    assert fwd(_filled(lib)) == 0                                          # few aligned rows: no scratch
    assert fwd(_filled(lib, rows=100)) >= 0
    odd = _filled(lib, rows=100, width=17)
    assert fwd(odd) > 0                                                    # copies with padded rows
    for field, value in [("dtype", 3), ("dtype", -1), ("activation", 5), ("rows", -1), ("rows", 1 << 31), ("width", 0),
                         ("hidden", 0), ("ld_x", 15), ("ld_gate", 15), ("ld_down", 23), ("ld_h", 25), ("ld_y", 15),
                         ("x", 0), ("x", 4097), ("w_gate", 0), ("w_down", 0), ("y", 0), ("h", 0), ("h", 4104), ("a", 4096),
                         ("b_gate", 4097)]:
        a = _filled(lib)
        setattr(a, field, value)
        assert fwd(a) < 0, field
        assert lib.butd_gated_ffn_fwd(ctypes.byref(a), None, 0, None) != 0, field
    a = _filled(lib)
    a.a, a.b, a.dy, a.dx, a.ld_dy, a.ld_dx = 4096, 8192, 12288, 16384, 16, 16
    assert bwd(a) > 0
    assert lib.butd_gated_ffn_bwd(ctypes.byref(a), None, 0, None) != 0     # no workspace
    assert lib.butd_gated_ffn_bwd(ctypes.byref(a), 4096, bwd(a) - 1, None) != 0
    assert lib.butd_gated_ffn_bwd(ctypes.byref(a), 4104, bwd(a), None) != 0
    for field, value in [("a", 0), ("dy", 0), ("ld_dy", 15), ("ld_dx", 15), ("dw_gate", 4097)]:
        b = _filled(lib)
        b.a, b.b, b.dy, b.dx, b.ld_dy, b.ld_dx = 4096, 8192, 12288, 16384, 16, 16
        setattr(b, field, value)
        assert bwd(b) < 0, field
    for tile, split in [(32, 1), (64, 0), (64, 65), (0, 1), (-64, 1)]:
        assert lib.butd_gated_ffn_set_tile(tile, split) != 0
    assert lib.butd_gated_ffn_set_tile(0, 0) == 0


def test_size_limits():
    from butd_detr_amd import _hiplib
    lib = _hiplib.load()
    fwd = lambda a: lib.butd_gated_ffn_fwd_workspace(ctypes.byref(a))      # noqa: E731
    assert fwd(_filled(lib, rows=1 << 27)) >= 0 and fwd(_filled(lib, rows=(1 << 27) + 1)) < 0
    most = 1 << 20
    assert fwd(_filled(lib, width=most)) >= 0 and fwd(_filled(lib, width=most + 1)) < 0
    assert fwd(_filled(lib, hidden=most)) >= 0 and fwd(_filled(lib, hidden=most + 1)) < 0
    a = _filled(lib)
    a.ld_y = most + 1
    assert fwd(a) < 0


_HOOK_WHILE_PLANNING = """
import ctypes, sys, threading
sys.path.insert(0, {root!r})
from butd_detr_amd import _hiplib
from tests.test_gated_ffn_cpu import _filled
lib = _hiplib.load()
a = _filled(lib, rows=4096, width=512, hidden=2048)
a.a, a.b, a.dy, a.dx, a.ld_dy, a.ld_dx, a.dw_gate, a.dw_up, a.dw_down = 4096, 8192, 12288, 16384, 512, 512, 4096, 4096, 4096
need = lambda: lib.butd_gated_ffn_bwd_workspace(ctypes.byref(a))
known = {{need()}}
lib.butd_gated_ffn_set_tile(64, 48)
known.add(need())
assert len(known) == 2 and min(known) > 0
done = threading.Event()
def turn():
    while not done.is_set():
        lib.butd_gated_ffn_set_tile(0, 0)
        lib.butd_gated_ffn_set_tile(64, 48)
threads = [threading.Thread(target=turn) for _ in range(2)]
for t in threads:
    t.start()
seen = {{need() for _ in range(200000)}}
done.set()
for t in threads:
    t.join()
assert seen <= known, (seen, known)
"""


def test_a_plan_is_made_of_one_setting_of_the_tuning_hook():
    """The hook set by other threads while a plan is made: the plan is the one setting's or the other's, never a mixture."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    out = subprocess.run([sys.executable, "-c", _HOOK_WHILE_PLANNING.format(root=root)], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0, (out.returncode, out.stderr[-1000:])


def test_what_a_launch_cannot_hold_is_refused_by_the_query():
    """2^27 rows: the rule takes tiles whose launch has room for them; the smallest tiles, forced, and copies of odd rows are
    refused by the workspace query as by the call, which launches nothing."""
    from butd_detr_amd import _hiplib
    lib = _hiplib.load()
    invalid = 1                                                            # hipErrorInvalidValue

    def refused(backward, **kw):
        a = _filled(lib, rows=1 << 27, **kw)
        if backward:
            a.a, a.b, a.dy, a.dx, a.ld_dy, a.ld_dx, a.dw_gate = 4096, 8192, 12288, 16384, kw["width"], kw["width"], 4096
        query, call = ((lib.butd_gated_ffn_bwd_workspace, lib.butd_gated_ffn_bwd) if backward
                       else (lib.butd_gated_ffn_fwd_workspace, lib.butd_gated_ffn_fwd))
        need = query(ctypes.byref(a))
        assert need >= 0 or need == -invalid
        if need < 0:
            assert call(ctypes.byref(a), 4096, 1 << 62, None) == invalid   # (a call that is accepted would launch: not made)
        return need < 0
    for dtype in (0, 1, 2):
        for backward in (False, True):
            for width, hidden in ((16, 512), (16, 4096), (512, 16), (768, 256)):
                # the largest tile: 128 rows x 64 columns of h (128 of the other products) on 256 threads, fp32; twice each, 16 bits
                n = 1 if dtype == 0 else 2
                columns = max(-(-hidden // ((128 if backward else 64) * n)), -(-width // (128 * n)))
                threads = (1 << 27) // (128 * n) * columns * 256 * n
                assert refused(backward, dtype=dtype, width=width, hidden=hidden) == (threads >= 1 << 32), (dtype, backward, width, hidden)
            assert refused(backward, dtype=dtype, width=777, hidden=256), (dtype, backward)
    lib.butd_gated_ffn_set_tile(64, 1)
    try:
        for backward in (False, True):
            assert refused(backward, width=16, hidden=1024)
            assert not refused(backward, width=16, hidden=24)
    finally:
        lib.butd_gated_ffn_set_tile(0, 0)
