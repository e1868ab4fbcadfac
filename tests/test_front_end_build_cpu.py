"""How the compiled front ends are built and found (butd_detr_amd/binding/build.py), without a GPU."""
import pytest


def test_the_opt_out_compiles_no_front_end(monkeypatch):
    import __graft_entry__
    from butd_detr_amd import build as hip_build
    from butd_detr_amd.binding import build as aten_build
    called = []

    class Module:
        gated_ffn = furthest_point_sampling = print

    monkeypatch.setattr(hip_build, "build", lambda **kw: hip_build.LIB_PATH)
    monkeypatch.setattr(aten_build, "compile_blocks", lambda **kw: called.append("blocks") or Module)
    monkeypatch.setattr(aten_build, "load", lambda **kw: called.append("pointnet2") or Module)
    monkeypatch.setenv("BUTD_SKIP_ATEN", "1")
    __graft_entry__.build()
    assert called == []
    monkeypatch.setenv("BUTD_SKIP_ATEN", "0")
    __graft_entry__.build()
    assert sorted(called) == ["blocks", "pointnet2"]


@pytest.fixture
def copied(monkeypatch, tmp_path):
    """blocks() looks into a folder of its own, which holds the built front end and its stamp"""
    import os
    import shutil
    from butd_detr_amd.binding import build as aten_build
    aten_build.blocks()
    for ext in (".so", ".stamp"):
        shutil.copy(os.path.join(aten_build.BLOCKS_DIR, aten_build.BLOCKS + ext), tmp_path)
    monkeypatch.setattr(aten_build, "BLOCKS_DIR", str(tmp_path))
    monkeypatch.setattr(aten_build, "_blocks", None)
    monkeypatch.setattr(aten_build, "compile_blocks", lambda **kw: pytest.fail("compiled"))
    return aten_build, tmp_path


def test_a_front_end_of_other_sources_is_refused(copied):
    aten_build, folder = copied
    assert callable(aten_build.blocks().gated_ffn)
    for stale in ("0" * 40, None):
        aten_build._blocks = None
        stamp = folder / (aten_build.BLOCKS + ".stamp")
        stamp.write_text(stale) if stale else stamp.unlink()
        with pytest.raises(RuntimeError, match="built from other sources"):
            aten_build.blocks()


def test_the_stamp_covers_source_headers_flags_and_torch(monkeypatch, tmp_path):
    import torch
    from butd_detr_amd import build as hip_build
    from butd_detr_amd.binding import build as aten_build
    seen = [aten_build._stamp("blocks_aten.cpp")]
    headers = [h.rsplit("/", 1)[1] for h in hip_build._headers(aten_build.HERE + "/blocks_aten.cpp", [])]
    assert {"butd_gated_ffn.h", "butd_residual_norm.h"} <= set(headers)
    with monkeypatch.context() as m:
        m.setattr(aten_build, "FLAGS", aten_build.FLAGS + ["-g"])
        seen.append(aten_build._stamp("blocks_aten.cpp"))
    with monkeypatch.context() as m:
        m.setattr(torch, "__version__", "0.0")
        seen.append(aten_build._stamp("blocks_aten.cpp"))
    with monkeypatch.context() as m:
        (tmp_path / "blocks_aten.cpp").write_text(open(aten_build.HERE + "/blocks_aten.cpp").read() + "\n")
        m.setattr(aten_build, "HERE", str(tmp_path))
        seen.append(aten_build._stamp("blocks_aten.cpp"))
    with monkeypatch.context() as m:
        (tmp_path / "butd_gated_ffn.h").write_text("/* another */")
        m.setattr(hip_build, "INCLUDE", str(tmp_path))
        seen.append(aten_build._stamp("blocks_aten.cpp"))
    assert len(set(seen)) == len(seen)


def test_nothing_is_compiled_during_a_capture(copied, monkeypatch):
    import torch
    aten_build, folder = copied
    (folder / (aten_build.BLOCKS + ".so")).unlink()
    monkeypatch.setattr(torch.cuda, "is_initialized", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="being captured"):
        aten_build.blocks()


@pytest.mark.parametrize("name", ["GatedFfnArgs", "ResidualNormArgs"])
def test_a_library_with_another_argument_struct_is_refused(name, monkeypatch):
    import ctypes
    from butd_detr_amd import _hiplib

    class Longer(ctypes.Structure):
        _fields_ = getattr(_hiplib, name)._fields_ + [("one_more", ctypes.c_long)]

    monkeypatch.setattr(_hiplib, "_lib", None)
    monkeypatch.setattr(_hiplib, name, Longer)
    with pytest.raises(_hiplib.HipLibraryMissing, match="build it again"):
        _hiplib.load()


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("how", ["jit", "fx"])
def test_tracing_is_refused(how):
    """Neither block is a registered operator: a trace would hold the allocation of its output only."""
    import torch
    from torch.fx.experimental.proxy_tensor import make_fx
    from butd_detr_amd.gated_ffn import gated_ffn
    from butd_detr_amd.residual_norm import residual_norm
    w = torch.randn(12, 8)
    trace = (lambda f, v: torch.jit.trace(f, (v,))) if how == "jit" else (lambda f, v: make_fx(f)(v))
    for block in (lambda v: gated_ffn(v, w, w, w.t().contiguous()), lambda v: residual_norm(v, pre_norm=torch.nn.RMSNorm(8))[1]):
        with torch.no_grad(), pytest.raises(RuntimeError, match="cannot be traced"):
            trace(block, torch.randn(3, 8))
