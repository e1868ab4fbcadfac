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
