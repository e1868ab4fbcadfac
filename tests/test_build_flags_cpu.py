"""What the units are compiled with, and what the set-abstraction unit becomes: no packed fp32 arithmetic."""
import os
import re
import subprocess

import pytest


def test_every_unit_is_built_without_packed_fp32_arithmetic():
    from butd_detr_amd import build
    for name in build._sources():
        flags = build._tu_flags(name)
        at = [i for i in range(len(flags)) if flags[i:i + 4] == build.NO_PACKED_F32]
        assert len(at) == 1, name


def test_the_set_abstraction_unit_has_no_packed_fp32_instruction(tmp_path):
    from butd_detr_amd import build
    if not os.path.exists(build.HIPCC):
        pytest.skip("no hipcc")
    out = tmp_path / "sa_ops.s"
    subprocess.run([build.HIPCC] + build.COMMON + build._tu_flags("sa_ops.hip")
                   + ["--cuda-device-only", "-S", os.path.join(build.CSRC, "sa_ops.hip"), "-o", str(out)],
                   check=True, capture_output=True, timeout=300)
    text = out.read_text()
    assert "v_fma" in text and not re.findall(r"v_pk_(?:add|mul|fma)_f32", text)
