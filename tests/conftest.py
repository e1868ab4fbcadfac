import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


# Tests that hold a value shown to be wrong: they stay as they were written and run, and are expected to fail.
SUPERSEDED = {
    "tests/test_gpu_residual_norm.py::test_default_epsilon_and_constant_rows":
        "takes the 16-bit type's epsilon for nn.RMSNorm(eps=None); the module itself uses float32's there "
        "(test_default_epsilon_against_the_module, test_default_epsilon_is_the_module_s_own)",
}


def pytest_collection_modifyitems(items):
    for item in items:
        if item.nodeid in SUPERSEDED:
            item.add_marker(pytest.mark.xfail(reason=SUPERSEDED[item.nodeid], raises=AssertionError, strict=True))


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a real MI355X (run with -m gpu on the GPU box)")


@pytest.fixture(scope="session")
def oracle():
    from oracle import pointnet2_oracle
    pointnet2_oracle.build()
    return pointnet2_oracle
