import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA GPU (B200, sm_100a)")
    config.addinivalue_line("markers", "first_gpu_run: GPU test that has not yet passed on hardware")


def pytest_collection_modifyitems(config, items):
    # Tests still waiting for their first pass on a GPU run after the established suite, so
    # that a failure among them (under -x) cannot hide the results of the others. They
    # still run and still fail the suite. The no-allocation entry point's file
    # (test_zz_no_alloc.py) always runs last of all. The drop-in binary can only be built beside
    # the reference checkout; where it is missing its test fails behind all others.
    dropin = os.path.exists(os.path.join(ROOT, "minitensor_b200", "overlay", "_build", "dropin_test"))
    items.sort(key=lambda it: (not dropin and os.path.basename(str(it.fspath)) == "test_dropin_gpu.py",
                               os.path.basename(str(it.fspath)).startswith("test_zz_"),
                               it.get_closest_marker("first_gpu_run") is not None))


@pytest.fixture(scope="session")
def port():
    import oracle
    return oracle.Port()


@pytest.fixture(scope="session")
def ref():
    import oracle
    if not oracle.have_ref():
        pytest.skip("reference CPU build (oracle/_ref) not present")
    return oracle.Ref()


@pytest.fixture(scope="session")
def eng():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from minitensor_b200 import engine
    engine.lib()
    return engine
