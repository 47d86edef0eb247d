import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a gfx950 GPU (runs on the MI355X box)")
    config.addinivalue_line("markers", "slow: long-running CPU test")


# Tests that ask for what is wrong. They run, and have to fail.
WRONG = {
    "test_m0_is_written_only_by_the_dma_asm":
        "asks for each load to LDS directly behind the write of M0, where the instruction set manual asks for a wait "
        "state between them; test_lds_loads.py asks for that and for the rest of what this one does",
}


def pytest_collection_modifyitems(items):
    for item in items:
        if item.name in WRONG:
            item.add_marker(pytest.mark.xfail(reason=WRONG[item.name], raises=AssertionError, strict=True))


@pytest.fixture(scope="session")
def oracle():
    """The CPU oracle (test infrastructure); built from oracle/ if missing."""
    import oracle as O

    O.build()
    O.lib()
    return O


@pytest.fixture(scope="session")
def gpu():
    """libnrq initialised on device 0; fails loudly if it cannot be."""
    import torch

    import nightrun_amd
    from nightrun_amd import _lib

    assert torch.cuda.is_available(), "GPU test needs a visible gfx950 device"
    _lib.lib()
    nightrun_amd.init(0)
    return nightrun_amd
