import gc
import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a gfx950 GPU (run with -m gpu on the GPU host)")


@pytest.fixture(scope="module", autouse=True)
def _collected():
    """What a module's tests left in reference cycles (a raised error's frames)
    ends with the module, not in a later test that counts what is freed."""
    yield
    gc.collect()
