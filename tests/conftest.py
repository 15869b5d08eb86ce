import os
import sys

import pytest
import torch  # noqa: F401  before the library loads, so that both use one HIP runtime (torch brings its own)

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "lightining-core_amd")
for p in (ROOT, PKG, os.path.dirname(os.path.abspath(__file__))):
    if p not in sys.path:
        sys.path.insert(0, p)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a real MI355X (HIP device); parity tests proper")


@pytest.fixture(scope="session")
def oracle():
    import oracle_lib

    return oracle_lib.load()
