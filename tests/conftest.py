import gc
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
if str(ROOT) not in sys.path:
    sys.path.insert(0, str(ROOT))


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a real MI355X (run with -m gpu)")


def _has_gpu():
    try:
        import torch

        # the package names its SDMA-engine tools library in HSA_TOOLS_LIB at
        # import; that has to happen before the first call into the GPU runtime
        import offload_adam_amd  # noqa: F401

        return torch.cuda.is_available()
    except Exception:
        return False


def pytest_collection_modifyitems(config, items):
    if _has_gpu():
        return
    skip = pytest.mark.skip(reason="no GPU in this environment")
    for item in items:
        if "gpu" in item.keywords:
            item.add_marker(skip)


def pytest_runtest_setup(item):
    # tests that compare counts of allocated memory: cycles that earlier tests left behind
    # are collected before they begin, not while they count
    if item.module.__name__.endswith("test_zz_no_alloc"):
        gc.collect()


@pytest.fixture(scope="session")
def oracle():
    import oracle as _oracle

    _oracle.lib()
    return _oracle
