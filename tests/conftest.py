import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a real MI355X (run with -m gpu on the GPU box)")


def pytest_collection_modifyitems(config, items):
    """Without a GPU the gpu-marked tests are skipped, not failed (plain `pytest tests` on a CPU-only machine)."""
    import torch
    if torch.cuda.is_available():
        return
    skip = pytest.mark.skip(reason="needs a real MI355X")
    for item in items:
        if "gpu" in item.keywords:
            item.add_marker(skip)


@pytest.fixture(scope="session")
def golden():
    from tests import util
    return util.Golden()


@pytest.hookimpl(tryfirst=True)
def pytest_pyfunc_call(pyfuncitem):
    """The tests of test_abi.py run in a thread each: iff_last_error() is a thread's, and what other tests' errors left is not theirs."""
    if pyfuncitem.path.name != "test_abi.py":
        return None
    from concurrent.futures import ThreadPoolExecutor
    with ThreadPoolExecutor(1) as one:
        one.submit(pyfuncitem.obj, **{a: pyfuncitem.funcargs[a] for a in pyfuncitem._fixtureinfo.argnames}).result()
    return True
