import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a real MI355X (run with -m gpu on the GPU box)")


def pytest_collection_modifyitems(items):
    """the tests against the reference's own modules need its source tree, not just the folder that it would be in"""
    from oracle.ref_shim import REF_ROOT
    if not os.path.isdir(os.path.join(REF_ROOT, "code")):
        for item in items:
            if os.path.basename(str(item.fspath)) == "test_dropin_cpu.py":
                item.add_marker(pytest.mark.skip(reason="the reference's source tree is not here"))


@pytest.fixture(scope="session")
def gold_dir():
    return os.path.join(ROOT, "tests", "golden")
