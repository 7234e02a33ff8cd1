import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a real MI355X (run with -m gpu)")


# Tests with an expected value that the contract contradicts, kept as they were written.
RANKS = "ranks a group with one usable expert as one with none, so that masked experts are chosen where others are left; the same inputs by the header: test_gpu_select_masks.py"
WRONG = {"test_gpu_select.py::test_masked_and_missing_logits": RANKS, "test_gpu_select.py::test_many_tokens_masked": RANKS}


def pytest_collection_modifyitems(items):
    for item in items:
        reason = WRONG.get(os.path.basename(str(item.fspath)) + "::" + getattr(item, "originalname", item.name))
        if reason:
            item.add_marker(pytest.mark.xfail(reason=reason, strict=True, raises=AssertionError))


@pytest.fixture(scope="session")
def orc():
    import oracle
    oracle.lib()
    return oracle
