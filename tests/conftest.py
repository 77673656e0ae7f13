import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a real MI355X (run with -m gpu)")


@pytest.fixture(scope="session")
def kat():
    import json
    with open(os.path.join(ROOT, "tests", "golden", "requant_kat.json")) as f:
        return json.load(f)


# Tests that hold a wrong value: they stay, run, and are known to fail.
WRONG_VALUE = {
    "test_gpu_vocab_layer.py::test_layer[":
        "expects the layer's integers from gradients rounded to bfloat16, whose empty low bits are no random number: PstoShift then rounds "
        "almost every fraction up (test_vocab_update.py shows both sides); the layer takes them from float32",
}


def pytest_collection_modifyitems(items):
    for item in items:
        for name, why in WRONG_VALUE.items():
            if name in item.nodeid:
                item.add_marker(pytest.mark.xfail(reason=why, raises=AssertionError, strict=True))
