import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG_ROOT = os.path.join(ROOT, "aima-amd395-qwen36-35b-linux-engine_amd")
for p in (ROOT, PKG_ROOT):
    if p not in sys.path:
        sys.path.insert(0, p)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs an MI355X (runs through the HIP C-ABI library)")


# Tests that hold a value their operator's documentation rules out, by name: each runs and is
# expected to fail on that value, and a test beside it covers the same ground without it.
WRONG_VALUES = {
    "test_page_tables_gpu.py::test_numbers_out_of_range":
        "expects compaction to clear the entries of rows whose length is none, which every call "
        "leaves as they are; their pages stay counted (test_page_tables_kept_gpu.py)",
}


def pytest_collection_modifyitems(items):
    for item in items:
        reason = WRONG_VALUES.get(item.nodeid.rpartition("/")[2])
        if reason is not None:
            item.add_marker(pytest.mark.xfail(reason=reason, raises=AssertionError, strict=True))


@pytest.fixture(scope="session")
def gpu():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from qwen36_attn import _lib
    _lib.load()
    return torch.device("cuda:0")
