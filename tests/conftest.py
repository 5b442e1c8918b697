"""Shared fixtures.  GPU tests are marked `gpu`; everything else runs on CPU."""
import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
GOLDEN = os.path.join(ROOT, "tests", "golden")
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs an MI355X (runs through the HIP library)")


# Tests as they were written whose expected value contradicts the header, and why.  They run, and have to
# fail (strict): what replaces them is named beside each.
WRONG_VALUES = {
    "test_gpu_paged.py::test_fork_bad_entries":
        "expects the second child of a parent whose last page is not there to take a fresh page that nothing was "
        "copied to: its attention would read what another sequence left in it "
        "(test_fork_of_a_last_page_that_is_not_there; its other values: test_fork_lengths_past_the_table)",
}


def pytest_collection_modifyitems(items):
    for item in items:
        for name, why in WRONG_VALUES.items():
            if item.nodeid.endswith(name):
                item.add_marker(pytest.mark.xfail(reason=why, strict=True))


@pytest.fixture(scope="session")
def ora():
    """The CPU oracle (built on demand; test infrastructure only)."""
    from oracle import ora as _ora
    _ora.lib()
    return _ora


@pytest.fixture(scope="session")
def rai():
    import rai_amd
    rai_amd.lib()
    return rai_amd


def golden(name: str) -> str:
    return os.path.join(GOLDEN, name)


def read_golden(name: str) -> bytes:
    with open(golden(name), "rb") as f:
        return f.read()
