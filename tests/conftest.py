import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a real MI355X (run with -m gpu)")


# Tests that stay as they are although a value they hold is wrong, and why it is
WRONG_VALUES = {
    "test_gpu_kv_pages.py::test_forks_from_pages_outside_the_pool":
        "expects a page from the free stack in the child's table where the parent's page lies outside the pool: page 8, which nothing is copied to, so that attention would take what its last "
        "owner left there for rows 64 .. 99 of the child, where the parent has none (test_forks_that_end_in_a_page_outside_the_pool)",
}


def pytest_collection_modifyitems(items):
    for item in items:
        for name, why in WRONG_VALUES.items():
            if item.nodeid.endswith(name):
                item.add_marker(pytest.mark.xfail(strict=True, raises=AssertionError, reason=why))


@pytest.fixture(scope="session")
def oracle():
    import oracle as orc
    orc.build()
    return orc
