import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs an MI355X (gfx950) GPU and the built HIP library")


def pytest_collection_modifyitems(items):
    """Tests without a GPU first: they pass made-up addresses to calls that the library
    refuses as long as no test has initialised it, and that would fault the GPU afterwards."""
    items.sort(key=lambda item: item.get_closest_marker("gpu") is not None)


@pytest.fixture(scope="session")
def rng_seed():
    return 0
