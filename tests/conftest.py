import os
import sys

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if REPO not in sys.path:
    sys.path.insert(0, REPO)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs an MI355X (gfx950) GPU")
    config.addinivalue_line("markers", "slow: long-running CPU check")


@pytest.fixture(scope="session")
def repo_root():
    return REPO


# Tests of the host's checks that go on to a call which is accepted, with addresses
# that no memory backs: its launch fails on a host without a GPU, and on one with a GPU
# the kernel would read them.
HOST_ONLY = {
    ("test_capi.py", "test_split_prefill_runs_without_a_workspace"),
    ("test_serve_capi.py", "test_packed_key_strides"),
}


def pytest_runtest_setup(item):
    if (item.path.name, getattr(item, "originalname", item.name)) in HOST_ONLY:
        import torch

        if torch.cuda.is_available():
            pytest.skip("an accepted call would run on addresses that are not real")
