"""No unmarked test launches a kernel where a GPU is visible: they pass addresses
that no memory backs."""
import os
import subprocess
import sys

import pytest

from tests.conftest import REPO

# Says that a GPU is visible, and names the tests whose calls get as far as HIP all the same.
PLUGIN = r"""
import ctypes
import torch
import kernelfoundry_amd as kf
torch.cuda.is_available = lambda: True
test = None
def pytest_runtest_protocol(item, nextitem):
    global test
    test = item.nodeid
def note(result, func, args):
    if result == kf.KF_ERR_HIP:
        print("\nREACHED", func.__name__, test, flush=True)
    return result
def pytest_sessionstart(session):
    lib = kf.load_library()
    for name in kf.exported_symbols():
        func = getattr(lib, name)
        if func.restype is ctypes.c_int and name != "kf_last_hip_error":
            func.errcheck = note
"""


def test_unmarked_tests_launch_nothing_beside_a_gpu(tmp_path):
    import torch

    if torch.cuda.is_available():
        pytest.skip("meant for a host whose launches fail")
    (tmp_path / "says_gpu.py").write_text(PLUGIN)
    files = [os.path.join("tests", f) for f in sorted(os.listdir(os.path.join(REPO, "tests")))
             if f.startswith("test_") and f != os.path.basename(__file__)
             and any(word in open(os.path.join(REPO, "tests", f)).read() for word in ("FAKE", "from tests.test_serve_capi"))]
    assert {"tests/test_capi.py", "tests/test_serve_capi.py", "tests/test_serve_refusals.py"} <= set(files)
    env = dict(os.environ, PYTHONPATH=os.pathsep.join([str(tmp_path), REPO]))
    r = subprocess.run([sys.executable, "-m", "pytest", "-p", "says_gpu", "-p", "no:cacheprovider", "-q", "-s",
                        "-m", "not gpu", *files], cwd=REPO, env=env, capture_output=True, text=True)
    assert " passed" in r.stdout, r.stdout + r.stderr
    reached = [line for line in r.stdout.splitlines() if line.startswith("REACHED")]
    assert not reached, reached
