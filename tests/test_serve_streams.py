"""The stream of a call is checked before anything is launched; no GPU."""
from types import SimpleNamespace

import pytest
import torch

from kernelfoundry_amd import serve


def test_a_stream_of_another_device_is_refused():
    def entry(*args):
        pytest.fail("launched")

    stream = SimpleNamespace(device=torch.device("cuda:1"), cuda_stream=0)
    with pytest.raises(ValueError, match="stream of cuda:0"):
        serve._launch(torch, torch.device("cuda:0"), stream, entry)
