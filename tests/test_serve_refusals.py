"""More refusals of the serving entry points; every check comes before the
first HIP call, and calls that are accepted run only where no GPU could read their
made-up pointers."""
import pytest
import torch

import kernelfoundry_amd as kf
from tests.test_serve_capi import lib, packed  # noqa: F401


@pytest.mark.parametrize("i", [2, 4])
def test_wide_key_strides_are_refused(lib, i):  # noqa: F811
    s = [1024] * 6
    s[i] = (1 << 28) + 8
    assert packed(lib, strides=s) == kf.KF_ERR_SIZE
    if not torch.cuda.is_available():
        s[i] = 1 << 28
        assert packed(lib, strides=s) == kf.KF_ERR_HIP
