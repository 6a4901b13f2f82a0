"""More refusals of the serving entry points; every check comes before the
first HIP call, and calls that are accepted run only where no GPU could read their
made-up pointers."""
import pytest
import torch

import kernelfoundry_amd as kf
from tests.test_serve_capi import append, decode, lib, packed, read  # noqa: F401


@pytest.mark.parametrize("i", [2, 4])
def test_wide_key_strides_are_refused(lib, i):  # noqa: F811
    s = [1024] * 6
    s[i] = (1 << 28) + 8
    assert packed(lib, strides=s) == kf.KF_ERR_SIZE
    if not torch.cuda.is_available():
        s[i] = 1 << 28
        assert packed(lib, strides=s) == kf.KF_ERR_HIP


# The largest grids that a launch can number: fewer than 2^32 threads.
@pytest.mark.parametrize("call", [append, read])
def test_cache_grids(lib, call):  # noqa: F811
    """Workgroups of 256 threads and, of 8 heads of 256, four tokens."""
    most = 4 * (2 ** 24 - 1)
    assert call(lib, T=most + 1, H_kv=8, D=256) == kf.KF_ERR_SIZE
    assert call(lib, T=1 << 27, H_kv=8, D=256) == kf.KF_ERR_SIZE
    if not torch.cuda.is_available():
        assert call(lib, T=most, H_kv=8, D=256) == kf.KF_ERR_HIP


def test_decode_merge_grid(lib):  # noqa: F811
    """The merge has a wave per sequence and KV head at least: refused before the
    decode is launched."""
    one = dict(H_q=1, H_kv=1, D=64, mp=1)
    assert decode(lib, B=1 << 26, **one) == kf.KF_ERR_SIZE
    assert kf.kv4_workspace_bytes(1 << 26, 1, 1, 1, 64, 16, 1) == 0
    assert kf.kv4_workspace_bytes((1 << 26) - 4, 1, 1, 1, 64, 16, 1) > 0
    if not torch.cuda.is_available():
        assert decode(lib, B=(1 << 26) - 4, **one) == kf.KF_ERR_HIP
