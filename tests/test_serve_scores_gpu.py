"""Scores of large magnitude, up to the documented 9e7, and rows of one weight."""
import pytest
import torch

import kernelfoundry_amd as kf
from tests.test_kv4_gpu import ints, new_cache, normal

pytestmark = pytest.mark.gpu

LENS = [300, 1, 70]


def keys_of_two_sizes(D, dtype):
    """Keys of 1536 or -1536 in every channel, exact in 4 bits: against queries of a
    power of two all products and sums are exact, so a row's weights are 1 and 0."""
    plus = torch.arange(sum(LENS), device="cuda") % 3 != 1
    plus[300] = True                       # the sequence of one key
    K = torch.where(plus, 1536.0, -1536.0).to(dtype)[:, None, None].expand(-1, 2, D).contiguous()
    return K, plus


def check(O, V, plus, dtype, rows):
    """O is the mean of V over the keys of the larger score: one weight, rounded to
    `dtype` where it meets V and not in the sum; sums of up to 300 terms in 32 bits."""
    at = 0
    for i, n in enumerate(LENS):
        v = V[at:at + n][plus[at:at + n]].double()
        mean = v.mean(0).repeat_interleave(rows, 0)          # [H_q, D]
        off = (torch.finfo(dtype).eps / 2 + 2.0 ** -24 * (n + 64)) * v.abs().mean(0).repeat_interleave(rows, 0)
        assert torch.isfinite(O[i]).all() and ((O[i].double() - mean).abs() <= off).all()
        at += n


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("q", [1, 1024, 4096])
def test_large_scores(D, dtype, q):
    """q 4096: q . k / sqrt(D) = 5.0e7, 7.1e7 and (2048) 5.0e7."""
    if D == 256 and q == 4096:
        q = 2048
    K, plus = keys_of_two_sizes(D, dtype)
    V = normal(sum(LENS), 2, D, dtype=dtype)
    starts = [0]
    for n in LENS:
        starts.append(starts[-1] + n)
    for Q in (torch.full((3, 8, D), q, device="cuda", dtype=dtype), torch.full((3, 24, D), q, device="cuda", dtype=dtype)):
        rows = Q.shape[1] // 2
        O = kf.attn_packed(Q, K, V, ints([0, 1, 2, 3]), kv_starts=ints(starts), causal=True)
        check(O, V, plus, dtype, rows)
        Kp, Vp, table = new_cache(LENS, 2, D, 16)
        kf.kv4_append(K, V, Kp, Vp, table, ints(starts), ints(LENS))
        K4, V4 = kf.kv4_read(Kp, Vp, table, ints(starts), ints(LENS), sum(LENS), D, out_dtype=dtype)
        assert torch.equal(K4, K)
        O = kf.attn_decode_kv4(Q[:, :, None].contiguous(), Kp, Vp, table, ints(LENS))
        check(O[:, :, 0], V4, plus, dtype, rows)
