"""The tests' elementwise bound of attention: it holds for rounded weights,
and one wrong row of V among thousands breaks it."""
import pytest
import torch

from tests import _serve_bounds as bounds


def emulated(q, k, v, dtype, wrong=None):
    """One head, weights rounded to `dtype`, the rest in 64 bits."""
    s = q @ k.t() / q.shape[1] ** 0.5
    e = torch.exp(s - s.amax(1, keepdim=True))
    if wrong is not None:
        v = v.clone()
        v[wrong] = v[wrong + 1]
    return (e.to(dtype).double() @ v / e.sum(1, keepdim=True))[None]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n", [1, 2, 33, 700, 4097])
def test_bound_of_rounded_weights(dtype, n):
    gen = torch.Generator().manual_seed(n)
    q, k, v = (torch.randn(m, 64, generator=gen).to(dtype).double() for m in (64, n, n))
    want, _, off = bounds.attention(q[None], k[None], v[None], False, dtype)
    bounds.check(emulated(q, k, v, dtype).float(), want, off)
    if n > 33:
        with pytest.raises(AssertionError):
            bounds.check(emulated(q, k, v, dtype, wrong=n // 3).float(), want, off)
        # The size of the bound against that of the outputs.
        assert float((off / want.pow(2).mean().sqrt()).max()) < (0.1 if dtype == torch.bfloat16 else 0.02) * (4097 / n) ** 0.5
