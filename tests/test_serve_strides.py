"""Strides as the Python entries hand them on; no GPU."""
import pytest
import torch

from kernelfoundry_amd import serve


@pytest.mark.parametrize("token", [3, 1 << 28, (1 << 28) + 8, 1 << 40])
def test_the_stride_of_one_token_or_head_does_not_count(token):
    x = torch.empty(512, dtype=torch.float16)
    at, head = serve._heads("K", x.as_strided((1, 2, 128), (token, 128, 1)))
    assert head == 128 and at in (0, 1 << 28)
    at, head = serve._heads("K", x.as_strided((2, 1, 128), (128, 5, 1)))
    assert (at, head) == (128, 0)


def test_strides_of_several_tokens_are_handed_on():
    wide = torch.empty(0, dtype=torch.float16, device="meta").as_strided((2, 2, 128), ((1 << 28) + 8, 128, 1))
    assert serve._heads("Q", wide) == ((1 << 28) + 8, 128)
    for bad in ((100, 128, 1), (1024, 100, 1), (1024, 128, 2)):
        with pytest.raises(ValueError, match="strides"):
            serve._heads("Q", torch.empty(4096, dtype=torch.float16).as_strided((2, 2, 128), bad))
