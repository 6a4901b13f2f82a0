"""Sizes past 32 bits: refused by the Python entries, which would hand the C entries
what is left of them in an int; no GPU."""
import pytest
import torch

import kernelfoundry_amd as kf
from kernelfoundry_amd import serve

BIG = 2 ** 32 + 4


def meta(*shape, dtype=torch.float16):
    return torch.empty([n if n < 1000 else 1 for n in shape], dtype=dtype, device="meta").expand(shape)


@pytest.fixture
def refused(monkeypatch):
    """Calls an entry whose checks of devices pass, and whose launch is a failure."""
    monkeypatch.setattr(serve, "_gpu", lambda *a: torch.device("cuda:0"))
    for name in ("_starts", "_ints"):
        monkeypatch.setattr(serve, name, lambda *a: 0)
    monkeypatch.setattr(serve, "_table", lambda *a: (0, 0))
    for name in ("_launch", "_like", "_new_at"):
        monkeypatch.setattr(serve, name, lambda *a: pytest.fail("not refused"))

    def check(call):
        with pytest.raises(kf.KfError) as e:
            call()
        assert e.value.status == kf.KF_ERR_SIZE

    return check


def test_packed(refused):
    q, k, s = meta(4, 8, 128), meta(4, 2, 128), meta(3, dtype=torch.int32)
    for Q, K in ((meta(BIG, 8, 128), k), (q, meta(BIG, 2, 128)), (meta(4, BIG, 128), k), (q, meta(4, BIG, 128))):
        refused(lambda: kf.attn_packed(Q, K, K, s))
    refused(lambda: kf.attn_packed(q, k, k, meta(BIG + 1, dtype=torch.int32)))


def test_rope(refused):
    q, k = meta(4, 8, 128), meta(4, 2, 128)
    for Q, K in ((meta(BIG, 8, 128), meta(BIG, 2, 128)), (meta(4, BIG, 128), k), (q, meta(4, BIG, 128))):
        refused(lambda: kf.qk_norm_rope(Q, K, None, None))


def test_cache(refused):
    k, s, t = meta(4, 2, 128), meta(3, dtype=torch.int32), meta(2, 8, dtype=torch.int32)
    long, wide = meta(BIG + 1, dtype=torch.int32), meta(2, BIG, dtype=torch.int32)
    pages = torch.empty(2, 2, kf.kv4_page_bytes(16, 128), dtype=torch.uint8)
    for K, starts, table in ((meta(BIG, 2, 128), s, t), (k, long, t), (k, s, wide)):
        refused(lambda: kf.kv4_append(K, K, pages, pages, table, starts, None))
    for total, starts, table in ((BIG, s, t), (4, long, t), (4, s, wide)):
        refused(lambda: kf.kv4_read(pages, pages, table, starts, None, total, 128))
    refused(lambda: kf.attn_decode_kv4(meta(2, 8, 1, 128).contiguous(), pages, pages, wide, None))
