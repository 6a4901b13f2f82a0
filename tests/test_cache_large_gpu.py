"""The 16-bit cache's entries on pools of more than 2^32 elements, whose last pages are
used: the same bits as on small pools."""
import pytest
import torch

import kernelfoundry_amd as kf
from tests import _cache_ref as ref
from tests.test_attn_paged_gpu import ints, queries
from tests.test_kv_cache_gpu import equal

pytestmark = pytest.mark.gpu

HEADS, D, PAGE = 8, 128, 64


class Large:
    """`small`, whose pages are the last ones of pools of more than 2^32 elements."""

    def __init__(self, small):
        self.n = small.K.shape[0]
        pages = (1 << 32) // (HEADS * D * PAGE) + 2 * self.n
        self.K, self.V = (torch.empty((pages, HEADS, PAGE, D), dtype=small.K.dtype, device="cuda") for _ in range(2))
        self.weights = torch.zeros((pages, HEADS, PAGE), device="cuda")
        self.table, self.lens = small.table + (pages - self.n), small.lens
        for x, y in self.pairs(small):
            x.copy_(y)

    def pairs(self, small):
        return ((self.K[-self.n:], small.K), (self.V[-self.n:], small.V), (self.weights[-self.n:], small.weights))


def same(large, small):
    torch.cuda.synchronize()
    return all(equal(x, y) for x, y in large.pairs(small)) and not large.weights[: -large.n].any()


@pytest.mark.parametrize("news,before", [([1, 1, 2], [900, 64, 300]), ([300, 90], [700, 0])])
def test_append_and_weights(news, before):
    small = ref.Cache([a + b for a, b in zip(news, before)], HEADS, D, torch.bfloat16, PAGE, spare=0)
    large, s = Large(small), ints(ref.starts_of(news))
    K, V = (queries(news, HEADS, D, torch.bfloat16, seed) for seed in (5, 6))
    Q = queries(news, 2 * HEADS, D, torch.bfloat16)
    for c in (small, large):
        kf.kv_append(K, V, c.K, c.V, c.table, s, c.lens, weights=c.weights)
    assert same(large, small)
    _, lse = kf.attn_paged(Q, small.K, small.V, small.table, s, small.lens, causal=True, return_lse=True)
    for c in (small, large):
        kf.kv_weigh(Q, c.K, c.weights, c.table, s, c.lens, lse, causal=True)
    assert same(large, small)


def test_eviction():
    """Keys that move from behind the new end, in any order, and from below it; the recent ones."""
    small = ref.Cache([9000, 700, 130], HEADS, D, torch.bfloat16, PAGE, spare=0)
    large = Large(small)
    for budgets, recent in (([4000, 600, 130], 200), ([3999, 100, 129], 64)):
        kept = [kf.kv_evict(c.K, c.V, c.weights, c.table, c.lens, ints(budgets), recent=recent) for c in (small, large)]
        assert kept[0].tolist() == kept[1].tolist() == budgets and same(large, small)
        small.lens = large.lens = kept[0]
