"""kv_weigh's rows whose log-sum-exp is no ordinary number: what they add, and to which keys
alone."""
import math

import pytest
import torch

import kernelfoundry_amd as kf
from tests import _cache_ref as ref
from tests.test_attn_paged_gpu import ints, queries
from tests.test_kv_cache_gpu import equal

pytestmark = pytest.mark.gpu

HEADS = [(8, 2, 128), (4, 1, 64), (6, 2, 256), (3, 3, 64)]
# Steps; a step, a chunk and rows of which some see no key; one chunk that shares cut.
MIXES = [([1, 3, 2], [200, 70, 1500]), ([1, 200, 90], [300, 130, -40]), ([700], [900])]


class Call:
    def __init__(self, heads, dtype, news, before, causal):
        H_q, H_kv, D = heads
        self.news, self.causal, self.ratio = news, causal, H_q // H_kv
        self.cache = ref.Cache([a + b for a, b in zip(news, before)], H_kv, D, dtype, 16)
        self.starts = ref.starts_of(news)
        self.Q = queries(news, H_q, D, dtype)
        _, self.lse = kf.attn_paged(self.Q, self.cache.K, self.cache.V, self.cache.table, ints(self.starts), self.cache.lens,
                                    causal=causal, return_lse=True)

    def __call__(self, Q=None, lse=None, K=None):
        w = self.cache.weights.clone()
        kf.kv_weigh(self.Q if Q is None else Q, self.cache.K if K is None else K, w, self.cache.table, ints(self.starts),
                    self.cache.lens, self.lse if lse is None else lse, causal=self.causal)
        torch.cuda.synchronize()
        return w

    def rows(self):
        """Of every sequence the first, the last and one more token: (sequence, token in it, head)."""
        for b, n in enumerate(self.news):
            for k, i in enumerate(sorted({0, n // 3, n - 1})):
                yield b, i, (5 * b + k) % (self.lse.shape[1])

    def seen(self, b, i):
        """Pages and rows of the keys that token i of sequence b sees."""
        n = self.cache.keys[b]
        sees = ref.seen_by(self.cache, b, self.news[b], n, self.causal)[i].cpu().nonzero()[:, 0].tolist()
        return self.cache.slots(b, sees)


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("news,before", MIXES)
def test_nan_reaches_the_keys_that_the_row_sees(heads, dtype, causal, news, before):
    """Whatever its sign and payload; all other weights are those of a call without it."""
    call = Call(heads, dtype, news, before, causal)
    want = call()
    for k, (b, i, h) in enumerate(call.rows()):
        lse = call.lse.clone()
        lse.view(torch.int32)[call.starts[b] + i, h] = [0x7fc00000, 0x7f800001, -1, -0x400000][k % 4]
        got, expect = call(lse=lse), want.clone()
        page, row = call.seen(b, i)
        assert torch.isnan(got[page, h // call.ratio, row]).all(), (b, i, h)
        expect[page, h // call.ratio, row] = got[page, h // call.ratio, row]
        assert equal(got, expect), (b, i, h)


def test_nan_in_every_row():
    call = Call((8, 2, 128), torch.float16, [1, 200, 90], [300, 130, -40], True)
    got, want = call(lse=torch.full_like(call.lse, math.nan)), call.cache.weights.clone()
    for b, n in enumerate(call.news):
        page, row = call.seen(b, n - 1)
        assert torch.isnan(got[page, :, row]).all()
        want[page, :, row] = got[page, :, row]
    assert equal(got, want)


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("news,before", MIXES)
def test_rows_of_minus_infinity_add_nothing(heads, dtype, causal, news, before):
    """Whatever they hold themselves."""
    call = Call(heads, dtype, news, before, causal)
    lse, Q = call.lse.clone(), call.Q.clone()
    for k, (b, i, h) in enumerate(call.rows()):
        lse[call.starts[b] + i, h] = -math.inf
        Q[call.starts[b] + i, h] = [math.nan, math.inf, -math.inf][k % 3]
        Q[call.starts[b] + i, h, ::2] = 1.0
    want = call(lse=lse)
    assert torch.isfinite(want).all() and equal(call(Q=Q, lse=lse), want)


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("news,before", MIXES)
def test_rows_of_minus_infinity_add_nothing_to_strange_keys(heads, news, before):
    """No row adds anything: keys that hold NaN and infinities keep their weights."""
    call = Call(heads, torch.bfloat16, news, before, True)
    K = call.cache.K.clone()
    K[..., 3] = math.nan
    K[:, :, ::3, 5] = math.inf
    assert equal(call(K=K, lse=torch.full_like(call.lse, -math.inf)), call.cache.weights)


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("value", [torch.finfo(torch.float32).min, -2.4e38, -1e30, 1e30, torch.finfo(torch.float32).max,
                                   math.inf])
@pytest.mark.parametrize("news,before", MIXES)
def test_extreme_rows(heads, causal, value, news, before):
    """exp(score - lse) is infinite, or 0; keys that the row does not see get nothing."""
    call = Call(heads, torch.float16, news, before, causal)
    want = call()
    for b, i, h in call.rows():
        lse = call.lse.clone()
        lse[call.starts[b] + i, h] = value
        got, expect = call(lse=lse), want.clone()
        page, row = call.seen(b, i)
        at = got[page, h // call.ratio, row]
        assert (torch.isposinf(at) if value < 0 else torch.isfinite(at)).all(), (b, i, h)
        expect[page, h // call.ratio, row] = at
        assert equal(got, expect), (b, i, h)


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("news,before", MIXES)
def test_strange_queries_reach_the_keys_that_the_row_sees(heads, causal, value, news, before):
    """One channel of a row with an ordinary log-sum-exp."""
    call = Call(heads, torch.bfloat16, news, before, causal)
    want = call()
    for b, i, h in call.rows():
        if not math.isfinite(float(call.lse[call.starts[b] + i, h])):
            continue
        Q = call.Q.clone()
        Q[call.starts[b] + i, h, 7] = value
        got, expect = call(Q=Q), want.clone()
        page, row = call.seen(b, i)
        at = got[page, h // call.ratio, row]
        assert math.isinf(value) or torch.isnan(at).all(), (b, i, h)
        expect[page, h // call.ratio, row] = at
        assert equal(got, expect), (b, i, h)


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("news,before", MIXES)
def test_strange_keys_change_their_own_weight_alone(heads, news, before):
    call = Call(heads, torch.bfloat16, news, before, True)
    K, want = call.cache.K.clone(), call()
    odd = torch.zeros_like(call.cache.weights, dtype=torch.bool)
    for b, n in enumerate(call.cache.keys):
        page, row = call.cache.slots(b, range(0, n, 7))
        K[page, :, row, 3], odd[page, :, row] = math.nan, True
        page, row = call.cache.slots(b, range(3, n, 14))
        K[page, :, row, 9], odd[page, :, row] = math.inf, True
    got = call(K=K)
    assert equal(torch.where(odd, 0.0, got), torch.where(odd, 0.0, want))
    for b, n in enumerate(call.cache.keys):
        page, row = call.cache.slots(b, range(0, n, 7))
        assert torch.isnan(got[page, :, row]).all()
