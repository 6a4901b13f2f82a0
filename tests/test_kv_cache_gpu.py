"""kv_append, kv_weigh and kv_evict against plain forms, and a bounded cache filled, attended to
and cut as a server does."""
import math

import pytest
import torch

import kernelfoundry_amd as kf
from tests import _cache_ref as ref
from tests.test_attn_paged_gpu import check, ints, queries

pytestmark = pytest.mark.gpu


def bits(x):
    return x.view({2: torch.int16, 4: torch.int32}[x.element_size()])


def equal(a, b):
    return torch.equal(bits(a), bits(b))


# ---------------------------------------------------------------------------
# New tokens.
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,D,page_size", [(8, 128, 16), (1, 64, 32), (3, 256, 128), (16, 64, 16)])
@pytest.mark.parametrize("news,before", [([1], [0]), ([1, 1, 1], [15, 16, 700]), ([0, 33, 1, 200, 0], [5, 14, 31, 0, 9]),
                                         ([1] * 70, list(range(70))), ([1000, 3], [40, 900])])
def test_append(dtype, heads, D, page_size, news, before):
    cache = ref.Cache([a + b for a, b in zip(news, before)], heads, D, dtype, page_size)
    T = sum(news) + 5                     # tokens behind the last sequence
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randint(-(1 << 15), 1 << 15, (T, 3 * heads, D), generator=gen, dtype=torch.int16, device="cuda").view(dtype)
    K, V = x[:, heads : 2 * heads], x[:, 2 * heads :]
    want, starts = cache.clone(), ref.starts_of(news)
    for b, n in enumerate(cache.keys):
        page, row = cache.slots(b, range(n - news[b], n))
        for pool, new in ((want.K, K), (want.V, V)):
            pool[page, :, row] = new[starts[b] : starts[b + 1]]
        want.weights[page, :, row] = 0
    weights = cache.weights.clone()
    kf.kv_append(K, V, cache.K, cache.V, cache.table, ints(starts), cache.lens)
    torch.cuda.synchronize()
    assert equal(cache.K, want.K) and equal(cache.V, want.V) and equal(cache.weights, weights)
    kf.kv_append(K, V, cache.K, cache.V, cache.table, ints(starts), cache.lens, weights=cache.weights)
    torch.cuda.synchronize()
    assert equal(cache.K, want.K) and equal(cache.V, want.V) and equal(cache.weights, want.weights)


def test_append_without_a_place():
    """Invalid pages, counts that are less than the new tokens or past the table: not written."""
    cache = ref.Cache([40, 40, 40], 2, 64, torch.float16, 16, wide=1)
    cache.table[0, 1], cache.table[1, 2] = -1, cache.K.shape[0]
    K = torch.randn(9, 2, 64, device="cuda").half()
    want, starts = cache.clone(), [0, 3, 6, 9]
    lens = [34, 2, 65]     # places 31 .. 33 (31 invalid), -1 .. 1, 62 .. 64 (64 past the table)
    for b, n in enumerate(lens):
        for i in range(3):
            at = n - 3 + i
            if 0 <= at < 64 and bool(cache.valid(b, at + 1)[-1]):
                page, row = cache.slots(b, [at])
                for pool in (want.K, want.V):
                    pool[page, :, row] = K[starts[b] + i]
                want.weights[page, :, row] = 0
    kf.kv_append(K, K, cache.K, cache.V, cache.table, ints(starts), ints(lens), weights=cache.weights)
    torch.cuda.synchronize()
    assert equal(cache.K, want.K) and equal(cache.V, want.V) and equal(cache.weights, want.weights)


# ---------------------------------------------------------------------------
# Gathered weights.
# ---------------------------------------------------------------------------
def weigh(cache, Q, news, lse, causal):
    """kv_weigh on the cache's weights against the plain form, all other weights bit for bit."""
    before = cache.weights.clone()
    kf.kv_weigh(Q, cache.K, cache.weights, cache.table, ints(ref.starts_of(news)), cache.lens, lse, causal=causal)
    torch.cuda.synchronize()
    rest, starts = cache.weights.clone(), ref.starts_of(news)
    for b, (q, n) in enumerate(zip(news, cache.keys)):
        if q == 0 or n == 0:
            continue
        k, = cache.rows(b, n, cache.K)
        ok = cache.valid(b, n)
        page, row = (x[ok] for x in cache.slots(b, range(n)))
        rows = slice(starts[b], starts[b + 1])
        sums, off = ref.gathered(Q[rows].double().transpose(0, 1).contiguous(), k, lse[rows].double().t().contiguous(),
                                 ref.seen_by(cache, b, q, n, causal))
        old = before[page, :, row].double().t()
        got = cache.weights[page, :, row].double().t()
        want = old + sums[:, ok]
        worst = ((got - want).abs() - off[:, ok] - 2.0 ** -24 * want.abs()).max() if got.numel() else torch.zeros(())
        assert torch.isfinite(got).all() and float(worst) <= 0, (b, float(worst))
        rest[page, :, row] = before[page, :, row]
    assert equal(rest, before)


HEADS = [(8, 2, 128), (4, 1, 64), (6, 2, 256), (3, 3, 64), (32, 1, 128)]


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("news,before", [([1] * 8, [0, 1, 15, 31, 63, 127, 500, 3000]),
                                         ([2, 31, 0, 33, 65, 300], [40, 0, 9, 95, 200, 33]), ([900], [700])])
def test_weights(heads, dtype, causal, news, before):
    H_q, H_kv, D = heads
    cache = ref.Cache([a + b for a, b in zip(news, before)], H_kv, D, dtype, 16)
    Q = queries(news, H_q, D, dtype)
    _, lse = kf.attn_paged(Q, cache.K, cache.V, cache.table, ints(ref.starts_of(news)), cache.lens, causal=causal,
                           return_lse=True)
    weigh(cache, Q, news, lse, causal)
    # All weights of a row add up to 1.
    total = cache.weights.clone()
    cache.weights.zero_()
    kf.kv_weigh(Q, cache.K, cache.weights, cache.table, ints(ref.starts_of(news)), cache.lens, lse, causal=causal)
    for b, n in enumerate(cache.keys):
        page, row = cache.slots(b, range(n))
        s = cache.weights[page, :, row].double().sum(0)
        assert float((s - news[b] * (H_q // H_kv)).abs().max()) <= news[b] * (H_q // H_kv) * 1e-4
    assert total.shape == cache.weights.shape


@pytest.mark.parametrize("page_size", [16, 64, 256])
def test_weights_of_invalid_pages_and_rows_without_keys(page_size):
    cache = ref.Cache([600, 10, 300], 2, 128, torch.float16, page_size)
    cache.table[0, 1], cache.table[2, 0] = -1, 1 << 30
    news = [3, 40, 50]          # 30 rows of the second see no key
    Q = queries(news, 8, 128, torch.float16)
    _, lse = kf.attn_paged(Q, cache.K, cache.V, cache.table, ints(ref.starts_of(news)), cache.lens, causal=True,
                           return_lse=True)
    assert (lse[3:33] == -math.inf).all()
    weigh(cache, Q, news, lse, True)


def test_weights_of_many_sequences():
    news = [i % 3 for i in range(300)]
    cache = ref.Cache([i % 50 + 2 for i in range(300)], 2, 64, torch.bfloat16, 16)
    Q = queries(news, 4, 64, torch.bfloat16)
    _, lse = kf.attn_paged(Q, cache.K, cache.V, cache.table, ints(ref.starts_of(news)), cache.lens, causal=True,
                           return_lse=True)
    weigh(cache, Q, news, lse, True)


def test_weights_of_a_long_prompt_of_one_kv_head():
    news = [2100, 1, 70]
    cache = ref.Cache([2100, 9000, 400], 1, 64, torch.float16, 64)
    Q = queries(news, 32, 64, torch.float16)
    _, lse = kf.attn_paged(Q, cache.K, cache.V, cache.table, ints(ref.starts_of(news)), cache.lens, causal=True,
                           return_lse=True)
    weigh(cache, Q, news, lse, True)


@pytest.mark.parametrize("heads,keys,news", [
    ((64, 64, 64), [70000, 40000, 3], [1, 2, 1]),                      # more runs of a wave than wait in LDS
    ((32, 32, 128), [9000, 20, 9000, 500], [1, 20, 30, 400]),          # steps and chunks in a share
    ((520, 520, 64), [300, 70, 900], [70, 1, 300]),                    # one share a KV head
    ((16, 2, 128), [5000, 4000, 3900], [700, 0, 1000]),                # blocks that several shares cut
    ((10, 2, 256), [1500, 1400], [37, 900])])
@pytest.mark.parametrize("causal", [True, False])
def test_weights_over_shares(heads, keys, news, causal):
    H_q, H_kv, D = heads
    cache = ref.Cache(keys, H_kv, D, torch.float16, 16)
    Q = queries(news, H_q, D, torch.float16)
    _, lse = kf.attn_paged(Q, cache.K, cache.V, cache.table, ints(ref.starts_of(news)), cache.lens, causal=causal,
                           return_lse=True)
    weigh(cache, Q, news, lse, causal)


def test_weights_repeat():
    """The same sums every time."""
    cache = ref.Cache([3000, 700, 5000], 2, 128, torch.bfloat16, 32)
    news = [300, 1, 64]
    Q, s = queries(news, 16, 128, torch.bfloat16), ints(ref.starts_of([300, 1, 64]))
    _, lse = kf.attn_paged(Q, cache.K, cache.V, cache.table, s, cache.lens, causal=True, return_lse=True)
    got = []
    for _ in range(3):
        w = cache.weights.clone()
        kf.kv_weigh(Q, cache.K, w, cache.table, s, cache.lens, lse, causal=True)
        got.append(w)
    assert equal(got[0], got[1]) and equal(got[0], got[2])


def test_weights_from_views_and_tokens_outside():
    cache = ref.Cache([300, 700], 2, 128, torch.float16, 16)
    x = torch.randn(60, 12 * 128, device="cuda").half()
    Q = x[:, : 8 * 128].unflatten(1, (8, 128))
    s = ints([4, 30, 50])
    _, lse = kf.attn_paged(Q, cache.K, cache.V, cache.table, s, cache.lens, causal=True, return_lse=True)
    x[:4], x[50:] = math.nan, math.inf
    lse[:4], lse[50:] = math.nan, math.nan
    a, b = cache.weights.clone(), cache.weights.clone()
    kf.kv_weigh(Q, cache.K, a, cache.table, s, cache.lens, lse, causal=True)
    kf.kv_weigh(Q[4:50].contiguous(), cache.K, b, cache.table, ints([0, 26, 46]), cache.lens, lse[4:50].contiguous(),
                causal=True)
    assert torch.isfinite(a).all() and equal(a, b)


# ---------------------------------------------------------------------------
# Eviction.
# ---------------------------------------------------------------------------
def evict(cache, budgets, recent, **kw):
    want = cache.clone()
    kept = ref.evict(want, budgets, recent)
    got = kf.kv_evict(cache.K, cache.V, cache.weights, cache.table, cache.lens, ints(budgets), recent=recent, **kw)
    torch.cuda.synchronize()
    assert got.tolist() == kept
    for a, b in ((cache.K, want.K), (cache.V, want.V), (cache.weights, want.weights)):
        assert equal(a, b)
    return got


@pytest.mark.parametrize("heads,D,page_size,dtype", [(2, 128, 16, torch.float16), (1, 64, 32, torch.bfloat16),
                                                     (3, 256, 128, torch.float16)])
@pytest.mark.parametrize("recent", [0, 1, 20, 5000])
def test_evict(heads, D, page_size, dtype, recent):
    keys = [0, 1, 2, 16, 17, 100, 300, 1100, 2500, 50, 64, 65, 128]
    cache = ref.Cache(keys, heads, D, dtype, page_size)
    budgets = [5, 0, 1, 15, 17, 99, 20, 1000, 300, -7, 1 << 30, 1, 127]
    evict(cache, budgets, recent)


@pytest.mark.parametrize("keys,budget,recent", [(9000, 8999, 128), (9000, 4500, 300), (9000, 10, 3), (20000, 18000, 2000),
                                                (9000, 8000, 8000), (9000, 8000, 0)])
def test_evict_long(keys, budget, recent):
    cache = ref.Cache([keys, keys // 3], 2, 64, torch.float16, 64)
    evict(cache, [budget, budget // 3], recent)


def test_evict_ties_and_strange_weights():
    """Equal weights go by their places; NaN above infinity, -0 as 0, -inf last."""
    cache = ref.Cache([400, 400, 400, 400], 2, 64, torch.float16, 16)
    w = cache.weights
    page, row = cache.slots(0, range(400))
    w[page, :, row] = 1.5
    page, row = cache.slots(1, range(400))
    w[page, :, row] = torch.arange(400, device="cuda").remainder(3).float()[:, None] - 1
    page, row = cache.slots(2, range(400))
    strange = torch.tensor([math.nan, math.inf, 0.0, -0.0, -math.inf, -1.0, 1e-45, -math.nan], device="cuda")
    w[page, :, row] = strange[torch.arange(400, device="cuda") % 8][:, None]
    evict(cache, [100, 270, 130, 1], 7)


@pytest.mark.parametrize("values", [1, 2, 300])
@pytest.mark.parametrize("wide", [0, 2000, 6000])
def test_evict_ties_of_many_keys(values, wide):
    """Few values among keys of many waves, in tables of different sizes."""
    cache = ref.Cache([5000, 3100, 1025], 2, 64, torch.float16, 16, wide=wide)
    w = torch.randint(0, values, cache.weights.shape, generator=torch.Generator("cuda").manual_seed(values), device="cuda")
    cache.weights.copy_(w.float() / 7 - 3)
    evict(cache, [2100, 3000, 1], 40)


def test_evict_more_keys_than_registers_hold():
    cache = ref.Cache([90000, 100, 82500], 1, 64, torch.bfloat16, 64)
    evict(cache, [30000, 90, 82400], 300)


def test_evict_on_invalid_pages():
    """A sequence with one among its keys is left, its count too; one behind its keys does not matter."""
    cache = ref.Cache([100, 100, 100, 100], 2, 128, torch.float16, 16, wide=2)
    cache.table[0, 3], cache.table[1, 6], cache.table[2, 7], cache.table[3, 0] = -1, cache.K.shape[0], -5, 1 << 30
    got = evict(cache, [50, 50, 50, 100], 10)
    assert got.tolist() == [100, 100, 50, 100]


def test_evict_writes_its_counts_over_its_inputs():
    for alias in ("lens", "budgets"):
        cache = ref.Cache([300, 40, 2000], 4, 128, torch.bfloat16, 16)
        budgets = ints([100, 100, 1999])
        out = cache.lens if alias == "lens" else budgets
        want = cache.clone()
        kept = ref.evict(want, [100, 100, 1999], 32)
        got = kf.kv_evict(cache.K, cache.V, cache.weights, cache.table, cache.lens, budgets, out, recent=32)
        torch.cuda.synchronize()
        assert got is out and got.tolist() == kept and equal(cache.K, want.K) and equal(cache.weights, want.weights)


def test_evict_again_and_again():
    """Counts that change on the device, one key at a time."""
    cache = ref.Cache([200, 130], 2, 64, torch.float16, 16)
    lens = cache.lens
    for step in range(6):
        budgets = [n - 1 - step * 5 for n in cache.keys]
        kept = evict(cache, budgets, 16)
        cache.keys = kept.tolist()
        lens.copy_(kept)


def test_evict_of_sequences_that_share_pages_stays_inside():
    """What the shared pages hold is undefined; nothing else is touched."""
    cache = ref.Cache([500, 500], 2, 64, torch.float16, 16)
    cache.table[1, :20] = cache.table[0, :20]
    cache.table[0, 25] = cache.table[0, 24]
    want = cache.clone()
    ws = torch.zeros(kf.evict_workspace_bytes(2, 2, 64, 16, cache.table.shape[1]) + 4096, dtype=torch.uint8, device="cuda")
    ws[-4096:] = 77
    kf.kv_evict(cache.K, cache.V, cache.weights, cache.table, cache.lens, ints([100, 250]), recent=9, workspace=ws[:-4096])
    torch.cuda.synchronize()
    used = torch.zeros(cache.K.shape[0], dtype=torch.bool, device="cuda")
    used[cache.table.flatten().long()] = True
    assert equal(cache.K[~used], want.K[~used]) and (ws[-4096:] == 77).all()


# ---------------------------------------------------------------------------
# Together.
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("heads,dtype", [((8, 2, 128), torch.float16), ((4, 1, 64), torch.bfloat16)])
def test_a_bounded_cache(heads, dtype):
    """Prompts in chunks, cut to a budget, then steps of which each evicts one key, eager and
    replayed from a graph; attention is checked over what the pages hold at each point."""
    H_q, H_kv, D = heads
    cache = ref.Cache([700, 90, 400], H_kv, D, dtype, 16, wide=2)
    whole, gen = cache.keys, torch.Generator(device="cuda").manual_seed(9)
    for x in (cache.K, cache.V):
        x.fill_(math.nan)
    cache.weights.fill_(math.nan)
    budget, recent = 80, 24

    def forward(news, keys):
        T = sum(news)
        qkv = torch.randn(T, (H_q + 2 * H_kv) * D, generator=gen, dtype=dtype, device="cuda")
        Q, K, V = (x.unflatten(1, (-1, D)) for x in qkv.split((H_q * D, H_kv * D, H_kv * D), 1))
        starts, lens = ints(ref.starts_of(news)), ints(keys)
        kf.kv_append(K, V, cache.K, cache.V, cache.table, starts, lens, weights=cache.weights)
        O, lse = kf.attn_paged(Q, cache.K, cache.V, cache.table, starts, lens, causal=True, return_lse=True)
        cache.keys, cache.lens = keys, lens
        check(cache, Q, news, O, lse, True)
        weigh(cache, Q, news, lse, True)

    done = [0, 0, 0]
    while done != whole:
        news = [min(150, n - d) for n, d in zip(whole, done)]
        done = [d + q for d, q in zip(done, news)]
        forward(news, done)
    cache.keys = evict(cache, [budget] * 3, recent).tolist()
    assert cache.keys == [80, 80, 80]
    for _ in range(3):
        forward([1, 1, 1], [n + 1 for n in cache.keys])
        cache.keys = evict(cache, [budget] * 3, recent).tolist()

    # The step as a graph.
    Q, K, V = (torch.empty(3, h, D, dtype=dtype, device="cuda") for h in (H_q, H_kv, H_kv))
    starts, lens, budgets, kept = ints([0, 1, 2, 3]), ints([81] * 3), ints([budget] * 3), ints([0] * 3)
    O = torch.empty(3, H_q, D, device="cuda")

    def step(c):
        kf.kv_append(K, V, c.K, c.V, c.table, starts, lens, weights=c.weights)
        _, lse = kf.attn_paged(Q, c.K, c.V, c.table, starts, lens, O, causal=True, return_lse=True)
        kf.kv_weigh(Q, c.K, c.weights, c.table, starts, lens, lse, causal=True)
        kf.kv_evict(c.K, c.V, c.weights, c.table, lens, budgets, kept, recent=recent)

    twin = cache.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(cache)
    for i in range(5):
        for x in (Q, K, V):
            x.copy_(torch.randn(x.shape, generator=gen, dtype=dtype, device="cuda"))
        O.zero_()
        kept.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = O.clone()
        assert kept.tolist() == [80, 80, 80]
        step(twin)
        torch.cuda.synchronize()
        assert torch.equal(got, O) and equal(cache.K, twin.K) and equal(cache.V, twin.V)
        assert equal(cache.weights, twin.weights)


def test_other_streams():
    cache = ref.Cache([300, 90], 2, 128, torch.float16, 16)
    want = cache.clone()
    ref.evict(want, [100, 50], 10)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = kf.kv_evict(cache.K, cache.V, cache.weights, cache.table, cache.lens, ints([100, 50]), recent=10, stream=side)
    side.synchronize()
    assert got.tolist() == [100, 50] and equal(cache.K, want.K) and equal(cache.weights, want.weights)


def test_refusals():
    cache = ref.Cache([20], 2, 128, torch.float16, 16)
    x, s, b = torch.randn(4, 2, 128, device="cuda").half(), ints([0, 4]), ints([7])
    K, V, w, t, n = cache.K, cache.V, cache.weights, cache.table, cache.lens
    lse = torch.zeros(4, 2, device="cuda")
    for bad in (lambda: kf.kv_append(x.bfloat16(), x.bfloat16(), K, V, t, s, n), lambda: kf.kv_append(x, x.bfloat16(), K, V, t, s, n),
                lambda: kf.kv_weigh(x, K.bfloat16(), w, t, s, n, lse), lambda: kf.kv_evict(K, V.bfloat16(), w, t, n, b),
                lambda: kf.kv_evict(K.float(), V.float(), w, t, n, b)):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: kf.kv_append(x, x, K, V, t, s, n, weights=w.half()), lambda: kf.kv_append(x, x, K, V, t, s, n, weights=w[:1]),
                lambda: kf.kv_append(x[:, :1], x[:, :1], K, V, t, s, n), lambda: kf.kv_append(x[..., :64], x[..., :64], K, V, t, s, n),
                lambda: kf.kv_append(x, x, K, V, t, s.long(), n), lambda: kf.kv_append(x.requires_grad_(), x, K, V, t, s, n),
                lambda: kf.kv_weigh(x.detach(), K, w, t, s, n, lse[:3]), lambda: kf.kv_weigh(x.detach(), K, w, t, s, n, lse.double()),
                lambda: kf.kv_weigh(x.detach(), K, w.transpose(1, 2), t, s, n, lse), lambda: kf.kv_weigh(x.detach(), K, w, t, s, n, lse.cpu()),
                lambda: kf.kv_evict(K, V, w, t, n, b.long()), lambda: kf.kv_evict(K, V, w, t, n, ints([1, 2])),
                lambda: kf.kv_evict(K, V, w, t[0], n, b), lambda: kf.kv_evict(K, V, w, t, n, b, recent=-1),
                lambda: kf.kv_evict(K, V[:1], w, t, n, b), lambda: kf.kv_evict(K, V, w, t, n, b, torch.zeros(1, device="cuda"))):
        with pytest.raises(ValueError):
            bad()
