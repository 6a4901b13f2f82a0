"""attn_paged against a plain 64-bit form: steps, chunks and mixes over pages, every
layout and type, invalid pages, lengths from none to long."""
import math

import pytest
import torch

import kernelfoundry_amd as kf
from tests import _cache_ref as ref
from tests import _serve_bounds as bounds

pytestmark = pytest.mark.gpu

HEADS = [(8, 2, 128), (4, 1, 64), (6, 2, 256), (3, 3, 64), (7, 1, 128), (2, 2, 256)]


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def queries(news, H_q, D, dtype, seed=1):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn((max(1, sum(news)), H_q, D), generator=gen, dtype=dtype, device="cuda")


def check(cache, Q, news, O, LSE, causal):
    """Every sequence's rows of O and LSE, and, of a slice of heads, how far they may be off."""
    starts = ref.starts_of(news)
    for b, (q, n) in enumerate(zip(news, cache.keys)):
        if q == 0:
            continue
        k, v = cache.rows(b, n, cache.K, cache.V)
        rows = slice(starts[b], starts[b + 1])
        qs = Q[rows].double().transpose(0, 1).contiguous()
        want, lse, off = ref.attention(qs, k, v, ref.seen_by(cache, b, q, n, causal), Q.dtype)
        bounds.check(O[rows].transpose(0, 1), want, off)
        if LSE is not None:
            bounds.check_lse(LSE[rows].transpose(0, 1), lse, qs, k, n)


def run(news, before, heads, dtype=torch.float16, page_size=16, causal=True, out_dtype=None, seed=0, cache=None, Q=None):
    H_q, H_kv, D = heads
    cache = cache or ref.Cache([a + b for a, b in zip(news, before)], H_kv, D, dtype, page_size, seed)
    Q = queries(news, H_q, D, dtype, seed + 1) if Q is None else Q
    O, LSE = kf.attn_paged(Q, cache.K, cache.V, cache.table, ints(ref.starts_of(news)), cache.lens, causal=causal,
                           out_dtype=out_dtype, return_lse=True)
    torch.cuda.synchronize()
    assert O.dtype == (out_dtype or torch.float32)
    check(cache, Q, news, O, LSE, causal)
    return O, LSE


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("page_size", [16, 64])
def test_steps(heads, dtype, page_size):
    """One token of each sequence, contexts around tiles, stages, pages and parts."""
    run([1] * 14, [0, 1, 14, 15, 16, 31, 32, 63, 64, 127, 255, 256, 1000, 4095], heads, dtype, page_size)


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("causal", [True, False])
def test_mixes(heads, dtype, causal):
    run([1, 2, 31, 0, 33, 64, 65, 1, 129, 5, 300], [700, 0, 1, 40, 95, 64, 200, 2100, 17, 31, 33], heads, dtype, 32, causal)


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("news", [[2, 3, 1], [9, 8, 7], [20, 30, 11], [100, 3, 200]])
def test_layouts_by_the_average_rows(heads, news):
    run(news, [500, 33, 1500], heads, torch.bfloat16)


@pytest.mark.parametrize("out_dtype", [None, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("before", [[0, 3, 20], [900, 2000, 60]])
def test_output_types(dtype, out_dtype, before):
    run([5, 77, 140], before, (8, 2, 128), dtype, out_dtype=out_dtype)


@pytest.mark.parametrize("page_size", [16, 32, 128, 1024])
def test_page_sizes(page_size):
    run([1, 40, 3], [2000, 1000, 129], (8, 2, 128), page_size=page_size)
    run([1, 1], [2000, 10], (4, 2, 64), page_size=page_size)


@pytest.mark.parametrize("heads", [(8, 2, 128), (4, 1, 64), (4, 2, 256)])
@pytest.mark.parametrize("causal", [True, False])
def test_fewer_keys_than_queries(heads, causal):
    """Rows that see no key get 0 and -inf; sequences without keys."""
    H_q, H_kv, D = heads
    cache = ref.Cache([10, 0, 33, 1, 200], H_kv, D, torch.float16, 16)
    news = [40, 5, 35, 2, 199]
    O, LSE = run(news, None, heads, causal=causal, cache=cache)
    assert (O[40:45] == 0).all() and (LSE[40:45] == -math.inf).all()
    if causal:
        assert (O[:30] == 0).all() and (LSE[:30] == -math.inf).all()


@pytest.mark.parametrize("heads", [(8, 2, 128), (4, 1, 64), (4, 2, 256)])
@pytest.mark.parametrize("news", [[1, 1, 1, 1], [30, 1, 200, 17]])
@pytest.mark.parametrize("page_size", [16, 64])
def test_invalid_pages(heads, news, page_size):
    """Their keys count as none, also where they are all, or the last."""
    H_q, H_kv, D = heads
    cache = ref.Cache([600, 300, 500, 150], H_kv, D, torch.float16, page_size)
    bad = [-1, cache.K.shape[0], 1 << 30, -(1 << 31)]
    for b, pages in enumerate([[0, 2, 3], [-1], [1, -1], list(range(64))]):
        used = -(-cache.keys[b] // page_size)
        for i in pages:
            cache.table[b, i % used] = bad[i % 4]
    O, LSE = run(news, None, heads, cache=cache)
    rows = slice(sum(news[:3]), sum(news))
    if len(range(64)) >= -(-150 // page_size):
        assert (O[rows] == 0).all() and (LSE[rows] == -math.inf).all()


@pytest.mark.parametrize("n", [63, 64, 65, 130, 700])
@pytest.mark.parametrize("long", [False, True])
def test_sequence_counts(n, long):
    """Up to 64 sequences have a lane each; more, runs of them, cut and whole tiles mixed."""
    news = [(37 * i * i + 11 * i) % (40 if long else 3) for i in range(n)]
    before = [(i * 7919) % (50 if i % 9 else 4000) for i in range(n)]
    run(news, before, (4, 2, 64))


@pytest.mark.parametrize("heads", [(8, 2, 128), (300, 300, 64), (4, 2, 256)])
@pytest.mark.parametrize("most", [250, 900])
def test_shares_of_many_short_sequences(heads, most):
    """Shares that begin inside tiles, several tiles and empty sequences in a share, few keys
    and one share a KV head."""
    news = [(7 * i) % 6 for i in range(40)]
    run(news, [(37 * i) % (most - 10) for i in range(40)], heads)


def test_many_sequences_of_one_token():
    run([1] * 3000, [i % 40 for i in range(3000)], (2, 1, 64))


@pytest.mark.parametrize("heads", [(32, 8, 128), (32, 1, 64), (16, 4, 256), (16, 16, 64)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_long_contexts(heads, dtype):
    """One sequence cut over the whole device; with a chunk, and beside short ones."""
    run([1], [20000], heads, dtype)
    run([130], [9000], heads, dtype, 64)
    run([1, 1, 40], [8191, 3, 2000], heads, dtype)


def test_large_chunks_without_cuts():
    run([2500, 100, 3], [0, 1100, 70], (16, 16, 64), torch.bfloat16, 64)


def test_tokens_outside_the_sequences_are_left_alone():
    H_q, H_kv, D = 8, 2, 128
    cache = ref.Cache([500, 40], H_kv, D, torch.float16, 16)
    Q = queries([60], H_q, D, torch.float16)
    Q[:7], Q[50:] = math.nan, math.inf
    out = torch.full((60, H_q, D), 3.25, device="cuda")
    O, LSE = kf.attn_paged(Q, cache.K, cache.V, cache.table, ints([7, 8, 50]), cache.lens, out, causal=True,
                           return_lse=True)
    torch.cuda.synchronize()
    assert O is out and (O[:7] == 3.25).all() and (O[50:] == 3.25).all()
    check(cache, Q[7:50], [1, 42], O[7:50], LSE[7:50], True)


def test_starts_and_counts_outside_the_tensors_are_clamped():
    cache = ref.Cache([64, 64], 2, 64, torch.float16, 16)
    Q = queries([100], 4, 64, torch.float16)
    a = kf.attn_paged(Q, cache.K, cache.V, cache.table, ints([-5, 40, 1 << 30]), ints([1 << 30, 64]), causal=True)
    b = kf.attn_paged(Q, cache.K, cache.V, cache.table, ints([0, 40, 100]), ints([64, 64]), causal=True)
    assert torch.equal(a, b)
    # In no order: nothing but the rows of O is undefined.
    for starts in ([100, 0, 100], [50, 20, 10], [-(1 << 31), (1 << 31) - 1, -(1 << 31)]):
        O = kf.attn_paged(Q, cache.K, cache.V, cache.table, ints(starts), ints([-3, 64]), causal=True)
        torch.cuda.synchronize()
        assert O.shape == Q.shape


def test_views_of_a_fused_projection_and_broadcast_heads():
    cache = ref.Cache([300, 700], 2, 128, torch.float16, 16)
    x = torch.randn(50, 12 * 128, device="cuda").half()
    Q = x[:, : 8 * 128].unflatten(1, (8, 128))
    s = ints([0, 30, 50])
    a = kf.attn_paged(Q, cache.K, cache.V, cache.table, s, cache.lens, causal=True)
    assert torch.equal(a, kf.attn_paged(Q.contiguous(), cache.K, cache.V, cache.table, s, cache.lens, causal=True))
    one = x[:, :128].unsqueeze(1).expand(50, 8, 128)
    a = kf.attn_paged(one, cache.K, cache.V, cache.table, s, cache.lens, causal=True)
    assert torch.equal(a, kf.attn_paged(one.contiguous(), cache.K, cache.V, cache.table, s, cache.lens, causal=True))


def test_pages_that_sequences_share():
    """A prefix in the same pages of both."""
    cache = ref.Cache([200, 170], 2, 128, torch.float16, 32)
    cache.table[1, :5] = cache.table[0, :5]
    run([1, 10], None, (8, 2, 128), cache=cache)


def test_offsets_past_32_bits():
    """A pool of more than 2^32 elements, whose last pages are used."""
    H, D, ps = 8, 128, 64
    pool = (1 << 32) // (H * D * ps) + 40
    small = ref.Cache([500, 90], H, D, torch.bfloat16, ps, spare=0)
    K, V = (torch.empty((pool, H, ps, D), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    n = small.K.shape[0]
    K[-n:], V[-n:] = small.K, small.V
    Q = queries([1, 50], 16, D, torch.bfloat16)
    s = ints([0, 1, 51])
    got = kf.attn_paged(Q, K, V, small.table + (pool - n), s, small.lens, causal=True)
    assert torch.equal(got, kf.attn_paged(Q, small.K, small.V, small.table, s, small.lens, causal=True))


def test_the_same_call_gives_the_same_bits():
    cache = ref.Cache([5000, 77, 900], 2, 128, torch.bfloat16, 16)
    Q = queries([1, 33, 200], 8, 128, torch.bfloat16)
    s = ints([0, 1, 34, 234])
    a = kf.attn_paged(Q, cache.K, cache.V, cache.table, s, cache.lens, causal=True)
    for _ in range(3):
        assert torch.equal(a, kf.attn_paged(Q, cache.K, cache.V, cache.table, s, cache.lens, causal=True))


def test_a_step_agrees_with_the_paged_decode():
    """Both within their roundings of the same values."""
    cache = ref.Cache([700, 1, 4000, 64], 2, 128, torch.float16, 16, wide=3)
    cache.K.nan_to_num_(0.0)
    cache.V.nan_to_num_(0.0)
    Q = queries([1] * 4, 8, 128, torch.float16)
    a, la = kf.attn_paged(Q, cache.K, cache.V, cache.table, ints([0, 1, 2, 3, 4]), cache.lens, return_lse=True)
    b, lb = kf.attn_decode_paged(Q[:, :, None].contiguous(), cache.K, cache.V, cache.table, cache.lens, return_lse=True)
    check(cache, Q, [1] * 4, a, la, True)
    check(cache, Q, [1] * 4, b[:, :, 0], lb[:, :, 0], True)


def test_streams_graphs_and_a_caller_workspace():
    cache = ref.Cache([3000, 64, 500], 2, 128, torch.float16, 16)
    Q = queries([1, 64, 3], 8, 128, torch.float16)
    s = ints([0, 1, 65, 68])
    call = lambda **kw: kf.attn_paged(Q, cache.K, cache.V, cache.table, s, cache.lens, causal=True, **kw)  # noqa: E731
    want = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = call(stream=side)
    side.synchronize()
    assert torch.equal(got, want)
    need = kf.paged_attn_workspace_bytes(3, 68, 8, 2, 128, 16, cache.table.shape[1])
    assert need > 0
    ws = torch.full((need,), 255, dtype=torch.uint8, device="cuda")
    assert torch.equal(call(workspace=ws), want)
    # Two graphs, replayed between eager calls with other starts and counts.
    outs, graphs = [torch.empty_like(want) for _ in range(2)], []
    for out in outs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            call(out=out)
    for cut, n in ((1, 3000), (10, 100), (60, 0), (0, 2999)):
        s.copy_(ints([0, cut, 65, 68]))
        cache.lens.copy_(ints([n, 64, 500]))
        Q.mul_(0.9)
        want = call()
        for out, graph in zip(outs, graphs):
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
            want = call()


def test_refusals():
    cache = ref.Cache([20], 2, 128, torch.float16, 16)
    Q, s = queries([20], 4, 128, torch.float16), ints([0, 20])
    K, V, t, n = cache.K, cache.V, cache.table, cache.lens
    for bad in (lambda: kf.attn_paged(Q.float(), K, V, t, s, n), lambda: kf.attn_paged(Q.bfloat16(), K, V, t, s, n),
                lambda: kf.attn_paged(Q, K, V.bfloat16(), t, s, n)):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: kf.attn_paged(Q[:, :, :64], K, V, t, s, n), lambda: kf.attn_paged(Q, K, V[:1], t, s, n),
                lambda: kf.attn_paged(Q, K[0], V[0], t, s, n), lambda: kf.attn_paged(Q, K, V, t.long(), s, n),
                lambda: kf.attn_paged(Q, K, V, t, s, n.cpu()), lambda: kf.attn_paged(Q, K, V, t[0], s, n),
                lambda: kf.attn_paged(Q, K, V, t, s[:1], n), lambda: kf.attn_paged(Q, K, V, t, ints([0, 5, 20]), n),
                lambda: kf.attn_paged(Q.transpose(1, 2), K, V, t, s, n),
                lambda: kf.attn_paged(Q, K.transpose(1, 2), V.transpose(1, 2), t, s, n),
                lambda: kf.attn_paged(Q, K, V, t, s, n, torch.empty(20, 4, 64, device="cuda")),
                lambda: kf.attn_paged(Q.clone().requires_grad_(), K, V, t, s, n),
                lambda: kf.attn_paged(Q, K.clone().requires_grad_(), V, t, s, n)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(kf.KfError) as e:
        kf.attn_paged(Q[:, :3].contiguous(), K, V, t, s, n)
    assert e.value.status == kf.KF_ERR_GQA
