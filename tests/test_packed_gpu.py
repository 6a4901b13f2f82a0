"""kf_attn_packed against a plain 64-bit form, a sequence and a head at a
time: lengths from none to long, odd sizes, strided views, several types."""
import math

import pytest
import torch

import kernelfoundry_amd as kf
from tests import _serve_ref as ref

pytestmark = pytest.mark.gpu


def starts_of(lens):
    s = [0]
    for n in lens:
        s.append(s[-1] + n)
    return s


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def make(lens, heads, dtype, kv_lens=None, seed=0, fused=False):
    H_q, H_kv, D = heads
    gen = torch.Generator(device="cuda").manual_seed(seed)
    T, Tk = max(1, sum(lens)), max(1, sum(kv_lens or lens))
    if fused:
        x = torch.randn(T, (H_q + 2 * H_kv) * D, generator=gen, device="cuda", dtype=dtype)
        return [v.unflatten(1, (-1, D)) for v in x.split((H_q * D, H_kv * D, H_kv * D), 1)]
    return [torch.randn(n, h, D, generator=gen, device="cuda", dtype=dtype)
            for n, h in ((T, H_q), (Tk, H_kv), (Tk, H_kv))]


def run(lens, heads, dtype=torch.float16, kv_lens=None, causal=True, out_dtype=None, seed=0, fused=False, tensors=None):
    Q, K, V = tensors or make(lens, heads, dtype, kv_lens, seed, fused)
    qs, ks = starts_of(lens), starts_of(kv_lens or lens)
    O, LSE = kf.attn_packed(Q, K, V, ints(qs), kv_starts=ints(ks) if kv_lens else None, causal=causal,
                            out_dtype=out_dtype, return_lse=True)
    torch.cuda.synchronize()
    want, want_lse = ref.packed(Q, K, V, qs, ks, causal)
    bounds = ref.attention_bounds(Q, K, V, out_dtype or torch.float32, max(kv_lens or lens))
    ref.check_attention(O, LSE, want, want_lse, bounds)
    return O, LSE


HEADS = [(8, 2, 128), (4, 1, 64), (6, 2, 256), (3, 3, 64), (7, 1, 128)]


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("causal", [True, False])
def test_lengths_around_tiles_and_stages(heads, dtype, causal):
    run([1, 2, 31, 32, 33, 63, 64, 65, 0, 127, 129, 0, 255, 257, 300], heads, dtype, causal=causal)


@pytest.mark.parametrize("out_dtype", [None, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_output_types(dtype, out_dtype):
    O, _ = run([5, 77, 140], (8, 2, 128), dtype, out_dtype=out_dtype)
    assert O.dtype == (out_dtype or torch.float32)


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("causal", [True, False])
def test_more_and_fewer_keys_than_queries(heads, causal):
    """Chunks over contexts; causal rows in front of the first key see none."""
    run([16, 70, 40, 100, 9, 0, 33, 200], heads, kv_lens=[200, 70, 0, 37, 1, 50, 300, 199], causal=causal)


@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 130, 700])
def test_sequence_counts(n):
    lens = [(37 * i * i + 11 * i) % 90 for i in range(n)]
    run(lens or [3], (4, 2, 64), causal=n % 2 == 0)


@pytest.mark.parametrize("n", [5000])
def test_many_sequences_of_one_token(n):
    run([1] * n, (2, 1, 64))


@pytest.mark.parametrize("S,heads", [(4097, (8, 2, 128)), (2500, (16, 1, 64)), (1800, (4, 2, 256))])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_long_prompts(S, heads, dtype):
    run([S, 5, S // 3], heads, dtype, fused=True)


@pytest.mark.parametrize("n,longest,heads,causal", [(64, 600, (64, 64, 64), True), (40, 900, (32, 32, 64), True),
                                                    (64, 600, (32, 32, 128), False), (64, 500, (32, 32, 256), True)])
def test_grids_of_many_rounds(n, longest, heads, causal):
    """Workgroups enough that several tiles of a sequence are numbered together."""
    lens = [(i * 7919 + 13) % longest for i in range(n)]
    run(lens, heads, kv_lens=[(k * 3) // 2 if i % 3 else k // 2 for i, k in enumerate(lens)], causal=causal)


def test_views_of_a_fused_projection_equal_their_copies():
    Q, K, V = make([300, 20], (8, 2, 128), torch.float16, fused=True)
    s = ints([0, 300, 320])
    a = kf.attn_packed(Q, K, V, s, causal=True)
    b = kf.attn_packed(Q.contiguous(), K.contiguous(), V.contiguous(), s, causal=True)
    assert torch.equal(a, b)


def test_head_major_and_broadcast_views():
    """[H, T, D] storage, and keys of one head shared by all through stride 0."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    Q = torch.randn(4, 150, 128, generator=gen, device="cuda", dtype=torch.float16).transpose(0, 1)
    K = torch.randn(150, 1, 128, generator=gen, device="cuda", dtype=torch.float16).expand(150, 2, 128)
    run([100, 50], (4, 2, 128), tensors=(Q, K, K))


@pytest.mark.parametrize("heads", [(8, 2, 128), (4, 1, 64), (4, 2, 256)])
def test_what_lies_outside_the_sequences_is_neither_read_nor_written(heads):
    """Infinities and NaN between the places of neighbouring sequences' rows:
    tokens before the first start and behind the last; keys of other sequences
    that share tiles."""
    H_q, H_kv, D = heads
    Q, K, V = make([400], heads, torch.float16)
    qs, ks = [7, 60, 60, 171, 300], [3, 50, 90, 90, 333]
    for x, s in ((Q, qs), (K, ks), (V, ks)):
        x[: s[0]] = math.nan
        x[s[-1]:] = math.inf
    K[50:90] = math.nan      # the keys of a sequence without queries
    V[50:90] = math.inf
    out = torch.full(Q.shape, 3.25, device="cuda", dtype=torch.float32)
    O, LSE = kf.attn_packed(Q, K, V, ints(qs), out, kv_starts=ints(ks), causal=False, return_lse=True)
    assert O.data_ptr() == out.data_ptr()
    torch.cuda.synchronize()
    want, want_lse = ref.packed(Q, K, V, qs, ks, False)
    clean = [torch.where(torch.isfinite(x), x, torch.zeros_like(x)) for x in (Q, K, V)]
    ref.check_attention(O, None, want, want_lse, ref.attention_bounds(*clean, torch.float32, 243))
    assert (O[:7] == 3.25).all() and (O[300:] == 3.25).all()
    assert (O[60:171] == 0).all() and torch.isinf(LSE[60:171]).all()


def test_one_token_may_have_any_stride():
    gen = torch.Generator(device="cuda").manual_seed(2)
    buf = torch.randn(4096, generator=gen, device="cuda", dtype=torch.float16)
    Q, K = buf.as_strided((1, 4, 128), (3, 128, 1)), buf.as_strided((1, 2, 128), (5, 128, 1), 1024)
    run([1], (4, 2, 128), tensors=(Q, K, K))
    Q1, K1 = kf.qk_norm_rope(Q, K, ints([7]), kf.rope_freqs(128, device="cuda")[0])
    Q2, K2 = kf.qk_norm_rope(Q.contiguous(), K.contiguous(), ints([7]), kf.rope_freqs(128, device="cuda")[0])
    assert torch.equal(Q1, Q2) and torch.equal(K1, K2)


def test_a_key_of_another_sequence_does_not_reach_its_neighbours():
    """NaN and infinities in the keys and values of one sequence: the others' bits."""
    Q, K, V = make([100, 40, 77], (8, 2, 128), torch.float16)
    s = ints([0, 100, 140, 217])
    want = kf.attn_packed(Q, K, V, s, causal=True)
    K[100:140], V[100:140] = math.nan, math.inf
    got = kf.attn_packed(Q, K, V, s, causal=True)
    assert torch.equal(got[:100], want[:100]) and torch.equal(got[140:], want[140:])


def test_starts_outside_the_tensors_are_clamped():
    Q, K, V = make([100], (4, 2, 64), torch.float16)
    a = kf.attn_packed(Q, K, V, ints([-5, 40, 1 << 30]), causal=True)
    b = kf.attn_packed(Q, K, V, ints([0, 40, 100]), causal=True)
    assert torch.equal(a, b)


def test_scores_of_one_size_and_of_extreme_sizes():
    """Constant scores (uniform weights) and scores whose exponentials
    overflow without the running maximum."""
    Q, K, V = make([257], (4, 2, 128), torch.float16, seed=3)
    Q.zero_()
    O, LSE = kf.attn_packed(Q, K, V, ints([0, 257]), causal=True, return_lse=True)
    mean = V.double().cumsum(0) / torch.arange(1, 258, device="cuda", dtype=torch.float64)[:, None, None]
    # Weights of 1 are exact; 257 terms are summed in 32 bits.
    assert float((O.double().view(257, 2, 2, 128) - mean[:, :, None]).abs().max()) < 300 * 2.0 ** -24 * 6
    assert float((LSE[:, 0].double() - torch.arange(1, 258, device="cuda").double().log()).abs().max()) < 2.0 ** -18
    Q, K, V = make([257], (4, 2, 128), torch.float16, seed=4)
    run([257], (4, 2, 128), tensors=(Q * 16, K * 16, V))


def test_the_result_does_not_depend_on_the_neighbours():
    Q, K, V = make([900], (8, 2, 128), torch.float16)
    whole = kf.attn_packed(Q, K, V, ints([0, 333, 900]), causal=True)
    one = kf.attn_packed(Q[333:], K[333:], V[333:], ints([0, 567]), causal=True)
    assert torch.equal(whole[333:], one)
    again = kf.attn_packed(Q, K, V, ints([0, 333, 900]), causal=True)
    assert torch.equal(whole, again)


def test_offsets_past_32_bits():
    """A token stride that puts the last tokens more than 4 GiB away."""
    stride, T = 1 << 22, 600
    buf = torch.empty(T * stride, dtype=torch.float16, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(1)
    data = [torch.randn(T, h, 128, generator=gen, device="cuda", dtype=torch.float16) for h in (4, 2, 2)]
    views, at = [], 0
    for x in data:
        v = buf.as_strided(x.shape, (stride, 128, 1), at)
        v.copy_(x)
        at += x.shape[1] * 128
        views.append(v)
    s = ints([0, 100, T])
    assert torch.equal(kf.attn_packed(*views, s, causal=True), kf.attn_packed(*data, s, causal=True))


@pytest.mark.parametrize("D", [64, 128, 256])
def test_the_widest_key_stride(D):
    """A copy's 8, 4 or 2 rows of 512 MiB each: 32-bit offsets with the top bit set."""
    T, stride = 36, 1 << 28
    buf = torch.empty((T - 1) * stride + 2 * D, dtype=torch.float16, device="cuda")
    Q, K, V = make([T], (4, 1, D), torch.float16)
    views = []
    for i, x in enumerate((K, V)):
        v = buf.as_strided(x.shape, (stride, D, 1), i * D)
        v.copy_(x)
        views.append(v)
    s = ints([0, T])
    got = kf.attn_packed(Q, *views, s, causal=True)
    assert torch.equal(got, kf.attn_packed(Q, K, V, s, causal=True))


def test_other_streams_and_graphs():
    Q, K, V = make([64, 500], (8, 2, 128), torch.float16)
    s = ints([0, 64, 564])
    want = kf.attn_packed(Q, K, V, s, causal=True, out_dtype=torch.float16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = kf.attn_packed(Q, K, V, s, causal=True, out_dtype=torch.float16, stream=side)
    side.synchronize()
    assert torch.equal(got, want)
    out = torch.empty_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kf.attn_packed(Q, K, V, s, out, causal=True, out_dtype=torch.float16)
    for cut in (64, 10, 500, 0):
        s.copy_(ints([0, cut, 564]))
        Q.mul_(0.9)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, kf.attn_packed(Q, K, V, s, causal=True, out_dtype=torch.float16))


def test_refusals():
    Q, K, V = make([20], (4, 2, 128), torch.float16)
    s = ints([0, 20])
    for bad in (lambda: kf.attn_packed(Q.float(), K, V, s), lambda: kf.attn_packed(Q, K.bfloat16(), V, s)):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: kf.attn_packed(Q, K[:, :, :64], V, s), lambda: kf.attn_packed(Q, K, V[:10], s),
                lambda: kf.attn_packed(Q, K, V, s.long()), lambda: kf.attn_packed(Q, K, V, s[:1]),
                lambda: kf.attn_packed(Q, K, V, s, kv_starts=ints([0, 5, 20])),
                lambda: kf.attn_packed(Q, K, V, s.cpu()), lambda: kf.attn_packed(Q[0], K, V, s),
                lambda: kf.attn_packed(Q.transpose(1, 2), K, V, s),
                lambda: kf.attn_packed(Q, K, V, s, torch.empty(20, 4, 64, device="cuda")),
                lambda: kf.attn_packed(Q.requires_grad_(), K, V, s)):
        with pytest.raises(ValueError):
            bad()
    with torch.no_grad():
        kf.attn_packed(Q, K, V, s)
    with pytest.raises(kf.KfError) as e:
        kf.attn_packed(Q.detach()[:, :3].contiguous(), K, V, s)
    assert e.value.status == kf.KF_ERR_GQA
