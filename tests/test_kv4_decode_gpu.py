"""attn_decode_kv4 against a 64-bit form with an elementwise bound, and the
same values read back; blocks that stand for NaN."""
import math

import pytest
import torch

import kernelfoundry_amd as kf
from tests import _serve_bounds as bounds
from tests import _serve_ref as ref
from tests.test_kv4_gpu import fill, ints, new_cache, normal, starts_of

pytestmark = pytest.mark.gpu

HEADS = [(8, 2, 64), (8, 2, 128), (8, 2, 256), (24, 1, 64), (32, 1, 128), (20, 1, 256)]


def against_64_bits(lens, heads, q_len, dtype, out_dtype, causal=True, page_size=16, seed=0):
    H_q, H_kv, D = heads
    Kp, Vp, table, K4, V4 = fill(lens, H_kv, D, page_size, dtype, seed)
    Q = normal(len(lens), H_q, q_len, D, dtype=dtype, seed=seed + 9)
    run = lambda: kf.attn_decode_kv4(Q, Kp, Vp, table, ints(lens), causal=causal, out_dtype=out_dtype, return_lse=True)
    O, LSE = run()
    again = run()
    assert torch.equal(O, again[0]) and torch.equal(LSE, again[1])
    s = starts_of(lens)
    for b, m in enumerate(lens):
        q = Q[b].double()
        k, v = (x[s[b]:s[b + 1]].transpose(0, 1).contiguous() for x in (K4, V4))
        want, lse, off = bounds.attention(q, k, v, causal, dtype)
        bounds.check(O[b], want, off)
        bounds.check_lse(LSE[b], lse, q, k, m)


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_elementwise(heads, dtype, out_dtype):
    against_64_bits([1, 0, 31, 33, 700, 100], heads, 1, dtype, out_dtype)


@pytest.mark.parametrize("heads,q_len", [((8, 2, 128), 8), ((8, 2, 64), 3), ((4, 2, 256), 5), ((8, 1, 64), 4)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_elementwise_of_several_tokens(heads, q_len, dtype):
    against_64_bits([2, 333, q_len, 0, 2000], heads, q_len, dtype, dtype)


@pytest.mark.parametrize("heads", [(8, 2, 128), (32, 1, 64), (4, 2, 256)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_elementwise_of_long_sequences(heads, dtype):
    against_64_bits([9000, 17, 20011], heads, 1, dtype, torch.float32, page_size=64)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows", [4, 24])
@pytest.mark.parametrize("keys", [70, 9000])      # of one wave and of many
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_a_block_without_finite_values_is_nan(D, dtype, rows, keys, bad):
    """Its key makes the rows of its KV head NaN, its value their 32 channels, as
    the rows read back do in attn_packed; other heads and sequences keep their bits."""
    lens, H_kv, at = [100, keys], 2, 137            # token 37 of the second sequence
    T, starts = sum(lens), ints(starts_of(lens))
    for which in ("K", "V"):
        Kp, Vp, table, _, _ = fill(lens, H_kv, D, 16, dtype)
        Q = normal(2, rows * H_kv, 1, D, dtype=dtype, seed=9)
        want = kf.attn_decode_kv4(Q, Kp, Vp, table, ints(lens))
        K, V = normal(T, H_kv, D, dtype=dtype), normal(T, H_kv, D, dtype=dtype, seed=1)
        (K if which == "K" else V)[at, 1, D - 27] = bad
        kf.kv4_append(K, V, Kp, Vp, table, starts, ints(lens))
        O = kf.attn_decode_kv4(Q, Kp, Vp, table, ints(lens))
        assert torch.equal(O[0], want[0]) and torch.equal(O[1, :rows], want[1, :rows])
        hit = torch.isnan(O[1, rows:, 0])
        assert hit.all() if which == "K" else hit[:, D - 32:].all()
        K, V = kf.kv4_read(Kp, Vp, table, starts, ints(lens), T, D, out_dtype=dtype)
        P = kf.attn_packed(Q[:, :, 0], K, V, ints([0, 1, 2]), kv_starts=starts)
        hit = torch.isnan(P[1, rows:])
        assert hit.all() if which == "K" else hit[:, D - 32:].all()
        assert torch.isfinite(P[0]).all() and torch.isfinite(P[1, :rows]).all()


def test_the_smallest_bf16_values_are_exact():
    """Every subnormal and the least normal numbers as a block's largest: written and
    read back without a flush to zero."""
    top = torch.arange(0x300, dtype=torch.int32).to(torch.int16).view(torch.bfloat16).cuda()
    part = torch.linspace(-1, 1, 31, device="cuda", dtype=torch.float64)
    x = torch.zeros(top.shape[0], 1, 64, device="cuda", dtype=torch.bfloat16)
    x[:, 0, 0], x[:, 0, 1:32] = top, (top.double()[:, None] * part).to(torch.bfloat16)
    n = x.shape[0]
    Kp, Vp, table = new_cache([n], 1, 64, 16)
    kf.kv4_append(x, x, Kp, Vp, table, ints([0, n]), ints([n]))
    K, V = kf.kv4_read(Kp, Vp, table, ints([0, n]), ints([n]), n, 64, out_dtype=torch.bfloat16)
    want = ref.quantise(x)
    assert torch.equal(K.double(), want) and torch.equal(V.double(), want)
