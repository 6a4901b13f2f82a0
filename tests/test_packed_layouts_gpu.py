"""Every layout of kf_attn_packed at every head dimension, with and without the
causal mask, for both input types and all output types, against a 64-bit form."""
import itertools
import math

import pytest
import torch

import kernelfoundry_amd as kf
from tests import _serve_bounds as bounds
from tests._packed_layout import layouts, packed_layout

# Queries and keys around tiles and stages; none, fewer and more keys than queries.
SHORT = ([1, 2, 33, 0, 64, 129, 31, 257, 300, 5], [1, 40, 7, 64, 200, 129, 0, 250, 301, 5])
CHUNK = ([200, 33], [2000, 1995])
# (D, layout): heads, (queries, keys) of the sequences.
CALLS = {
    (64, 0): ((64, 16, 64), SHORT), (64, 1): ((4, 1, 64), SHORT), (64, 2): ((4, 1, 64), CHUNK),
    (128, 0): ((32, 8, 128), SHORT), (128, 1): ((8, 2, 128), SHORT), (128, 2): ((8, 2, 128), CHUNK),
    (256, 0): ((6, 2, 256), SHORT), (256, 1): ((4, 1, 256), CHUNK),
}
# Several tiles of a sequence, in the layouts of long prompts.
LONG = {(64, 0): ((32, 8, 64), ([1500, 700, 1, 1100], [1500, 700, 1, 1100])),
        (128, 0): ((16, 4, 128), ([1500, 700, 1, 1100], [1500, 700, 1, 1100])),
        (256, 0): ((32, 8, 256), ([900, 700, 1, 500], [900, 700, 1, 500]))}
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


@pytest.mark.parametrize("causal", [True, False])
def test_the_calls_reach_every_layout(causal):
    assert {(D, i) for D, found in layouts().items() for i in range(len(found))} == set(CALLS)
    for (D, layout), (heads, lens) in itertools.chain(CALLS.items(), LONG.items()):
        assert packed_layout(heads, *lens, causal) == layout, (D, layout)


def starts_of(lens):
    return torch.tensor([0, *itertools.accumulate(lens)], dtype=torch.int32)


def run(layout, call, causal, dtype, out_dtype, seed):
    heads, (lens, kv_lens) = call
    H_q, H_kv, D = heads
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    assert packed_layout(heads, lens, kv_lens, causal, cus) == layout
    gen = torch.Generator(device="cuda").manual_seed(seed)
    Q, K, V = (torch.randn(sum(n), h, D, generator=gen, device="cuda").to(dtype)
               for n, h in ((lens, H_q), (kv_lens, H_kv), (kv_lens, H_kv)))
    qs, ks = starts_of(lens), starts_of(kv_lens)
    O, LSE = kf.attn_packed(Q, K, V, qs.cuda(), kv_starts=ks.cuda(), causal=causal, out_dtype=out_dtype, return_lse=True)
    again = kf.attn_packed(Q, K, V, qs.cuda(), kv_starts=ks.cuda(), causal=causal, out_dtype=out_dtype)
    assert O.dtype == out_dtype and torch.equal(O, again)
    for i, (n, m) in enumerate(zip(lens, kv_lens)):
        a, b = slice(int(qs[i]), int(qs[i + 1])), slice(int(ks[i]), int(ks[i + 1]))
        q, k, v = (x.double().transpose(0, 1).contiguous() for x in (Q[a], K[b], V[b]))
        want, lse, off = bounds.attention(q, k, v, causal, dtype)
        bounds.check(O[a].transpose(0, 1), want, off)
        if n:
            bounds.check_lse(LSE[a].transpose(0, 1), lse, q, k, m)


@pytest.mark.gpu
@pytest.mark.parametrize("key", CALLS, ids=lambda k: f"D{k[0]}-layout{k[1]}")
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("out_dtype", ["f32", "f16", "bf16"])
def test_layouts(key, causal, dtype, out_dtype):
    run(key[1], CALLS[key], causal, TYPES[dtype], TYPES[out_dtype], 11 * key[0] + key[1])


@pytest.mark.gpu
@pytest.mark.parametrize("key", LONG, ids=lambda k: f"D{k[0]}")
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_long_prompts(key, causal, dtype):
    run(key[1], LONG[key], causal, TYPES[dtype], TYPES[dtype], 5)


@pytest.mark.gpu
@pytest.mark.parametrize("key", CALLS, ids=lambda k: f"D{k[0]}-layout{k[1]}")
def test_views_between_other_values(key):
    """Rows of a wider tensor, whose other columns hold NaN, behind and in front of
    tokens that do: neither read; and no row outside the sequences written."""
    heads, (lens, kv_lens) = CALLS[key]
    H_q, H_kv, D = heads
    gen = torch.Generator(device="cuda").manual_seed(3)
    plain, views = [], []
    for n, h in ((lens, H_q), (kv_lens, H_kv), (kv_lens, H_kv)):
        x = torch.randn(sum(n), h, D, generator=gen, device="cuda").to(torch.bfloat16)
        wide = torch.full((sum(n) + 9, h, D + 24), math.nan, device="cuda", dtype=torch.bfloat16)
        wide[4: 4 + sum(n), :, 8: 8 + D] = x
        plain.append(x)
        views.append(wide[:, :, 8: 8 + D])
    qs, ks = starts_of(lens).cuda(), starts_of(kv_lens).cuda()
    want = kf.attn_packed(*plain, qs, kv_starts=ks, causal=True)
    out = torch.full((sum(lens) + 9, H_q, D), 3.25, device="cuda")
    kf.attn_packed(*views, qs + 4, out, kv_starts=ks + 4, causal=True)
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    # (The nine tokens beside the sequences count in the averages that the layout goes by.)
    more = [list(n[:-1]) + [n[-1] + 9] for n in (lens, kv_lens)]
    assert packed_layout(heads, *more, True, cus) == key[1]
    assert torch.equal(out[4:-5], want)
    assert torch.isfinite(out).all() and (out[:4] == 3.25).all() and (out[-5:] == 3.25).all()
