"""kf_qk_norm_rope against the plain 64-bit form."""
import pytest
import torch

import kernelfoundry_amd as kf
from tests import _serve_ref as ref

pytestmark = pytest.mark.gpu


def make(T, H_q, H_kv, D, dtype, seed=0, fused=False):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(T, (H_q + 2 * H_kv) * D, generator=gen, device="cuda", dtype=dtype)
    Q, K, _ = (v.unflatten(1, (-1, D)) for v in x.split((H_q * D, H_kv * D, H_kv * D), 1))
    if not fused:
        Q, K = Q.contiguous(), K.contiguous()
    w = [(1 + 0.2 * torch.randn(D, generator=gen, device="cuda", dtype=dtype)) for _ in range(2)]
    return Q, K, w


def check(got, x, w, eps, positions, freqs, interleaved, scale):
    """Rounding to the output type, and 64 units of 2^-24 of the magnitudes that
    make a channel up: the norm's sum (D / 8 terms in a lane, then halving: at
    most 38 roundings, halved by the root), sine, cosine (2^-25 of the series'
    end and 4 roundings of up to 1) and 5 products and sums."""
    want, mag = ref.norm_rope(x, w, eps, positions, freqs, interleaved, scale)
    # Below the type's least normal number a rounding is half its last place.
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    room = torch.finfo(got.dtype).eps / 2 * want.abs() + 64 * 2.0 ** -24 * mag + tiny
    err = (got.double() - want).abs()
    assert (err <= room).all(), float((err / room).max())


@pytest.mark.parametrize("D,rot", [(16, 16), (64, 64), (64, 32), (64, 48), (128, 128), (128, 64), (128, 16),
                                   (128, 112), (256, 256), (256, 64), (256, 208)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("norm", [False, True])
def test_layouts_parts_and_types(D, rot, interleaved, dtype, norm):
    Q, K, w = make(37, 5, 2, D, dtype, fused=True)
    freqs, _ = kf.rope_freqs(rot, device="cuda")
    pos = torch.randint(0, 1 << 20, (37,), device="cuda", dtype=torch.int32)
    qw, kw = w if norm else (None, None)
    Qo, Ko = kf.qk_norm_rope(Q, K, pos, freqs, q_weight=qw, k_weight=kw, eps=1e-5, interleaved=interleaved, scale=1.25)
    assert Qo.is_contiguous() and Qo.dtype == dtype
    check(Qo, Q, qw, 1e-5, pos, freqs, interleaved, 1.25)
    check(Ko, K, kw, 1e-5, pos, freqs, interleaved, 1.25)


@pytest.mark.parametrize("T", [1, 2, 3, 5, 255, 2559, 2560, 4095, 4099, 9001])
@pytest.mark.parametrize("heads", [(32, 8, 128), (1, 1, 64), (3, 1, 256), (40, 1, 16)])
def test_token_and_head_counts(T, heads):
    if T > 5000 and heads[0] > 4:
        T = 5001
    H_q, H_kv, D = heads
    Q, K, w = make(T, H_q, H_kv, D, torch.float16)
    freqs, _ = kf.rope_freqs(D, device="cuda")
    pos = torch.arange(T, device="cuda", dtype=torch.int32)
    Qo, Ko = kf.qk_norm_rope(Q, K, pos, freqs, q_weight=w[0], k_weight=w[1])
    check(Qo, Q, w[0], 1e-6, pos, freqs, False, 1.0)
    check(Ko, K, w[1], 1e-6, pos, freqs, False, 1.0)


@pytest.mark.parametrize("scaling", [None, "linear", "ntk", "yarn"])
def test_far_and_negative_positions_in_scaled_contexts(scaling):
    Q, K, w = make(11, 4, 2, 128, torch.float16)
    freqs, scale = kf.rope_freqs(128, scaling=scaling, factor=8.0 if scaling else 1.0, original_len=8192, device="cuda")
    pos = torch.tensor([0, 1, -1, -1000, 8191, 65535, 1 << 20, (1 << 20) + 1, 1 << 24, 2 ** 31 - 1, -2 ** 31],
                       device="cuda", dtype=torch.int32)
    Qo, Ko = kf.qk_norm_rope(Q, K, pos, freqs, scale=scale)
    # (2^31 radians in 64 bits are known to 2^-22; the reference has the same.)
    near = pos.abs() <= 1 << 24
    near &= pos != -2 ** 31
    check(Qo[near], Q[near], None, 0, pos[near], freqs, False, scale)
    check(Ko[near], K[near], None, 0, pos[near], freqs, False, scale)
    assert torch.isfinite(Qo).all()


def test_norm_alone_and_rotation_of_nothing():
    Q, K, w = make(9, 4, 2, 128, torch.bfloat16)
    Qo, Ko = kf.qk_norm_rope(Q, K, None, None, q_weight=w[0])
    check(Qo, Q, w[0], 1e-6, None, None, False, 1.0)
    assert torch.equal(Ko, K)
    freqs, _ = kf.rope_freqs(128, device="cuda")
    Qo, Ko = kf.qk_norm_rope(Q, K, torch.zeros(9, device="cuda", dtype=torch.int32), freqs)
    assert torch.equal(Qo, Q) and torch.equal(Ko, K)


def test_zero_rows_and_large_values():
    Q, K, w = make(4, 4, 2, 64, torch.float16)
    Q[0] = 0
    Q[1] = 60000.0
    Q[2] = 2.0 ** -24
    pos = torch.zeros(4, device="cuda", dtype=torch.int32)
    Qo, _ = kf.qk_norm_rope(Q, K, pos, kf.rope_freqs(64, device="cuda")[0], q_weight=w[0], k_weight=w[1])
    check(Qo, Q, w[0], 1e-6, pos, kf.rope_freqs(64, device="cuda")[0], False, 1.0)
    assert (Qo[0] == 0).all()


def test_in_place_equals_out_of_place():
    for fused in (False, True):
        Q, K, w = make(300, 8, 2, 128, torch.float16, fused=fused)
        freqs, _ = kf.rope_freqs(96, device="cuda")
        pos = torch.arange(300, device="cuda", dtype=torch.int32)
        want = kf.qk_norm_rope(Q, K, pos, freqs, q_weight=w[0], k_weight=w[1])
        got = kf.qk_norm_rope(Q, K, pos, freqs, (Q, K), q_weight=w[0], k_weight=w[1])
        assert got[0] is Q and torch.equal(Q, want[0]) and torch.equal(K, want[1])


def test_turning_back_and_relative_positions():
    """Rotation by -p undoes rotation by p, and scores depend on the distance."""
    Q, K, _ = make(64, 2, 2, 128, torch.float16)
    freqs, _ = kf.rope_freqs(128, device="cuda")
    pos = torch.arange(1000, 1064, device="cuda", dtype=torch.int32)
    there = kf.qk_norm_rope(Q, K, pos, freqs)
    back, _ = kf.qk_norm_rope(*there, -pos, freqs)
    # Two roundings of fp16 of values of at most the pair's length.
    assert float((back.double() - Q.double()).abs().max()) <= 2 * 2.0 ** -11 * 1.5 * float(Q.abs().max())


def test_streams_and_graphs():
    Q, K, w = make(33, 8, 2, 128, torch.float16)
    freqs, _ = kf.rope_freqs(128, device="cuda")
    pos = torch.arange(33, device="cuda", dtype=torch.int32)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = kf.qk_norm_rope(Q, K, pos, freqs, stream=side)
    side.synchronize()
    assert torch.equal(got[0], kf.qk_norm_rope(Q, K, pos, freqs)[0])
    out = torch.empty_like(Q), torch.empty_like(K)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kf.qk_norm_rope(Q, K, pos, freqs, out, q_weight=w[0])
    for step in range(4):
        pos.add_(17)
        graph.replay()
        torch.cuda.synchronize()
        want = kf.qk_norm_rope(Q, K, pos, freqs, q_weight=w[0])
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_refusals():
    Q, K, w = make(8, 4, 2, 128, torch.float16)
    freqs, _ = kf.rope_freqs(128, device="cuda")
    pos = torch.arange(8, device="cuda", dtype=torch.int32)
    for bad in (lambda: kf.qk_norm_rope(Q.float(), K, pos, freqs), lambda: kf.qk_norm_rope(Q, K.bfloat16(), pos, freqs),
                lambda: kf.qk_norm_rope(Q, K, pos, freqs, q_weight=w[0].float())):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: kf.qk_norm_rope(Q, K[:4], pos, freqs), lambda: kf.qk_norm_rope(Q, K, pos.long(), freqs),
                lambda: kf.qk_norm_rope(Q, K, pos[:4], freqs), lambda: kf.qk_norm_rope(Q, K, pos, freqs.float()),
                lambda: kf.qk_norm_rope(Q, K, None, freqs), lambda: kf.qk_norm_rope(Q, K, pos, freqs.cpu()),
                lambda: kf.qk_norm_rope(Q, K, pos, freqs, q_weight=w[0][:64]),
                lambda: kf.qk_norm_rope(Q, K, pos, freqs, (torch.empty_like(Q)[:4], torch.empty_like(K))),
                lambda: kf.qk_norm_rope(Q, K, pos, freqs,
                                        (torch.empty(4, 8, 128, dtype=Q.dtype, device="cuda").transpose(0, 1),
                                         torch.empty_like(K))),
                lambda: kf.qk_norm_rope(Q, K.requires_grad_(), pos, freqs)):
        with pytest.raises(ValueError):
            bad()
    K.requires_grad_(False)
    with pytest.raises(kf.KfError) as e:
        kf.qk_norm_rope(Q, K, pos, freqs[:4].contiguous())
    assert e.value.status == kf.KF_ERR_SIZE
