"""Calls that the serving entry points refuse or bound, on the GPU."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

import kernelfoundry_amd as kf
from tests.test_kv4_gpu import fill, ints, normal

pytestmark = pytest.mark.gpu


def calls():
    """Per differentiable argument of an entry: its value, and the entry as a function of it."""
    Kp, Vp, table, _, _ = fill([20], 2, 128, 16)
    Q, K, V, s, n = normal(20, 8, 128), normal(20, 2, 128), normal(20, 2, 128, seed=1), ints([0, 20]), ints([20])
    w, f, pos = normal(128), kf.rope_freqs(128, device="cuda")[0], ints(list(range(20)))
    return {
        "packed Q": (Q, lambda x: kf.attn_packed(x, K, V, s)), "packed K": (K, lambda x: kf.attn_packed(Q, x, V, s)),
        "packed V": (V, lambda x: kf.attn_packed(Q, K, x, s)),
        "rope Q": (Q, lambda x: kf.qk_norm_rope(x, K, pos, f)), "rope K": (K, lambda x: kf.qk_norm_rope(Q, x, pos, f)),
        "rope q_weight": (w, lambda x: kf.qk_norm_rope(Q, K, pos, f, q_weight=x)),
        "rope k_weight": (w, lambda x: kf.qk_norm_rope(Q, K, pos, f, k_weight=x)),
        "rope freqs": (f, lambda x: kf.qk_norm_rope(Q, K, pos, x)),
        "append K": (K, lambda x: kf.kv4_append(x, V, Kp, Vp, table, s, n)),
        "append V": (V, lambda x: kf.kv4_append(K, x, Kp, Vp, table, s, n)),
        "decode Q": (Q[:1, :, None], lambda x: kf.attn_decode_kv4(x, Kp, Vp, table, n)),
    }


def test_an_input_that_requires_grad_is_refused():
    for name, (x, call) in calls().items():
        call(x)
        leaf = x.detach().clone().requires_grad_()
        with pytest.raises(ValueError, match="requires grad"):
            call(leaf)
            pytest.fail(name)
        with torch.no_grad():
            call(leaf)


def test_an_input_with_a_tangent_is_refused():
    for name, (x, call) in calls().items():
        with fwd.dual_level():
            call(x)
            dual = fwd.make_dual(x, torch.ones_like(x))
            with pytest.raises(ValueError, match="tangent"):
                call(dual)
                pytest.fail(name)
            with torch.no_grad(), pytest.raises(ValueError, match="tangent"):
                call(dual)
                pytest.fail(name)
        call(x)
        # torch.func's wrapped tensors have no memory of their own.
        with pytest.raises((ValueError, RuntimeError)):
            torch.func.jvp(call, (x,), (torch.ones_like(x),))
            pytest.fail(name)


def test_calls_without_tokens_rows_or_pages_are_refused():
    Kp, Vp, table, _, _ = fill([20], 2, 128, 16)
    Q, K, s, n, f = normal(20, 8, 128), normal(20, 2, 128), ints([0, 20]), ints([20]), kf.rope_freqs(128, device="cuda")[0]
    none = ints([0, 0])
    for call in (lambda: kf.attn_packed(Q[:0], K, K, none, kv_starts=s), lambda: kf.attn_packed(Q, K[:0], K[:0], s, kv_starts=none),
                 lambda: kf.qk_norm_rope(Q[:0], K[:0], n[:0], f), lambda: kf.kv4_append(K[:0], K[:0], Kp, Vp, table, none, n),
                 lambda: kf.kv4_append(K, K, Kp, Vp, table[:, :0].contiguous(), s, n),
                 lambda: kf.kv4_append(K, K, Kp[:0], Vp[:0], table, s, n),
                 lambda: kf.kv4_read(Kp, Vp, table, none, n, 0, 128),
                 lambda: kf.attn_decode_kv4(Q[:0, :, None], Kp, Vp, table[:0], n[:0]),
                 lambda: kf.attn_decode_kv4(Q[:1, :, None], Kp[:0], Vp[:0], table, n)):
        with pytest.raises(kf.KfError) as e:
            call()
        assert e.value.status == kf.KF_ERR_SIZE
    with pytest.raises(ValueError):
        kf.attn_packed(Q, K, K, s[:1])
    # Sequences without tokens or keys among others.
    O, LSE = kf.attn_packed(Q, K, K, ints([0, 0, 20, 20]), kv_starts=ints([0, 20, 20, 20]), return_lse=True)
    assert (O == 0).all() and (LSE == -float("inf")).all()
