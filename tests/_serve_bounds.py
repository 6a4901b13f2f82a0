"""Attention in 64 bits with an elementwise bound of what the kernels' roundings
may do to it.

With e_j = exp(s_j - m), w_j = e_j / sum e and O_d = sum_j w_j v_jd:

* A weight e_j is rounded to the 16-bit type before it meets V: e_j (1 + d_j), |d_j|
  <= h = 2^-11 (fp16) or 2^-8 (bf16).  O moves by sum_j w_j d_j v_jd.  For up to 64 keys
  that is at most h sum |w_j v_jd| <= 8 h sqrt(sum (w_j v_jd)^2) (Cauchy); for more,
  d_j are as independent numbers of mean zero, and by Hoeffding's inequality a
  sum beyond 8 h sqrt(sum (w_j v_jd)^2) has a probability below 2 exp(-32) = 3e-14.
* fp16 weights below 2^-14 are off by 2^-25 instead; the largest of a row is at least 1,
  so sum e >= 1, and O moves by 8 2^-25 sqrt(sum v_jd^2) at most, likewise.
* Scores: D products summed in 32 bits, the scale, the subtraction and the
  exponential: each weight relative u ((D + 8) |q| |k| / sqrt(D) + 8), u = 2^-24,
  in the numerator and the denominator.
* Sums over the keys in 32 bits: 16 keys to a product, 32 to a step of the row's sum, a
  few more for lanes, partials and rescalings: relative u (keys / 16 + keys / 32 + 64).
* O is rounded to its own type.
"""
import math

import torch

U = 2.0 ** -24


def attention(q, k, v, causal, dtype):
    """q [H_q, n, D], k and v [H_kv, m, D] in 64 bits, of which the kernel had `dtype`
    -> O [H_q, n, D], LSE [H_q, n], bound of O before its last rounding."""
    H_q, n, D = q.shape
    m, ratio = k.shape[1], H_q // k.shape[0]
    out, lse, off = torch.zeros_like(q), q.new_full((H_q, n), -math.inf), torch.zeros_like(q)
    if m == 0 or n == 0:
        return out, lse, off
    half = torch.finfo(dtype).eps / 2
    seen = torch.ones(n, m, dtype=torch.bool, device=q.device)
    if causal:
        seen = torch.arange(m, device=q.device) <= torch.arange(n, device=q.device)[:, None] + (m - n)
    some = seen.any(1)[:, None]
    for h in range(H_q):
        kh, vh = k[h // ratio], v[h // ratio]
        s = (q[h] @ kh.t().contiguous() / math.sqrt(D)).masked_fill(~seen, -math.inf)
        lse[h] = torch.logsumexp(s, 1)
        w = torch.exp(s - torch.where(some, lse[h][:, None], 0.0))
        out[h] = w @ vh
        size = q[h].norm(dim=1, keepdim=True) * kh.norm(dim=1).max() / math.sqrt(D)
        fp32 = 2 * U * ((D + 8) * size + 8) + U * (m / 16 + m / 32 + 64)
        off[h] = 8 * half * torch.sqrt((w * w) @ (vh * vh)) + fp32 * (w @ vh.abs())
        if dtype == torch.float16:
            off[h] += 8 * 2.0 ** -25 * torch.sqrt(seen.double() @ (vh * vh))
    return out, lse, off


def check(O, want, off):
    """O within `off` of `want`, and its own rounding."""
    info = torch.finfo(O.dtype)
    rounding = info.eps / 2 * (want.abs() + off) + info.tiny * info.eps / 2
    worst = ((O.double() - want).abs() / (off + rounding)).max() if O.numel() else torch.zeros(())
    assert torch.isfinite(O).all() and float(worst) <= 1.0, float(worst)


def check_lse(LSE, want, q, k, keys):
    """The log-sum-exp sums unrounded weights: the scores' and the sum's errors, and
    its own rounding."""
    D = q.shape[-1]
    size = float(q.norm(dim=-1).max() * k.norm(dim=-1).max()) / math.sqrt(D) if k.numel() else 0.0
    some = torch.isfinite(want)
    assert torch.equal(LSE[~some].double(), want[~some])
    if some.any():
        worst = float((LSE.double() - want)[some].abs().max())
        assert worst <= U * ((D + 10) * size + keys + 32), worst
