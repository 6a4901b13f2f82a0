"""Plain 64-bit forms of the serving operators, a sequence and a head at a
time, for the tests: packed attention, norm and rotary positions, and the 4-bit
rows.  On the CPU or the GPU, without the library."""
import math

import torch

def exp2i(e):
    """2^e of an integer tensor in 64 bits, by its bits (a library's power is only near it)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


LEVELS = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def attention(q, k, v, causal):
    """q [H_q, n, D], k and v [H_kv, m, D] in 64 bits -> O [H_q, n, D], LSE [H_q, n]."""
    H_q, n, D = q.shape
    m, ratio = k.shape[1], H_q // k.shape[0]
    out, lse = torch.zeros_like(q), torch.full(q.shape[:2], -math.inf, dtype=q.dtype, device=q.device)
    if m == 0:
        return out, lse
    for h in range(H_q):
        s = q[h] @ k[h // ratio].t().contiguous() / math.sqrt(D)
        if causal:
            seen = torch.arange(m, device=q.device) <= torch.arange(n, device=q.device)[:, None] + (m - n)
            s = s.masked_fill(~seen, -math.inf)
        lse[h] = torch.logsumexp(s, 1)
        w = torch.exp(s - lse[h][:, None])
        out[h] = torch.where(torch.isinf(lse[h])[:, None], torch.zeros_like(w), w) @ v[h // ratio]
    return out, lse


def packed(Q, K, V, q_starts, k_starts, causal):
    """Rows outside the sequences stay NaN."""
    out = torch.full(Q.shape, math.nan, dtype=torch.float64, device=Q.device)
    lse = out[..., 0].clone()
    for q0, q1, k0, k1 in zip(q_starts[:-1], q_starts[1:], k_starts[:-1], k_starts[1:]):
        q, k, v = (x.double().transpose(0, 1).contiguous() for x in (Q[q0:q1], K[k0:k1], V[k0:k1]))
        o, e = attention(q, k, v, causal)
        out[q0:q1], lse[q0:q1] = o.transpose(0, 1), e.transpose(0, 1)
    return out, lse


def attention_bounds(Q, K, V, out_dtype, keys):
    """How far O and the LSE may be off, elementwise, for finite inputs.

    A weight p (at most 2^8, the largest of a row at least 1) is rounded to the
    16-bit type: relative 2^-11 (fp16) or 2^-8 (bf16), and fp16's weights
    below 2^-14 by 2^-25 at most; D products of a score are summed in 32 bits
    (relative 2^-24 a term of |q| |k|), the exponential and the sums over the
    keys likewise.  O is an average of V's rows with those weights, over the sum
    of the unrounded ones; then it is rounded to its own type."""
    half = torch.finfo(Q.dtype).eps / 2
    D, u = Q.shape[-1], 2.0 ** -24
    finite = [torch.nan_to_num(x.double(), 0.0, 0.0, 0.0) for x in (Q, K, V)]
    size = float(finite[0].norm(dim=-1).max() * finite[1].norm(dim=-1).max()) / math.sqrt(D)
    score = u * ((D + 4) * size + 4)
    lse = score + u * (keys + 16) + u * size
    top = float(finite[2].abs().max())
    weights = half + (keys * 2.0 ** -25 if Q.dtype == torch.float16 else 0.0) + 2 * score + 2 * u * (keys + 16)
    return weights * top, (torch.finfo(out_dtype).eps / 2), lse


def check_attention(O, LSE, ref, ref_lse, bounds):
    off, rel, lse_off = bounds
    here = ~torch.isnan(ref)
    err = (O.double() - ref).abs() - rel * ref.abs()
    worst = float(err[here].max()) if here.any() else 0.0
    assert torch.isfinite(O[here]).all() and worst <= off, (worst, off)
    if LSE is not None:
        some = torch.isfinite(ref_lse)
        assert torch.equal(LSE[~some & ~torch.isnan(ref_lse)].double(), ref_lse[~some & ~torch.isnan(ref_lse)])
        if some.any():
            d = float((LSE.double() - ref_lse)[some].abs().max())
            assert d <= lse_off, (d, lse_off)


def norm_rope(x, w, eps, positions, freqs, interleaved, scale):
    """[T, H, D] in 64 bits -> turned rows, and per channel the sum of the magnitudes
    that make it up."""
    y = x.double()
    if w is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * w.double()
    out, mag = y.clone(), y.abs()
    half = 0 if freqs is None else freqs.shape[0]
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        angle = positions.double() * freqs[i]
        c, s = torch.cos(angle)[:, None] * scale, torch.sin(angle)[:, None] * scale
        out[..., a] = y[..., a] * c - y[..., b] * s
        out[..., b] = y[..., b] * c + y[..., a] * s
        both = (y[..., a].abs() + y[..., b].abs()) * abs(scale)
        mag[..., a] = mag[..., b] = both
    return out, mag


def quantise(x):
    """[..., D] -> the values of its 4-bit form, in 64 bits; finite inputs."""
    b = x.double().unflatten(-1, (-1, 32))
    top = b.abs().amax(-1, keepdim=True)
    # floor(log2) by frexp: exact, also of subnormals (E is at least 1 then).
    e = torch.frexp(top)[1] - 1
    unit = exp2i(torch.where(top > 0, e - 2, torch.full_like(e, -126)).clamp(min=-126))
    levels = LEVELS.to(x.device)
    a = b.abs() / unit
    # Ties to the even code: distances compared, the even code first.
    d = (a[..., None] - levels).abs()
    order = torch.tensor([0, 2, 4, 6, 1, 3, 5, 7], device=x.device)
    code = order[d[..., order].argmin(-1)]
    return (torch.sign(b) * levels[code] * unit).flatten(-2)


def unpack(pages, D, dtype=torch.float64):
    """Page pools [num_pages, H_kv, bytes] -> values [num_pages, H_kv, page_size, D]."""
    rows = pages.shape[2] * 32 // (17 * D)
    cut = rows * (D // 2)
    codes, E = pages[..., :cut].unflatten(-1, (rows, D // 2)), pages[..., cut:].unflatten(-1, (rows, D // 32))
    both = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()
    v = LEVELS.to(pages.device)[both & 7] * (1.0 - 2.0 * (both >> 3).double())
    v = v.unflatten(-1, (-1, 32)) * exp2i(E.int() - 127)[..., None]
    return v.flatten(-2).to(dtype)
