"""What a server runs beside the attention forward, on torch GPU tensors:
packed prompts, head norms with rotary positions, and a paged K/V cache in 4
bits with the decode that reads it (include/kf/attn.h: kf_attn_packed,
kf_qk_norm_rope, kf_kv4_append, kf_kv4_read, kf_attn_decode_kv4).

    freqs, scale = rope_freqs(128, scaling="yarn", factor=4.0, original_len=8192, device="cuda")
    Q, K = qk_norm_rope(Q, K, positions, freqs, q_weight=wq, k_weight=wk, scale=scale)
    kv4_append(K, V, K_pages, V_pages, block_table, seq_starts, kv_lens)
    O = attn_packed(Q, K, V, seq_starts, causal=True)                          # prompts
    O = attn_decode_kv4(Q, K_pages, V_pages, block_table, kv_lens)             # a step
    K, V = kv4_read(K_pages, V_pages, block_table, kv_starts, kv_lens, total, 128)
    O = attn_packed(Q, K, V, seq_starts, kv_starts=kv_starts, causal=True)     # a later chunk

The entries run asynchronously on ``stream``, one of the tensors' device (default:
torch's current one), and check their arguments on the host only; what device arrays hold
(sequence starts, key counts, page ids) is bounded by the kernels.  They have
no derivatives: an input that requires grad is refused while torch records
gradients, and one with a tangent always.  A call needs at least one token, sequence,
row of K and V and page (else KfError, KF_ERR_SIZE); a sequence among others may be
empty.  None of them has a counterpart in the reference.
"""
from __future__ import annotations

import ctypes
import functools
import math

from . import (KF_ATTN_CAUSAL, KF_ERR_HIP, KF_ERR_SIZE, KF_OK, KfError, _new, _out_flags, _output, _raw_stream,
               _workspace, load_library, status_string)

KF_BF16 = 16
KF_ROPE_INTERLEAVED = 32

_STRIDES = {n: ctypes.c_int64 * n for n in (4, 6, 8)}
_WIDE_STRIDE = 1 << 28   # of tokens: the most that attn_packed takes of K and V
_MOST = 2 ** 31 - 1      # a size of the C entries: an int, to which ctypes cuts without a word


# The checks below run on every call, and a small call's time is the host's:
# they compare by device index and identity, and look for words only when
# something is wrong.
def _gpu(torch, names, *tensors):
    """The device of tensors (or None, but the first) that are all on one GPU and
    record no gradient, backward or forward."""
    index = tensors[0].get_device()
    for t in tensors:
        if t is not None and (t.get_device() != index or index < 0 or t.requires_grad):
            break
    else:
        # Tangents exist only inside a level of forward-mode differentiation, whose
        # number torch keeps in a variable (a call a tensor where it has none).
        if getattr(torch.autograd.forward_ad, "_current_level", 0) < 0:
            return tensors[0].device
    for name, t in zip(names, tensors):
        if t is None:
            continue
        if t.get_device() != index or index < 0:
            where = tensors[0].device if index >= 0 else "a GPU"
            raise ValueError(f"{name} must be a GPU tensor, on {where}")
        if t.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{name} requires grad, but there is no backward pass: call under torch.no_grad()")
        if torch.autograd.forward_ad.unpack_dual(t).tangent is not None:
            raise ValueError(f"{name} has a tangent, but there is no forward-mode derivative")
    return tensors[0].device


def _half(torch, names, *tensors):
    """KF_BF16 or 0 by the one 16-bit type of the tensors."""
    dtype = tensors[0].dtype
    if dtype is not torch.float16 and dtype is not torch.bfloat16:
        raise TypeError(f"{names[0]} must be float16 or bfloat16")
    for t in tensors:
        if t.dtype is not dtype:
            raise TypeError(f"{' and '.join(names)} must be of one type")
    return KF_BF16 if dtype is torch.bfloat16 else 0


def _heads(name, t):
    """A [tokens, heads, D] tensor's token and head strides (0 where there is one
    token or head, whose stride may be anything): D contiguous."""
    if t.dim() != 3:
        raise ValueError(f"{name} must be [tokens, heads, D]")
    token, head, channel = t.stride()
    if channel != 1 or token % 8 or head % 8 or token > _WIDE_STRIDE:
        tokens, heads, D = t.shape
        token, head = token if tokens > 1 else 0, head if heads > 1 else 0
        if (channel != 1 and D > 1) or token % 8 or head % 8:
            raise ValueError(f"{name}: the channels must be contiguous, token and head strides multiples of 8")
    return token, head


def _ints(torch, name, t, device, shape):
    if t.dtype is not torch.int32 or t.get_device() != device.index or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor of shape {tuple(shape)} on {device}")
    return t.data_ptr()


def _starts(torch, name, t, device):
    if t.dim() != 1 or t.shape[0] < 2:
        raise ValueError(f"{name} must be [sequences + 1]")
    return _ints(torch, name, t, device, t.shape)


def _new_at(torch, t, shape, dtype, stream):
    """_new on t's device (new_empty takes less time than empty)."""
    return t.new_empty(shape, dtype=dtype) if stream is None else _new(torch, shape, dtype, t.device, stream)


def _like(torch, t, dtype, stream):
    """A new contiguous tensor of t's shape (empty_like takes less time again)."""
    if stream is None:
        return torch.empty_like(t, dtype=dtype, memory_format=torch.contiguous_format)
    return _new(torch, t.shape, dtype, t.device, stream)


def _too_many():
    return KfError(KF_ERR_SIZE, status_string(KF_ERR_SIZE))


def _launch(torch, device, stream, entry, *args):
    """entry(*args, stream) with `device` current: its streams are the current device's."""
    if stream is not None and stream.device != device:
        raise ValueError(f"stream must be a stream of {device}")
    if device.index == torch.cuda.current_device():
        st = entry(*args, _raw_stream(torch, stream, device))
    else:
        with torch.cuda.device(device):
            st = entry(*args, _raw_stream(torch, stream, device))
    if st != KF_OK:
        msg = status_string(st)
        if st == KF_ERR_HIP:
            msg += f" (hipError_t {load_library().kf_last_hip_error()})"
        raise KfError(st, msg)


def attn_packed(Q, K, V, seq_starts, out=None, *, kv_starts=None, causal=False, stream=None,
                out_dtype=None, return_lse=False):
    """Attention over packed sequences.

    Q [T, H_q, D], K and V [T_kv, H_kv, D], float16 or bfloat16, D = 64, 128 or
    256; views with other token and head strides (multiples of 8, those of K's and V's
    tokens at most 2^28), as those of a fused projection, are read in place.
    ``seq_starts`` int32 [N + 1]: sequence b has the tokens seq_starts[b] ..
    seq_starts[b + 1] - 1, none or more; ``kv_starts`` the same for the keys
    (default: seq_starts).  ``causal`` is aligned to the last key: query i of n
    sees keys j <= i + keys - n.
    Returns O [T, H_q, D] (fp32, or ``out_dtype``), or (O, LSE [T, H_q]) with
    ``return_lse``; a row without keys gets O = 0, LSE = -inf.  Rows outside
    the sequences are not written.  The softmax weights are rounded to the inputs' type
    before they meet V; scores q . k / sqrt(D) may reach 9e7.
    """
    import torch

    device = _gpu(torch, "QKV", Q, K, V)
    flags = _out_flags(torch, out_dtype, return_lse) | _half(torch, "QKV", Q, K, V)
    strides = _STRIDES[6](*_heads("Q", Q), *_heads("K", K), *_heads("V", V))
    T, H_q, D = Q.shape
    T_kv, H_kv, Dk = K.shape
    if V.shape != K.shape or Dk != D:
        raise ValueError("K and V must be [T_kv, H_kv, D], with Q's D")
    starts = kstarts = _starts(torch, "seq_starts", seq_starts, device)
    n = seq_starts.shape[0] - 1
    if T > _MOST or T_kv > _MOST or H_q > _MOST or H_kv > _MOST or n > _MOST:
        raise _too_many()
    if kv_starts is not None:
        kstarts = _ints(torch, "kv_starts", kv_starts, device, seq_starts.shape)
    if out is None:
        out = _like(torch, Q, out_dtype or torch.float32, stream)
    else:
        out = _output(torch, out, (T, H_q, D), out_dtype, device, stream)
    lse = _new_at(torch, Q, (T, H_q), torch.float32, stream) if return_lse else None
    if causal:
        flags |= KF_ATTN_CAUSAL
    _launch(torch, device, stream, load_library().kf_attn_packed,
            Q.data_ptr(), K.data_ptr(), V.data_ptr(), out.data_ptr(), lse.data_ptr() if return_lse else None, None,
            strides, starts, kstarts, n, T, T_kv, H_q, H_kv, D, flags)
    return (out, lse) if return_lse else out


def rope_freqs(rot, base=10000.0, *, scaling=None, factor=1.0, original_len=None, beta_fast=32.0,
               beta_slow=1.0, device=None):
    """Rotary frequencies [rot / 2] (float64, radians per position) and the
    factor that rotated channels are multiplied by, for qk_norm_rope.

    f_i = base ** (-2 i / rot), and for contexts ``factor`` times as long as
    those trained on, with ``scaling``:
    "linear"  f_i / factor (positions interpolated);
    "ntk"     base * factor ** (rot / (rot - 2)): the lowest frequency
              interpolated, the highest kept;
    "yarn"    by the turns f_i makes over ``original_len`` positions: kept from
              beta_fast turns on, interpolated up to beta_slow, in between
              linearly mixed; the rotated channels times 1 + ln(factor) / 10.  The
              mix is linear in the turns; a checkpoint that was tuned with one linear
              in the channel index brings its own frequencies.
    """
    import torch

    if rot <= 0 or rot % 2:
        raise ValueError("rot must be a positive even number of channels")
    if scaling not in (None, "linear", "ntk", "yarn"):
        raise ValueError('scaling must be None, "linear", "ntk" or "yarn"')
    if scaling is not None and factor < 1.0:
        raise ValueError("factor must be at least 1")
    if scaling == "ntk":
        if rot < 4:
            raise ValueError('scaling "ntk" needs rot >= 4')
        base = base * factor ** (rot / (rot - 2))
    i = torch.arange(rot // 2, dtype=torch.float64)
    freqs = float(base) ** (-2.0 * i / rot)
    scale = 1.0
    if scaling == "linear":
        freqs = freqs / factor
    elif scaling == "yarn":
        if not original_len or original_len <= 0:
            raise ValueError('scaling "yarn" needs original_len')
        if beta_fast <= beta_slow:
            raise ValueError("beta_fast must be above beta_slow")
        turns = original_len * freqs / (2.0 * math.pi)
        keep = ((turns - beta_slow) / (beta_fast - beta_slow)).clamp(0.0, 1.0)
        freqs = freqs * keep + freqs / factor * (1.0 - keep)
        scale = 1.0 + 0.1 * math.log(factor)
    return freqs.to(device) if device is not None else freqs, scale


def qk_norm_rope(Q, K, positions, freqs, out=None, *, q_weight=None, k_weight=None, eps=1e-6,
                 interleaved=False, scale=1.0, stream=None):
    """RMS norm of every query and key head, then rotary positions.

    Q [T, H_q, D], K [T, H_kv, D], float16 or bfloat16, D = 16, 64, 128 or 256,
    with any token and head strides (multiples of 8).  ``q_weight`` /
    ``k_weight`` [D] of the same type: x / sqrt(mean(x^2) + eps) * weight
    (None: not normed).  The first 2 * len(freqs) channels (a multiple of 16)
    are turned by positions[t] * freqs[i] (int32 [T]; float64, see rope_freqs) in the
    pairs (i, i + len(freqs)), or (2 i, 2 i + 1) with ``interleaved``, and
    multiplied by ``scale``.  ``positions`` and ``freqs`` None: no rotation.
    Returns new contiguous tensors, or ``out``, a pair that may be (Q, K)
    themselves.
    """
    import torch

    device = _gpu(torch, ("Q", "K", "q_weight", "k_weight", "freqs"), Q, K, q_weight, k_weight, freqs)
    flags = _half(torch, "QK", Q, K) | (KF_ROPE_INTERLEAVED if interleaved else 0)
    strides = (*_heads("Q", Q), *_heads("K", K))
    T, H_q, D = Q.shape
    T_k, H_kv, Dk = K.shape
    if T_k != T or Dk != D:
        raise ValueError("K must be [T, H_kv, D], with Q's T and D")
    if T > _MOST or H_q > _MOST or H_kv > _MOST:
        raise _too_many()
    wq = wk = pos = frq = None
    if q_weight is not None:
        wq = _weight(torch, "q_weight", q_weight, Q, D)
    if k_weight is not None:
        wk = _weight(torch, "k_weight", k_weight, Q, D)
    rot = 0
    if freqs is not None:
        if freqs.dtype is not torch.float64 or freqs.dim() != 1 or not freqs.is_contiguous():
            raise ValueError(f"freqs must be a contiguous float64 [rot / 2] tensor on {device}")
        rot, frq = 2 * freqs.shape[0], freqs.data_ptr()
        if positions is None:
            raise ValueError("freqs without positions")
        pos = _ints(torch, "positions", positions, device, (T,))
    if out is None:
        out = (_like(torch, Q, Q.dtype, stream), _like(torch, K, Q.dtype, stream))
        strides += (H_q * D, D, H_kv * D, D)
    else:
        for name, y, x in (("out[0]", out[0], Q), ("out[1]", out[1], K)):
            if y.shape != x.shape or y.dtype != x.dtype or y.device != device:
                raise ValueError(f"{name} must have the shape, type and device of its input")
            in_place = y.data_ptr() == x.data_ptr() and y.stride() == x.stride()
            if not (in_place or y.is_contiguous()):
                raise ValueError(f"{name} must be contiguous, or its input itself")
            strides += _heads(name, y)
    _launch(torch, device, stream, load_library().kf_qk_norm_rope,
            Q.data_ptr(), K.data_ptr(), out[0].data_ptr(), out[1].data_ptr(), _STRIDES[8](*strides), wq, wk, pos, frq,
            T, H_q, H_kv, D, rot, eps, scale, flags)
    return out


def _weight(torch, name, w, Q, D):
    if w.dtype is not Q.dtype:
        _half(torch, ("Q", name), Q, w)
    if w.shape != (D,) or not w.is_contiguous():
        raise ValueError(f"{name} must be a contiguous tensor of D elements")
    return w.data_ptr()


def kv4_page_bytes(page_size, D) -> int:
    """Bytes of one KV head's page of the 4-bit cache: pools are uint8 [num_pages,
    H_kv, kv4_page_bytes(page_size, D)] tensors."""
    n = int(load_library().kf_kv4_page_bytes(page_size, D))
    if n == 0:
        raise ValueError("page_size must be a power of two in [16, 2^20] and D 64, 128 or 256")
    return n


def _pages(torch, K_pages, V_pages, D):
    """num_pages, H_kv and page_size of a pair of pools."""
    if K_pages.dim() != 3 or K_pages.shape != V_pages.shape:
        raise ValueError("K_pages and V_pages must be [num_pages, H_kv, kv4_page_bytes(page_size, D)]")
    if K_pages.dtype is not torch.uint8 or V_pages.dtype is not torch.uint8 or not K_pages.is_contiguous() \
            or not V_pages.is_contiguous():
        raise ValueError("K_pages and V_pages must be contiguous uint8 tensors")
    n, H_kv, nbytes = K_pages.shape
    page_size, rest = divmod(nbytes * 32, 17 * D) if D > 0 else (0, 1)
    if rest:
        raise ValueError(f"a page of {nbytes} bytes does not hold whole rows of D = {D}")
    return n, H_kv, page_size


def _table(torch, block_table, kv_lens, device, n_seqs):
    if block_table.dim() != 2 or block_table.shape[0] != n_seqs:
        raise ValueError("block_table must be [sequences, max_pages_per_seq]")
    return (_ints(torch, "block_table", block_table, device, block_table.shape),
            _ints(torch, "kv_lens", kv_lens, device, (n_seqs,)))


def kv4_append(K, V, K_pages, V_pages, block_table, seq_starts, kv_lens, *, stream=None):
    """Quantise new tokens into a paged 4-bit cache.

    K, V [T, H_kv, D] float16 or bfloat16, packed by ``seq_starts`` (int32 [N + 1]),
    with any token and head strides (multiples of 8).  Sequence b's tokens
    become the last of its ``kv_lens[b]`` keys (int32 [N], counted with them);
    ``block_table`` int32 [N, max_pages].  Tokens of an invalid page are not
    written; no two tokens of a call may have the same row.
    """
    import torch

    device = _gpu(torch, ("K", "V", "K_pages", "V_pages"), K, V, K_pages, V_pages)
    flags = _half(torch, "KV", K, V)
    strides = _STRIDES[4](*_heads("K", K), *_heads("V", V))
    T, H_kv, D = K.shape
    num_pages, heads, page_size = _pages(torch, K_pages, V_pages, D)
    if V.shape != K.shape or heads != H_kv:
        raise ValueError("K and V must be [T, H_kv, D], with the pools' H_kv")
    starts, n = _starts(torch, "seq_starts", seq_starts, device), seq_starts.shape[0] - 1
    table, lens = _table(torch, block_table, kv_lens, device, n)
    max_pages = block_table.shape[1]
    if T > _MOST or H_kv > _MOST or n > _MOST or max_pages > _MOST:
        raise _too_many()
    _launch(torch, device, stream, load_library().kf_kv4_append,
            K.data_ptr(), V.data_ptr(), strides, K_pages.data_ptr(), V_pages.data_ptr(), table, starts, lens, n, T,
            H_kv, D, page_size, max_pages, num_pages, flags)


def kv4_read(K_pages, V_pages, block_table, seq_starts, kv_lens, total, D, out=None, *, out_dtype=None,
             stream=None):
    """Read the cache back: (K, V) [total, H_kv, D], float16 or ``out_dtype``
    bfloat16, the values that the codes stand for.

    Sequence b's packed rows ``seq_starts[b] .. seq_starts[b + 1] - 1`` are the last
    of its ``kv_lens[b]`` keys: with seq_starts the running sum of kv_lens and
    total = seq_starts[-1], whole contexts for attn_packed.  Rows of an
    invalid page are zeros; rows outside the sequences are not written.
    """
    import torch

    dtype = torch.float16 if out_dtype is None else out_dtype
    if dtype not in (torch.float16, torch.bfloat16):
        raise ValueError("out_dtype must be float16 or bfloat16")
    device = _gpu(torch, ("K_pages", "V_pages"), K_pages, V_pages)
    num_pages, H_kv, page_size = _pages(torch, K_pages, V_pages, D)
    starts, n = _starts(torch, "seq_starts", seq_starts, device), seq_starts.shape[0] - 1
    table, lens = _table(torch, block_table, kv_lens, device, n)
    max_pages = block_table.shape[1]
    if total > _MOST or n > _MOST or max_pages > _MOST:
        raise _too_many()
    shape = (total, H_kv, D)
    if out is None:
        K = _new_at(torch, K_pages, shape, dtype, stream)
        V = _like(torch, K, dtype, stream)
    else:
        K, V = (_output(torch, x, shape, dtype, device, stream) for x in out)
    _launch(torch, device, stream, load_library().kf_kv4_read,
            K_pages.data_ptr(), V_pages.data_ptr(), table, starts, lens, K.data_ptr(), V.data_ptr(), n, total, H_kv, D,
            page_size, max_pages, num_pages, KF_BF16 if dtype is torch.bfloat16 else 0)
    return K, V


def kv4_workspace_bytes(B, q_len, H_q, H_kv, D, page_size, max_pages_per_seq) -> int:
    """Workspace of attn_decode_kv4 (kf_attn_decode_kv4_workspace_bytes)."""
    return int(load_library().kf_attn_decode_kv4_workspace_bytes(B, q_len, H_q, H_kv, D, page_size,
                                                                 max_pages_per_seq))


@functools.lru_cache(maxsize=1024)
def _kv4_need(index, *sizes):
    """kv4_workspace_bytes on device `index`, by the sizes alone (0.6 us a call to ask)."""
    import torch

    with torch.cuda.device(index):
        return kv4_workspace_bytes(*sizes)


def attn_decode_kv4(Q, K_pages, V_pages, block_table, kv_lens, out=None, *, causal=False, workspace=None,
                    stream=None, out_dtype=None, return_lse=False):
    """Decode over the paged 4-bit cache that kv4_append writes.

    Q [B, H_q, q_len, D] float16 or bfloat16, at most 32 query rows per KV head
    (H_q / H_kv * q_len); the other arguments and the results are those of
    attn_decode_paged: O [B, H_q, q_len, D] fp32 or ``out_dtype``, (O, LSE) with
    ``return_lse``.  The softmax weights are rounded to Q's type before they meet V.
    K and V are what kv4_read with Q's type gives (fp16 cannot hold all of a cache
    written from bfloat16).  ``workspace``: a buffer of kv4_workspace_bytes to use
    instead of a new one.
    """
    import torch

    device = _gpu(torch, ("Q", "K_pages", "V_pages"), Q, K_pages, V_pages)
    flags = _out_flags(torch, out_dtype, return_lse) | _half(torch, "Q", Q)
    if Q.dim() != 4 or not Q.is_contiguous():
        raise ValueError("Q must be a contiguous [B, H_q, q_len, D] tensor")
    B, H_q, q_len, D = Q.shape
    num_pages, H_kv, page_size = _pages(torch, K_pages, V_pages, D)
    table, lens = _table(torch, block_table, kv_lens, device, B)
    max_pages = block_table.shape[1]
    if max_pages > _MOST:
        raise _too_many()
    if out is None:
        out = _like(torch, Q, out_dtype or torch.float32, stream)
    else:
        out = _output(torch, out, (B, H_q, q_len, D), out_dtype, device, stream)
    lse = _new_at(torch, Q, (B, H_q, q_len), torch.float32, stream) if return_lse else None
    need = _kv4_need(device.index, B, q_len, H_q, H_kv, D, page_size, max_pages)
    if workspace is None and need:
        workspace = _new_at(torch, Q, need, torch.uint8, stream)
    else:
        workspace, need = _workspace(torch, workspace, need, lambda: need, device, stream)
    if causal:
        flags |= KF_ATTN_CAUSAL
    _launch(torch, device, stream, load_library().kf_attn_decode_kv4,
            Q.data_ptr(), K_pages.data_ptr(), V_pages.data_ptr(), table, lens, out.data_ptr(),
            lse.data_ptr() if return_lse else None, None, B, q_len, H_q, H_kv, D, page_size, max_pages, num_pages,
            flags, workspace.data_ptr() if workspace is not None else None, need)
    return (out, lse) if return_lse else out
