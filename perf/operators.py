"""What stands around attention in a server with a 4-bit cache, as cases to
time: packed prompts, norms and rotary positions, the cache's write and read,
and decode over it.

``own`` False computes the operators in their plain form, elementary torch
operations in 32 bits; True calls the library.  The field "op" of a case says
which operator it is:

packed  attention over prompts of different lengths, one after the other in
        [tokens, heads, D] tensors (views of one fused projection where
        "fused"), causal; "prefix": every sequence has that many times as many
        keys as queries (a chunk of a prompt over its context).
rope    RMS norm of every query and key head and rotary positions.
cache   the new tokens of every sequence are quantised into the pages of a
        4-bit cache and the last "back" times as many tokens read back.
decode  attention of q_len new tokens over a paged 4-bit cache.

Four bits: blocks of 32 channels with a power-of-two scale (exponent byte E,
2^(E - 127)) and the values 0, .5, 1, 1.5, 2, 3, 4, 6 with a sign bit.  E is
that of the block's largest magnitude less 2, at least 1; a value is rounded to
the nearest, ties to the even code, 7 and more to 6.  A page holds, per KV
head, the codes of its rows (channel 2 i in the low half of byte i), then
their scale bytes.
"""
import math
import random
from itertools import accumulate

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
# H_q, H_kv, D: the repository's GQA and MQA rows, its D = 256 rows, multi-head.
HEADS = ((32, 8, 128), (32, 8, 128), (32, 8, 128), (32, 1, 64), (16, 4, 256), (32, 8, 64),
         (16, 16, 64), (32, 1, 128), (8, 8, 128))


def _case(name, op, n, lo, hi, heads=(32, 8, 128), dtype="f16", **more):
    """n sequences whose lengths (queries of "packed", new tokens of "rope" and
    "cache", keys of "decode") are spread over lo .. hi."""
    H_q, H_kv, D = heads
    c = {"op": op, "n": n, "lo": lo, "hi": hi, "H_q": H_q, "H_kv": H_kv, "D": D, "dtype": dtype,
         "lens_seed": 1, **more}
    return dict(c, name=name) if name else c


def listed():
    return [
        # A burst of short requests, MQA: little work, many ends of sequences.
        _case("prompts_short_b64", "packed", 64, 1, 128, heads=(32, 1, 64), prefix=1, fused=False, lse=True),
        # A serving batch: prompts of very different lengths, straight from
        # the fused projection.
        _case("prompts_mixed_b16", "packed", 16, 16, 4096, prefix=1, fused=True, lse=False),
        # One long prompt.
        _case("prompt_8192", "packed", 1, 8192, 8192, dtype="bf16", prefix=1, fused=True, lse=False),
        # Chunked prefill: 512 more tokens for each of 4 long contexts, D = 256.
        _case("chunks_512_over_4096", "packed", 4, 512, 512, heads=(16, 4, 256), prefix=8, fused=False,
              lse=True),
        # One token of each of 32 sequences: all latency.
        _case("rope_step_b32", "rope", 32, 1, 1, norm=True, interleaved=False, rot=128, scaling=1.0, far=8192),
        # The tokens of long prompts in a scaled context, half of the head rotated.
        _case("rope_prompts_16k", "rope", 4, 2048, 8192, dtype="bf16", norm=True, interleaved=True, rot=64,
              scaling=8.0, far=1 << 20),
        # One token for each of 64 sequences.
        _case("cache_step_b64", "cache", 64, 1, 1, page_size=16, back=1),
        # A chunk of prompts, then the contexts back for attention over them.
        _case("cache_chunk_back", "cache", 4, 300, 512, dtype="bf16", page_size=64, back=16),
        # Whole prompts into the cache, D = 64, and back.
        _case("cache_prompts_b24", "cache", 24, 32, 4096, heads=(32, 8, 64), page_size=32, back=1),
        # One token of one sequence with a 4096-token context.
        _case("decode4_b1", "decode", 1, 4096, 4096, page_size=16, q_len=1),
        # A serving step over contexts of different lengths.
        _case("decode4_ragged_b32", "decode", 32, 512, 8192, page_size=16, q_len=1),
        # Long contexts, 4 tokens to verify for each.
        _case("decode4_verify_long_b8", "decode", 8, 50000, 65536, dtype="bf16", page_size=64, q_len=4),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    most = [work(c) for c in listed()]
    flops, nbytes = max(w["flops"] for w in most), max(w["bytes"] for w in most)
    while True:
        heads = rng.choice(HEADS)
        H_q, H_kv, D = heads
        op = rng.choice(("packed", "rope", "cache", "decode"))
        kw = {"heads": heads, "dtype": rng.choice(("f16", "bf16"))}
        if op == "packed":
            n, hi = _log(rng, 1, 64), _log(rng, 2, 8192)
            lo = hi if rng.random() < 0.25 else max(1, hi // rng.choice((2, 8, 64)))
            more = {"prefix": rng.choice((1, 1, 1, 2, 8)), "fused": rng.random() < 0.5, "lse": rng.random() < 0.3}
        elif op == "rope":
            n, hi = _log(rng, 1, 64), _log(rng, 1, 8192)
            lo = max(1, hi // rng.choice((1, 4, 64)))
            more = {"norm": rng.random() < 0.7, "interleaved": rng.random() < 0.5,
                    "rot": rng.choice((D, D, D // 2, D // 4)), "scaling": rng.choice((1.0, 4.0, 32.0)),
                    "far": rng.choice((8192, 1 << 17, 1 << 20))}
        elif op == "cache":
            n, hi = _log(rng, 1, 64), _log(rng, 1, 4096)
            lo = max(1, hi // rng.choice((1, 4, 64)))
            more = {"page_size": rng.choice((16, 16, 32, 64, 128)), "back": rng.choice((1, 1, 2, 16))}
        else:
            n, hi = _log(rng, 1, 64), _log(rng, 64, 65536)
            lo = max(1, hi // rng.choice((1, 2, 16)))
            more = {"page_size": rng.choice((16, 16, 32, 64, 128)),
                    "q_len": rng.choice([q for q in (1, 1, 1, 2, 4) if H_q // H_kv * q <= 32])}
        c = _case("", op, n, lo, hi, **kw, **more)
        c["lens_seed"] = rng.randrange(1 << 20)
        # The plain form's padded scores have to fit the card.
        if op == "packed" and n * H_q * max(_lens(c)) ** 2 * c["prefix"] > 2.2e9:
            continue
        w = work(c)
        if w["flops"] <= flops and w["bytes"] <= nbytes:
            return c


def _lens(case):
    r = random.Random(case["lens_seed"])
    return [_log(r, case["lo"], case["hi"]) for _ in range(case["n"])]


def work(case):
    H_q, H_kv, D = case["H_q"], case["H_kv"], case["D"]
    lens = _lens(case)
    tokens = sum(lens)
    kv_row = H_kv * D * 2 * 2           # K and V of a token in 16 bits
    kv4_row = H_kv * D * 2 * 17 // 32   # the same in 4 bits with the scales
    if case["op"] == "packed":
        before = case["prefix"] - 1
        pairs = sum(n * n * before + n * (n + 1) // 2 for n in lens)
        nbytes = tokens * H_q * (D * 4 + (4 if case["lse"] else 0)) + tokens * case["prefix"] * kv_row
        return {"bytes": nbytes, "flops": 4 * pairs * H_q * D}
    if case["op"] == "rope":
        return {"bytes": tokens * ((H_q + H_kv) * D * 4 + 4), "flops": tokens * (H_q + H_kv) * D * 7}
    if case["op"] == "cache":
        return {"bytes": tokens * (1 + case["back"]) * (kv_row + kv4_row),
                "flops": tokens * (1 + case["back"]) * H_kv * D * 4}
    q = case["q_len"]
    nbytes = tokens * kv4_row + len(lens) * H_q * q * D * 4
    return {"bytes": nbytes, "flops": 4 * H_q * D * sum(q * n - q * (q - 1) // 2 for n in lens)}


# ---------------------------------------------------------------------------
# Four bits.
# ---------------------------------------------------------------------------
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
# Half way between neighbouring levels; a value at one goes to the even code.
BORDERS = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)


def _power(E):
    """2^(E - 127), exactly: E is the exponent field of a 32-bit number."""
    return (E.to(torch.int32) << 23).view(torch.float32)


def _quantise(x):
    """[..., D] -> codes [..., D / 2] and scale bytes [..., D / 32], uint8.
    Dividing by a power of two is exact in 32 bits."""
    b = x.float().unflatten(-1, (-1, 32))
    E = ((b.abs().amax(-1).view(torch.int32) >> 23) - 2).clamp(min=1)
    v = (b / _power(E).unsqueeze(-1)).flatten(-2)
    a = v.abs()
    # Borders below even codes are passed only from above, below odd ones at them.
    code = (a > 0.25).to(torch.uint8)
    code += a >= 0.75
    code += a > 1.25
    code += a >= 1.75
    code += a > 2.5
    code += a >= 3.5
    code += a > 5.0
    code += torch.signbit(v).to(torch.uint8) * 8
    pair = code.unflatten(-1, (-1, 2))
    return pair[..., 0] + pair[..., 1] * 16, E.to(torch.uint8)


def _values(codes, scales):
    """The 32-bit values that codes [..., D / 2] and scales [..., D / 32] stand for."""
    lut = torch.tensor(LEVELS + tuple(-v for v in LEVELS), dtype=torch.float32, device=codes.device)
    both = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    v = lut[both.int()].unflatten(-1, (-1, 32))
    return (v * _power(scales).unsqueeze(-1)).flatten(-2)


def _page_views(pages, D):
    """Codes [pages, H_kv, rows, D / 2] and scales [pages, H_kv, rows, D / 32]
    of page pools [pages, H_kv, bytes of a page]."""
    rows = pages.shape[2] // (D // 2 + D // 32)
    cut = rows * (D // 2)
    return (pages[..., :cut].unflatten(-1, (rows, D // 2)), pages[..., cut:].unflatten(-1, (rows, D // 32)))


def prepare(case, seed):
    dev = "cuda" if torch.cuda.is_available() else "cpu"
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    order = random.Random(seed)
    dtype = DTYPES[case["dtype"]]
    H_q, H_kv, D, op = case["H_q"], case["H_kv"], case["D"], case["op"]
    lens = _lens(case)
    order.shuffle(lens)
    T, n = sum(lens), len(lens)
    s = {"case": case, "lens": lens}

    def starts(lens):
        return torch.tensor([0, *accumulate(lens)], dtype=torch.int32, device=dev)

    def table(lens):
        """Pages placed at random in a pool with some to spare."""
        need = [-(-m // case["page_size"]) for m in lens]
        pool = sum(need) + sum(need) // 16 + 1
        ids = list(range(pool))
        order.shuffle(ids)
        rows = []
        for m in need:
            rows.append(ids[:m] + [0] * (max(need) - m))
            ids = ids[m:]
        return torch.tensor(rows, dtype=torch.int32, device=dev), pool

    def new_pages(pool):
        """Pages that hold quantised normal values."""
        rows = case["page_size"]
        pages = torch.empty((pool, H_kv, rows * (D // 2 + D // 32)), dtype=torch.uint8, device=dev)
        codes, scales = _page_views(pages, D)
        step = max(1, (1 << 26) // (H_kv * rows * D))
        for at in range(0, pool, step):
            shape = codes[at : at + step].shape[:-1] + (D,)
            x = torch.randn(shape, generator=gen, dtype=torch.float16, device=dev)
            codes[at : at + step], scales[at : at + step] = _quantise(x)
        return pages

    def normal(*shape):
        return torch.randn(shape, generator=gen, dtype=dtype, device=dev)

    def fused_qkv():
        """Views of one projection's output, as a layer has them."""
        x = normal(T, (H_q + 2 * H_kv) * D)
        return [v.unflatten(1, (-1, D)) for v in x.split((H_q * D, H_kv * D, H_kv * D), 1)]

    if op == "packed":
        s["starts"] = starts(lens)
        s["kv_starts"] = None
        if case["prefix"] > 1:
            s["kv_starts"] = starts([m * case["prefix"] for m in lens])
        if case["fused"] and case["prefix"] == 1:
            s["Q"], s["K"], s["V"] = fused_qkv()
        else:
            s["Q"] = normal(T, H_q, D)
            s["K"], s["V"] = (normal(T * case["prefix"], H_kv, D) for _ in range(2))
    elif op == "rope":
        s["Q"], s["K"], _ = fused_qkv()
        # Consecutive positions that begin anywhere below the context's end.
        at = [order.randrange(max(1, case["far"] - m)) for m in lens]
        s["pos"] = torch.cat([torch.arange(a, a + m, dtype=torch.int32, device=dev) for a, m in zip(at, lens)])
        i = torch.arange(case["rot"] // 2, dtype=torch.float64, device=dev)
        s["freqs"] = 10000.0 ** (-2.0 * i / case["rot"]) / case["scaling"]
        s["scale"] = 1.0 + 0.1 * math.log(case["scaling"])
        s["qw"] = s["kw"] = None
        if case["norm"]:
            s["qw"], s["kw"] = (1 + 0.1 * normal(D) for _ in range(2))
    elif op == "cache":
        _, s["K"], s["V"] = fused_qkv()
        whole = [m * case["back"] for m in lens]
        s["table"], pool = table(whole)
        s["K_pages"], s["V_pages"] = (new_pages(pool) for _ in range(2))
        s["starts"], s["back"] = starts(lens), starts(whole)
        s["total"] = sum(whole)
        s["kv_lens"] = torch.tensor(whole, dtype=torch.int32, device=dev)
    else:
        s["Q"] = normal(n, H_q, case["q_len"], D)
        s["table"], pool = table(lens)
        s["K_pages"], s["V_pages"] = (new_pages(pool) for _ in range(2))
        s["kv_lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    return s


# ---------------------------------------------------------------------------
# The plain forms.
# ---------------------------------------------------------------------------
def _attention(Q, K, V, q_lens, kv_lens):
    """Causal attention, aligned to the last key, of Q [n, H_q, q, D] over K,
    V [n, H_kv, k, D] (32 bits), rows and keys behind a sequence's own masked.
    Returns O and the log-sum-exp; rows without a key get 0 and -inf."""
    n, H_q, q, D = Q.shape
    H_kv, k = K.shape[1:3]
    rows = Q.reshape(n, H_kv, H_q // H_kv * q, D)
    s = rows @ K.transpose(2, 3) * D ** -0.5
    # Query i of a sequence sees keys j <= i + keys - queries.
    last = torch.arange(q, device=Q.device) + (kv_lens - q_lens).unsqueeze(1)
    last = torch.minimum(last, kv_lens.unsqueeze(1) - 1).repeat(1, H_q // H_kv)[:, None, :, None]
    s.masked_fill_(torch.arange(k, device=Q.device) > last, float("-inf"))
    top = s.amax(-1, keepdim=True)
    top = torch.where(top > float("-inf"), top, torch.zeros_like(top))
    s.sub_(top).exp_()
    total = s.sum(-1, keepdim=True)
    out = (s @ V) / torch.where(total > 0, total, torch.ones_like(total))
    lse = top + torch.log(total)
    return out.reshape(n, H_q, q, D), lse.reshape(n, H_q, q)


def _places(starts, total):
    """Sequence and place in it of each of `total` packed tokens."""
    t = torch.arange(total, device=starts.device, dtype=torch.int32)
    seq = torch.searchsorted(starts[1:].contiguous(), t, right=True)
    return seq, t - starts[seq]


def _plain_packed(s):
    c, Q, K, V, starts = s["case"], s["Q"], s["K"], s["V"], s["starts"]
    kv_starts = starts if s["kv_starts"] is None else s["kv_starts"]
    n, q_top = len(s["lens"]), max(s["lens"])
    k_top = q_top * c["prefix"]
    q_seq, q_at = _places(starts, Q.shape[0])
    k_seq, k_at = _places(kv_starts, K.shape[0])
    padded = [torch.zeros((n, m, x.shape[1], c["D"]), dtype=torch.float32, device=Q.device)
              for x, m in ((Q, q_top), (K, k_top), (V, k_top))]
    padded[0][q_seq, q_at] = Q.float()
    padded[1][k_seq, k_at] = K.float()
    padded[2][k_seq, k_at] = V.float()
    Qp, Kp, Vp = (x.transpose(1, 2).contiguous() for x in padded)
    out, lse = _attention(Qp, Kp, Vp, starts.diff(), kv_starts.diff())
    out = out.transpose(1, 2)[q_seq, q_at].to(Q.dtype)
    return (out, lse.transpose(1, 2)[q_seq, q_at]) if c["lse"] else out


def _turn(x, w, cos, sin, c):
    x = x.float()
    if w is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w.float()
    r, rest = x[..., : c["rot"]], x[..., c["rot"] :]
    a, b = (r[..., 0::2], r[..., 1::2]) if c["interleaved"] else r.chunk(2, -1)
    y = (a * cos - b * sin, a * sin + b * cos)
    y = torch.stack(y, -1).flatten(-2) if c["interleaved"] else torch.cat(y, -1)
    return torch.cat((y, rest), -1)


def _plain_rope(s):
    angle = s["pos"].double()[:, None, None] * s["freqs"]
    cos, sin = (angle.cos() * s["scale"]).float(), (angle.sin() * s["scale"]).float()
    return tuple(_turn(s[x], s[w], cos, sin, s["case"]).to(s[x].dtype) for x, w in (("Q", "qw"), ("K", "kw")))


def _slots(s, starts, total):
    """Page and row of the last tokens of every sequence, packed by `starts`."""
    seq, at = _places(starts, total)
    at = at + (s["kv_lens"] - starts.diff())[seq]
    page_size = s["case"]["page_size"]
    return s["table"][seq, at // page_size].long(), at % page_size


def _plain_cache(s):
    D, out = s["case"]["D"], []
    page, row = _slots(s, s["starts"], s["K"].shape[0])
    page2, row2 = _slots(s, s["back"], s["total"])

    def one(x, pages):
        codes, scales = _page_views(pages, D)
        codes[page, :, row], scales[page, :, row] = _quantise(x)
        return _values(codes[page2, :, row2], scales[page2, :, row2]).to(x.dtype)

    return one(s["K"], s["K_pages"]), one(s["V"], s["V_pages"])


def _plain_decode(s):
    Q, D, table = s["Q"], s["case"]["D"], s["table"].long()

    def rows(pages):
        codes, scales = _page_views(pages, D)
        x = _values(codes[table], scales[table])  # [n, pages, H_kv, rows, D]
        return x.transpose(1, 2).flatten(2, 3)

    q_lens = torch.full_like(s["kv_lens"], Q.shape[2])
    return _attention(Q.float(), rows(s["K_pages"]), rows(s["V_pages"]), q_lens, s["kv_lens"])[0].to(Q.dtype)


def run(s):
    c = s["case"]
    if not own:
        return {"packed": _plain_packed, "rope": _plain_rope, "cache": _plain_cache,
                "decode": _plain_decode}[c["op"]](s)
    import kernelfoundry_amd as kf

    if c["op"] == "packed":
        return kf.attn_packed(s["Q"], s["K"], s["V"], s["starts"], kv_starts=s["kv_starts"], causal=True,
                              out_dtype=s["Q"].dtype, return_lse=c["lse"])
    if c["op"] == "rope":
        return kf.qk_norm_rope(s["Q"], s["K"], s["pos"], s["freqs"], q_weight=s["qw"], k_weight=s["kw"],
                               eps=1e-6, interleaved=c["interleaved"], scale=s["scale"])
    if c["op"] == "cache":
        kf.kv4_append(s["K"], s["V"], s["K_pages"], s["V_pages"], s["table"], s["starts"], s["kv_lens"])
        return kf.kv4_read(s["K_pages"], s["V_pages"], s["table"], s["back"], s["kv_lens"], s["total"], c["D"],
                           out_dtype=s["K"].dtype)
    return kf.attn_decode_kv4(s["Q"], s["K_pages"], s["V_pages"], s["table"], s["kv_lens"], causal=True,
                              out_dtype=s["Q"].dtype)


# ---------------------------------------------------------------------------
# The definitions in 64 bits, a sequence at a time.
# ---------------------------------------------------------------------------
def _exact_read(pages, table_row, count, D):
    """The first `count` rows of a sequence, [H_kv, count, D] in 64 bits."""
    H_kv, size = pages.shape[1:]
    rows = size * 32 // (17 * D)
    at = torch.arange(count, device=pages.device)
    page, row = table_row[at // rows].long(), at % rows
    d = torch.arange(D, device=pages.device)
    byte = pages[page[:, None], :, (row[:, None] * (D // 2) + d // 2)]       # [count, D, H_kv]
    E = pages[page[:, None], :, rows * (D // 2) + row[:, None] * (D // 32) + d // 32]
    code = torch.where(d[None, :, None] % 2 == 1, byte >> 4, byte & 15).long()
    sign, exponent, half = 1 - 2 * (code >> 3), (code >> 1) & 3, code & 1
    # e2m1: subnormal half steps below 1, else (1 + half / 2) 2^(exponent - 1).
    low = half.double() / 2
    high = (1 + half.double() / 2) * 2.0 ** (exponent.double() - 1)
    v = sign * torch.where(exponent == 0, low, high) * 2.0 ** (E.double() - 127)
    return v.permute(2, 0, 1).contiguous()


def _exact_round(x):
    """x [..., D] in 64 bits through the 4-bit form, by the nearest of its levels."""
    b = x.unflatten(-1, (-1, 32))
    top = b.abs().amax(-1, keepdim=True)
    unit = 2.0 ** (torch.floor(torch.log2(torch.where(top > 0, top, torch.ones_like(top)))) - 2)
    a = (b / unit).abs().contiguous()
    levels = torch.tensor(LEVELS, dtype=torch.float64, device=x.device)
    borders = torch.tensor(BORDERS, dtype=torch.float64, device=x.device)
    up = torch.searchsorted(borders, a, right=True)   # at a border: the code above it
    down = torch.searchsorted(borders, a)             # at a border: the code below it
    code = torch.where(up % 2 == 0, up, down)
    return (torch.sign(b) * levels[code] * unit).flatten(-2)


def exact(case, seed):
    s = prepare(case, seed)
    D, op = case["D"], case["op"]

    def attention(q, k, v):
        """Causal attention of q [H_q, n, D] over k, v [H_kv, m, D]."""
        H_q, n, _ = q.shape
        m, ratio = k.shape[1], H_q // k.shape[0]
        out, lse = torch.empty_like(q), torch.empty_like(q[..., 0])
        step = max(1, (1 << 27) // m)
        for h in range(H_q):
            kt, vh = k[h // ratio].t().contiguous(), v[h // ratio]
            for at in range(0, n, step):
                last = torch.arange(at, min(n, at + step), device=q.device)[:, None] + (m - n)
                x = q[h, at : at + step] @ kt / math.sqrt(D)
                x.masked_fill_(torch.arange(m, device=q.device) > last, float("-inf"))
                lse[h, at : at + step] = torch.logsumexp(x, 1)
                # A row that sees no key gets 0.
                out[h, at : at + step] = torch.where(last >= 0, torch.softmax(x, 1), torch.zeros_like(x)) @ vh
        return out, lse

    if op == "rope":
        turns = s["pos"].double()[:, None] * s["freqs"]
        z = torch.polar(torch.full_like(turns, s["scale"]), turns)[:, None]
        outs = []
        for x, w in ((s["Q"], s["qw"]), (s["K"], s["kw"])):
            x = x.double()
            if w is not None:
                x = x * torch.rsqrt((x * x).sum(-1, keepdim=True) / D + 1e-6) * w.double()
            r = x[..., : case["rot"]]
            if case["interleaved"]:
                y = torch.view_as_real(torch.view_as_complex(r.unflatten(-1, (-1, 2)).contiguous()) * z).flatten(-2)
            else:
                y = torch.complex(*(p.contiguous() for p in r.chunk(2, -1))) * z
                y = torch.cat((y.real, y.imag), -1)
            outs.append(torch.cat((y, x[..., case["rot"] :]), -1))
        return tuple(outs)
    if op == "cache":
        outs = []
        for x, pages in ((s["K"], s["K_pages"]), (s["V"], s["V_pages"])):
            parts, at = [], 0
            for i, m in enumerate(s["lens"]):
                old = _exact_read(pages, s["table"][i], m * (case["back"] - 1), D).transpose(0, 1)
                parts += [old, _exact_round(x[at : at + m].double())]
                at += m
            outs.append(torch.cat(parts))
        return tuple(outs)
    if op == "decode":
        if sum(s["lens"]) * case["H_q"] > 1 << 25:
            return None
        outs = [attention(s["Q"][i].double(), *(_exact_read(s[p], s["table"][i], m, D)
                                                  for p in ("K_pages", "V_pages")))[0]
                for i, m in enumerate(s["lens"])]
        return torch.stack(outs)
    outs, lses, at = [], [], 0
    for m in s["lens"]:
        q = s["Q"][at : at + m].double().transpose(0, 1).contiguous()
        keys = slice(at * case["prefix"], (at + m) * case["prefix"])
        k, v = (s[x][keys].double().transpose(0, 1).contiguous() for x in ("K", "V"))
        out, lse = attention(q, k, v)
        outs.append(out.transpose(0, 1))
        lses.append(lse.transpose(0, 1))
        at += m
    return (torch.cat(outs), torch.cat(lses)) if case["lse"] else torch.cat(outs)
