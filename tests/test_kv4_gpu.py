"""The 4-bit cache: what kv4_append writes and kv4_read reads, exactly, and
attn_decode_kv4 over it, against plain 64-bit forms."""
import math
import random

import pytest
import torch

import kernelfoundry_amd as kf
from tests import _serve_ref as ref

pytestmark = pytest.mark.gpu


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def starts_of(lens):
    s = [0]
    for n in lens:
        s.append(s[-1] + n)
    return s


def new_cache(capacity, H_kv, D, page_size, seed=0, spare=3):
    """Pools full of 0xff (scales that stand for NaN), a table of shuffled pages for
    sequences of up to `capacity` keys."""
    need = [-(-n // page_size) for n in capacity]
    pool = sum(need) + spare
    ids = list(range(pool))
    random.Random(seed).shuffle(ids)
    top, rows = max(1, max(need)), []
    for n in need:
        rows.append(ids[:n] + [-1] * (top - n))
        ids = ids[n:]
    pages = [torch.full((pool, H_kv, kf.kv4_page_bytes(page_size, D)), 255, dtype=torch.uint8, device="cuda")
             for _ in range(2)]
    return pages[0], pages[1], ints(rows)


def normal(*shape, dtype=torch.float16, seed=0):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda", dtype=dtype)


def fill(lens, H_kv, D, page_size, dtype=torch.float16, seed=0):
    """A cache that holds `lens` keys a sequence, and the values it stands for."""
    Kp, Vp, table = new_cache(lens, H_kv, D, page_size, seed)
    K, V = normal(sum(lens), H_kv, D, dtype=dtype, seed=seed), normal(sum(lens), H_kv, D, dtype=dtype, seed=seed + 1)
    kf.kv4_append(K, V, Kp, Vp, table, ints(starts_of(lens)), ints(lens))
    return Kp, Vp, table, ref.quantise(K), ref.quantise(V)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("page_size", [16, 64])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_append_and_read_are_exact(D, page_size, dtype):
    lens = [1, 15, 16, 17, 0, 100, 33]
    Kp, Vp, table, K4, V4 = fill(lens, 3, D, page_size, dtype)
    K, V = kf.kv4_read(Kp, Vp, table, ints(starts_of(lens)), ints(lens), sum(lens), D, out_dtype=dtype)
    assert torch.equal(K.double(), K4) and torch.equal(V.double(), V4)
    # Every row where the format says, and no other row touched.
    values, at = ref.unpack(Kp, D), 0
    used = torch.zeros(Kp.shape[0], page_size, dtype=torch.bool, device="cuda")
    for i, n in enumerate(lens):
        for j in range(n):
            page, row = int(table[i, j // page_size]), j % page_size
            used[page, row] = True
            assert torch.equal(values[page, :, row], K4[at + j])
        at += n
    codes = Kp[..., : page_size * (D // 2)].unflatten(-1, (page_size, D // 2))
    assert (codes.transpose(1, 2)[~used] == 255).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_every_kind_of_block(dtype):
    """Blocks of one magnitude after the other: all finite values of the
    type as the block's largest beside smaller ones, ties among them, zeros,
    negative zeros, least numbers."""
    bits = torch.arange(0, 0x7c00 if dtype == torch.float16 else 0x7f80, 37, dtype=torch.int32)
    top = bits.to(torch.int16).view(dtype).cuda()                       # [n]
    part = torch.linspace(-1, 1, 31, device="cuda", dtype=torch.float64)
    ties = torch.tensor([0.0, -0.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 4.0, 6.0, 0.5, -0.25, -1.25, -2.5, -5.0],
                        device="cuda", dtype=torch.float64)
    unit = ref.exp2i(torch.frexp(top.double())[1] - 3)
    rows = torch.empty(top.shape[0], 64, device="cuda", dtype=dtype)
    rows[:, 0] = top
    rows[:, 1:32] = (top.double()[:, None] * part).to(dtype)
    rows[:, 32] = -top
    rows[:, 33:49] = (unit[:, None] * ties).to(dtype)
    rows[:, 49:] = 0
    x = rows[:, None, :].contiguous()
    n = x.shape[0]
    Kp, Vp, table = new_cache([n], 1, 64, 16)
    kf.kv4_append(x, x, Kp, Vp, table, ints([0, n]), ints([n]))
    K, V = kf.kv4_read(Kp, Vp, table, ints([0, n]), ints([n]), n, 64, out_dtype=dtype)
    want = ref.quantise(x)
    # bf16: results below its least normal number stand for themselves in the
    # cache; a conversion may flush them.
    least = torch.finfo(dtype).smallest_normal if dtype == torch.bfloat16 else 0.0
    far = (K.double() != want) & ~((want.abs() < least) & (K == 0))
    assert not far.any(), (x[far][:4], K[far][:4], want[far][:4])
    assert torch.equal(K, V)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_infinity_and_nan_mark_their_block_alone(dtype):
    x = normal(4, 1, 128, dtype=dtype)
    clean = ref.quantise(x)
    x[0, 0, 5], x[1, 0, 40], x[2, 0, 127] = math.inf, math.nan, -math.inf
    Kp, Vp, table = new_cache([4], 1, 128, 16)
    kf.kv4_append(x, x, Kp, Vp, table, ints([0, 4]), ints([4]))
    K, _ = kf.kv4_read(Kp, Vp, table, ints([0, 4]), ints([4]), 4, 128, out_dtype=dtype)
    bad = torch.zeros(4, 128, dtype=torch.bool, device="cuda")
    bad[0, :32] = bad[1, 32:64] = bad[2, 96:] = True
    got = K[:, 0]
    # By the bits: the build does not promise what a comparison makes of NaN.
    nan = got.view(torch.int16).int() & 0x7fff
    assert (nan[bad] > (0x7c00 if dtype == torch.float16 else 0x7f80)).all()
    assert torch.equal(got[~bad].double(), clean[:, 0][~bad])


def test_tokens_are_appended_behind_the_context_and_windows_read():
    lens, more = [5, 0, 40, 17], [1, 3, 0, 30]
    total = [a + b for a, b in zip(lens, more)]
    Kp, Vp, table = new_cache(total, 2, 128, 16)
    parts = []
    for n, at, seed in ((lens, lens, 1), (more, total, 2)):
        x = normal(sum(n), 2 * 2 * 128, seed=seed)
        K, V = (v.unflatten(1, (2, 128)) for v in x.split(256, 1))     # strided views
        kf.kv4_append(K, V, Kp, Vp, table, ints(starts_of(n)), ints(at))
        parts.append((ref.quantise(K), ref.quantise(V)))
    K, V = kf.kv4_read(Kp, Vp, table, ints(starts_of(total)), ints(total), sum(total), 128)
    s0, s1, s2 = starts_of(lens), starts_of(more), starts_of(total)
    for b in range(4):
        for got, i in ((K, 0), (V, 1)):
            want = torch.cat((parts[0][i][s0[b]:s0[b + 1]], parts[1][i][s1[b]:s1[b + 1]]))
            assert torch.equal(got[s2[b]:s2[b + 1]].double(), want)
    last, _ = kf.kv4_read(Kp, Vp, table, ints(s1), ints(total), sum(more), 128)
    assert torch.equal(last.double(), parts[1][0])


def test_bad_places_are_skipped():
    """Invalid pages, tokens beyond the table, counts smaller than the new
    tokens, tokens outside the sequences: neither written nor read."""
    Kp, Vp, table = new_cache([40, 40, 40], 1, 64, 16)
    table[0, 1], table[1, 2] = Kp.shape[0], -7
    x = normal(100, 1, 64)
    starts, lens = ints([3, 38, 70, 80]), ints([35, 70, 4])
    kf.kv4_append(x, x, Kp, Vp, table, starts, lens)
    out = [torch.full((100, 1, 64), 9.0, device="cuda", dtype=torch.float16) for _ in range(2)]
    K, _ = kf.kv4_read(Kp, Vp, table, starts, lens, 100, 64, out)
    want = torch.full((100, 64), 9.0, device="cuda", dtype=torch.float64)
    want[3:80] = 0
    q = ref.quantise(x)[:, 0]
    want[3:19], want[35:38] = q[3:19], q[35:38]     # 0..15, 32..34 of a sequence without its second page
    # The second: keys 38..69, of which 38..47 lie on its invalid third page and the
    # rest outside the table; the third: its last 4 of 10 tokens.
    want[76:80] = q[76:80]
    assert torch.equal(K[:, 0].double(), want)


def test_many_sequences_of_one_token():
    n = 3000
    lens = [1 + i % 40 for i in range(n)]
    Kp, Vp, table, K4, _ = fill(lens, 1, 64, 16)
    step = normal(n, 1, 64, seed=7)
    kf.kv4_append(step, step, Kp, Vp, table, ints(list(range(n + 1))), ints(lens))
    K, _ = kf.kv4_read(Kp, Vp, table, ints(list(range(n + 1))), ints(lens), n, 64)
    assert torch.equal(K.double(), ref.quantise(step))


# ---------------------------------------------------------------------------
# Decode.
# ---------------------------------------------------------------------------
def decode(lens, heads, q_len, page_size, dtype=torch.float16, causal=True, out_dtype=None, seed=0, cache=None):
    H_q, H_kv, D = heads
    Kp, Vp, table, K4, V4 = cache or fill(lens, H_kv, D, page_size, dtype, seed)
    Q = normal(len(lens), H_q, q_len, D, dtype=dtype, seed=seed + 9)
    O, LSE = kf.attn_decode_kv4(Q, Kp, Vp, table, ints(lens), causal=causal, out_dtype=out_dtype, return_lse=True)
    torch.cuda.synchronize()
    s, want, want_lse = starts_of(lens), [], []
    for b in range(len(lens)):
        o, e = ref.attention(Q[b].double(), *(x[s[b]:s[b + 1]].transpose(0, 1).contiguous() for x in (K4, V4)), causal)
        want.append(o)
        want_lse.append(e)
    bounds = ref.attention_bounds(Q, K4, V4, out_dtype or torch.float32, max(lens)) if sum(lens) else (0, 0, 0)
    ref.check_attention(O, LSE, torch.stack(want), torch.stack(want_lse), bounds)
    return O, LSE


HEADS = [(8, 2, 128), (4, 1, 64), (8, 2, 256), (3, 3, 64), (14, 2, 128), (20, 1, 128), (24, 1, 64), (32, 1, 256)]


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("page_size", [16, 32, 128])
def test_decode_lengths(heads, dtype, page_size):
    decode([1, 0, 15, 16, 17, 31, 32, 33, 64, 100, 0, 257, 700], heads, 1, page_size, dtype)


@pytest.mark.parametrize("heads,q_len", [((8, 2, 128), 4), ((8, 2, 128), 8), ((8, 2, 64), 3), ((4, 2, 256), 5),
                                         ((2, 1, 128), 16), ((5, 1, 64), 6)])
@pytest.mark.parametrize("causal", [True, False])
def test_decode_of_several_tokens(heads, q_len, causal):
    """Rows in front of the first key of a sequence shorter than q_len see none."""
    decode([1, 2, q_len, q_len + 1, 40, 0, 333], heads, q_len, 16, causal=causal)


@pytest.mark.parametrize("out_dtype", [None, torch.float16, torch.bfloat16])
def test_decode_output_types(out_dtype):
    assert decode([50, 3], (8, 2, 128), 1, 16, out_dtype=out_dtype)[0].dtype == (out_dtype or torch.float32)


@pytest.mark.parametrize("lens,heads", [([20000], (8, 2, 128)), ([9000, 1, 30000, 4000], (4, 1, 64)),
                                        ([5000] * 6, (8, 4, 256)), ([7777, 12345], (32, 1, 128))])
def test_decode_long(lens, heads):
    decode(lens, heads, 1, 64)


@pytest.mark.parametrize("n", [70, 300, 1200])
def test_decode_many_sequences(n):
    decode([(i * i * 7 + i) % 130 for i in range(n)], (4, 2, 64), 1, 16)


def test_decode_invalid_pages_hold_no_keys():
    """Also where the sequence's keys behind its last one are garbage (0xff)."""
    lens = [100, 50]
    cache = fill(lens, 2, 128, 16)
    Kp, Vp, table, K4, V4 = cache
    bad = table.clone()
    bad[0, 2], bad[0, 5], bad[1, :] = -1, Kp.shape[0], -1
    Q = normal(2, 8, 1, 128, seed=3)
    O, LSE = kf.attn_decode_kv4(Q, Kp, Vp, bad, ints(lens), return_lse=True)
    keep = torch.ones(100, dtype=torch.bool, device="cuda")
    keep[32:48] = keep[80:96] = False
    k, v = (x[:100][keep].transpose(0, 1).contiguous() for x in (K4, V4))
    want, want_lse = ref.attention(Q[0].double(), k, v, False)
    ref.check_attention(O[0], LSE[0], want, want_lse, ref.attention_bounds(Q, K4, V4, torch.float32, 100))
    assert (O[1] == 0).all() and torch.isinf(LSE[1]).all()


def test_decode_counts_outside_the_table_are_clamped():
    Kp, Vp, table, _, _ = fill([64, 64], 2, 64, 16)
    Q = normal(2, 4, 1, 64)
    a = kf.attn_decode_kv4(Q, Kp, Vp, table, ints([1 << 30, -3]))
    b = kf.attn_decode_kv4(Q, Kp, Vp, table, ints([64, 0]))
    assert torch.equal(a, b) and (a[1] == 0).all()


def test_decode_pages_past_32_bits():
    """A pool of more than 4 GiB, whose last pages are used."""
    page_size, D, H_kv = 64, 128, 8
    per = H_kv * kf.kv4_page_bytes(page_size, D)
    pool = (9 << 29) // per + 8
    Kp, Vp = (torch.empty(pool, H_kv, per // H_kv, dtype=torch.uint8, device="cuda") for _ in range(2))
    small_k, small_v, table, K4, V4 = fill([500], H_kv, D, page_size)
    far = table.clone()
    for i in range(table.shape[1]):
        far[0, i] = pool - 1 - i
        Kp[pool - 1 - i], Vp[pool - 1 - i] = small_k[int(table[0, i])], small_v[int(table[0, i])]
    Q = normal(1, 32, 1, D)
    want = kf.attn_decode_kv4(Q, small_k, small_v, table, ints([500]))
    assert torch.equal(kf.attn_decode_kv4(Q, Kp, Vp, far, ints([500])), want)
    s = ints([0, 500])
    K, _ = kf.kv4_read(Kp, Vp, far, s, ints([500]), 500, D)
    assert torch.equal(K.double(), K4)
    x = normal(500, H_kv, D, seed=4)
    kf.kv4_append(x, x, Kp, Vp, far, s, ints([500]))
    K, _ = kf.kv4_read(Kp, Vp, far, s, ints([500]), 500, D)
    assert torch.equal(K.double(), ref.quantise(x))


def test_decode_workspace_streams_and_graphs():
    lens = [700, 33, 1500]
    Kp, Vp, table, _, _ = fill(lens, 2, 128, 16)
    Q, n = normal(3, 8, 1, 128), ints(lens)
    want = kf.attn_decode_kv4(Q, Kp, Vp, table, n)
    need = kf.kv4_workspace_bytes(3, 1, 8, 2, 128, 16, table.shape[1])
    ws = torch.full((need,), 255, dtype=torch.uint8, device="cuda")   # holds NaN: no initialisation needed
    assert torch.equal(kf.attn_decode_kv4(Q, Kp, Vp, table, n, workspace=ws), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = kf.attn_decode_kv4(Q, Kp, Vp, table, n, stream=side)
    side.synchronize()
    assert torch.equal(got, want)
    out, x = torch.empty_like(want), normal(3, 2, 128, seed=5)
    one = ints([0, 1, 2, 3])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kf.kv4_append(x, x, Kp, Vp, table, one, n)
        kf.attn_decode_kv4(Q, Kp, Vp, table, n, out, workspace=ws)
    for step in range(5):
        # One more key for some, fewer for others, no key for one at the last.
        n.copy_(ints([700 - 100 * step, 33 + step, 0 if step == 4 else 1500]))
        x.mul_(1.5)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, kf.attn_decode_kv4(Q, Kp, Vp, table, n))


def test_refusals():
    Kp, Vp, table, _, _ = fill([20], 2, 128, 16)
    Q, n = normal(1, 8, 1, 128), ints([20])
    for bad in (lambda: kf.attn_decode_kv4(Q.float(), Kp, Vp, table, n),):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: kf.attn_decode_kv4(Q, Kp.half(), Vp, table, n),
                lambda: kf.attn_decode_kv4(Q, Kp[:, :, :1000], Vp, table, n),
                lambda: kf.attn_decode_kv4(Q, Kp[:, :, :1000].contiguous(), Vp[:, :, :1000].contiguous(), table, n),
                lambda: kf.attn_decode_kv4(Q, Kp, Vp, table.long(), n),
                lambda: kf.attn_decode_kv4(Q, Kp, Vp, table, ints([1, 2])),
                lambda: kf.attn_decode_kv4(Q[:, :, :, ::2], Kp, Vp, table, n),
                lambda: kf.attn_decode_kv4(Q, Kp, Vp, table, n, workspace=torch.empty(1 << 20, dtype=torch.uint8)),
                lambda: kf.kv4_append(Q[:, :3, 0], Q[:, :3, 0], Kp, Vp, table, ints([0, 1]), n),
                lambda: kf.kv4_append(Q[:, :2, 0], Q[:, :2, 0], Kp, Vp, table, ints([0, 1, 2]), n),
                lambda: kf.kv4_read(Kp, Vp, table, ints([0, 20]), n, 20, 96),
                lambda: kf.kv4_read(Kp, Vp, table, ints([0, 20]), n, 20, 128, (Q, Q))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(kf.KfError) as e:
        kf.attn_decode_kv4(normal(1, 66, 1, 128), Kp, Vp, table, n)
    assert e.value.status == kf.KF_ERR_SIZE
