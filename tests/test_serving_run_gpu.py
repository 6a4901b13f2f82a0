"""The serving operators together, as a server runs them: prompts (norm and
rotation, cache, attention), steps of one token, and a later chunk of a prompt
over its context read back from the cache; also as one captured step."""
import math

import pytest
import torch

import kernelfoundry_amd as kf
from tests import _serve_ref as ref

pytestmark = pytest.mark.gpu

H_q, H_kv, D, PAGE = 8, 2, 128, 16


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def starts_of(lens):
    s = [0]
    for n in lens:
        s.append(s[-1] + n)
    return s


class Server:
    """Three sequences with room for `room` keys each."""

    def __init__(self, room, dtype, seed=0):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.gen, self.dtype, self.B = gen, dtype, 3
        per = -(-room // PAGE)
        ids = torch.randperm(3 * per + 2, generator=gen, device="cuda")[: 3 * per]
        self.table = ids.to(torch.int32).view(3, per).contiguous()
        shape = (3 * per + 2, H_kv, kf.kv4_page_bytes(PAGE, D))
        self.Kp, self.Vp = (torch.full(shape, 255, dtype=torch.uint8, device="cuda") for _ in range(2))
        self.freqs, self.scale = kf.rope_freqs(D, scaling="yarn", factor=4.0, original_len=64, device="cuda")
        self.wq, self.wk = ((1 + 0.1 * torch.randn(D, generator=gen, device="cuda")).to(dtype) for _ in range(2))
        self.have = [0, 0, 0]
        # What a sequence's keys and values stand for in the cache, in 64 bits.
        self.keys = [torch.empty(0, H_kv, D, dtype=torch.float64, device="cuda") for _ in range(3)]
        self.values = [k.clone() for k in self.keys]

    def qkv(self, lens):
        x = torch.randn(sum(lens), (H_q + 2 * H_kv) * D, generator=self.gen, device="cuda").to(self.dtype)
        return [v.unflatten(1, (-1, D)) for v in x.split((H_q * D, H_kv * D, H_kv * D), 1)]

    def take(self, lens):
        """Norm, rotation and cache of the next tokens: their Q, K, V and starts."""
        Q, K, V = self.qkv(lens)
        pos = ints([self.have[b] + i for b in range(3) for i in range(lens[b])])
        Qr, Kr = kf.qk_norm_rope(Q, K, pos, self.freqs, q_weight=self.wq, k_weight=self.wk, scale=self.scale)
        s = starts_of(lens)
        self.have = [h + n for h, n in zip(self.have, lens)]
        kf.kv4_append(Kr, V, self.Kp, self.Vp, self.table, ints(s), ints(self.have))
        half = torch.finfo(self.dtype).eps / 2
        for got, x, w in ((Qr, Q, self.wq), (Kr, K, self.wk)):
            # Its rounding, and 64 units of 2^-24 of the magnitudes for the arithmetic in 32 bits.
            exact, mag = ref.norm_rope(x, w, 1e-6, pos, self.freqs, False, self.scale)
            assert ((got.double() - exact).abs() <= half * exact.abs() + 64 * 2.0 ** -24 * mag).all()
        k4, v4 = ref.quantise(Kr), ref.quantise(V)
        for b in range(3):
            self.keys[b] = torch.cat((self.keys[b], k4[s[b]:s[b + 1]]))
            self.values[b] = torch.cat((self.values[b], v4[s[b]:s[b + 1]]))
        return Qr, Kr, V, s

    def check(self, O, LSE, Q, s, keys, values):
        for b in range(3):
            q, k, v = (x.double().transpose(0, 1).contiguous() for x in (Q[s[b]:s[b + 1]], keys[b], values[b]))
            want, lse = ref.attention(q, k, v, True)
            if q.shape[1]:
                bounds = ref.attention_bounds(Q, keys[b], values[b], O.dtype, k.shape[1])
                ref.check_attention(O[s[b]:s[b + 1]].transpose(0, 1), LSE[s[b]:s[b + 1]].transpose(0, 1), want, lse, bounds)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_prompts_steps_and_a_later_chunk(dtype):
    sv = Server(400, dtype)
    # Prompts, one of them empty for now: over their own keys in 16 bits.
    lens = [50, 0, 133]
    Q, K, V, s = sv.take(lens)
    O, LSE = kf.attn_packed(Q, K, V, ints(s), causal=True, out_dtype=dtype, return_lse=True)
    sv.check(O, LSE, Q, s, [K[s[b]:s[b + 1]].double() for b in range(3)], [V[s[b]:s[b + 1]].double() for b in range(3)])
    # Steps of one token over the cache.
    for _ in range(3):
        Q, _, _, s = sv.take([1, 1, 1])
        O, LSE = kf.attn_decode_kv4(Q.view(3, H_q, 1, D), sv.Kp, sv.Vp, sv.table, ints(sv.have), out_dtype=dtype,
                                    return_lse=True)
        sv.check(O.view(3, H_q, D), LSE.view(3, H_q), Q, s, sv.keys, sv.values)
    # A chunk for each over its whole context, read back from the cache.
    Q, _, _, s = sv.take([70, 200, 33])
    ks = starts_of(sv.have)
    K, V = kf.kv4_read(sv.Kp, sv.Vp, sv.table, ints(ks), ints(sv.have), ks[-1], D, out_dtype=dtype)
    assert torch.equal(K.double(), torch.cat(sv.keys)) and torch.equal(V.double(), torch.cat(sv.values))
    O, LSE = kf.attn_packed(Q, K, V, ints(s), kv_starts=ints(ks), causal=True, out_dtype=dtype, return_lse=True)
    sv.check(O, LSE, Q, s, sv.keys, sv.values)
    # The two ways to attend to the cache agree: the chunk's last token.
    last = torch.stack([Q[s[b + 1] - 1] for b in range(3)])
    one, _ = kf.attn_decode_kv4(last.view(3, H_q, 1, D), sv.Kp, sv.Vp, sv.table, ints(sv.have), out_dtype=dtype,
                                return_lse=True)
    both = torch.stack([O[s[b + 1] - 1] for b in range(3)])
    off, rel, _ = ref.attention_bounds(Q, K, V, dtype, max(sv.have))
    assert ((one.view(3, H_q, D).double() - both.double()).abs() <= 2 * (off + rel * both.double().abs())).all()


def test_a_captured_step_replayed():
    """One step in a graph on a side stream, its inputs rewritten between the
    replays: the eager step's bits each time, and no row of the cache beside the
    new ones touched."""
    dtype = torch.float16
    sv, eager = Server(200, dtype, 5), Server(200, dtype, 5)
    for x in (sv, eager):
        x.take([20, 61, 100])
    assert torch.equal(sv.Kp, eager.Kp)
    x = torch.zeros(3, (H_q + 2 * H_kv) * D, device="cuda", dtype=dtype)
    pos, lens, s = ints(sv.have), ints([h + 1 for h in sv.have]), ints([0, 1, 2, 3])

    def step(sv, x, pos, lens, out=None, rows=None, ws=None):
        Q, K, V = (v.unflatten(1, (-1, D)) for v in x.split((H_q * D, H_kv * D, H_kv * D), 1))
        Qr, Kr = kf.qk_norm_rope(Q, K, pos, sv.freqs, rows, q_weight=sv.wq, k_weight=sv.wk, scale=sv.scale)
        kf.kv4_append(Kr, V, sv.Kp, sv.Vp, sv.table, s, lens)
        return kf.attn_decode_kv4(Qr.view(3, H_q, 1, D), sv.Kp, sv.Vp, sv.table, lens, out, workspace=ws)

    rows = (torch.empty(3, H_q, D, device="cuda", dtype=dtype), torch.empty(3, H_kv, D, device="cuda", dtype=dtype))
    out = torch.empty(3, H_q, 1, D, device="cuda")
    ws = torch.empty(kf.kv4_workspace_bytes(3, 1, H_q, H_kv, D, PAGE, sv.table.shape[1]), dtype=torch.uint8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(sv, x, pos, lens, out, rows, ws)
    for i in range(4):
        x.copy_(torch.randn(x.shape, generator=sv.gen, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        want = step(eager, x, pos, lens)
        assert torch.equal(out, want) and torch.equal(sv.Kp, eager.Kp) and torch.equal(sv.Vp, eager.Vp)
        pos.add_(1)
        lens.add_(1)


def test_two_steps_at_once_on_two_streams():
    """Two servers' steps queued on two streams side by side, each with its own
    workspace from its stream's pool: the bits of the steps one after the other."""
    servers = [Server(300, torch.float16, i) for i in (1, 2)]
    data = []
    for sv in servers:
        sv.take([150, 280, 7])
        data.append(torch.randn(3, H_q, 1, D, generator=sv.gen, device="cuda").half())
    lens = [ints(sv.have) for sv in servers]
    want = [kf.attn_decode_kv4(q, sv.Kp, sv.Vp, sv.table, n) for q, sv, n in zip(data, servers, lens)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in servers]
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(20):
        for i, (q, sv, n) in enumerate(zip(data, servers, lens)):
            got[i].append(kf.attn_decode_kv4(q, sv.Kp, sv.Vp, sv.table, n, stream=streams[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in got[i])
    assert not math.isnan(float(want[0].sum()))
