"""Each serving entry captured into a graph as a process's first call of it, and
replayed between eager work."""
import os
import subprocess
import sys

import pytest

from tests.conftest import REPO

pytestmark = pytest.mark.gpu

CHILD = r"""
import sys
import torch
import kernelfoundry_amd as kf

def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")

def half(*shape):
    return torch.randn(shape, device="cuda").half()

Q, K, V, T = half(90, 8, 128), half(90, 2, 128), half(90, 2, 128), 90
starts, lens, table = ints([0, 50, 90]), ints([50, 40]), ints([[3, 0, 5, 1], [2, 7, 4, 6]])
pages = [torch.zeros(8, 2, kf.kv4_page_bytes(16, 128), dtype=torch.uint8, device="cuda") for _ in range(2)]
freqs, pos = kf.rope_freqs(128, device="cuda")[0], ints(list(range(90)))
O, Q1 = torch.empty(90, 8, 128, device="cuda"), half(2, 8, 1, 128)
O1, Qr, Kr, K4, V4 = torch.empty(2, 8, 1, 128, device="cuda"), *(torch.empty_like(x) for x in (Q, K, K, K))
calls = {
    "packed": (lambda: kf.attn_packed(Q, K, V, starts, O, causal=True), [O]),
    "rope": (lambda: kf.qk_norm_rope(Q, K, pos, freqs, (Qr, Kr)), [Qr, Kr]),
    "append": (lambda: kf.kv4_append(K, V, *pages, table, starts, lens), pages),
    "read": (lambda: kf.kv4_read(*pages, table, starts, lens, T, 128, (K4, V4)), [K4, V4]),
    "decode": (lambda: kf.attn_decode_kv4(Q1, *pages, table, lens, O1), [O1]),
}
for name in sys.argv[1:]:
    call, outs = calls[name]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for step in range(4):
        for x in (Q, K, V, Q1):
            x.mul_(0.9)
        for x in outs:
            x.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in outs]
        for x in outs:
            x.zero_()
        call()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, outs)), (name, step)
        assert name in ("read", "decode") or any(bool(x.any()) for x in outs)
    print("ok", name, flush=True)
"""


@pytest.mark.parametrize("names", [["packed"], ["rope"], ["append", "read"], ["decode"]], ids="-".join)
def test_the_first_call_is_captured(names, tmp_path):
    child = tmp_path / "child.py"
    child.write_text(CHILD)
    r = subprocess.run([sys.executable, str(child), *names], cwd=REPO, env=dict(os.environ, PYTHONPATH=REPO),
                       capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and r.stdout.split() == [w for n in names for w in ("ok", n)], r.stdout + r.stderr
