"""Each entry of the 16-bit cache captured into a graph as a process's first call of it, and
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
from tests import _cache_ref as ref

def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")

def half(*shape):
    return torch.randn(shape, device="cuda").half()

cache = ref.Cache([700, 3000, 90], 2, 128, torch.float16, 16)
first = cache.clone()
starts, T = ints([0, 1, 201, 231]), 231
Q, K, V, lse = half(T, 8, 128), half(T, 2, 128), half(T, 2, 128), torch.rand(T, 8, device="cuda") + 5
O, kept, budgets = torch.empty(T, 8, 128, device="cuda"), ints([0] * 3), ints([300, 1000, 80])
c, pools = cache, [cache.K, cache.V, cache.weights]
calls = {
    "append": (lambda: kf.kv_append(K, V, c.K, c.V, c.table, starts, c.lens, weights=c.weights), pools),
    "attend": (lambda: kf.attn_paged(Q, c.K, c.V, c.table, starts, c.lens, O, causal=True), [O]),
    "weigh": (lambda: kf.kv_weigh(Q, c.K, c.weights, c.table, starts, c.lens, lse, causal=True), [c.weights]),
    "evict": (lambda: kf.kv_evict(c.K, c.V, c.weights, c.table, c.lens, budgets, kept, recent=20), pools + [kept]),
}

def reset():
    for x, y in ((c.K, first.K), (c.V, first.V), (c.weights, first.weights)):
        x.copy_(y)
    O.zero_()
    kept.zero_()

for name in sys.argv[1:]:
    call, outs = calls[name]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for step in range(4):
        for x in (Q, K, V, lse, first.weights):
            x.mul_(0.9)
        budgets.sub_(7)
        reset()
        before = [x.clone() for x in outs]
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in outs]
        reset()
        call()
        torch.cuda.synchronize()
        bits = lambda x: x.view(torch.int16 if x.element_size() == 2 else torch.int32)
        assert all(torch.equal(bits(a), bits(b)) for a, b in zip(got, outs)), (name, step)
        assert not any(torch.equal(bits(a), bits(b)) for a, b in zip(got, before)), (name, step)
    print("ok", name, flush=True)
"""


@pytest.mark.parametrize("name", ["append", "attend", "weigh", "evict"])
def test_the_first_call_is_captured(name, tmp_path):
    child = tmp_path / "child.py"
    child.write_text(CHILD)
    r = subprocess.run([sys.executable, str(child), name], cwd=REPO, env=dict(os.environ, PYTHONPATH=REPO),
                       capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and r.stdout.split() == ["ok", name], r.stdout + r.stderr
