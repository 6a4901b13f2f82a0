"""The 16-bit cache's entries with starts, counts, budgets and page ids that no caller should
pass: nothing outside the tensors and the workspace is read or written."""
import pytest
import torch

import kernelfoundry_amd as kf
from tests import _cache_ref as ref
from tests.test_kv4_gpu import normal
from tests.test_kv_cache_gpu import equal
from tests.test_serve_starts_gpu import between, disorder, untouched

pytestmark = pytest.mark.gpu

EDGE = 1 << 20   # bytes on either side of a workspace


def guarded(need):
    ws = torch.full((need + 2 * EDGE,), 77, dtype=torch.uint8, device="cuda")
    return ws, ws[EDGE : EDGE + need] if need else None


def test_sums_of_parts_that_pass_32_bits():
    """Starts by which every second sequence has the tokens that it says: 2^32 - 1 parts of
    one run's tiles in front of a sequence whose parts would lie in front of the workspace."""
    n, T, ratio, rows, unit = 512, 8184, 16, 128, 256
    tiles = T * ratio // rows
    lens, starts = [0] * n, [0] * (n + 1)
    # (tiles, units) of 8 sequences a run: one tile that is not cut, four with 2^32 - 1 parts, four tiles of two.
    work = {0: (1, 1), 8: (1023, 1229135), 10: (1023, 1229136), 12: (1023, 1229136), 14: (1022, 511497), 16: (4, 2)}
    assert tiles == 1023 and sum(a * b for i, (a, b) in work.items() if 8 <= i <= 14) == 2 ** 32 - 1
    for i, (a, b) in work.items():
        starts[i + 1], lens[i] = a * rows // ratio, b * unit
    pages = 341                                   # of 2^20 rows: a unit is 256 keys
    Q = torch.zeros(T, ratio, 64, dtype=torch.float16, device="cuda")
    K = torch.zeros(1, 1, 1 << 20, 64, dtype=torch.float16, device="cuda")
    table = torch.zeros(n, pages, dtype=torch.int32, device="cuda")
    need = kf.paged_attn_workspace_bytes(n, T, ratio, 1, 64, 1 << 20, pages)
    assert need > 0 and EDGE >= rows * 64 * 4     # a partial
    whole, ws = guarded(need)
    out, O, edge = between((T, ratio, 64), torch.float32, 3.25)
    kf.attn_paged(Q, K, K, table, torch.tensor(starts, dtype=torch.int32, device="cuda"),
                  torch.tensor(lens, dtype=torch.int32, device="cuda"), O, workspace=ws)
    torch.cuda.synchronize()
    assert untouched(whole, EDGE, 77) and untouched(out, edge, 3.25)


@pytest.mark.parametrize("n", [1, 10, 64, 65, 700])
@pytest.mark.parametrize("heads", [(8, 2, 128), (4, 1, 64), (4, 2, 256), (64, 1, 64)])
@pytest.mark.parametrize("T", [3, 600])
def test_arrays_in_no_order(n, heads, T):
    """As uninitialised memory holds them."""
    H_q, H_kv, D = heads
    cols, pages = 40, 14
    (wk, Kp, edge), (wv, Vp, _) = (between((pages, H_kv, 16, D), torch.float16, 3.25) for _ in range(2))
    (ww, W, wedge), (wo, O, oedge) = between(Kp.shape[:3], torch.float32, 3.25), between((T, H_q, D), torch.float32, 3.25)
    spaces = [guarded(size) for size in (kf.paged_attn_workspace_bytes(n, T, H_q, H_kv, D, 16, cols),
                                         kf.weigh_workspace_bytes(n, T, H_q, H_kv, D, 16, cols),
                                         kf.evict_workspace_bytes(n, H_kv, D, 16, cols))]
    Q, K = normal(T, H_q, D), normal(T, H_kv, D, seed=1)
    for seed in range(3):
        # (disorder(n, ...) has n + 1 numbers.)
        table = disorder(n * cols - 1, pages, seed).view(n, cols)
        table[::2] = torch.arange(table[::2].numel(), dtype=torch.int32, device="cuda").view(-1, cols) % pages   # all valid
        starts, lens, budgets = disorder(n, T, seed + 3), disorder(n - 1, 16 * cols, seed + 6), disorder(n - 1, 200, seed + 7)
        kf.kv_append(K, K, Kp, Vp, table, starts, lens, weights=W)
        for causal in (True, False):
            _, lse = kf.attn_paged(Q, Kp, Vp, table, starts, lens, O, causal=causal, return_lse=True, workspace=spaces[0][1])
            kf.kv_weigh(Q, Kp, W, table, starts, lens, lse, causal=causal, workspace=spaces[1][1])
        kept = kf.kv_evict(Kp, Vp, W, table, lens, budgets, recent=seed * 5, workspace=spaces[2][1])
        torch.cuda.synchronize()
        for whole, _ in spaces:
            assert untouched(whole, EDGE, 77)
        assert untouched(wk, edge, 3.25) and untouched(wv, edge, 3.25) and untouched(ww, wedge, 3.25)
        assert untouched(wo, oedge, 3.25) and kept.shape == (n,) and bool((kept >= 0).all() and (kept <= 16 * cols).all())


@pytest.mark.parametrize("D", [64, 128, 256])
def test_evictions_that_share_pages_stay_inside(D):
    """Sequences that are cut with pages of each other, and one with a page twice."""
    cache = ref.Cache([500, 500, 1000], 2, D, torch.float16, 16)
    cache.table[1, :20] = cache.table[0, :20]
    cache.table[0, 25] = cache.table[0, 24]
    cache.table[2, 10:30] = cache.table[2, 30:50]
    used = torch.zeros(cache.K.shape[0], dtype=torch.bool, device="cuda")
    for b, n in enumerate(cache.keys):
        used[cache.table[b, : -(-n // 16)].long()] = True
    assert not used.all()
    want = cache.clone()
    whole, ws = guarded(kf.evict_workspace_bytes(3, 2, D, 16, cache.table.shape[1]))
    got = kf.kv_evict(cache.K, cache.V, cache.weights, cache.table, cache.lens,
                      torch.tensor([100, 250, 900], dtype=torch.int32, device="cuda"), recent=9, workspace=ws)
    torch.cuda.synchronize()
    assert got.tolist() == [100, 250, 900] and untouched(whole, EDGE, 77)
    for a, b in ((cache.K, want.K), (cache.V, want.V), (cache.weights, want.weights)):
        assert equal(a[~used], b[~used])
