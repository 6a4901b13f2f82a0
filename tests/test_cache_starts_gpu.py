"""The 16-bit cache's entries with starts, counts, budgets and page ids that no caller should
pass: nothing outside the tensors and the workspace is read or written."""
import pytest
import torch

import kernelfoundry_amd as kf
from tests.test_serve_starts_gpu import between, untouched

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
