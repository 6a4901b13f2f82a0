"""kf_attn_packed's choice of a layout, from the constants in serve_capi.hip, for
tests that have to reach each of them."""
import math
import os
import re

from tests.conftest import REPO

SOURCE = os.path.join(REPO, "kernelfoundry_amd", "csrc", "serve_capi.hip")


def layouts():
    """{D: [(rows, KV groups, start, chain, workgroup, tile), ...]} of the cost model."""
    text = open(SOURCE).read()
    found = {}
    for D, body in re.findall(r"PackedLayout kPacked(\d+)\[\d\] = \{(.*?)\};", text, re.S):
        found[int(D)] = [tuple(float(v) for v in row.split(",")) for row in re.findall(r"\{([^{}]+)\}", body)]
    return found


def packed_layout(heads, lens, kv_lens, causal, cus=256):
    """packed_layout() of serve_capi.hip: the cheapest by the averages."""
    H_q, H_kv, D = heads
    n, ratio = len(lens), H_q // H_kv
    queries, keys = max(1.0, sum(lens) / n), sum(kv_lens) / n
    costs = []
    for rows, groups, start, chain, workgroup, tile in layouts()[D]:
        tiles = math.ceil(queries * ratio / rows)
        seen = min(keys, keys - (queries - 1) / 2 + rows / (2 * ratio)) if causal and tiles > 1 else keys
        key_tiles = max(seen, 0.0) / 32 + 0.5 + (0.5 * groups if groups > 1 else 0.0)
        longest = start + chain * math.ceil(math.ceil(keys / 32) / groups)
        work = n * H_kv * tiles * (workgroup + tile * key_tiles / groups) / cus
        costs.append((longest ** 4 + work ** 4) ** 0.25)
    return costs.index(min(costs))
