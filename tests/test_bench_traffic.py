"""The committed HBM traffic of the headline prefill is that of the sources in the tree."""
import json

import bench


def test_the_traffic_was_collected_on_these_sources():
    traffic, note = bench.committed_traffic()
    assert traffic is not None, note
    with open(bench.TRAFFIC_FILE) as f:
        t = json.load(f)
    assert traffic == (t["fetch_size_kib_raw"] * t["fetch_scale"] + t["write_size_kib_raw"] * t["write_scale"]) * 1024
    # Q, K, V in fp16 and O in fp32, each once: what no kernel can do without.
    assert t["algorithmic_bytes_per_launch"] == 4096 * 128 * (32 * 2 + 2 * 8 * 2 + 32 * 4) <= traffic
