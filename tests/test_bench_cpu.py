"""Host-side helpers of bench.py: no GPU needed."""
import json
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)


def test_traffic_record_goes_by_the_sources_not_by_its_name(tmp_path):
    import bench
    assert bench.traffic_record(tmp_path, "a") == (None, None)
    for name, sha in (("r01", "a"), ("recorded", "b"), ("r99", "c")):
        (tmp_path / f"{name}_pmc_step_traffic.json").write_text(json.dumps({"_meta": {"csrc_sha256": sha}, "classes": {"k": name}}))
    for name, sha in (("r01", "a"), ("recorded", "b"), ("r99", "c")):
        got, rec = bench.traffic_record(tmp_path, sha)
        assert got == f"{name}_pmc_step_traffic.json" and rec["classes"] == {"k": name}
    name, rec = bench.traffic_record(tmp_path, "d")
    assert name.endswith("_pmc_step_traffic.json") and rec is None
