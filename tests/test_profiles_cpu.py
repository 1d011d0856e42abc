"""CPU: counters kept under profiles/ belong to the build that they were collected on."""
import json
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)


def test_r06_counters_are_those_of_their_build():
    """the figures quoted from this file are of that build: later sources' counters go to step_pmc_traffic.json"""
    with open(os.path.join(ROOT, "profiles", "r06_pmc_traffic.json")) as f:
        assert json.load(f)["source_fingerprint"] == "8b2c24a6a73243e6"


def test_traffic_is_taken_from_the_file_of_the_running_sources(tmp_path, monkeypatch):
    import bench
    from vision_longformer_amd import _lib
    os.mkdir(tmp_path / "profiles")
    for name, fp, n in (("r06", "other", 1), ("step", _lib.source_fingerprint(), 2), ("z", "another", 3)):
        with open(tmp_path / "profiles" / (name + "_pmc_traffic.json"), "w") as f:
            json.dump({"source_fingerprint": fp, "configs": {"c": {"per_gpu_batch": 8, "kernels": {"k": {"s": {"hbm_bytes_per_launch": n}}}}}}, f)
    monkeypatch.setattr(bench, "ROOT", str(tmp_path))
    assert bench.pmc_traffic("c", 8, "k", "s") == 2
    assert bench.pmc_traffic("c", 9, "k", "s") is None and bench.pmc_traffic("c", 8, "k", "t") is None
