"""`roofline.traffic_source` of the bench line names the build that a committed counter summary is of, where it
is not the library that was timed (no GPU)."""
import hashlib
import json

import bench


def test_a_summary_of_another_build_says_so(tmp_path, monkeypatch):
    lib = tmp_path / "lib.so"
    lib.write_bytes(b"one build")
    here = hashlib.sha256(b"one build").hexdigest()[:16]
    (tmp_path / "profiles").mkdir()
    monkeypatch.setattr(bench, "ROOT", str(tmp_path))
    monkeypatch.setattr(bench, "library_path", lambda: str(lib))
    for theirs, source in ((None, "r50_summary.json"), (here, "r50_summary.json"),
                           ("0123456789abcdef", f"r50_summary.json, of library 0123456789abcdef; this one is {here}")):
        d = {"hbm_bytes_per_launch": 5e9, "library_sha256": theirs,
             "bench_line_under_profiler": {"config": {"workload": "W", "prune_interval": 25},
                                           "roofline": {"utterance_frames_per_launch": 1000}}}
        (tmp_path / "profiles" / "r50_summary.json").write_text(json.dumps(d))
        assert bench.profiled_traffic("W", 1000, 25) == (5e9, source)
