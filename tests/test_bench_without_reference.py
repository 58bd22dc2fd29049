"""bench.py where CacheFlow's own CPU build is missing: its own arm prints its
line all the same, the reference arm says that it is unavailable, and why."""

import json
import sys
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]
sys.path.insert(0, str(ROOT))


def test_reference_arm_says_why(monkeypatch, capsys, tmp_path):
    import bench
    from oracle import oracle

    monkeypatch.setattr(oracle, "REF_CPU_LIB", tmp_path / "libcf_ref_cpu.so")
    monkeypatch.setattr(sys, "argv", ["bench.py", "--impl", "reference", "--steps", "1"])
    bench.main()
    lines = capsys.readouterr().out.splitlines()
    assert len(lines) == 1
    d = json.loads(lines[0])
    assert d["impl"] == "reference" and "libcf_ref_cpu.so" in d["unavailable"] and set(d) == {"impl", "unavailable"}


def test_own_arm_keeps_its_line(monkeypatch, tmp_path):
    import bench
    from cacheflow_b200 import workloads
    from oracle import oracle

    monkeypatch.setattr(oracle, "REF_CPU_LIB", tmp_path / "libcf_ref_cpu.so")
    monkeypatch.setattr(bench, "cpu_port_baseline", lambda w: {"kind": "port", "of": w.name})
    d = bench.cpu_baselines(workloads.make("cpu_decode_fp32"), 0.1)
    assert "libcf_ref_cpu.so" in d["cpu_baseline"]["unavailable"]
    assert d["cpu_port"] == {"kind": "port", "of": "cpu_decode_fp32"}
