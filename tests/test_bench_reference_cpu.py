"""The reference arm of bench.py where the reference is not installed: it says so, and times nothing in its place."""
import json

import pytest


@pytest.mark.parametrize("workload", ["config1", "config2"])
def test_an_absent_reference_is_unavailable(workload, monkeypatch, capsys, tmp_path):
    import bench
    monkeypatch.setattr(bench, "REF_DIR", str(tmp_path))
    monkeypatch.setattr(bench, "cpu_baseline", lambda *a, **k: pytest.fail("something else was timed as the reference"))
    monkeypatch.setattr("sys.argv", ["bench.py", "--impl", "reference", "--workload", workload, "--steps", "1",
                                     "--warmup", "1"])
    bench.main()
    line = json.loads(capsys.readouterr().out.strip().splitlines()[-1])
    assert line["impl"] == "reference" and "baseline/_ref" in line["unavailable"] and "value" not in line
