"""bench.py where the reference and its weight image are not at hand."""
import json
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
sys.path.insert(0, str(ROOT))

import bench  # noqa: E402


@pytest.mark.parametrize("workload", ["config1", "config2", "config4", "config5"])
def test_the_reference_arm_says_why_it_cannot_run(workload, monkeypatch, capsys, tmp_path):
    import oracle.oracle
    monkeypatch.setattr(oracle.oracle, "REF_SO", tmp_path / "libhkbref.so")
    monkeypatch.setattr(sys, "argv", ["bench.py", "--impl", "reference", "--workload", workload])
    assert bench.main() == 0
    line = json.loads(capsys.readouterr().out)
    assert line["impl"] == "reference" and "sources" in line["unavailable"]
    (tmp_path / "libhkbref.so").write_bytes(b"")
    monkeypatch.setattr(bench, "WEIGHTS", tmp_path / "none.safetensors")
    assert bench.main() == 0
    assert "weight image" in json.loads(capsys.readouterr().out)["unavailable"]


def test_random_weights_are_named(monkeypatch, tmp_path):
    monkeypatch.setattr(bench, "WEIGHTS", tmp_path / "none.safetensors")
    assert isinstance(bench.engine_weights(), bytes) and "random weights" in bench.data_note("x")
    image = tmp_path / "some.safetensors"
    image.write_bytes(b"")
    monkeypatch.setattr(bench, "WEIGHTS", image)
    assert bench.engine_weights() == image and bench.data_note("x") == "x"


def test_the_reference_arm_exits_with_0_as_a_command():
    from oracle.oracle import REF_SO
    if REF_SO.exists() and bench.published_weights():
        pytest.skip("the reference is at hand and would run")
    done = subprocess.run([sys.executable, "bench.py", "--impl", "reference"], cwd=ROOT,
                          capture_output=True, text=True)
    assert done.returncode == 0 and "unavailable" in json.loads(done.stdout), done.stderr
