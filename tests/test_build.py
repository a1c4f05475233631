"""The build on a machine without torch, and after torch was replaced."""
import subprocess
import sys
from pathlib import Path

from hikoboshi_b200 import _build

ROOT = Path(__file__).resolve().parents[1]


def test_the_library_builds_without_torch():
    code = ("import sys; sys.modules['torch'] = None; from hikoboshi_b200 import _build; "
            "assert _build.build_library() == _build.LIB and _build.LIB.exists(); "
            "assert _build.build_vocab_module() is None")
    done = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)
    assert done.returncode == 0, done.stderr
    assert "torch cannot be imported" in done.stdout


def test_the_binding_is_compiled_anew_for_another_torch(tmp_path, monkeypatch):
    import torch
    module, stamp, runs = tmp_path / "_vocab.so", tmp_path / "_vocab.stamp", []

    def compiler(cmd, check):
        runs.append(cmd)
        module.write_bytes(b"")

    monkeypatch.setattr(_build, "VOCAB_MODULE", module)
    monkeypatch.setattr(_build, "VOCAB_STAMP", stamp, raising=False)
    monkeypatch.setattr(_build.subprocess, "run", compiler)
    assert _build.build_vocab_module() == module and len(runs) == 1
    assert _build.build_vocab_module() == module and len(runs) == 1  # nothing has changed
    monkeypatch.setattr(torch, "__version__", "99.0")
    assert _build.build_vocab_module() == module and len(runs) == 2
    assert _build.build_vocab_module() == module and len(runs) == 2
    stamp.unlink()  # of unknown origin
    assert _build.build_vocab_module() == module and len(runs) == 3


def test_the_build_script_runs_without_a_weight_image(tmp_path):
    import os
    env = dict(os.environ, HKB_REFERENCE_ROOT=str(tmp_path))
    done = subprocess.run([sys.executable, str(ROOT / "hikoboshi_b200" / "_build.py")], env=env,
                          capture_output=True, text=True)
    assert done.returncode == 0, done.stderr
