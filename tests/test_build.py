"""The build on a machine without torch."""
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
