"""The block operators' tests on the bounds-checked build (libgfield_check.so):
the same results, and no access outside its extent (every test there asserts
that no condition bit is set)."""
from __future__ import annotations

import os
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parent.parent


def test_block_operators_stay_in_bounds():
    from guass_b200 import _build

    assert _build.LIB_CHECK.exists(), "build it with python -m guass_b200._build"
    env = dict(os.environ, GUASS_B200_LIB=str(_build.LIB_CHECK))
    few = ("test_ff and not many_tiles or test_dropout and not large or test_quantize or test_int8 and not many_rows "
           "or test_calls")
    res = subprocess.run([sys.executable, "-m", "pytest", "-x", "-q", "-m", "gpu", "-k", few, "-p", "no:cacheprovider",
                          str(ROOT / "tests" / "test_gpu_block.py")], env=env, capture_output=True, text=True,
                         timeout=900, cwd=ROOT)
    assert res.returncode == 0, (res.stdout + res.stderr)[-3000:]
    assert " passed" in res.stdout and "skipped" not in res.stdout
