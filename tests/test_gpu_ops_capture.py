"""GPU tests of what the operators' calls do to a capture and to one another after
a failure, each in a process of its own (tests/ops_capture_calls.py)."""
from __future__ import annotations

import json
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

ROOT = Path(__file__).resolve().parent.parent


def worker(cuda_lib, name):
    if not torch.cuda.is_available():
        pytest.fail("gpu tests need a CUDA device")
    r = subprocess.run([sys.executable, str(ROOT / "tests" / "ops_capture_calls.py"), name], capture_output=True,
                       text=True, timeout=300, cwd=ROOT)
    assert r.returncode == 0, r.stderr[-2000:]
    return json.loads(r.stdout.strip().splitlines()[-1])


def test_a_failed_call_leaves_nothing_behind(cuda_lib):
    """The error of a failed call is that call's alone."""
    got = worker(cuda_lib, "a_failed_call")
    assert got["inside"].startswith("VerboCudaError")
    assert got["next layer"] == "" and got["next check"] == ""


def test_a_layer_made_during_a_capture(cuda_lib):
    got = worker(cuda_lib, "a_layer")
    assert "being captured" in got["inside"]
    assert got["other stream"] == "" and got["other thread"] == "" and got["capture"] == ""
    assert got["replayed"] and got["read"] == [True, True]
