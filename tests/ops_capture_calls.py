"""Worker of tests/test_gpu_ops_capture.py: calls that cannot be captured, made while
a stream is being captured, in a process of its own.  Prints one JSON line."""
from __future__ import annotations

import json
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

import verbo_b200 as vb  # noqa: E402


def layer():
    q = torch.randint(0, 256, (64, 32), dtype=torch.uint8)
    return vb.Q4Linear(q, torch.full((64, 2), 0.01, dtype=torch.float16))


def said(fn):
    """What a call answers: "" or its error's text."""
    try:
        fn()
        return ""
    except Exception as e:
        return f"{type(e).__name__}: {e}"


def a_failed_call():
    """vb.check() synchronises, so it fails inside a capture, which it ends."""
    x = torch.ones(8, device="cuda")
    out = {}

    def capture():
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            x + 1
            out["inside"] = said(vb.check)

    out["capture"] = said(capture)
    out["next layer"] = said(layer)
    out["next check"] = said(vb.check)
    return out


if __name__ == "__main__":
    layer()
    torch.cuda.synchronize()
    print(json.dumps({"a_failed_call": a_failed_call}[sys.argv[1]]()))
