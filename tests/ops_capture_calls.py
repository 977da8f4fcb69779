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


def a_layer():
    """Refused on the captured stream; beside it, on another stream or from another
    thread, it is made.  The capture goes on."""
    import threading

    x = torch.ones(8, device="cuda")
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    out, made = {}, []

    def beside():
        made.append(layer())

    def capture():
        with torch.cuda.graph(graph):
            y = x + 1
            out["inside"] = said(layer)
            with torch.cuda.stream(side):
                out["other stream"] = said(beside)
            t = threading.Thread(target=lambda: out.update({"other thread": said(beside)}))
            t.start()
            t.join()
            made.append(y * 2)

    out["capture"] = said(capture)
    graph.replay()
    a, b, y = made
    torch.cuda.synchronize()
    out["replayed"] = bool((y == 4).all())
    eye = torch.eye(64, device="cuda")
    out["read"] = [bool(((m.matvec(eye) / 0.01).abs() <= 8.01).all()) for m in (a, b)]
    vb.check()
    return out


if __name__ == "__main__":
    layer()
    torch.cuda.synchronize()
    print(json.dumps({"a_failed_call": a_failed_call, "a_layer": a_layer}[sys.argv[1]]()))
