"""Worker of tests/test_gpu_beam_search.py: the first call of every operator of beam search and of the cache
in a process is one that is captured.  Prints "same"."""
from __future__ import annotations

import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

import verbo_b200 as vb  # noqa: E402


def made(width):
    c = vb.PagedCache.new(1, 60, 2, 64, 4, width, 16)
    g = torch.Generator(device="cuda").manual_seed(1)
    kv = torch.randn(4, 2, 64, generator=g, device="cuda")
    q = torch.randn(4, 8, 64, generator=g, device="cuda").half()
    x = torch.randn(4, 1000, generator=g, device="cuda")
    return c, kv, q, x, torch.ones(4, dtype=torch.int32, device="cuda"), torch.zeros(4, device="cuda")


def step(c, kv, q, x, one, scores):
    start, status = c.reserve(one)
    c.append(0, kv, kv, start)
    y = c.attend(0, q)
    s, p, t = vb.beam_select(x, scores, 2, 4)
    c.fork(p, 2)
    state = x[:, :8].contiguous()
    vb.beam_reorder(state, p, 2)
    c.free(one)
    info = c.compact()
    return start, status, y, s, p, t, state, info, c.table, c.lens, c.refs


for width in (4, 8000):
    a, b = made(width), made(width)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(*a)
    graph.replay()
    want = step(*b)
    vb.check()
    assert all(torch.equal(x, y) for x, y in zip(got, want))
print("same")
