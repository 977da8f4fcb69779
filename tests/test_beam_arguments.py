"""CPU tests of include/verbo_beam.h and verbo_b200/beam.py (no kernel launches):
the exported symbols and the refusals, which come before the GPU is touched."""
from __future__ import annotations

import ctypes
import re
import subprocess
from pathlib import Path

import pytest

import verbo_b200 as vb
from verbo_b200 import beam, build

torch = pytest.importorskip("torch")

ROOT = Path(__file__).resolve().parent.parent
F32, F16, BF16 = 0, 1, 2
BIG = 1 << 40


@pytest.fixture(scope="module")
def lib():
    build.build()
    return beam._beam()[0]


def test_exports_match_header(lib):
    text = (ROOT / "include" / "verbo_beam.h").read_text()
    declared = sorted(set(re.findall(r"VERBO_CUDA_API\s+[^;(]*?\b(verbo_beam_\w+)\s*\(", text)))
    out = subprocess.run(["nm", "-D", "--defined-only", str(build.LIB)], capture_output=True, text=True,
                         check=True).stdout
    assert sorted(ln.split()[-1] for ln in out.splitlines() if ln.split()[-1].startswith("verbo_beam_")) == declared
    assert declared == ["verbo_beam_reorder", "verbo_beam_select", "verbo_beam_workspace"]


def test_header_compiles_as_c(lib, tmp_path):
    src = tmp_path / "use.c"
    src.write_text('#include "verbo_beam.h"\nint main(void) { return verbo_beam_workspace(1, 4, 8) > 0 ? 0 : 1; }\n')
    exe = tmp_path / "use"
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", f"-I{ROOT / 'include'}", str(src), f"-L{build.LIB.parent}",
                    "-lverbo_cuda", f"-Wl,-rpath,{build.LIB.parent}", "-o", str(exe)], check=True, capture_output=True)
    assert subprocess.run([str(exe)]).returncode == 0


def refused(lib, rc, msg):
    assert rc == -1
    text = lib.verbo_cuda_last_error().decode()
    assert msg in text, text


def select(lib, **kw):
    a = dict(logits=1 << 20, dtype=F32, requests=2, beams=2, vocab=8, ld=8, scores=1 << 21, take=4, out=1 << 22,
             parents=1 << 23, tokens=1 << 24, ws=1 << 25, bytes=1 << 20)
    a.update(kw)
    return lib.verbo_beam_select(a["logits"], a["dtype"], a["requests"], a["beams"], a["vocab"], a["ld"], a["scores"],
                                 a["take"], a["out"], a["parents"], a["tokens"], a["ws"], a["bytes"], None)


@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=3), "dtype"),
    (dict(requests=-1), "requests"),
    (dict(requests=2**31 - 1), "rows"),
    (dict(beams=0), "beams"),
    (dict(beams=33), "beams"),
    (dict(take=0), "take"),
    (dict(take=65), "take"),
    (dict(vocab=0), "vocab"),
    (dict(vocab=4194305, ld=4194305), "vocab"),
    (dict(ld=7), "stride"),
    (dict(ld=1 << 61), "stride"),
    (dict(logits=None), "NULL"),
    (dict(scores=None), "NULL"),
    (dict(out=None), "NULL"),
    (dict(parents=None), "NULL"),
    (dict(tokens=None), "NULL"),
    (dict(logits=(1 << 20) + 2), "aligned"),
    (dict(scores=6), "scores must be aligned"),
    (dict(out=6), "out_scores must be aligned"),
    (dict(parents=6), "parents must be aligned"),
    (dict(tokens=6), "tokens must be aligned"),
    (dict(ws=None), "workspace"),
    (dict(bytes=4 * 6 * 8 - 1), "workspace"),
    (dict(ws=(1 << 25) + 8), "workspace must be aligned"),
    (dict(out=1 << 21), "overlaps scores"),
    (dict(take=2, out=(1 << 21) + 4), "overlaps scores"),
    (dict(parents=1 << 21), "overlaps scores"),
    (dict(tokens=(1 << 20) + 32), "overlaps logits"),
    (dict(tokens=1 << 22), "overlap"),
    (dict(parents=(1 << 22) + 28), "overlap"),
    (dict(out=1 << 25), "overlaps the workspace"),
    (dict(ws=1 << 20), "overlaps logits"),
    (dict(ws=1 << 21), "overlaps logits or scores"),
])
def test_select_refusals(lib, kw, msg):
    refused(lib, select(lib, **kw), msg)


def test_select_of_nothing(lib):
    assert select(lib, requests=0, logits=None, ws=None, bytes=0) == 0


def test_workspace(lib):
    assert lib.verbo_beam_workspace(2, 2, 4) == 4 * 6 * 8
    assert lib.verbo_beam_workspace(0, 1, 1) == 0
    refused(lib, lib.verbo_beam_workspace(1, 33, 1), "beams")
    refused(lib, lib.verbo_beam_workspace(1, 1, 65), "take")
    refused(lib, lib.verbo_beam_workspace(-1, 1, 1), "requests")


def reorder(lib, states, requests=2, beams=2, parents=1 << 20, ld=2, n=None):
    items = (beam._State * max(1, len(states)))(*[beam._State(*s) for s in states])
    return lib.verbo_beam_reorder(items, len(states) if n is None else n, requests, beams, parents, ld, None)


@pytest.mark.parametrize("states,kw,msg", [
    ([(1 << 24, 16, 16)], dict(requests=-1), "requests"),
    ([(1 << 24, 16, 16)], dict(beams=0), "beams"),
    ([(1 << 24, 16, 16)], dict(beams=33), "beams"),
    ([(1 << 24, 16, 16)], dict(n=-1), "n must"),
    ([(1 << 24, 16, 16)], dict(parents=None), "NULL"),
    ([(1 << 24, 16, 16)], dict(parents=6), "aligned"),
    ([(1 << 24, 16, 16)], dict(ld=1), "ld_parents"),
    ([(1 << 24, 16, 16)], dict(ld=1 << 60), "ld_parents"),
    ([(None, 16, 16)], {}, "NULL"),
    ([(1 << 24, -1, 16)], {}, "row_bytes"),
    ([(1 << 24, 16, 15)], {}, "stride"),
    ([(1 << 24, 16, 1 << 60)], {}, "stride"),
    ([((1 << 20) - 48, 16, 16)], {}, "overlaps parents"),
    ([(1 << 24, 16, 16), (1 << 24, 16, 16)], {}, "two states overlap"),
    ([(1 << 24, 16, 32), ((1 << 24) + 8, 16, 32)], {}, "two states overlap"),
])
def test_reorder_refusals(lib, states, kw, msg):
    refused(lib, reorder(lib, states, **kw), msg)


def test_reorder_of_nothing(lib):
    assert reorder(lib, []) == 0
    assert reorder(lib, [(1 << 24, 16, 16)], requests=0) == 0
    assert reorder(lib, [(None, 0, 0)]) == 0


@pytest.mark.parametrize("kw,msg", [
    (dict(beams=0), "beams"),
    (dict(beams=33), "beams"),
    (dict(beams=2**32 + 1), "beams"),
    (dict(take=0), "take"),
    (dict(take=65), "take"),
    (dict(take=2**32 + 1), "take"),
    (dict(), "CUDA"),
])
def test_python_select(kw, msg):
    with pytest.raises(vb.VerboCudaError, match=msg):
        vb.beam_select(**{**dict(logits=torch.zeros(4, 8), scores=torch.zeros(4), beams=2, take=2), **kw})


def test_python_reorder():
    p = torch.zeros(2, 2, dtype=torch.int32)
    for states, parents, beams in ((torch.zeros(4, 3), p, 2), (torch.zeros(3, 3), p, 2), (torch.zeros(()), p, 2),
                                   (torch.zeros(4, 3), p[:1], 2), (torch.zeros(4, 3), p, 33),
                                   (torch.zeros(4, 3), p.long(), 2)):
        with pytest.raises(vb.VerboCudaError):
            vb.beam_reorder(states, parents, beams)
    vb.beam_reorder([], p, 2)
