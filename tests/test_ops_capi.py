"""CPU tests of include/verbo_ops.h (no kernel launches): the exported symbols
and the refusals, which come before the GPU is touched."""
from __future__ import annotations

import ctypes
import re
import subprocess
from pathlib import Path

import pytest

import verbo_b200 as vb
from verbo_b200 import build, ops

ROOT = Path(__file__).resolve().parent.parent
F32, F16, BF16 = 0, 1, 2


@pytest.fixture(scope="module")
def lib():
    build.build()
    return ops._ops()[0]


def test_exports_match_header(lib):
    text = (ROOT / "include" / "verbo_ops.h").read_text()
    declared = sorted(set(re.findall(r"VERBO_CUDA_API\s+[^;(]*?\b(verbo_ops_\w+)\s*\(", text)))
    out = subprocess.run(["nm", "-D", "--defined-only", str(build.LIB)], capture_output=True, text=True,
                         check=True).stdout
    assert sorted(ln.split()[-1] for ln in out.splitlines() if ln.split()[-1].startswith("verbo_ops_")) == declared
    assert len(declared) == 7


def test_header_compiles_as_c(lib, tmp_path):
    src = tmp_path / "use.c"
    src.write_text('#include "verbo_ops.h"\nint main(void) { verbo_ops_penalties p = verbo_ops_default_penalties();\n'
                   'return p.repeat == 1.0f && p.frequency == 0.0f && p.presence == 0.0f && p.last == 0 ? 0 : 1; }\n')
    exe = tmp_path / "use"
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", f"-I{ROOT / 'include'}", str(src), f"-L{build.LIB.parent}",
                    "-lverbo_cuda", f"-Wl,-rpath,{build.LIB.parent}", "-o", str(exe)], check=True, capture_output=True)
    assert subprocess.run([str(exe)]).returncode == 0


def refused(lib, rc, msg):
    assert rc == -1
    text = lib.verbo_cuda_last_error().decode()
    assert msg in text, text


def process(lib, **kw):
    a = dict(logits=1 << 20, dtype=F32, rows=2, vocab=8, ld=8, opts=vb.Penalties(1.1), row=None, hist=None, off=None,
             bias_ids=None, bias=None, bias_off=None, mask=None, ld_mask=0, out=1 << 24, ld_out=8)
    a.update(kw)
    o = a["opts"]
    return lib.verbo_ops_process_logits(a["logits"], a["dtype"], a["rows"], a["vocab"], a["ld"],
                                        ctypes.byref(o) if o is not None else None, a["row"], a["hist"], a["off"],
                                        a["bias_ids"], a["bias"], a["bias_off"], a["mask"], a["ld_mask"], a["out"],
                                        a["ld_out"], None)


@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=3), "dtype"),
    (dict(dtype=-1), "dtype"),
    (dict(rows=-1), "rows"),
    (dict(vocab=0), "vocab"),
    (dict(vocab=5000000, ld=5000000, ld_out=5000000), "vocab"),
    (dict(ld=7), "stride"),
    (dict(ld_out=7), "stride"),
    (dict(ld=1 << 61), "stride"),
    (dict(logits=None), "NULL"),
    (dict(out=None), "NULL"),
    (dict(logits=(1 << 20) + 2), "aligned"),
    (dict(out=(1 << 24) + 1), "aligned"),
    (dict(hist=1), "hist"),
    (dict(off=1), "hist"),
    (dict(bias=4, bias_ids=4), "bias"),
    (dict(bias=4, bias_off=8), "bias"),
    (dict(bias_off=8), "bias"),
    (dict(row=4, opts=None), "row_penalties"),
    (dict(opts=vb.Penalties(0.0)), "repeat"),
    (dict(opts=vb.Penalties(-1.1)), "repeat"),
    (dict(opts=vb.Penalties(float("nan"))), "repeat"),
    (dict(opts=vb.Penalties(float("inf"))), "repeat"),
    (dict(opts=vb.Penalties(1.0, float("inf"))), "frequency"),
    (dict(opts=vb.Penalties(1.0, 0.0, float("nan"))), "presence"),
    (dict(mask=4, ld_mask=1, vocab=40, ld=40, ld_out=40), "ld_mask"),
    (dict(mask=6), "aligned"),
    (dict(row=6), "row_penalties must be aligned"),
    (dict(hist=6, off=8), "hist must be aligned"),
    (dict(hist=4, off=4), "hist_off must be aligned"),
    (dict(bias=4, bias_ids=5, bias_off=8), "bias_ids must be aligned"),
    (dict(bias=6, bias_ids=4, bias_off=8), "bias must be aligned"),
    (dict(bias=4, bias_ids=4, bias_off=4), "bias_off must be aligned"),
    (dict(dtype=BF16, out=1 << 20), "out may be logits"),
    (dict(out=1 << 20, ld_out=9), "out may be logits"),
    (dict(out=(1 << 20) + 4), "overlaps"),
    (dict(out=(1 << 20) + 32), "overlaps"),
    (dict(out=(1 << 20) - 32), "overlaps"),
    (dict(dtype=F16, out=(1 << 20) + 16), "overlaps"),
    (dict(ld=16, ld_out=16, out=(1 << 20) + 40), "overlaps"),
])
def test_process_refusals(lib, kw, msg):
    refused(lib, process(lib, **kw), msg)


def test_process_of_nothing(lib):
    assert process(lib, rows=0, logits=None, out=None) == 0
    # in place with nothing to change: no launch
    assert process(lib, out=1 << 20) == 0
    assert process(lib, out=1 << 20, opts=vb.Penalties(), hist=4, off=8) == 0


def logprobs(lib, **kw):
    a = dict(logits=1 << 20, dtype=F32, rows=2, vocab=8, ld=8, temp=1.0, ids=4, lp=4, rank=4, top=0, tid=None, tlp=None)
    a.update(kw)
    return lib.verbo_ops_token_logprobs(a["logits"], a["dtype"], a["rows"], a["vocab"], a["ld"], a["temp"], a["ids"],
                                        a["lp"], a["rank"], a["top"], a["tid"], a["tlp"], None)


@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=9), "dtype"),
    (dict(rows=-2), "rows"),
    (dict(vocab=0), "vocab"),
    (dict(ld=4), "stride"),
    (dict(logits=None), "NULL"),
    (dict(dtype=F16, logits=(1 << 20) + 1), "aligned"),
    (dict(ids=5), "ids must be aligned"),
    (dict(lp=6), "logprob must be aligned"),
    (dict(rank=7), "rank must be aligned"),
    (dict(top=1, tid=6, tlp=4), "top_ids must be aligned"),
    (dict(top=1, tid=4, tlp=6), "top_logprobs must be aligned"),
    (dict(temp=0.0), "temp"),
    (dict(temp=-1.0), "temp"),
    (dict(temp=float("nan")), "temp"),
    (dict(temp=float("inf")), "temp"),
    (dict(top=33, tid=4, tlp=4), "top"),
    (dict(top=-1), "top"),
    (dict(top=1, tid=4), "top_ids"),
    (dict(lp=None), "logprob"),
    (dict(rank=None), "rank"),
])
def test_logprobs_refusals(lib, kw, msg):
    refused(lib, logprobs(lib, **kw), msg)


def test_logprobs_of_nothing(lib):
    assert logprobs(lib, rows=0, logits=None) == 0
    assert logprobs(lib, ids=None, lp=None, rank=None) == 0


@pytest.mark.parametrize("kw,msg", [
    (dict(q=None), "NULL"),
    (dict(s=None), "NULL"),
    (dict(outs=0), "outs"),
    (dict(outs=(1 << 22) + 1), "outs"),
    (dict(ins=0), "ins"),
    (dict(ins=48), "ins"),
    (dict(ins=32800), "ins"),
    (dict(group=0), "group"),
    (dict(group=16), "group"),
    (dict(group=48), "group"),
    (dict(s=5), "aligned"),
    (dict(bias=6), "aligned"),
])
def test_q4_new_refusals(lib, kw, msg):
    a = dict(outs=4, ins=64, group=32, q=4, s=4, zeros=None, bias=None)
    a.update(kw)
    assert lib.verbo_ops_q4_new(a["outs"], a["ins"], a["group"], a["q"], a["s"], a["zeros"], a["bias"], 0, None) is None
    assert msg in lib.verbo_cuda_last_error().decode()


def test_q4_null_handle(lib):
    refused(lib, lib.verbo_ops_q4_matvec(None, 4, 0, 1, 64, 4, 0, 64, None, 0, None), "NULL")
    refused(lib, lib.verbo_ops_q4_workspace(None, 0, 1), "NULL")
    lib.verbo_ops_q4_free(None)


def test_python_refuses_host_tensors():
    import torch

    x = torch.zeros(2, 8)
    with pytest.raises(vb.VerboCudaError, match="CUDA"):
        vb.process_logits(x)
    with pytest.raises(vb.VerboCudaError, match="CUDA"):
        vb.token_logprobs(x, top=1)


def test_q4_python_refusals():
    import torch

    if not torch.cuda.is_available():
        device = "cuda:0"
    else:
        device = 0
    q, s = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.float16)
    bad = [dict(q=q.int()), dict(q=q[0]), dict(s=s.float()), dict(s=s[:, :1]), dict(group=64), dict(group=0),
           dict(zeros=torch.zeros(4, 1, dtype=torch.uint8)), dict(bias=torch.zeros(3)), dict(bias=torch.zeros(4).half())]
    for kw in bad:
        with pytest.raises(vb.VerboCudaError):
            vb.Q4Linear(**{**dict(q=q, s=s, group=32, device=device), **kw})
