"""CPU tests of include/verbo_cache.h and verbo_b200/cache.py (no kernel launches):
the exported symbols and the refusals, which come before the GPU is touched."""
from __future__ import annotations

import copy
import ctypes
import pickle
import re
import subprocess
from pathlib import Path

import pytest

import verbo_b200 as vb
from verbo_b200 import build, cache

torch = pytest.importorskip("torch")

ROOT = Path(__file__).resolve().parent.parent
F32, F16, BF16 = 0, 1, 2
M = 1 << 20


@pytest.fixture(scope="module")
def lib():
    build.build()
    return cache._cache()[0]


def test_exports_match_header(lib):
    text = (ROOT / "include" / "verbo_cache.h").read_text()
    declared = sorted(set(re.findall(r"VERBO_CUDA_API\s+[^;(]*?\b(verbo_cache_\w+)\s*\(", text)))
    out = subprocess.run(["nm", "-D", "--defined-only", str(build.LIB)], capture_output=True, text=True,
                         check=True).stdout
    assert sorted(ln.split()[-1] for ln in out.splitlines() if ln.split()[-1].startswith("verbo_cache_")) == declared
    assert len(declared) == 8


def test_header_compiles_as_c(lib, tmp_path):
    src = tmp_path / "use.c"
    src.write_text('#include "verbo_cache.h"\nint main(void) { verbo_cache c = {1, 8, 2, 64, 16, 2, 4, 0, 0, 0, 0, 0, 0, 0};\n'
                   'return verbo_cache_workspace(&c) > 0 && sizeof c == %d ? 0 : 1; }\n' % ctypes.sizeof(cache._Cache))
    exe = tmp_path / "use"
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", f"-I{ROOT / 'include'}", str(src), f"-L{build.LIB.parent}",
                    "-lverbo_cuda", f"-Wl,-rpath,{build.LIB.parent}", "-o", str(exe)], check=True, capture_output=True)
    assert subprocess.run([str(exe)]).returncode == 0


def made(**kw):
    """A cache of made-up addresses, 1 MB apart: 2 layers, 8 pages, 2 heads of 64, 3 rows of up to 4 pages."""
    a = dict(layers=2, pages=8, heads=2, dim=64, page=16, rows=3, width=4, k=16 * M, v=17 * M, k_scale=18 * M,
             v_scale=19 * M, table=20 * M, lens=21 * M, refs=22 * M)
    a.update(kw)
    return ctypes.byref(cache._Cache(**a))


def refused(lib, rc, msg):
    assert rc == -1
    text = lib.verbo_cuda_last_error().decode()
    assert msg in text, text


BAD_CACHES = [
    (dict(layers=0), "layers"), (dict(layers=65537), "layers"), (dict(pages=0), "pages"),
    (dict(pages=4194305), "pages"), (dict(heads=0), "heads"), (dict(heads=257), "heads"), (dict(dim=0), "dim"),
    (dict(dim=72), "dim"), (dict(dim=144), "dim"), (dict(page=0), "page"), (dict(page=24), "page"),
    (dict(page=272), "page"), (dict(rows=-1), "rows"), (dict(rows=4097), "rows"), (dict(width=0), "width"),
    (dict(width=(1 << 26) + 1), "width"), (dict(rows=4096, width=1 << 20), "rows * width"),
    (dict(pages=4194304, heads=256, page=256), "pages * heads"),
]
BAD_ARRAYS = [
    (dict(k=None), "k must not be NULL"), (dict(v=None), "v must not be NULL"), (dict(k_scale=None), "NULL"),
    (dict(v_scale=None), "NULL"), (dict(table=None), "NULL"), (dict(lens=None), "NULL"), (dict(refs=None), "NULL"),
    (dict(k=16 * M + 8), "k must be aligned"), (dict(v=17 * M + 4), "v must be aligned"),
    (dict(k_scale=18 * M + 2), "aligned"), (dict(table=20 * M + 1), "aligned"), (dict(lens=21 * M + 2), "aligned"),
    (dict(refs=22 * M + 3), "aligned"), (dict(v=16 * M), "v overlaps k"), (dict(v=16 * M + 16), "v overlaps k"),
    (dict(lens=20 * M + 44), "lens overlaps table"), (dict(refs=16 * M), "refs overlaps k"),
]


@pytest.mark.parametrize("kw,msg", BAD_CACHES)
def test_sizes(lib, kw, msg):
    refused(lib, lib.verbo_cache_workspace(made(**kw)), msg)
    refused(lib, lib.verbo_cache_attend_workspace(made(**kw), 2, 1, F16), msg)
    refused(lib, lib.verbo_cache_free(made(**kw), 30 * M, None), msg)


@pytest.mark.parametrize("kw,msg", BAD_ARRAYS)
def test_arrays(lib, kw, msg):
    c = made(**kw)
    refused(lib, lib.verbo_cache_free(c, 30 * M, None), msg)
    refused(lib, lib.verbo_cache_fork(c, 30 * M, 3, 3, None), msg)
    refused(lib, lib.verbo_cache_reserve(c, 30 * M, 31 * M, 32 * M, 33 * M, 1 << 20, None), msg)
    refused(lib, lib.verbo_cache_compact(c, 30 * M, 33 * M, 1 << 20, None), msg)
    refused(lib, append(lib, cache=kw), msg)
    refused(lib, attend(lib, cache=kw), msg)


def test_null_cache(lib):
    refused(lib, lib.verbo_cache_workspace(None), "NULL")
    refused(lib, lib.verbo_cache_free(None, 30 * M, None), "NULL")


def reserve(lib, add=30 * M, start=31 * M, status=32 * M, ws=33 * M, size=1 << 20, **kw):
    return lib.verbo_cache_reserve(made(**kw), add, start, status, ws, size, None)


@pytest.mark.parametrize("kw,msg", [
    (dict(add=None), "add"), (dict(start=None), "start"), (dict(status=None), "status"), (dict(ws=None), "workspace"),
    (dict(size=100), "workspace"), (dict(size=-1), "workspace"), (dict(ws=33 * M + 4), "workspace must be aligned"),
    (dict(add=30 * M + 2), "add must be aligned"), (dict(start=31 * M + 2), "start must be aligned"),
    (dict(status=32 * M + 2), "status must be aligned"), (dict(start=30 * M), "start overlaps add"),
    (dict(status=31 * M + 8), "status overlaps start"), (dict(start=21 * M), "start overlaps lens"),
    (dict(status=22 * M), "status overlaps refs"), (dict(ws=16 * M), "workspace overlaps k"),
    (dict(ws=30 * M), "workspace overlaps add"),
])
def test_reserve(lib, kw, msg):
    refused(lib, reserve(lib, **kw), msg)


@pytest.mark.parametrize("kw,msg", [
    (dict(beams=0), "beams"), (dict(beams=33), "beams"), (dict(beams=2), "multiple of beams"),
    (dict(parents=None), "NULL"), (dict(parents=30 * M + 2), "aligned"), (dict(beams=1, ld=0), "ld_parents"),
    (dict(beams=1, ld=1 << 60), "ld_parents"), (dict(parents=20 * M), "overlaps table"),
])
def test_fork(lib, kw, msg):
    a = {**dict(parents=30 * M, ld=3, beams=3), **kw}
    refused(lib, lib.verbo_cache_fork(made(), a["parents"], a["ld"], a["beams"], None), msg)


def test_free_and_compact(lib):
    refused(lib, lib.verbo_cache_free(made(), None, None), "keep")
    refused(lib, lib.verbo_cache_free(made(), 30 * M + 1, None), "aligned")
    refused(lib, lib.verbo_cache_free(made(), 21 * M, None), "overlaps lens")
    refused(lib, lib.verbo_cache_compact(made(), None, 33 * M, 1 << 20, None), "info")
    refused(lib, lib.verbo_cache_compact(made(), 30 * M + 2, 33 * M, 1 << 20, None), "aligned")
    refused(lib, lib.verbo_cache_compact(made(), 22 * M, 33 * M, 1 << 20, None), "overlaps refs")
    refused(lib, lib.verbo_cache_compact(made(), 30 * M, 33 * M, 64, None), "workspace")
    refused(lib, lib.verbo_cache_compact(made(), 30 * M, 30 * M, 1 << 20, None), "overlaps info")


def append(lib, cache=(), **kw):
    a = dict(layer=1, k=40 * M, ldk=128, hdk=64, v=41 * M, ldv=128, hdv=64, dtype=F16, tokens=6, start=42 * M, off=None)
    a.update(kw)
    return lib.verbo_cache_append(made(**dict(cache)), a["layer"], a["k"], a["ldk"], a["hdk"], a["v"], a["ldv"],
                                  a["hdv"], a["dtype"], a["tokens"], a["start"], a["off"], None)


@pytest.mark.parametrize("kw,msg", [
    (dict(layer=-1), "layer"), (dict(layer=2), "layer"), (dict(dtype=3), "dtype"), (dict(tokens=-1), "tokens"),
    (dict(tokens=4), "multiple of rows"), (dict(k=None), "new k"), (dict(v=None), "new v"),
    (dict(start=None), "start"), (dict(start=42 * M + 2), "start must be aligned"),
    (dict(off=43 * M + 4), "off must be aligned"), (dict(k=40 * M + 1), "new k must be aligned"),
    (dict(ldk=63), "token stride"), (dict(hdv=63), "head stride"), (dict(ldk=-128), "stride"),
    (dict(ldk=1 << 60), "too large"), (dict(hdk=1 << 60), "too large"), (dict(k=16 * M), "new k overlaps k"),
    (dict(v=20 * M), "new v overlaps table"), (dict(start=22 * M), "start overlaps refs"),
    (dict(off=21 * M), "off overlaps lens"),
])
def test_append(lib, kw, msg):
    refused(lib, append(lib, **kw), msg)


LONG = dict(width=40000)  # few rows of a short table need no workspace


def attend(lib, cache=(), **kw):
    a = dict(layer=0, q=40 * M, q_type=BF16, ldq=256, hdq=64, heads=4, steps=2, scale=0.1, out=41 * M, o_type=F32,
             ldo=256, hdo=64, ws=64 * M, size=1 << 30)
    a.update(kw)
    return lib.verbo_cache_attend(made(**dict(cache)), a["layer"], a["q"], a["q_type"], a["ldq"], a["hdq"], a["heads"],
                                  a["steps"], a["scale"], a["out"], a["o_type"], a["ldo"], a["hdo"], a["ws"],
                                  a["size"], None)


@pytest.mark.parametrize("kw,msg", [
    (dict(layer=2), "layer"), (dict(q_type=5), "q_type"), (dict(o_type=-1), "out_type"), (dict(steps=0), "steps"),
    (dict(steps=33), "steps"), (dict(heads=3), "heads"), (dict(heads=0), "heads"), (dict(heads=130), "heads"),
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(q=None), "q must not be NULL"),
    (dict(out=None), "out must not be NULL"), (dict(q=40 * M + 1), "q must be aligned"),
    (dict(out=41 * M + 2), "out must be aligned"), (dict(ldq=60), "token stride"), (dict(hdq=32), "head stride"),
    (dict(ldo=128), "tokens and heads overlap"), (dict(out=40 * M), "out overlaps q"),
    (dict(out=18 * M), "out overlaps k_scale"), (dict(ws=None, cache=LONG), "workspace"),
    (dict(size=1000, cache=LONG), "workspace"), (dict(ws=64 * M + 8, cache=LONG), "workspace must be aligned"),
    (dict(ws=41 * M, cache=LONG), "workspace overlaps"),
])
def test_attend(lib, kw, msg):
    refused(lib, attend(lib, **kw), msg)


def test_nothing(lib):
    none = dict(rows=0)
    assert lib.verbo_cache_free(made(**none), None, None) == 0
    assert lib.verbo_cache_fork(made(**none), None, 1, 1, None) == 0
    assert append(lib, cache=none, tokens=0, start=None) == 0
    assert append(lib, tokens=0, k=None, v=None, start=None) == 0
    assert attend(lib, cache=none, q=None, out=None, ws=None) == 0
    refused(lib, append(lib, cache=none, tokens=4), "multiple of rows")
    empty = dict(rows=0, table=None, lens=None)
    assert lib.verbo_cache_free(made(**empty), None, None) == 0


@pytest.mark.parametrize("how", [copy.copy, copy.deepcopy, pickle.dumps], ids=["copy", "deepcopy", "pickle"])
def test_a_cache_is_not_copied(how):
    """Nor can its tensors be exchanged: the library has their addresses."""
    c = object.__new__(vb.PagedCache)
    c._held = {"lens": torch.zeros(2)}
    with pytest.raises(TypeError, match="PagedCache"):
        how(c)
    with pytest.raises(AttributeError):
        c.lens = torch.zeros(3)
    c.lens += 1
    assert c.lens.tolist() == [1, 1]


def test_python_refusals():
    e4m3 = torch.float8_e4m3fn
    t = dict(k=torch.zeros(1, 4, 2, 16, 64).to(e4m3), v=torch.zeros(1, 4, 2, 16, 64).to(e4m3),
             k_scale=torch.ones(1, 4, 2, 1), v_scale=torch.ones(1, 4, 2, 1),
             table=torch.zeros(2, 3, dtype=torch.int32), lens=torch.zeros(2, dtype=torch.int32),
             refs=torch.zeros(4, dtype=torch.int32))
    with pytest.raises(vb.VerboCudaError, match="CUDA"):
        vb.PagedCache(**t)
    with pytest.raises(vb.VerboCudaError, match="layers, pages"):
        vb.PagedCache(**{**t, "k": t["k"][0]})
    with pytest.raises(vb.VerboCudaError, match="rows, width"):
        vb.PagedCache(**{**t, "table": t["lens"]})
    for kw in (dict(pages=2**32 + 1), dict(rows=-1), dict(width=2**31), dict(page=24)):
        with pytest.raises(vb.VerboCudaError):
            vb.PagedCache.new(**{**dict(layers=1, pages=4, heads=1, dim=64, rows=1, width=2, device="cuda:0"), **kw})
