"""CPU tests of the memory that PagedCache.reserve and compact work in (no kernel
launches): it has to belong to the stream of the call, for the allocator gives a
dropped cache's memory to the stream that it was made on without waiting for others."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

import verbo_b200 as vb  # noqa: E402
from verbo_b200 import cache  # noqa: E402


class Lib:
    verbo_cache_reserve, verbo_cache_compact = "reserve", "compact"


@pytest.fixture
def calls(monkeypatch):
    """(stream, tensor) of what is allocated, and the arguments of the library's calls."""
    made, ran = [], []

    def new(torch, like, stream, shape, dtype):
        made.append((stream, torch.empty(shape, dtype=dtype)))
        return made[-1][1]

    monkeypatch.setattr(cache, "_new", new)
    monkeypatch.setattr(cache, "_stream_of", lambda torch, dev, stream: stream or 0)
    c = object.__new__(vb.PagedCache)
    c._torch, c._lib, c._dev, c.rows, c._need = torch, Lib, -1, 2, 64
    c._held = {"lens": torch.zeros(2, dtype=torch.int32)}
    c._ws = torch.empty(64, dtype=torch.uint8)
    c._run = lambda fn, *args: ran.append((fn, *args))
    return c, made, ran


def workspace_of(call):
    return call[4] if call[0] == "reserve" else call[2]


@pytest.mark.parametrize("what", ["reserve", "compact"])
def test_a_call_on_another_stream_has_its_own(calls, what):
    c, made, ran = calls
    for stream in (7, 9):
        c.reserve(torch.ones(2, dtype=torch.int32), stream=stream) if what == "reserve" else c.compact(stream=stream)
        own = [t for s, t in made if s == stream and t.dtype == torch.uint8 and t.numel() >= 64]
        assert ran[-1][0] == what and ran[-1][-1] == stream
        assert workspace_of(ran[-1]) in [t.data_ptr() for t in own]


@pytest.mark.parametrize("what", ["reserve", "compact"])
def test_a_cache_made_on_another_stream_keeps_none(calls, what):
    c, made, ran = calls
    c._ws = None
    c.reserve(torch.ones(2, dtype=torch.int32)) if what == "reserve" else c.compact()
    assert workspace_of(ran[-1]) in [t.data_ptr() for _, t in made if t.dtype == torch.uint8]
