"""A step whose tokens the cache does not hold ends the search: PagedCache.reserve answers with a
status in device memory, and BeamSearch reads those of its model's calls.  On the CPU with made-up
answers, and on the GPU with a table and a pool that are too small."""
from __future__ import annotations

import ctypes

import pytest

torch = pytest.importorskip("torch")

import verbo_b200 as vb  # noqa: E402
from verbo_b200 import cache as cache_module  # noqa: E402
from verbo_b200.serving import BeamSearch  # noqa: E402


class Lib:
    verbo_cache_reserve, verbo_cache_fork = "reserve", "fork"


@pytest.fixture
def cache(monkeypatch):
    """A cache of four rows whose reserves answer what c.answers holds."""
    monkeypatch.setattr(cache_module, "_new", lambda torch, like, stream, shape, dtype: torch.empty(shape, dtype=dtype))
    monkeypatch.setattr(cache_module, "_stream_of", lambda torch, dev, stream: 0)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    c = object.__new__(vb.PagedCache)
    c._torch, c._lib, c._dev, c.rows, c._need = torch, Lib, -1, 4, 64
    c._held = {"lens": torch.zeros(4, dtype=torch.int32)}
    c._ws = torch.empty(64, dtype=torch.uint8)
    c.answers, c.forked = [], 0

    def run(fn, *args):
        if fn == "reserve":
            ctypes.cast(args[2], ctypes.POINTER(ctypes.c_int))[0] = c.answers.pop(0)
        else:
            c.forked += 1

    c._run = run
    return c


def search(monkeypatch, cache, reserves=1):
    def model(tokens, out):
        out.copy_(torch.arange(7.0).expand_as(out))
        for _ in range(reserves):
            cache.reserve(torch.ones(4, dtype=torch.int32))

    def select(logits, scores, beams, take):
        n = logits.shape[0] // beams
        return (-torch.arange(take).float().expand(n, take), torch.zeros(n, take, dtype=torch.int32),
                torch.arange(take).int().expand(n, take))

    monkeypatch.setattr(vb, "beam_select", select)
    s = object.__new__(BeamSearch)
    s.torch, s.model, s.device, s.cache = torch, model, torch.device("cpu"), cache
    s.requests, s.beams, s.vocab, s.max_tokens = 2, 2, 7, 9
    s.stop_ids, s.length_penalty, s.states, s.steps, s.tokens = frozenset(), 1.0, [], 0, None
    s.logits, s.scores = torch.zeros(4, 7), torch.zeros(2, 2)
    s.beam_tokens, s.done, s.open = [[[], []], [[], []]], [[], []], [True, True]
    return s


@pytest.mark.parametrize("answers,msg", [([3], "3 pages"), ([-2], "row 1"), ([0, 5], "5 pages"), ([7, 0], "7 pages")])
def test_a_refused_reserve_ends_the_search(monkeypatch, cache, answers, msg):
    cache.answers = list(answers)
    s = search(monkeypatch, cache, len(answers))
    with pytest.raises(vb.VerboCudaError, match=msg):
        s.step()
    assert s.steps == 0 and cache.forked == 0


def test_others_do_not(monkeypatch, cache):
    cache.answers = [0, 0, 4]
    s = search(monkeypatch, cache)
    assert s.step() and s.step() and cache.forked == 2
    cache.reserve(torch.ones(4, dtype=torch.int32))  # not the search's
    cache.answers = [0]
    assert s.step() and cache.forked == 3


def test_a_model_that_answers_itself(monkeypatch, cache):
    cache.answers = [2, 0]
    s = search(monkeypatch, cache)
    model = s.model

    def tries(tokens, out):
        with cache.statuses() as said:
            model(tokens, out)
            if int(said[0]):
                cache.reserve(torch.ones(4, dtype=torch.int32))

    s.model = tries
    assert s.step() and cache.answers == [] and cache.forked == 1


def test_captured_reserves_are_left_out(monkeypatch, cache):
    """Their statuses are written by the replays."""
    cache.answers = [3]
    with cache.statuses() as said:
        monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
        cache.reserve(torch.ones(4, dtype=torch.int32))
    assert said == []


def test_statuses(cache):
    cache.answers = [0, 6, 1]
    one = torch.ones(4, dtype=torch.int32)
    cache.reserve(one)
    with cache.statuses() as said:
        _, status = cache.reserve(one)
        assert [t.tolist() for t in said] == [[6]] and said[0] is status
    cache.reserve(one)
    assert len(said) == 1


@pytest.mark.gpu
@pytest.mark.parametrize("pages,width,msg", [(40, 2, "row 0"), (9, 40, "pages")])
def test_on_the_gpu(cuda_lib, pages, width, msg):
    """Four rows of two requests: 30 tokens of a prompt each, then a token a step."""
    c = vb.PagedCache.new(1, pages, 2, 64, 4, width, 16)
    kv = torch.randn(120, 2, 64, device="cuda")
    one = torch.ones(4, dtype=torch.int32, device="cuda")

    def model(tokens, out):
        out.copy_(torch.arange(50.0, device="cuda").expand_as(out))
        n = 30 if tokens is None else 1
        start, _ = c.reserve(one * n)
        c.append(0, kv[:4 * n], kv[:4 * n], start)

    s = BeamSearch(model, 2, 2, 50, 30, cache=c)
    with pytest.raises(vb.VerboCudaError, match=msg):
        s.run()
    # three pages of two rows each: the table ends at 32 tokens, the pool with a copy of a shared page
    assert s.steps == 3 if width == 2 else s.steps >= 1
    vb.check()
