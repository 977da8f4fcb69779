"""CPU tests of BeamSearch's host part (verbo_b200/serving.py): which continuations
end a hypothesis, which live on, and when a request is over."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from verbo_b200.serving import BeamSearch  # noqa: E402

INF = float("inf")


def search(requests=1, beams=2, max_tokens=5, stop_ids=(9,), length_penalty=1.0):
    """A search whose device part is not used."""
    s = object.__new__(BeamSearch)
    s.requests, s.beams, s.max_tokens = requests, beams, max_tokens
    s.stop_ids, s.length_penalty = frozenset(stop_ids), length_penalty
    s.steps = 0
    s.beam_tokens = [[[] for _ in range(beams)] for _ in range(requests)]
    s.done = [[] for _ in range(requests)]
    s.open = [True] * requests
    return s


def test_live_beams_are_the_first_without_a_stop():
    s = search()
    out = s._advance([[-1.0, -2.0, -3.0, -4.0]], [[0, 0, 0, 0]], [[5, 9, 6, 7]])
    assert out == ([[-1.0, -3.0]], [[0, 0]], [[5, 6]])
    assert s.beam_tokens == [[[5], [6]]] and s.open == [True]
    assert [(h.tokens, h.score, h.stopped) for h in s.done[0]] == [([], -2.0, True)]
    out = s._advance([[-1.5, -3.5, -4.0, -5.0]], [[1, 0, 1, 0]], [[1, 2, 3, 4]])
    assert out[1] == [[1, 0]] and s.beam_tokens == [[[6, 1], [5, 2]]]


def test_a_late_stop_does_not_count():
    """A stop behind the first `beams` continuations is dropped."""
    s = search()
    s._advance([[-1.0, -2.0, -3.0, -4.0]], [[0, 0, 0, 0]], [[5, 6, 9, 9]])
    assert s.done == [[]]


def test_token_limit():
    s = search(max_tokens=1)
    out = s._advance([[-1.0, -2.0, -3.0, -4.0]], [[0, 0, 0, 0]], [[5, 9, 6, 7]])
    assert s.open == [False]
    assert [(h.tokens, h.stopped) for h in s.done[0]] == [([5], False), ([], True)]
    assert out == ([[-INF, -INF]], [[-1, -1]], [[0, 0]])


def test_over_when_nothing_better_can_come():
    s = search(length_penalty=0.0, max_tokens=50)
    s._advance([[-1.0, -1.5, -3.0, -4.0]], [[0, 0, 0, 0]], [[9, 9, 6, 7]])
    assert s.open == [False] and [h.value for h in s.done[0]] == [-1.0, -1.5]
    s = search(length_penalty=1.0, max_tokens=50)  # long hypotheses may still be better
    s._advance([[-1.0, -1.5, -3.0, -4.0]], [[0, 0, 0, 0]], [[9, 9, 6, 7]])
    assert s.open == [True]


def test_fewer_continuations_than_beams():
    s = search(beams=3)
    out = s._advance([[-1.0] + [-INF] * 5], [[0] + [-1] * 5], [[4] + [-1] * 5])
    assert out == ([[-1.0, -INF, -INF]], [[0, -1, -1]], [[4, 0, 0]]) and s.open == [True]
    s = search(beams=2)
    out = s._advance([[-INF] * 4], [[-1] * 4], [[-1] * 4])
    assert s.open == [False] and out[1] == [[-1, -1]]


def test_requests_are_apart():
    s = search(requests=2, max_tokens=2)
    s._advance([[-1.0, -2.0, -INF, -INF], [-INF] * 4], [[0, 0, -1, -1], [-1] * 4], [[1, 2, -1, -1], [-1] * 4])
    assert s.open == [True, False]
    s._advance([[-1.0, -2.0, -3.0, -4.0]] * 2, [[0, 1, 0, 1]] * 2, [[1, 2, 3, 4]] * 2)
    assert [h.tokens for h in s.done[0]] == [[1, 1], [2, 2]] and s.done[1] == []


def test_refusals():
    for kw in (dict(requests=0), dict(beams=0), dict(beams=33), dict(max_tokens=0)):
        with pytest.raises(ValueError):
            BeamSearch(None, **{**dict(requests=1, beams=2, vocab=8, max_tokens=4), **kw})
