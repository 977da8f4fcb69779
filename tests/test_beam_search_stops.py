"""BeamSearch with several stop ids against a search in 64 bits that looks at every
continuation: on the CPU with beam_select's definition in plain torch in its place,
and on the GPU with the kernels."""
from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import verbo_b200 as vb  # noqa: E402
from verbo_b200.serving import BeamSearch  # noqa: E402

INF = float("inf")


def plain_select(logits, scores, beams, take, vocab=None, stream=None):
    """beam_select's definition, on the CPU."""
    assert 1 <= beams <= 32 and 1 <= take <= 64
    n, v = logits.shape[0] // beams, logits.shape[1]
    value = (torch.log_softmax(logits.double(), 1) + scores.double().view(-1, 1)).view(n, beams * v)
    top, at = torch.sort(value, dim=1, descending=True, stable=True)
    top, at = top[:, :take], at[:, :take]
    missing = max(0, take - top.shape[1])
    top = torch.nn.functional.pad(top, (0, missing), value=-INF)
    at = torch.nn.functional.pad(at, (0, missing))
    none = top == -INF
    return top.float(), torch.where(none, -1, at // v).int(), torch.where(none, -1, at % v).int()


def reference(logp, first, beams, steps, stops):
    live, done = [(0.0, [], first)], []
    for _ in range(steps):
        cand = sorted(((s + logp[last][v], t + [v], v) for s, t, last in live for v in range(logp.shape[1])),
                      key=lambda c: -c[0])
        done += [(s, t[:-1], len(t)) for s, t, v in cand[:beams] if v in stops]
        live = [c for c in cand if c[2] not in stops][:beams]
    done += [(s, t, len(t)) for s, t, _ in live]
    return sorted(done, key=lambda d: -d[0] / d[2])[:beams]


def made_up(model, requests, beams, vocab, steps, stops):
    """A search on the CPU."""
    s = object.__new__(BeamSearch)
    s.torch, s.model, s.device = torch, model, torch.device("cpu")
    s.requests, s.beams, s.vocab, s.max_tokens = requests, beams, vocab, steps
    s.stop_ids, s.length_penalty = frozenset(stops), 1.0
    s.cache, s.states, s.steps, s.tokens = None, [], 0, None
    s.logits = torch.zeros(requests * beams, vocab)
    s.beam_tokens = [[[] for _ in range(beams)] for _ in range(requests)]
    s.done, s.open = [[] for _ in range(requests)], [True] * requests
    s.scores = torch.tensor([[0.0] + [-INF] * (beams - 1)] * requests)
    return s


def run(beams, vocab, stops, seed, device, more):
    g = np.random.default_rng(seed)
    w = g.standard_normal((vocab, vocab)).astype(np.float32) * 2
    w[:, sorted(i for i in stops if 0 <= i < vocab)] += more  # the stop ids are likely
    logp = w.astype(np.float64)
    logp = logp - np.log(np.exp(logp).sum(1, keepdims=True))
    first = [int(i) for i in g.integers(0, vocab, 4)]
    rows = torch.tensor(first, device=device).repeat_interleave(beams)
    table = torch.from_numpy(w).to(device)

    def model(tokens, out):
        out.copy_(table[rows if tokens is None else tokens.long()])

    if device == "cpu":
        s = made_up(model, 4, beams, vocab, 5, stops)
    else:
        s = BeamSearch(model, 4, beams, vocab, 5, stop_ids=sorted(stops))
    got = s.run()
    for r in range(4):
        want = reference(logp, first[r], beams, 5, stops)
        assert [h.tokens for h in got[r]] == [t for _, t, _ in want]
        assert np.allclose([h.score for h in got[r]], [sc for sc, _, _ in want], rtol=0, atol=1e-4)


CASES = [(3, 23, {0, 1}), (3, 23, {5, 6, 7, 22}), (1, 9, {0, 1, 2, 3}), (5, 40, {1, 2, -7, 400}), (8, 30, set(range(9))),
         (20, 60, {3, 4, 5}), (32, 60, {0, 59}), (32, 50, set(range(10)))]


@pytest.mark.parametrize("more", [0.0, 4.0])
@pytest.mark.parametrize("beams,vocab,stops", CASES)
def test_several_stop_ids(monkeypatch, beams, vocab, stops, more):
    monkeypatch.setattr(vb, "beam_select", plain_select)
    run(beams, vocab, stops, beams, "cpu", more)


def test_a_step_that_cannot_be_told(monkeypatch):
    """More stop ids than a beam's list holds, all of them before the others."""
    monkeypatch.setattr(vb, "beam_select", plain_select)

    def model(tokens, out):
        out.zero_()
        out[:, :70] = 5.0

    with pytest.raises(vb.VerboCudaError, match="stop ids"):
        made_up(model, 1, 4, 200, 5, range(70)).step()
    s = made_up(model, 2, 4, 200, 5, range(70))  # the first request is over
    s.open[0], s.scores[0] = False, -INF
    with pytest.raises(vb.VerboCudaError, match="stop ids"):
        s.step()
    s = made_up(lambda tokens, out: out.copy_(torch.arange(200.0).expand_as(out)), 1, 4, 200, 5, range(70))
    assert s.step() and s.beam_tokens == [[[199], [198], [197], [196]]]


@pytest.mark.gpu
@pytest.mark.parametrize("more", [0.0, 4.0])
@pytest.mark.parametrize("beams,vocab,stops", CASES)
def test_on_the_gpu(cuda_lib, beams, vocab, stops, more):
    run(beams, vocab, stops, 100 + beams, "cuda", more)
    vb.check()
