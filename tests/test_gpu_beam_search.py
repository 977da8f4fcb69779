"""GPU tests of beam search's operators together, as a decoder uses them: the search
itself against one in 64 bits, and a small decoder (4-bit layers, the paged 8-bit
cache, its attention, selection, forks) against the same decoder whose beams own
their pages and are copied."""
from __future__ import annotations

import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import verbo_b200 as vb  # noqa: E402
from verbo_b200.serving import BeamSearch  # noqa: E402


ROOT = Path(__file__).resolve().parent.parent


@pytest.fixture(autouse=True)
def _needs(cuda_lib):
    if not torch.cuda.is_available():
        pytest.fail("gpu tests need a CUDA device")


def reference(table, first, beams, steps, stop):
    """Beam search in 64 bits over a table of next-token log-probabilities: finished and live (score, tokens)."""
    live, done = [(0.0, [], first)], []
    for n in range(steps):
        cand = sorted(((s + table[last][v], t + [v], v) for s, t, last in live for v in range(table.shape[1])),
                      key=lambda c: -c[0])[:2 * beams]
        done += [(s, t[:-1], len(t)) for i, (s, t, v) in enumerate(cand) if v == stop and i < beams]
        live = [c for c in cand if c[2] != stop][:beams]
    done += [(s, t, len(t)) for s, t, _ in live]
    return sorted(done, key=lambda d: -d[0] / d[2])[:beams]


def test_first_calls_are_captured(cuda_lib):
    r = subprocess.run([sys.executable, str(ROOT / "tests" / "beam_capture_calls.py")], capture_output=True, text=True,
                       timeout=300, cwd=ROOT)
    assert r.returncode == 0 and r.stdout.strip().endswith("same"), r.stderr[-2000:]


@pytest.mark.parametrize("beams", [1, 2, 5])
def test_the_search(beams):
    g = np.random.default_rng(beams)
    V, requests, steps, stop = 23, 4, 6, 7
    w = g.standard_normal((V, V)).astype(np.float32) * 2
    logp = w.astype(np.float64)
    logp = logp - np.log(np.exp(logp).sum(1, keepdims=True))
    first = [3, 11, 0, 22]
    rows = torch.tensor(first, device="cuda").repeat_interleave(beams)
    table = torch.from_numpy(w).cuda()
    seen = torch.zeros(requests * beams, 2, dtype=torch.int32, device="cuda")  # a state: step and last token

    def model(tokens, out):
        last = rows if tokens is None else tokens.long()
        if tokens is not None:
            seen[:, 0] += 1
            seen[:, 1] = tokens
        out.copy_(table[last])

    s = BeamSearch(model, requests, beams, V, steps, stop_ids=[stop], states=[seen])
    got = s.run()
    vb.check()
    for r in range(requests):
        want = reference(logp, first[r], beams, steps, stop)
        assert [h.tokens for h in got[r]] == [t for _, t, _ in want]
        assert np.allclose([h.score for h in got[r]], [sc for sc, _, _ in want], rtol=0, atol=1e-4)
        assert np.allclose([h.value for h in got[r]], [sc / n for sc, _, n in want], rtol=0, atol=1e-4)


class Decoder:
    """One attention layer and a head, on the library's operators."""

    V, D, H, KV, DIM = 97, 64, 4, 2, 32

    def __init__(self, seed):
        g = torch.Generator().manual_seed(seed)

        def layer(outs, ins):
            q = torch.randint(0, 256, (outs, ins // 2), generator=g, dtype=torch.uint8)
            return vb.Q4Linear(q, torch.full((outs, ins // 32), 0.03, dtype=torch.float16))

        self.embed = (torch.randn(self.V, self.D, generator=g)).cuda()
        self.qkv = layer((self.H + 2 * self.KV) * self.DIM, self.D)
        self.out, self.head = layer(self.D, self.H * self.DIM), layer(self.V, self.D)

    def __call__(self, tokens, cache, add, out):
        """The rows' next tokens through the decoder; tokens [rows * steps]."""
        x = self.embed[tokens.long()]
        rows, steps = cache.rows, tokens.numel() // cache.rows
        qkv = self.qkv.matvec(x).view(-1, self.H + 2 * self.KV, self.DIM)
        q, k, v = qkv.split([self.H, self.KV, self.KV], 1)
        start, self.status = cache.reserve(add)
        cache.append(0, k, v, start)
        y = cache.attend(0, q)
        x = x + self.out.matvec(y.view(rows * steps, -1))
        self.head.matvec(x.view(rows, steps, -1)[:, -1].contiguous(), out=out)


class Owned(vb.PagedCache):
    """The same cache without sharing: a fork copies every page."""

    def fork(self, parents, beams, stream=None):
        rows = torch.arange(self.rows, device="cuda").view(-1, beams)
        src = (rows[:, :1] + parents.clamp(min=0)).view(-1)
        for pool in (self.k, self.v, self.k_scale, self.v_scale):
            bits = pool.view(torch.uint8) if pool.dtype == torch.float8_e4m3fn else pool
            table = self.own.view(self.rows, -1)
            bits[:, table.view(-1)] = bits[:, table[src].view(-1)]
        live = (parents.view(-1) >= 0).int()
        self.lens.copy_(self.lens[src] * live)
        used = (self.lens + self.page - 1) // self.page
        inside = torch.arange(self.width, device="cuda") < used[:, None]
        self.table.copy_(torch.where(inside, self.own.view(self.rows, -1).int(), -1))
        self.refs.zero_()
        self.refs[self.table[self.table >= 0].long()] = 1

    def reserve(self, add, stream=None):
        start = self.lens.clone()
        self.lens += add
        used = (self.lens + self.page - 1) // self.page
        inside = torch.arange(self.width, device="cuda") < used[:, None]
        self.table.copy_(torch.where(inside, self.own.view(self.rows, -1).int(), -1))
        return start, torch.zeros(1, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("beams,prompt", [(4, 30), (3, 16), (5, 5)])
def test_a_decoder(beams, prompt):
    requests, steps, page = 3, 40, 16
    rows, width = requests * beams, (prompt + steps) // page + 2
    g = torch.Generator().manual_seed(beams)
    ids = torch.randint(0, Decoder.V, (requests, prompt), generator=g).cuda()
    found, lowest = [], []
    for owned in (False, True):
        net = Decoder(1)
        cache = (Owned if owned else vb.PagedCache).new(1, rows * width, Decoder.KV, Decoder.DIM, rows, width, page)
        cache.own = torch.arange(rows * width, device="cuda")
        one = torch.ones(rows, dtype=torch.int32, device="cuda")
        free = []

        def model(tokens, out):
            if tokens is None:  # the prompt through a request's first row, which the others fork from
                alone = torch.zeros(rows, dtype=torch.int32, device="cuda")
                alone[::beams] = prompt - 1
                start, _ = cache.reserve(alone if not owned else one * (prompt - 1))
                x = net.embed[ids[:, :-1].reshape(-1)]
                kv = net.qkv.matvec(x).view(requests, prompt - 1, -1, Decoder.DIM)[:, :, Decoder.H:]
                kv = kv.repeat_interleave(beams, 0).flatten(0, 1)
                off = torch.arange(rows + 1, device="cuda") * (prompt - 1)
                cache.append(0, kv[:, :Decoder.KV], kv[:, Decoder.KV:], start, off=off)
                if not owned:
                    cache.fork(torch.zeros(requests, beams, dtype=torch.int32, device="cuda"), beams)
                tokens = ids[:, -1].repeat_interleave(beams)
            net(tokens, cache, one, out)
            assert net.status.tolist() == [0] or owned
            free.append(int((cache.refs == 0).sum()))

        s = BeamSearch(model, requests, beams, Decoder.V, steps, stop_ids=[0], cache=cache)
        found.append(s.run())
        lowest.append(min(free))
        vb.check()
        counted = torch.bincount(cache.table[cache.table >= 0].long(), minlength=cache.pages)
        assert torch.equal(cache.refs.long(), counted)
    a, b = found  # the same tokens read: the same scores, bit for bit
    for x, y in zip(a, b):
        assert [(h.tokens, h.score, h.stopped) for h in x] == [(h.tokens, h.score, h.stopped) for h in y]
    assert all(x for x in a)
    assert lowest[0] > lowest[1]  # pages are shared
