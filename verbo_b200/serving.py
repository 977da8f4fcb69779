"""Request batching for a server, over the library's verbo_cuda_server_*, and beam
search over a batch of requests, over verbo_beam_* (``BeamSearch``, at the end).

The reference's server (cli/serve.cpp:139-218) runs one request at a time
behind a global mutex (:168), each through verbo::generate
(src/sampler.cpp:111-181) with the request's own Sampling (:149-157): accept
the prompt, then pick / stop check / accept until a stop id or max_tokens.
``BatchServer`` keeps up to ``slots`` requests in flight in one
``verbo_b200.Server`` instead: a request takes a free row (its Sampler seeded
with its seed, its prompt accepted), every step samples all rows from the
logits rows the caller's model produced, one launch chain per option set, and
a request leaves when it meets a stop id (not emitted, as in generate) or its
token limit, letting the next queued request in.  Only the ids cross to the
host each step; the scheduling itself is the C ABI's, so a C++ server can drive
the same object (verbo_cuda_server_prepare / _step / _result).
"""
from __future__ import annotations

import contextlib
from dataclasses import dataclass, field
from typing import Callable, Dict, List, Optional, Sequence


@dataclass
class Request:
    prompt: List[int]
    max_tokens: int
    seed: int
    opts: object = None
    rid: int = -1
    tokens: List[int] = field(default_factory=list)
    stopped: bool = False  # ended on a stop id (else on max_tokens)


class BatchServer:
    """Continuous batching of generation requests on one GPU.

    ``model(row_requests, out)`` fills ``out`` (CUDA float32 [slots, vocab])
    with the next logits row of each row's request (``None`` for an idle row,
    whose row may hold anything finite).  ``opts`` is the default Sampling; a
    request may bring its own.  ``stop_ids`` is the model's stop set."""

    def __init__(self, opts, slots: int, vocab: int, model: Callable, device: int = 0, stop_ids: Sequence[int] = (),
                 max_window: int = 256):
        import torch

        import verbo_b200 as vb

        self.opts, self.vocab, self.slots, self.model = opts, vocab, slots, model
        self.server = vb.Server(slots, vocab, max_window=max_window, stop_ids=stop_ids, device=device)
        self.logits = torch.zeros((slots, vocab), dtype=torch.float32, device=f"cuda:{device}")
        self.reqs: Dict[int, Request] = {}
        self.done: Dict[int, Request] = {}

    def submit(self, prompt: Sequence[int], max_tokens: int, seed: int, opts=None) -> int:
        import dataclasses

        if seed == 0:
            raise ValueError("seed 0 means the clock in the reference; give each request its own seed")
        o = dataclasses.replace(opts if opts is not None else self.opts, seed=int(seed))
        rid = self.server.submit(list(prompt), o, int(max_tokens))
        r = Request(list(prompt), int(max_tokens), int(seed), o, rid=rid)
        if r.max_tokens <= 0:
            self.server.result(rid, release=True)
            self.done[rid] = r
        else:
            self.reqs[rid] = r
        return rid

    def step(self) -> bool:
        """One sampling step over the active rows; False when nothing is left."""
        rows, n = self.server.prepare()
        if n == 0:
            return False
        active: List[Optional[Request]] = [self.reqs[int(rid)] if rid >= 0 else None for rid in rows]
        self.model(active, self.logits)
        self.server.step(self.logits)
        for r in active[:n]:
            finished, ids, stopped = self.server.result(r.rid, release=True)
            r.tokens = ids
            if finished:
                r.stopped = stopped
                self.done[r.rid] = self.reqs.pop(r.rid)
        return True

    def run(self) -> Dict[int, Request]:
        while self.step():
            pass
        return self.done


@dataclass
class Hypothesis:
    tokens: List[int]
    score: float  # the summed log-probability, the stop token's with it
    value: float  # what hypotheses are ordered by: score / tokens ** length_penalty
    stopped: bool  # ended on a stop id (else at the token limit)


class BeamSearch:
    """Beam search of ``requests`` requests with ``beams`` beams each on one GPU.

    ``model(tokens, out)`` fills ``out`` (CUDA float32 [requests * beams, vocab], row
    r * beams + b is beam b of request r) with each row's next logits.  ``tokens`` is
    None in the first step, in which all rows of a request hold its prompt, and after
    that int32 [requests * beams], the token that each row has got.

    A step takes the best continuations of each request (``beam_select``): those that
    end on a stop id among the first ``beams`` of them are finished hypotheses, the
    first ``beams`` of the others live on.  With n stop ids (1 + n) * beams are taken,
    enough for both, or 64: where those do not hold ``beams`` that live on, every beam's own
    first 64 are.  What the rows carry follows them:
    ``cache`` (a ``PagedCache`` with a row per beam) forks, ``states`` (tensors with a
    row per beam) are reordered in place.  A request ends when it has ``beams``
    finished hypotheses and no live one can be better than the worst of them, or after
    ``max_tokens`` tokens.  Only continuations cross to the host, and the statuses of the
    ``cache.reserve`` calls of the model (not of a graph that it replays): one that was
    refused raises ``VerboCudaError``, unless the model collects it itself
    (``cache.statuses``)."""

    def __init__(self, model: Callable, requests: int, beams: int, vocab: int, max_tokens: int,
                 stop_ids: Sequence[int] = (), length_penalty: float = 1.0, cache=None, states: Sequence = (),
                 device: int = 0):
        import torch

        if requests < 1 or max_tokens < 1:
            raise ValueError("requests and max_tokens must be at least 1")
        if not 1 <= beams <= 32:
            raise ValueError("beams must be in [1, 32]")
        if cache is not None and cache.rows != requests * beams:
            raise ValueError("the cache must have a row per beam")
        self.torch, self.model = torch, model
        self.requests, self.beams, self.vocab, self.max_tokens = requests, beams, vocab, max_tokens
        self.stop_ids, self.length_penalty = frozenset(int(i) for i in stop_ids), float(length_penalty)
        self.cache, self.states = cache, list(states)
        self.device = torch.device("cuda", device)
        self.logits = torch.zeros((requests * beams, vocab), dtype=torch.float32, device=self.device)
        self.steps = 0
        self.beam_tokens: List[List[List[int]]] = [[[] for _ in range(beams)] for _ in range(requests)]
        self.done: List[List[Hypothesis]] = [[] for _ in range(requests)]
        self.open = [True] * requests
        first = [0.0] + [float("-inf")] * (beams - 1)
        self.scores = torch.tensor([first] * requests, dtype=torch.float32, device=self.device)
        self.tokens = None

    def _value(self, score: float, tokens: int) -> float:
        return score / max(1, tokens) ** self.length_penalty

    def _advance(self, scores, parents, tokens):
        """The host's part of a step, from its continuations ([requests][2 * beams] lists):
        the live beams' (scores, parents, tokens)."""
        beams, n = self.beams, self.steps + 1
        out_s, out_p, out_t = [], [], []
        for r in range(self.requests):
            live_s, live_p, live_t, kept = [], [], [], []
            if self.open[r]:
                for i, (s, p, t) in enumerate(zip(scores[r], parents[r], tokens[r])):
                    if p < 0 or len(live_s) == beams:
                        break
                    if t in self.stop_ids:
                        if i < beams:
                            self.done[r].append(Hypothesis(self.beam_tokens[r][p], s, self._value(s, n), True))
                        continue
                    live_s.append(s)
                    live_p.append(p)
                    live_t.append(t)
                    kept.append(self.beam_tokens[r][p] + [t])
                if n == self.max_tokens:
                    self.done[r] += [Hypothesis(k, s, self._value(s, n), False) for k, s in zip(kept, live_s)]
                self.done[r] = sorted(self.done[r], key=lambda h: -h.value)[:beams]
                # what the best beam can still reach: its score only falls, its length may grow to the limit
                best = live_s[0] if live_s else float("-inf")
                reach = self._value(best, self.max_tokens if self.length_penalty > 0 else n)
                full = len(self.done[r]) == beams and self.done[r][-1].value >= reach
                if n == self.max_tokens or not live_s or full:
                    self.open[r] = False
            if not self.open[r]:
                live_s, live_p, live_t, kept = [], [], [], []
            # beams without a continuation stay where they are, with no score
            spare = beams - len(live_s)
            self.beam_tokens[r] = kept + [[]] * spare
            out_s.append(live_s + [float("-inf")] * spare)
            out_p.append(live_p + [-1] * spare)
            out_t.append(live_t + [0] * spare)
        self.steps = n
        return out_s, out_p, out_t

    def _short(self, parents, tokens) -> bool:
        """Whether an open request's continuations are fewer that live on than beams, and not all there are."""
        return any(is_open and p[-1] >= 0 and sum(i not in self.stop_ids for i in t) < self.beams
                   for is_open, p, t in zip(self.open, parents, tokens))

    def _find(self):
        """The step's continuations of each request: (scores, parents, tokens) as lists."""
        import verbo_b200 as vb

        most, beams = 64, self.beams  # beam_select's limit
        ends = sum(0 <= i < self.vocab for i in self.stop_ids)
        take = min(most, max(2, 1 + ends) * beams)
        found = [f.tolist() for f in vb.beam_select(self.logits, self.scores, beams, take)]
        if take == max(2, 1 + ends) * beams or not self._short(*found[1:]):
            return found
        # a beam at a time: no more than `beams` of one live on.  These scores are rounded to fp32, equal ones
        # go by the beam.
        scores, parents, tokens = (f.tolist() for f in vb.beam_select(self.logits, self.scores, 1, most))
        found = [], [], []
        for r in range(self.requests):
            rows = range(r * beams, (r + 1) * beams)
            best = sorted(((s, b, t) for b, i in enumerate(rows) for s, p, t in zip(scores[i], parents[i], tokens[i])
                           if p >= 0), key=lambda c: -c[0])
            live = [s for s, _, t in best if t not in self.stop_ids]
            worst = live[beams - 1] if len(live) >= beams else float("-inf")
            if any(parents[i][-1] >= 0 and scores[i][-1] > worst for i in rows):
                raise vb.VerboCudaError(f"too many stop ids among the first {most} continuations of a beam")
            for out, column in zip(found, ([c[k] for c in best] for k in range(3))):
                out.append(column)
        return found

    def step(self) -> bool:
        """One token for every open request; False when none is left."""
        import verbo_b200 as vb

        if not any(self.open):
            return False
        torch = self.torch
        with getattr(self.cache, "statuses", contextlib.nullcontext)() as said:
            self.model(self.tokens, self.logits)
        found = self._find()
        for status in torch.cat(said).tolist() if said else ():
            if status:
                raise vb.VerboCudaError("the cache does not hold the step's tokens: " + (
                    f"{status} pages are missing" if status > 0 else f"row {-status - 1} would be longer than its table"))
        live = self._advance(*found)
        self.scores = torch.tensor(live[0], dtype=torch.float32, device=self.device)
        parents = torch.tensor(live[1], dtype=torch.int32, device=self.device)
        self.tokens = torch.tensor(live[2], dtype=torch.int32, device=self.device).view(-1)
        if self.cache is not None:
            self.cache.fork(parents, self.beams)
        if self.states:
            vb.beam_reorder(self.states, parents, self.beams)
        return any(self.open)

    def run(self) -> List[List[Hypothesis]]:
        """The requests' finished hypotheses, the best first."""
        while self.step():
            pass
        return self.done
