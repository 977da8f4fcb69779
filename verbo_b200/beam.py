"""Beam search beside the sampler (include/verbo_beam.h), for CUDA tensors.

``beam_select``   the best continuations of each request's beams
``beam_reorder``  the beams' states in the order of the chosen parents, in place

They are the library's kernels and nothing else: no fallback.  Arguments are
checked here and in the C ABI; both raise ``VerboCudaError``.
"""
from __future__ import annotations

import ctypes

from . import VerboCudaError, _err
from .ops import _call, _INT_MAX, _list, _new, _ops, _rows, _stream_of

__all__ = ["beam_select", "beam_reorder"]

_P = ctypes.c_void_p
_I = ctypes.c_int
_L = ctypes.c_longlong
MAX_BEAMS, MAX_TAKE = 32, 64


class _State(ctypes.Structure):
    _fields_ = [("data", _P), ("row_bytes", _L), ("stride_bytes", _L)]


_ready = None
_needs = {}  # workspace bytes by (requests, beams, take)


def _beam():
    """(library, torch, type codes); the signatures are set at the first use."""
    global _ready
    if _ready is None:
        lib, torch, types = _ops()
        for name, res, args in (
            ("verbo_beam_select", _I, [_P, _I, _I, _I, _I, _L, _P, _I, _P, _P, _P, _P, _L, _P]),
            ("verbo_beam_workspace", _L, [_I, _I, _I]),
            ("verbo_beam_reorder", _I, [ctypes.POINTER(_State), _I, _I, _I, _P, _L, _P]),
        ):
            fn = getattr(lib, name)
            fn.restype, fn.argtypes = res, args
        _ready = lib, torch, types
    return _ready


def _whole(v, low, high, what):
    v = int(v)
    if not low <= v <= high:
        raise VerboCudaError(f"{what} must be in [{low}, {high}]")
    return v


def _parents(parents, torch, requests, beams, dev):
    """(address, row stride) of int32 parents [requests, >= beams]."""
    if parents.dim() != 2 or parents.shape[0] != requests or parents.shape[1] < beams:
        raise VerboCudaError("parents must be [requests, at least beams]")
    if parents.get_device() != dev or parents.dtype != torch.int32:
        raise VerboCudaError("parents must be an int32 CUDA tensor on the device of the rows")
    ld, step = parents.stride()
    if step != 1 and parents.shape[1] > 1:
        raise VerboCudaError("parents: rows must be contiguous (stride(1) == 1)")
    return parents.data_ptr(), (ld if requests > 1 else max(beams, 1))


def beam_select(logits, scores, beams, take, vocab=None, stream=None):
    """The ``take`` best continuations of each request (verbo_beam_select):
    (scores, parents, tokens), each [requests, take].

    logits: CUDA rows [requests * beams, >= vocab] in float32, float16 or bfloat16,
    rows contiguous, any row stride; row r * beams + b is beam b of request r.
    scores: float32 with one value per row, the beams' summed log-probabilities;
    -inf for a beam without continuations (all but one of a request's beams in its
    first step).  beams <= 32, take <= 64.

    A continuation's score is the beam's plus the token's log-probability; they come
    in descending order, of equal ones the lower beam's first, then the larger
    logit's, then the lower token's.  Where there are fewer: -inf, -1, -1."""
    lib, torch, types = _beam()
    beams, take = _whole(beams, 1, MAX_BEAMS, "beams"), _whole(take, 1, MAX_TAKE, "take")
    rows, cols, ld, code, dev = _rows(logits, types, "logits")
    if rows % beams:
        raise VerboCudaError("logits must have beams rows per request")
    if vocab is None:
        vocab = cols
    elif not 0 < vocab <= cols:
        raise VerboCudaError("vocab must be in [1, columns of logits]")
    requests = rows // beams
    sp = _list(scores, torch.float32, dev, "scores", rows)
    at = _stream_of(torch, dev, stream)
    need = _needs.get((requests, beams, take))
    if need is None:
        need = lib.verbo_beam_workspace(requests, beams, take)
        if need < 0:
            raise _err()
        _needs[requests, beams, take] = need
    out = _new(torch, logits, stream, requests, take, torch.float32)
    parents = _new(torch, logits, stream, requests, take, torch.int32)
    tokens = _new(torch, logits, stream, requests, take, torch.int32)
    # the workspace belongs to the call's stream: freed here, it is reused behind the call
    ws = _new(torch, logits, stream, need, None, torch.uint8)
    _call(lib.verbo_beam_select, torch, dev, logits.data_ptr(), code, requests, beams, vocab, ld, sp, take,
          out.data_ptr(), parents.data_ptr(), tokens.data_ptr(), ws.data_ptr(), need, at)
    return out, parents, tokens


def beam_reorder(states, parents, beams, stream=None):
    """Puts the rows of one state or of a list of states in the order of their
    parents, in place (verbo_beam_reorder).

    states: CUDA tensors [requests * beams, ...] of any type, each row contiguous,
    any row stride, on one device and not overlapping.  parents: int32 [requests, >= beams] (what
    ``beam_select`` returns, or its first columns): row b of a request becomes what
    row parents[request, b] of that request was; a parent outside [0, beams) leaves
    its row as it was."""
    lib, torch, _ = _beam()
    beams = _whole(beams, 1, MAX_BEAMS, "beams")
    if isinstance(states, torch.Tensor):
        states = [states]
    if not states:
        return
    dev = states[0].get_device()
    rows = states[0].shape[0] if states[0].dim() else -1
    if rows < 0 or rows % beams or rows > _INT_MAX:
        raise VerboCudaError("a state must have beams rows per request")
    pp, ldp = _parents(parents, torch, rows // beams, beams, dev)
    items = (_State * len(states))()
    for item, t in zip(items, states):
        if t.get_device() != dev or dev < 0:
            raise VerboCudaError("states must be CUDA tensors on one device")
        if t.dim() == 0 or t.shape[0] != rows:
            raise VerboCudaError("states must have the same number of rows")
        if t.numel() == 0:
            continue
        inner = t.numel() // rows
        span = 1
        for n, step in zip(reversed(t.shape[1:]), reversed(t.stride()[1:])):
            if n > 1 and step != span:
                raise VerboCudaError("a state's rows must be contiguous")
            span *= n
        size = t.element_size()
        item.data, item.row_bytes = t.data_ptr(), inner * size
        item.stride_bytes = (t.stride(0) if rows > 1 else inner) * size
    _call(lib.verbo_beam_reorder, torch, dev, items, len(states), rows // beams, beams, pp, ldp,
          _stream_of(torch, dev, stream))
