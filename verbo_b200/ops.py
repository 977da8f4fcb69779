"""Operators around the sampler (include/verbo_ops.h), for CUDA tensors.

``process_logits``   penalties for repeated tokens, biases and masks, before the pick
``token_logprobs``   log-probability and rank of a token, and the most likely tokens
``Q4Linear``         products with 4-bit weights and group scales

They are the library's kernels and nothing else: no fallback.  Arguments are
checked here and in the C ABI; both raise ``VerboCudaError``.
"""
from __future__ import annotations

import ctypes

from . import VerboCudaError, _err, load_library

__all__ = ["Penalties", "process_logits", "token_logprobs", "Q4Linear"]

_P = ctypes.c_void_p
_I = ctypes.c_int
_L = ctypes.c_longlong
_INT_MAX = 2**31 - 1  # what ctypes takes for an int it cuts to 32 bits, without an error
_MAX_TOP = 32


class Penalties(ctypes.Structure):
    """Penalties on the ids of a row's history: ``repeat`` is that of ``Sampling``
    (v > 0 ? v / repeat : v * repeat), then ``frequency`` times the number of
    occurrences and ``presence`` once are subtracted.  ``last`` is the window:
    the last ``last`` ids, all of them if <= 0.  (verbo_ops_penalties itself.)"""

    _fields_ = [("repeat", ctypes.c_float), ("frequency", ctypes.c_float), ("presence", ctypes.c_float),
                ("last", ctypes.c_int)]

    def __init__(self, repeat: float = 1.0, frequency: float = 0.0, presence: float = 0.0, last: int = 0):
        if not -_INT_MAX - 1 <= last <= _INT_MAX:
            raise VerboCudaError("last must be in [-2147483648, 2147483647]")
        super().__init__(repeat, frequency, presence, last)

    def __repr__(self):
        return f"Penalties(repeat={self.repeat}, frequency={self.frequency}, presence={self.presence}, last={self.last})"


_state = None


def _ops():
    """(library, torch, type codes); the signatures are set at the first use."""
    global _state
    if _state is None:
        import torch

        lib = load_library()
        for name, res, args in (
            ("verbo_ops_default_penalties", Penalties, []),
            ("verbo_ops_process_logits", _I, [_P, _I, _I, _I, _L, ctypes.POINTER(Penalties), _P, _P, _P, _P, _P, _P, _P,
                                              _L, _P, _L, _P]),
            ("verbo_ops_token_logprobs", _I, [_P, _I, _I, _I, _L, ctypes.c_float, _P, _P, _P, _I, _P, _P, _P]),
            ("verbo_ops_q4_new", _P, [_I, _I, _I, _P, _P, _P, _P, _I, _P]),
            ("verbo_ops_q4_free", None, [_P]),
            ("verbo_ops_q4_workspace", _L, [_P, _I, _I]),
            ("verbo_ops_q4_matvec", _I, [_P, _P, _I, _I, _L, _P, _I, _L, _P, _L, _P]),
        ):
            fn = getattr(lib, name)
            fn.restype, fn.argtypes = res, args
        _state = lib, torch, {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
    return _state


def _rows(t, types, what):
    """(rows, columns, row stride, type code, device index) of a CUDA matrix with
    contiguous rows."""
    if t.dim() != 2:
        raise VerboCudaError(f"{what} must have two dimensions")
    rows, cols = t.shape
    if rows > _INT_MAX or cols > _INT_MAX:
        raise VerboCudaError(f"{what} must have at most {_INT_MAX} rows and columns")
    index = t.get_device()
    if index < 0:
        raise VerboCudaError(f"{what} must be a CUDA tensor")
    code = types.get(t.dtype)
    if code is None:
        raise VerboCudaError(f"{what} must be float32, float16 or bfloat16")
    ld, step = t.stride()
    if step != 1 and cols > 1:
        raise VerboCudaError(f"{what}: rows must be contiguous (stride(1) == 1)")
    return rows, cols, (ld if rows > 1 else max(cols, 1)), code, index


def _list(t, dtype, index, what, size=None):
    """Device address of a contiguous CUDA tensor of one type on a device, or None."""
    if t is None:
        return None
    if t.get_device() != index:
        raise VerboCudaError(f"{what} must be a CUDA tensor on the device of the rows")
    if t.dtype != dtype:
        raise VerboCudaError(f"{what} must be {str(dtype)[6:]}")
    if not t.is_contiguous():
        raise VerboCudaError(f"{what} must be contiguous")
    if size is not None and t.numel() != size:
        raise VerboCudaError(f"{what} must have {size} elements")
    return t.data_ptr()


def _call(fn, torch, index, *args):
    """One library call with the device current (the calls on rows take the
    current device's)."""
    if torch.cuda.current_device() == index:
        rc = fn(*args)
    else:
        with torch.cuda.device(index):
            rc = fn(*args)
    if rc < 0:
        raise _err()


def _stream_of(torch, index, stream):
    """The address of the call's stream (the device's current one if None)."""
    if stream is None:
        return torch._C._cuda_getCurrentRawStream(index)
    at = getattr(stream, "device", None)
    if at is not None and at.index != index:
        raise VerboCudaError("stream must be one of the rows' device")
    return getattr(stream, "cuda_stream", stream)


def _new(torch, like, stream, rows, cols, dtype):
    """A new matrix (or vector: cols None) that belongs to the call's stream."""
    if stream is not None:
        if not isinstance(stream, torch.cuda.Stream):
            stream = torch.cuda.ExternalStream(stream, device=like.device)
        with torch.cuda.stream(stream):
            return _new(torch, like, None, rows, cols, dtype)
    if cols is None:
        return torch.empty(rows, dtype=dtype, device=like.device)
    return torch.empty(rows, cols, dtype=dtype, device=like.device)


def process_logits(logits, penalties=None, hist=None, hist_off=None, row_penalties=None, bias_ids=None, bias=None,
                   bias_off=None, mask=None, out=None, vocab=None, stream=None):
    """What a request does to its logits before the pick: penalties for repeated
    tokens, then biases, then a mask (verbo_ops_process_logits).

    logits: CUDA rows [rows, >= vocab] in float32, float16 or bfloat16, rows
    contiguous, any row stride.  penalties: ``Penalties``, on each row's
    history hist/hist_off (int32 ids, int64 CSR offsets [rows + 1], as for
    ``sample``); row_penalties: float32 [rows, 3], each row's own repeat,
    frequency and presence in their place (``penalties`` then gives the window
    alone).  bias_ids/bias/bias_off: int32 ids, float32 values and int64 CSR
    offsets; of an id listed twice in a row the last value counts.  mask: int32
    words [rows or 1, >= ceil(vocab / 32)], bit i % 32 of word i // 32 set where
    id i is allowed; one row of words is shared by all.

    Returns float32 rows [rows, vocab]: new ones, or ``out``, which may be
    ``logits`` itself (float32): then only the columns that change are touched.
    Pass them to ``sample`` or ``Batch.step`` with repeat = 1."""
    lib, torch, types = _ops()
    rows, cols, ld, code, dev = _rows(logits, types, "logits")
    if vocab is None:
        vocab = cols
    elif not 0 < vocab <= cols:
        raise VerboCudaError("vocab must be in [1, columns of logits]")
    at = _stream_of(torch, dev, stream)
    if out is None:
        out = _new(torch, logits, stream, rows, vocab, torch.float32)
        ld_out = vocab
    elif out is logits and code == 0:
        ld_out = ld
    else:
        orows, ocols, ld_out, ocode, odev = _rows(out, types, "out")
        if ocode != 0 or orows != rows or ocols < vocab or odev != dev:
            raise VerboCudaError("out must be float32 with one row per row of logits, on their device")
    mp, ld_mask = None, 0
    if mask is not None:
        shape = mask.shape
        if len(shape) != 2 or (shape[0] != rows and shape[0] != 1) or shape[1] * 32 < vocab:
            raise VerboCudaError("mask must be [rows or 1, at least ceil(vocab / 32)]")
        if mask.get_device() != dev or mask.dtype != torch.int32:
            raise VerboCudaError("mask must be an int32 CUDA tensor on the device of the rows")
        stride = mask.stride()
        if stride[1] != 1 and shape[1] > 1:
            raise VerboCudaError("mask: rows must be contiguous (stride(1) == 1)")
        mp = mask.data_ptr()
        if shape[0] > 1:
            ld_mask = stride[0]
    hp = op = rp = bi = bv = bo = pen = None
    if hist is not None or hist_off is not None:
        if hist is None or hist_off is None:
            raise VerboCudaError("hist and hist_off must both be given or both be None")
        hp = _list(hist, torch.int32, dev, "hist")
        op = _list(hist_off, torch.int64, dev, "hist_off", rows + 1)
        if hist.numel() == 0:
            hp = op = None
    if bias is not None or bias_ids is not None or bias_off is not None:
        if bias is None or bias_ids is None or bias_off is None:
            raise VerboCudaError("bias_ids, bias and bias_off must all be given or all be None")
        bv = _list(bias, torch.float32, dev, "bias")
        bi = _list(bias_ids, torch.int32, dev, "bias_ids", bias.numel())
        bo = _list(bias_off, torch.int64, dev, "bias_off", rows + 1)
        if bias.numel() == 0:
            bi = bv = bo = None
    if penalties is not None:
        if not isinstance(penalties, Penalties):
            raise VerboCudaError("penalties must be Penalties")
        pen = penalties
    if row_penalties is not None:
        rp = _list(row_penalties, torch.float32, dev, "row_penalties", 3 * rows)
        if row_penalties.dim() != 2 or row_penalties.shape[0] != rows:
            raise VerboCudaError("row_penalties must be [rows, 3]")
        if pen is None:
            pen = Penalties(1.0, 0.0, 0.0, 0)
    _call(lib.verbo_ops_process_logits, torch, dev, logits.data_ptr(), code, rows, vocab, ld,
          None if pen is None else ctypes.byref(pen), rp, hp, op, bi, bv, bo, mp, ld_mask, out.data_ptr(), ld_out, at)
    return out


def token_logprobs(logits, ids=None, top=0, temp=1.0, vocab=None, stream=None):
    """Log-probabilities of softmax(logits / temp) over each row's first ``vocab``
    columns (verbo_ops_token_logprobs): (logprob, rank, top_ids, top_logprobs).

    logits: CUDA rows as for ``process_logits``.  ids: int32 [rows], one token a
    row; logprob float32 [rows] is its log-probability and rank int32 [rows]
    the number of columns before it in the sampler's order (value descending,
    id ascending); both None without ids; -inf and -1 for an id outside
    [0, vocab).  top_ids int32 and top_logprobs float32 [rows, top]: the first
    ``top`` <= 32 columns of that order, (-1, -inf) where fewer are above
    -inf.  A NaN counts as -inf."""
    lib, torch, types = _ops()
    top = int(top)
    if not 0 <= top <= _MAX_TOP:
        raise VerboCudaError(f"top must be in [0, {_MAX_TOP}]")
    rows, cols, ld, code, dev = _rows(logits, types, "logits")
    if vocab is None:
        vocab = cols
    elif not 0 < vocab <= cols:
        raise VerboCudaError("vocab must be in [1, columns of logits]")
    at = _stream_of(torch, dev, stream)
    f32, i32 = torch.float32, torch.int32
    tid, tlp = _new(torch, logits, stream, rows, top, i32), _new(torch, logits, stream, rows, top, f32)
    if ids is None:
        lp = rank = ip = lpp = rp = None
    else:
        ip = _list(ids, i32, dev, "ids", rows)
        lp, rank = _new(torch, logits, stream, rows, None, f32), _new(torch, logits, stream, rows, None, i32)
        lpp, rp = lp.data_ptr(), rank.data_ptr()
    _call(lib.verbo_ops_token_logprobs, torch, dev, logits.data_ptr(), code, rows, vocab, ld, temp, ip, lpp, rp, top,
          tid.data_ptr(), tlp.data_ptr(), at)
    return lp, rank, tid, tlp


class Q4Linear:
    """A weight matrix of 4-bit integers with group scales on the device
    (verbo_ops_q4_*), for products with a few rows.

    q: uint8 [outs, ins / 2], the reference's Q4 rows (byte j of a block of 32
    holds element j in its low half, element j + 16 in its high half); s: float16
    [outs, ceil(ins / group)]; zeros: uint8 [outs, ceil(ins / group)] with values
    0..15, or None for 8 everywhere; bias: float32 [outs] or None.  Each a numpy
    array or a tensor of any device; they are read before the constructor
    returns.  W[o, i] = s[o, i // group] * (q[o, i] - zeros[o, i // group]).

    Keep a layer as long as the CUDA graphs that were captured with it.  It cannot
    be copied or pickled: its weights belong to one object."""

    def __init__(self, q, s, zeros=None, bias=None, group: int = 32, device=None):
        lib, torch, self._types = _ops()
        self._lib, self._torch = lib, torch
        self._h = None
        self._need = {}  # workspace bytes by (rows, type)

        def hold(v, dtype, what):
            t = torch.as_tensor(v)
            if t.dtype != dtype:
                raise VerboCudaError(f"{what} must be {str(dtype)[6:]}")
            return t.contiguous()

        q = hold(q, torch.uint8, "q")
        if q.dim() != 2:
            raise VerboCudaError("q must have two dimensions")
        if device is None:
            device = q.device.index if q.is_cuda else torch.cuda.current_device()
        device = torch.device("cuda", device) if isinstance(device, int) else torch.device(device)
        self.device = torch.device("cuda", torch.cuda.current_device() if device.index is None else device.index)
        self.outs, self.ins, self.group = q.shape[0], 2 * q.shape[1], int(group)
        if not 1 <= self.group <= _INT_MAX:
            raise VerboCudaError("group must be a multiple of 32 in [32, 2^31)")
        if max(self.outs, self.ins) > _INT_MAX:
            raise VerboCudaError(f"q must have at most {_INT_MAX} rows and weights of a row")
        cells = (self.outs, -(-self.ins // self.group))
        s = hold(s, torch.float16, "s")
        zeros = None if zeros is None else hold(zeros, torch.uint8, "zeros")
        bias = None if bias is None else hold(bias, torch.float32, "bias")
        if tuple(s.shape) != cells or (zeros is not None and tuple(zeros.shape) != cells):
            raise VerboCudaError("s and zeros must be [outs, ceil(ins / group)]")
        if bias is not None and tuple(bias.shape) != (self.outs,):
            raise VerboCudaError("bias must be [outs]")
        given = [t for t in (q, s, zeros, bias) if t is not None]
        for d in {t.device for t in given if t.is_cuda and t.device != self.device}:
            torch.cuda.current_stream(d).synchronize()
        h = lib.verbo_ops_q4_new(self.outs, self.ins, self.group, q.data_ptr(), s.data_ptr(),
                                 None if zeros is None else zeros.data_ptr(), None if bias is None else bias.data_ptr(),
                                 self.device.index, torch.cuda.current_stream(self.device).cuda_stream
                                 if torch.cuda.is_available() else None)
        if not h:
            raise _err()
        self._h = h

    def __reduce_ex__(self, protocol):
        raise TypeError("a Q4Linear cannot be copied or pickled")

    def close(self):
        if getattr(self, "_h", None):
            self._lib.verbo_ops_q4_free(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def matvec(self, x, out=None, dtype=None, stream=None):
        """x W^T + bias for CUDA rows x [n, ins] (float32, float16 or bfloat16, rows
        contiguous, any row stride) -> rows [n, outs] of ``dtype`` (x's if None), or
        into ``out``.  Sums are fp32 whatever the types."""
        torch = self._torch
        if self._h is None:
            raise VerboCudaError("the layer is closed")
        n, cols, ldx, xt, dev = _rows(x, self._types, "x")
        if cols != self.ins or dev != self.device.index:
            raise VerboCudaError(f"x must be [n, {self.ins}] on {self.device}")
        at = _stream_of(torch, dev, stream)
        if out is None:
            if dtype is None:
                dtype = x.dtype
            yt = self._types.get(dtype)
            if yt is None:
                raise VerboCudaError("dtype must be float32, float16 or bfloat16")
            out = _new(torch, x, stream, n, self.outs, dtype)
            ldy = self.outs
        else:
            rows, ocols, ldy, yt, odev = _rows(out, self._types, "out")
            if rows != n or ocols != self.outs or odev != dev or (dtype is not None and dtype != out.dtype):
                raise VerboCudaError(f"out must be [n, {self.outs}] on {self.device}")
        need = self._need.get((n, xt))
        if need is None:
            need = self._lib.verbo_ops_q4_workspace(self._h, xt, n)
            if need < 0:
                raise _err()
            self._need[n, xt] = need
        # the workspace belongs to the call's stream: freed here, it is reused behind the call
        ws = _new(torch, x, stream, need, None, torch.uint8) if need else None
        if self._lib.verbo_ops_q4_matvec(self._h, x.data_ptr(), xt, n, ldx, out.data_ptr(), yt, ldy,
                                         ws.data_ptr() if need else None, need, at) < 0:
            raise _err()
        return out
