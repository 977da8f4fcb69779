"""The paged cache of keys and values in 8 bits (include/verbo_cache.h), on CUDA
tensors: what the rows of a decode step, or the beams of a search, keep of their
tokens, and the attention that reads it.

The compute is the library's kernels and nothing else: no fallback.  Arguments
are checked here and in the C ABI; both raise ``VerboCudaError``.
"""
from __future__ import annotations

import contextlib
import ctypes
import math

from . import VerboCudaError, _err
from .beam import _parents
from .ops import _call, _INT_MAX, _list, _ops, _stream_of

__all__ = ["PagedCache"]

_P = ctypes.c_void_p
_I = ctypes.c_int
_L = ctypes.c_longlong
BLOCK = 16  # tokens that share a scale


class _Cache(ctypes.Structure):
    _fields_ = [("layers", _I), ("pages", _I), ("heads", _I), ("dim", _I), ("page", _I), ("rows", _I), ("width", _I),
                ("k", _P), ("v", _P), ("k_scale", _P), ("v_scale", _P), ("table", _P), ("lens", _P), ("refs", _P)]


_ready = None


def _cache():
    """(library, torch, type codes); the signatures are set at the first use."""
    global _ready
    if _ready is None:
        lib, torch, types = _ops()
        c = ctypes.POINTER(_Cache)
        for name, res, args in (
            ("verbo_cache_workspace", _L, [c]),
            ("verbo_cache_reserve", _I, [c, _P, _P, _P, _P, _L, _P]),
            ("verbo_cache_fork", _I, [c, _P, _L, _I, _P]),
            ("verbo_cache_free", _I, [c, _P, _P]),
            ("verbo_cache_compact", _I, [c, _P, _P, _L, _P]),
            ("verbo_cache_append", _I, [c, _I, _P, _L, _L, _P, _L, _L, _I, _I, _P, _P, _P]),
            ("verbo_cache_attend", _I, [c, _I, _P, _I, _L, _L, _I, _I, ctypes.c_float, _P, _I, _L, _L, _P, _L, _P]),
            ("verbo_cache_attend_workspace", _L, [c, _I, _I, _I]),
        ):
            fn = getattr(lib, name)
            fn.restype, fn.argtypes = res, args
        _ready = lib, torch, types
    return _ready


def _new(torch, like, stream, shape, dtype):
    """A new tensor that belongs to the call's stream."""
    if stream is not None:
        if not isinstance(stream, torch.cuda.Stream):
            stream = torch.cuda.ExternalStream(stream, device=like.device)
        with torch.cuda.stream(stream):
            return torch.empty(shape, dtype=dtype, device=like.device)
    return torch.empty(shape, dtype=dtype, device=like.device)


def _tensor(name):
    """A tensor of the cache: changed in place (``cache.lens += 1`` too), not exchanged."""

    def get(self):
        return self._held[name]

    def put(self, t):
        if t is not self._held[name]:
            raise AttributeError(f"the cache's {name} cannot be another tensor")

    return property(get, put)


class PagedCache:
    """Keys and values of ``rows`` rows in pages that they may share.

    k, v: float8_e4m3fn [layers, pages, heads, page, dim]; k_scale, v_scale: float32
    [layers, pages, heads, page / 16], one scale for 16 tokens of a head; table: int32
    [rows, width], the rows' pages, -1 behind the last; lens: int32 [rows], their
    tokens; refs: int32 [pages], how many entries of the table hold a page (0: free).
    All contiguous CUDA tensors on one device, the caller's own: the object keeps
    them, and, where it is made on the default stream, a workspace of about 12 bytes a page for
    the calls there.  ``new`` makes an empty cache.

    A decode step: ``reserve`` makes room for the rows' new tokens, then per layer
    ``append`` writes their keys and values and ``attend`` reads them.  A step of
    beam search ends with ``fork``.  Nothing waits for the device; what a call has to
    say (``status``, ``info``) it writes into a tensor.  Calls on one cache have to follow
    one another (one stream, or streams that wait for one another), but for ``append`` and
    ``attend`` of different layers."""

    def __init__(self, k, v, k_scale, v_scale, table, lens, refs):
        self._lib, self._torch, self._types = lib, torch, _ = _cache()
        if k.dim() != 5:
            raise VerboCudaError("k must be [layers, pages, heads, page, dim]")
        layers, pages, heads, page, dim = k.shape
        if table.dim() != 2:
            raise VerboCudaError("table must be [rows, width]")
        rows, width = table.shape
        if max(*k.shape, rows, width) > _INT_MAX:
            raise VerboCudaError(f"sizes must be at most {_INT_MAX}")
        if page % BLOCK:
            raise VerboCudaError("page must be a multiple of 16")
        dev = k.get_device()
        if dev < 0:
            raise VerboCudaError("the cache must be CUDA tensors")
        codes, f32, i32 = torch.float8_e4m3fn, torch.float32, torch.int32
        blocks = (layers, pages, heads, page // BLOCK)
        c = self._c = _Cache(layers, pages, heads, dim, page, rows, width)
        self._held = {}  # the library has their addresses: other tensors are another cache
        for name, t, dtype, shape in (("k", k, codes, k.shape), ("v", v, codes, k.shape),
                                      ("k_scale", k_scale, f32, blocks), ("v_scale", v_scale, f32, blocks),
                                      ("table", table, i32, table.shape), ("lens", lens, i32, (rows,)),
                                      ("refs", refs, i32, (pages,))):
            if tuple(t.shape) != tuple(shape):
                raise VerboCudaError(f"{name} must be {list(shape)}")
            setattr(c, name, _list(t, dtype, dev, name))
            self._held[name] = t
        self.layers, self.pages, self.heads, self.page, self.dim = layers, pages, heads, page, dim
        self.rows, self.width = rows, width
        self.device = k.device
        self._dev, self._ref = dev, ctypes.byref(c)
        self._need = lib.verbo_cache_workspace(ctypes.byref(c))
        if self._need < 0:
            raise _err()
        # reserve's and compact's on the default stream (0): what is made there and used there alone may be
        # dropped at any time, and no graph holds its address, for that stream cannot be captured
        self._ws = None
        if torch._C._cuda_getCurrentRawStream(dev) == 0:
            self._ws = torch.empty(self._need, dtype=torch.uint8, device=k.device)
        self._attend_need = {}  # workspace bytes by (heads, steps, type)

    @classmethod
    def new(cls, layers, pages, heads, dim, rows, width, page=64, device=None):
        """An empty cache on a CUDA device (the current one if None)."""
        torch = _cache()[1]
        for name, n in (("layers", layers), ("pages", pages), ("heads", heads), ("dim", dim), ("rows", rows),
                        ("width", width), ("page", page)):
            if not 0 <= n <= _INT_MAX:
                raise VerboCudaError(f"{name} must be in [0, {_INT_MAX}]")
        device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        if page % BLOCK:
            raise VerboCudaError("page must be a multiple of 16")

        def make(shape, dtype, value):
            return torch.full(shape, value, dtype=dtype, device=device)

        def pool():
            return make((layers, pages, heads, page, dim), torch.uint8, 0).view(torch.float8_e4m3fn)

        def scales():
            return make((layers, pages, heads, page // BLOCK), torch.float32, 1.0)

        i32 = torch.int32
        return cls(pool(), pool(), scales(), scales(), make((rows, width), i32, -1), make((rows,), i32, 0),
                   make((pages,), i32, 0))

    def __reduce_ex__(self, protocol):
        raise TypeError("a PagedCache cannot be copied or pickled")

    _said = None  # what `statuses` collects

    @contextlib.contextmanager
    def statuses(self):
        """A list of the statuses (device tensors) of the reserves that are called inside, but for captured ones, which
        a replay writes.  Of two collections, one inside the other, the inner one has what is called in it."""
        before, self._said = self._said, []
        try:
            yield self._said
        finally:
            self._said = before

    k, v, k_scale, v_scale = _tensor("k"), _tensor("v"), _tensor("k_scale"), _tensor("v_scale")
    table, lens, refs = _tensor("table"), _tensor("lens"), _tensor("refs")

    def _run(self, fn, *args):
        _call(fn, self._torch, self._dev, self._ref, *args)

    def _workspace(self, stream, at):
        """Memory for a reserve or a compact on a stream: the kept one, or one that belongs to the call's stream
        (freed behind the call, it is reused behind the call's work)."""
        if at == 0 and self._ws is not None:
            return self._ws
        return _new(self._torch, self.lens, stream, self._need, self._torch.uint8)

    def _ints(self, t, what):
        """Address of int32 [rows] on the cache's device."""
        return _list(t, self._torch.int32, self._dev, what, self.rows)

    def reserve(self, add, stream=None):
        """Room for ``add`` more tokens of each row (int32 [rows]; 0: none): pages, the
        lowest free ones first, and a copy of a row's last page where other rows hold
        it too (verbo_cache_reserve).  lens grows by add.

        Returns (start, status): int32 [rows], where the new tokens begin (-1: none),
        and int32 [1], 0, or the number of pages that were missing, or -(r + 1) for a
        row r that the table is too narrow for.  Unless status is 0 nothing was changed
        and every start is -1, for which ``append`` writes nothing."""
        torch = self._torch
        at = _stream_of(torch, self._dev, stream)
        ap = self._ints(add, "add")
        start = _new(torch, self.lens, stream, self.rows, torch.int32)
        status = _new(torch, self.lens, stream, 1, torch.int32)
        ws = self._workspace(stream, at)
        self._run(self._lib.verbo_cache_reserve, ap, start.data_ptr(), status.data_ptr(), ws.data_ptr(), self._need, at)
        if self._said is not None and not torch.cuda.is_current_stream_capturing():
            self._said.append(status)
        return start, status

    def fork(self, parents, beams, stream=None):
        """Rows take over their parents' pages, and share them (verbo_cache_fork):
        row b of a group of ``beams`` rows becomes what row parents[group, b] of it was.
        parents: int32 [rows / beams, >= beams], as ``beam_select`` returns them; a
        parent outside [0, beams) empties the row."""
        torch = self._torch
        beams = int(beams)
        if not 1 <= beams <= 32 or self.rows % beams:
            raise VerboCudaError("beams must be in [1, 32] and divide the rows")
        pp, ld = _parents(parents, torch, self.rows // beams, beams, self._dev)
        self._run(self._lib.verbo_cache_fork, pp, ld, beams, _stream_of(torch, self._dev, stream))

    def free(self, keep, stream=None):
        """Row r keeps its first keep[r] tokens (int32 [rows]; negative: all), and gives
        the pages behind them back (verbo_cache_free).  Kept tokens stay rounded to the scale
        of their block, also where a token that is not kept has raised it."""
        self._run(self._lib.verbo_cache_free, self._ints(keep, "keep"),
                  _stream_of(self._torch, self._dev, stream))

    def compact(self, stream=None):
        """Moves the live pages to the front of the pool, in all layers
        (verbo_cache_compact).  Returns int32 [2]: live pages, pages that moved."""
        torch = self._torch
        at = _stream_of(torch, self._dev, stream)
        info = _new(torch, self.lens, stream, 2, torch.int32)
        ws = self._workspace(stream, at)
        self._run(self._lib.verbo_cache_compact, info.data_ptr(), ws.data_ptr(), self._need, at)
        return info

    def _tokens(self, t, what, heads=None):
        """(tokens, heads, token stride, head stride, type code) of [tokens, heads, dim]."""
        if t.dim() != 3 or t.shape[2] != self.dim or (heads is not None and t.shape[1] != heads):
            raise VerboCudaError(f"{what} must be [tokens, {heads or 'heads'}, {self.dim}]")
        if t.shape[0] > _INT_MAX or t.shape[1] > _INT_MAX:
            raise VerboCudaError(f"{what} must have at most {_INT_MAX} tokens and heads")
        if t.get_device() != self._dev:
            raise VerboCudaError(f"{what} must be a CUDA tensor on the device of the cache")
        code = self._types.get(t.dtype)
        if code is None:
            raise VerboCudaError(f"{what} must be float32, float16 or bfloat16")
        ld, hd, step = t.stride()
        if step != 1:
            raise VerboCudaError(f"{what}: its last dimension must be contiguous")
        # a dimension of one element may have any stride: it is not used
        return t.shape[0], t.shape[1], ld if t.shape[0] > 1 else 0, hd if t.shape[1] > 1 else 0, code

    def append(self, layer, k, v, start, off=None, stream=None):
        """Quantises keys and values of new tokens into a layer (verbo_cache_append).

        k, v: [tokens, heads, dim] in float32, float16 or bfloat16, any strides but the
        last.  Row r's tokens are off[r] .. off[r + 1] - 1 (int64 [rows + 1]), or, without
        off, its tokens / rows of them; they go to the places from start[r] on (int32
        [rows], as ``reserve`` returns it; negative: none)."""
        torch = self._torch
        n, _, ldk, hdk, code = self._tokens(k, "k", self.heads)
        nv, _, ldv, hdv, vcode = self._tokens(v, "v", self.heads)
        if nv != n or vcode != code:
            raise VerboCudaError("k and v must have the same tokens and type")
        dev = self._dev
        sp = self._ints(start, "start")
        op = _list(off, torch.int64, dev, "off", self.rows + 1)
        self._run(self._lib.verbo_cache_append, self._layer(layer), k.data_ptr(), ldk, hdk, v.data_ptr(), ldv, hdv,
                  code, n, sp, op, _stream_of(torch, dev, stream))

    def _layer(self, layer):
        layer = int(layer)
        if not 0 <= layer < self.layers:
            raise VerboCudaError(f"layer must be in [0, {self.layers})")
        return layer

    def attend(self, layer, q, scale=None, out=None, dtype=None, stream=None):
        """softmax(scale q k^T) v of the rows' last tokens over a layer
        (verbo_cache_attend).

        q: [rows * steps, heads, dim] in float32, float16 or bfloat16, any strides but the
        last; row r's are its last ``steps`` <= 32 tokens, each of which sees the places up to its
        own; heads a multiple of the cache's (head h reads the cache's head h * kv_heads
        // heads).  scale: 1 / sqrt(dim) if None.  Returns [rows * steps, heads, dim] of
        ``dtype`` (q's if None), or ``out``; zeros where nothing is seen."""
        torch = self._torch
        n, heads, ldq, hdq, code = self._tokens(q, "q")
        if self.rows and (n == 0 or n % self.rows):
            raise VerboCudaError("q must have the same number of tokens for every row")
        if not self.rows and n:
            raise VerboCudaError("q must have no tokens for no rows")
        steps = n // self.rows if self.rows else 1
        if scale is None:
            scale = 1.0 / math.sqrt(self.dim)
        if out is None:
            out_dtype = q.dtype if dtype is None else dtype
            if out_dtype not in self._types:
                raise VerboCudaError("dtype must be float32, float16 or bfloat16")
            out = _new(torch, q, stream, (n, heads, self.dim), out_dtype)
            ldo, hdo, ocode = heads * self.dim, self.dim, self._types[out_dtype]
        else:
            if dtype is not None and dtype != out.dtype:
                raise VerboCudaError("out must be of dtype")
            on, _, ldo, hdo, ocode = self._tokens(out, "out", heads)
            if on != n:
                raise VerboCudaError("out must have the tokens of q")
        at = _stream_of(torch, self._dev, stream)
        need = self._attend_need.get((heads, steps, code))
        if need is None:
            with torch.cuda.device(self.device):
                need = self._lib.verbo_cache_attend_workspace(self._ref, heads, steps, code)
            if need < 0:
                raise _err()
            self._attend_need[heads, steps, code] = need
        # this workspace belongs to the call's stream: freed here, it is reused behind the call
        ws = _new(torch, q, stream, need, torch.uint8) if need else None
        self._run(self._lib.verbo_cache_attend, self._layer(layer), q.data_ptr(), code, ldq, hdq, heads, steps, scale,
                  out.data_ptr(), ocode, ldo, hdo, ws.data_ptr() if need else None, need, at)
        return out
