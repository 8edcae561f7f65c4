"""An embedding model's operators on the GPU that holds the index.

The reference leaves text -> vector to another library
(src/embed/transformers.ts); ``EmbedOps`` has the operators such a model's
forward pass is made of (``linear``, ``rotary``, ``attention``, ``norm``), and
``pool``, whose rows are what ``append_device`` and ``search_device`` take.

Inputs and outputs are torch tensors on the context's device; torch is only
imported by this class.  Calls run on torch's current stream and return without
waiting; inside ``torch.cuda.stream(torch.cuda.ExternalStream(index.stream_ptr()))``
that is an index's, and its appends and searches follow in order.
"""

from __future__ import annotations

import ctypes
import math

import numpy as np

from . import _lib as L

ACTIVATIONS = {None: 0, "none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}
NORMS = {None: 0, "none": 0, "layer": 1, "rms": 2}
POOLS = {"mean": 1, "first": 2, "last": 3}
SCALINGS = {None: 0, "none": 0, "linear": 1, "base": 2, "parts": 3}


def rotary_table(rows: int, rot_dim: int, base: float = 10000.0, scaling: str | None = None, factor: float = 1.0,
                 original_rows: float = 0.0, low_turns: float = 1.0, high_turns: float = 32.0,
                 magnitude: float = 1.0) -> np.ndarray:
    """Cosines and sines by position for ``EmbedOps.rotary``: float32
    [rows, rot_dim / 2, 2], computed in 64 bits (bv_embed_rotary_table has the
    scalings' formulas)."""
    if rows < 0 or rot_dim < 0:
        raise L.BVError(L.BV_E_INVALID, "rows and rot_dim are not negative")
    if scaling not in SCALINGS:
        raise L.BVError(L.BV_E_INVALID, f"unknown scaling {scaling!r}")
    if magnitude == 0:  # the library's word for its default
        raise L.BVError(L.BV_E_INVALID, "magnitude is 0")
    s = L.RotaryScaling(ctypes.sizeof(L.RotaryScaling), SCALINGS[scaling], base, factor, original_rows,
                        low_turns, high_turns, magnitude)
    out = np.empty((rows, rot_dim // 2, 2), np.float32)
    L.check(L.load().bv_embed_rotary_table(ctypes.addressof(s), rows, rot_dim, out.ctypes.data, rows * rot_dim))
    return out


def _bad(msg: str):
    raise L.BVError(L.BV_E_INVALID, msg)


def _too_many(what: str, *sizes):
    """Of sizes that the library takes as 32 bits: a ctypes field would cut them
    down to these without an error."""
    raise L.BVError(L.BV_E_UNSUPPORTED, f"{what}: a dimension of {max(sizes)} exceeds 32 bits")


class EmbedOps:
    """Operators on one device, for one thread at a time.  Inputs whose last
    dimension is not contiguous, or whose rows overlap, are copied first.

    Torch's autograd does not see these calls: results of tensors that require
    gradients have none, and writes to ``out`` leave its version as it was."""

    def __init__(self, ctx):
        import torch

        self.ctx = ctx
        self.lib = ctx.lib
        h = ctypes.c_void_p()
        L.check(self.lib.bv_embed_create(ctx.handle, ctypes.byref(h)))
        self.handle = h
        self._ordinal = ctx.ordinal
        self._dtypes = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
        self._int32, self._f32, self._empty = torch.int32, torch.float32, torch.empty
        # the arguments of each operator, filled in anew by every call, with
        # their address
        self._linear, self._rotary, self._attention, self._norm = (
            (t, ctypes.addressof(t)) for t in (c(ctypes.sizeof(c)) for c in (L.LinearArgs, L.RotaryArgs, L.AttentionArgs,
                                                                             L.NormArgs)))
        # the current stream as an int, without the object around it where torch has that
        raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
        self._current = raw or (lambda ordinal: torch.cuda.current_stream(ordinal).cuda_stream)
        self._stream = None

    def destroy(self) -> None:
        if self.handle:
            self.lib.bv_embed_destroy(self.handle)
            self.handle = None

    def sync(self) -> None:
        """Waits for the stream of the last call."""
        L.check(self.lib.bv_embed_sync(self.handle))

    # -- plumbing (a call's checks cost as much as its launch: no message is
    # -- made up unless it is needed) ------------------------------------------
    def _call(self, fn, address) -> None:
        stream = self._current(self._ordinal)
        if stream != self._stream:
            L.check(self.lib.bv_embed_set_stream(self.handle, stream))
            self._stream = stream
        rc = fn(self.handle, address)
        if rc:
            L.check(rc)

    def _here(self, what: str, *tensors) -> None:
        """Every tensor is on the context's device."""
        for t in tensors:
            if t is not None and t.get_device() != self._ordinal:
                _bad(f"{what}: tensors must be on GPU {self._ordinal}, not {t.device}")

    def _dtype(self, t, what: str) -> int:
        code = self._dtypes.get(t.dtype)
        if code is None:
            raise L.BVError(L.BV_E_UNSUPPORTED, f"{what}: {t.dtype} is not float32, float16 or bfloat16")
        return code

    def _vector(self, t, n: int, what: str):
        if t.shape != (n,):
            _bad(f"{what} has shape {tuple(t.shape)}, not ({n},)")
        return t.contiguous()

    def _offsets(self, t, what: str):
        if t.dim() != 1 or t.shape[0] < 1 or t.dtype != self._int32:
            _bad(f"{what} is not a vector of int32 offsets")
        return t.contiguous()

    # -- operators -----------------------------------------------------------
    def linear(self, x, weight, bias=None, residual=None, activation=None, out=None, out_dtype=None):
        """act(x weight^T + bias) + residual: x [..., k], weight [n, k], bias
        [n], residual and the result [..., n].  x and weight float16 or
        bfloat16, the result of that type or float32."""
        a, address = self._linear
        act = ACTIVATIONS.get(activation)
        if act is None:
            _bad(f"unknown activation {activation!r}")
        self._here("linear", x, weight, bias, residual, out)
        sx, sw, dtype = x.shape, weight.shape, x.dtype
        if len(sw) != 2 or len(sx) < 1 or sx[-1] != sw[1]:
            _bad(f"linear: x {tuple(sx)} and weight {tuple(sw)} do not fit")
        if weight.dtype != dtype or (bias is not None and bias.dtype != dtype):
            _bad("linear: x, weight and bias differ in type")
        n, k = sw
        if (n | k) >> 32:
            _too_many("linear", n, k)
        flat = len(sx) == 2
        shape = (sx[0], n) if flat else (*sx[:-1], n)
        if out is None:
            out = self._empty(shape, dtype=out_dtype or dtype, device=x.device)
        elif out.shape != shape or (out_dtype is not None and out.dtype != out_dtype):
            _bad(f"linear: out has shape {tuple(out.shape)}, not {tuple(shape)}, or another type")
        y = out if flat else _flat(out, "linear")
        a.dtype, a.out_dtype, a.activation = self._dtype(x, "linear"), self._dtype(out, "linear"), act
        x2, a.x_stride = _rows(x)
        w2, a.w_stride = _rows(weight)
        a.y_stride = _out_stride(y, "linear")
        a.m, a.n, a.k = x2.shape[0], n, k
        a.x, a.w, a.y = x2.data_ptr(), w2.data_ptr(), y.data_ptr()
        if bias is None:
            a.bias = None
        else:
            bias = self._vector(bias, n, "linear: bias")
            a.bias = bias.data_ptr()
        if residual is None:
            a.residual = None
        elif residual is out:
            a.residual, a.residual_stride = a.y, a.y_stride
        else:
            if residual.shape != shape or residual.dtype != out.dtype:
                _bad("linear: residual differs from the result in shape or type")
            residual, a.residual_stride = _rows(residual)
            a.residual = residual.data_ptr()
        self._call(self.lib.bv_embed_linear, address)
        return out

    def rotary(self, q, k, table, positions=None, interleaved: bool = False, out_q=None, out_k=None):
        """q [tokens, heads, d] and k (or None) with their first
        2 * table.shape[1] elements turned by the table's rows at each token's
        position; ``table`` float32 [rows, pairs, 2] (``rotary_table``),
        ``positions`` int32 [tokens], None: 0, 1, ...  out_q = q and out_k = k
        turn them in place."""
        a, address = self._rotary
        self._here("rotary", q, k, table, positions, out_q, out_k)
        sq, st = q.shape, table.shape
        if len(sq) != 3 or (k is not None and (k.dim() != 3 or k.shape[0] != sq[0] or k.shape[2] != sq[2] or k.dtype != q.dtype)):
            _bad("rotary: q and k are not [tokens, heads, d] alike")
        if len(st) != 3 or st[2] != 2 or table.dtype != self._f32 or not table.is_contiguous():
            _bad("rotary: the table is not contiguous float32 [rows, pairs, 2]")
        hk = 0 if k is None else k.shape[1]
        if (sq[1] | sq[2] | hk | 2 * st[1] | st[0]) >> 32:
            _too_many("rotary", sq[1], sq[2], hk, 2 * st[1], st[0])
        if positions is None:
            a.positions = None
        else:
            if positions.shape != sq[:1] or positions.dtype != self._int32:
                _bad("rotary: positions are not one int32 per token")
            positions = positions.contiguous()
            a.positions = positions.data_ptr()
        a.dtype = self._dtype(q, "rotary")
        a.tokens, a.heads_q, a.head_dim = sq
        a.rot_dim, a.table_rows, a.interleaved, a.table = 2 * st[1], st[0], bool(interleaved), table.data_ptr()
        qi, out_q = self._turned(q, out_q)
        a.q, a.q_out = qi.data_ptr(), out_q.data_ptr()
        a.q_stride, a.q_head_stride, _ = qi.stride()
        a.q_out_stride, a.q_out_head_stride, _ = out_q.stride()
        if k is None:
            a.k, a.k_out, a.heads_k = None, None, 0
        else:
            ki, out_k = self._turned(k, out_k)
            a.heads_k = hk
            a.k, a.k_out = ki.data_ptr(), out_k.data_ptr()
            a.k_stride, a.k_head_stride, _ = ki.stride()
            a.k_out_stride, a.k_out_head_stride, _ = out_k.stride()
        self._call(self.lib.bv_embed_rotary, address)
        return out_q, out_k

    def _turned(self, x, out):
        if out is None:
            return _heads(x), self._empty(x.shape, dtype=x.dtype, device=x.device)
        if out.shape != x.shape or out.dtype != x.dtype:
            _bad("rotary: an output differs from its input in shape or type")
        _out_heads(out, "rotary")
        return (x if out is x else _heads(x)), out

    def attention(self, q, k, v, cu_q, cu_k=None, max_q: int = 0, max_k: int = 0, causal: bool = True, scale: float | None = None,
                  out=None):
        """softmax(scale q k^T) v of packed sequences: q [tokens, heads, d], k
        and v [keys, key heads, d] in float16 or bfloat16, cu_q and cu_k int32
        offsets [batch + 1] (cu_k None: cu_q).  causal: a sequence's last query
        sees its last key.  scale None: 1 / sqrt(d); 0 is refused.  max_q and
        max_k: the longest lengths where they are known; they steer how the
        work is split."""
        a, address = self._attention
        if cu_k is None:
            cu_k = cu_q
            max_k = max_k or max_q
        self._here("attention", q, k, v, cu_q, cu_k, out)
        sq, sk, dtype = q.shape, k.shape, q.dtype
        if len(sq) != 3 or len(sk) != 3 or v.shape != sk or sk[2] != sq[2]:
            _bad("attention: q is not [tokens, heads, d], or k and v are not [keys, key heads, d] alike")
        if k.dtype != dtype or v.dtype != dtype:
            _bad("attention: q, k and v differ in type")
        if (sq[1] | sq[2] | sk[1] | cu_q.shape[0]) >> 32:
            _too_many("attention", sq[1], sq[2], sk[1], cu_q.shape[0])
        cu_q = self._offsets(cu_q, "attention: cu_q")
        cu_k = self._offsets(cu_k, "attention: cu_k")
        if cu_q.shape != cu_k.shape or max_q < 0 or max_k < 0:
            _bad("attention: cu_q and cu_k differ in length, or max_q or max_k is negative")
        if out is None:
            out = self._empty(sq, dtype=dtype, device=q.device)
        elif out.shape != sq or out.dtype != dtype:
            _bad("attention: out differs from q in shape or type")
        else:
            _out_heads(out, "attention")
        q, k, v = _heads(q), _heads(k), _heads(v)
        a.dtype, a.causal, a.batch = self._dtype(q, "attention"), bool(causal), cu_q.shape[0] - 1
        a.tokens_q, a.heads_q, a.head_dim = sq
        a.tokens_k, a.heads_k, _ = sk
        a.max_q, a.max_k, a.scale = min(max_q, sq[0]), min(max_k, sk[0]), 0.0 if scale is None else scale
        if scale is not None and a.scale == 0:  # in 32 bits; the library's word for its default
            _bad(f"attention: scale {scale} is 0 in 32 bits")
        a.q, a.k, a.v, a.o = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr()
        a.cu_q, a.cu_k = cu_q.data_ptr(), cu_k.data_ptr()
        a.q_stride, a.q_head_stride, _ = q.stride()
        a.k_stride, a.k_head_stride, _ = k.stride()
        a.v_stride, a.v_head_stride, _ = v.stride()
        a.o_stride, a.o_head_stride, _ = out.stride()
        self._call(self.lib.bv_embed_attention, address)
        return out

    def _normed(self, what: str, x, weight, bias, kind, eps, pool, unit, cu, out):
        a, address = self._norm
        norm = NORMS.get(kind)
        if norm is None:
            _bad(f"unknown norm {kind!r}")
        self._here(what, x, weight, bias, cu, out)
        if x.dim() < 1:
            _bad(f"{what}: x has no dimension")
        dim = x.shape[-1]
        if (dim | (0 if cu is None else cu.shape[0])) >> 32:
            _too_many(what, dim, 0 if cu is None else cu.shape[0])
        a.weight = a.bias = None
        if weight is not None:
            weight = self._vector(weight, dim, "weight")
            a.weight, a.weight_dtype = weight.data_ptr(), self._dtype(weight, what)
        if bias is not None:
            bias = self._vector(bias, dim, "bias")
            if weight is not None and weight.dtype != bias.dtype:
                _bad(f"{what}: weight and bias differ in type")
            a.bias, a.weight_dtype = bias.data_ptr(), self._dtype(bias, what)
        y = out if out.dim() == 2 else _flat(out, what)
        a.dtype, a.out_dtype = self._dtype(x, what), self._dtype(out, what)
        a.y_stride = _out_stride(y, what)
        x2, a.x_stride = (y, a.y_stride) if out is x else _rows(x)
        a.norm, a.pool, a.unit, a.dim, a.eps, a.tokens = norm, pool, unit, dim, eps, x2.shape[0]
        a.x, a.y = x2.data_ptr(), y.data_ptr()
        a.cu, a.batch = (None, 0) if cu is None else (cu.data_ptr(), cu.shape[0] - 1)
        self._call(self.lib.bv_embed_norm, address)
        return out

    def norm(self, x, weight=None, bias=None, kind: str = "layer", eps: float = 1e-5, out=None, out_dtype=None):
        """Layer or RMS norm of x [..., dim] (kind "layer", "rms" or None)
        times weight plus bias; out = x works in place."""
        if out is None:
            out = self._empty(x.shape, dtype=out_dtype or x.dtype, device=x.device)
        elif out.shape != x.shape or (out_dtype is not None and out.dtype != out_dtype):
            _bad("norm: out differs from x in shape, or in type from out_dtype")
        return self._normed("norm", x, weight, bias, kind, eps, 0, False, None, out)

    def pool(self, x, cu, mode: str = "mean", kind: str | None = None, weight=None, bias=None, eps: float = 1e-5,
             unit: bool = True, out=None):
        """One float32 vector per packed sequence of x [tokens, dim]: the mean,
        first or last of its rows after the norm (kind None: the rows as they
        are), divided by its 2-norm with ``unit``."""
        pool = POOLS.get(mode)
        if pool is None or x.dim() != 2:
            _bad(f"unknown pooling {mode!r}, or x is not [tokens, dim]")
        cu = self._offsets(cu, "pool: cu")
        shape = (cu.shape[0] - 1, x.shape[1])
        if out is None:
            out = self._empty(shape, dtype=self._f32, device=x.device)
        elif out.shape != shape or out.dtype != self._f32:
            _bad(f"pool: out is not float32 {shape}")
        return self._normed("pool", x, weight, bias, kind, eps, pool, bool(unit), cu, out)


def _rows(t):
    """t [..., n] as rows and their stride: itself where the last dimension is
    contiguous and the others are one stride apart, or a copy.  0: packed."""
    if t.dim() != 2:
        t = t.reshape(math.prod(t.shape[:-1]), t.shape[-1])
    if t.is_contiguous():
        return t, 0
    rows, n = t.shape
    step, one = t.stride()
    if (one != 1 and n > 1) or (step < n and rows > 1):
        return t.contiguous(), 0
    return t, step if rows > 1 else 0


def _flat(out, what: str):
    """out [..., n] as rows of the same memory."""
    try:
        return out.view(math.prod(out.shape[:-1]), out.shape[-1])
    except RuntimeError:
        _bad(f"{what}: out's rows do not lie one stride apart")


def _out_stride(y, what: str) -> int:
    if y.is_contiguous():
        return 0
    rows, n = y.shape
    step, one = y.stride()
    if one != 1 and n > 1:
        _bad(f"{what}: out's last dimension is not contiguous")
    if rows > 1 and step < n:  # an expanded tensor's 0 among them, which would mean packed
        _bad(f"{what}: out's rows overlap")
    return step if rows > 1 else 0


def _out_heads(out, what: str) -> None:
    """Refuses what the library would take for packed heads (other strides that
    make heads overlap it refuses itself)."""
    tokens, heads, d = out.shape
    st, sh, one = out.stride()
    if one != 1 and d > 1:
        _bad(f"{what}: out's last dimension is not contiguous")
    if (st == 0 and tokens > 1) or (sh == 0 and heads > 1):
        _bad(f"{what}: out's rows overlap")


def _heads(t):
    if t.is_contiguous():
        return t
    tokens, heads, d = t.shape
    st, sh, one = t.stride()
    if (one != 1 and d > 1) or (sh < d and heads > 1) or (st < d and tokens > 1):
        return t.contiguous()
    return t
