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

import numpy as np

from . import _lib as L

ACTIVATIONS = {None: 0, "none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}
NORMS = {None: 0, "none": 0, "layer": 1, "rms": 2}
POOLS = {"mean": 1, "first": 2, "last": 3}
SCALINGS = {None: 0, "none": 0, "linear": 1, "base": 2, "parts": 3}


def _named(table: dict, name, what: str) -> int:
    try:
        return table[name]
    except KeyError:
        raise L.BVError(L.BV_E_INVALID, f"unknown {what} {name!r}") from None


def rotary_table(rows: int, rot_dim: int, base: float = 10000.0, scaling: str | None = None, factor: float = 1.0,
                 original_rows: float = 0.0, low_turns: float = 1.0, high_turns: float = 32.0,
                 magnitude: float = 1.0) -> np.ndarray:
    """Cosines and sines by position for ``EmbedOps.rotary``: float32
    [rows, rot_dim / 2, 2], computed in 64 bits (bv_embed_rotary_table has the
    scalings' formulas)."""
    if rows < 0 or rot_dim < 0:
        raise L.BVError(L.BV_E_INVALID, "rows and rot_dim are not negative")
    s = L.RotaryScaling(ctypes.sizeof(L.RotaryScaling), _named(SCALINGS, scaling, "scaling"), base, factor, original_rows,
                        low_turns, high_turns, magnitude)
    out = np.empty((rows, rot_dim // 2, 2), np.float32)
    L.check(L.load().bv_embed_rotary_table(ctypes.addressof(s), rows, rot_dim, out.ctypes.data, rows * rot_dim))
    return out


class EmbedOps:
    """Operators on one device, for one thread at a time.  Inputs whose last
    dimension is not contiguous, or whose rows overlap, are copied first."""

    def __init__(self, ctx):
        import torch

        self.torch = torch
        self.ctx = ctx
        self.lib = ctx.lib
        h = ctypes.c_void_p()
        L.check(self.lib.bv_embed_create(ctx.handle, ctypes.byref(h)))
        self.handle = h
        self._dtypes = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
        self._args = {}
        for t in (L.LinearArgs, L.RotaryArgs, L.AttentionArgs, L.NormArgs):
            self._args[t] = t(ctypes.sizeof(t))
        self._stream = None

    def destroy(self) -> None:
        if self.handle:
            self.lib.bv_embed_destroy(self.handle)
            self.handle = None

    def sync(self) -> None:
        """Waits for the stream of the last call."""
        L.check(self.lib.bv_embed_sync(self.handle))

    # -- plumbing ------------------------------------------------------------
    def _call(self, fn, a, device) -> None:
        stream = self.torch.cuda.current_stream(device).cuda_stream
        if stream != self._stream:
            L.check(self.lib.bv_embed_set_stream(self.handle, stream))
            self._stream = stream
        L.check(fn(self.handle, ctypes.addressof(a)))

    def _dtype(self, t, what: str) -> int:
        try:
            return self._dtypes[t.dtype]
        except KeyError:
            raise L.BVError(L.BV_E_UNSUPPORTED, f"{what}: {t.dtype} is not float32, float16 or bfloat16") from None

    @staticmethod
    def _need(ok: bool, msg: str) -> None:
        if not ok:
            raise L.BVError(L.BV_E_INVALID, msg)

    def _same(self, what: str, ref, **tensors) -> None:
        """Every tensor is on the context's device."""
        if not ref.is_cuda or ref.device.index != self.ctx.ordinal:
            raise L.BVError(L.BV_E_INVALID, f"{what}: tensors must be on GPU {self.ctx.ordinal}, not {ref.device}")
        for name, t in tensors.items():
            if t is not None and t.device != ref.device:
                raise L.BVError(L.BV_E_INVALID, f"{what}: {name} is on {t.device}, not {ref.device}")

    @staticmethod
    def _rows(t):
        """t [..., n] as rows for the library: itself where the last dimension
        is contiguous and the others are one stride apart, or a copy."""
        t = t if t.dim() == 2 else t.reshape(-1, t.shape[-1])
        st = t.stride()
        if (st[1] != 1 and t.shape[1] > 1) or (st[0] < t.shape[1] and t.shape[0] > 1):
            t = t.contiguous()
        return t

    @staticmethod
    def _heads(t):
        st, sh = t.stride(), t.shape
        if (st[2] != 1 and sh[2] > 1) or (st[1] < sh[2] and sh[1] > 1) or (st[0] < sh[2] and sh[0] > 1):
            t = t.contiguous()
        return t

    def _vector(self, t, n: int, what: str):
        self._need(t.dim() == 1 and t.shape[0] == n, f"{what} has shape {tuple(t.shape)}, not ({n},)")
        return t.contiguous()

    def _offsets(self, t, what: str):
        self._need(t.dim() == 1 and t.shape[0] >= 1 and t.dtype == self.torch.int32, f"{what} is not a vector of int32 offsets")
        return t.contiguous()

    # -- operators -----------------------------------------------------------
    def linear(self, x, weight, bias=None, residual=None, activation=None, out=None, out_dtype=None):
        """act(x weight^T + bias) + residual: x [..., k], weight [n, k], bias
        [n], residual and the result [..., n].  x and weight float16 or
        bfloat16, the result of that type or float32."""
        a = self._args[L.LinearArgs]
        act = _named(ACTIVATIONS, activation, "activation")
        self._same("linear", x, weight=weight, bias=bias, residual=residual, out=out)
        self._need(weight.dim() == 2 and x.dim() >= 1 and x.shape[-1] == weight.shape[1],
                   f"linear: x {tuple(x.shape)} and weight {tuple(weight.shape)} do not fit")
        self._need(weight.dtype == x.dtype and (bias is None or bias.dtype == x.dtype), "linear: x, weight and bias differ in type")
        n, shape = weight.shape[0], x.shape[:-1] + weight.shape[:1]
        x2, w2 = self._rows(x), self._rows(weight)
        if out is None:
            out = x.new_empty(shape, dtype=out_dtype or x.dtype)
            y = out if out.dim() == 2 else out.view(-1, n)
        else:
            self._need(out.shape == shape and (out_dtype is None or out.dtype == out_dtype), f"linear: out has shape {tuple(out.shape)}, not {tuple(shape)}, or another type")
            y = out if out.dim() == 2 else out.view(-1, n)
            self._need(y.stride(1) == 1 or n <= 1, "linear: out's last dimension is not contiguous")
        r = None
        if residual is not None:
            self._need(residual.shape == shape and residual.dtype == out.dtype, "linear: residual differs from the result in shape or type")
            r = y if residual is out else self._rows(residual)
        b = None if bias is None else self._vector(bias, n, "linear: bias")
        a.dtype, a.out_dtype, a.activation = self._dtype(x, "linear"), self._dtype(out, "linear"), act
        a.m, a.n, a.k = x2.shape[0], n, x2.shape[1]
        a.x, a.w, a.y = x2.data_ptr(), w2.data_ptr(), y.data_ptr()
        a.bias = None if b is None else b.data_ptr()
        a.residual = None if r is None else r.data_ptr()
        a.x_stride, a.w_stride, a.y_stride = self._stride(x2), self._stride(w2), self._stride(y)
        a.residual_stride = 0 if r is None else self._stride(r)
        self._call(self.lib.bv_embed_linear, a, x.device)
        return out

    @staticmethod
    def _stride(t) -> int:
        return t.stride(0) if t.shape[0] > 1 else 0

    def rotary(self, q, k, table, positions=None, interleaved: bool = False, out_q=None, out_k=None):
        """q [tokens, heads, d] and k (or None) with their first
        2 * table.shape[1] elements turned by the table's rows at each token's
        position; ``table`` float32 [rows, pairs, 2] (``rotary_table``),
        ``positions`` int32 [tokens], None: 0, 1, ...  out_q = q and out_k = k
        turn them in place."""
        a = self._args[L.RotaryArgs]
        self._same("rotary", q, k=k, table=table, positions=positions, out_q=out_q, out_k=out_k)
        self._need(q.dim() == 3 and (k is None or (k.dim() == 3 and k.shape[0] == q.shape[0] and k.shape[2] == q.shape[2] and
                                                   k.dtype == q.dtype)), "rotary: q and k are not [tokens, heads, d] alike")
        self._need(table.dim() == 3 and table.shape[2] == 2 and table.dtype == self.torch.float32 and table.is_contiguous(),
                   "rotary: the table is not contiguous float32 [rows, pairs, 2]")
        if positions is not None:
            self._need(positions.dim() == 1 and positions.shape[0] == q.shape[0] and positions.dtype == self.torch.int32,
                       "rotary: positions are not one int32 per token")
            positions = positions.contiguous()
        a.dtype = self._dtype(q, "rotary")
        a.tokens, a.heads_q, a.head_dim = q.shape
        a.heads_k = 0 if k is None else k.shape[1]
        a.rot_dim, a.table_rows, a.interleaved = 2 * table.shape[1], table.shape[0], bool(interleaved)
        a.table = table.data_ptr()
        a.positions = None if positions is None else positions.data_ptr()
        qi, qo, out_q = self._turned(q, out_q, "q")
        a.q, a.q_out = qi.data_ptr(), qo.data_ptr()
        a.q_stride, a.q_head_stride, _ = qi.stride()
        a.q_out_stride, a.q_out_head_stride, _ = qo.stride()
        if k is None:
            a.k = a.k_out = None
            a.k_stride = a.k_head_stride = a.k_out_stride = a.k_out_head_stride = 0
        else:
            ki, ko, out_k = self._turned(k, out_k, "k")
            a.k, a.k_out = ki.data_ptr(), ko.data_ptr()
            a.k_stride, a.k_head_stride, _ = ki.stride()
            a.k_out_stride, a.k_out_head_stride, _ = ko.stride()
        self._call(self.lib.bv_embed_rotary, a, q.device)
        return out_q, out_k

    def _turned(self, x, out, name: str):
        if out is None:
            out = x.new_empty(x.shape)
        elif out is not x:
            self._need(out.shape == x.shape and out.dtype == x.dtype, f"rotary: out_{name} differs from {name} in shape or type")
        self._need(out.shape[2] <= 1 or out.stride(2) == 1, f"rotary: out_{name}'s last dimension is not contiguous")
        return (x if out is x else self._heads(x)), out, out

    def attention(self, q, k, v, cu_q, cu_k=None, max_q: int = 0, max_k: int = 0, causal: bool = True, scale: float | None = None,
                  out=None):
        """softmax(scale q k^T) v of packed sequences: q [tokens, heads, d], k
        and v [keys, key heads, d] in float16 or bfloat16, cu_q and cu_k int32
        offsets [batch + 1] (cu_k None: cu_q).  causal: a sequence's last query
        sees its last key.  max_q and max_k: the longest lengths where they are
        known; they steer how the work is split."""
        a = self._args[L.AttentionArgs]
        if cu_k is None:
            cu_k = cu_q
            max_k = max_k or max_q
        self._same("attention", q, k=k, v=v, cu_q=cu_q, cu_k=cu_k, out=out)
        self._need(q.dim() == 3 and k.dim() == 3 and v.shape == k.shape and k.shape[2] == q.shape[2],
                   "attention: q is not [tokens, heads, d], or k and v are not [keys, key heads, d] alike")
        self._need(k.dtype == q.dtype and v.dtype == q.dtype, "attention: q, k and v differ in type")
        cu_q, cu_k = self._offsets(cu_q, "attention: cu_q"), self._offsets(cu_k, "attention: cu_k")
        self._need(cu_q.shape == cu_k.shape, "attention: cu_q and cu_k differ in length")
        self._need(max_q >= 0 and max_k >= 0, "attention: max_q and max_k are not negative")
        if out is None:
            out = q.new_empty(q.shape)
        else:
            self._need(out.shape == q.shape and out.dtype == q.dtype and (out.shape[2] <= 1 or out.stride(2) == 1),
                       "attention: out differs from q in shape or type, or its last dimension is not contiguous")
        q2, k2, v2 = self._heads(q), self._heads(k), self._heads(v)
        a.dtype, a.causal, a.batch = self._dtype(q, "attention"), bool(causal), cu_q.shape[0] - 1
        a.tokens_q, a.heads_q, a.head_dim = q.shape
        a.tokens_k, a.heads_k = k.shape[0], k.shape[1]
        a.max_q, a.max_k, a.scale = max_q, max_k, 0.0 if scale is None else scale
        a.q, a.k, a.v, a.o = q2.data_ptr(), k2.data_ptr(), v2.data_ptr(), out.data_ptr()
        a.cu_q, a.cu_k = cu_q.data_ptr(), cu_k.data_ptr()
        a.q_stride, a.q_head_stride, _ = q2.stride()
        a.k_stride, a.k_head_stride, _ = k2.stride()
        a.v_stride, a.v_head_stride, _ = v2.stride()
        a.o_stride, a.o_head_stride, _ = out.stride()
        self._call(self.lib.bv_embed_attention, a, q.device)
        return out

    def _norm(self, what: str, x, weight, bias, kind, eps, pool, unit, cu, out):
        a = self._args[L.NormArgs]
        self._same(what, x, weight=weight, bias=bias, cu=cu, out=out)
        dim = x.shape[-1]
        w = None if weight is None else self._vector(weight, dim, f"{what}: weight")
        b = None if bias is None else self._vector(bias, dim, f"{what}: bias")
        self._need(w is None or b is None or w.dtype == b.dtype, f"{what}: weight and bias differ in type")
        x2 = self._rows(x)
        y = out if out.dim() == 2 else out.view(-1, dim)
        self._need(y.stride(1) == 1 or dim <= 1, f"{what}: out's last dimension is not contiguous")
        if out is x:
            x2 = y
        a.dtype, a.out_dtype = self._dtype(x, what), self._dtype(out, what)
        either = w if w is not None else b
        a.weight_dtype = 0 if either is None else self._dtype(either, what)
        a.norm, a.pool, a.unit = _named(NORMS, kind, "norm"), pool, bool(unit)
        a.dim, a.eps, a.tokens = dim, eps, x2.shape[0]
        a.batch = 0 if cu is None else cu.shape[0] - 1
        a.x, a.y = x2.data_ptr(), y.data_ptr()
        a.weight = None if w is None else w.data_ptr()
        a.bias = None if b is None else b.data_ptr()
        a.cu = None if cu is None else cu.data_ptr()
        a.x_stride, a.y_stride = self._stride(x2), self._stride(y)
        self._call(self.lib.bv_embed_norm, a, x.device)
        return out

    def norm(self, x, weight=None, bias=None, kind: str = "layer", eps: float = 1e-5, out=None, out_dtype=None):
        """Layer or RMS norm of x [..., dim] (kind "layer", "rms" or None)
        times weight plus bias; out = x works in place."""
        if out is None:
            out = x.new_empty(x.shape, dtype=out_dtype or x.dtype)
        else:
            self._need(out.shape == x.shape and (out_dtype is None or out.dtype == out_dtype), "norm: out differs from x in shape, or in type from out_dtype")
        return self._norm("norm", x, weight, bias, kind, eps, 0, False, None, out)

    def pool(self, x, cu, mode: str = "mean", kind: str | None = None, weight=None, bias=None, eps: float = 1e-5,
             unit: bool = True, out=None):
        """One float32 vector per packed sequence of x [tokens, dim]: the mean,
        first or last of its rows after the norm (kind None: the rows as they
        are), divided by its 2-norm with ``unit``."""
        self._need(x.dim() == 2, "pool: x is not [tokens, dim]")
        cu = self._offsets(cu, "pool: cu")
        shape = (cu.shape[0] - 1, x.shape[1])
        if out is None:
            out = x.new_empty(shape, dtype=self.torch.float32)
        else:
            self._need(out.shape == shape and out.dtype == self.torch.float32, f"pool: out is not float32 {shape}")
        return self._norm("pool", x, weight, bias, kind, eps, _named(POOLS, mode, "pooling"), unit, cu, out)
