"""The operators of the paged key/value cache of include/tsn.h on torch tensors: :class:`CacheAppend`,
:class:`PagedAttention` and :class:`SparseAttention`.

They are made and called as the transformer-block operators are: an object holds a layer's weights and options and the
arguments of its last call, results go into tensors that the caller owns, calls are issued on the device handle's stream and do
not synchronise. What a batch is, for all three:

``k_pages``, ``v_pages`` [P, page, Hk, head_dim], any strides whose last dimension is contiguous; ``table`` int32 [B, M], the pages
of each sequence; ``lens`` int32 [B], its tokens in the cache, the new ones included; ``q_start`` int32 [B + 1], the
rows at which each sequence's new tokens start, or None for one new token a sequence.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import CacheAppendArgs, Paged, PagedAttnArgs, RopePlan, SparseAttnArgs, check, lib
from .block_ops import LAYOUTS, TYPES, _address, _form_of, _here, _known, _put, _record, _want, _weights


def _ints(name, t, shape):
    if t.dtype is not torch.int32 or tuple(t.shape) != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor of shape {list(shape)}")


def _cache(c, rows, D, k_pages, v_pages, table, lens, q_start):
    """Checks the cache and the batch of a call with `rows` new tokens, and describes them."""
    if k_pages.dim() != 4 or k_pages.shape[3] != D:
        raise ValueError(f"k_pages must be [P, page, Hk, {D}]")
    dtype = k_pages.dtype
    if dtype not in (torch.float16, torch.bfloat16):
        raise TypeError("k_pages must be float16 or bfloat16")
    _want("v_pages", v_pages, k_pages.shape, dtype)
    _put(c.k, "k_pages", k_pages)
    _put(c.v, "v_pages", v_pages)
    if table.dim() != 2 or table.dtype is not torch.int32 or (table.stride(1) != 1 and table.shape[1] > 1):
        raise ValueError("table must be int32 [B, M], its last dimension contiguous")
    B = table.shape[0]
    _ints("lens", lens, (B,))
    if q_start is not None:
        _ints("q_start", q_start, (B + 1,))
    elif rows != B:
        raise ValueError(f"{rows} new tokens for {B} sequences: q_start is wanted")
    c.P, c.page, c.Hk, c.D = k_pages.shape
    c.B, c.M = table.shape
    c.N, c.type, c.table_sb = rows, TYPES[dtype], table.stride(0)
    return dtype


def _rows(name, t, D, dtype, rows=None):
    if t.dim() != 3 or t.shape[2] != D or (rows is not None and t.shape[0] != rows):
        raise ValueError(f"{name} must be [{'N' if rows is None else rows}, heads, {D}], got {tuple(t.shape)}")
    if t.dtype is not dtype:
        raise TypeError(f"{name} is {t.dtype}, expected {dtype}")


def _paged(args):
    """The places that the cache's and the batch's addresses go to."""
    at = C.addressof(args.c)
    return (C.addressof(args.c.k), C.addressof(args.c.v), at + Paged.table.offset, at + Paged.len.offset, at + Paged.q_start.offset)


def _scale(scale):
    """The factor on the scores as the arguments have it, where 0 stands for the default; the rest the library checks."""
    if scale is None:
        return 0.0
    if scale == 0:
        raise ValueError("scale must be positive")
    return scale


def _count(name, n):
    """A whole number that the arguments' 32 bits hold: what exceeds them would arrive as another number."""
    if not 0 <= n < 2 ** 32:
        raise ValueError(f"{name} must be a whole number of 32 bits, got {n}")
    return n


class _Op:
    def _ready(self, args, call, *places):
        self._a, self._ref, self._call = args, C.byref(args), call
        self._places = [C.c_void_p.from_address(p) for p in places]
        self._form, self._formed = _form_of(*places)

    def _take(self, tensors):
        if not _known(self._formed, tensors):
            self._check(*tensors)
            _record(self._formed, tensors)
            for place, t in zip(self._places, tensors):
                place.value = _address(t)


class CacheAppend(_Op):
    """Appends new tokens to a paged cache (tsn_cache_append): an optional RMSNorm of each head and rotary positions for queries
    and keys, keys and values into their pages.

    `pairs`, `theta`, `scale`, `layout`, `q_norm`, `k_norm`: as :class:`tsn.RopeAxes`; head_dim a multiple of 8."""

    def __init__(self, dev, head_dim: int, pairs, theta=10000.0, scale=1.0, layout: str = "interleaved", q_norm=None,
                 k_norm=None, eps: float = 1e-6):
        if layout not in LAYOUTS:
            raise ValueError("layout must be 'interleaved' or 'half'")
        n = len(pairs)
        theta = [theta] * n if isinstance(theta, (int, float)) else list(theta)
        scale = [scale] * n if isinstance(scale, (int, float)) else list(scale)
        if len(theta) != n or len(scale) != n:
            raise ValueError("theta and scale: one value, or one per axis")
        self.dev, self.D, self.axes = dev, head_dim, n
        self._plan = RopePlan()
        check(lib().tsn_rope_plan(head_dim, n, (C.c_uint32 * n)(*pairs), (C.c_double * n)(*theta),
                                  (C.c_double * n)(*scale), LAYOUTS[layout], C.byref(self._plan)))
        self._plan_ref = C.byref(self._plan)
        self._keep = [_weights(dev, "q_norm", q_norm, (head_dim,)), _weights(dev, "k_norm", k_norm, (head_dim,))]
        a = CacheAppendArgs()
        a.eps = eps
        a.q_norm, a.k_norm = (_address(t) for t in self._keep)
        self._ready(a, lib().tsn_cache_append, C.addressof(a.q), C.addressof(a.k), C.addressof(a.v), *_paged(a),
                    C.addressof(a.q_out), C.addressof(a) + CacheAppendArgs.pos.offset, C.addressof(a.means))

    def __call__(self, q, k, v, k_pages, v_pages, table, lens, q_out=None, q_start=None, pos=None, means=None):
        """q [N, Hq, head_dim] or None, k, v [N, Hk, head_dim], of the cache's type or float32. q_out: of the cache's type; None:
        in place. pos int32 [N, axes], or None: a token's place in its sequence (one axis). means [P, Hk, head_dim] of the
        cache's type, or None: the mean key of each page that the tokens go into is written."""
        if q_out is None:
            q_out = q
        self._take((q, k, v, k_pages, v_pages, table, lens, q_start, q_out, pos, means))
        rc = self._call(self.dev.h, self._plan_ref, self._ref)
        if rc:
            check(rc)

    def _check(self, q, k, v, k_pages, v_pages, table, lens, q_start, q_out, pos, means):
        a, D = self._a, self.D
        _here(self.dev, ("q", q), ("k", k), ("v", v), ("k_pages", k_pages), ("v_pages", v_pages), ("table", table), ("lens", lens),
              ("q_start", q_start), ("q_out", q_out), ("pos", pos), ("means", means))
        N = k.shape[0]
        dtype = _cache(a.c, N, D, k_pages, v_pages, table, lens, q_start)
        if k.dtype not in (dtype, torch.float32):
            raise TypeError(f"k is {k.dtype}, expected {dtype} or float32")
        a.xtype, a.Hq = TYPES[k.dtype], 0
        _rows("k", k, D, k.dtype)
        _want("v", v, k.shape, k.dtype)
        if k.shape[1] != a.c.Hk:
            raise ValueError(f"k has {k.shape[1]} heads, the cache {a.c.Hk}")
        _put(a.k, "k", k)
        _put(a.v, "v", v)
        if q is not None:
            _rows("q", q, D, k.dtype, N)
            _want("q_out", q_out, q.shape, dtype)
            _put(a.q, "q", q)
            _put(a.q_out, "q_out", q_out)
            a.Hq = q.shape[1]
        if pos is not None:
            if pos.dtype is not torch.int32 or tuple(pos.shape) != (N, self.axes) or (pos.stride(1) != 1 and self.axes > 1):
                raise ValueError(f"pos must be int32 [{N}, {self.axes}], its last dimension contiguous")
            a.pos_ss = pos.stride(0)
        elif self.axes > 1:
            raise ValueError("pos is wanted: the positions have several axes")
        if means is not None:
            _want("means", means, (a.c.P, a.c.Hk, D), dtype)
            _put(a.means, "means", means)


class PagedAttention(_Op):
    """Attention of new tokens over a paged cache that they have been appended to (tsn_paged_attn):
    ``softmax(scale q k') v``; head_dim 64 or 128, `scale` 1 / sqrt(head_dim) where it is None."""

    def __init__(self, dev, head_dim: int, scale: float | None = None):
        self.dev, self.D = dev, head_dim
        a = PagedAttnArgs()
        a.scale = _scale(scale)
        self._ready(a, lib().tsn_paged_attn, C.addressof(a.q), C.addressof(a.out), *_paged(a))

    def __call__(self, q, k_pages, v_pages, table, lens, out, q_start=None, causal: bool = True, window: int = 0, most: int = 0):
        """q, out [N, H, head_dim] of the cache's type. causal: a token sees its own place and those before it, with a window
        the last `window` of them. most: new tokens of a sequence at most, where the caller knows it; 0: unknown."""
        a = self._a
        self._take((q, out, k_pages, v_pages, table, lens, q_start))
        a.causal, a.window, a.most = 1 if causal else 0, _count("window", window), _count("most", most)
        rc = self._call(self.dev.h, self._ref)
        if rc:
            check(rc)

    def _check(self, q, out, k_pages, v_pages, table, lens, q_start):
        a = self._a
        _here(self.dev, ("q", q), ("out", out), ("k_pages", k_pages), ("v_pages", v_pages), ("table", table), ("lens", lens),
              ("q_start", q_start))
        dtype = _cache(a.c, q.shape[0], self.D, k_pages, v_pages, table, lens, q_start)
        _rows("q", q, self.D, dtype)
        _want("out", out, q.shape, dtype)
        _put(a.q, "q", q)
        _put(a.out, "out", out)
        a.H = q.shape[1]


class SparseAttention(_Op):
    """Causal attention over `picks` pages of a paged cache, chosen for each token and kv head by the score of the page's mean key
    (tsn_sparse_attn). The `first` pages of a sequence and the `last` up to the token's own are always among them."""

    def __init__(self, dev, head_dim: int, picks: int, first: int = 1, last: int = 1, scale: float | None = None):
        self.dev, self.D, self.picks = dev, head_dim, picks
        a = SparseAttnArgs()
        a.picks, a.first, a.last, a.scale = _count("picks", picks), _count("first", first), _count("last", last), _scale(scale)
        self._ready(a, lib().tsn_sparse_attn, C.addressof(a.q), C.addressof(a.out), C.addressof(a.means),
                    C.addressof(a) + SparseAttnArgs.chosen.offset, *_paged(a))

    def __call__(self, q, k_pages, v_pages, means, table, lens, out, chosen, q_start=None):
        """q, out [N, H, head_dim] and means [P, Hk, head_dim] of the cache's type, means as :class:`CacheAppend` keeps them; chosen
        int32 [N, Hk, picks], the chosen pages of each token in ascending order, then -1."""
        self._take((q, out, means, chosen, k_pages, v_pages, table, lens, q_start))
        rc = self._call(self.dev.h, self._ref)
        if rc:
            check(rc)

    def _check(self, q, out, means, chosen, k_pages, v_pages, table, lens, q_start):
        a = self._a
        _here(self.dev, ("q", q), ("out", out), ("means", means), ("chosen", chosen), ("k_pages", k_pages), ("v_pages", v_pages),
              ("table", table), ("lens", lens), ("q_start", q_start))
        dtype = _cache(a.c, q.shape[0], self.D, k_pages, v_pages, table, lens, q_start)
        _rows("q", q, self.D, dtype)
        _want("out", out, q.shape, dtype)
        _want("means", means, (a.c.P, a.c.Hk, self.D), dtype)
        _ints("chosen", chosen, (q.shape[0], a.c.Hk, self.picks))
        _put(a.q, "q", q)
        _put(a.out, "out", out)
        _put(a.means, "means", means)
        a.H = q.shape[1]
