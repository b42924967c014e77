"""The transformer-block operators of include/tsn.h on torch tensors: :class:`BlockNorm`,
:class:`RopeAxes` and :class:`DiffAttention`.

Each object holds a layer's weights and options (kept alive by it) and is called with the tensors of one
pass; results go into tensors that the caller owns. Calls are issued on the device handle's stream and do
not synchronise. Tensors may have any strides whose last dimension is contiguous; what the library refuses
raises :class:`tsn.TsnError`, what does not fit together, or lies on another GPU than the handle's, raises
:class:`ValueError` or :class:`TypeError`. An object holds the arguments of its last call, so one thread at a time
calls it.
"""
from __future__ import annotations

import ctypes as C
import sys

import torch

from . import BlockNormArgs, DiffAttnArgs, Form, RopeArgs, RopePlan, check, form_take, lib

TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
NORMS = {"none": 0, "rms": 1, "layer": 2}
LAYOUTS = {"interleaved": 0, "half": 1}


def _weights(dev, name, t, shape):
    """A float32 weight on the handle's GPU, contiguous; None stays None."""
    if t is None:
        return None
    if tuple(t.shape) != tuple(shape) or t.dtype is not torch.float32:
        raise ValueError(f"{name} must be a float32 tensor of shape {tuple(shape)}")
    _here(dev, (name, t))
    if not t.is_contiguous():
        t = t.contiguous()
        torch.cuda.current_stream(t.device).synchronize()   # the copy's stream; calls are issued on the handle's
    return t


def _address(t):
    return None if t is None else t.data_ptr()


def _want(name, t, shape, dtype):
    if t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if t.dtype is not dtype:
        raise TypeError(f"{name} is {t.dtype}, expected {dtype}")


def _put(view, name, t):
    """Strides of a [., ., C] or [., ., ., C] tensor whose last dimension is contiguous."""
    st = t.stride()
    if st[-1] != 1 and t.shape[-1] > 1:
        raise ValueError(f"{name}: the last dimension must be contiguous")
    view.sb = st[0]
    if len(st) == 3:
        view.st = st[1]
    else:
        view.ss = st[1]
        view.sh = st[2]


def _here(dev, *named):
    """Every tensor lies on the handle's GPU."""
    for name, t in named:
        if t is not None and (t.get_device() != dev.ordinal or getattr(t, "is_meta", False)):
            raise ValueError(f"{name} must be a CUDA tensor on GPU {dev.ordinal}")


def _view():
    """The address of the function that describes a torch tensor as a DLTensor, from torch's DLPack exchange table
    (ABI version 1: version, previous table, then five functions, this one the fourth); 0 where there is none."""
    table = getattr(torch.Tensor, "__dlpack_c_exchange_api__", None)
    if table is None or object.__basicsize__ != 16 or not getattr(sys, "_is_gil_enabled", lambda: True)():
        return 0
    get = C.PyDLL(None).PyCapsule_GetPointer
    get.restype, get.argtypes = C.c_void_p, [C.py_object, C.c_char_p]
    at = get(table, b"dlpack_exchange_api")
    if C.c_uint32.from_address(at).value != 1:
        return 0
    return C.c_void_p.from_address(at + 5 * C.sizeof(C.c_void_p)).value or 0


_VIEW, _take, _python = _view(), form_take(), C.PyDLL(None)


def _form_of(*places):
    """A call's form and a reference to it: the tensors' addresses go to `places`."""
    f = Form()
    f.view, f.item = _VIEW, C.cast(_python.PyTuple_GetItem, C.c_void_p)
    f.type, f.none, f.n = id(torch.Tensor), id(None), len(places)
    for i, p in enumerate(places):
        f.to[i] = p
    return f, C.byref(f)


def _known(ref, tensors):
    """Whether the tensors have the form of the call before; then their addresses are set. What the view refuses (a
    tensor without storage, say) goes through the checks instead."""
    try:
        return _take(ref, 0, tensors)
    except (BufferError, RuntimeError):
        return 0


def _record(ref, tensors):
    """Records the form of tensors that have passed the checks, several microseconds of Python, for the next call."""
    if not _VIEW:
        return
    try:
        _take(ref, 1, tensors)
    except (BufferError, RuntimeError):
        pass


class BlockNorm:
    """Norms before and after a block, with its gate and residual scale (tsn_block_norm):
    ``x_out = r * x + act(gate) * Npost(y)``, ``h = Npre(x_out) * (1 + scale) + shift``.

    `post`, `pre`: "rms", "layer" or "none"; weights and biases float32 [C] or None; `residual_scale` a number
    or a float32 [C]; `gate_tanh` takes tanh of the gate."""

    def __init__(self, dev, C_: int, post: str = "rms", pre: str = "layer", post_weight=None, post_bias=None,
                 pre_weight=None, pre_bias=None, post_eps: float = 1e-6, pre_eps: float = 1e-6, residual_scale=1.0,
                 gate_tanh: bool = False):
        if post not in NORMS or pre not in NORMS:
            raise ValueError("post and pre must be 'rms', 'layer' or 'none'")
        self.dev, self.C = dev, C_
        vec = residual_scale if isinstance(residual_scale, torch.Tensor) else None
        self._keep = [_weights(dev, n, t, (C_,)) for n, t in (("post_weight", post_weight), ("post_bias", post_bias),
                                                         ("pre_weight", pre_weight), ("pre_bias", pre_bias),
                                                         ("residual_scale", vec))]
        a = BlockNormArgs()
        a.C, a.post, a.pre, a.gate_tanh = C_, NORMS[post], NORMS[pre], int(gate_tanh)
        a.post_eps, a.pre_eps, a.res_scale = post_eps, pre_eps, 1.0 if vec is not None else residual_scale
        a.post_w, a.post_b, a.pre_w, a.pre_b, a.res_vec = (_address(t) for t in self._keep)
        self._a, self._ref, self._call = a, C.byref(a), lib().tsn_block_norm
        self._views = a.x, a.y, a.gate, a.shift, a.scale, a.x_out, a.h
        self._form, self._formed = _form_of(*(C.addressof(v) for v in self._views))

    def __call__(self, x, y=None, gate=None, shift=None, scale=None, x_out=None, h=None):
        """x, x_out [B, T, C] of the residual's type; y, h [B, T, C] of the branch's type, which is the residual's or
        narrower than its float32; gate, shift, scale [B or 1, T or 1, C] of the branch's type, each or None.
        x_out may be x and h may be y."""
        tensors = x, y, gate, shift, scale, x_out, h
        if not _known(self._formed, tensors):
            self._check(*tensors)
            _record(self._formed, tensors)
            for view, t in zip(self._views, tensors):
                view.p = _address(t)
        rc = self._call(self.dev.h, self._ref)
        if rc:
            check(rc)

    def _check(self, x, y, gate, shift, scale, x_out, h):
        a = self._a
        _here(self.dev, ("x", x), ("y", y), ("gate", gate), ("shift", shift), ("scale", scale), ("x_out", x_out), ("h", h))
        shape = x.shape
        if len(shape) != 3 or shape[2] != self.C:
            raise ValueError(f"x must be [B, T, {self.C}], got {tuple(shape)}")
        typed = y if y is not None else h if h is not None else x
        dtype = typed.dtype
        if dtype not in TYPES or x.dtype not in TYPES:
            raise TypeError("float32, float16 or bfloat16 tensors are wanted")
        a.B, a.T, a.xtype, a.type = shape[0], shape[1], TYPES[x.dtype], TYPES[dtype]
        _put(a.x, "x", x)
        for name, t, of in (("y", y, dtype), ("x_out", x_out, x.dtype), ("h", h, dtype)):
            if t is not None:
                _want(name, t, shape, of)
                _put(getattr(a, name), name, t)
        for name, t in (("gate", gate), ("shift", shift), ("scale", scale)):
            if t is None:
                continue
            if t.dtype is not dtype:
                raise TypeError(f"{name} is {t.dtype}, expected {dtype}")
            ts = t.shape
            if len(ts) != 3 or ts[2] != self.C or ts[0] not in (1, shape[0]) or ts[1] not in (1, shape[1]):
                raise ValueError(f"{name} must be [B or 1, T or 1, {self.C}], got {tuple(ts)}")
            view = getattr(a, name)
            _put(view, name, t)
            if ts[0] == 1:
                view.sb = 0
            if ts[1] == 1:
                view.st = 0


class RopeAxes:
    """Rotary positions with 1 to 4 axes after an optional RMSNorm of each head (tsn_rope_axes).

    `pairs`: rotated pairs of each axis (2 * sum(pairs) <= head_dim; the rest passes through); `theta`: base, one
    or one per axis; `scale`: factor on the positions, one or one per axis; `layout`: "interleaved" (pair j is
    elements 2j, 2j + 1) or "half" (j, j + sum(pairs)); `q_norm`, `k_norm`: float32 [head_dim] or None."""

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
        self._keep = [_weights(dev, "q_norm", q_norm, (head_dim,)), _weights(dev, "k_norm", k_norm, (head_dim,))]
        a = RopeArgs()
        a.eps = eps
        a.q_norm, a.k_norm = (_address(t) for t in self._keep)
        self._a, self._ref, self._plan_ref = a, C.byref(a), C.byref(self._plan)
        self._call = lib().tsn_rope_axes
        self._views = a.q, a.k, a.q_out, a.k_out
        self._form, self._formed = _form_of(*(C.addressof(v) for v in self._views), C.addressof(a) + RopeArgs.pos.offset)

    def __call__(self, q, k, pos, q_out=None, k_out=None):
        """q [B, S, Hq, head_dim] and k [B, S, Hk, head_dim], either may be None; pos int32 [S, axes] or [B, S, axes].
        Results into q_out and k_out, or in place where those are None."""
        if q_out is None:
            q_out = q
        if k_out is None:
            k_out = k
        tensors = q, k, q_out, k_out, pos
        if not _known(self._formed, tensors):
            self._check(q, k, pos, q_out, k_out)
            _record(self._formed, tensors)
            for view, t in zip(self._views, tensors):
                view.p = _address(t)
            self._a.pos = pos.data_ptr()
        rc = self._call(self.dev.h, self._plan_ref, self._ref)
        if rc:
            check(rc)

    def _check(self, q, k, pos, q_out, k_out):
        a = self._a
        _here(self.dev, ("q", q), ("k", k), ("pos", pos), ("q_out", q_out), ("k_out", k_out))
        first = q if q is not None else k
        if first is None or first.dim() != 4:
            raise ValueError("q or k is wanted, [B, S, heads, head_dim]")
        B, S = first.shape[0], first.shape[1]
        dtype = first.dtype
        if dtype not in TYPES:
            raise TypeError("float32, float16 or bfloat16 tensors are wanted")
        a.B, a.S, a.type = B, S, TYPES[dtype]
        for name, t, out in (("q", q, q_out), ("k", k, k_out)):
            if t is None:
                continue
            if t.dim() != 4:
                raise ValueError(f"{name} must be [B, S, heads, head_dim]")
            H = t.shape[2]
            _want(name, t, (B, S, H, self.D), dtype)
            _want(name + "_out", out, t.shape, dtype)
            _put(getattr(a, name), name, t)
            _put(getattr(a, name + "_out"), name + "_out", out)
            if name == "q":
                a.Hq = H
            else:
                a.Hk = H
        ps = pos.shape
        if pos.dtype is not torch.int32 or ps[-2:] != (S, self.axes) or (len(ps) == 3 and ps[0] not in (1, B)) or len(ps) > 3:
            raise ValueError(f"pos must be int32 [S, {self.axes}] or [B, S, {self.axes}]")
        st = pos.stride()
        if st[-1] != 1 and self.axes > 1:
            raise ValueError("pos: the last dimension must be contiguous")
        a.pos_ss = st[-2]
        a.pos_sb = st[0] if len(ps) == 3 and ps[0] > 1 else 0


class DiffAttention:
    """Differential attention with its per-head RMSNorm (tsn_diff_attn):
    ``(softmax(q1 k1') - lambda softmax(q2 k2')) v``, normalised over 2 d and scaled by ``1 - lambda_init``.

    `lambda_q1` .. `lambda_k2`: float32 [d], shared by the heads, or [H, d]; `norm_weight`: float32 [2 d] or None."""

    def __init__(self, dev, d: int, lambda_q1, lambda_k1, lambda_q2, lambda_k2, lambda_init: float, norm_weight=None,
                 eps: float = 1e-5, scale: float | None = None):
        self.dev, self.d = dev, d
        vectors = (("lambda_q1", lambda_q1), ("lambda_k1", lambda_k1), ("lambda_q2", lambda_q2), ("lambda_k2", lambda_k2))
        shape = tuple(lambda_q1.shape)
        if shape[-1:] != (d,) or len(shape) > 2:
            raise ValueError(f"the lambda vectors must be [{d}] or [H, {d}]")
        self.heads = shape[0] if len(shape) == 2 else None
        self._keep = [_weights(dev, n, t, shape) for n, t in vectors] + [_weights(dev, "norm_weight", norm_weight, (2 * d,))]
        a = DiffAttnArgs()
        a.d, a.lambda_init, a.eps, a.scale = d, lambda_init, eps, 0.0 if scale is None else scale
        a.lq1, a.lk1, a.lq2, a.lk2, a.norm_w = (_address(t) for t in self._keep)
        a.lam_sh = d if self.heads else 0
        self._a, self._ref, self._call = a, C.byref(a), lib().tsn_diff_attn
        self._views = a.q, a.k, a.v, a.out
        self._form, self._formed = _form_of(*(C.addressof(v) for v in self._views), C.addressof(a) + DiffAttnArgs.key_len.offset,
                                            C.addressof(a) + DiffAttnArgs.key_mask.offset)

    def __call__(self, q, k, v, out, key_len=None, key_mask=None, causal: bool = False):
        """q, out [B, Sq, H, 2 d], k, v [B, Sk, Hk, 2 d], all float16 or bfloat16. key_len: int32 [B], the keys each
        sequence has; key_mask: uint8 or bool [B or 1, Sk], nonzero where a key is seen; causal: counted from the
        end, the last query sees the last key."""
        a = self._a
        tensors = q, k, v, out, key_len, key_mask
        if not _known(self._formed, tensors):
            self._check(*tensors)
            _record(self._formed, tensors)
            for view, t in zip(self._views, tensors):
                view.p = t.data_ptr()
            a.key_len, a.key_mask = _address(key_len), _address(key_mask)
        a.causal = 1 if causal else 0
        rc = self._call(self.dev.h, self._ref)
        if rc:
            check(rc)

    def _check(self, q, k, v, out, key_len, key_mask):
        a = self._a
        _here(self.dev, ("q", q), ("k", k), ("v", v), ("out", out), ("key_len", key_len), ("key_mask", key_mask))
        if q.dim() != 4 or k.dim() != 4:
            raise ValueError("q and k must be [B, S, heads, 2 d]")
        B, Sq, H, D = q.shape
        Sk, Hk = k.shape[1], k.shape[2]
        dtype = q.dtype
        if D != 2 * self.d:
            raise ValueError(f"q must be [B, Sq, H, {2 * self.d}]")
        if dtype not in TYPES:
            raise TypeError("float16 or bfloat16 tensors are wanted")
        if self.heads and H != self.heads:
            raise ValueError(f"the lambda vectors are of {self.heads} heads, q has {H}")
        _want("k", k, (B, Sk, Hk, D), dtype)
        _want("v", v, (B, Sk, Hk, D), dtype)
        _want("out", out, q.shape, dtype)
        a.B, a.Sq, a.Sk, a.H, a.Hk, a.type = B, Sq, Sk, H, Hk, TYPES[dtype]
        for name, t in (("q", q), ("k", k), ("v", v), ("out", out)):
            _put(getattr(a, name), name, t)
        if key_len is not None and (key_len.dtype is not torch.int32 or tuple(key_len.shape) != (B,)
                                    or not key_len.is_contiguous()):
            raise ValueError("key_len must be a contiguous int32 tensor of shape [B]")
        if key_mask is not None:
            ms = key_mask.shape
            if key_mask.dtype not in (torch.uint8, torch.bool) or len(ms) != 2 or ms[1] != Sk or ms[0] not in (1, B):
                raise ValueError("key_mask must be uint8 or bool [B or 1, Sk]")
            if key_mask.stride(1) != 1 and Sk > 1:
                raise ValueError("key_mask: the last dimension must be contiguous")
            a.mask_sb = key_mask.stride(0) if ms[0] > 1 else 0
