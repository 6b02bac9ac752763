"""Layers along an axis and their training step, on arrays of the b200 backend.

* :func:`linear_recurrence` / :func:`linear_recurrence_backward` -- the gated
  linear recurrence ``h_t = alpha_t h_{t-1} + u_t`` along an axis, from one step
  with a kept state (serving) to long sequences, and its gradients;
* :func:`group_norm` / :func:`group_norm_backward` -- group norm with an
  activation, channels last, and its gradients (layer norm is one group);
* :class:`AdamW` -- the optimizer step over many tensors in one call, and
  :func:`adamw_step`, the same on lists that the caller keeps.

OpenPacho has none of these (its reductions, src/openpacho/_reductions.py, and
its norm, src/openpacho/_norm.py, are the nearest).  Arrays are anything with
the backend protocol's ``shape``/``dtype``/``_data`` (OpenPacho arrays on the
b200 backend, :class:`~pacho_b200.backend.DeviceArray`,
``B200Backend.view`` of another library's array); float32 or float64, one dtype
in a call; results come back as the same kind.  ``out`` names arrays to write
into instead of new ones: with it a call allocates nothing, as
``B200Backend.capture`` needs.  An output must not share memory with an input
or another output, except ``final`` with ``state``.
"""

from __future__ import annotations

import ctypes as C
from array import array
from math import prod
from operator import index

import numpy as np

from . import _lib
from . import exceptions as _exc
from .backend import B200Backend, wrap_like

_FLOATS = {np.dtype(np.float32): _lib.PB_F32, np.dtype(np.float64): _lib.PB_F64}


def _context(x, what):
    """(backend, dtype, dtype code) of a call's first operand."""
    try:
        backend, dtype = x._data.backend, x.dtype
    except AttributeError:
        backend = None
    if not isinstance(backend, B200Backend):
        raise TypeError(f"{what} takes arrays of the b200 backend, not {type(x).__name__}")
    code = _FLOATS.get(dtype)
    if code is None:
        raise _exc.UnsupportedDtypeError(f"{what} requires float32 or float64, not {dtype}")
    return backend, dtype, code


def _stranger(name, x):
    return TypeError(f"{name} is no array of the b200 backend: {type(x).__name__}")


def _pointer(name, x, shape, dtype, backend):
    """The device pointer of an operand that has to have this shape and dtype
    (None for an operand that is not there)."""
    if x is None:
        return None
    # The usual case in three comparisons: a call's time on the host is what its
    # smallest sizes take.
    try:
        data = x._data
        if data.backend is backend and x.shape == shape and (x.dtype is dtype or x.dtype == dtype) and data.ptr:
            return data.ptr
    except AttributeError:
        raise _stranger(name, x) from None
    if data.backend is not backend:
        raise _exc.BackendMismatchError(f"{name} belongs to another backend")
    if tuple(x.shape) != shape:
        raise ValueError(f"{name} has shape {tuple(x.shape)}, expected {shape}")
    if x.dtype != dtype:
        raise ValueError(f"{name} has dtype {x.dtype}, expected {dtype}")
    # To the C entries a null pointer is an operand that is not there.
    if not data.ptr and prod(shape):
        raise ValueError(f"the memory of {name} has been released")
    return data.ptr


def _output(name, given, shape, dtype, backend, template):
    """``given`` checked, or a new array like ``template``: (array, pointer)."""
    if given is not None:
        return given, _pointer(name, given, shape, dtype, backend)
    data = backend.empty(shape, dtype)
    return wrap_like(template, data, shape, dtype, backend), data.ptr


def _outputs(out, count, what):
    if out is None:
        return (None,) * count
    if not isinstance(out, (tuple, list)) or len(out) != count:
        raise ValueError(f"out of {what} is a tuple of {count} arrays")
    return out


def _choice(what, choices, value):
    try:
        return choices[value]
    except (KeyError, TypeError):
        raise ValueError(f"unknown {what} {value!r}: {', '.join(map(repr, choices))}") from None


def _axis_view(shape, axis, what):
    """(outer, length, inner, shape without the axis)."""
    ndim = len(shape)
    if ndim == 3 and (axis == -2 or axis == 1):
        return shape[0], shape[1], shape[2], (shape[0], shape[2])
    if not -ndim <= axis < ndim:
        raise ValueError(f"{what}: axis {axis} is out of range for {ndim} dimensions")
    axis %= ndim
    before, after = shape[:axis], shape[axis + 1:]
    return prod(before), shape[axis], prod(after), before + after


def linear_recurrence(a, b, *, state=None, gate="linear", axis=-2, out=None, final=None):
    """``h_t = alpha_t * h_{t-1} + u_t`` along ``axis``, elementwise over the
    other dimensions, from ``h_{-1} = state`` (zeros without one).

    ``gate="linear"``: alpha = a, u = b.  ``gate="sigmoid"``: ``a`` holds logits,
    alpha = sigmoid(a), u = (1 - alpha) * b.  The default axis is the sequence of
    ``(..., sequence, channels)`` arrays.  ``state`` has the shape of ``b``
    without the axis; ``final``, an array of that shape, receives the last h
    and may be ``state`` itself, which serving a stream step by step does.
    Returns h (``out`` if given)."""
    backend, dtype, code = _context(a, "linear_recurrence")
    shape = tuple(a.shape)
    mode = _choice("gate", _lib.GATES, gate)
    outer, length, inner, rest = _axis_view(shape, axis, "linear_recurrence")
    pa = a._data.ptr
    pb = _pointer("b", b, shape, dtype, backend)
    ps = _pointer("state", state, rest, dtype, backend)
    pf = _pointer("final", final, rest, dtype, backend)
    with backend._lock:
        backend._require_open()
        h, ph = _output("out", out, shape, dtype, backend, a)
        status = backend._lib.pb_recurrence(backend._ctx, 0, code, mode, outer, length, inner, pa, pb, ps, ph, pf)
        if status:
            backend._check(status, "pb_recurrence")
    return h


def linear_recurrence_backward(a, b, h, dh, *, state=None, dfinal=None, gate="linear", axis=-2, out=None):
    """Gradients ``(da, db, dstate)`` of :func:`linear_recurrence` at the same
    ``a``, ``b`` and ``state``, given its result ``h``, the gradient ``dh`` of it
    and, where ``final`` was used, the gradient ``dfinal`` of that.  ``b`` may be
    None with ``gate="linear"``, whose gradients do not depend on it."""
    backend, dtype, code = _context(a, "linear_recurrence_backward")
    shape = tuple(a.shape)
    mode = _choice("gate", _lib.GATES, gate)
    outer, length, inner, rest = _axis_view(shape, axis, "linear_recurrence_backward")
    if b is None and mode != _lib.GATES["linear"]:
        raise ValueError(f"the gradients of gate={gate!r} need b")
    pa = a._data.ptr
    pb = _pointer("b", b, shape, dtype, backend)
    ph = _pointer("h", h, shape, dtype, backend)
    pg = _pointer("dh", dh, shape, dtype, backend)
    ps = _pointer("state", state, rest, dtype, backend)
    pf = _pointer("dfinal", dfinal, rest, dtype, backend)
    da, db, ds = _outputs(out, 3, "linear_recurrence_backward")
    with backend._lock:
        backend._require_open()
        da, pda = _output("da", da, shape, dtype, backend, a)
        db, pdb = _output("db", db, shape, dtype, backend, a)
        ds, pds = _output("dstate", ds, rest, dtype, backend, a)
        status = backend._lib.pb_recurrence_backward(backend._ctx, 0, code, mode, outer, length, inner, pa, pb, ph,
                                                     pg, ps, pf, pda, pdb, pds)
        if status:
            backend._check(status, "pb_recurrence_backward")
    return da, db, ds


def _norm_view(x, groups, what):
    """(N, S, C, groups) of a channels-last array ``(N, ..., C)``."""
    shape = tuple(x.shape)
    if len(shape) < 2:
        raise ValueError(f"{what} takes (N, ..., C) arrays, channels last")
    groups = index(groups)
    if groups < 1 or shape[-1] % groups:
        raise ValueError(f"{what}: {shape[-1]} channels do not divide into {groups} groups")
    return shape[0], shape[1] if len(shape) == 3 else prod(shape[1:-1]), shape[-1], groups


def group_norm(x, groups, weight=None, bias=None, *, eps=1e-5, activation=None, out=None):
    """``act((x - mean) * rstd * weight + bias)`` of a channels-last array
    ``(N, ..., C)``, with the mean and ``rstd = 1/sqrt(var + eps)`` of each sample's
    each group of ``C / groups`` channels over all positions.

    ``activation``: None, ``"relu"``, ``"silu"`` or ``"gelu"`` (the exact one).
    ``groups=1`` on ``(N, C)`` is a layer norm, and per-token head norms are
    ``(tokens, C)`` with a group per head.  Returns ``(y, mean, rstd)``, the
    statistics ``(N, groups)`` for the backward pass; ``out`` takes the three."""
    backend, dtype, code = _context(x, "group_norm")
    act = _choice("activation", _lib.ACTIVATIONS, activation)
    n, s, c, groups = _norm_view(x, groups, "group_norm")
    shape = tuple(x.shape)
    px = x._data.ptr
    pw = _pointer("weight", weight, (c,), dtype, backend)
    pb = _pointer("bias", bias, (c,), dtype, backend)
    y, mean, rstd = _outputs(out, 3, "group_norm")
    with backend._lock:
        backend._require_open()
        y, py = _output("y", y, shape, dtype, backend, x)
        mean, pm = _output("mean", mean, (n, groups), dtype, backend, x)
        rstd, pr = _output("rstd", rstd, (n, groups), dtype, backend, x)
        status = backend._lib.pb_group_norm(backend._ctx, 0, code, act, n, s, c, groups, float(eps), px, pw, pb,
                                            py, pm, pr)
        if status:
            backend._check(status, "pb_group_norm")
    return y, mean, rstd


def group_norm_backward(dy, x, groups, mean, rstd, weight=None, bias=None, *, activation=None, out=None):
    """Gradients ``(dx, dweight, dbias)`` of :func:`group_norm` at the same
    ``x``, ``weight``, ``bias`` and activation, with the ``mean`` and ``rstd`` it
    returned.  ``dweight`` is None without a weight, ``dbias`` without a bias."""
    backend, dtype, code = _context(x, "group_norm_backward")
    act = _choice("activation", _lib.ACTIVATIONS, activation)
    n, s, c, groups = _norm_view(x, groups, "group_norm_backward")
    shape = tuple(x.shape)
    px = x._data.ptr
    pd = _pointer("dy", dy, shape, dtype, backend)
    pm = _pointer("mean", mean, (n, groups), dtype, backend)
    pr = _pointer("rstd", rstd, (n, groups), dtype, backend)
    pw = _pointer("weight", weight, (c,), dtype, backend)
    pb = _pointer("bias", bias, (c,), dtype, backend)
    dx, dweight, dbias = _outputs(out, 3, "group_norm_backward")
    if (weight is None and dweight is not None) or (bias is None and dbias is not None):
        raise ValueError("group_norm_backward has no gradient of a weight or bias that is not there")
    with backend._lock:
        backend._require_open()
        dx, pdx = _output("dx", dx, shape, dtype, backend, x)
        pdw = pdb = None
        if weight is not None:
            dweight, pdw = _output("dweight", dweight, (c,), dtype, backend, x)
        if bias is not None:
            dbias, pdb = _output("dbias", dbias, (c,), dtype, backend, x)
        status = backend._lib.pb_group_norm_backward(backend._ctx, 0, code, act, n, s, c, groups, pd, px, pm, pr, pw,
                                                     pb, pdx, pdw, pdb)
        if status:
            backend._check(status, "pb_group_norm_backward")
    return dx, dweight, dbias


def _table(name, arrays, shapes, dtype, backend):
    """The host table of device pointers of one list, an array for each shape."""
    if len(arrays) != len(shapes):
        raise ValueError(f"{name}: {len(arrays)} arrays for {len(shapes)} parameters")
    try:
        pointers = [x._data.ptr for x, s in zip(arrays, shapes)
                    if x._data.backend is backend and x.dtype is dtype and x.shape == s and x._data.ptr]
    except AttributeError:
        raise _stranger(name, next((x for x in arrays if not hasattr(getattr(x, "_data", None), "backend")),
                                   arrays)) from None
    if len(pointers) != len(arrays):  # one is not quite so: checked one by one
        pointers = [_pointer(name, x, s, dtype, backend) or 0 for x, s in zip(arrays, shapes)]
    # Through an array of integers: ctypes takes four times as long for each item.
    return (C.c_void_p * len(pointers)).from_buffer(array("Q", pointers))


def _sizes(shapes):
    return (C.c_int64 * len(shapes))(*[prod(s) for s in shapes])


def _two(betas):
    betas = tuple(float(v) for v in betas)
    if len(betas) != 2:
        raise ValueError("betas are two numbers")
    return betas


def _adamw(backend, dtype, code, tables, sizes, grad_scale, lr, betas, eps, weight_decay, step):
    """One step over host tables of parameters, gradients and the two moments."""
    scale = None
    if grad_scale is not None:
        shape = getattr(grad_scale, "shape", None)
        if shape is None:
            raise _stranger("grad_scale", grad_scale)
        if prod(shape) != 1:
            raise ValueError("grad_scale has one element")
        scale = _pointer("grad_scale", grad_scale, tuple(shape), dtype, backend)
    with backend._lock:
        backend._require_open()
        status = backend._lib.pb_adamw(backend._ctx, 0, code, len(sizes), *tables, sizes, float(lr), *betas,
                                       float(eps), float(weight_decay), step, scale)
        if status:
            backend._check(status, "pb_adamw")


def adamw_step(params, grads, exp_avg, exp_avg_sq, *, step, lr=1e-3, betas=(0.9, 0.999), eps=1e-8,
               weight_decay=0.01, grad_scale=None):
    """One AdamW step with decoupled weight decay over lists of arrays, in place and
    in one call: parameters, their gradients and the two moments, each list with
    an array of the parameter's shape and dtype for each parameter.

    ``step`` counts from 1 and is the caller's to keep; :class:`AdamW` keeps it and
    the moments.  ``grad_scale``, a one-element array on the GPU, multiplies every
    gradient (a clipping coefficient, the inverse of a loss scale) without a copy to
    the host."""
    params = list(params)
    if not params:
        raise ValueError("adamw_step needs at least one parameter")
    backend, dtype, code = _context(params[0], "adamw_step")
    shapes = [tuple(p.shape) for p in params]
    tables = [_table(name, arrays, shapes, dtype, backend) for name, arrays in
              (("params", params), ("grads", grads), ("exp_avg", exp_avg), ("exp_avg_sq", exp_avg_sq))]
    _adamw(backend, dtype, code, tables, _sizes(shapes), grad_scale, lr, _two(betas), eps, weight_decay, index(step))


class AdamW:
    """AdamW with decoupled weight decay over a list of parameter arrays, which
    :meth:`step` updates in place, all tensors in one call.

    The two moments are arrays of the parameters' dtype: new zeros, or the
    lists given as ``exp_avg`` and ``exp_avg_sq`` (to resume; with ``steps`` the
    number of steps already taken).  ``lr`` and ``weight_decay`` may be changed
    between steps.  The parameters' and moments' memory must stay the same: a step
    after one of them was released or replaced is refused."""

    def __init__(self, params, *, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01,
                 exp_avg=None, exp_avg_sq=None, steps=0):
        self.params = list(params)
        if not self.params:
            raise ValueError("AdamW needs at least one parameter")
        self._backend, self._dtype, self._code = _context(self.params[0], "AdamW")
        self.lr, self.eps, self.weight_decay = float(lr), float(eps), float(weight_decay)
        self.betas = _two(betas)
        self.steps = int(steps)
        self._shapes = [tuple(p.shape) for p in self.params]
        p = self._table("params", self.params)
        self.exp_avg = self._moment("exp_avg", exp_avg)
        self.exp_avg_sq = self._moment("exp_avg_sq", exp_avg_sq)
        self._tables = p, self._table("exp_avg", self.exp_avg), self._table("exp_avg_sq", self.exp_avg_sq)
        self._known = [[x._data.ptr for x in q] for q in (self.params, self.exp_avg, self.exp_avg_sq)]
        self._sizes = _sizes(self._shapes)

    def _moment(self, name, given):
        if given is not None:
            return list(given)
        b = self._backend
        return [wrap_like(p, b.full(s, 0.0, self._dtype), s, self._dtype, b)
                for p, s in zip(self.params, self._shapes)]

    def _table(self, name, arrays):
        return _table(name, arrays, self._shapes, self._dtype, self._backend)

    def step(self, grads, *, grad_scale=None):
        """One step with a gradient array per parameter (shape and dtype of
        the parameter) and ``grad_scale`` as of :func:`adamw_step`."""
        # One step at a time, its number with it: threads that share an optimizer.
        with self._backend._lock:
            for arrays, known in zip((self.params, self.exp_avg, self.exp_avg_sq), self._known):
                if [x._data.ptr for x in arrays] != known:
                    raise ValueError("the memory of a parameter or moment has been released or replaced")
            p, m, v = self._tables
            _adamw(self._backend, self._dtype, self._code, (p, self._table("grads", grads), m, v), self._sizes,
                   grad_scale, self.lr, self.betas, self.eps, self.weight_decay, self.steps + 1)
            self.steps += 1


__all__ = [
    "AdamW",
    "adamw_step",
    "group_norm",
    "group_norm_backward",
    "linear_recurrence",
    "linear_recurrence_backward",
]
