"""Host side of the layer operators, on CPU with a recording library: the view
each call passes on, its checks of arguments, and that the reference formulas
used by the GPU tests are the derivatives of the forward ones."""

from __future__ import annotations

import ast
import ctypes as C
import pathlib
import threading
import time
import weakref

import numpy as np
import pytest

import layer_reference as ref
import pacho_b200 as pb
from pacho_b200 import _lib
from pacho_b200.backend import B200Backend, DeviceArray
from test_host_logic import RecordingLib


def _backend():
    b = object.__new__(B200Backend)
    b._lib, b._ctx, b._lock, b._closed = RecordingLib(), C.c_void_p(1), threading.RLock(), False
    b._buffers = weakref.WeakSet()
    return b


@pytest.fixture
def backend():
    b = _backend()
    yield b
    b._closed = True


def _arr(backend, *shape, dtype=np.float32):
    return DeviceArray(backend, backend.empty(shape, dtype), shape, dtype)


def _call(backend, name):
    (args,) = [a for n, a in backend._lib.calls if n == name]
    return args


@pytest.mark.parametrize("shape,axis,view", [
    ((4, 7, 5), -2, (4, 7, 5)), ((4, 7, 5), 1, (4, 7, 5)), ((4, 7, 5), 0, (1, 4, 35)),
    ((4, 7, 5), -1, (28, 5, 1)), ((7, 5), -2, (1, 7, 5)), ((2, 3, 7, 5), 2, (6, 7, 5)), ((9,), 0, (1, 9, 1)),
    ((4, 0, 5), 1, (4, 0, 5))])
def test_recurrence_passes_the_axis_view(backend, shape, axis, view):
    a, b = _arr(backend, *shape), _arr(backend, *shape)
    rest = tuple(d for i, d in enumerate(shape) if i != axis % len(shape))
    state = _arr(backend, *rest)
    h = pb.linear_recurrence(a, b, state=state, final=state, gate="sigmoid", axis=axis)
    args = _call(backend, "pb_recurrence")
    assert args[2:7] == (_lib.PB_F32, 1) + view
    assert args[7:] == (a._data.ptr, b._data.ptr, state._data.ptr, h._data.ptr, state._data.ptr)
    da, db, ds = pb.linear_recurrence_backward(a, b, h, b, state=state, gate="sigmoid", axis=axis)
    assert _call(backend, "pb_recurrence_backward")[4:7] == view
    assert da.shape == db.shape == shape and ds.shape == rest


def test_recurrence_without_state_passes_nulls_and_uses_out(backend):
    a, b, out = (_arr(backend, 2, 3, 4, dtype=np.float64) for _ in range(3))
    before = backend._lib.next_ptr
    assert pb.linear_recurrence(a, b, out=out) is out
    assert backend._lib.next_ptr == before  # nothing was allocated
    args = _call(backend, "pb_recurrence")
    assert args[2] == _lib.PB_F64 and args[9] is None and args[11] is None and args[10] == out._data.ptr
    pb.linear_recurrence_backward(a, None, b, out)
    assert _call(backend, "pb_recurrence_backward")[8] is None


@pytest.mark.parametrize("call,error", [
    (lambda b, a: pb.linear_recurrence(a, _arr(b, 2, 3, 5)), ValueError),
    (lambda b, a: pb.linear_recurrence(a, _arr(b, 2, 3, 4, dtype=np.float64)), ValueError),
    (lambda b, a: pb.linear_recurrence(a, a, state=_arr(b, 2, 3)), ValueError),
    (lambda b, a: pb.linear_recurrence(a, a, final=_arr(b, 3, 4)), ValueError),
    (lambda b, a: pb.linear_recurrence(a, a, out=_arr(b, 2, 3, 5)), ValueError),
    (lambda b, a: pb.linear_recurrence(a, a, axis=3), ValueError),
    (lambda b, a: pb.linear_recurrence(a, a, axis=-4), ValueError),
    (lambda b, a: pb.linear_recurrence(a, a, gate="tanh"), ValueError),
    (lambda b, a: pb.linear_recurrence(a, a, gate=["linear"]), ValueError),
    (lambda b, a: pb.linear_recurrence(_arr(b, 2, 3, 4, dtype=np.bool_), a), TypeError),
    (lambda b, a: pb.linear_recurrence(np.zeros((2, 3, 4), np.float32), a), TypeError),
    (lambda b, a: pb.linear_recurrence(a, _arr(_backend(), 2, 3, 4)), pb.BackendMismatchError),
    (lambda b, a: pb.linear_recurrence_backward(a, None, a, a, gate="sigmoid"), ValueError),
    (lambda b, a: pb.linear_recurrence_backward(a, a, a, a, out=(a, a)), ValueError),
    (lambda b, a: pb.linear_recurrence_backward(a, a, a, a, dfinal=a), ValueError),
    (lambda b, a: pb.group_norm(a, 3), ValueError),
    (lambda b, a: pb.group_norm(a, 0), ValueError),
    (lambda b, a: pb.group_norm(_arr(b, 4), 1), ValueError),
    (lambda b, a: pb.group_norm(a, 2, activation="tanh"), ValueError),
    (lambda b, a: pb.group_norm(a, 2, _arr(b, 3)), ValueError),
    (lambda b, a: pb.group_norm(a, 2, None, _arr(b, 1, 4)), ValueError),
    (lambda b, a: pb.group_norm(a, 2, out=a), ValueError),
    (lambda b, a: pb.group_norm(a, 2, out=(None, _arr(b, 4), None)), ValueError),
    (lambda b, a: pb.group_norm_backward(a, a, 2, _arr(b, 2, 1), _arr(b, 2, 2)), ValueError),
    (lambda b, a: pb.group_norm_backward(a, a, 2, _arr(b, 2, 2), _arr(b, 2, 2), out=(None, _arr(b, 4), None)),
     ValueError),
    (lambda b, a: pb.AdamW([]), ValueError),
    (lambda b, a: pb.AdamW([a, _arr(b, 3, dtype=np.float64)]), ValueError),
    (lambda b, a: pb.AdamW([a], betas=(0.9,)), ValueError),
    (lambda b, a: pb.AdamW([a], exp_avg=[]), ValueError),
    (lambda b, a: pb.AdamW([a]).step([]), ValueError),
    (lambda b, a: pb.AdamW([a]).step([_arr(b, 2, 3, 5)]), ValueError),
    (lambda b, a: pb.AdamW([a]).step([a], grad_scale=a), ValueError),
    (lambda b, a: pb.AdamW([a]).step([_arr(_backend(), 2, 3, 4)]), pb.BackendMismatchError),
])
def test_refused_arguments_reach_no_kernel(backend, call, error):
    with pytest.raises(error):
        call(backend, _arr(backend, 2, 3, 4))
    assert not [n for n, _ in backend._lib.calls if n in (
        "pb_recurrence", "pb_recurrence_backward", "pb_group_norm", "pb_group_norm_backward", "pb_adamw")]


class _HostArray:
    """An array of another backend, its data a NumPy array."""

    def __init__(self, *shape):
        self._data = np.zeros(shape, np.float32)
        self.shape, self.dtype = shape, self._data.dtype


@pytest.mark.parametrize("make", [lambda *s: np.zeros(s, np.float32), _HostArray])
@pytest.mark.parametrize("call", [
    lambda a, o: pb.linear_recurrence(o(2, 3, 4), a),
    lambda a, o: pb.linear_recurrence(a, o(2, 3, 4)),
    lambda a, o: pb.linear_recurrence(a, a, state=o(2, 4)),
    lambda a, o: pb.linear_recurrence(a, a, out=o(2, 3, 4)),
    lambda a, o: pb.linear_recurrence_backward(a, a, a, o(2, 3, 4)),
    lambda a, o: pb.group_norm(a, 2, o(4)),
    lambda a, o: pb.group_norm(a, 2, out=(o(2, 3, 4), None, None)),
    lambda a, o: pb.group_norm_backward(o(2, 3, 4), a, 2, a, a),
    lambda a, o: pb.AdamW([a, o(4)]),
    lambda a, o: pb.AdamW([a], exp_avg=[o(2, 3, 4)]),
    lambda a, o: pb.AdamW([a]).step([o(2, 3, 4)]),
    lambda a, o: pb.AdamW([a]).step([None]),
    lambda a, o: pb.AdamW([a]).step([a], grad_scale=o(1)),
    lambda a, o: pb.AdamW([a]).step([a], grad_scale=0.5),
    lambda a, o: pb.adamw_step([a], [o(2, 3, 4)], [a], [a], step=1),
])
def test_arrays_of_other_kinds_are_a_type_error(backend, call, make):
    with pytest.raises(TypeError, match="b200 backend"):
        call(_arr(backend, 2, 3, 4), make)


def test_a_closed_backend_is_refused(backend):
    a = _arr(backend, 2, 3, 4)
    opt = pb.AdamW([a])
    backend._closed = True
    for call in (lambda: pb.linear_recurrence(a, a), lambda: pb.group_norm(a, 2), lambda: opt.step([a])):
        with pytest.raises(RuntimeError):
            call()


def _released(backend, *shape):
    x = _arr(backend, *shape)
    x._data.release()
    return x


@pytest.mark.parametrize("call", [
    lambda b, a: pb.linear_recurrence(a, a, state=_released(b, 2, 4)),
    lambda b, a: pb.linear_recurrence(a, a, final=_released(b, 2, 4)),
    lambda b, a: pb.linear_recurrence(a, a, out=_released(b, 2, 3, 4)),
    lambda b, a: pb.linear_recurrence_backward(a, _released(b, 2, 3, 4), a, a),
    lambda b, a: pb.linear_recurrence_backward(a, a, a, a, dfinal=_released(b, 2, 4)),
    lambda b, a: pb.group_norm(a, 2, _released(b, 4)),
    lambda b, a: pb.group_norm(a, 2, None, _released(b, 4)),
    lambda b, a: pb.group_norm(a, 2, out=(None, None, _released(b, 2, 2))),
    lambda b, a: pb.group_norm_backward(a, a, 2, *(_arr(b, 2, 2) for _ in range(2)), _arr(b, 4),
                                        out=(None, _released(b, 4), None)),
    lambda b, a: pb.AdamW([a, _released(b, 3)]),
    lambda b, a: pb.AdamW([a]).step([_released(b, 2, 3, 4)]),
    lambda b, a: pb.AdamW([a]).step([a], grad_scale=_released(b, 1)),
])
def test_a_released_operand_is_not_taken_for_an_absent_one(backend, call):
    a = _arr(backend, 2, 3, 4)
    backend._lib.pb_free = lambda *args: 0
    with pytest.raises(ValueError, match="released"):
        call(backend, a)


@pytest.mark.parametrize("which", ["params", "exp_avg", "exp_avg_sq"])
def test_adamw_refuses_memory_that_was_released_or_replaced(backend, which):
    backend._lib.pb_free = lambda *args: 0
    for change in (lambda opt: getattr(opt, which)[1]._data.release(),
                   lambda opt: getattr(opt, which).__setitem__(1, _arr(backend, 5)),
                   lambda opt: getattr(opt, which).pop()):
        ps = [_arr(backend, 3, 4), _arr(backend, 5), _arr(backend, 0)]
        opt = pb.AdamW(ps)
        gs = [_arr(backend, *p.shape) for p in ps]
        opt.step(gs)
        change(opt)
        with pytest.raises(ValueError, match="released or replaced"):
            opt.step(gs)
        assert opt.steps == 1


def test_group_norm_takes_whole_groups_only(backend):
    with pytest.raises(TypeError):
        pb.group_norm(_arr(backend, 2, 3, 4), 2.5)
    pb.group_norm(_arr(backend, 2, 3, 4), np.int64(2))


def test_group_norm_views_and_outputs(backend):
    x, w = _arr(backend, 3, 5, 7, 8), _arr(backend, 8)
    y, mean, rstd = pb.group_norm(x, 4, w, activation="silu", eps=1e-3)
    args = _call(backend, "pb_group_norm")
    assert args[2:9] == (_lib.PB_F32, 2, 3, 35, 8, 4, 1e-3)
    assert args[9:] == (x._data.ptr, w._data.ptr, None, y._data.ptr, mean._data.ptr, rstd._data.ptr)
    assert y.shape == x.shape and mean.shape == rstd.shape == (3, 4)
    dx, dw, db = pb.group_norm_backward(y, x, 4, mean, rstd, w, activation="silu")
    assert dx.shape == x.shape and dw.shape == (8,) and db is None
    assert _call(backend, "pb_group_norm_backward")[4:8] == (3, 35, 8, 4)
    rows = _arr(backend, 6, 8)
    pb.group_norm(rows, 1)
    assert backend._lib.calls[-1][1][4:8] == (6, 1, 8, 1)


class _FrontArray:
    """An array of a front end that wraps a backend's buffers, as OpenPacho's does
    (src/openpacho/_array.py:43-51)."""

    @classmethod
    def _wrap(cls, data, shape, dtype, backend):
        x = cls()
        x._data, x.shape, x.dtype, x._backend = data, shape, dtype, backend
        return x


def test_arrays_of_the_front_end_are_taken_and_returned(backend):
    def arr(*shape):
        return _FrontArray._wrap(backend.empty(shape, np.float32), shape, np.dtype(np.float32), backend)

    a, w = arr(2, 3, 4), arr(4)
    h = pb.linear_recurrence(a, a, state=arr(2, 4), gate="sigmoid")
    y, mean, rstd = pb.group_norm(h, 2, w, w)
    grads = pb.group_norm_backward(y, h, 2, mean, rstd, w, w)
    more = pb.linear_recurrence_backward(a, a, h, grads[0], gate="sigmoid")
    opt = pb.AdamW([w])
    opt.step([grads[1]])
    pb.adamw_step([w], [grads[1]], opt.exp_avg, opt.exp_avg_sq, step=2)
    shapes = [x.shape for x in (h, y, mean, rstd, *grads, *more, *opt.exp_avg)]
    assert shapes == [(2, 3, 4)] * 2 + [(2, 2)] * 2 + [(2, 3, 4), (4,), (4,)] + [(2, 3, 4)] * 2 + [(2, 4), (4,)]
    assert all(type(x) is _FrontArray for x in (h, y, mean, rstd, *grads, *more, *opt.exp_avg))


def test_adamw_tables_and_step_count(backend):
    ps = [_arr(backend, 3, 4), _arr(backend, 5), _arr(backend, 0, 2)]
    opt = pb.AdamW(ps, lr=0.1, betas=(0.8, 0.95), eps=1e-6, weight_decay=0.2)
    assert [n for n, _ in backend._lib.calls if n == "pb_fill"] == ["pb_fill"] * 4  # moments of the two that hold values
    gs = [_arr(backend, *p.shape) for p in ps]
    scale = _arr(backend, 1)
    opt.step(gs)
    opt.lr = 0.05
    opt.step(gs, grad_scale=scale)
    first, second = [a for n, a in backend._lib.calls if n == "pb_adamw"]
    assert first[3] == 3 and [first[8][i] for i in range(3)] == [12, 5, 0]
    assert [first[4][i] for i in range(3)] == [p._data.ptr for p in ps]
    assert [first[5][i] for i in range(3)] == [g._data.ptr for g in gs]
    assert first[9:] == (0.1, 0.8, 0.95, 1e-6, 0.2, 1, None)
    assert second[9:] == (0.05, 0.8, 0.95, 1e-6, 0.2, 2, scale._data.ptr)


def test_adamw_steps_of_two_threads_have_numbers_of_their_own(backend):
    p, g = _arr(backend, 4), _arr(backend, 4)
    opt = pb.AdamW([p])
    steps, both = [], threading.Barrier(2)

    def slow(*args):
        steps.append(args[14])
        time.sleep(0.05)
        return 0

    backend._lib.pb_adamw = slow

    def work():
        both.wait()
        for _ in range(3):
            opt.step([g])

    threads = [threading.Thread(target=work) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert steps == [1, 2, 3, 4, 5, 6] and opt.steps == 6


def test_adamw_step_on_the_callers_lists(backend):
    ps = [_arr(backend, 3, 4), _arr(backend, 5), _arr(backend, 0, 2)]
    gs, m, v = ([_arr(backend, *p.shape) for p in ps] for _ in range(3))
    scale = _arr(backend, 1)
    before = backend._lib.next_ptr
    pb.adamw_step(ps, gs, m, v, step=7, lr=0.1, betas=(0.8, 0.95), eps=1e-6, weight_decay=0.2, grad_scale=scale)
    assert backend._lib.next_ptr == before  # nothing was allocated
    args = _call(backend, "pb_adamw")
    assert args[2:4] == (_lib.PB_F32, 3) and [args[8][i] for i in range(3)] == [12, 5, 0]
    for table, arrays in zip(args[4:8], (ps, gs, m, v)):
        assert [table[i] for i in range(3)] == [x._data.ptr for x in arrays]
    assert args[9:] == (0.1, 0.8, 0.95, 1e-6, 0.2, 7, scale._data.ptr)


@pytest.mark.parametrize("change,error", [
    (dict(params=[]), ValueError), (dict(grads=[]), ValueError), (dict(exp_avg_sq=[None, None]), ValueError),
    (dict(step=1.5), TypeError), (dict(betas=(0.9,)), ValueError), (dict(grads=lambda b: [_arr(b, 5)]), ValueError),
    (dict(exp_avg=lambda b: [_arr(b, 4, dtype=np.float64)]), ValueError),
    (dict(exp_avg=lambda b: [_released(b, 4)]), ValueError),
    (dict(exp_avg=lambda b: [_arr(_backend(), 4)]), pb.BackendMismatchError),
    (dict(grad_scale=lambda b: _arr(b, 2)), ValueError),
])
def test_adamw_step_refuses(backend, change, error):
    backend._lib.pb_free = lambda *args: 0
    args = {k: [_arr(backend, 4)] for k in ("params", "grads", "exp_avg", "exp_avg_sq")} | dict(step=1)
    args |= {k: v(backend) if callable(v) else v for k, v in change.items()}
    with pytest.raises(error):
        pb.adamw_step(**args)
    assert not [n for n, _ in backend._lib.calls if n == "pb_adamw"]


def test_the_operator_cases_call_what_the_package_has():
    """Every pacho_b200 name that the cases of perf/operators.py call is there."""
    tree = ast.parse((pathlib.Path(__file__).parent.parent / "perf" / "operators.py").read_text())
    aliases = {a.asname or a.name for n in ast.walk(tree) if isinstance(n, ast.Import) for a in n.names
               if a.name == "pacho_b200"}
    called = {n.attr for n in ast.walk(tree) if isinstance(n, ast.Attribute) and isinstance(n.value, ast.Name)
              and n.value.id in aliases}
    called |= {a.name for n in ast.walk(tree) if isinstance(n, ast.ImportFrom) and n.module == "pacho_b200"
               for a in n.names}
    assert called and not [name for name in called if not hasattr(pb, name)]


def test_c_entries_refuse_before_any_device_call():
    lib, bad = _lib.load(), _lib.PB_ERR_INVALID
    assert lib.pb_recurrence(None, 0, 0, 0, 1, 1, 1, None, None, None, None, None) == bad
    assert lib.pb_recurrence_backward(None, 0, 0, 0, 1, 1, 1, *([None] * 9)) == bad
    assert lib.pb_group_norm(None, 0, 0, 0, 1, 1, 1, 1, 1e-5, *([None] * 6)) == bad
    assert lib.pb_group_norm_backward(None, 0, 0, 0, 1, 1, 1, 1, *([None] * 9)) == bad
    assert lib.pb_adamw(None, 0, 0, 0, None, None, None, None, None, 0, 0, 0, 0, 0, 1, None) == bad


# A context that is never entered: every one of these calls is refused by the
# checks that come before the device is touched.
_FAKE = (C.c_char * 4096)()


def _ptr(i):
    return 0x10000 * (i + 1)


@pytest.mark.parametrize("call,text", [
    (lambda lib, c: lib.pb_recurrence(c, 0, 2, 0, 1, 1, 1, *map(_ptr, range(5))), b"float32 or float64"),
    (lambda lib, c: lib.pb_recurrence(c, 0, 0, 7, 1, 1, 1, *map(_ptr, range(5))), b"gate"),
    (lambda lib, c: lib.pb_recurrence(c, 0, 0, 0, -1, 1, 1, *map(_ptr, range(5))), b"negative"),
    (lambda lib, c: lib.pb_recurrence(c, 0, 0, 0, 1 << 40, 1 << 40, 1, *map(_ptr, range(5))), b"large"),
    (lambda lib, c: lib.pb_recurrence(c, 0, 0, 0, 1, 4, 4, None, *map(_ptr, range(4))), b"null"),
    (lambda lib, c: lib.pb_recurrence(c, 0, 0, 0, 1, 4, 4, _ptr(0), _ptr(1), None, _ptr(0), None), b"overlap"),
    (lambda lib, c: lib.pb_recurrence(c, 0, 0, 0, 1, 4, 4, _ptr(0), _ptr(1), None, _ptr(1) + 60, None), b"overlap"),
    (lambda lib, c: lib.pb_recurrence(c, 0, 0, 0, 1, 4, 4, _ptr(0), _ptr(1), None, _ptr(2), _ptr(2)), b"overlap"),
    (lambda lib, c: lib.pb_recurrence(c, 0, 0, 0, 1, 4, 4, _ptr(0), _ptr(1), _ptr(2), _ptr(3), _ptr(2) + 4),
     b"overlap"),
    (lambda lib, c: lib.pb_recurrence(c, 0, 0, 0, 1, 4, 4, _ptr(0) + 2, _ptr(1), None, _ptr(2), None), b"aligned"),
    (lambda lib, c: lib.pb_recurrence_backward(c, 0, 0, 1, 1, 4, 4, _ptr(0), None, *map(_ptr, range(1, 8))), b"need b"),
    (lambda lib, c: lib.pb_recurrence_backward(c, 0, 0, 0, 1, 4, 4, *map(_ptr, range(7)), _ptr(3), None), b"overlap"),
    (lambda lib, c: lib.pb_group_norm(c, 0, 0, 9, 1, 1, 4, 2, 0.0, *map(_ptr, range(6))), b"activation"),
    (lambda lib, c: lib.pb_group_norm(c, 0, 0, 0, 1, 1, 4, 3, 0.0, *map(_ptr, range(6))), b"divide"),
    (lambda lib, c: lib.pb_group_norm(c, 0, 0, 0, 1, 0, 4, 2, 0.0, *map(_ptr, range(6))), b"empty"),
    (lambda lib, c: lib.pb_group_norm(c, 0, 0, 0, 1, 1, 0, 2, 0.0, *map(_ptr, range(6))), b"empty"),
    (lambda lib, c: lib.pb_group_norm(c, 0, 0, 0, 1, 1, 4, 2, -1.0, *map(_ptr, range(6))), b"eps"),
    (lambda lib, c: lib.pb_group_norm(c, 0, 0, 0, 1, 1, 4, 2, float("nan"), *map(_ptr, range(6))), b"eps"),
    (lambda lib, c: lib.pb_group_norm(c, 0, 0, 0, 1, 1, 4, 2, 0.0, _ptr(0), None, None, _ptr(0), None, None),
     b"overlap"),
    (lambda lib, c: lib.pb_group_norm_backward(c, 0, 0, 0, 1, 1, 4, 2, *map(_ptr, range(6)), _ptr(0), None, None),
     b"overlap"),
    (lambda lib, c: lib.pb_group_norm_backward(c, 0, 0, 0, 1, 1, 4, 2, _ptr(0), _ptr(1), None, *map(_ptr, range(6))),
     b"null"),
])
def test_c_entries_refuse_bad_operands(call, text):
    lib = _lib.load()
    assert call(lib, C.addressof(_FAKE)) == _lib.PB_ERR_INVALID
    assert text in lib.pb_last_error(), lib.pb_last_error()


@pytest.mark.parametrize("change,text", [
    (dict(dtype=2), b"float32 or float64"), (dict(beta1=1.0), b"betas"), (dict(beta2=-0.1), b"betas"),
    (dict(step=0), b"step"), (dict(lr=-1.0), b"negative"), (dict(eps=float("nan")), b"negative"),
    (dict(sizes=[4, -1]), b"size"), (dict(p=[_ptr(0), None]), b"null"),
    (dict(p=[_ptr(0), _ptr(0)]), b"overlap"), (dict(p=[_ptr(0), _ptr(0) + 12]), b"overlap"),
    (dict(m=[_ptr(2), _ptr(4)], v=[_ptr(4), _ptr(5)]), b"overlap"), (dict(g=[_ptr(8), _ptr(1) + 8]), b"overlap"),
    (dict(scale=_ptr(5) + 4), b"overlap"), (dict(p=[_ptr(0), _ptr(1) + 2]), b"aligned"),
])
def test_c_adamw_refuses_bad_operands(change, text):
    lib = _lib.load()
    a = dict(dtype=0, p=[_ptr(0), _ptr(1)], m=[_ptr(2), _ptr(3)], v=[_ptr(4), _ptr(5)], g=[_ptr(8), _ptr(9)],
             sizes=[4, 4], lr=1e-3, beta1=0.9, beta2=0.99, eps=1e-8, step=1, scale=None) | change
    table = [(C.c_void_p * 2)(*a[k]) for k in ("p", "g", "m", "v")]
    status = lib.pb_adamw(C.addressof(_FAKE), 0, a["dtype"], 2, *table, (C.c_int64 * 2)(*a["sizes"]), a["lr"],
                          a["beta1"], a["beta2"], a["eps"], 0.0, a["step"], a["scale"])
    assert status == _lib.PB_ERR_INVALID and text in lib.pb_last_error(), lib.pb_last_error()


# --------------------- the reference gradients against differences


def _difference(f, x, direction, step=1e-6):
    return (f(x + step * direction) - f(x - step * direction)) / (2 * step)


@pytest.mark.parametrize("gate", ["linear", "sigmoid"])
def test_reference_recurrence_gradients(gate):
    rng = np.random.default_rng(1)
    a, b = rng.uniform(0.2, 0.95, (2, 9, 3)), rng.standard_normal((2, 9, 3))
    s, dh, df = rng.standard_normal((2, 3)), rng.standard_normal((2, 9, 3)), rng.standard_normal((2, 3))

    def loss(a, b, s):
        h = ref.recurrence(a, b, s, gate, 0.0)[0]
        return np.sum(h * dh) + np.sum(h[:, -1] * df)

    h = ref.recurrence(a, b, s, gate, 0.0)[0]
    (da, db, ds), _ = ref.recurrence_backward(a, b, h, dh, s, df, gate, 0.0)
    for x, grad, f in ((a, da, lambda v: loss(v, b, s)), (b, db, lambda v: loss(a, v, s)),
                       (s, ds, lambda v: loss(a, b, v))):
        d = rng.standard_normal(x.shape)
        assert abs(_difference(f, x, d) - np.sum(grad * d)) <= 1e-7 * (1 + np.sum(np.abs(grad * d)))


@pytest.mark.parametrize("act", [None, "relu", "silu", "gelu"])
def test_reference_group_norm_gradients(act):
    rng = np.random.default_rng(2)
    x, dy = rng.standard_normal((2, 5, 6)), rng.standard_normal((2, 5, 6))
    w, b = rng.uniform(0.5, 1.5, 6), rng.standard_normal(6) * 0.3

    def loss(x, w, b):
        return np.sum(ref.group_norm(x, 3, w, b, 1e-3, act, 0.0)[0][0] * dy)

    (_, mean, rstd), _ = ref.group_norm(x, 3, w, b, 1e-3, act, 0.0)
    (dx, dw, db), _ = ref.group_norm_backward(dy, x, 3, mean, rstd, w, b, act, 0.0)
    for v, grad, f in ((x, dx, lambda q: loss(q, w, b)), (w, dw, lambda q: loss(x, q, b)),
                       (b, db, lambda q: loss(x, w, q))):
        d = rng.standard_normal(v.shape)
        assert abs(_difference(f, v, d) - np.sum(grad * d)) <= 1e-6 * (1 + np.sum(np.abs(grad * d)))
