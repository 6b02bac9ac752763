"""Arrays over memory that another library owns (B200Backend.view) and the
order of its streams and the library's: the refusals on CPU with a recording
library, the memory and the order on the GPU with torch as the owner."""

from __future__ import annotations

import ctypes as C
import threading
import weakref

import numpy as np
import pytest

from pacho_b200 import _lib
from pacho_b200.backend import B200Backend


class Recording:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, args))
            return 0

        return call


@pytest.fixture
def host_backend():
    b = object.__new__(B200Backend)
    b._lib, b._ctx, b._lock, b._closed = Recording(), C.c_void_p(1), threading.RLock(), False
    b._buffers = weakref.WeakSet()
    yield b
    b._closed = True


def _face(ptr=4096, shape=(3, 5), typestr="<f4", strides=None, read_only=False, **more):
    return type("Owner", (), {"__cuda_array_interface__": dict(
        shape=shape, typestr=typestr, data=(ptr, read_only), strides=strides, version=2, **more)})()


@pytest.mark.parametrize("face,error", [
    (_face(ptr=4100), ValueError),                      # not 16-byte aligned
    (_face(strides=(4, 12)), ValueError),               # transposed
    (_face(strides=(24, 4)), ValueError),               # rows with a gap
    (_face(read_only=True), ValueError),
    (_face(typestr="<f2"), TypeError),
    (_face(typestr=">f4"), TypeError),
    (_face(typestr="<i4"), TypeError),
])
def test_refused_views(host_backend, face, error):
    with pytest.raises(error):
        host_backend.view(face)
    assert host_backend._lib.calls == []


def test_a_masked_array_is_refused(host_backend):
    """The interface's mask marks values that are not there: they are not to be read as values."""
    with pytest.raises(ValueError, match="mask"):
        host_backend.view(_face(mask=_face(typestr="|b1")))
    assert host_backend._lib.calls == []
    assert host_backend.view(_face(mask=None)).shape == (3, 5)


def test_view_without_the_interface(host_backend):
    with pytest.raises(AttributeError):
        host_backend.view(np.zeros(3, np.float32))


@pytest.mark.parametrize("more,stream,joined", [
    ({}, None, [None]),                 # no stream named: the legacy default stream
    ({"stream": 7}, None, [7]),         # the interface's
    ({"stream": None}, None, []),       # it asks for no ordering
    ({"stream": 7}, 9, [9]),            # the caller's
    ({}, 0, [None]),
])
def test_view_orders_the_stream_that_is_named(host_backend, more, stream, joined):
    x = host_backend.view(_face(**more), stream=stream)
    assert x.shape == (3, 5) and x.dtype == np.float32 and x._data.ptr == 4096
    calls = host_backend._lib.calls
    assert calls[0][0] == "pb_pointer_check" and calls[0][1][3] == 60
    assert [c[1][2].value for c in calls[1:]] == joined
    assert all(c[0] == "pb_stream_join" and c[1][3] == _lib.PB_JOIN_WAIT for c in calls[1:])


def test_empty_view_and_unit_dimensions(host_backend):
    assert host_backend.view(_face(ptr=0, shape=(0, 4))).size == 0
    assert host_backend._lib.calls[0][0] == "pb_stream_join"  # no memory to check
    assert host_backend.view(_face(shape=(1, 5), strides=(999, 4))).shape == (1, 5)


def test_signal_stream(host_backend):
    host_backend.signal_stream(11)
    (name, args), = host_backend._lib.calls
    assert name == "pb_stream_join" and args[2].value == 11 and args[3] == _lib.PB_JOIN_SIGNAL


def test_null_context_is_refused_without_a_gpu():
    lib = _lib.load()
    assert lib.pb_pointer_check(None, 0, None, 4) == _lib.PB_ERR_INVALID
    assert lib.pb_stream_join(None, 0, None, 0) == _lib.PB_ERR_INVALID


# ------------------------------------------------------------------ on a GPU


@pytest.mark.gpu
def test_view_shares_memory_in_both_directions(b200):
    torch = pytest.importorskip("torch")
    t = torch.arange(1000, dtype=torch.float32, device="cuda")
    x = b200.view(t)
    assert x.numpy().tobytes() == np.arange(1000, dtype=np.float32).tobytes()
    t.mul_(2)
    b200.wait_stream(torch.cuda.current_stream().cuda_stream)
    out = b200.view(torch.empty(1, device="cuda"))
    _lib.check(b200._lib.pb_dot(b200._ctx, 0, _lib.PB_F32, 1000, C.c_void_p(x._data.ptr),
                                C.c_void_p(x._data.ptr), C.c_void_p(out._data.ptr)))
    b200.signal_stream(torch.cuda.current_stream().cuda_stream)
    got = out._data.owner.item()
    want = 4.0 * float(np.sum(np.arange(1000.0) ** 2))
    assert abs(got - want) <= 1e-5 * want


@pytest.mark.gpu
def test_streams_are_ordered_in_both_directions(b200):
    """A long producer on a stream of torch's own, then the library, then a
    consumer on that stream: no host synchronisation between them."""
    torch = pytest.importorskip("torch")
    side = torch.cuda.Stream()
    n = 1 << 24
    for turn in range(5):
        with torch.cuda.stream(side):
            t = torch.zeros(n, device="cuda")
            for _ in range(20):
                t.add_(1.0)
            x = b200.view(t, stream=side.cuda_stream)
            data = b200.elementwise("multiply", [x, x], (n,), np.float32)  # 400
            b200.signal_stream(side.cuda_stream)
            t.fill_(-1.0)  # must come after the product has read t
        got = np.empty(n, np.float32)
        _lib.check(b200._lib.pb_d2h(b200._ctx, 0, C.c_void_p(got.ctypes.data), C.c_void_p(data.ptr), got.nbytes))
        assert got.min() == got.max() == 400.0, turn
    side.synchronize()


@pytest.mark.gpu
def test_host_memory_is_refused(b200):
    host = np.zeros(64, np.float32)
    lib, ctx = b200._lib, b200._ctx
    assert lib.pb_pointer_check(ctx, 0, C.c_void_p(host.ctypes.data), host.nbytes) == _lib.PB_ERR_INVALID
    buf = b200.empty((64,), np.float32)
    assert lib.pb_pointer_check(ctx, 0, C.c_void_p(buf.ptr), buf.nbytes) == _lib.PB_OK
    # The refusal leaves nothing behind: the next launch succeeds.
    assert np.all(b200.download(type("A", (), {"shape": (4,), "dtype": np.dtype(np.float32),
                                               "_data": b200.full((4,), 3.0, np.float32)})()) == 3.0)


@pytest.mark.gpu
def test_join_is_refused_while_either_side_is_captured(b200):
    torch = pytest.importorskip("torch")
    with pytest.raises(NotImplementedError):
        b200.capture(lambda: b200.wait_stream(0))
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(NotImplementedError):
        with torch.cuda.graph(graph, stream=side, capture_error_mode="relaxed"):
            b200.wait_stream(side.cuda_stream)
    b200.wait_stream(side.cuda_stream)
    b200.synchronize()
