"""The layer operators on the GPU against their definitions in float64
(layer_reference), within bounds that follow from the formulas and the unit
roundoff of the type.

FACTOR covers what the bounds leave out on purpose: terms of second order, and
a recurrence cut into pieces, whose pieces are first run from zero and then
again from their true start (at most two roundings where one was counted)."""

from __future__ import annotations

import ctypes as C
import threading

import numpy as np
import pytest

import layer_reference as ref
import pacho_b200 as pb
from pacho_b200 import _lib
from pacho_b200.backend import DeviceArray

pytestmark = pytest.mark.gpu
FACTOR = 3.0
FLOATS = [np.float32, np.float64]


def up(b200, x):
    return None if x is None else DeviceArray(b200, b200.upload(x), x.shape, x.dtype)


def poisoned(b200, shape, dtype):
    """An output full of NaN: a value that is not written shows."""
    return DeviceArray(b200, b200.full(shape, np.nan, dtype), shape, dtype)


def close(got, want, bound, dtype, what):
    got = got.astype(np.float64)
    tiny = float(np.finfo(dtype).tiny)
    off = np.abs(got - want) - FACTOR * bound - 8 * tiny
    bad = ~(off <= 0)  # a NaN is bad too
    assert not bad.any(), (f"{what}: {bad.sum()} of {bad.size} off, first at {np.argwhere(bad)[0]}: "
                           f"{got[bad][0]!r} for {want[bad][0]!r}, bound {bound[bad][0]!r}")


# ------------------------------------------------------------ recurrence --

SHAPES = [  # (outer, length, inner): single steps, short, odd, long, wide, one column
    (1, 1, 1), (32, 1, 2048), (3, 2, 5), (1, 7, 33), (2, 8, 31), (5, 17, 64), (2, 127, 40), (2, 128, 32),
    (2, 129, 96), (1, 1000, 515), (3, 2047, 100), (1, 4100, 8), (1, 20011, 1), (700, 9, 1), (9, 300, 3),
    (1, 16381, 65), (64, 40, 1024), (2, 70, 33), (3, 211, 71), (5, 641, 38), (1, 333, 1), (2, 4099, 149), (300, 50, 31),
    (1, 40, 8193), (13, 97, 701),
]


def _recurrence_inputs(shape, dtype, gate, seed=0):
    rng = np.random.default_rng(sum(shape) + seed)
    z = rng.standard_normal(shape) * 2 + 2
    a = (z if gate == "sigmoid" else ref.sigmoid(z)[0] * np.where(rng.random(shape) < 0.2, -1, 1)).astype(dtype)
    b = rng.standard_normal(shape).astype(dtype)
    state = rng.standard_normal((shape[0], shape[2])).astype(dtype)
    return a, b, state, rng


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("gate", ["linear", "sigmoid"])
@pytest.mark.parametrize("shape", SHAPES)
def test_recurrence(b200, shape, gate, dtype):
    a, b, state, _ = _recurrence_inputs(shape, dtype, gate)
    u = ref.U[np.dtype(dtype)]
    for s in (state, None):
        out, final = poisoned(b200, shape, dtype), poisoned(b200, state.shape, dtype)
        h = pb.linear_recurrence(up(b200, a), up(b200, b), state=up(b200, s), gate=gate, out=out, final=final)
        assert h is out
        got = h.numpy()
        want, bound = ref.recurrence(a, b, s, gate, u)
        close(got, want, bound, dtype, "h")
        assert final.numpy().tobytes() == got[:, -1].tobytes()


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("gate", ["linear", "sigmoid"])
@pytest.mark.parametrize("shape", SHAPES)
def test_recurrence_backward(b200, shape, gate, dtype):
    a, b, state, rng = _recurrence_inputs(shape, dtype, gate, 1)
    u = ref.U[np.dtype(dtype)]
    dh = rng.standard_normal(shape).astype(dtype)
    dfinal = rng.standard_normal(state.shape).astype(dtype)
    for s, df in ((state, dfinal), (None, None)):
        h = ref.recurrence(a, b, s, gate, u)[0].astype(dtype)
        out = tuple(poisoned(b200, v, dtype) for v in (shape, shape, state.shape))
        got = pb.linear_recurrence_backward(up(b200, a), up(b200, b), up(b200, h), up(b200, dh), state=up(b200, s),
                                            dfinal=up(b200, df), gate=gate, out=out)
        want, bounds = ref.recurrence_backward(a, b, h, dh, s, df, gate, u)
        for name, g, w, e in zip(("da", "db", "dstate"), got, want, bounds):
            close(g.numpy(), w, e, dtype, name)


@pytest.mark.parametrize("gate", ["linear", "sigmoid"])
def test_recurrence_axes(b200, gate):
    shape = (3, 6, 10, 4)
    a, b, _, rng = _recurrence_inputs(shape[:3], np.float64, gate)
    a, b = (np.broadcast_to(v[..., None], shape) * rng.uniform(0.9, 1.0, shape) for v in (a, b))
    for axis in range(4):
        rest = tuple(d for i, d in enumerate(shape) if i != axis)
        s = rng.standard_normal(rest)
        final = poisoned(b200, rest, np.float64)
        h = pb.linear_recurrence(up(b200, a), up(b200, b), state=up(b200, s), gate=gate, axis=axis,
                                 final=final).numpy()
        # The same view, the axis in the middle.
        view = (int(np.prod(shape[:axis], dtype=int)), shape[axis], int(np.prod(shape[axis + 1:], dtype=int)))
        want, bound = ref.recurrence(a.reshape(view), b.reshape(view), s.reshape(view[0], view[2]), gate, 2.0 ** -53)
        close(h.reshape(view), want, bound, np.float64, f"axis {axis}")
        assert np.array_equal(final.numpy(), np.take(h, -1, axis))


@pytest.mark.parametrize("dtype", FLOATS)
def test_recurrence_empty_axes(b200, dtype):
    state = np.arange(6, dtype=dtype).reshape(2, 3)
    a = up(b200, np.zeros((2, 0, 3), dtype))
    final = poisoned(b200, (2, 3), dtype)
    assert pb.linear_recurrence(a, a, state=up(b200, state), final=final).shape == (2, 0, 3)
    assert np.array_equal(final.numpy(), state)
    pb.linear_recurrence(a, a, final=final)
    assert np.array_equal(final.numpy(), np.zeros_like(state))
    _, _, ds = pb.linear_recurrence_backward(a, a, a, a, dfinal=up(b200, state))
    assert np.array_equal(ds.numpy(), state)
    none = up(b200, np.zeros((0, 5, 3), dtype))
    assert pb.linear_recurrence(none, none).size == 0
    none = up(b200, np.zeros((4, 5, 0), dtype))
    assert pb.linear_recurrence_backward(none, none, none, none)[2].shape == (4, 0)


@pytest.mark.parametrize("shape", [(8, 1, 96), (1, 3000, 96)])
def test_recurrence_state_kept_in_place(b200, shape):
    """`final` may be `state`: a stream read in two parts gives the whole one's bits
    at every position that starts a piece of its own, and the definition's values."""
    a, b, state, _ = _recurrence_inputs((shape[0], 2 * shape[1], shape[2]), np.float32, "sigmoid")
    keep = up(b200, state)
    parts = []
    for half in (slice(0, shape[1]), slice(shape[1], None)):
        h = pb.linear_recurrence(up(b200, np.ascontiguousarray(a[:, half])), up(b200, np.ascontiguousarray(b[:, half])),
                                 state=keep, final=keep, gate="sigmoid").numpy()
        assert keep.numpy().tobytes() == h[:, -1].tobytes()
        parts.append(h)
    want, bound = ref.recurrence(a, b, state, "sigmoid", 2.0 ** -24)
    close(np.concatenate(parts, 1), want, bound, np.float32, "parts")


@pytest.mark.parametrize("dtype", FLOATS)
def test_recurrence_resets_growth_and_saturated_gates(b200, dtype):
    """alpha = 0 forgets what came before, whatever it was; gates above 1
    that overflow as a product over zeros; logits far out on both sides."""
    n, c = 3000, 40
    rng = np.random.default_rng(3)
    a = np.full((1, n, c), 2.0, dtype)
    b = np.zeros((1, n, c), dtype)
    a[0, n - 30:] = 0.5
    b[0, n - 20] = 1.0
    h = pb.linear_recurrence(up(b200, a), up(b200, b)).numpy()
    want = np.zeros(n)
    want[n - 20:] = 0.5 ** np.arange(20)
    assert np.array_equal(h, np.broadcast_to(want[None, :, None], h.shape).astype(dtype))
    a = rng.uniform(0.9, 1.0, (2, n, c)).astype(dtype)
    b = rng.standard_normal((2, n, c)).astype(dtype)
    a[:, 777] = 0.0  # a new sequence starts here
    whole = pb.linear_recurrence(up(b200, a), up(b200, b)).numpy()
    want, bound = ref.recurrence(a[:, 777:], b[:, 777:], None, "linear", ref.U[np.dtype(dtype)])
    close(whole[:, 777:], want, bound, dtype, "after the reset")
    z = np.tile(np.array([-1e4, -100, -40, 40, 100, 1e4, -np.inf, np.inf], dtype), c // 8)
    z = np.broadcast_to(z, (1, n, c)).copy()
    b = np.ones_like(z)
    h = pb.linear_recurrence(up(b200, z), up(b200, b), gate="sigmoid").numpy()
    want, bound = ref.recurrence(z, b, None, "sigmoid", ref.U[np.dtype(dtype)])
    close(h, want, bound, dtype, "saturated")


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_recurrence_confines_what_is_not_finite_to_its_column(b200, bad):
    a, b, state, _ = _recurrence_inputs((1, 2000, 64), np.float32, "linear")
    clean = pb.linear_recurrence(up(b200, a), up(b200, b), state=up(b200, state)).numpy()
    b[0, 700, 13] = bad
    h = pb.linear_recurrence(up(b200, a), up(b200, b), state=up(b200, state)).numpy()
    others = np.arange(64) != 13
    assert h[..., others].tobytes() == clean[..., others].tobytes()
    assert h[0, :700, 13].tobytes() == clean[0, :700, 13].tobytes()
    assert not np.isfinite(h[0, 700:, 13]).any()


def test_recurrence_repeats_its_bits(b200):
    a, b, state, rng = _recurrence_inputs((2, 9001, 200), np.float32, "sigmoid")
    da, db, ds = (up(b200, v) for v in (a, b, state))
    first = pb.linear_recurrence(da, db, state=ds, gate="sigmoid")
    dh = up(b200, rng.standard_normal(a.shape).astype(np.float32))
    back = [g.numpy().tobytes() for g in pb.linear_recurrence_backward(da, db, first, dh, state=ds, gate="sigmoid")]
    for _ in range(4):
        assert pb.linear_recurrence(da, db, state=ds, gate="sigmoid").numpy().tobytes() == first.numpy().tobytes()
        again = pb.linear_recurrence_backward(da, db, first, dh, state=ds, gate="sigmoid")
        assert [g.numpy().tobytes() for g in again] == back


# ------------------------------------------------------------ group norm --

NORMS = [  # (N, S, C, G)
    (1, 1, 1, 1), (1, 1, 8, 1), (32, 1, 2048, 16), (7, 1, 96, 3), (5, 1, 100, 4), (300, 1, 24, 3), (2, 1, 7, 7),
    (3, 1, 5000, 1), (2, 1, 12289, 1), (9, 1, 1030, 2), (1000, 1, 64, 1), (130, 1, 512, 2), (3, 5, 6, 2),
    (2, 49, 32, 8), (1, 1000, 3, 1), (3, 37 * 41, 90, 9), (2, 4096, 20, 4), (4, 256, 320, 32), (1, 20000, 16, 2),
    (17, 3, 1300, 26), (600, 4, 8, 1), (20, 1, 4000, 1), (70, 1, 1000, 2), (50, 1, 1024, 1), (6, 64, 160, 4),
    (33, 10, 64, 2),
    # Rows that do not end on 16 bytes, the ends of the array among them; wider than a block spans.
    (1, 2049, 1, 1), (3, 5000, 21, 3), (5, 1031, 91, 7), (3, 700, 319, 11), (2, 333, 959, 7), (3, 333, 1919, 19),
    (2, 150, 1921, 17), (2, 2050, 5, 1), (1, 40001, 7, 7),
    # Rows of single values, from a few lanes to the most that a block holds, and one more.
    (40, 1, 39, 3), (60, 1, 62, 2), (30, 1, 507, 3), (20, 1, 510, 1), (9, 1, 1022, 1), (6, 1, 4095, 1), (5, 1, 8191, 1),
    (3, 1, 8193, 1), (9, 3, 25, 1), (7, 41, 50, 2), (5, 101, 15, 1),
]
ACTS = [None, "relu", "silu", "gelu"]


def _norm_inputs(shape, dtype, seed=0):
    n, s, c, g = shape
    rng = np.random.default_rng(n + s + c + seed)
    x = (rng.standard_normal((n, s, c)) * 1.5 + 0.3).astype(dtype)
    w = (rng.standard_normal(c) * 0.3 + 1).astype(dtype)
    b = (rng.standard_normal(c) * 0.3).astype(dtype)
    return x, w, b, rng


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("shape", NORMS)
def test_group_norm(b200, shape, dtype):
    x, w, b, _ = _norm_inputs(shape, dtype)
    g = shape[3]
    for k, act in enumerate(ACTS):
        w_, b_ = (w if k != 1 else None), (b if k != 2 else None)
        out = tuple(poisoned(b200, v, dtype) for v in (x.shape, (shape[0], g), (shape[0], g)))
        got = pb.group_norm(up(b200, x), g, up(b200, w_), up(b200, b_), eps=1e-3, activation=act, out=out)
        want, bounds = ref.group_norm(x, g, w_, b_, 1e-3, act, ref.U[np.dtype(dtype)])
        for name, q, v, e in zip(("y", "mean", "rstd"), got, want, bounds):
            close(q.numpy(), v, e, dtype, f"{act} {name}")


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("shape", NORMS)
def test_group_norm_backward(b200, shape, dtype):
    x, w, b, rng = _norm_inputs(shape, dtype, 1)
    g = shape[3]
    dy = rng.standard_normal(x.shape).astype(dtype)
    for k, act in enumerate(ACTS):
        w_, b_ = (w if k != 1 else None), (b if k != 2 else None)
        (_, mean, rstd), _ = ref.group_norm(x, g, w_, b_, 1e-3, act, 0.0)
        mean, rstd = mean.astype(dtype), rstd.astype(dtype)
        out = (poisoned(b200, x.shape, dtype),) + tuple(
            None if v is None else poisoned(b200, v.shape, dtype) for v in (w_, b_))
        got = pb.group_norm_backward(up(b200, dy), up(b200, x), g, up(b200, mean), up(b200, rstd), up(b200, w_),
                                     up(b200, b_), activation=act, out=out)
        want, bounds = ref.group_norm_backward(dy, x, g, mean, rstd, w_, b_, act, ref.U[np.dtype(dtype)])
        for name, q, v, e in zip(("dx", "dweight", "dbias"), got, want, bounds):
            if q is not None:
                close(q.numpy(), v, e, dtype, f"{act} {name}")


@pytest.mark.parametrize("shape", [(3, 1, 64, 2), (2, 900, 12, 3)])
@pytest.mark.parametrize("offset", [1e4, -3e6])
def test_group_norm_far_from_zero(b200, shape, offset):
    """The variance of values that lie far from zero is not lost."""
    x, w, b, _ = _norm_inputs(shape, np.float32)
    x = (x + offset).astype(np.float32)
    got = pb.group_norm(up(b200, x), shape[3], up(b200, w), up(b200, b))
    want, bounds = ref.group_norm(x, shape[3], w, b, 1e-5, None, 2.0 ** -24)
    for name, q, v, e in zip(("y", "mean", "rstd"), got, want, bounds):
        close(q.numpy(), v, e, np.float32, name)


@pytest.mark.parametrize("shape", [(5, 1, 100, 4), (7, 1, 96, 3), (3, 1, 5000, 1), (9, 1, 1030, 2), (17, 3, 1300, 26),
                                   (2, 4096, 20, 4), (3, 1517, 90, 9), (1, 20000, 16, 2)])
def test_group_norm_backward_where_the_mean_over_the_deviation_overflows(b200, shape):
    """x = mean = 1e30 and rstd = 1e10: xhat is 0 and every gradient finite,
    though (0 - mean) rstd, what a place without a value would give, is not.
    Sums of 2^20 equal float32 values are exact in float64."""
    _, w, b, rng = _norm_inputs(shape, np.float32)
    n, s, c, g = shape
    x, mean = np.full((n, s, c), 1e30, np.float32), np.full((n, g), 1e30, np.float32)
    rstd, dy = np.full((n, g), 1e10, np.float32), rng.standard_normal(x.shape).astype(np.float32)
    for act in ACTS:
        got = pb.group_norm_backward(*(up(b200, v) for v in (dy, x)), g, *(up(b200, v) for v in (mean, rstd, w, b)),
                                     activation=act)
        want, bounds = ref.group_norm_backward(dy, x, g, mean, rstd, w, b, act, 2.0 ** -24)
        for name, q, v, e in zip(("dx", "dweight", "dbias"), got, want, bounds):
            close(q.numpy(), v, e, np.float32, f"{act} {name}")


def _scaled_inputs(shape, scale, seed):
    n, s, c, g = shape
    rng = np.random.default_rng(n + s + c + seed)
    x = ((rng.standard_normal((n, s, c)) + 0.3) * scale).astype(np.float32)
    w, b = (rng.standard_normal(c) * 0.3 + 1).astype(np.float32), (rng.standard_normal(c) * 0.3).astype(np.float32)
    return x, w, b, rng


# A shape of each kernel and way through it: rows in a part of a warp, a warp and a
# block, of packs and of single values, of several positions; the ring with packs
# and with single values; the samples kernel.
KERNELS = [(300, 1, 24, 3), (130, 1, 512, 2), (20, 1, 4000, 1), (60, 1, 62, 2), (9, 1, 1022, 1), (3, 1, 8191, 1),
           (17, 3, 1300, 26), (9, 3, 25, 1), (2, 4096, 20, 4), (3, 5000, 21, 3), (2, 150, 1921, 17), (2, 80, 2048, 8),
           (3, 1, 8193, 1)]


@pytest.mark.parametrize("scale,eps", [(1e30, 1e-5), (1e20, 0.0), (1e-15, 0.0), (1e-24, 0.0), (1e-30, 0.0)])
@pytest.mark.parametrize("shape", KERNELS)
def test_group_norm_of_values_whose_squares_leave_float32(b200, shape, scale, eps):
    """Deviations of 1e20 and more or 1e-24 and less: mean, rstd and y are ordinary float32
    values, the squares are not."""
    x, w, b, _ = _scaled_inputs(shape, scale, 3)
    for act in (None, "silu"):
        got = pb.group_norm(up(b200, x), shape[3], up(b200, w), up(b200, b), eps=eps, activation=act)
        want, bounds = ref.group_norm(x, shape[3], w, b, eps, act, 2.0 ** -24)
        for name, q, v, e in zip(("y", "mean", "rstd"), got, want, bounds):
            close(q.numpy(), v, e, np.float32, f"{act} {name}")


@pytest.mark.parametrize("scale", [1e30, 1e22, 1e-22, 1e-30])
@pytest.mark.parametrize("size", [1.0, 1e10, 1e-10])
@pytest.mark.parametrize("shape", KERNELS)
def test_group_norm_backward_of_large_and_small_values(b200, shape, size, scale):
    """rstd far from 1: dx is of the size of dy rstd, while rstd^2 and dy (x - mean) leave
    float32's range on one side or the other.  dy = 1e10 at rstd = 1e30 is beyond it
    itself: such a dx is the infinity of its sign."""
    x, w, b, rng = _scaled_inputs(shape, scale, 4)
    g = shape[3]
    dy = (rng.standard_normal(x.shape) * size).astype(np.float32)
    (_, mean, rstd), _ = ref.group_norm(x, g, w, b, 0.0, None, 0.0)
    mean, rstd = mean.astype(np.float32), rstd.astype(np.float32)
    for act in (None, "silu"):
        got = pb.group_norm_backward(*(up(b200, v) for v in (dy, x)), g, *(up(b200, v) for v in (mean, rstd, w, b)),
                                     activation=act)
        want, bounds = ref.group_norm_backward(dy, x, g, mean, rstd, w, b, act, 2.0 ** -24)
        for name, q, v, e in zip(("dx", "dweight", "dbias"), got, want, bounds):
            q, most = q.numpy(), float(np.finfo(np.float32).max)
            beyond = np.abs(v) - FACTOR * e > most
            assert np.array_equal(q[beyond], np.sign(v[beyond]) * np.float32(np.inf)), f"{act} {name}"
            here = np.abs(v) + FACTOR * e <= most
            close(q[here], v[here], e[here], np.float32, f"{act} {name}")


@pytest.mark.parametrize("dtype", FLOATS)
def test_gelu_keeps_its_relative_accuracy(b200, dtype):
    """With weights of zero an activation is of the bias alone.  From -12 on, where the
    density is a normal float32, z Phi(z) is off by ACT roundings of itself, and its slope
    Phi + z phi of the two terms.  In float64 the argument of erfc, z over the root of 2, has two
    roundings in the kernel and two in the definition; erfc(x) passes on 2 x^2 = z^2 of
    each, and exp(-z^2 / 2) as many."""
    b = np.concatenate([np.linspace(-12, 12, 4001), np.linspace(-0.3, 0.3, 800), [0.0]]).astype(dtype)
    c = b.size
    rng = np.random.default_rng(5)
    u = ref.U[np.dtype(dtype)]
    z = b.astype(np.float64)
    k = u * (ref.ACT + (4 * z * z if dtype == np.float64 else 0))
    x = rng.standard_normal((1, 1, c)).astype(dtype)
    y, _, _ = pb.group_norm(up(b200, x), 1, up(b200, np.zeros(c, dtype)), up(b200, b), activation="gelu")
    want = ref.activate(z, "gelu")
    close(y.numpy()[0, 0], want, k * np.abs(want), dtype, "gelu")
    stats = [up(b200, v) for v in (np.zeros((1, 1), dtype), np.ones((1, 1), dtype))]
    dy = rng.standard_normal((1, 1, c)).astype(dtype)
    _, _, dbias = pb.group_norm_backward(up(b200, dy), up(b200, x), 1, *stats, up(b200, np.zeros(c, dtype)), up(b200, b),
                                         activation="gelu")
    terms = np.abs(ref._erfc(-z / np.sqrt(2.0)) / 2) + np.abs(z) * np.exp(-z * z / 2) / np.sqrt(2 * np.pi)
    g = dy[0, 0].astype(np.float64)
    close(dbias.numpy(), g * ref.slope(z, "gelu"), k * np.abs(g) * terms, dtype, "slope")


@pytest.mark.parametrize("shape", [(4, 1, 64, 2), (3, 700, 8, 2)])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("where", [0, 5])
def test_group_norm_confines_what_is_not_finite_to_its_group(b200, shape, bad, where):
    x, w, b, _ = _norm_inputs(shape, np.float32)
    g, m = shape[3], shape[2] // shape[3]
    clean = pb.group_norm(up(b200, x), g, up(b200, w), up(b200, b), activation="silu")[0].numpy()
    x.reshape(shape[0], -1)[1, where % m] = bad  # sample 1, group 0
    y, mean, rstd = (q.numpy() for q in pb.group_norm(up(b200, x), g, up(b200, w), up(b200, b), activation="silu"))
    hit = np.zeros(y.shape, bool)
    hit[1, :, :m] = True
    assert np.isnan(y[hit]).all() and y[~hit].tobytes() == clean[~hit].tobytes()
    assert np.isnan(rstd[1, 0]) and (np.isnan(mean[1, 0]) if np.isnan(bad) else mean[1, 0] == bad)


def test_group_norm_of_constants_and_of_no_samples(b200):
    x = np.full((2, 10, 8), 7.0, np.float32)
    y, mean, rstd = pb.group_norm(up(b200, x), 2, eps=1e-2)
    assert np.all(y.numpy() == 0) and np.all(mean.numpy() == 7) and np.allclose(rstd.numpy(), 10.0)
    none = up(b200, np.zeros((0, 10, 8), np.float32))
    w = up(b200, np.ones(8, np.float32))
    y, mean, rstd = pb.group_norm(none, 2, w)
    assert y.shape == (0, 10, 8) and mean.shape == (0, 2)
    dw, db = poisoned(b200, (8,), np.float32), poisoned(b200, (8,), np.float32)
    pb.group_norm_backward(none, none, 2, mean, rstd, w, w, out=(None, dw, db))
    assert np.all(dw.numpy() == 0) and np.all(db.numpy() == 0)
    with pytest.raises(ValueError, match="empty"):
        pb.group_norm(up(b200, np.zeros((3, 0, 8), np.float32)), 2)


def test_group_norm_without_statistics(b200):
    """The C entry gives y alone when mean and rstd are not wanted."""
    for shape in ((5, 1, 64, 4), (2, 600, 16, 4)):
        x, w, b, _ = _norm_inputs(shape, np.float32)
        dx, y = up(b200, x), poisoned(b200, x.shape, np.float32)
        want = pb.group_norm(dx, shape[3])[0].numpy()
        _lib.check(b200._lib.pb_group_norm(b200._ctx, 0, _lib.PB_F32, 0, *shape, 1e-5, dx._data.ptr, None, None,
                                           y._data.ptr, None, None))
        assert y.numpy().tobytes() == want.tobytes()


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("shape", [(5, 1, 100, 4), (6, 64, 160, 4), (5, 101, 15, 1), (2, 333, 24, 3), (3, 2000, 8, 8),
                                   (3, 4000, 2, 1), (2, 8000, 3, 3), (2, 5000, 21, 3), (2, 150, 1921, 17)])
def test_group_norm_backward_without_weight_and_bias(b200, shape, dtype):
    x, _, _, rng = _norm_inputs(shape, dtype, 2)
    g = shape[3]
    dy = rng.standard_normal(x.shape).astype(dtype)
    (_, mean, rstd), _ = ref.group_norm(x, g, None, None, 1e-3, "silu", 0.0)
    mean, rstd = mean.astype(dtype), rstd.astype(dtype)
    dx, dw, db = pb.group_norm_backward(up(b200, dy), up(b200, x), g, up(b200, mean), up(b200, rstd),
                                        activation="silu", out=(poisoned(b200, x.shape, dtype), None, None))
    want, bounds = ref.group_norm_backward(dy, x, g, mean, rstd, None, None, "silu", ref.U[np.dtype(dtype)])
    close(dx.numpy(), want[0], bounds[0], dtype, "dx")
    assert dw is None and db is None


@pytest.mark.parametrize("shape", [(2, 700, 64, 4), (3, 1, 64, 4), (2, 700, 9, 3)])
@pytest.mark.parametrize("odd", ["x", "dy", "weight", "dx", "dweight"])
def test_group_norm_backward_of_arrays_that_start_anywhere(b200, shape, odd):
    """The C entry takes pointers that are aligned to a value only, and leaves
    what lies around its results."""
    x, w, b, rng = _norm_inputs(shape, np.float32)
    n, s, c, g = shape
    dy = rng.standard_normal(x.shape).astype(np.float32)
    (_, mean, rstd), _ = ref.group_norm(x, g, w, b, 1e-3, "silu", 0.0)
    mean, rstd = mean.astype(np.float32), rstd.astype(np.float32)
    arrays = dict(dy=dy, x=x, mean=mean, rstd=rstd, weight=w, bias=b, dx=np.full_like(x, np.nan),
                  dweight=np.full_like(w, np.nan), dbias=np.full_like(b, np.nan))
    held = {k: up(b200, np.concatenate([np.full(8, 7, np.float32), v.ravel(), np.full(8, 7, np.float32)]))
            for k, v in arrays.items()}
    at = {k: 9 if k == odd else 8 for k in arrays}
    held[odd] = up(b200, np.concatenate([np.full(9, 7, np.float32), arrays[odd].ravel(), np.full(7, 7, np.float32)]))
    _lib.check(b200._lib.pb_group_norm_backward(b200._ctx, 0, _lib.PB_F32, _lib.ACTIVATIONS["silu"], *shape,
                                                *(held[k]._data.ptr + 4 * at[k] for k in arrays)))
    want, bounds = ref.group_norm_backward(dy, x, g, mean, rstd, w, b, "silu", 2.0 ** -24)
    for k, v, e in zip(("dx", "dweight", "dbias"), want, bounds):
        got = held[k].numpy()
        close(got[at[k]:at[k] + v.size].reshape(v.shape), v, e, np.float32, k)
        assert np.all(got[:at[k]] == 7) and np.all(got[at[k] + v.size:] == 7)


def _check_group_norm(b200, shape, dtype):
    """Forward and backward of one shape with weight, bias and silu."""
    x, w, b, rng = _norm_inputs(shape, dtype, 6)
    g = shape[3]
    dy = rng.standard_normal(x.shape).astype(dtype)
    dx, dw, db, ddy = (up(b200, v) for v in (x, w, b, dy))
    out = tuple(poisoned(b200, v, dtype) for v in (x.shape, (shape[0], g), (shape[0], g)))
    got = pb.group_norm(dx, g, dw, db, eps=1e-3, activation="silu", out=out)
    want, bounds = ref.group_norm(x, g, w, b, 1e-3, "silu", ref.U[np.dtype(dtype)])
    for name, q, v, e in zip(("y", "mean", "rstd"), got, want, bounds):
        close(q.numpy(), v, e, dtype, name)
    mean, rstd = (v.astype(dtype) for v in want[1:])
    out = tuple(poisoned(b200, v.shape, dtype) for v in (x, w, b))
    got = pb.group_norm_backward(ddy, dx, g, up(b200, mean), up(b200, rstd), dw, db, activation="silu", out=out)
    want, bounds = ref.group_norm_backward(dy, x, g, mean, rstd, w, b, "silu", ref.U[np.dtype(dtype)])
    for name, q, v, e in zip(("dx", "dweight", "dbias"), got, want, bounds):
        close(q.numpy(), v, e, dtype, name)


# Shapes on either side of the choice between rows and ring: samples of few positions and
# many rounds, short runs.
CHOICES = [(1300, 70, 32, 4), (1300, 129, 8, 1), (1100, 65, 32, 4), (30, 600, 64, 64), (60, 64, 256, 256),
           (60, 64, 256, 64), (4, 4096, 33, 33), (9, 65, 48, 6), (2, 2000, 96, 24)]


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("shape", CHOICES)
def test_group_norm_on_either_side_of_a_choice(b200, shape, dtype):
    _check_group_norm(b200, shape, dtype)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("shape", [(2048, 64, 8, 1), (300, 33, 100, 5), (60, 2, 16, 2), (3, 64, 8, 1)])
def test_group_norm_of_many_samples_of_few_positions(b200, shape, dtype):
    _check_group_norm(b200, shape, dtype)


@pytest.mark.parametrize("shape,backward", [((20000, 65, 32, 4), True), ((40000, 65, 32, 1), True),
                                            ((8, 4096, 320, 320), False), ((16, 8192, 64, 64), False),
                                            ((1000, 64, 640, 640), False), ((1000, 64, 640, 640), True)])
def test_group_norm_does_not_fall_to_a_tenth_of_the_copy_rate(b200, shape, backward):
    """A wrong choice of the kernel takes 10 to 20 times what the bytes need at 6.4 TB/s on
    these, the right one 2 to 4."""
    n, s, c, g = shape
    x, y, dy = (DeviceArray(b200, b200.full((n, s, c), v, np.float32), (n, s, c), np.float32) for v in (0.5, 0, 1))
    w, b, dw, db = (DeviceArray(b200, b200.full((c,), 1, np.float32), (c,), np.float32) for _ in range(4))
    mean, rstd = (DeviceArray(b200, b200.full((n, g), 0.5, np.float32), (n, g), np.float32) for _ in range(2))
    lib, ctx, best = b200._lib, b200._ctx, np.inf
    for _ in range(6):
        ms = C.c_float()
        _lib.check(lib.pb_timer_start(ctx, 0))
        if backward:
            pb.group_norm_backward(dy, x, g, mean, rstd, w, b, activation="silu", out=(y, dw, db))
        else:
            pb.group_norm(x, g, w, b, activation="silu", out=(y, mean, rstd))
        _lib.check(lib.pb_timer_stop(ctx, 0, C.byref(ms)))
        best = min(best, ms.value * 1e3)
    floor = (3 if backward else 2) * n * s * c * 4 / 6.4e6
    assert best <= 7 * floor, f"{best:.1f} us for {floor:.1f}"


def test_the_kernel_timer_counts_the_sums_of_dweight(b200):
    """Many rows of sums for few channels: adding them up is most of the call."""
    n, s, c, g = 2048, 64, 8, 1
    x, y, dy = (DeviceArray(b200, b200.full((n, s, c), v, np.float32), (n, s, c), np.float32) for v in (0.5, 0, 1))
    w, dw = (DeviceArray(b200, b200.full((c,), 1, np.float32), (c,), np.float32) for _ in range(2))
    mean, rstd = (DeviceArray(b200, b200.full((n, g), 0.5, np.float32), (n, g), np.float32) for _ in range(2))
    lib, ctx = b200._lib, b200._ctx
    whole, kernels, count, ms = np.inf, np.inf, C.c_uint64(), C.c_float()
    for timed in [False] * 4 + [True] * 4:
        total = C.c_double()
        _lib.check(lib.pb_ktimer_enable(ctx, 0, 2 if timed else 0))
        _lib.check(lib.pb_timer_start(ctx, 0))
        pb.group_norm_backward(dy, x, g, mean, rstd, w, out=(y, dw, None))
        _lib.check(lib.pb_timer_stop(ctx, 0, C.byref(ms)))
        if timed:
            _lib.check(lib.pb_ktimer_read(ctx, 0, C.byref(total), C.byref(count)))
            assert count.value == 1
            kernels = min(kernels, total.value)
        else:
            whole = min(whole, ms.value)
    _lib.check(lib.pb_ktimer_enable(ctx, 0, 0))
    assert kernels >= whole / 2, (kernels, whole)


@pytest.mark.parametrize("dtype", FLOATS)
def test_silu_is_off_by_its_argument_in_roundings(b200, dtype):
    """As for gelu.  The float32 exponent z log2 e is rounded once (1.3 |z| roundings of
    the result with the constant's own), and the slope's 1 - s is off by up to four of 1."""
    b = np.concatenate([np.linspace(-85, 85, 4001), np.linspace(-0.3, 0.3, 800), [0.0]]).astype(dtype)
    c = b.size
    rng = np.random.default_rng(6)
    u = ref.U[np.dtype(dtype)]
    z = b.astype(np.float64)
    x = rng.standard_normal((1, 1, c)).astype(dtype)
    y, _, _ = pb.group_norm(up(b200, x), 1, up(b200, np.zeros(c, dtype)), up(b200, b), activation="silu")
    want = ref.activate(z, "silu")
    k = u * (ref.ACT + 1.3 * np.abs(z))
    close(y.numpy()[0, 0], want, k * np.abs(want), dtype, "silu")
    stats = [up(b200, v) for v in (np.zeros((1, 1), dtype), np.ones((1, 1), dtype))]
    dy = rng.standard_normal((1, 1, c)).astype(dtype)
    _, _, dbias = pb.group_norm_backward(up(b200, dy), up(b200, x), 1, *stats, up(b200, np.zeros(c, dtype)), up(b200, b),
                                         activation="silu")
    s, rest = ref.sigmoid(z)
    g = np.abs(dy[0, 0].astype(np.float64))
    close(dbias.numpy(), dy[0, 0] * ref.slope(z, "silu"), g * (k * (s + np.abs(s * z) * rest) + 4 * u * np.abs(s * z)),
          dtype, "slope")


# (N, S, C, G) of the ring's further ways: sums of more blocks and groups than each
# block adds up for itself (8192, or 512 groups), with packs and with single values; and
# several rounds of samples, the per-block sums of dweight and dbias carried on.
RINGS = [((1, 20000, 64, 64), np.float32), ((1, 20000, 64, 64), np.float64), ((1, 9000, 1200, 600), np.float32),
         ((1, 9000, 640, 640), np.float64), ((1, 20000, 65, 65), np.float32), ((1, 9000, 1201, 1201), np.float32),
         ((1, 5000, 701, 701), np.float64), ((300, 200, 48, 1), np.float32), ((300, 200, 49, 1), np.float32),
         ((40, 2000, 160, 8), np.float32), ((40, 1000, 160, 8), np.float64), ((700, 700, 13, 1), np.float32),
         ((200, 400, 13, 1), np.float64)]


@pytest.mark.parametrize("shape,dtype", RINGS)
def test_group_norm_in_rounds_and_with_many_group_sums(b200, shape, dtype):
    _check_group_norm(b200, shape, dtype)


def test_group_norm_repeats_its_bits(b200):
    for shape in ((500, 1, 256, 4), (3, 5000, 24, 3)):
        x, w, b, rng = _norm_inputs(shape, np.float32)
        dx, dw, db, dy = (up(b200, v) for v in (x, w, b, rng.standard_normal(x.shape).astype(np.float32)))
        runs = set()
        for _ in range(4):
            y, mean, rstd = pb.group_norm(dx, shape[3], dw, db, activation="silu")
            grads = pb.group_norm_backward(dy, dx, shape[3], mean, rstd, dw, db, activation="silu")
            runs.add(b"".join(q.numpy().tobytes() for q in (y, mean, rstd) + grads))
        assert len(runs) == 1


# ----------------------------------------------------------------- AdamW --


def _adamw_inputs(sizes, dtype, seed=0):
    rng = np.random.default_rng(len(sizes) + seed)
    draw = {"p": lambda n: rng.standard_normal(n), "g": lambda n: rng.standard_normal(n) * 10.0 ** rng.uniform(-6, 2, n),
            "m": lambda n: rng.standard_normal(n) * 0.1, "v": lambda n: rng.standard_normal(n) ** 2 * 1e-2}
    return {k: [f(n).astype(dtype) for n in sizes] for k, f in draw.items()}


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("sizes", [[1], [4096], [3, 0, 1, 2049, 5000, 8192], [(i * 37) % 900 for i in range(70)],
                                   [1 + i % 5 for i in range(1100)], [1 << 20, 7]])
@pytest.mark.parametrize("scale", [None, 0.37])
def test_adamw(b200, sizes, dtype, scale):
    u = ref.U[np.dtype(dtype)]
    a = _adamw_inputs(sizes, dtype)
    d = {k: [up(b200, x) for x in v] for k, v in a.items()}
    opt = pb.AdamW(d["p"], lr=0.02, betas=(0.9, 0.99), eps=1e-6, weight_decay=0.1, exp_avg=d["m"], exp_avg_sq=d["v"],
                   steps=4)
    s = None if scale is None else np.array([scale], dtype)
    opt.step(d["g"], grad_scale=up(b200, s))
    assert opt.steps == 5
    for j in range(len(sizes)):
        want, bounds = ref.adamw(*(a[k][j] for k in "pgmv"), 1.0 if s is None else float(s[0]), 0.02, (0.9, 0.99), 1e-6,
                                 0.1, 5, u)
        for k, w, e in zip("pmv", want, bounds):
            close(d[k][j].numpy(), w, e, dtype, f"{k}[{j}]")


@pytest.mark.parametrize("dtype", FLOATS)
def test_adamw_step_on_the_callers_lists(b200, dtype):
    """The optimizer's bits, from lists and a step number that the caller keeps."""
    sizes = [3, 0, 2049, 8192]
    a = _adamw_inputs(sizes, dtype)
    mine, its = ({k: [up(b200, x) for x in v] for k, v in a.items()} for _ in range(2))
    scale = up(b200, np.array([0.37], dtype))
    opt = pb.AdamW(its["p"], lr=0.02, betas=(0.9, 0.99), eps=1e-6, weight_decay=0.1, exp_avg=its["m"],
                   exp_avg_sq=its["v"], steps=4)
    for step in (5, 6):
        pb.adamw_step(mine["p"], mine["g"], mine["m"], mine["v"], step=step, lr=0.02, betas=(0.9, 0.99), eps=1e-6,
                      weight_decay=0.1, grad_scale=scale)
        opt.step(its["g"], grad_scale=scale)
    for k in "pmv":
        for x, y, old in zip(mine[k], its[k], a[k]):
            assert x.numpy().tobytes() == y.numpy().tobytes()
            assert not x.size or x.numpy().tobytes() != old.tobytes()


@pytest.mark.parametrize("dtype", FLOATS)
def test_adamw_views_at_odd_places_leave_their_neighbours(b200, dtype):
    """Tensors inside one buffer that start anywhere (the C entry asks only for
    whole elements): what lies between them stays as it was."""
    rng = np.random.default_rng(8)
    spans = [(1, 3), (5, 4097), (4103, 2048), (6152, 1), (6154, 9000)]
    n, item = 16000, np.dtype(dtype).itemsize
    host = {k: rng.uniform(0.1, 1.0, n).astype(dtype) for k in "pgmv"}
    dev = {k: up(b200, x) for k, x in host.items()}
    table = [(C.c_void_p * 5)(*[dev[k]._data.ptr + at * item for at, _ in spans]) for k in "pgmv"]
    _lib.check(b200._lib.pb_adamw(b200._ctx, 0, _lib.dtype_code(dtype), 5, *table,
                                  (C.c_int64 * 5)(*[m for _, m in spans]), 0.1, 0.9, 0.99, 1e-8, 0.0, 1, None))
    want, bounds = ref.adamw(*(host[k] for k in "pgmv"), 1.0, 0.1, (0.9, 0.99), 1e-8, 0.0, 1, ref.U[np.dtype(dtype)])
    live = np.zeros(n, bool)
    for at, m in spans:
        live[at:at + m] = True
    for k, w, e in zip("pmv", want, bounds):
        got = dev[k].numpy()
        close(got[live], w[live], e[live], dtype, k)
        assert got[~live].tobytes() == host[k][~live].tobytes()
    assert dev["g"].numpy().tobytes() == host["g"].tobytes()


def test_adamw_refuses_a_tensor_given_twice_and_a_capture(b200):
    p = up(b200, np.ones(8, np.float32))
    g = up(b200, np.ones(8, np.float32))
    with pytest.raises(ValueError, match="overlap"):
        pb.AdamW([p, p]).step([g, g])
    with pytest.raises(ValueError, match="overlap"):
        pb.AdamW([p]).step([p])
    opt = pb.AdamW([p])
    with pytest.raises(NotImplementedError, match="captur"):
        b200.capture(lambda: opt.step([g]))
    assert opt.steps == 0 and np.all(p.numpy() == 1)
    opt.step([g])
    assert opt.steps == 1 and np.all(p.numpy() < 1)


# ------------------------------------------ together, captured, other streams


def test_calls_in_a_graph(b200):
    """A captured step with `out` gives the eager bits, on new contents too, and
    keeps its state from replay to replay."""
    shape = (2, 3000, 64)
    a, b, state, rng = _recurrence_inputs(shape, np.float32, "sigmoid")
    da, db, keep = up(b200, a), up(b200, b), up(b200, state)
    h, y = (poisoned(b200, shape, np.float32) for _ in range(2))
    stats = [poisoned(b200, (2, 4), np.float32) for _ in range(2)]
    dx = poisoned(b200, shape, np.float32)
    grads = [poisoned(b200, v, np.float32) for v in (shape, shape, state.shape)]

    def step():
        pb.linear_recurrence(da, db, state=keep, final=keep, gate="sigmoid", out=h)
        pb.group_norm(h, 4, activation="silu", out=(y, *stats))
        pb.group_norm_backward(y, h, 4, *stats, activation="silu", out=(dx, None, None))
        pb.linear_recurrence_backward(da, db, h, dx, gate="sigmoid", out=tuple(grads))

    outs = [h, y, dx, keep] + stats + grads
    step()
    eager = [[o.numpy() for o in outs]]
    step()
    eager.append([o.numpy() for o in outs])

    def reset():
        _lib.check(b200._lib.pb_h2d(b200._ctx, 0, keep._data.ptr, state.ctypes.data, state.nbytes, 1))

    reset()
    with b200.capture(step) as graph:
        assert graph.launches >= 4
        for turn in range(2):
            graph.launch()
            for want, o in zip(eager[turn], outs):
                assert o.numpy().tobytes() == want.tobytes()
        # Two graphs that share the library's workspaces, in turn.
        with b200.capture(step) as other:
            reset()
            graph.launch()
            other.launch()
            for want, o in zip(eager[1], outs):
                assert o.numpy().tobytes() == want.tobytes()


def test_a_capture_that_would_grow_a_workspace_is_refused(b200):
    x = up(b200, np.ones((3, 40000, 96), np.float32))
    out = tuple(poisoned(b200, v, np.float32) for v in (x.shape, (3, 4), (3, 4)))
    b200.release_cached_memory()
    try:
        with b200.capture(lambda: pb.group_norm(x, 4, out=out)):
            pass
    except NotImplementedError as exc:
        assert "grow" in str(exc)
    pb.group_norm(x, 4, out=out)
    assert np.all(out[0].numpy() == 0)


def test_a_capture_that_grows_a_workspace_raises(b200):
    x = up(b200, np.ones((3, 40000, 96), np.float32))
    out = tuple(poisoned(b200, v, np.float32) for v in (x.shape, (3, 4), (3, 4)))
    b200.release_cached_memory()
    with pytest.raises(NotImplementedError, match="grow"):
        b200.capture(lambda: pb.group_norm(x, 4, out=out))
    pb.group_norm(x, 4, out=out)
    assert np.all(out[0].numpy() == 0)


def test_arrays_of_torch_on_a_stream_of_its_own(b200):
    torch = pytest.importorskip("torch")
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        a = torch.zeros(2, 500, 96, device="cuda")
        for _ in range(50):
            a.add_(0.01)
        b = torch.ones_like(a)
        h = torch.empty_like(a)
        va, vb, vh = (b200.view(t, stream=side.cuda_stream) for t in (a, b, h))
        pb.linear_recurrence(va, vb, out=vh)
        b200.signal_stream(side.cuda_stream)
        last = h[:, -1].cpu().numpy()
    assert np.allclose(last, 2.0, rtol=1e-4)  # 1 / (1 - 1/2)


def _gather(b200, x, shape, offset, strides):
    return DeviceArray(b200, b200.gather(x, shape, offset, strides), shape, x.dtype)


def _matmul(b200, a, b):
    shape = a.shape[:-1] + b.shape[-1:]
    return DeviceArray(b200, b200.matmul(a, b, shape, a.dtype), shape, a.dtype)


def _transpose(b200, a):
    r, c = a.shape
    return _gather(b200, a, (c, r), 0, (1, c))


def _layer(b200, x, w, gamma, beta):
    """x @ W gives logits and inputs; recurrence; per-head norm with silu."""
    n, t, _ = x.shape
    c = w.shape[1] // 2
    z = _matmul(b200, DeviceArray(b200, x._data, (n * t, x.shape[2]), x.dtype), w)
    gate, put = (_gather(b200, z, (n, t, c), k * c, (t * 2 * c, 2 * c, 1)) for k in (0, 1))
    h = pb.linear_recurrence(gate, put, gate="sigmoid")
    flat = DeviceArray(b200, h._data, (n * t, c), h.dtype)
    y, mean, rstd = pb.group_norm(flat, 4, gamma, beta, activation="silu")
    return y, (gate, put, h, flat, mean, rstd)


def test_a_training_step_of_a_layer(b200):
    """Forward, gradients against differences of the loss, and an AdamW step
    that lowers it by what the gradient says (float64 throughout)."""
    rng = np.random.default_rng(11)
    n, t, d, c = 2, 300, 12, 16
    x, w = rng.standard_normal((n, t, d)), rng.standard_normal((d, 2 * c)) * 0.4
    gamma, beta, goal = 1 + 0.1 * rng.standard_normal(c), 0.1 * rng.standard_normal(c), rng.standard_normal((n * t, c))
    dx = up(b200, x)

    def loss(w, gamma, beta):
        y, _ = _layer(b200, dx, up(b200, w), up(b200, gamma), up(b200, beta))
        return float(np.sum((y.numpy() - goal) ** 2) / 2)

    dw_, dg_, db_ = up(b200, w), up(b200, gamma), up(b200, beta)
    y, (gate, put, h, flat, mean, rstd) = _layer(b200, dx, dw_, dg_, db_)
    dy = DeviceArray(b200, b200.elementwise("subtract", [y, up(b200, goal)], y.shape, np.float64), y.shape, np.float64)
    dflat, dgamma, dbeta = pb.group_norm_backward(dy, flat, 4, mean, rstd, dg_, db_, activation="silu")
    dgate, dput, _ = pb.linear_recurrence_backward(gate, put, h, DeviceArray(b200, dflat._data, h.shape, h.dtype),
                                                   gate="sigmoid")
    xt = _transpose(b200, DeviceArray(b200, dx._data, (n * t, d), dx.dtype))
    halves = [_matmul(b200, xt, DeviceArray(b200, g._data, (n * t, c), g.dtype)).numpy() for g in (dgate, dput)]
    grads = [np.concatenate(halves, 1), dgamma.numpy(), dbeta.numpy()]
    values = [w, gamma, beta]
    for k, grad in enumerate(grads):
        direction = rng.standard_normal(grad.shape)
        step = 1e-5

        def at(e):
            return loss(*[v + e * direction if i == k else v for i, v in enumerate(values)])

        slope = (at(step) - at(-step)) / (2 * step)
        # Central differences: third derivatives times step^2, and the loss's rounding over step.
        assert abs(slope - np.sum(grad * direction)) <= 1e-5 * np.sum(np.abs(grad * direction)), k
    params = [dw_, dg_, db_]
    opt = pb.AdamW(params, lr=1e-3, weight_decay=0.01)
    opt.step([up(b200, g) for g in grads])
    for v, g, p in zip(values, grads, params):
        want, bound = ref.adamw(v, g, np.zeros_like(v), np.zeros_like(v), 1.0, 1e-3, (0.9, 0.999), 1e-8, 0.01, 1,
                                2.0 ** -53)
        close(p.numpy(), want[0], bound[0], np.float64, "parameter")


def test_serving_token_by_token_gives_the_whole_sequence(b200):
    """A prompt at once, then single tokens with the kept state, against the whole
    sequence in one call."""
    n, t, c = 3, 200, 64
    a, b, state, _ = _recurrence_inputs((n, t, c), np.float32, "sigmoid")
    want = ref.recurrence(a, b, state, "sigmoid", 2.0 ** -24)
    keep = up(b200, state)
    rows, prompt = [], 150
    h = pb.linear_recurrence(up(b200, a[:, :prompt].copy()), up(b200, b[:, :prompt].copy()), state=keep, final=keep,
                             gate="sigmoid")
    rows.append(h.numpy())
    out = poisoned(b200, (n, 1, c), np.float32)
    for k in range(prompt, t):
        pb.linear_recurrence(up(b200, a[:, k:k + 1].copy()), up(b200, b[:, k:k + 1].copy()), state=keep, final=keep,
                             gate="sigmoid", out=out)
        rows.append(out.numpy())
    close(np.concatenate(rows, 1), *want, np.float32, "tokens")


@pytest.mark.parametrize("dtype", FLOATS)
def test_recurrence_in_several_windows(b200, dtype):
    """Few columns, more operands than fit L2: the chain is read in windows."""
    n, c = (300001, 32) if dtype == np.float32 else (150001, 32)
    rng = np.random.default_rng(12)
    a = rng.uniform(0.5, 1.0, (1, n, c)).astype(dtype)
    b = rng.standard_normal((1, n, c)).astype(dtype)
    state = rng.standard_normal((1, c)).astype(dtype)
    keep = up(b200, state)
    da, db = up(b200, a), up(b200, b)
    h = pb.linear_recurrence(da, db, state=keep, final=keep)
    got = h.numpy()
    want, bound = ref.recurrence(a, b, state, "linear", ref.U[np.dtype(dtype)])
    close(got, want, bound, dtype, "h")
    assert keep.numpy().tobytes() == got[:, -1].tobytes()
    dh = rng.standard_normal(a.shape).astype(dtype)
    grads = pb.linear_recurrence_backward(da, db, h, up(b200, dh), state=up(b200, state))
    want, bounds = ref.recurrence_backward(a, b, got, dh, state, None, "linear", ref.U[np.dtype(dtype)])
    for name, g, w, e in zip(("da", "db", "dstate"), grads, want, bounds):
        close(g.numpy(), w, e, dtype, name)


@pytest.mark.parametrize("shape", [(1, 20000, 64), (1, 20000, 1600), (1, 3000, 9000), (1, 60, 50000)])
@pytest.mark.parametrize("dtype", FLOATS)
def test_recurrence_resets_behind_growth_and_poison_behind_zeros(b200, shape, dtype):
    """A zero gate forgets whatever follows it in the product; a gate that is not
    finite leaves nothing finite behind it, even where all it meets is zero."""
    _, n, c = shape
    a, b = np.full(shape, 2.0, dtype), np.zeros(shape, dtype)
    reset, tail = n // 2, n - 25
    a[0, reset] = 0.0
    a[0, tail:] = 0.5
    b[0, tail] = 1.0
    state = np.ones((1, c), dtype)
    state[0, 1::2] = 0.0
    h = pb.linear_recurrence(up(b200, a), up(b200, b), state=up(b200, state)).numpy()
    # Powers of two: the recurrence itself in the type is exact.  A column that
    # has grown to Inf is NaN from the reset on (0 * Inf).
    want, x = np.empty_like(h), state.copy()
    with np.errstate(all="ignore"):
        for t in range(n):
            x = a[:, t] * x + b[:, t]
            want[:, t] = x
    finite = np.isfinite(want)
    assert np.array_equal(h[finite], want[finite]) and not np.isfinite(h[~finite]).any()
    assert finite[0, :, 1::2].all() and np.array_equal(h[0, tail:, 1], (0.5 ** np.arange(25)).astype(dtype))
    a[0] = 0.5
    b[0] = 0.0
    a[0, 7, 3], a[0, 7, 5] = np.nan, np.inf
    h = pb.linear_recurrence(up(b200, a), up(b200, b)).numpy()
    assert not np.isfinite(h[0, 7:, [3, 5]]).any() and np.array_equal(np.delete(h[0], [3, 5], 1), np.zeros((n, c - 2)))


# ---------------------------------------------------- offsets beyond 32 bits


@pytest.mark.parametrize("steps,width", [(8200, 131072), (16400, 65600), (262500, 4100)])
def test_recurrence_beyond_4_gib(b200, steps, width):
    """Arrays above 4 GiB on the three ways a chain is walked: constant gates, whose
    sums are known."""
    torch = pytest.importorskip("torch")
    a = torch.full((1, steps, width), 0.5, device="cuda")
    b = torch.empty_like(a)
    b.copy_(torch.arange(width, device="cuda", dtype=torch.float32).remainder_(7).add_(1.0))
    h, g = torch.empty_like(a), torch.empty_like(a)
    va, vb, vh, vg = (b200.view(t) for t in (a, b, h, g))
    final = b200.view(torch.empty(1, width, device="cuda"))
    pb.linear_recurrence(va, vb, out=vh, final=final)
    # h -> 2 b; da = g h[t-1] = 2 * 2 b, db = g = 2 far from both ends.
    pb.linear_recurrence_backward(va, None, vh, va, out=(vb, vg, final))
    b200.synchronize()
    want = torch.arange(width, device="cuda", dtype=torch.float32).remainder_(7).add_(1.0) * 2
    for t in (100, steps // 2, steps - 1):
        assert torch.allclose(h[0, t], want, rtol=1e-6), t
    for t in (100, steps // 2, steps - 100):
        assert torch.allclose(g[0, t], torch.ones_like(want), rtol=1e-6), t  # dh = 0.5: g = 1
        assert torch.allclose(b[0, t], want, rtol=1e-6), t


@pytest.mark.parametrize("shape,groups", [((2, (1 << 20) + 5, 1026), 3), ((2, 1 << 20, 1032), 8), ((1 << 21, 1, 1028), 2)])
def test_group_norm_beyond_32_bits(b200, shape, groups):
    """More than 2^31 values, on each kernel; the last sample against torch."""
    torch = pytest.importorskip("torch")
    x = torch.empty(shape, device="cuda").normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    y = torch.empty_like(x)
    stats = [torch.empty(shape[0], groups, device="cuda") for _ in range(2)]
    pb.group_norm(b200.view(x), groups, activation="relu", out=tuple(b200.view(t) for t in (y, *stats)))
    b200.synchronize()
    last = x[-1].reshape(shape[1], groups, -1).double()
    mean = last.mean((0, 2), keepdim=True)
    want = ((last - mean) / (last.var((0, 2), unbiased=False, keepdim=True) + 1e-5).sqrt()).clamp(min=0)
    assert (y[-1].reshape_as(want) - want).abs().max().item() <= 1e-5
    del last, want
    # dx of dy = 1 without weight and activation is 0 up to rounding.
    x.fill_(1.0)
    x[..., ::2] = -1.0
    pb.group_norm(b200.view(x), groups, out=tuple(b200.view(t) for t in (y, *stats)))
    dy = torch.ones_like(x)
    pb.group_norm_backward(b200.view(dy), b200.view(x), groups, *(b200.view(t) for t in stats),
                           out=(b200.view(y), None, None))
    b200.synchronize()
    assert y[-1].abs().max().item() <= 1e-5 and y[0].abs().max().item() <= 1e-5


def test_two_contexts_at_once(b200):
    """Kernels whose blocks wait for one another, from two threads on two streams
    of one GPU: each is launched whole, so neither waits for the other."""
    shapes = [(2, 2048, 320, 32), (2, 4096, 20, 4), (3, 1517, 90, 9)]
    backends = [pb.B200Backend(), pb.B200Backend()]
    failed = []

    def work(backend, seed):
        try:
            rng = np.random.default_rng(seed)
            sets = []
            for n, s, c, g in shapes:
                x, dy = (up(backend, rng.standard_normal((n, s, c)).astype(np.float32)) for _ in range(2))
                w, b = (up(backend, rng.standard_normal(c).astype(np.float32)) for _ in range(2))
                sets.append((x, dy, g, w, b))
            first = None
            for _ in range(15):
                bits = []
                for x, dy, g, w, b in sets:
                    y, mean, rstd = pb.group_norm(x, g, w, b, activation="silu")
                    grads = pb.group_norm_backward(dy, x, g, mean, rstd, w, b, activation="silu")
                    h = pb.linear_recurrence(x, dy, gate="sigmoid")
                    bits += [v.numpy().tobytes() for v in (y, mean, rstd, h) + grads]
                first = first or bits
                assert bits == first
        except BaseException as e:  # noqa: BLE001 - reported by the test's own thread
            failed.append(e)

    threads = [threading.Thread(target=work, args=(b, i)) for i, b in enumerate(backends)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for b in backends:
        b.close()
    assert not failed, failed[0]
