"""Layer norm and its gradients on the device against the formulas in 64 bits."""
import numpy as np
import pytest

from langhelp import *
from recpulse_amd import capi

pytestmark = pytest.mark.gpu
EPS = 1e-5

# a wave's rows, a workgroup's, rows that end inside a vector, one that is shorter than a vector, one element, and widths on either side of each kind of team
SIZES = [(1, 1), (3, 2), (5, 7), (1, 8), (4, 64), (7, 513), (300, 96), (2, 1031), (33, 2048), (6, 2049), (3, 4096), (2, 5001), (2, 9001), (1, 16384), (2, 40000), (1, 70001)]


def forward(x, w, b, dtype, y_rs=None, stats=True, eps=EPS):
    rows, d = x.shape
    y = Output(rows, d, dtype, y_rs)
    st = Output(rows, 2, ACC[dtype]) if stats else None
    capi.check(capi.lib().rp_hip_layer_norm_forward(y.ptr, at(st), x.ptr, at(w), at(b), rows, d, y.rs, x.rs, eps, dtype), "rp_hip_layer_norm_forward")
    return y, st


def bounds(x, w, b, dtype):
    """What the sums' order and the roundings of the values between can change: a sum of d values by teams of 64 to 1024 adds fewer than 100 of them one after the other."""
    mean, r, h, y = norm_reference(x, w, b, EPS)
    u, ww = UNIT[dtype], 1.0 if w is None else np.abs(w)
    steps = 100 + x.shape[1] / 256                              # (rows longer than registers: 256 threads walk them)
    size = np.abs(x).mean(1, keepdims=True)
    off_mean = steps * u * size
    off_h = r * (off_mean + 4 * u * np.abs(x)) + steps * u * np.abs(h) + np.abs(h) * (off_mean * r) ** 2
    return mean, r, h, y, off_h, off_h * ww + 4 * u * (np.abs(h) * ww + np.abs(0.0 if b is None else b))


@pytest.mark.parametrize("dtype", ALL, ids=NAMES.get)
@pytest.mark.parametrize("rows,d", SIZES)
def test_forward(rows, d, dtype):
    rng = np.random.default_rng(d * 7 + rows)
    x = Operand(rng.normal(1.5, 2.0, (rows, d)), dtype)
    w, b = (vector(1 + 0.3 * rng.normal(size=d), dtype), vector(rng.normal(size=d), dtype)) if d % 2 else (None, None)
    y, stats = forward(x, w, b, dtype, y_rs=d + 3 if rows > 1 else None)
    mean, r, h, want, _, off = bounds(x.values, w and w.values, b and b.values, dtype)
    assert_within(y.read(), want, rounded(off, want, dtype), "y")
    got = stats.read()
    steps = 100 + d / 256
    assert_within(got[:, :1], mean, steps * UNIT[dtype] * np.abs(x.values).mean(1, keepdims=True), "mean")
    assert_within(got[:, 1:], r, r * (steps * UNIT[dtype] * 2 + (steps * UNIT[dtype] * np.abs(x.values).mean(1, keepdims=True) * r) ** 2), "1 / deviation")


@pytest.mark.parametrize("dtype", ALL, ids=NAMES.get)
@pytest.mark.parametrize("rows,d", SIZES + [(2000, 40), (1500, 3), (700, 1024)])
def test_backward(rows, d, dtype):
    rng = np.random.default_rng(d * 5 + rows)
    x, dy = Operand(rng.normal(-1.0, 1.5, (rows, d)), dtype, rs=d + 5), Operand(rng.normal(size=(rows, d)), dtype, rs=d + 1)
    w = vector(1 + 0.3 * rng.normal(size=d), dtype) if (rows + d) % 2 else None
    mean, r, h, _, off_h, _ = bounds(x.values, w and w.values, None, dtype)
    stats = Operand(np.concatenate([mean, r], 1), ACC[dtype])
    accumulate = rows % 2
    start = [rng.normal(size=s) if accumulate else None for s in ((rows, d), (1, d), (1, d))]
    dx, dw, db = Output(rows, d, dtype, d + 2, start=start[0]), Output(1, d, dtype, start=start[1]), Output(1, d, dtype, start=start[2])
    was = [o.values if accumulate else 0.0 for o in (dx, dw, db)]
    size = capi.lib().rp_hip_layer_norm_workspace(rows, d, dtype)
    space = room(size)
    capi.check(capi.lib().rp_hip_layer_norm_backward(dx.ptr, dw.ptr, db.ptr, dy.ptr, x.ptr, at(w), stats.ptr, space.ptr, rows, d, dy.rs, x.rs, dx.rs, accumulate, accumulate, accumulate, dtype),
               "rp_hip_layer_norm_backward")
    u, steps = UNIT[dtype], 100 + d / 256
    ww = 1.0 if w is None else w.values
    g = dy.values * ww
    want = r * (g - g.mean(1, keepdims=True) - h * (g * h).mean(1, keepdims=True))
    # stats are rounded to the accumulate type: h is off by u |h| and u r |mean|
    off_h = 6 * u * (np.abs(h) + r * np.abs(mean) + r * np.abs(x.values))
    mean_off = steps * u * np.abs(g).mean(1, keepdims=True)
    cross_off = (steps * u * np.abs(g * h) + np.abs(g) * off_h).mean(1, keepdims=True)
    off = r * (4 * u * np.abs(g) + mean_off + off_h * np.abs((g * h).mean(1, keepdims=True)) + np.abs(h) * cross_off) + 6 * u * np.abs(want)
    off = off + u * np.abs(was[0])
    assert_within(dx.read(), want + was[0], rounded(off, want + was[0], dtype), "dx")
    terms = dy.values * h
    steps = rows + 120
    for out, want, off, old, what in ((dw, terms.sum(0), (steps * u * np.abs(terms) + np.abs(dy.values) * off_h).sum(0), was[1], "dw"), (db, dy.values.sum(0), steps * u * np.abs(dy.values).sum(0), was[2], "db")):
        assert_within(out.read(), want + old, rounded(off + u * np.abs(old), want + old, dtype), what)


@pytest.mark.parametrize("asked", ["dx", "dw", "db"])
@pytest.mark.parametrize("d", [96, 1031, 4096, 5])
def test_an_output_does_not_depend_on_the_others(asked, d):
    rng = np.random.default_rng(d)
    rows, dtype = 37, BF16
    x, dy, w = Operand(rng.normal(size=(rows, d)), dtype), Operand(rng.normal(size=(rows, d)), dtype), vector(rng.normal(size=d), dtype)
    _, stats = forward(x, w, None, dtype)
    space = room(capi.lib().rp_hip_layer_norm_workspace(rows, d, dtype))
    results = []
    for names in (("dx", "dw", "db"), (asked,)):
        out = {"dx": Output(rows, d, dtype), "dw": Output(1, d, dtype), "db": Output(1, d, dtype)}
        p = {n: out[n].ptr if n in names else None for n in out}
        capi.check(capi.lib().rp_hip_layer_norm_backward(p["dx"], p["dw"], p["db"], dy.ptr, x.ptr, w.ptr, stats.ptr, space.ptr, rows, d, d, d, d, 0, 0, 0, dtype), "backward")
        results.append(out[asked].bits())
        for n in out:
            if n not in names:
                assert np.all(out[n].read() == MARK)
    assert np.array_equal(*results)


def test_rows_far_from_zero_keep_their_variance():
    """Differences of one around a mean of 4096: the sum of squares less the square of the sum would have no digit left."""
    rng = np.random.default_rng(3)
    x = Operand(4096 + rng.normal(size=(4, 1000)), F32)
    y, _ = forward(x, None, None, F32)
    _, _, _, want, off, _ = bounds(x.values, None, None, F32)
    assert off.max() < 0.05
    assert_within(y.read(), want, rounded(off, want, F32), "y")


def test_constant_rows_are_zeros_and_not_finite_ones_stay_in_their_row():
    x = np.full((4, 520), 3.0)
    x[1, 7] = np.inf
    x[2, 9] = np.nan
    x = Operand(x, BF16)
    y, _ = forward(x, None, None, BF16)
    got = y.read()
    assert np.all(got[[0, 3]] == 0) and np.all(np.isnan(got[2])) and np.all(np.isnan(got[1]))


def test_gradient_agrees_with_differences():
    rng = np.random.default_rng(11)
    rows, d, eps, step = 3, 37, 1e-3, 1e-5
    x, w, c = rng.normal(size=(rows, d)), rng.normal(size=d), rng.normal(size=(rows, d))

    def value(xv, wv):
        y, _ = forward(Operand(xv, F64), vector(wv, F64), None, F64, eps=eps)
        return (y.read() * c).sum()

    xo = Operand(x, F64)
    _, stats = forward(xo, vector(w, F64), None, F64, eps=eps)
    dx, dw = Output(rows, d, F64), Output(1, d, F64)
    space = room(capi.lib().rp_hip_layer_norm_workspace(rows, d, F64))
    capi.check(capi.lib().rp_hip_layer_norm_backward(dx.ptr, dw.ptr, None, Operand(c, F64).ptr, xo.ptr, vector(w, F64).ptr, stats.ptr, space.ptr, rows, d, d, d, d, 0, 0, 0, F64), "backward")
    for i, j in ((0, 0), (1, 20), (2, 36)):
        e = np.zeros((rows, d))
        e[i, j] = step
        # a central difference is off by step^2 / 6 times the third derivative (below 100 here) and 1e-13 / step
        assert abs((value(x + e, w) - value(x - e, w)) / (2 * step) - dx.read()[i, j]) < 1e-7
        assert abs((value(x, w + e[i]) - value(x, w - e[i])) / (2 * step) - dw.read()[0, j]) < 1e-7


def test_recorded_calls_replay_to_the_eager_result():
    rng = np.random.default_rng(5)
    rows, d, dtype = 65, 1031, F16
    x, dy, w = Operand(rng.normal(size=(rows, d)), dtype), Operand(rng.normal(size=(rows, d)), dtype), vector(rng.normal(size=d), dtype)
    y, dx, dw, db, stats = Output(rows, d, dtype), Output(rows, d, dtype), Output(1, d, dtype), Output(1, d, dtype), Output(rows, 2, F32)
    space = room(capi.lib().rp_hip_layer_norm_workspace(rows, d, dtype))

    def step():
        capi.check(capi.lib().rp_hip_layer_norm_forward(y.ptr, stats.ptr, x.ptr, w.ptr, None, rows, d, d, d, EPS, dtype), "forward")
        capi.check(capi.lib().rp_hip_layer_norm_backward(dx.ptr, dw.ptr, db.ptr, dy.ptr, x.ptr, w.ptr, stats.ptr, space.ptr, rows, d, d, d, d, 0, 0, 0, dtype), "backward")

    step()
    eager = [o.bits() for o in (y, dx, dw, db)]
    with capi.Stream() as s:
        with capi.Graph.capture() as graph:
            step()
        for _ in range(3):
            for o in (y, dx, dw, db):
                capi.check(capi.lib().rp_hip_memset(o.buf.ptr, 0, o.buf.nbytes), "memset")
            capi.synchronize()
            graph.launch()
            capi.check(capi.lib().rp_hip_stream_synchronize(), "sync")
            assert all(np.array_equal(a, o.bits()) for a, o in zip(eager, (y, dx, dw, db)))
