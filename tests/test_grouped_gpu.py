"""Layers whose weight depends on the row, on the GPU, against plain implementations in 64 bits: routing and its sort, the exchange
of rows, the grouped linear layer, the adapters, and a run of them together.

Tolerances, elementwise: a sum of `terms` products in the accumulate type is off by at most (terms + 8) u times the sum of the
products' magnitudes, u = 2^-24 (2^-53), and each rounding to the tensor type by at most half a step, eps / 2 of the value (2^-25 below
float16's normal numbers).  The oracle's own sums in float64 are off by as much with u = 2^-53, which the factor 2 on u covers there.
"""
import ctypes

import numpy as np
import pytest

import oracle
from recpulse_amd import capi
from devhelp import ALL, BF16, F16, F32, F64, NAMES, Dev, rand_storage

pytestmark = pytest.mark.gpu

HALF_STEP = {F32: 2.0 ** -24, F64: 2.0 ** -53, F16: 2.0 ** -11, BF16: 2.0 ** -8}
UNIT = {F32: 2.0 ** -24, F64: 2.0 ** -52, F16: 2.0 ** -24, BF16: 2.0 ** -24}
TINY = {F32: 0.0, F64: 0.0, F16: 2.0 ** -25, BF16: 0.0}


def ids_of(dt):
    return NAMES[dt]


def within(got, want, magnitude, terms, dt, roundings=1, added=0.0):
    """got and want float64; magnitude: the sum of the products' magnitudes; added: what the rounded product (want - added) was added to,
    which is a rounding of the product's value and one of the sum's."""
    fine = np.isfinite(want)
    assert np.array_equal(np.isfinite(got), fine) and np.array_equal(np.isnan(got), np.isnan(want))
    value = np.abs(want) + (np.abs(want - added) if added else 0.0)
    bound = roundings * (HALF_STEP[dt] * value * (1 + HALF_STEP[dt]) + 2 * TINY[dt]) + (terms + 8) * UNIT[dt] * magnitude * (1 + HALF_STEP[dt])
    worst = np.max(np.where(fine, np.abs(np.where(fine, got - want, 0)) - bound, -1.0), initial=-1.0)
    assert worst <= 0, f"{worst} beyond the bound"


def ints(a):
    return capi.DeviceBuffer.from_numpy(np.ascontiguousarray(a, dtype=np.int32))


def read_ints(buf, shape):
    capi.synchronize()
    return buf.to_numpy(np.int32, shape)


def call(name, *args):
    capi.check(getattr(capi.lib(), name)(*args), name)


def ptr(x):
    return None if x is None else x.ptr


def cuts(rng, rows, parts, empty=(), behind=0):
    """Offsets of `parts` uneven groups over rows - behind rows; the groups named in `empty` hold none."""
    share = np.exp(0.5 * rng.normal(0, 1, parts))
    share[list(empty)] = 0
    sizes = rng.multinomial(rows - behind, share / share.sum())
    return np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)


# ---- routing -----------------------------------------------------------------------------------------------------------

def weight_dt(dt):
    return F64 if dt == F64 else F32


def route_want(logits, k, normalize):
    """experts, weights, offsets, order, position from float64 logits."""
    t, e = logits.shape
    key = np.where(np.isnan(logits), np.inf, logits)
    rank = np.lexsort((np.broadcast_to(np.arange(e), (t, e)), -key, ~np.isnan(logits)), axis=1)[:, :k]        # NaN first, then by value, then by index
    picked = ~(np.take_along_axis(logits, rank, 1) == -np.inf)
    with np.errstate(invalid="ignore", divide="ignore"):
        best = np.take_along_axis(logits, rank, 1)
        top = np.where(picked[:, :1], best[:, :1], 0)
        ex = np.where(picked, np.exp(best - top), 0)
        total = ex.sum(1, keepdims=True) if normalize else np.where(logits == -np.inf, 0, np.exp(logits - top)).sum(1, keepdims=True)
        weights = np.where(picked, ex / np.where(total == 0, 1, total), 0)
    experts = np.where(picked, rank, -1)
    return (experts, weights) + sort_want(experts.reshape(-1), e)


def sort_want(ids, groups):
    inside = (ids >= 0) & (ids < groups)
    slots = np.flatnonzero(inside)
    order = slots[np.argsort(ids[slots], kind="stable")]
    offsets = np.concatenate([[0], np.cumsum(np.bincount(ids[slots], minlength=groups))])
    position = np.full(ids.size, -1)
    position[order] = np.arange(order.size)
    return offsets, np.concatenate([order, np.full(ids.size - order.size, -1)]), position


def route(dlogits, rs, t, e, k, normalize, dt):
    w = Dev.empty((t, k), weight_dt(dt))
    bufs = [capi.DeviceBuffer(4 * n) for n in (t * k, e + 1, t * k, t * k)]
    call("rp_hip_route_forward", w.ptr, *[b.ptr for b in bufs], dlogits.ptr, rs, t, e, k, int(normalize), dt)
    return w, bufs


def special_rows(logits, rng):
    """The rows where a routing can go wrong, as far as there are rows: nothing left, fewer than k left, ties, zeros of both signs, infinity, NaN."""
    t, e = logits.shape
    for i, fill in enumerate(("none", "one", "ties", "zeros", "inf", "nan")):
        if i + 1 >= t:
            return
        row = logits[i + 1]
        if fill == "none":
            row[:] = -np.inf
        elif fill == "one":
            row[:] = -np.inf
            row[e // 2] = 0.5
        elif fill == "ties":
            row[:] = 1.0
            row[: e // 3] = 0.25
        elif fill == "zeros":
            row[:] = np.where(np.arange(e) % 2, 0.0, -0.0)
        elif fill == "inf":
            row[e - 1] = np.inf
        else:
            row[e // 2] = np.nan
            row[0] = np.inf


@pytest.mark.parametrize("normalize", [True, False], ids=["among-k", "among-all"])
@pytest.mark.parametrize("dt", ALL, ids=ids_of)
@pytest.mark.parametrize("t, e, k", [(1, 1, 1), (1, 64, 6), (7, 5, 5), (16, 65, 8), (17, 300, 3), (64, 128, 2), (65, 17, 4), (300, 256, 16), (700, 1000, 7), (5000, 130, 2), (40000, 8, 2)])
def test_route(t, e, k, dt, normalize):
    rng = np.random.default_rng(7 * t + e)
    values = rng.normal(0, 2, (t, e))
    values[rng.random((t, e)) < 0.05] = -np.inf
    special_rows(values, rng)
    wide = oracle.to_storage(np.concatenate([values, np.full((t, 3), 100.0)], 1), dt)         # rows further apart than they are long
    logits = oracle.to_f64(wide, dt)[:, :e]
    d = Dev(wide, dt)
    w, (experts, offsets, order, position) = route(d, e + 3, t, e, k, normalize, dt)
    want = route_want(logits, k, normalize)
    assert np.array_equal(read_ints(experts, (t, k)), want[0])
    for got, ref in zip((read_ints(offsets, (e + 1,)), read_ints(order, (t * k,)), read_ints(position, (t * k,))), want[2:]):
        assert np.array_equal(got, ref)
    got = w.numpy().astype(np.float64)
    # exp of a difference that is off by |difference| u, two units for exp itself, a sum of at most e terms, a division
    with np.errstate(invalid="ignore"):
        span = np.nan_to_num(np.abs(logits - np.nanmax(np.where(np.isinf(logits), np.nan, logits), axis=1, keepdims=True, initial=0)), nan=0, posinf=0).max()
    u = UNIT[weight_dt(dt)]
    with np.errstate(invalid="ignore"):
        assert np.all((np.abs(got - want[1]) <= (2 * span + e + 12) * u * np.abs(want[1])) | (np.isnan(got) & np.isnan(want[1])))

    g = rng.normal(0, 1, (t, k)).astype(np.float64 if dt == F64 else np.float32)
    g[want[0] < 0] = np.nan                                                                     # never looked at
    dg, out = Dev(g, weight_dt(dt)), Dev.empty((t, e), dt)
    call("rp_hip_route_backward", out.ptr, dg.ptr, w.ptr, experts.ptr, d.ptr, e + 3, t, e, k, int(normalize), dt)
    got = oracle.to_f64(out.numpy(), dt)
    picked = want[0] >= 0
    gz = np.where(picked, g, 0).astype(np.float64)
    hot = np.zeros((t, e))
    among = np.zeros((t, e))
    rows = np.broadcast_to(np.arange(t)[:, None], (t, k))
    hot[rows[picked], want[0][picked]] = gz[picked]
    with np.errstate(invalid="ignore"):
        if normalize:
            among[rows[picked], want[0][picked]] = want[1][picked]
        else:
            top = np.max(np.where(np.isnan(logits), -np.inf, logits), 1, keepdims=True)
            p = np.where(logits == -np.inf, 0, np.exp(logits - np.where(np.isfinite(top), top, np.where(top > 0, top, 0))))
            total = p.sum(1, keepdims=True)
            among = p / np.where(total == 0, 1, total)
        mean = (np.where(picked, want[1], 0) * gz).sum(1, keepdims=True)
        ref = among * (hot - mean)
        size = among * (np.abs(hot) + (np.where(picked, np.abs(want[1]), 0) * np.abs(gz)).sum(1, keepdims=True))
    odd = np.isnan(want[1]).any(1)                                                              # rows with NaN or infinity: NaN somewhere, no more is promised
    assert np.isnan(got[odd]).any(1).all()
    # twice the weights' error (p, and the weights in the mean) and k additions
    within(got[~odd], ref[~odd], size[~odd], 2 * (2 * span + e + 12) + k, dt)


def test_route_backward_matches_differences():
    rng = np.random.default_rng(3)
    t, e, k = 9, 40, 3
    x = rng.normal(0, 1, (t, e))
    g = rng.normal(0, 1, (t, k))
    for normalize in (True, False):
        d = Dev(x, F64)
        w, (experts, *_) = route(d, e, t, e, k, normalize, F64)
        taken = read_ints(experts, (t, k))
        out, dg = Dev.empty((t, e), F64), Dev(g, F64)
        call("rp_hip_route_backward", out.ptr, dg.ptr, w.ptr, experts.ptr, d.ptr, e, t, e, k, int(normalize), F64)
        got = out.numpy()
        step = 1e-5

        def loss(v):
            p = np.exp(v - v.max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
            q = np.take_along_axis(p, taken, 1)
            return (g * (q / q.sum(1, keepdims=True) if normalize else q)).sum(1)

        for c in range(e):
            up, down = x.copy(), x.copy()
            up[:, c] += step
            down[:, c] -= step
            # the difference quotient is off by step^2 times a third derivative of order 1 and by 2^-52 / step
            assert np.max(np.abs((loss(up) - loss(down)) / (2 * step) - got[:, c])) <= 1e-9


@pytest.mark.parametrize("count, groups", [(1, 1), (7, 3), (64, 64), (1000, 1), (4096, 1024), (4097, 5), (5000, 1000), (6143, 64), (70001, 130), (262144, 256)])
def test_group_rows(count, groups):
    rng = np.random.default_rng(count)
    ids = rng.integers(-1, groups + 1, count).astype(np.int32)          # some on either side
    ids[rng.integers(0, count, 2)] = [-2 ** 31, 2 ** 31 - 1]
    d = ints(ids)
    offsets, order, position = (capi.DeviceBuffer(4 * n) for n in (groups + 1, count, count))
    for _ in range(2):
        call("rp_hip_group_rows", offsets.ptr, order.ptr, position.ptr, d.ptr, count, groups)
        want = sort_want(ids.astype(np.int64), groups)
        for got, ref in zip((read_ints(offsets, (groups + 1,)), read_ints(order, (count,)), read_ints(position, (count,))), want):
            assert np.array_equal(got, ref)


# ---- exchange ----------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dt", ALL, ids=ids_of)
@pytest.mark.parametrize("t, k, d", [(1, 1, 1), (3, 2, 64), (16, 6, 136), (33, 3, 129), (5, 2, 4096), (7, 4, 5000), (200, 1, 1027), (1000, 2, 512)])
def test_exchange(t, k, d, dt):
    rng = np.random.default_rng(t + d)
    rows = t * k
    pos = rng.permutation(rows).reshape(t, k).astype(np.int32)
    pos[rng.random((t, k)) < 0.2] = -1
    if t > 2:
        pos[1] = -1                                                     # a token that is sent nowhere
        pos[2, 0] = rows + 5                                            # no such row
    there = (pos >= 0) & (pos < rows)
    wdt = np.float64 if dt == F64 else np.float32
    w = rng.random((t, k)).astype(wdt)
    w[~there] = np.nan                                                  # weights and rows that nothing names are never used
    pad = 8 if d % 8 == 0 else 3
    x, g = rand_storage(rng, (t, d), dt), rand_storage(rng, (t, d), dt)
    z = rng.normal(0, 1, (rows, d + pad))
    z[np.setdiff1d(np.arange(rows), pos[there])] = np.nan
    z = oracle.to_storage(z, dt)
    filled = oracle.to_storage(np.full((rows, d + pad), 7.0), dt)
    dx, dg, dz, dw, dp = Dev(x, dt), Dev(g, dt), Dev(z, dt), Dev(w, weight_dt(dt)), ints(pos)
    out, y, gz, gw, back = Dev(filled, dt), Dev.empty((t, d), dt), Dev(filled, dt), Dev.empty((t, k), weight_dt(dt)), Dev.empty((t, d), dt)
    call("rp_hip_dispatch_rows", out.ptr, dx.ptr, dp.ptr, t, k, d, d, d + pad, dt)
    call("rp_hip_combine_forward", y.ptr, dz.ptr, dw.ptr, dp.ptr, t, k, d, d, d + pad, dt)
    call("rp_hip_combine_backward", gz.ptr, gw.ptr, dg.ptr, dz.ptr, dw.ptr, dp.ptr, t, k, d, d, d + pad, d + pad, dt)
    call("rp_hip_combine_forward", back.ptr, dz.ptr, None, dp.ptr, t, k, d, d, d + pad, dt)
    want = filled.copy()
    tt, jj = np.nonzero(there)
    want[pos[tt, jj], :d] = x[tt]
    assert np.array_equal(out.numpy(), want)
    z64, x64, g64, w64 = oracle.to_f64(z, dt)[:, :d], oracle.to_f64(x, dt), oracle.to_f64(g, dt), np.where(there, w, 0).astype(np.float64)
    zr = np.where(there[..., None], z64[np.where(there, pos, 0)], 0)
    within(oracle.to_f64(y.numpy(), dt), (w64[..., None] * zr).sum(1), np.abs(w64[..., None] * zr).sum(1), 2 * k, dt)
    within(oracle.to_f64(back.numpy(), dt), zr.sum(1), np.abs(zr).sum(1), k, dt)
    ref = oracle.to_f64(filled, dt)
    ref[pos[tt, jj], :d] = w64[tt, jj][:, None] * g64[tt]
    within(oracle.to_f64(gz.numpy(), dt), ref, np.abs(ref), 1, dt)
    within(gw.numpy().astype(np.float64), (g64[:, None] * zr).sum(2), np.abs(g64[:, None] * zr).sum(2), d, weight_dt(dt))


# ---- the grouped linear layer ----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dt", ALL, ids=ids_of)
@pytest.mark.parametrize("rows, last, width, pad", [(1, 0, 1, 0), (9, 4, 7, 3), (3000, 1, 65, 0), (40, 40, 8, 0), (5, 90, 8, 0), (5, -2, 8, 1)])
def test_zero_rows_behind(rows, last, width, pad, dt):
    x = rand_storage(np.random.default_rng(rows), (rows, width + pad), dt)
    buf = capi.DeviceBuffer.from_numpy(x)
    call("rp_hip_zero_rows_behind", buf.ptr, ints([0, last]).ptr, 1, rows, width, width + pad, dt)
    capi.synchronize()
    x[max(last, 0):, :width] = 0
    assert np.array_equal(buf.to_numpy(x.dtype, x.shape), x)


def grouped_want(x, w, bias, offsets):
    rows, n = x.shape[0], w.shape[2]
    y, size = np.zeros((rows, n)), np.zeros((rows, n))
    for e, (b, f) in enumerate(zip(offsets, offsets[1:])):
        y[b:f], size[b:f] = x[b:f] @ w[e], np.abs(x[b:f]) @ np.abs(w[e])
        if bias is not None:
            y[b:f] += bias[e]
            size[b:f] += np.abs(bias[e])
    return y, size


class Grouped:
    """A grouped layer's operands on the device; rows behind the last group hold NaN in x and dy and a mark in the outputs."""

    def __init__(self, dt, groups, rows, k, n, empty=(), behind=0, bias=True, seed=0, x_pad=0, y_pad=0, transposed=False, nan=True):
        rng = np.random.default_rng(seed + rows + 3 * k + 7 * n)
        self.dt, self.groups, self.rows, self.k, self.n = dt, groups, rows, k, n
        self.offsets = cuts(rng, rows, groups, empty, behind)
        self.x_rs, self.y_rs = k + x_pad, n + y_pad
        x, g = rng.normal(0, 1, (rows, self.x_rs)), rng.normal(0, 1, (rows, self.y_rs))
        if nan:
            x[self.offsets[-1]:], g[self.offsets[-1]:] = np.nan, np.nan
            x[:, k:], g[:, n:] = np.nan, np.nan
        w = rng.normal(0, k ** -0.5, (groups, n, k) if transposed else (groups, k, n))
        if nan:
            for e in empty:
                w[e] = np.nan                                           # a weight that no row uses is not read into any result
        self.w_st = (k * n, 1, k) if transposed else (k * n, n, 1)
        self.sx, self.sg, self.sw = (oracle.to_storage(a, dt) for a in (x, g, w))
        self.sb = oracle.to_storage(rng.normal(0, 1, (groups, n)), dt) if bias else None
        self.x, self.g, self.w = oracle.to_f64(self.sx, dt)[:, :k], oracle.to_f64(self.sg, dt)[:, :n], oracle.to_f64(self.sw, dt)
        if transposed:
            self.w = self.w.transpose(0, 2, 1)
        self.b = oracle.to_f64(self.sb, dt) if bias else None
        self.dx, self.dg, self.dw, self.do = Dev(self.sx, dt), Dev(self.sg, dt), Dev(self.sw, dt), ints(self.offsets)
        self.db = Dev(self.sb, dt) if bias else None
        self.mark = lambda *shape: Dev(oracle.to_storage(np.full(shape, 3.0), dt), dt)

    def forward(self, y=None):
        y = y or self.mark(self.rows, self.y_rs)
        call("rp_hip_grouped_linear_forward", y.ptr, self.dx.ptr, self.dw.ptr, ptr(self.db), self.do.ptr, self.groups, self.rows, self.k, self.n,
             self.x_rs, 1, *self.w_st, self.y_rs, self.dt)
        return y

    def check_forward(self, y):
        got = oracle.to_f64(y.numpy(), self.dt)
        last = self.offsets[-1]
        y64, size = grouped_want(self.x, self.w, self.b, self.offsets)
        within(got[:last, :self.n], y64[:last], size[:last], self.k + 1, self.dt)
        assert np.all(got[last:] == 3.0) and np.all(got[:, self.n:] == 3.0)

    def backward(self, accumulate=0, which=(1, 1, 1)):
        out = [self.mark(*shape) if use else None for use, shape in zip(which, ((self.rows, self.x_rs), (self.groups, self.k, self.n), (self.groups, self.n)))]
        call("rp_hip_grouped_linear_backward", *[ptr(o) for o in out], self.dg.ptr, self.dx.ptr, self.dw.ptr, self.do.ptr, self.groups, self.rows, self.k, self.n,
             self.y_rs, self.x_rs, 1, *self.w_st, self.x_rs, accumulate, accumulate, accumulate, self.dt)
        return out

    def check_backward(self, out, accumulate=0):
        dx, dw, db = out
        last, dt, old = self.offsets[-1], self.dt, 3.0 if accumulate else 0.0
        if dx is not None:
            got = oracle.to_f64(dx.numpy(), dt)
            ref, size = grouped_want(self.g, self.w.transpose(0, 2, 1), None, self.offsets)
            within(got[:last, :self.k], ref[:last] + old, size[:last] + old, self.n + 1, dt, added=old)
            assert np.all(got[last:] == 3.0) and np.all(got[:, self.k:] == 3.0)
        spans = list(zip(self.offsets, self.offsets[1:]))
        most = max(f - b for b, f in spans)
        if dw is not None:
            ref = np.stack([self.x[b:f].T @ self.g[b:f] for b, f in spans])
            size = np.stack([np.abs(self.x[b:f]).T @ np.abs(self.g[b:f]) for b, f in spans])
            within(oracle.to_f64(dw.numpy(), dt), ref + old, size + old, most + 1, dt, added=old)
        if db is not None:
            ref, size = (np.stack([f(self.g[b:e]).sum(0) for b, e in spans]) for f in (lambda a: a, np.abs))
            within(oracle.to_f64(db.numpy(), dt), ref + old, size + old, most + 1, dt, added=old)


SHAPES = [  # groups, rows, k, n, empty groups, rows behind the last
    (1, 1, 1, 1, (), 0), (3, 5, 3, 2, (1,), 1), (2, 40, 8, 8, (), 0), (5, 70, 24, 40, (0, 4), 3), (4, 300, 72, 136, (2,), 0), (3, 200, 33, 61, (), 5), (70, 500, 64, 64, (5, 69), 0),
    (2, 3, 512, 264, (), 0), (8, 16, 1024, 512, (), 0), (4, 130, 520, 384, (), 1), (3, 700, 256, 512, (), 0), (2, 257, 519, 263, (), 0), (6, 33, 320, 1000, (3,), 0), (2, 1500, 320, 320, (), 7)]


@pytest.mark.parametrize("dt", ALL, ids=ids_of)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s[:4])))
def test_grouped_linear(shape, dt):
    groups, rows, k, n, empty, behind = shape
    p = Grouped(dt, groups, rows, k, n, empty, behind, bias=rows % 2 == 0)
    p.check_forward(p.forward())
    p.check_backward(p.backward())
    p.check_backward(p.backward(accumulate=1), accumulate=1)


# sizes at which a product goes on tiles of 256 (forward; dx; dw) or of 128, aligned and ragged
@pytest.mark.parametrize("dt", [BF16, F16], ids=ids_of)
@pytest.mark.parametrize("shape", [(3, 4000, 512, 3584), (3, 4000, 3584, 512), (16, 16000, 1024, 1024), (8, 4100, 519, 1031), (7, 2500, 264, 2056)], ids=lambda s: "x".join(map(str, s)))
def test_grouped_linear_large_tiles(shape, dt):
    groups, rows, k, n = shape
    p = Grouped(dt, groups, rows, k, n, empty=(1,), behind=5)
    p.check_forward(p.forward())
    p.check_backward(p.backward(accumulate=1), accumulate=1)


@pytest.mark.parametrize("dt", ALL, ids=ids_of)
@pytest.mark.parametrize("pad, transposed", [(8, False), (3, False), (0, True), (8, True), (5, True)])
def test_grouped_linear_strides(pad, transposed, dt):
    for rows, k, n in ((90, 136, 72), (7, 264, 520)):
        p = Grouped(dt, 3, rows, k, n, (1,), 2, x_pad=pad, y_pad=pad, transposed=transposed)
        p.check_forward(p.forward())
        p.check_backward(p.backward())


@pytest.mark.parametrize("dt", [BF16, F32], ids=ids_of)
def test_grouped_linear_single_gradients(dt):
    for rows, k, n in ((90, 136, 72), (400, 256, 256)):
        p = Grouped(dt, 3, rows, k, n)
        whole = [o.numpy() for o in p.backward()]
        for i in range(3):
            one = p.backward(which=[j == i for j in range(3)])[i]
            assert np.array_equal(one.numpy(), whole[i])


@pytest.mark.parametrize("dt", ALL, ids=ids_of)
def test_grouped_linear_strided_columns(dt):
    """x with a column stride (every second column of wider rows)."""
    rng = np.random.default_rng(5)
    groups, rows, k, n = 3, 80, 40, 48
    offsets = cuts(rng, rows, groups)
    x, w = rand_storage(rng, (rows, 2 * k), dt), rand_storage(rng, (groups, k, n), dt)
    dx, dw, do, y = Dev(x, dt), Dev(w, dt), ints(offsets), Dev.empty((rows, n), dt)
    call("rp_hip_grouped_linear_forward", y.ptr, dx.ptr, dw.ptr, None, do.ptr, groups, rows, k, n, 2 * k, 2, k * n, n, 1, n, dt)
    ref, size = grouped_want(oracle.to_f64(x, dt)[:, ::2], oracle.to_f64(w, dt), None, offsets)
    within(oracle.to_f64(y.numpy(), dt), ref, size, k, dt)


@pytest.mark.parametrize("dt", [BF16, F32], ids=ids_of)
def test_grouped_linear_offsets_out_of_range(dt):
    """Offsets before 0, past the rows and decreasing are clamped: no access goes out of range, whole groups keep their results."""
    rng = np.random.default_rng(8)
    groups, rows, k, n = 4, 100, 64, 72
    p = Grouped(dt, groups, rows, k, n, bias=False, nan=False)
    bad = np.array([-50, 30, 20, 60, 4000], dtype=np.int32)            # groups 0: [0, 30), 1: none, 2: [20, 60), 3: [60, 100)
    p.do = ints(bad)
    got = oracle.to_f64(p.forward().numpy(), dt)
    for e, b, f in ((0, 0, 20), (3, 60, 100)):
        ref, size = p.x[b:f] @ p.w[e], np.abs(p.x[b:f]) @ np.abs(p.w[e])
        within(got[b:f], ref, size, k, dt)
    dw = oracle.to_f64(p.backward()[1].numpy(), dt)
    for e, b, f in ((0, 0, 30), (1, 0, 0), (2, 20, 60), (3, 60, 100)):
        within(dw[e], p.x[b:f].T @ p.g[b:f], np.abs(p.x[b:f]).T @ np.abs(p.g[b:f]), rows, dt)


@pytest.mark.parametrize("dt", [BF16, F16, F32], ids=ids_of)
def test_grouped_rows_do_not_mix(dt):
    """A row of NaN and one of infinities stay in their own rows of y and dx, and in their own group's dw."""
    for rows, k, n in ((60, 64, 96), (500, 320, 256), (12, 1024, 512)):
        p = Grouped(dt, 3, rows, k, n, bias=False)
        o = p.offsets
        bad = int(o[1])                                                  # the first row of group 1
        sx = p.sx.copy()
        sx[bad, :k] = oracle.to_storage(np.full(k, np.nan), dt)
        p.dx = Dev(sx, dt)
        got = oracle.to_f64(p.forward().numpy(), dt)
        keep = np.arange(rows) != bad
        ref, size = grouped_want(p.x, p.w, None, o)
        within(got[keep], ref[keep], size[keep], k, dt)
        assert np.isnan(got[bad]).all()
        dw = oracle.to_f64(p.backward()[1].numpy(), dt)
        for e in (0, 2):
            b, f = o[e], o[e + 1]
            within(dw[e], p.x[b:f].T @ p.g[b:f], np.abs(p.x[b:f]).T @ np.abs(p.g[b:f]), rows, dt)
        assert np.isnan(dw[1]).all()


# ---- adapters ------------------------------------------------------------------------------------------------------------

class Adapters:
    def __init__(self, dt, segments, adapters, rows, k, n, rank, behind=0, bias=True, scaled=True, empty=(), seed=0, transposed=False, ids=None):
        rng = np.random.default_rng(seed + rows + 5 * k + 11 * n)
        self.dt, self.sizes = dt, (segments, adapters, rows, k, n, rank)
        self.offsets = cuts(rng, rows, segments, empty, behind)
        self.ids = np.asarray(ids if ids is not None else rng.integers(-1, adapters, segments), dtype=np.int32)
        arrays = dict(x=(rows, k), g=(rows, n), w=(n, k) if transposed else (k, n), a=(adapters, k, rank), b=(adapters, rank, n))
        scale = dict(w=k ** -0.5, a=k ** -0.5, b=rank ** -0.5)
        self.s = {name: oracle.to_storage(rng.normal(0, scale.get(name, 1.0), shape), dt) for name, shape in arrays.items()}
        self.s["bias"] = rand_storage(rng, (n,), dt) if bias else None
        self.d = {name: None if a is None else Dev(a, dt) for name, a in self.s.items()}
        self.f = {name: None if a is None else oracle.to_f64(a, dt) for name, a in self.s.items()}
        if transposed:
            self.f["w"] = self.f["w"].T
        self.w_st = (1, k) if transposed else (n, 1)
        self.scales = (0.5 + rng.random(adapters)).astype(np.float32) if scaled else None
        self.dscales = Dev(self.scales, F32) if scaled else None
        self.dids, self.doff = ints(self.ids), ints(self.offsets)
        self.acc = F64 if dt == F64 else F32

    def plan(self):
        return (ptr(self.dscales), self.dids.ptr, self.doff.ptr) + self.sizes

    def spans(self):
        segments, adapters = self.sizes[:2]
        for s in range(segments):
            a = int(self.ids[s])
            if 0 <= a < adapters:
                yield slice(self.offsets[s], self.offsets[s + 1]), a, float(self.scales[a]) if self.scales is not None else 1.0

    def forward(self):
        _, _, rows, k, n, rank = self.sizes
        d = self.d
        self.y, self.h = Dev(oracle.to_storage(np.full((rows, n), 3.0), self.dt), self.dt), Dev(np.full((rows, rank), 3.0, dtype=capi.NP_STORAGE[self.acc]), self.acc)
        call("rp_hip_adapter_linear_forward", self.y.ptr, self.h.ptr, d["x"].ptr, d["w"].ptr, ptr(d["bias"]), d["a"].ptr, d["b"].ptr, *self.plan(), k, 1, *self.w_st, n, self.dt)

    def check_forward(self):
        _, _, rows, k, n, rank = self.sizes
        f, dt = self.f, self.dt
        y, size = f["x"] @ f["w"], np.abs(f["x"]) @ np.abs(f["w"])
        if f["bias"] is not None:
            y, size = y + f["bias"], size + np.abs(f["bias"])
        low, h = np.zeros((rows, rank)), self.h.numpy().astype(np.float64)
        base, reach = y.copy(), np.zeros((rows, n))
        used = np.zeros(rows, dtype=bool)
        for at, a, scale in self.spans():
            used[at] = True
            low[at] = scale * (f["x"][at] @ f["a"][a])
            hsize = scale * (np.abs(f["x"][at]) @ np.abs(f["a"][a]))
            within(h[at], low[at], hsize, k + 1, self.acc)
            y[at] += low[at] @ f["b"][a]
            reach[at] = hsize @ np.abs(f["b"][a])
        assert np.all(h[~used] == 3.0)
        got = oracle.to_f64(self.y.numpy(), dt)
        if dt in (F32, F64):
            within(got, y, size + reach, k + rank + 2, dt, roundings=2)
        else:
            self.thrice_rounded(got, y, base, 0.0 if f["bias"] is None else f["bias"], size + reach, k + rank + 2)

    def thrice_rounded(self, got, want, base, added, magnitude, terms):
        """The shared product p is rounded to the tensor type, p + added (a bias, or what dx held) = base again, and base plus the adapter's
        part a third time: each by half a step of its own value, |p| + |base| + |want| half steps in all.  Or p and the adapter's part are rounded
        together, want - added, and their sum with what dx held again: |want - added| + |want| half steps.  Neither bounds the other: with p = -3,
        added = 3 and an adapter's part of t < 0 they are 3 + |t| and 3 + 2 |t|."""
        dt = self.dt
        rounded = np.maximum(np.abs(base - added) + np.abs(base), np.abs(want - added)) + np.abs(want)
        bound = HALF_STEP[dt] * (1 + 2 * HALF_STEP[dt]) * rounded + 3 * TINY[dt] + (terms + 8) * UNIT[dt] * magnitude * (1 + HALF_STEP[dt])
        worst = np.max(np.abs(got - want) - bound)
        assert worst <= 0, f"{worst} beyond the bound"

    def backward(self, accumulate=0, which=(1, 1, 1)):
        segments, adapters, rows, k, n, rank = self.sizes
        d = self.d
        out = [Dev(oracle.to_storage(np.full(shape, 3.0), self.dt), self.dt) if use else None for use, shape in zip(which, ((rows, k), (adapters, k, rank), (adapters, rank, n)))]
        u = Dev.empty((rows, rank), self.acc)
        call("rp_hip_adapter_linear_backward", *[ptr(o) for o in out], u.ptr, d["g"].ptr, d["x"].ptr, d["w"].ptr, d["a"].ptr, d["b"].ptr, self.h.ptr, *self.plan(),
             n, k, 1, *self.w_st, k, accumulate, accumulate, accumulate, self.dt)
        return out

    def check_backward(self, out, accumulate=0):
        segments, adapters, rows, k, n, rank = self.sizes
        f, dt, old = self.f, self.dt, 3.0 if accumulate else 0.0
        dx, size = f["g"] @ f["w"].T + old, np.abs(f["g"]) @ np.abs(f["w"]).T + old
        base, reach = dx.copy(), np.zeros((rows, k))
        da, da_size, db, db_size = np.zeros((adapters, k, rank)), np.zeros((adapters, k, rank)), np.zeros((adapters, rank, n)), np.zeros((adapters, rank, n))
        for at, a, scale in self.spans():
            u, u_size = scale * (f["g"][at] @ f["b"][a].T), scale * (np.abs(f["g"][at]) @ np.abs(f["b"][a]).T)
            low, low_size = scale * (f["x"][at] @ f["a"][a]), scale * (np.abs(f["x"][at]) @ np.abs(f["a"][a]))
            dx[at] += u @ f["a"][a].T
            reach[at] = u_size @ np.abs(f["a"][a]).T
            da[a] += f["x"][at].T @ u
            da_size[a] += np.abs(f["x"][at]).T @ u_size
            db[a] += low.T @ f["g"][at]
            db_size[a] += low_size.T @ np.abs(f["g"][at])
        if out[0] is not None:
            got = oracle.to_f64(out[0].numpy(), dt)
            if dt in (F32, F64):
                within(got, dx, size + reach, n + rank + 2, dt, roundings=2)
            else:
                self.thrice_rounded(got, dx, base, old, size + reach, n + rank + 2)
        if out[1] is not None:
            within(oracle.to_f64(out[1].numpy(), dt), da + old, da_size + old, rows + n + 2, dt, added=old)
        if out[2] is not None:
            within(oracle.to_f64(out[2].numpy(), dt), db + old, db_size + old, rows + k + 2, dt, added=old)


ADAPTER_SHAPES = [  # segments, adapters, rows, k, n, rank, rows behind the last segment
    (1, 1, 1, 1, 1, 1, 0), (3, 2, 7, 16, 24, 4, 1), (32, 5, 32, 256, 512, 16, 0), (5, 3, 100, 72, 136, 8, 3), (4, 4, 300, 260, 130, 32, 0), (3, 2, 150, 33, 61, 5, 2),
    (6, 2, 513, 512, 320, 64, 0), (2, 1, 64, 1024, 512, 16, 0), (40, 30, 200, 128, 264, 100, 0), (9, 6, 1030, 264, 520, 16, 4)]


@pytest.mark.parametrize("dt", ALL, ids=ids_of)
@pytest.mark.parametrize("shape", ADAPTER_SHAPES, ids=lambda s: "x".join(map(str, s[:6])))
def test_adapter_linear(shape, dt):
    *sizes, behind = shape
    for transposed in (False, True):
        p = Adapters(dt, *sizes, behind=behind, bias=sizes[2] % 2 == 0, scaled=sizes[0] != 4, transposed=transposed)
        p.forward()
        p.check_forward()
        p.check_backward(p.backward())
        p.check_backward(p.backward(accumulate=1), accumulate=1)


@pytest.mark.parametrize("dt", ALL, ids=ids_of)
@pytest.mark.parametrize("pad", [8, 3])
@pytest.mark.parametrize("shape", [(5, 3, 100, 72, 136, 8, 3), (3, 2, 700, 264, 520, 16, 0), (32, 5, 32, 256, 512, 16, 0), (4, 2, 90, 129, 95, 12, 2), (3, 3, 200, 40, 48, 200, 0)], ids=lambda s: "x".join(map(str, s[:6])))
def test_adapter_linear_strides(shape, pad, dt):
    """Rows of x, dy, y and dx further apart than they are long, NaN between them: never read, and never written."""
    *sizes, behind = shape
    segments, adapters, rows, k, n, rank = sizes
    p = Adapters(dt, *sizes, behind=behind)

    def wide(name, width, value):
        a = oracle.to_storage(np.full((rows, width + pad), value), dt)
        if name:
            a[:, :width] = p.s[name]
        return Dev(a, dt)

    def dense(d, width):
        a = d.numpy()
        assert np.all(oracle.to_f64(a, dt)[:, width:] == 3.0)
        return Dev(np.ascontiguousarray(a[:, :width]), dt)

    x, g, y, dx = wide("x", k, np.nan), wide("g", n, np.nan), wide(None, n, 3.0), wide(None, k, 3.0)
    p.h = Dev(np.full((rows, rank), 3.0, dtype=capi.NP_STORAGE[p.acc]), p.acc)
    d = p.d
    call("rp_hip_adapter_linear_forward", y.ptr, p.h.ptr, x.ptr, d["w"].ptr, ptr(d["bias"]), d["a"].ptr, d["b"].ptr, *p.plan(), k + pad, 1, *p.w_st, n + pad, dt)
    p.y = dense(y, n)
    p.check_forward()
    u, da, db = Dev.empty((rows, rank), p.acc), Dev.empty((adapters, k, rank), dt), Dev.empty((adapters, rank, n), dt)
    call("rp_hip_adapter_linear_backward", dx.ptr, da.ptr, db.ptr, u.ptr, g.ptr, x.ptr, d["w"].ptr, d["a"].ptr, d["b"].ptr, p.h.ptr, *p.plan(),
         n + pad, k + pad, 1, *p.w_st, k + pad, 0, 0, 0, dt)
    p.check_backward([dense(dx, k), da, db])


@pytest.mark.parametrize("dt", ALL, ids=ids_of)
@pytest.mark.parametrize("groups, rows, k, n", [(3, 90, 72, 136), (4, 700, 264, 520), (2, 20, 256, 128)])
def test_grouped_linear_broadcast_operands(groups, rows, k, n, dt):
    """One row for all rows of x or of dy, one weight for all groups, rows of x that overlap."""
    p = Grouped(dt, groups, rows, k, n, nan=False)
    dw, db = Dev.empty((groups, k, n), dt), Dev.empty((groups, n), dt)
    y, dx = p.mark(rows, n), p.mark(rows, k)
    flat = p.sx.reshape(-1)
    x0, w0 = p.x, p.w
    for x_rs, g_rs, w_gs in ((0, n, k * n), (k, 0, k * n), (k, n, 0), (0, 0, 0), (k // 2, n, k * n)):
        p.x = oracle.to_f64(np.stack([flat[i * x_rs:i * x_rs + k] for i in range(rows)]), dt)
        p.g = np.broadcast_to(oracle.to_f64(p.sg, dt)[:1], (rows, n)) if g_rs == 0 else oracle.to_f64(p.sg, dt)
        p.w = np.broadcast_to(w0[:1], w0.shape) if w_gs == 0 else w0
        call("rp_hip_grouped_linear_forward", y.ptr, p.dx.ptr, p.dw.ptr, ptr(p.db), p.do.ptr, groups, rows, k, n, x_rs, 1, w_gs, n, 1, n, dt)
        p.check_forward(y)
        call("rp_hip_grouped_linear_backward", dx.ptr, dw.ptr, db.ptr, p.dg.ptr, p.dx.ptr, p.dw.ptr, p.do.ptr, groups, rows, k, n, g_rs, x_rs, 1, w_gs, n, 1, k, 0, 0, 0, dt)
        p.check_backward([dx, dw, db])


# ranks that are no whole vectors, rows that end and start inside one, widths below a vector, tiles of every edge
ODD_ADAPTER_SHAPES = [(3, 2, 700, 264, 520, 5, 0), (2, 2, 300, 129, 515, 3, 1), (1, 1, 2000, 136, 264, 1, 0), (2, 2, 20, 5, 300, 4, 0), (2, 2, 20, 300, 5, 4, 0), (4, 2, 90, 9, 15, 12, 0),
                      (20, 3, 1500, 264, 1032, 12, 7), (3, 2, 2100, 264, 2056, 7, 0), (48, 2, 400, 1031, 130, 64, 0), (5, 3, 70, 2040, 94, 33, 0), (1, 9, 1, 168, 93, 64, 0)]


@pytest.mark.parametrize("dt", [BF16, F16, F32], ids=ids_of)
@pytest.mark.parametrize("shape", ODD_ADAPTER_SHAPES, ids=lambda s: "x".join(map(str, s[:6])))
def test_adapter_linear_odd_sizes(shape, dt):
    test_adapter_linear(shape, dt)


# the term as a launch of its own: each segment a row or a few, large and small shared products
@pytest.mark.parametrize("dt", [BF16, F16], ids=ids_of)
@pytest.mark.parametrize("shape", [(300, 40, 700, 1024, 2048, 16, 9), (500, 7, 2100, 264, 1032, 33, 0), (90, 90, 90, 520, 2047, 8, 0), (64, 9, 200, 2064, 24, 100, 3), (33, 5, 70, 40, 9, 4, 1)], ids=lambda s: "x".join(map(str, s[:6])))
def test_adapter_linear_many_segments(shape, dt):
    """y and dx are rounded once (and once more where dx is added to what is there)."""
    *sizes, behind = shape
    segments, adapters, rows, k, n, rank = sizes
    for transposed in (False, True):
        p = Adapters(dt, *sizes, behind=behind, transposed=transposed)
        p.forward()
        p.check_forward()
        for accumulate in (0, 1):
            out = p.backward(accumulate=accumulate)
            p.check_backward(out, accumulate=accumulate)
        f, size, y = p.f, np.abs(p.f["x"]) @ np.abs(p.f["w"]) + np.abs(p.f["bias"]), p.f["x"] @ p.f["w"] + p.f["bias"]
        for at, a, scale in p.spans():
            y[at] += scale * (f["x"][at] @ f["a"][a]) @ f["b"][a]
            size[at] += scale * (np.abs(f["x"][at]) @ np.abs(f["a"][a])) @ np.abs(f["b"][a])
        # h is multiplied as two values that add up to it to 2^-17 (bfloat16): 128 units of 2^-24 of the term's magnitude
        within(oracle.to_f64(p.y.numpy(), dt), y, size, k + rank + 2 + 128, dt)


# the shared product on tiles of 256 and of 128, aligned and ragged, the rank in one and in several steps
@pytest.mark.parametrize("dt", [BF16, F16], ids=ids_of)
@pytest.mark.parametrize("shape", [(5, 3, 4100, 512, 4096, 32, 0), (5, 3, 4096, 4096, 512, 100, 6), (3, 2, 2049, 1031, 4099, 12, 0), (7, 4, 2048, 520, 2048, 8, 0)], ids=lambda s: "x".join(map(str, s[:6])))
def test_adapter_linear_large_tiles(shape, dt):
    *sizes, behind = shape
    p = Adapters(dt, *sizes, behind=behind)
    p.forward()
    p.check_forward()
    p.check_backward(p.backward(accumulate=1), accumulate=1)


@pytest.mark.parametrize("dt", [BF16, F32], ids=ids_of)
def test_adapter_linear_without_any(dt):
    """No segment has an adapter: the layer is the shared projection, and the adapters' gradients are zeros."""
    p = Adapters(dt, 3, 2, 50, 64, 96, 8, ids=[-1, 7, -3])
    p.forward()
    p.check_forward()
    out = p.backward()
    p.check_backward(out)
    assert not out[1].numpy().any() and not out[2].numpy().any()


@pytest.mark.parametrize("dt", [BF16, F32], ids=ids_of)
def test_adapter_linear_one_adapter_for_all(dt):
    """Segments that share an adapter, empty ones among them: its gradients are sums over all of them."""
    p = Adapters(dt, 6, 3, 120, 136, 72, 16, empty=(0, 3, 5), ids=[1, 1, 1, 0, 1, 2])
    p.forward()
    p.check_forward()
    whole = p.backward()
    p.check_backward(whole)
    for i in range(3):
        one = p.backward(which=[j == i for j in range(3)])[i]
        assert np.array_equal(one.numpy(), whole[i].numpy())


# ---- together ----------------------------------------------------------------------------------------------------------------

def moe_buffers(dt, t, e, k, d, f, rng):
    r = t * k
    dev = {name: Dev(rand_storage(rng, shape, dt), dt) for name, shape in dict(logits=(t, e), x=(t, d), gy=(t, d)).items()}
    for name, shape, scale in (("w1", (e, d, f), d ** -0.5), ("b1", (e, f), 0.1), ("w2", (e, f, d), f ** -0.5)):
        dev[name] = Dev(oracle.to_storage(rng.normal(0, scale, shape), dt), dt)
    for name, shape in dict(xs=(r, d), h=(r, f), a=(r, f), z=(r, d), y=(t, d), gz=(r, d), ga=(r, f), gh=(r, f), gxs=(r, d), gx=(t, d), glogits=(t, e),
                            gw1=(e, d, f), gb1=(e, f), gw2=(e, f, d)).items():
        dev[name] = Dev(oracle.to_storage(np.zeros(shape), dt), dt)
    for name in ("weights", "gweights"):
        dev[name] = Dev.empty((t, k), weight_dt(dt))
    for name, n in dict(experts=r, offsets=e + 1, order=r, position=r).items():
        dev[name] = capi.DeviceBuffer(4 * n)
    return dev


def moe_step(v, dt, t, e, k, d, f):
    """A mixture of experts, forward and backward: route, dispatch, two grouped layers with a ReLU, combine, and the way back."""
    r = t * k
    p = {name: b.ptr for name, b in v.items()}
    call("rp_hip_route_forward", p["weights"], p["experts"], p["offsets"], p["order"], p["position"], p["logits"], e, t, e, k, 1, dt)
    call("rp_hip_dispatch_rows", p["xs"], p["x"], p["position"], t, k, d, d, d, dt)
    call("rp_hip_grouped_linear_forward", p["h"], p["xs"], p["w1"], p["b1"], p["offsets"], e, r, d, f, d, 1, d * f, f, 1, f, dt)
    call("relu_kernel_device", p["a"], p["h"], r * f, dt)
    call("rp_hip_grouped_linear_forward", p["z"], p["a"], p["w2"], None, p["offsets"], e, r, f, d, f, 1, d * f, d, 1, d, dt)
    call("rp_hip_combine_forward", p["y"], p["z"], p["weights"], p["position"], t, k, d, d, d, dt)
    call("rp_hip_combine_backward", p["gz"], p["gweights"], p["gy"], p["z"], p["weights"], p["position"], t, k, d, d, d, d, dt)
    call("rp_hip_grouped_linear_backward", p["ga"], p["gw2"], None, p["gz"], p["a"], p["w2"], p["offsets"], e, r, f, d, d, f, 1, d * f, d, 1, f, 0, 0, 0, dt)
    call("backwards_relu_device", p["ga"], p["h"], p["gh"], r * f, dt)
    call("rp_hip_grouped_linear_backward", p["gxs"], p["gw1"], p["gb1"], p["gh"], p["xs"], p["w1"], p["offsets"], e, r, d, f, f, d, 1, d * f, f, 1, d, 0, 0, 0, dt)
    call("rp_hip_combine_forward", p["gx"], p["gxs"], None, p["position"], t, k, d, d, d, dt)
    call("rp_hip_route_backward", p["glogits"], p["gweights"], p["weights"], p["experts"], p["logits"], e, t, e, k, 1, dt)


RESULTS = ("y", "gx", "glogits", "gw1", "gb1", "gw2")


def moe_want(v, dt, t, e, k):
    f64 = {name: oracle.to_f64(v[name].numpy(), dt) for name in ("logits", "x", "gy", "w1", "b1", "w2")}
    experts, weights, *_ = route_want(f64["logits"], k, True)
    y, gx, gw = np.zeros_like(f64["x"]), np.zeros_like(f64["x"]), np.zeros((t, k))
    gw1, gb1, gw2 = np.zeros_like(f64["w1"]), np.zeros_like(f64["b1"]), np.zeros_like(f64["w2"])
    for i in range(t):
        for j in range(k):
            q, w = experts[i, j], weights[i, j]
            if q < 0:
                continue
            h = f64["x"][i] @ f64["w1"][q] + f64["b1"][q]
            a = np.maximum(h, 0)
            z = a @ f64["w2"][q]
            y[i] += w * z
            gw[i, j] = f64["gy"][i] @ z
            gz = w * f64["gy"][i]
            gh = (f64["w2"][q] @ gz) * (h > 0)
            gw2[q] += np.outer(a, gz)
            gw1[q] += np.outer(f64["x"][i], gh)
            gb1[q] += gh
            gx[i] += f64["w1"][q] @ gh
    glogits = np.zeros_like(f64["logits"])
    mean = (weights * gw).sum(1)
    for j in range(k):
        live = experts[:, j] >= 0
        glogits[live, experts[live, j]] = (weights[:, j] * (gw[:, j] - mean))[live]
    return dict(y=y, gx=gx, glogits=glogits, gw1=gw1, gb1=gb1, gw2=gw2)


@pytest.mark.parametrize("dt", [F32, BF16], ids=ids_of)
def test_mixture_of_experts_forward_and_backward(dt):
    t, e, k, d, f = 37, 6, 2, 64, 136
    v = moe_buffers(dt, t, e, k, d, f, np.random.default_rng(21))
    moe_step(v, dt, t, e, k, d, f)
    want = moe_want(v, dt, t, e, k)
    # A chain of at most five products, each rounded (h, a, z, gz, gh ...): normwise about five half steps, and where an h next to zero
    # changes its sign with its rounding, one term of 136.
    for name in RESULTS:
        assert oracle.rel_err(oracle.to_f64(v[name].numpy(), dt), want[name]) <= (8 * HALF_STEP[dt] if dt != F32 else 2e-5), name


@pytest.mark.parametrize("dt", [F32, F16, BF16], ids=ids_of)
def test_captured_and_replayed(dt):
    """The step recorded into a graph, twice with outputs of their own, replayed with other work between: the eager results each time."""
    t, e, k, d, f = 50, 5, 2, 72, 264
    args = (dt, t, e, k, d, f)
    eager = moe_buffers(*args, np.random.default_rng(4))
    one, two = (moe_buffers(*args, np.random.default_rng(seed)) for seed in (4, 5))
    moe_step(eager, *args)
    want = {name: eager[name].numpy() for name in RESULTS}
    stream = capi.Stream()
    graphs = []
    with stream:
        for v in (one, two):
            moe_step(v, *args)
            with capi.Graph.capture() as g:
                moe_step(v, *args)
            graphs.append(g)
        for _ in range(3):
            for name in RESULTS:
                call("rp_hip_memset", one[name].ptr, 0, one[name].buf.nbytes)
            graphs[1].launch()
            graphs[0].launch()
            moe_step(two, *args)
            capi.check(capi.lib().rp_hip_stream_synchronize(), "rp_hip_stream_synchronize")
            for name in RESULTS:
                assert np.array_equal(one[name].numpy(), want[name]), name


def test_two_streams_at_once():
    """Two steps on streams of their own, side by side: neither touches the other's results."""
    args = (BF16, 64, 8, 2, 128, 264)
    alone, here, there = (moe_buffers(*args, np.random.default_rng(seed)) for seed in (1, 1, 2))
    moe_step(alone, *args)
    want = {name: alone[name].numpy() for name in RESULTS}
    streams = [capi.Stream(), capi.Stream()]
    for _ in range(5):
        for s, v in zip(streams, (here, there)):
            with s:
                moe_step(v, *args)
        capi.synchronize()
        for name in RESULTS:
            assert np.array_equal(here[name].numpy(), want[name]), name


@pytest.mark.parametrize("t, e, k", [(3000, 130, 2), (20001, 8, 2), (40000, 64, 6), (700, 1000, 7), (9000, 1024, 1)])
def test_routing_on_other_streams_and_in_graphs(t, e, k):
    """Long lists are sorted with other memory there; the results are the null stream's."""
    rng = np.random.default_rng(t)
    logits = oracle.to_storage(rng.normal(0, 1, (t, e)), F32)
    special_rows(logits, rng)
    dlogits = Dev(logits, F32)
    shapes = [(t * k,), (e + 1,), (t * k,), (t * k,)]
    ids = rng.integers(-1, e + 1, t * k).astype(np.int32)
    dids, sort = ints(ids), sort_want(ids.astype(np.int64), e)

    def results(r):
        return [r[0].numpy()] + [read_ints(b, s) for b, s in zip(r[1], shapes)]

    def buffers():
        return [capi.DeviceBuffer.from_numpy(np.full(n, 7, np.int32)) for n in (e + 1, t * k, t * k)]

    def sort_into(outs):
        call("rp_hip_group_rows", *(o.ptr for o in outs), dids.ptr, t * k, e)

    def check_sort(outs):
        for got, ref in zip(outs, sort):
            assert np.array_equal(read_ints(got, np.shape(ref)), ref)

    want = results(route(dlogits, e, t, e, k, 1, F32))
    streams, outs, routed = [capi.Stream(), capi.Stream()], [buffers(), buffers()], []
    for s, o in zip(streams, outs):                            # both at work at once
        with s:
            routed.append(route(dlogits, e, t, e, k, 1, F32))
            sort_into(o)
    capi.synchronize()
    for r, o in zip(routed, outs):
        check_sort(o)
        for got, ref in zip(results(r), want):
            assert np.array_equal(got, ref, equal_nan=True)
    with streams[0]:
        with capi.Graph.capture() as g:
            sort_into(outs[0])
        for _ in range(3):
            for o in outs[0]:
                call("rp_hip_memset", o.ptr, 0, o.nbytes)
            g.launch()
            capi.check(capi.lib().rp_hip_stream_synchronize(), "rp_hip_stream_synchronize")
            check_sort(outs[0])


@pytest.mark.parametrize("dt", [BF16, F16], ids=ids_of)
@pytest.mark.parametrize("shape", [(1, 1, 4100, 136, 264, 8, 0), (3, 2, 9000, 96, 200, 33, 5), (2, 25, 6000, 264, 520, 16, 0), (1, 1, 8192, 1032, 24, 64, 0)], ids=lambda s: "x".join(map(str, s[:6])))
def test_adapter_gradients_of_many_rows(shape, dt):
    """Several workgroups share an adapter's rows; one gradient alone has the same bits, on another stream and in a graph too."""
    *sizes, behind = shape
    p = Adapters(dt, *sizes, behind=behind)
    p.forward()
    whole = p.backward()
    p.check_backward(whole)
    p.check_backward(p.backward(accumulate=1), accumulate=1)
    for i in range(3):
        one = p.backward(which=[j == i for j in range(3)])[i]
        assert np.array_equal(one.numpy(), whole[i].numpy())
    segments, adapters, rows, k, n, rank = p.sizes
    out, u, d = [Dev.empty(w.shape, dt) for w in whole], Dev.empty((rows, rank), p.acc), p.d

    def into():
        call("rp_hip_adapter_linear_backward", *[o.ptr for o in out], u.ptr, d["g"].ptr, d["x"].ptr, d["w"].ptr, d["a"].ptr, d["b"].ptr, p.h.ptr, *p.plan(), n, k, 1, *p.w_st, k, 0, 0, 0, dt)

    def check():
        capi.check(capi.lib().rp_hip_stream_synchronize(), "rp_hip_stream_synchronize")
        for a, b in zip(out, whole):
            assert np.array_equal(a.numpy(), b.numpy())
            call("rp_hip_memset", a.ptr, 0, a.buf.nbytes)

    with capi.Stream():
        into()
        check()
        with capi.Graph.capture() as g:
            into()
        for _ in range(3):
            g.launch()
            check()


@pytest.mark.parametrize("dt", [F32, F64], ids=ids_of)
def test_grouped_linear_groups_of_few_rows(dt):
    for groups, rows, k, n in ((40, 60, 264, 520), (7, 50, 130, 70), (30, 2, 300, 300)):
        p = Grouped(dt, groups, rows, k, n, empty=(2, 5))
        p.check_forward(p.forward())
        p.check_backward(p.backward())
        p.check_backward(p.backward(accumulate=1), accumulate=1)
