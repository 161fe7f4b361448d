"""Adapters of many requests side by side: what one adapter, or one request's range of values, may not do to the others."""
import numpy as np
import pytest

import oracle
from recpulse_amd import capi
from devhelp import BF16, F16, F32, Dev
from test_grouped_gpu import UNIT, Adapters, Grouped, call, ids_of, ptr, within

pytestmark = pytest.mark.gpu

# h and u are multiplied as two values of a 16-bit type that add up to them to 2^-17 (bfloat16) or 2^-22 (float16) of the product's magnitude: units of 2^-24
SPLIT = {BF16: 128, F16: 4, F32: 0}


def layer(p):
    """y and its magnitudes, from the operands as they are."""
    f = p.f
    with np.errstate(invalid="ignore"):
        y, size = f["x"] @ f["w"] + f["bias"], np.abs(f["x"]) @ np.abs(f["w"]) + np.abs(f["bias"])
        for at, a, scale in p.spans():
            y[at] += scale * (f["x"][at] @ f["a"][a]) @ f["b"][a]
            size[at] += scale * (np.abs(f["x"][at]) @ np.abs(f["a"][a])) @ np.abs(f["b"][a])
    return y, size


def input_gradient(p):
    f = p.f
    with np.errstate(invalid="ignore"):
        dx, size = f["g"] @ f["w"].T, np.abs(f["g"]) @ np.abs(f["w"]).T
        for at, a, scale in p.spans():
            dx[at] += scale * (f["g"][at] @ f["b"][a].T) @ f["a"][a].T
            size[at] += scale * (np.abs(f["g"][at]) @ np.abs(f["b"][a]).T) @ np.abs(f["a"][a]).T
    return dx, size


def put(p, name, where, values):
    """values into the operand, here and on the device"""
    s = p.s[name]
    s[where] = oracle.to_storage(np.broadcast_to(np.asarray(values, dtype=np.float64), s[where].shape), p.dt) if s[where].shape else oracle.to_storage(np.array([values], dtype=np.float64), p.dt)[0]
    p.d[name] = Dev(s, p.dt)
    p.f[name] = oracle.to_f64(s, p.dt)


def once(got, want, size, terms, dt):
    """Rounded once (in float32 the shared product and the sum); NaN and infinities where the exact values have them."""
    both = np.isinf(want)
    assert np.array_equal(got[both], want[both])
    within(np.where(both, 0, got), np.where(both, 0, want), np.where(np.isfinite(size), size, 0), terms + SPLIT[dt], dt, roundings=2 if dt == F32 else 1)


# few rows; the term as a launch of its own; tiles of 64, of 128 and of 256, whole and not; segments that end inside a tile, one row long and without an adapter
SMALL = [(9, 4, 32, 256, 512, 16), (90, 5, 300, 264, 136, 8), (7, 3, 700, 264, 520, 12), (6, 3, 2100, 264, 1031, 16)]
LARGE = [(9, 4, 4100, 136, 4096, 32), (9, 4, 4096, 128, 4096, 40)]


@pytest.mark.parametrize("shape, dt", [(s, d) for s in SMALL for d in (BF16, F16, F32)] + [(s, d) for s in LARGE for d in (BF16, F16)], ids=lambda v: "x".join(map(str, v)) if isinstance(v, tuple) else ids_of(v))
def test_rows_beside_an_adapter_that_is_not_finite(shape, dt):
    """An infinity and a NaN in one adapter's factors reach the rows of that adapter and no others, and there the columns they belong to."""
    segments, adapters, rows, k, n, rank = shape
    ids = [s % (adapters + 1) - 1 for s in range(segments)]
    p = Adapters(dt, *shape, behind=2, ids=ids)
    p.offsets[2] = p.offsets[1] + 1                            # (one row of adapter 0)
    p.doff = capi.DeviceBuffer.from_numpy(p.offsets)
    put(p, "b", (0, rank // 2, slice(3, 6)), [np.inf, np.nan, -np.inf])
    put(p, "b", (1, 0, 7), np.inf)
    p.forward()
    once(oracle.to_f64(p.y.numpy(), dt), *layer(p), k + rank + 2, dt)
    p = Adapters(dt, *shape, behind=2, ids=ids)
    p.forward()
    put(p, "a", (0, slice(3, 6), rank // 2), [np.inf, np.nan, -np.inf])
    put(p, "a", (1, 7, 0), np.inf)
    want, size = input_gradient(p)
    once(oracle.to_f64(p.backward()[0].numpy(), dt), want, size, n + rank + 2, dt)
    got = oracle.to_f64(p.backward(accumulate=1)[0].numpy(), dt)         # (added to 3: the same places)
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got[np.isinf(want)], want[np.isinf(want)])
    fine = np.isfinite(want)
    within(np.where(fine, got, 3), np.where(fine, want + 3, 3), np.where(np.isfinite(size), size, 0) + 3, n + rank + 2 + SPLIT[dt], dt, roundings=2 if dt == F32 else 1, added=3.0)


# the shapes above, many rows of one adapter
RANGES = SMALL + [(1, 1, 4100, 136, 264, 8)]
MAGNITUDES = [(2.0 ** 8, 2.0 ** -10, 2.0 ** -14, 2.0 ** -14), (2.0 ** -10, 2.0 ** -10, 2.0 ** 10, 2.0 ** 4), (2.0 ** 7, 2.0 ** 12, 2.0 ** -12, 2.0 ** -12), (2.0 ** -8, 2.0 ** -4, 2.0 ** 10, 1)]


def ranged(dt, shape, **scales):
    """Operands times a power of two each; without a shared weight, whose product would hide the term, and without a bias."""
    p = Adapters(dt, *shape, ids=[s % (shape[1] + 1) - 1 for s in range(shape[0])] if shape[0] > 1 else [0], scaled=False)
    put(p, "w", slice(None), 0.0)
    put(p, "bias", slice(None), 0.0)
    for name, scale in scales.items():
        put(p, name, slice(None), p.f[name] * scale)
    return p


def gradients(p):
    """da and db, their magnitudes, and what a value 2^-22 of the largest of its column would change."""
    _, adapters, rows, k, n, rank = p.sizes
    f = p.f
    da, db = np.zeros((3, adapters, k, rank)), np.zeros((3, adapters, rank, n))
    for at, a, _ in p.spans():
        if at.start == at.stop:
            continue
        u, h = f["g"][at] @ f["b"][a].T, f["x"][at] @ f["a"][a]
        usize, hsize = np.abs(f["g"][at]) @ np.abs(f["b"][a]).T, np.abs(f["x"][at]) @ np.abs(f["a"][a])
        x, g = np.abs(f["x"][at]), np.abs(f["g"][at])
        for out, parts in ((da, ((f["x"][at].T, u), (x.T, usize), (x.T, np.broadcast_to(np.abs(u).max(0), u.shape)))), (db, ((h.T, f["g"][at]), (hsize.T, g), (np.broadcast_to(np.abs(h).max(0), h.shape).T, g)))):
            for i, (left, right) in enumerate(parts):
                out[i, a] += left @ right
    return da, db


@pytest.mark.parametrize("shape, magnitude, dt", [(s, m, F16) for s in RANGES for m in range(4)] + [(s, 1, BF16) for s in RANGES] + [((9, 4, 4100, 72, 4096, 32), 2, F16)],
                         ids=lambda v: "x".join(map(str, v)) if isinstance(v, tuple) else str(v))
def test_term_of_any_magnitude(shape, magnitude, dt):
    """h and u far below and above what the tensors' type holds, results within it: they are float32 sums, and their products keep their digits.  (u is about
    2^-25 in the first, h 2^-20 and u 2^17 in the second, h 2^19 and u 2^-20 in the third.)  An h or u that is off by 2^-22 of the largest of its row, or of its column in a gradient, is allowed for."""
    p = ranged(dt, shape, **dict(zip("xabg", MAGNITUDES[magnitude])))
    _, adapters, rows, k, n, rank = shape
    f, unit = p.f, SPLIT[dt] * 2.0 ** -24
    p.forward()
    y, size = layer(p)
    row = np.zeros((rows, n))
    for at, i, _ in p.spans():
        row[at] = np.abs(f["x"][at] @ f["a"][i]).max(1, keepdims=True, initial=0) @ np.abs(f["b"][i]).sum(0, keepdims=True)
    within(oracle.to_f64(p.y.numpy(), dt), y, size + unit / UNIT[dt] / (k + rank + 10) * row, k + rank + 2 + SPLIT[dt], dt)
    dx, da, db = p.backward()
    want, size = input_gradient(p)
    row = np.zeros((rows, k))
    for at, i, _ in p.spans():
        row[at] = np.abs(f["g"][at] @ f["b"][i].T).max(1, keepdims=True, initial=0) @ np.abs(f["a"][i]).sum(1, keepdims=True).T
    within(oracle.to_f64(dx.numpy(), dt), want, size + unit / UNIT[dt] / (n + rank + 10) * row, n + rank + 2 + SPLIT[dt], dt)
    for got, (want, size, column), width in zip((da, db), gradients(p), (n, k)):
        within(oracle.to_f64(got.numpy(), dt), want, size + unit / UNIT[dt] / (rows + width + 10) * column, rows + width + 2 + SPLIT[dt], dt)


@pytest.mark.parametrize("shape", RANGES, ids=lambda s: "x".join(map(str, s)))
def test_term_of_rows_of_every_magnitude(shape):
    """float16: neighbouring rows 2^16 apart, in h and in u."""
    p = ranged(F16, shape, b=2.0 ** -6)
    _, adapters, rows, k, n, rank = shape
    steps = 2.0 ** np.random.default_rng(rows).integers(-12, 5, (rows, 1))
    put(p, "x", slice(None), p.f["x"] * steps)
    put(p, "g", slice(None), p.f["g"] * steps)
    p.forward()
    once(oracle.to_f64(p.y.numpy(), F16), *layer(p), k + rank + 2, F16)
    dx, da, db = p.backward()
    once(oracle.to_f64(dx.numpy(), F16), *input_gradient(p), n + rank + 2, F16)
    for got, (want, size, _), width in zip((da, db), gradients(p), (n, k)):
        once(oracle.to_f64(got.numpy(), F16), want, size, rows + width + 2, F16)


@pytest.mark.parametrize("dt", [BF16, F16], ids=ids_of)
@pytest.mark.parametrize("k, n, x_cs", [(136, 5, 1), (5, 136, 1), (72, 136, 2), (200, 72, 1)])
def test_gradients_asked_for_alone(k, n, x_cs, dt):
    """A factor's gradient has the same bits whichever others are asked for, also where the kernels take one of the two only (widths below a vector, x with a column stride)."""
    rows, rank, adapters = 700, 12, 3
    p = Adapters(dt, 7, adapters, rows, k, n, rank, behind=2)
    p.forward()
    wide = oracle.to_storage(np.zeros((rows, k * x_cs)), dt)
    wide[:, ::x_cs] = p.s["x"]
    x, d = Dev(wide, dt), p.d

    def backward(which):
        out = [Dev(oracle.to_storage(np.full(shape, 3.0), dt), dt) if use else None for use, shape in zip(which, ((rows, k), (adapters, k, rank), (adapters, rank, n)))]
        u = Dev.empty((rows, rank), p.acc)
        call("rp_hip_adapter_linear_backward", *[ptr(o) for o in out], u.ptr, d["g"].ptr, x.ptr, d["w"].ptr, d["a"].ptr, d["b"].ptr, p.h.ptr, *p.plan(),
             n, k * x_cs, x_cs, *p.w_st, k, 0, 0, 0, dt)
        return out

    whole = backward((1, 1, 1))
    p.check_backward(whole)
    for which in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 1, 1), (1, 1, 0), (1, 0, 1)):
        for one, ref in zip(backward(which), whole):
            assert one is None or np.array_equal(one.numpy(), ref.numpy()), which


@pytest.mark.parametrize("dt", [BF16, F16, F32], ids=ids_of)
@pytest.mark.parametrize("groups, rows, k, n, transposed", [(6, 1999, 519, 1031, False), (3, 14949, 104, 427, False), (4, 130, 520, 384, True), (3, 700, 256, 5, False), (5, 900, 7, 264, False), (9, 40, 2048, 264, True)])
def test_gradients_of_groups_asked_for_alone(groups, rows, k, n, transposed, dt):
    p = Grouped(dt, groups, rows, k, n, transposed=transposed)
    whole = [o.numpy() for o in p.backward()]
    for which in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 1, 1), (1, 1, 0), (1, 0, 1)):
        for one, ref in zip(p.backward(which=which), whole):
            assert one is None or np.array_equal(one.numpy(), ref), which


@pytest.mark.parametrize("dt", [BF16, F16], ids=ids_of)
@pytest.mark.parametrize("shape", SMALL + [(5, 3, 2048, 264, 2056, 24)] + LARGE[:1], ids=lambda s: "x".join(map(str, s)))
def test_rounded_once(shape, dt):
    """y and dx: the shared product, the bias and the term together.  (dx added to what is there: that sum is a rounding of its own.)"""
    p = Adapters(dt, *shape, behind=2)
    _, _, rows, k, n, rank = shape
    p.forward()
    once(oracle.to_f64(p.y.numpy(), dt), *layer(p), k + rank + 2, dt)
    want, size = input_gradient(p)
    once(oracle.to_f64(p.backward(which=(1, 0, 0))[0].numpy(), dt), want, size, n + rank + 2, dt)
    got = oracle.to_f64(p.backward(accumulate=1, which=(1, 0, 0))[0].numpy(), dt)
    within(got, want + 3, size + 3, n + rank + 2 + SPLIT[dt], dt, added=3.0)


@pytest.mark.parametrize("dt", [BF16, F16, F32], ids=ids_of)
@pytest.mark.parametrize("rows, k, n", [(60, 64, 96), (500, 317, 256), (12, 1024, 512), (500, 136, 523), (900, 1032, 1048), (9, 2048, 264)])
def test_infinities_of_one_group(rows, k, n, dt):
    """An infinity and a NaN in one group's weight, and one in a row of x, reach that group's rows, or that row, in the columns they belong to."""
    p = Grouped(dt, 3, rows, k, n, bias=False)
    p.sw[1, k // 2, 5:8] = oracle.to_storage(np.array([np.inf, np.nan, -np.inf]), dt)
    p.dw, p.w = Dev(p.sw, dt), oracle.to_f64(p.sw, dt)
    y, dx = (oracle.to_f64(o.numpy(), dt) for o in (p.forward(), p.backward(which=(1, 0, 0))[0]))
    with np.errstate(invalid="ignore"):
        for got, left, right, terms in ((y, p.x, p.w, k), (dx, p.g, p.w.transpose(0, 2, 1), n)):
            for i, (f, t) in enumerate(zip(p.offsets, p.offsets[1:])):
                want = left[f:t] @ right[i]
                assert np.array_equal(np.isnan(got[f:t]), np.isnan(want)) and np.array_equal(got[f:t][np.isinf(want)], want[np.isinf(want)])
                fine = np.isfinite(want)
                within(np.where(fine, got[f:t], 0), np.where(fine, want, 0), np.where(fine, np.abs(left[f:t]) @ np.where(np.isfinite(right[i]), np.abs(right[i]), 0), 0), terms, dt)
    p = Grouped(dt, 3, rows, k, n, bias=False)
    b = rows // 2
    group = int(np.searchsorted(p.offsets, b, "right")) - 1
    p.sx[b, 3] = oracle.to_storage(np.array([np.inf]), dt)[0]
    p.dx, p.x = Dev(p.sx, dt), oracle.to_f64(p.sx, dt)[:, :k]
    y, dw = oracle.to_f64(p.forward().numpy(), dt), oracle.to_f64(p.backward(which=(0, 1, 0))[1].numpy(), dt)
    with np.errstate(invalid="ignore"):                     # (zero times infinity is NaN)
        assert np.array_equal(y[b], p.w[group, 3] * np.inf, equal_nan=True)
        assert np.array_equal(dw[group, 3], p.g[b] * np.inf, equal_nan=True)
    assert np.isfinite(np.delete(y, b, axis=0)).all()
    dw[group, 3] = 0
    assert np.isfinite(dw).all()
