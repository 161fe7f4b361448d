"""Adapters of many requests side by side: what one adapter, or one request's range of values, may not do to the others."""
import numpy as np
import pytest

import oracle
from recpulse_amd import capi
from devhelp import BF16, F16, F32, Dev
from test_grouped_gpu import HALF_STEP, TINY, UNIT, Adapters, call, ids_of, ptr, within

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
BESIDE = [(9, 4, 32, 256, 512, 16), (90, 5, 300, 264, 136, 8), (7, 3, 700, 264, 520, 12), (6, 3, 2100, 520, 1031, 16), (9, 4, 4100, 512, 4096, 32), (9, 4, 4096, 512, 4096, 40)]


@pytest.mark.parametrize("dt", [BF16, F16, F32], ids=ids_of)
@pytest.mark.parametrize("shape", BESIDE, ids=lambda s: "x".join(map(str, s)))
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
    once(oracle.to_f64(p.backward()[0].numpy(), dt), *input_gradient(p), n + rank + 2, dt)
