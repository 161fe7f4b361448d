"""Calls of more tiles than one launch takes (fewer than 2^32 threads), and of hundreds of thousands of groups.  What is far too large to check in full is checked at its first, last
and some other rows."""
import numpy as np
import pytest

import oracle
from recpulse_amd import capi
from devhelp import BF16, F16, F32, Dev
from test_grouped_gpu import Adapters, call, ids_of, ints, within

pytestmark = pytest.mark.gpu


def rows_of(buf, at, width, dt):
    """Row `at` of a device array of rows of `width`."""
    out = np.empty(width, capi.NP_STORAGE[dt])
    call("rp_hip_memcpy_d2h", out.ctypes.data, buf.ptr + int(at) * out.nbytes, out.nbytes)
    return oracle.to_f64(out, dt)


def some(rng, rows, count=40):
    return np.unique(np.concatenate([[0, 1, rows - 2, rows - 1], rng.integers(0, rows, count)]))


def small(rng, shape, dt, scale=1.0):
    s = oracle.to_storage(rng.normal(0, scale, shape), dt)
    return Dev(s, dt), oracle.to_f64(s, dt)


@pytest.mark.parametrize("dt, rows, k, n, rank", [(BF16, 131072, 16, 4096, 8), (BF16, 4300000, 8, 8, 1), (F32, 280000, 8, 4096, 4), (F32, 280000, 8, 8, 256), (F16, 20000, 24, 264, 12)])
def test_adapters_of_a_segment_a_row(dt, rows, k, n, rank):
    rng = np.random.default_rng(rows)
    adapters = 50
    (x, fx), (w, fw), (a, fa), (b, fb) = (small(rng, s, dt) for s in ((rows, k), (k, n), (adapters, k, rank), (adapters, rank, n)))
    ids = rng.integers(-1, adapters, rows)
    acc = F32
    y, h = Dev.empty((rows, n), dt), Dev.empty((rows, rank), acc)
    dids, off = ints(ids), ints(np.arange(rows + 1))
    call("rp_hip_adapter_linear_forward", y.ptr, h.ptr, x.ptr, w.ptr, None, a.ptr, b.ptr, None, dids.ptr, off.ptr, rows, adapters, rows, k, n, rank, k, 1, n, 1, n, dt)
    for i in some(rng, rows):
        want, size = fx[i] @ fw, np.abs(fx[i]) @ np.abs(fw)
        if ids[i] >= 0:
            low, lsize = fx[i] @ fa[ids[i]], np.abs(fx[i]) @ np.abs(fa[ids[i]])
            within(rows_of(h, i, rank, acc), low, lsize, k, acc)
            want, size = want + low @ fb[ids[i]], size + lsize @ np.abs(fb[ids[i]])
        within(rows_of(y, i, n, dt), want, size, k + rank + 130, dt, roundings=2)


def test_grouped_rows_of_a_group_a_row():
    """One weight for all groups (a stride of 0): 16-bit rows that stream it, and rows of no whole vectors; on either side of where the groups are bisected and left to the generic kernel."""
    for rows, k, n, dt in ((280000, 8, 4096, BF16), (70000, 9, 520, BF16), (256, 16, 264, F16), (257, 16, 264, F16), (4096, 17, 261, BF16), (4097, 17, 261, BF16), (2048, 20, 70, F32), (2049, 20, 70, F32)):
        rng = np.random.default_rng(n)
        (x, fx), (w, fw) = (small(rng, s, dt) for s in ((rows, k), (k, n)))
        y, off = Dev.empty((rows, n), dt), ints(np.arange(rows + 1))
        call("rp_hip_grouped_linear_forward", y.ptr, x.ptr, w.ptr, None, off.ptr, rows, rows, k, n, k, 1, 0, n, 1, n, dt)
        for i in some(rng, rows):
            within(rows_of(y, i, n, dt), fx[i] @ fw, np.abs(fx[i]) @ np.abs(fw), k, dt)


@pytest.mark.parametrize("dt", [BF16, F32], ids=ids_of)
@pytest.mark.parametrize("groups", [300, 5000, 300000])
def test_very_many_uneven_groups(groups, dt):
    """Most groups empty, rows before the first and behind the last left as they are, forward and backward."""
    rng = np.random.default_rng(groups)
    rows, k, n, first, behind = 3000, 24, 72, 7, 11
    sizes = rng.multinomial(rows - first - behind, rng.dirichlet(np.full(groups, 0.05)))
    offsets = first + np.concatenate([[0], np.cumsum(sizes)])
    (x, fx), (g, fg), (w, fw) = small(rng, (rows, k), dt), small(rng, (rows, n), dt), small(rng, (k, n), dt)
    mark = [Dev(oracle.to_storage(np.full(s, 3.0), dt), dt) for s in ((rows, n), (rows, k), (groups, k, n))]
    y, dx, dw = mark
    off = ints(offsets)
    call("rp_hip_grouped_linear_forward", y.ptr, x.ptr, w.ptr, None, off.ptr, groups, rows, k, n, k, 1, 0, n, 1, n, dt)
    call("rp_hip_grouped_linear_backward", dx.ptr, dw.ptr, None, g.ptr, x.ptr, w.ptr, off.ptr, groups, rows, k, n, n, k, 1, 0, n, 1, k, 0, 0, 0, dt)
    inside = slice(first, rows - behind)
    for out, left, right, terms in ((y, fx, fw, k), (dx, fg, fw.T, n)):
        got = oracle.to_f64(out.numpy(), dt)
        within(got[inside], left[inside] @ right, np.abs(left[inside]) @ np.abs(right), terms, dt)
        assert np.all(got[:first] == 3.0) and np.all(got[rows - behind:] == 3.0)
    for e in np.concatenate([np.argsort(sizes)[-20:], some(rng, groups)]):
        s = slice(offsets[e], offsets[e + 1])
        within(rows_of(dw, e, k * n, dt), (fx[s].T @ fg[s]).reshape(-1), (np.abs(fx[s]).T @ np.abs(fg[s])).reshape(-1), rows, dt)


@pytest.mark.parametrize("dt", [BF16, F16, F32], ids=ids_of)
@pytest.mark.parametrize("segments", [300, 5000])
def test_very_many_uneven_segments(segments, dt):
    rows, k, n, rank, adapters = 2500, 40, 136, 8, 5
    p = Adapters(dt, segments, adapters, rows, k, n, rank, behind=9)
    rng = np.random.default_rng(segments)
    p.offsets = np.concatenate([[0], np.cumsum(rng.multinomial(rows - 16, rng.dirichlet(np.full(segments, 0.05))))]).astype(np.int32) + 7
    p.doff = ints(p.offsets)
    p.forward()
    p.check_forward()
    p.check_backward(p.backward())


@pytest.mark.parametrize("dt, groups, width", [(BF16, 2200000, 8), (BF16, 17000000, 4), (F32, 2200000, 8)])
def test_weights_of_millions_of_groups(dt, groups, width):
    rng = np.random.default_rng(groups)
    rows = 4000
    (x, fx), (g, fg) = (small(rng, (rows, width), dt) for _ in range(2))
    sizes = np.zeros(groups, dtype=np.int64)
    at = np.unique(np.concatenate([[0, groups - 1], rng.integers(0, groups, 300)]))
    sizes[at] = rng.multinomial(rows, np.full(at.size, 1 / at.size))
    offsets = np.concatenate([[0], np.cumsum(sizes)])
    dw, off = Dev.empty((groups, width * width), dt), ints(offsets)
    call("rp_hip_memset", dw.ptr, 0xff, dw.buf.nbytes)
    call("rp_hip_grouped_linear_backward", None, dw.ptr, None, g.ptr, x.ptr, None, off.ptr, groups, rows, width, width, width, width, 1, 0, 0, 0, width, 0, 0, 0, dt)
    for e in np.concatenate([at, some(rng, groups)]):
        s = slice(offsets[e], offsets[e + 1])
        within(rows_of(dw, e, width * width, dt), (fx[s].T @ fg[s]).reshape(-1), (np.abs(fx[s]).T @ np.abs(fg[s])).reshape(-1), rows, dt)


@pytest.mark.parametrize("dt, adapters", [(BF16, 6400000), (F32, 4300000)])
def test_gradients_of_millions_of_adapters(dt, adapters):
    rng = np.random.default_rng(adapters)
    rows, width = 300, 8
    (x, fx), (g, fg), (h, fh) = small(rng, (rows, width), dt), small(rng, (rows, width), dt), small(rng, (rows, 1), F32)
    offsets, ids = np.array([0, 100, 130, 300]), np.array([0, adapters - 1, 77])
    b = Dev.empty((adapters, 1, width), dt)
    call("rp_hip_memset", b.ptr, 0x3c, b.buf.nbytes)
    fb = oracle.to_f64(np.full(width * capi.DTYPE_SIZE[dt], 0x3c, np.uint8).view(capi.NP_STORAGE[dt]), dt)
    u, da, db = Dev.empty((rows, 1), F32), Dev.empty((adapters, width), dt), Dev.empty((adapters, width), dt)
    dids, off = ints(ids), ints(offsets)
    for o in (da, db):
        call("rp_hip_memset", o.ptr, 0xff, o.buf.nbytes)
    call("rp_hip_adapter_linear_backward", None, da.ptr, db.ptr, u.ptr, g.ptr, x.ptr, None, None, b.ptr, h.ptr, None, dids.ptr, off.ptr, 3, adapters, rows, width, width, 1,
         width, width, 1, 0, 0, width, 0, 0, 0, dt)
    fu = fg @ fb
    for s, (i, j) in enumerate(zip(offsets, offsets[1:])):
        for got, low, other in ((da, fu, fx), (db, fh[:, 0], fg)):
            within(rows_of(got, ids[s], width, dt), low[i:j] @ other[i:j], np.abs(low[i:j]) @ np.abs(other[i:j]) + (np.abs(fg[i:j]) @ fb) @ np.abs(other[i:j]) * (got is da), rows + width + 130, dt)
    for e in some(rng, adapters):
        if e not in ids:
            assert not rows_of(da, e, width, dt).any() and not rows_of(db, e, width, dt).any()


def test_route_backward_of_more_tokens_than_a_launch():
    tokens, experts = (1 << 28) + 100, 2
    logits, grad = Dev.empty((tokens, experts), BF16), Dev.empty((tokens, experts), BF16)
    weights, gw, ids = Dev.empty((tokens, 1), F32), Dev.empty((tokens, 1), F32), capi.DeviceBuffer(4 * tokens)
    call("rp_hip_memset", logits.ptr, 0, logits.buf.nbytes)                # equal logits: expert 0 with weight 1 / 2
    call("rp_hip_memset", ids.ptr, 0, ids.nbytes)
    for buf, value in ((weights, 0x3f), (gw, 0x3f)):                       # 0.747...
        call("rp_hip_memset", buf.ptr, value, buf.buf.nbytes)
    call("rp_hip_memset", grad.ptr, 0xff, grad.buf.nbytes)
    call("rp_hip_route_backward", grad.ptr, gw.ptr, weights.ptr, ids.ptr, logits.ptr, experts, tokens, experts, 1, 0, BF16)
    v = float(np.full(4, 0x3f, np.uint8).view(np.float32)[0])
    want = np.array([0.5 * (v - v * v), -0.5 * v * v])
    for t in (0, 1, 12345678, (1 << 28) - 1, 1 << 28, tokens - 1):
        got = rows_of(grad, t, experts, BF16)
        assert np.all(np.abs(got - want) <= 2.0 ** -8 * np.abs(want) + 2.0 ** -22)
