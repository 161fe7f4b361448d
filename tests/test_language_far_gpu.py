"""Layer norm, gated layers, the loss of a large vocabulary and distillation where sizes and offsets are large, beside each other on two streams, and with rows whose values do not count."""
import ctypes

import numpy as np
import pytest

from langhelp import *
from recpulse_amd import capi

pytestmark = pytest.mark.gpu

FAR = 1 << 21                                                   # elements from row to row: 1200 rows pass 2^31


class Far:
    """[rows, cols] on the device with rows `rs` apart, zeros between and where no values are given: {row: values}, or all rows."""

    def __init__(self, rows, cols, dtype, values=None, rs=FAR):
        self.shape, self.dtype, self.rs, self.cs = (rows, cols), dtype, rs, 1
        self.size = capi.DTYPE_SIZE[dtype]
        self.buf = capi.DeviceBuffer(((rows - 1) * rs + cols) * self.size)
        capi.check(capi.lib().rp_hip_memset(self.buf.ptr, 0, self.buf.nbytes), "memset")
        capi.synchronize()
        self.stored = np.dtype(storage(np.zeros(1), dtype).dtype)
        for row, v in (values.items() if isinstance(values, dict) else enumerate([] if values is None else values)):
            self.write(row, 0, v)

    def write(self, row, col, values):
        v = np.ascontiguousarray(storage(values, self.dtype))
        capi.check(capi.lib().rp_hip_memcpy_h2d(self.buf.at((row * self.rs + col) * self.size), v.ctypes.data_as(ctypes.c_void_p), v.nbytes), "h2d")

    def bits(self, row, col=0, width=None):
        out = np.empty(width or self.shape[1], self.stored)
        capi.check(capi.lib().rp_hip_memcpy_d2h(out.ctypes.data_as(ctypes.c_void_p), self.buf.at((row * self.rs + col) * self.size), out.nbytes), "d2h")
        return out

    def read(self, row, col=0, width=None):
        return f64(self.bits(row, col, width), self.dtype)

    @property
    def ptr(self):
        return self.buf.ptr


def same_rows(near, far, rows, what):
    bits = near.bits()
    for row in rows:
        assert np.array_equal(bits[row], far.bits(row)), f"{what}, row {row}"


SOME = [0, 1, 63, 512, 1022, 1023, 1024, 1025, 1100, 1198, 1199]


@pytest.mark.parametrize("d", [512, 520, 5])
def test_norm_of_rows_far_apart(d):
    rows, dtype = 1200, BF16
    rng = np.random.default_rng(d)
    xv, gv, w = rng.normal(size=(rows, d)), rng.normal(size=(rows, d)), vector(rng.normal(size=d), dtype)
    space = room(capi.lib().rp_hip_layer_norm_workspace(rows, d, dtype))
    results = []
    for make in (lambda v: Operand(v, dtype), lambda v: Far(rows, d, dtype, v)):
        x, dy = make(xv), make(gv)
        y, dx = (Output(rows, d, dtype), Output(rows, d, dtype)) if not results else (Far(rows, d, dtype), Far(rows, d, dtype))
        stats, dw, db = Output(rows, 2, F32), Output(1, d, dtype), Output(1, d, dtype)
        capi.check(capi.lib().rp_hip_layer_norm_forward(y.ptr, stats.ptr, x.ptr, w.ptr, None, rows, d, y.rs, x.rs, 1e-5, dtype), "forward")
        capi.check(capi.lib().rp_hip_layer_norm_backward(dx.ptr, dw.ptr, db.ptr, dy.ptr, x.ptr, w.ptr, stats.ptr, space.ptr, rows, d, dy.rs, x.rs, dx.rs, 0, 0, 0, dtype), "backward")
        capi.synchronize()
        results.append((y, dx, stats, dw, db))
    same_rows(results[0][0], results[1][0], SOME, "y")
    same_rows(results[0][1], results[1][1], SOME, "dx")
    for near, far in zip(results[0][2:], results[1][2:]):
        assert np.array_equal(near.bits(), far.bits())


def test_distillation_of_rows_far_apart():
    rows, classes, k = 1200, 1000, 20
    rng = np.random.default_rng(1)
    lv, teacher = rng.normal(size=(rows, classes)), Operand(rng.normal(size=(rows, k)), BF16)
    ids = ints(rng.integers(0, classes, (rows, k)))
    results = []
    for logits in (Operand(lv, BF16), Far(rows, classes, BF16, lv)):
        loss, stats, grad, again = Output(1, rows, F32), Output(1, 3 * rows, F32), Output(rows, classes, BF16), Output(rows, classes, BF16)
        capi.check(capi.lib().rp_hip_distillation_forward(loss.ptr, grad.ptr, stats.ptr, logits.ptr, ids.ptr, teacher.ptr, None, rows, classes, k, logits.rs, 2.0, 0, BF16), "forward")
        capi.check(capi.lib().rp_hip_distillation_backward(again.ptr, stats.ptr, logits.ptr, ids.ptr, teacher.ptr, None, rows, classes, k, logits.rs, 2.0, 0, BF16), "backward")
        results.append([o.bits() for o in (loss, stats, grad, again)])
    for near, far in zip(*results):
        assert np.array_equal(near, far)


def test_distillation_of_more_than_2_to_31_logits():
    rows, classes, k, ends = 40000, 65536, 10, 48
    rng = np.random.default_rng(2)
    at_ends = list(range(ends)) + list(range(rows - ends, rows))
    values, idv, tv = rng.normal(size=(2 * ends, classes)), rng.integers(0, classes, (2 * ends, k)), rng.normal(size=(2 * ends, k))
    all_ids, all_teacher = np.full((rows, k), -1), np.zeros((rows, k))
    all_ids[at_ends], all_teacher[at_ends] = idv, tv
    logits, grad = Far(rows, classes, BF16, dict(zip(at_ends, values)), rs=classes), Far(rows, classes, BF16, rs=classes)
    few_grad = Output(2 * ends, classes, BF16)
    losses = []
    for count, l, g, i, t in ((rows, logits, grad, all_ids, all_teacher), (2 * ends, Operand(values, BF16), few_grad, idv, tv)):
        loss, stats = Output(1, count, F32), Output(1, 3 * count, F32)
        idev, tdev = ints(i), Operand(t, BF16)
        capi.check(capi.lib().rp_hip_distillation_forward(loss.ptr, g.ptr, stats.ptr, l.ptr, idev.ptr, tdev.ptr, None, count, classes, k, classes, 1.0, 0, BF16), "forward")
        losses.append(loss.bits()[0])
    assert np.array_equal(losses[0][at_ends], losses[1]) and np.all(losses[0][ends:-ends] == 0)
    bits = few_grad.bits()
    for i, row in enumerate(at_ends):
        assert np.array_equal(grad.bits(row), bits[i]), row
    assert np.all(grad.bits(rows // 2) == 0)


@pytest.mark.parametrize("n,dtype", [(64, BF16), (264, F16)])
def test_gated_layer_of_rows_far_apart(n, dtype):
    rows, k = 1200, 136
    rng = np.random.default_rng(n)
    xv, gv = rng.normal(size=(rows, k)), rng.normal(size=(rows, n))
    w = Operand(rng.normal(0, k ** -0.5, size=(k, 2 * n)), dtype)
    results = []
    for make, out in ((lambda v: Operand(v, dtype), lambda c: Output(rows, c, dtype)), (lambda v: Far(rows, v.shape[1], dtype, v), lambda c: Far(rows, c, dtype))):
        x, dh, h, dx = make(xv), make(gv), out(n), out(k)
        z, dz, dw = Output(rows, 2 * n, F32), Output(rows, 2 * n, dtype), Output(k, 2 * n, dtype)
        capi.check(capi.lib().rp_hip_gated_linear_forward(h.ptr, z.ptr, x.ptr, w.ptr, None, rows, k, n, 0, x.rs, 1, w.rs, 1, h.rs, dtype), "forward")
        capi.check(capi.lib().rp_hip_gated_linear_backward(dx.ptr, dw.ptr, None, dz.ptr, dh.ptr, z.ptr, x.ptr, w.ptr, rows, k, n, 0, dh.rs, x.rs, 1, w.rs, 1, dx.rs, 2 * n, 1, 0, 0, 0, dtype), "backward")
        capi.synchronize()
        results.append((h, dx, z, dz, dw))
    same_rows(results[0][0], results[1][0], SOME, "h")
    same_rows(results[0][1], results[1][1], SOME, "dx")
    for near, far in zip(results[0][2:4], results[1][2:4]):
        assert np.array_equal(near.bits(), far.bits())
    # dw may be added up on other tiles (x^T has rows of another alignment): both within a sum of `rows` products in any order, and a rounding
    dw, other, dz = results[0][4].read(), results[1][4].read(), results[0][3].read()
    xs = f64(storage(xv, dtype), dtype)
    assert_within(other, dw, 2 * (rows + 8) * 2.0 ** -24 * (np.abs(xs).T @ np.abs(dz)) + 2 * HALF[dtype] * (np.abs(dw) + np.abs(other)) + TINY[dtype], "dw")


def test_gated_layer_of_more_than_2_to_31_sums():
    rows, k, n, dtype = 70000, 64, 16384, BF16
    rng = np.random.default_rng(4)
    x, w = Operand(rng.normal(size=(rows, k)), dtype), Operand(rng.normal(0, k ** -0.5, size=(k, 2 * n)), dtype)
    z, h, dh = Far(rows, 2 * n, F32, rs=2 * n), Far(rows, n, dtype, rs=n), Far(rows, n, dtype, rs=n)
    dz, dx = Far(rows, 2 * n, dtype, rs=2 * n), Output(rows, k, dtype)
    some = [0, 1, 32767, 32768, 65535, 65536, rows - 65, rows - 1]
    for row in some:
        dh.write(row, 0, rng.normal(size=n))
    capi.check(capi.lib().rp_hip_gated_linear_forward(h.ptr, z.ptr, x.ptr, w.ptr, None, rows, k, n, 0, k, 1, 2 * n, 1, n, dtype), "forward")
    capi.check(capi.lib().rp_hip_gated_linear_backward(dx.ptr, None, None, dz.ptr, dh.ptr, z.ptr, x.ptr, w.ptr, rows, k, n, 0, n, k, 1, 2 * n, 1, k, 0, 1, 0, 0, 0, dtype), "backward")
    got_dx = dx.read()
    for row in some:
        zr, size = z.read(row), np.abs(x.values[row]) @ np.abs(w.values)
        assert_within(zr, x.values[row] @ w.values, (k + 8) * 2.0 ** -24 * size, "z")
        act, slope = gate_reference(zr[:n], "silu")
        # (from the device's z: float32 exp, divisions and products, and the one rounding)
        assert_within(h.read(row), act * zr[n:], rounded(2.0 ** -20 * np.abs(act * zr[n:]), act * zr[n:], dtype), "h")
        up = dh.read(row)
        want = np.concatenate([up * zr[n:] * slope, up * act])
        slack = 2.0 ** -20 * np.concatenate([np.abs(up * zr[n:]), np.abs(up * act)])
        d = dz.read(row)
        assert_within(d, want, rounded(slack, want, dtype), "dz")
        assert_within(got_dx[row], d @ w.values.T, rounded((2 * n + 8) * 2.0 ** -24 * (np.abs(d) @ np.abs(w.values).T), d @ w.values.T, dtype), "dx")


@pytest.mark.parametrize("dtype", [BF16, F16], ids=NAMES.get)
@pytest.mark.parametrize("rows,n", [(40, 5), (40, 64), (600, 300), (4, (1 << 21) + 8)])
def test_sums_of_a_gated_layer_are_made_before_dz_is_rounded(rows, n, dtype):
    """Rows whose dz are 1 + 2^-12 and -1 by turns: rounded, each pair would cancel."""
    z, dh = np.full((rows, 2 * n), 1.0), np.ones((rows, n))
    z[::2, :n], z[::2, n:] = 1 + 2.0 ** -12, 1 + 2.0 ** -11
    dh[1::2] = -1
    zd, dhd, dz, db = Operand(z, F32), Operand(dh, dtype), Output(rows, 2 * n, dtype), Output(1, 2 * n, dtype)
    capi.check(capi.lib().rp_hip_gated_linear_backward(None, None, db.ptr, dz.ptr, dhd.ptr, zd.ptr, None, None, rows, 8, n, GATES["relu"], n, 8, 1, 2 * n, 1, 8, 2 * n, 1, 0, 0, 0, dtype), "backward")
    got = db.read()[0]
    assert np.all(got[:n] == rows / 2 * 2.0 ** -11) and np.all(got[n:] == rows / 2 * 2.0 ** -12)      # (exact in every type)
    # dz: bf16 steps by 2^-7 above 1, float16 by 2^-10
    assert np.array_equal(np.abs(dz.read()), np.ones((rows, 2 * n)))


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=NAMES.get)
def test_vocabulary_loss_of_rows_far_apart(dtype):
    rows, k, classes = 1200, 136, 1000
    rng = np.random.default_rng(5)
    xv, w = rng.normal(size=(rows, k)), Operand(rng.normal(0, k ** -0.5, size=(k, classes)), dtype)
    targets = ints(np.where(np.arange(rows) % 5, rng.integers(0, classes, rows), -1))
    space = room(capi.lib().rp_hip_linear_cross_entropy_workspace(rows, k, classes, 1, dtype))
    results = []
    for x, dx in ((Operand(xv, dtype), Output(rows, k, dtype)), (Far(rows, k, dtype, xv), Far(rows, k, dtype))):
        loss, stats, dw = Output(1, 1, F32), Output(1, 2 * rows + 1, F32), Output(k, classes, dtype)
        capi.check(capi.lib().rp_hip_linear_cross_entropy_forward(loss.ptr, stats.ptr, x.ptr, w.ptr, None, targets.ptr, space.ptr, rows, k, classes, 1, x.rs, 1, classes, 1, dtype), "forward")
        capi.check(capi.lib().rp_hip_linear_cross_entropy_backward(dx.ptr, dw.ptr, None, x.ptr, w.ptr, None, targets.ptr, stats.ptr, None, space.ptr, rows, k, classes, 1,
                                                                   x.rs, 1, classes, 1, dx.rs, classes, 1, 0, 0, 0, dtype), "backward")
        capi.synchronize()
        results.append((dx, loss, stats, dw))
    same_rows(results[0][0], results[1][0], SOME, "dx")
    for near, far in zip(results[0][1:3], results[1][1:3]):
        assert np.array_equal(near.bits(), far.bits())
    # float32's dw comes from another kernel where x passes 2^31 bytes: both sums of `rows` products are off by (rows + 8) half steps of their sizes, and 2^-22 where the products are split
    # into halves; d itself is the same (dx is), and known to better than a thousandth
    xs = f64(storage(xv, dtype), dtype)
    d = np.abs(vocab_reference(xs, w.values, None, targets.to_numpy(np.int32, rows), 1, 1.0)[2]) * 1.001 + 1e-9
    dw, other = results[0][3].read(), results[1][3].read()
    assert_within(other, dw, 2 * ((rows + 8) * 2.0 ** -24 + 2.0 ** -22) * (np.abs(xs).T @ d) + 2 * HALF[dtype] * (np.abs(dw) + np.abs(other)) + TINY[dtype], "dw")


@pytest.mark.parametrize("tied", [False, True], ids=["rows", "transposed"])
def test_weights_of_more_than_2_to_31_elements(tied):
    """... that are zeros but for those of some classes at either end: the others' logits are zeros, and their gradients one number a row."""
    rows, k, classes, dtype = 24, 8192, 300008, BF16
    rng = np.random.default_rng(6)
    some = np.array([0, 1, 7, classes // 2, classes - 257, classes - 2, classes - 1])
    wv = f64(storage(rng.normal(0, k ** -0.5, size=(some.size, k)), dtype), dtype)
    w, dw = (Far(classes, k, dtype, dict(zip(some, wv)), rs=k), Far(classes, k, dtype, rs=k)) if tied else (Far(k, classes, dtype, rs=classes), Far(k, classes, dtype, rs=classes))
    if not tied:
        line = np.zeros((k, classes), storage(np.zeros(1), dtype).dtype)
        line[:, some] = storage(wv.T, dtype)
        capi.check(capi.lib().rp_hip_memcpy_h2d(w.ptr, line.ctypes.data_as(ctypes.c_void_p), line.nbytes), "h2d")
        del line
    x = Operand(rng.normal(size=(rows, k)), dtype)
    targets = some[np.arange(rows) % some.size]
    targets[3] = 12345                                          # one whose weights are zeros
    loss, stats, dx, tdev = Output(1, rows, F32), Output(1, 2 * rows + 1, F32), Output(rows, k, dtype), ints(targets)
    space = room(capi.lib().rp_hip_linear_cross_entropy_workspace(rows, k, classes, 1, dtype))
    strides = (1, k) if tied else (classes, 1)
    capi.check(capi.lib().rp_hip_linear_cross_entropy_forward(loss.ptr, stats.ptr, x.ptr, w.ptr, None, tdev.ptr, space.ptr, rows, k, classes, 0, k, 1, *strides, dtype), "forward")
    capi.check(capi.lib().rp_hip_linear_cross_entropy_backward(dx.ptr, dw.ptr, None, x.ptr, w.ptr, None, tdev.ptr, stats.ptr, None, space.ptr, rows, k, classes, 0,
                                                               k, 1, *strides, k, *strides, 0, 0, 0, dtype), "backward")
    u = 2.0 ** -24
    z, size = x.values @ wv.T, np.abs(x.values) @ np.abs(wv).T
    z_off = (k + 8) * u * size
    lse = np.log(classes - some.size + np.exp(z).sum(1))
    lse_off = z_off.max(1) + u * (300 + 4 * size.max(1)) + 2 * u * lse      # (a sum by teams adds fewer than 300 of these one after the other)
    of = np.array([np.flatnonzero(some == t)[0] if t in some else -1 for t in targets])
    zt = np.where(of >= 0, z[np.arange(rows), of], 0.0)
    assert_within(loss.read()[0], lse - zt, lse_off + np.where(of >= 0, z_off[np.arange(rows), of], 0.0) + 2 * u * lse, "loss")
    # the gradient of the logits of the classes with weights, and of another
    p = np.exp(z - lse[:, None])
    d = p - (of[:, None] == np.arange(some.size))
    d_off = p * 1.1 * (z_off + lse_off[:, None] + 16 * u * (1 + np.abs(np.log(p)))) + 4 * u
    d_off = d_off + HALF[dtype] * (np.abs(d) + d_off)
    want = d @ wv
    assert_within(dx.read(), want, rounded(d_off @ np.abs(wv) + (classes + 8) * u * ((np.abs(d) + d_off) @ np.abs(wv)), want, dtype), "dx")
    other = np.exp(-lse)
    other_off = other * (1.1 * lse_off + 64 * u * lse) + HALF[dtype] * other * 1.01
    places = [0, 1, 4095, 4096, k - 1]
    for j, v in list(enumerate(some)) + [(-1, 12346), (-1, classes - 3)]:
        dv, off = (d[:, j], d_off[:, j]) if j >= 0 else (other, other_off)
        want = x.values.T @ dv
        bound = rounded(np.abs(x.values).T @ off + (rows + 8) * u * (np.abs(x.values).T @ (np.abs(dv) + off)), want, dtype)
        if tied:
            assert_within(dw.read(v), want, bound, "dw")
        else:
            for i in places:
                assert_within(dw.read(i, v, 1), want[i:i + 1], bound[i:i + 1], "dw")


@pytest.mark.parametrize("k", [16384, 33000])
def test_few_rows_of_a_wide_float32_layer(k):
    """The gradient of x is a product whose partial sums may be more than the workspace has room for.  Weights that overlap, w[i, v] = h[i + 4 v], take little memory."""
    rows, classes, dtype = 8, 70000, F32
    rng = np.random.default_rng(7)
    h = vector(rng.normal(0, k ** -0.5, size=k + 4 * classes), dtype)
    x, targets = Operand(rng.normal(size=(rows, k)), dtype), rng.integers(0, classes, rows)
    view = np.lib.stride_tricks.as_strided(h.values[0], (classes, k), (4 * 8, 8))
    steps = range(0, classes, 2000)
    z = np.concatenate([x.values @ np.ascontiguousarray(view[v:v + 2000]).T for v in steps], 1)
    size = np.concatenate([np.abs(x.values) @ np.abs(view[v:v + 2000]).T for v in steps], 1)
    loss, stats, dx, tdev = Output(1, rows, F32), Output(1, 2 * rows + 1, F32), Output(rows, k, dtype), ints(targets)
    space = room(capi.lib().rp_hip_linear_cross_entropy_workspace(rows, k, classes, 1, dtype))
    capi.check(capi.lib().rp_hip_linear_cross_entropy_forward(loss.ptr, stats.ptr, x.ptr, h.ptr, None, tdev.ptr, space.ptr, rows, k, classes, 0, k, 1, 1, 4, dtype), "forward")
    capi.check(capi.lib().rp_hip_linear_cross_entropy_backward(dx.ptr, None, None, x.ptr, h.ptr, None, tdev.ptr, stats.ptr, None, space.ptr, rows, k, classes, 0,
                                                               k, 1, 1, 4, k, 0, 1, 0, 0, 0, dtype), "backward")
    u = 2.0 ** -24
    z_off = ((k + 8) * u + 2.0 ** -22) * size
    lse = np.log(np.exp(z).sum(1))
    lse_off = z_off.max(1) + u * (300 + 4 * size.max(1)) + 2 * u * lse
    want = lse - z[np.arange(rows), targets]
    assert_within(loss.read()[0], want, lse_off + z_off.max(1) + 2 * u * np.abs(want), "loss")
    p = np.exp(z - lse[:, None])
    d = p.copy()
    d[np.arange(rows), targets] -= 1
    d_off = p * 1.1 * (z_off + lse_off[:, None] + 16 * u * (1 + np.abs(np.log(p)))) + 4 * u * np.abs(d) + 4 * u * p
    want, off = np.zeros((rows, k)), np.zeros((rows, k))
    for v in steps:
        piece = np.ascontiguousarray(view[v:v + 2000])
        want += d[:, v:v + 2000] @ piece
        off += (d_off[:, v:v + 2000] + ((classes + 8) * u + 2.0 ** -22) * (np.abs(d) + d_off)[:, v:v + 2000]) @ np.abs(piece)
    assert_within(dx.read(), want, rounded(off, want, dtype), "dx")


@pytest.mark.parametrize("dtype", ALL, ids=NAMES.get)
@pytest.mark.parametrize("rows,k,classes", [(24, 128, 1000), (300, 136, 1104), (9, 5, 33)])
def test_rows_without_a_target_may_hold_anything(rows, k, classes, dtype):
    """... where dw, which adds zeros times them, is not asked for: loss, dx and db are what they are with zeros there."""
    rng = np.random.default_rng(8)
    xv, w = rng.normal(size=(rows, k)), Operand(rng.normal(0, k ** -0.5, size=(k, classes)), dtype)
    targets = np.where(np.arange(rows) % 3, rng.integers(0, classes, rows), -1)
    space = room(capi.lib().rp_hip_linear_cross_entropy_workspace(rows, k, classes, 1, dtype))
    results = []
    for hole in (0.0, np.nan, np.inf):
        v = xv.copy()
        v[targets < 0] = hole
        x, tdev = Operand(v, dtype), ints(targets)
        loss, stats, dx, db = Output(1, 1, ACC[dtype]), Output(1, 2 * rows + 1, ACC[dtype]), Output(rows, k, dtype), Output(1, classes, dtype)
        capi.check(capi.lib().rp_hip_linear_cross_entropy_forward(loss.ptr, stats.ptr, x.ptr, w.ptr, None, tdev.ptr, space.ptr, rows, k, classes, 1, k, 1, classes, 1, dtype), "forward")
        capi.check(capi.lib().rp_hip_linear_cross_entropy_backward(dx.ptr, None, db.ptr, x.ptr, w.ptr, None, tdev.ptr, stats.ptr, None, space.ptr, rows, k, classes, 1,
                                                                   k, 1, classes, 1, k, 0, 1, 0, 0, 0, dtype), "backward")
        results.append([o.read() for o in (loss, dx, db)])
    assert np.all(results[0][1][targets < 0] == 0)
    for other in results[1:]:
        for a, b in zip(results[0], other):
            assert np.array_equal(a, b)
