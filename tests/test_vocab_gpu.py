"""The cross entropy of a large vocabulary from the rows before it, and its gradients, on the device against the formulas in 64 bits."""
import numpy as np
import pytest

from langhelp import *
from recpulse_amd import capi

pytestmark = pytest.mark.gpu

# (rows, k, classes): one of everything, fewer classes than a vector, sizes that end inside every tile, few rows, several tiles of each edge, several pieces
SIZES = [(1, 1, 1), (3, 5, 7), (1, 64, 1000), (16, 256, 1031), (130, 72, 520), (64, 520, 2050), (300, 64, 777), (257, 129, 1537), (520, 256, 2304)]


def problem(rows, k, classes, dtype, seed, tied=False, bias=True, without=4, lead=0, scale=1.5):
    rng = np.random.default_rng(seed)
    x = Operand(rng.normal(size=(rows, k)), dtype, rs=k + 8 * (seed % 2), lead=lead)
    w = rng.normal(0, scale * k ** -0.5, size=(k, classes))
    w = Operand(w, dtype, rs=1, cs=k, lead=lead) if tied else Operand(w, dtype, lead=lead)
    b = vector(rng.normal(size=classes), dtype) if bias else None
    targets = rng.integers(0, classes, rows)
    if without and rows > 1:
        targets[::without] = -1
        targets[1] = 0
        targets[-1] = classes - 1
    return rng, x, w, b, targets


def forward(x, w, b, targets, dtype, reduction, space=None):
    rows, k = x.shape
    classes = w.shape[1]
    loss, stats = Output(1, rows if reduction == 0 else 1, ACC[dtype]), Output(1, 2 * rows + 1, ACC[dtype])
    space = space or room(capi.lib().rp_hip_linear_cross_entropy_workspace(rows, k, classes, 0, dtype))
    capi.check(capi.lib().rp_hip_linear_cross_entropy_forward(loss.ptr, stats.ptr, x.ptr, w.ptr, at(b), ints(targets).ptr, space.ptr, rows, k, classes, reduction, x.rs, x.cs, w.rs, w.cs, dtype),
               "rp_hip_linear_cross_entropy_forward")
    return loss, stats


def offs(x, w, b, dtype):
    """What a sum of k products in any order can change in a row's logits, and in their log sum: a sum of at most 2^17 exponentials by teams adds fewer than 300 one after the other, and an
    argument of exp is rounded to 2^-24 of a value whose weight falls with it."""
    u = UNIT[dtype]
    size = np.abs(x.values) @ np.abs(w.values) + (0.0 if b is None else np.abs(b.values))
    z_off = (x.shape[1] + 8) * u * size + (2.0 ** -22 * size if dtype == F32 else 0.0)
    lse_off = z_off.max(1) + u * (300 + 4 * size.max(1))
    return z_off, lse_off


@pytest.mark.parametrize("dtype", ALL, ids=NAMES.get)
@pytest.mark.parametrize("tied", [False, True], ids=["rows", "transposed"])
@pytest.mark.parametrize("rows,k,classes", SIZES)
def test_forward(rows, k, classes, tied, dtype):
    _, x, w, b, targets = problem(rows, k, classes, dtype, rows + k + classes, tied, bias=classes % 2 == 1)
    z_off, lse_off = offs(x, w, b, dtype)
    off = z_off.max(1) + lse_off
    u = UNIT[dtype]
    for reduction in (0, 1, 2):
        want, lse, _, _, _ = vocab_reference(x.values, w.values, b and b.values, targets, reduction, 1.0)
        loss, stats = forward(x, w, b, targets, dtype, reduction)
        total = off if reduction == 0 else off.sum() / (max(1, (targets >= 0).sum()) if reduction == 1 else 1)
        assert_within(loss.read()[0], want, total + 2 * u * np.abs(want), "loss")
        got = stats.read()[0]
        assert_within(got[:rows], lse, lse_off + 2 * u * np.abs(lse), "log sums")
        assert got[-1] == (targets >= 0).sum()


@pytest.mark.parametrize("dtype", ALL, ids=NAMES.get)
@pytest.mark.parametrize("tied", [False, True], ids=["rows", "transposed"])
@pytest.mark.parametrize("rows,k,classes", SIZES)
def test_backward(rows, k, classes, tied, dtype):
    check_backward(rows, k, classes, tied, dtype, reduction=(rows + k) % 3, bias=classes % 2 == 1)


def check_backward(rows, k, classes, tied, dtype, reduction, bias=True, without=4, lead=0, upstream=None):
    rng, x, w, b, targets = problem(rows, k, classes, dtype, rows * 3 + k + classes, tied, bias, without, lead)
    up = rng.uniform(0.5, 2.0, rows if reduction == 0 else 1) if upstream is None else upstream
    space = room(capi.lib().rp_hip_linear_cross_entropy_workspace(rows, k, classes, 1, dtype))
    _, stats = forward(x, w, b, targets, dtype, reduction, space)
    up = vector(up, ACC[dtype])
    _, _, d, f, p = vocab_reference(x.values, w.values, b and b.values, targets, reduction, up.values[0])
    z_off, lse_off = offs(x, w, b, dtype)
    u, half = UNIT[dtype], HALF[dtype]
    accumulate = rows % 2
    start = [rng.normal(size=s) * np.abs(f).max() if accumulate else None for s in ((rows, k), (k, classes), (1, classes))]
    dx, db = Output(rows, k, dtype, k + 4, start=start[0]), Output(1, classes, dtype, start=start[2])
    dw = Output(k, classes, dtype, 1, k + 2, start=start[1]) if tied else Output(k, classes, dtype, classes + 2, start=start[1])
    capi.check(capi.lib().rp_hip_linear_cross_entropy_backward(dx.ptr, dw.ptr, db.ptr, x.ptr, w.ptr, at(b), ints(targets).ptr, stats.ptr, up.ptr, space.ptr, rows, k, classes, reduction,
                                                               x.rs, x.cs, w.rs, w.cs, dx.rs, dw.rs, dw.cs, accumulate, accumulate, accumulate, dtype), "rp_hip_linear_cross_entropy_backward")
    # d: what the logits' and the log sum's errors change in p, its last places, and one rounding to the tensors' type (for 16 bits; subnormal results are 2^-24 of a row's largest)
    held = (np.abs(f) > 0)[:, None]
    d_off = np.where(held, np.abs(f)[:, None] * (p * 1.1 * (z_off + lse_off[:, None] + 16 * u * (1 + np.abs(np.log(np.maximum(p, 1e-300))))) + 4 * u * np.abs(p)), 0.0)
    d_off = d_off + 4 * u * np.abs(d)
    if half > u:
        d_off = d_off + half * (np.abs(d) + d_off) + np.abs(f).max() * 2.0 ** -38
    wide = np.abs(d) + d_off
    steps = 2.0 ** -22 if dtype == F32 else 0.0
    pieces = 1 + rows * classes * 8 / (64 << 20)                # (float32 and float64 add the pieces' products one after the other)
    for out, want, off, what in ((dx, d @ w.values.T, d_off @ np.abs(w.values).T + ((classes + 8 + pieces) * u + steps) * (wide @ np.abs(w.values).T), "dx"),
                                 (dw, x.values.T @ d, np.abs(x.values).T @ d_off + ((rows + 8) * u + steps) * (np.abs(x.values).T @ wide), "dw"),
                                 (db, d.sum(0)[None], (d_off + (rows + 8) * u * wide).sum(0)[None], "db")):
        bound = rounded(off, want, dtype)
        if accumulate:
            want = want + out.values
            bound = bound + half * (np.abs(want) + np.abs(out.values) + bound) + TINY[dtype]
        assert_within(out.read(), want, bound, what)


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=NAMES.get)
def test_several_pieces_of_the_vocabulary(dtype):
    check_backward(3000, 16, 50000 if dtype == F32 else 60008, dtype == F16, dtype, reduction=1, bias=True)


@pytest.mark.parametrize("dtype", [BF16, F16], ids=NAMES.get)
@pytest.mark.parametrize("rows,k,classes,tied", [(4096, 2048, 4096, False), (4000, 2056, 4104, True), (4001, 2056, 4104, False)])
def test_the_largest_tiles(rows, k, classes, tied, dtype):
    check_backward(rows, k, classes, tied, dtype, reduction=1, bias=tied)


@pytest.mark.parametrize("dtype,tied", [(BF16, False), (F16, True)], ids=["bf16", "f16"])
def test_several_pieces_on_the_largest_tiles(dtype, tied):
    """... checked at some rows of dx and some classes of dW, whose logits are few."""
    rows, k, classes = 8192, 1024, 20008
    rng, x, w, _, targets = problem(rows, k, classes, dtype, 12, tied, bias=False, without=8)
    space = room(capi.lib().rp_hip_linear_cross_entropy_workspace(rows, k, classes, 1, dtype))
    _, stats = forward(x, w, None, targets, dtype, 1, space)
    dx, dw = Output(rows, k, dtype), Output(k, classes, dtype, 1, k) if tied else Output(k, classes, dtype)
    capi.check(capi.lib().rp_hip_linear_cross_entropy_backward(dx.ptr, dw.ptr, None, x.ptr, w.ptr, None, ints(targets).ptr, stats.ptr, None, space.ptr, rows, k, classes, 1,
                                                               x.rs, x.cs, w.rs, w.cs, dx.rs, dw.rs, dw.cs, 0, 0, 0, dtype), "rp_hip_linear_cross_entropy_backward")
    held = targets >= 0
    f = np.where(held, 1.0 / held.sum(), 0.0)
    # z is off by at most (k + 8) 2^-24 of the sum of |x w|, below 1e-3 here; lse, from the device, by as much and a little; d by that and its rounding
    rel = (k + 8) * 2.0 ** -24 * 2.2 * np.sqrt(2 / np.pi) ** 2 * 1.5 * np.sqrt(k) + 1e-4 + HALF[dtype]
    lse = stats.read()[0, :rows]
    some = rng.choice(rows, 48, replace=False)
    z = x.values[some] @ w.values
    assert np.abs(np.log(np.exp(z).sum(1)) - lse[some]).max() < 1e-3
    d = np.exp(z - lse[some, None])
    d[np.arange(48)[held[some]], targets[some][held[some]]] -= 1
    d *= f[some, None]
    d_off = rel * np.abs(d) + 2 * rel * np.abs(f[some, None]) * np.exp(z - lse[some, None]) + f.max() * 2.0 ** -38
    want = d @ w.values.T
    assert_within(dx.read()[some], want, rounded(d_off @ np.abs(w.values).T + classes * 2.0 ** -24 * (np.abs(d) @ np.abs(w.values).T), want, dtype), "dx")
    some = rng.choice(classes, 48, replace=False)
    z = x.values @ w.values[:, some]
    p = np.exp(z - lse[:, None])
    d = (p - (targets[:, None] == some)) * f[:, None]
    d_off = rel * np.abs(d) + 2 * rel * np.abs(f[:, None]) * p + f.max() * 2.0 ** -38
    want = x.values.T @ d
    assert_within(dw.read()[:, some], want, rounded(np.abs(x.values).T @ d_off + rows * 2.0 ** -24 * (np.abs(x.values).T @ np.abs(d)), want, dtype), "dw")


@pytest.mark.parametrize("dtype", [BF16, F16], ids=NAMES.get)
def test_rows_that_start_at_any_element(dtype):
    for tied in (False, True):
        check_backward(70, 136, 520, tied, dtype, reduction=1, lead=3)


@pytest.mark.parametrize("dtype", ALL, ids=NAMES.get)
def test_operands_of_any_stride(dtype):
    rng = np.random.default_rng(9)
    rows, k, classes = 21, 19, 45
    x, w = Operand(rng.normal(size=(rows, k)), dtype, rs=2 * k + 3, cs=2, lead=3), Operand(rng.normal(0, k ** -0.5, size=(k, classes)), dtype, rs=3 * classes, cs=3, lead=1)
    targets = rng.integers(0, classes, rows)
    want = vocab_reference(x.values, w.values, None, targets, 0, 1.0)[0]
    loss, _ = forward(x, w, None, targets, dtype, 0)
    z_off, lse_off = offs(x, w, None, dtype)
    assert_within(loss.read()[0], want, z_off.max(1) + lse_off + 2 * UNIT[dtype] * np.abs(want), "loss")


@pytest.mark.parametrize("dtype", [F16, BF16, F32], ids=NAMES.get)
def test_small_and_uneven_upstream_gradients_keep_their_digits(dtype):
    """Rows weighted from 2^-20 to 1, and a mean over thousands: in float16 the gradient of a rare class would be zero if it were stored as it is."""
    rows = 96
    check_backward(rows, 64, 2000, False, dtype, reduction=0, bias=False, without=0, upstream=2.0 ** -np.arange(0.0, 12.0, 12.0 / rows))
    check_backward(rows, 64, 2000, False, dtype, reduction=2, bias=True, without=3, upstream=np.array([2.0 ** -6]))


@pytest.mark.parametrize("dtype", [BF16, F16], ids=NAMES.get)
@pytest.mark.parametrize("rows", [37, 300])
def test_a_mean_does_not_round_all_rows_alike(rows, dtype):
    """With logits of zero over 128 classes p = 2^-7 and p - 1 are exact in 16 bits; 1.3 / rows is not, and must not be part of what is rounded."""
    rng = np.random.default_rng(13)
    k, classes = 64, 128
    x, w = Operand(rng.normal(size=(rows, k)), dtype), Operand(np.zeros((k, classes)), dtype)
    targets, up = rng.integers(0, classes, rows), vector([1.3], F32)
    space = room(capi.lib().rp_hip_linear_cross_entropy_workspace(rows, k, classes, 1, dtype))
    _, stats = forward(x, w, None, targets, dtype, 1, space)
    dw = Output(k, classes, dtype)
    capi.check(capi.lib().rp_hip_linear_cross_entropy_backward(None, dw.ptr, None, x.ptr, w.ptr, None, ints(targets).ptr, stats.ptr, up.ptr, space.ptr, rows, k, classes, 1,
                                                               k, 1, classes, 1, k, classes, 1, 0, 0, 0, dtype), "backward")
    d = (np.full((rows, classes), 2.0 ** -7) - (targets[:, None] == np.arange(classes))) * up.values[0, 0] / rows
    # log 128 in float32 and exp of it: 2^-7 to 2^-20 of itself, which 16 bits round back
    off = (rows + 16) * 2.0 ** -24 * (np.abs(x.values).T @ np.abs(d))
    assert_within(dw.read(), x.values.T @ d, rounded(off, x.values.T @ d, dtype), "dw")


@pytest.mark.parametrize("dtype", ALL, ids=NAMES.get)
@pytest.mark.parametrize("rows,k,classes", [(9, 40, 300), (150, 128, 1100)])
def test_without_any_target_everything_is_zero(rows, k, classes, dtype):
    _, x, w, b, targets = problem(rows, k, classes, dtype, 1)
    targets[:] = np.where(np.arange(rows) % 2, -1, classes)      # (behind the last class is outside as well)
    for reduction in (0, 1, 2):
        space = room(capi.lib().rp_hip_linear_cross_entropy_workspace(rows, k, classes, 1, dtype))
        loss, stats = forward(x, w, b, targets, dtype, reduction, space)
        assert np.all(loss.read() == 0)
        dx, dw, db = Output(rows, k, dtype), Output(k, classes, dtype), Output(1, classes, dtype)
        capi.check(capi.lib().rp_hip_linear_cross_entropy_backward(dx.ptr, dw.ptr, db.ptr, x.ptr, w.ptr, b.ptr, ints(targets).ptr, stats.ptr, None, space.ptr, rows, k, classes, reduction,
                                                                   x.rs, 1, classes, 1, k, classes, 1, 0, 0, 0, dtype), "backward")
        assert all(np.all(o.read() == 0) for o in (dx, dw, db))


@pytest.mark.parametrize("dtype", ALL, ids=NAMES.get)
@pytest.mark.parametrize("classes", [60, 1000])
def test_classes_that_a_bias_of_minus_infinity_takes_out(classes, dtype):
    """... have no share in the sum, and none of the gradient; a vocabulary padded to whole tiles is masked like this, whole tiles of it too."""
    rng, x, w, _, _ = problem(40, 64, classes, dtype, 2, bias=False)
    bias = rng.normal(size=classes)
    bias[classes // 3:] = -np.inf
    b = vector(bias, dtype)
    targets = rng.integers(0, classes // 3, 40)
    with np.errstate(all="ignore"):
        want, _, d, _, _ = vocab_reference(x.values, w.values[:, :classes // 3], b.values[:, :classes // 3], targets, 1, 1.0)
    space = room(capi.lib().rp_hip_linear_cross_entropy_workspace(40, 64, classes, 1, dtype))
    loss, stats = forward(x, w, b, targets, dtype, 1, space)
    assert abs(loss.read()[0, 0] - want[0]) < {F64: 1e-10}.get(dtype, 2e-5)          # (a sum of 64 products of size 4: 64 * 4 * 2^-24)
    dw = Output(64, classes, dtype)
    capi.check(capi.lib().rp_hip_linear_cross_entropy_backward(None, dw.ptr, None, x.ptr, w.ptr, b.ptr, ints(targets).ptr, stats.ptr, None, space.ptr, 40, 64, classes, 1,
                                                               x.rs, 1, classes, 1, 64, classes, 1, 0, 0, 0, dtype), "backward")
    got = dw.read()
    assert np.all(got[:, classes // 3:] == 0)
    # every d is off by its rounding and by 1e-5 of itself, the sum by one rounding more
    bound = (np.abs(x.values).T @ np.abs(d)) * (HALF[dtype] + (1e-10 if dtype == F64 else 3e-5)) + 1e-7 * (dtype != F64)
    assert_within(got[:, :classes // 3], x.values.T @ d, rounded(bound, x.values.T @ d, dtype), "dw")


def test_large_logits_do_not_run_over():
    """Logits of several thousand: exp of any of them alone would be infinite."""
    for dtype in ALL:
        rng = np.random.default_rng(1)
        rows, k, classes = 20, 32, 400
        x, w = Operand(rng.normal(size=(rows, k)) * 40, dtype), Operand(rng.normal(size=(k, classes)) * 10, dtype)
        targets = rng.integers(0, classes, rows)
        want = vocab_reference(x.values, w.values, None, targets, 0, 1.0)[0]
        z_off, lse_off = offs(x, w, None, dtype)
        loss, _ = forward(x, w, None, targets, dtype, 0)
        assert_within(loss.read()[0], want, z_off.max(1) + lse_off + 2 * UNIT[dtype] * np.abs(want), "loss")


@pytest.mark.parametrize("asked", [0, 1, 2])
@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=NAMES.get)
def test_an_output_does_not_depend_on_the_others(asked, dtype):
    rows, k, classes = 140, 136, 1000
    _, x, w, b, targets = problem(rows, k, classes, dtype, 4)
    space = room(capi.lib().rp_hip_linear_cross_entropy_workspace(rows, k, classes, 1, dtype))
    _, stats = forward(x, w, b, targets, dtype, 1, space)
    results = []
    for names in ((0, 1, 2), (asked,)):
        outs = [Output(rows, k, dtype), Output(k, classes, dtype), Output(1, classes, dtype)]
        p = [o.ptr if i in names else None for i, o in enumerate(outs)]
        capi.check(capi.lib().rp_hip_linear_cross_entropy_backward(*p, x.ptr, w.ptr, b.ptr, ints(targets).ptr, stats.ptr, None, space.ptr, rows, k, classes, 1,
                                                                   x.rs, 1, classes, 1, k, classes, 1, 0, 0, 0, dtype), "backward")
        results.append(outs[asked].bits())
    assert np.array_equal(*results)


def test_gradient_agrees_with_differences():
    rng = np.random.default_rng(8)
    rows, k, classes, step = 5, 6, 11, 1e-5
    x, w, targets = rng.normal(size=(rows, k)), rng.normal(size=(k, classes)), np.array([3, -1, 10, 0, 3])

    def value(xv, wv):
        return forward(Operand(xv, F64), Operand(wv, F64), None, targets, F64, 1)[0].read()[0, 0]

    xo, wo = Operand(x, F64), Operand(w, F64)
    space = room(capi.lib().rp_hip_linear_cross_entropy_workspace(rows, k, classes, 1, F64))
    _, stats = forward(xo, wo, None, targets, F64, 1, space)
    dx, dw = Output(rows, k, F64), Output(k, classes, F64)
    capi.check(capi.lib().rp_hip_linear_cross_entropy_backward(dx.ptr, dw.ptr, None, xo.ptr, wo.ptr, None, ints(targets).ptr, stats.ptr, None, space.ptr, rows, k, classes, 1,
                                                               k, 1, classes, 1, k, classes, 1, 0, 0, 0, F64), "backward")
    for i, j in ((0, 0), (1, 2), (4, 5)):
        e = np.zeros((rows, k))
        e[i, j] = step
        assert abs((value(x + e, w) - value(x - e, w)) / (2 * step) - dx.read()[i, j]) < 1e-7
    for i, j in ((0, 0), (5, 10), (2, 3)):
        e = np.zeros((k, classes))
        e[i, j] = step
        assert abs((value(x, w + e) - value(x, w - e)) / (2 * step) - dw.read()[i, j]) < 1e-7


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=NAMES.get)
@pytest.mark.parametrize("rows,k,classes", [(24, 128, 1000), (300, 136, 1104)])
def test_recorded_calls_replay_to_the_eager_result(rows, k, classes, dtype):
    _, x, w, b, targets = problem(rows, k, classes, dtype, 6)
    tdev = ints(targets)
    loss, stats = Output(1, 1, F32), Output(1, 2 * rows + 1, F32)
    dx, dw, db = Output(rows, k, dtype), Output(k, classes, dtype), Output(1, classes, dtype)
    space = room(capi.lib().rp_hip_linear_cross_entropy_workspace(rows, k, classes, 1, dtype))
    outs = (loss, stats, dx, dw, db)

    def step():
        capi.check(capi.lib().rp_hip_linear_cross_entropy_forward(loss.ptr, stats.ptr, x.ptr, w.ptr, b.ptr, tdev.ptr, space.ptr, rows, k, classes, 1, x.rs, 1, classes, 1, dtype), "forward")
        capi.check(capi.lib().rp_hip_linear_cross_entropy_backward(dx.ptr, dw.ptr, db.ptr, x.ptr, w.ptr, b.ptr, tdev.ptr, stats.ptr, None, space.ptr, rows, k, classes, 1,
                                                                   x.rs, 1, classes, 1, k, classes, 1, 0, 0, 0, dtype), "backward")

    with capi.Stream() as s:
        step()
        eager = [o.bits() for o in outs]
        with capi.Graph.capture() as graph:
            step()
        for _ in range(3):
            for o in outs:
                capi.check(capi.lib().rp_hip_memset(o.buf.ptr, 0, o.buf.nbytes), "memset")
            capi.check(capi.lib().rp_hip_memset(space.ptr, 255, space.nbytes), "memset")
            capi.synchronize()
            graph.launch()
            capi.check(capi.lib().rp_hip_stream_synchronize(), "sync")
            assert all(np.array_equal(a, o.bits()) for a, o in zip(eager, outs))


@pytest.mark.parametrize("dtype", ALL, ids=NAMES.get)
@pytest.mark.parametrize("rows,k,classes", [(24, 128, 1000), (300, 136, 1104)])
@pytest.mark.parametrize("upstream", [0.0, np.inf, np.nan, -2.0 ** -100])
def test_upstream_gradients_that_are_not_ordinary_numbers(upstream, rows, k, classes, dtype):
    """Rows without a target stay zeros; with a gradient of zero, or one too small for any product of it, all are."""
    _, x, w, _, targets = problem(rows, k, classes, dtype, 15, bias=False)
    for reduction in (0, 1, 2):
        space = room(capi.lib().rp_hip_linear_cross_entropy_workspace(rows, k, classes, 1, dtype))
        _, stats = forward(x, w, None, targets, dtype, reduction, space)
        up = vector(np.full(rows if reduction == 0 else 1, upstream), ACC[dtype])
        dx, db = Output(rows, k, dtype), Output(1, classes, dtype)
        capi.check(capi.lib().rp_hip_linear_cross_entropy_backward(dx.ptr, None, db.ptr, x.ptr, w.ptr, None, ints(targets).ptr, stats.ptr, up.ptr, space.ptr, rows, k, classes, reduction,
                                                                   x.rs, 1, classes, 1, k, 0, 1, 0, 0, 0, dtype), "backward")
        got = dx.read()
        assert np.all(got[targets < 0] == 0)
        if np.isfinite(upstream):
            assert np.all(np.abs(got) <= abs(upstream) * 64)             # (|d| adds up to less than two, |w| is below 32)
            assert np.all(np.abs(db.read()) <= abs(upstream) * rows)
        else:
            assert not np.any(np.isfinite(got[targets >= 0])) and not np.any(np.isfinite(db.read()))


@pytest.mark.parametrize("tied", [False, True], ids=["rows", "transposed"])
@pytest.mark.parametrize("accumulate", [0, 1])
@pytest.mark.parametrize("rows,k,classes", [(300, 200, 9001), (130, 520, 4160), (128, 128, 2048)])
def test_dense_gradients_of_few_tiles_in_float32(rows, k, classes, accumulate, tied):
    """The classes in shares, with some left over; the shares' sums are added up in float32."""
    rng, x, w, _, targets = problem(rows, k, classes, F32, 21, tied, bias=False)
    space = room(capi.lib().rp_hip_linear_cross_entropy_workspace(rows, k, classes, 1, F32))
    _, stats = forward(x, w, None, targets, F32, 1, space)
    _, _, d, f, p = vocab_reference(x.values, w.values, None, targets, 1, 1.0)
    z_off, lse_off = offs(x, w, None, F32)
    start = rng.normal(size=(rows, k)) * np.abs(f).max() if accumulate else None
    dx = Output(rows, k, F32, start=start)
    capi.check(capi.lib().rp_hip_linear_cross_entropy_backward(dx.ptr, None, None, x.ptr, w.ptr, None, ints(targets).ptr, stats.ptr, None, space.ptr, rows, k, classes, 1,
                                                               x.rs, 1, w.rs, w.cs, k, 0, 1, accumulate, 0, 0, F32), "backward")
    u = UNIT[F32]
    d_off = np.abs(f)[:, None] * (p * 1.1 * (z_off + lse_off[:, None] + 16 * u * (1 + np.abs(np.log(p)))) + 4 * u * p) + 4 * u * np.abs(d)
    wide, want = np.abs(d) + d_off, d @ w.values.T
    off = d_off @ np.abs(w.values).T + ((classes + 8) * u + 2.0 ** -22) * (wide @ np.abs(w.values).T)      # (in any order; 2^-22 where the products are split into halves)
    bound = rounded(off, want, F32)
    if accumulate:
        want = want + dx.values
        bound = bound + HALF[F32] * (np.abs(want) + np.abs(dx.values) + bound)
    assert_within(dx.read(), want, bound, "dx")
