"""The loss of a large vocabulary for 16-bit operands of any stride, whose W is widened to float32 a piece at a time: gradients over several pieces against the formulas in 64 bits."""
import numpy as np
import pytest

import test_vocab_gpu as vocab
from langhelp import *
from recpulse_amd import capi

pytestmark = pytest.mark.gpu
HALF_TYPES = [BF16, F16]


def gradients(x, w, b, targets, up, reduction, dtype, accumulate, dx, dw, db):
    (rows, k), classes = x.shape, w.shape[1]
    space = room(capi.lib().rp_hip_linear_cross_entropy_workspace_strided(rows, k, classes, 1, x.rs, x.cs, w.rs, w.cs, dtype))
    _, stats = vocab.forward(x, w, b, targets, dtype, reduction, space)
    capi.check(capi.lib().rp_hip_linear_cross_entropy_backward(dx.ptr, dw.ptr, at(db), x.ptr, w.ptr, at(b), ints(targets).ptr, stats.ptr, up.ptr, space.ptr, rows, k, classes, reduction,
                                                               x.rs, x.cs, w.rs, w.cs, dx.rs, dw.rs, dw.cs, accumulate, accumulate, accumulate, dtype), "rp_hip_linear_cross_entropy_backward")
    return stats


@pytest.mark.parametrize("dtype", HALF_TYPES, ids=NAMES.get)
@pytest.mark.parametrize("rows,k,classes,tied", [(7, 5, 70000, False), (8, 7, 66000, True), (3001, 5, 8000, False), (3000, 3, 6000, True)])
def test_rows_too_short_for_the_tiles(rows, k, classes, tied, dtype):
    """... of few rows in pieces of 65536 classes, and of many in pieces whose logits take 64 MiB; dx with gaps, everything added to what is there where the rows are odd."""
    vocab.check_backward(rows, k, classes, tied, dtype, reduction=1, bias=True)


@pytest.mark.parametrize("dtype", ALL, ids=NAMES.get)
@pytest.mark.parametrize("accumulate", [0, 1])
@pytest.mark.parametrize("rows,k,classes,reduction", [(21, 19, 45, 0), (70, 136, 520, 1), (257, 33, 1031, 2)])
def test_operands_of_any_stride(rows, k, classes, reduction, accumulate, dtype):
    rng = np.random.default_rng(rows + accumulate)
    x, w = Operand(rng.normal(size=(rows, k)), dtype, rs=2 * k + 3, cs=2, lead=3), Operand(rng.normal(0, k ** -0.5, size=(k, classes)), dtype, rs=3 * classes, cs=3, lead=1)
    b, targets = vector(rng.normal(size=classes), dtype), rng.integers(-1, classes, rows)
    up = vector(rng.uniform(0.5, 2.0, rows if reduction == 0 else 1), ACC[dtype])
    start = [rng.normal(size=s) if accumulate else None for s in ((rows, k), (k, classes), (1, classes))]
    dx, dw, db = Output(rows, k, dtype, k + 4, start=start[0]), Output(k, classes, dtype, classes + 2, start=start[1]), Output(1, classes, dtype, start=start[2])
    gradients(x, w, b, targets, up, reduction, dtype, accumulate, dx, dw, db)
    _, _, d, f, p = vocab.vocab_reference(x.values, w.values, b.values, targets, reduction, up.values[0])
    z_off, lse_off = vocab.offs(x, w, b, dtype)
    u = UNIT[dtype]
    # d stays in the accumulate type: the errors of z and of the log sum, and its own last places
    d_off = np.abs(f)[:, None] * (p * 1.1 * (z_off + lse_off[:, None] + 16 * u * (1 + np.abs(np.log(p)))) + 4 * u * p) + 4 * u * np.abs(d)
    wide, split = np.abs(d) + d_off, 0.0 if dtype == F64 else 2.0 ** -22      # (products of float32 as six of bfloat16)
    for out, want, off, what in ((dx, d @ w.values.T, d_off @ np.abs(w.values).T + ((classes + 8) * u + split) * (wide @ np.abs(w.values).T), "dx"),
                                 (dw, x.values.T @ d, np.abs(x.values).T @ d_off + ((rows + 8) * u + split) * (np.abs(x.values).T @ wide), "dw"),
                                 (db, d.sum(0)[None], (d_off + (rows + 8) * u * wide).sum(0)[None], "db")):
        if accumulate:                                          # (16-bit sums are added before they are rounded, the others are sums themselves)
            want = want + out.values
            off = off + 2 * u * (np.abs(want) + np.abs(out.values))
        assert_within(out.read(), want, rounded(off, want, dtype), what)


@pytest.mark.parametrize("dtype", HALF_TYPES, ids=NAMES.get)
def test_pieces_that_end_because_of_the_width(dtype):
    """Rows of 36864 columns, of whose W a piece is 768 classes.  Values are small whole numbers, W's over 64: every logit is exact in float32 whatever the order of its sum."""
    rng = np.random.default_rng(5)
    rows, k, classes = 3, 36864, 1100
    x = Operand(rng.integers(-2, 3, (rows, k)), dtype, rs=2 * k, cs=2)
    w = Operand(rng.integers(-1, 2, (k, classes)) / 64.0, dtype)
    targets, up = np.array([0, 800, 1099]), vector([1.0], F32)
    dx, dw, db = Output(rows, k, dtype, k + 8), Output(k, classes, dtype), Output(1, classes, dtype)
    stats = gradients(x, w, None, targets, up, 2, dtype, 0, dx, dw, db)
    _, lse, d, _, p = vocab.vocab_reference(x.values, w.values, None, targets, 2, 1.0)
    # (sums of 1100 exponentials by 1024 threads; arguments below 32)
    lse_off = 2.0 ** -24 * (64 + 4 * 32)
    assert np.abs(stats.read()[0, :rows] - lse).max() <= lse_off
    # z - lse is rounded to 2^-20, that times log2 e as the exponential's argument by 46 * 2^-24 * log 2
    d_off = p * 1.1 * (lse_off + 2.0 ** -18) + 4 * 2.0 ** -24 * np.abs(d)
    wide = np.abs(d) + d_off
    assert_within(dx.read(), d @ w.values.T, rounded((d_off + (classes * 2.0 ** -24 + 2.0 ** -22) * wide) @ np.abs(w.values).T, d @ w.values.T, dtype), "dx")
    assert_within(dw.read(), x.values.T @ d, rounded(np.abs(x.values).T @ (d_off + 2.0 ** -21 * wide), x.values.T @ d, dtype), "dw")
    assert_within(db.read(), d.sum(0)[None], rounded((d_off + 2.0 ** -21 * wide).sum(0)[None], d.sum(0)[None], dtype), "db")
