"""The gated linear layer and its gradients on the device against the formulas in 64 bits."""
import numpy as np
import pytest

from langhelp import *
from recpulse_amd import capi

pytestmark = pytest.mark.gpu

# decoding and a few rows, sizes that end inside every tile, widths below a vector, one of everything, several tiles of each edge
SIZES = [(1, 1, 1), (1, 64, 8), (3, 7, 5), (16, 256, 520), (33, 129, 67), (64, 512, 128), (70, 72, 264), (130, 64, 130), (300, 200, 1031), (257, 320, 512), (5, 4096, 1024), (520, 96, 768)]


def layer(rows, k, n, dtype, bias, seed, tied=False, lead=0):
    """x, W (row-major, or the transposed view of [2 n, k]) and bias."""
    rng = np.random.default_rng(seed)
    x = Operand(rng.normal(size=(rows, k)), dtype, rs=k + 8 * (seed % 2), lead=lead)
    w = rng.normal(0, k ** -0.5, size=(k, 2 * n))
    w = Operand(w, dtype, rs=1, cs=k) if tied else Operand(w, dtype, lead=lead)
    return rng, x, w, vector(0.3 * rng.normal(size=2 * n), dtype) if bias else None


def forward(x, w, bias, n, gate, dtype, keep=True, h_rs=None):
    rows, k = x.shape
    h, z = Output(rows, n, dtype, h_rs), Output(rows, 2 * n, ACC[dtype]) if keep else None
    capi.check(capi.lib().rp_hip_gated_linear_forward(h.ptr, at(z), x.ptr, w.ptr, at(bias), rows, k, n, GATES[gate], x.rs, x.cs, w.rs, w.cs, h.rs, dtype), "rp_hip_gated_linear_forward")
    return h, z


def reference(x, w, bias, n, gate, dtype):
    """z, h and what a sum of k products in any order, and the functions' own last places, can change in them."""
    k, u = x.shape[1], UNIT[dtype]
    b = 0.0 if bias is None else bias.values
    z = x.values @ w.values + b
    z_off = (k + 8) * u * (np.abs(x.values) @ np.abs(w.values) + np.abs(b))
    if dtype == F32:
        z_off = z_off + 2.0 ** -22 * (np.abs(x.values) @ np.abs(w.values))      # (products of float32 as six of bfloat16: what is left out is below 2^-24 of each)
    act, slope = gate_reference(z[:, :n], gate)
    g, up = z[:, :n], z[:, n:]
    # the slopes are below 1.2 and change by less than 1.2 a unit of g; exp of an argument rounded to u |g|
    act_off = 1.2 * z_off[:, :n] + 16 * u * (1 + np.abs(g)) * (np.abs(act) + u)
    h_off = act_off * (np.abs(up) + z_off[:, n:]) + np.abs(act) * z_off[:, n:] + 2 * u * np.abs(act * up)
    return z, z_off, act, act_off, slope, 1.2 * z_off[:, :n] + 16 * u * (1 + np.abs(g)), act * up, h_off


@pytest.mark.parametrize("dtype", ALL, ids=NAMES.get)
@pytest.mark.parametrize("tied", [False, True], ids=["rows", "transposed"])
@pytest.mark.parametrize("rows,k,n", SIZES)
def test_forward(rows, k, n, tied, dtype):
    gate = sorted(GATES)[(rows + k + n) % 5]
    _, x, w, bias = layer(rows, k, n, dtype, n % 2, rows + 3 * k + n, tied)
    z, z_off, _, _, _, _, want, off = reference(x, w, bias, n, gate, dtype)
    h, kept = forward(x, w, bias, n, gate, dtype, True, n + 3)
    assert_within(h.read(), want, rounded(off, want, dtype), "h")
    assert_within(kept.read(), z, rounded(z_off, z, ACC[dtype]), "z")
    again, _ = forward(x, w, bias, n, gate, dtype, False)
    assert_within(again.read(), want, rounded(off, want, dtype), "h where z is not kept")


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=NAMES.get)
@pytest.mark.parametrize("gate", sorted(GATES))
def test_gates(gate, dtype):
    _, x, w, bias = layer(48, 96, 200, dtype, True, 5)
    want, off = reference(x, w, bias, 200, gate, dtype)[6:]
    h, _ = forward(x, w, bias, 200, gate, dtype)
    assert_within(h.read(), want, rounded(off, want, dtype), "h")


@pytest.mark.parametrize("dtype", ALL, ids=NAMES.get)
def test_operands_of_any_stride(dtype):
    rng = np.random.default_rng(9)
    rows, k, n = 37, 45, 29
    x, w = Operand(rng.normal(size=(rows, k)), dtype, rs=2 * k + 3, cs=2, lead=3), Operand(rng.normal(0, k ** -0.5, size=(k, 2 * n)), dtype, rs=6 * n, cs=3, lead=1)
    want, off = reference(x, w, None, n, "silu", dtype)[6:]
    h, _ = forward(x, w, None, n, "silu", dtype)
    assert_within(h.read(), want, rounded(off, want, dtype), "h")


@pytest.mark.parametrize("dtype", [BF16, F16], ids=NAMES.get)
@pytest.mark.parametrize("tied", [False, True], ids=["rows", "transposed"])
@pytest.mark.parametrize("rows,k,n", [(2048, 320, 2048), (2000, 328, 2056), (1999, 321, 2051)])
def test_the_largest_tiles(rows, k, n, tied, dtype):
    _, x, w, bias = layer(rows, k, n, dtype, n % 2 == 0, rows, tied)
    z, z_off, _, _, _, _, want, off = reference(x, w, bias, n, "silu", dtype)
    h, kept = forward(x, w, bias, n, "silu", dtype, True, n + 8 * (rows % 2))
    assert_within(h.read(), want, rounded(off, want, dtype), "h")
    assert_within(kept.read(), z, rounded(z_off, z, ACC[dtype]), "z")


def test_rows_that_start_at_any_element():
    for rows, k, n in ((40, 128, 96), (150, 200, 264), (9, 520, 72)):
        _, x, w, bias = layer(rows, k, n, BF16, True, 1, lead=3)
        want, off = reference(x, w, bias, n, "gelu", BF16)[6:]
        h, _ = forward(x, w, bias, n, "gelu", BF16)
        assert_within(h.read(), want, rounded(off, want, BF16), "h")


def test_a_broadcast_row():
    """x with a row stride of 0: every row of h is the same."""
    rng = np.random.default_rng(2)
    x, w = Operand(rng.normal(size=(1, 64)), F16), Operand(rng.normal(0, 0.1, size=(64, 48)), F16)
    h = Output(5, 24, F16)
    capi.check(capi.lib().rp_hip_gated_linear_forward(h.ptr, None, x.ptr, w.ptr, None, 5, 64, 24, 0, 0, 1, 48, 1, 24, F16), "forward")
    got = h.bits()
    assert all(np.array_equal(got[0], row) for row in got)


@pytest.mark.parametrize("dtype", ALL, ids=NAMES.get)
@pytest.mark.parametrize("tied", [False, True], ids=["rows", "transposed"])
@pytest.mark.parametrize("rows,k,n", SIZES)
def test_backward(rows, k, n, tied, dtype):
    gate = sorted(GATES)[(rows + 2 * k + n) % 5]
    rng, x, w, _ = layer(rows, k, n, dtype, False, rows + 5 * k + n, tied)
    u, half = UNIT[dtype], HALF[dtype]
    z0 = x.values @ w.values
    z = Operand(z0, ACC[dtype])
    act, slope = gate_reference(z.values[:, :n], gate)
    dh = Operand(rng.normal(size=(rows, n)), dtype, rs=n + 1)
    dz = np.concatenate([dh.values * z.values[:, n:] * slope, dh.values * act], 1)
    # dz: the functions' last places, then one rounding
    dz_off = 24 * u * np.concatenate([np.abs(dh.values * z.values[:, n:]), np.abs(dh.values)], 1) * np.tile(1 + np.abs(z.values[:, :n]), 2)
    dz_off = rounded(dz_off, dz, dtype)
    wide = np.abs(dz) + dz_off
    accumulate = rows % 2
    start = [rng.normal(size=s) if accumulate else None for s in ((rows, k), (k, 2 * n), (1, 2 * n))]
    dx, db = Output(rows, k, dtype, k + 4, start=start[0]), Output(1, 2 * n, dtype, start=start[2])
    dw = Output(k, 2 * n, dtype, 1, k + 2, start=start[1]) if tied else Output(k, 2 * n, dtype, 2 * n + 2, start=start[1])
    made = Output(rows, 2 * n, dtype)
    capi.check(capi.lib().rp_hip_gated_linear_backward(dx.ptr, dw.ptr, db.ptr, made.ptr, dh.ptr, z.ptr, x.ptr, w.ptr, rows, k, n, GATES[gate], dh.rs, x.rs, x.cs, w.rs, w.cs,
                                                       dx.rs, dw.rs, dw.cs, accumulate, accumulate, accumulate, dtype), "rp_hip_gated_linear_backward")
    assert_within(made.read(), dz, dz_off, "dz")
    for out, want, off, what in ((dx, dz @ w.values.T, dz_off @ np.abs(w.values).T + (2 * n + 8) * u * (wide @ np.abs(w.values).T), "dx"),
                                 (dw, x.values.T @ dz, np.abs(x.values).T @ dz_off + (rows + 8) * u * (np.abs(x.values).T @ wide), "dw"),
                                 (db, dz.sum(0)[None], (dz_off + (rows + 8) * u * wide).sum(0)[None], "db")):
        if dtype == F32:
            off = off * (1 + 2.0 ** -20) + 2.0 ** -22 * (wide @ np.abs(w.values).T if what == "dx" else np.abs(x.values).T @ wide if what == "dw" else wide.sum(0)[None])
        bound = rounded(off, want, dtype)
        if accumulate:                                          # the product is rounded, then the sum
            want = want + out.values
            bound = bound + half * (np.abs(want) + bound) + TINY[dtype]
        assert_within(out.read(), want, bound, what)


def test_gradient_agrees_with_differences():
    rng = np.random.default_rng(4)
    rows, k, n, step = 4, 9, 6, 1e-5
    for gate in GATES:
        if gate == "relu":
            continue                                            # (no derivative at 0)
        x, w, c = rng.normal(size=(rows, k)), rng.normal(0, 0.3, size=(k, 2 * n)), rng.normal(size=(rows, n))

        def value(xv, wv):
            return (forward(Operand(xv, F64), Operand(wv, F64), None, n, gate, F64)[0].read() * c).sum()

        xo, wo = Operand(x, F64), Operand(w, F64)
        _, z = forward(xo, wo, None, n, gate, F64)
        dx, dw, dz = Output(rows, k, F64), Output(k, 2 * n, F64), Output(rows, 2 * n, F64)
        capi.check(capi.lib().rp_hip_gated_linear_backward(dx.ptr, dw.ptr, None, dz.ptr, Operand(c, F64).ptr, z.ptr, xo.ptr, wo.ptr, rows, k, n, GATES[gate], n, k, 1, 2 * n, 1, k, 2 * n, 1, 0, 0, 0, F64), "backward")
        for i, j in ((0, 0), (3, 8)):
            e = np.zeros((rows, k))
            e[i, j] = step
            assert abs((value(x + e, w) - value(x - e, w)) / (2 * step) - dx.read()[i, j]) < 1e-7      # (third derivatives below 100)
        for i, j in ((0, 0), (8, 2 * n - 1), (2, n)):
            e = np.zeros((k, 2 * n))
            e[i, j] = step
            assert abs((value(x, w + e) - value(x, w - e)) / (2 * step) - dw.read()[i, j]) < 1e-7


@pytest.mark.parametrize("gate", sorted(GATES))
def test_large_gates_stay_finite(gate):
    """Where exp runs over, the value and its slope are those of the limit."""
    n, rows = 8, 2
    g = np.array([[-3e4, -300.0, -90.0, -30.0, 30.0, 90.0, 300.0, 3e4]] * rows)
    x, w = Operand(np.ones((rows, 1)), F32), Operand(np.concatenate([g[:1], np.full((1, n), 2.0)], 1), F32)
    h, z = forward(x, w, None, n, gate, F32)
    act, slope = gate_reference(g, gate)
    assert_within(h.read(), 2 * act, 64 * 2.0 ** -24 * np.abs(2 * act) * (1 + np.minimum(np.abs(g), 100)) + 1e-12, "h")
    dz = Output(rows, 2 * n, F32)
    capi.check(capi.lib().rp_hip_gated_linear_backward(None, None, None, dz.ptr, Operand(np.ones((rows, n)), F32).ptr, z.ptr, x.ptr, w.ptr, rows, 1, n, GATES[gate], n, 1, 1, 2 * n, 1, 1, 2 * n, 1, 0, 0, 0, F32), "backward")
    assert_within(dz.read(), np.concatenate([2 * slope, act], 1), 1e-5 * (1 + np.abs(np.concatenate([2 * slope, act], 1))), "dz")


@pytest.mark.parametrize("dtype", [BF16, F32], ids=NAMES.get)
@pytest.mark.parametrize("rows,k,n", [(16, 512, 264), (300, 136, 256), (20, 1024, 4096)])
def test_recorded_calls_replay_to_the_eager_result(rows, k, n, dtype):
    rng, x, w, _ = layer(rows, k, n, dtype, False, 3)
    dh = Operand(rng.normal(size=(rows, n)), dtype)
    h, z, dz, dx, dw, db = Output(rows, n, dtype), Output(rows, 2 * n, ACC[dtype]), Output(rows, 2 * n, dtype), Output(rows, k, dtype), Output(k, 2 * n, dtype), Output(1, 2 * n, dtype)
    outs = (h, z, dz, dx, dw, db)

    def step():
        capi.check(capi.lib().rp_hip_gated_linear_forward(h.ptr, z.ptr, x.ptr, w.ptr, None, rows, k, n, 0, x.rs, 1, 2 * n, 1, n, dtype), "forward")
        capi.check(capi.lib().rp_hip_gated_linear_backward(dx.ptr, dw.ptr, db.ptr, dz.ptr, dh.ptr, z.ptr, x.ptr, w.ptr, rows, k, n, 0, n, x.rs, 1, 2 * n, 1, k, 2 * n, 1, 0, 0, 0, dtype), "backward")

    with capi.Stream() as s:
        step()
        eager = [o.bits() for o in outs]
        with capi.Graph.capture() as graph:
            step()
        for _ in range(3):
            for o in outs:
                capi.check(capi.lib().rp_hip_memset(o.buf.ptr, 0, o.buf.nbytes), "memset")
            capi.synchronize()
            graph.launch()
            capi.check(capi.lib().rp_hip_stream_synchronize(), "sync")
            assert all(np.array_equal(a, o.bits()) for a, o in zip(eager, outs))
