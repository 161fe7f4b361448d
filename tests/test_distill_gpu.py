"""Distillation from a teacher's top logits on the device against the formulas in 64 bits."""
import numpy as np
import pytest

from langhelp import *
from recpulse_amd import capi

pytestmark = pytest.mark.gpu

# (rows, classes, k): one of everything, fewer classes than a vector, a workgroup's registers of every size and the classes that no longer fit, more entries than threads
SIZES = [(1, 1, 1), (2, 3, 2), (7, 10, 4), (33, 1000, 10), (3, 2048, 64), (2, 2051, 300), (2, 8200, 7), (2, 16391, 20), (1, 33000, 64), (1, 65536, 8), (2, 70001, 5), (1, 140000, 6), (5, 1500, 1024)]


def problem(rows, classes, k, dtype, seed, twice=False, padded=True):
    rng = np.random.default_rng(seed)
    logits = Operand(rng.normal(0, 2, size=(rows, classes)), dtype, rs=classes + 3)
    ids = np.stack([rng.choice(classes, k, replace=twice or k > classes) for _ in range(rows)]).astype(np.int32)
    teacher = rng.normal(2, 2, size=(rows, k))
    if padded and rows > 1:
        ids[0, k // 2:] = -1
        ids[1, 0] = classes                                     # (behind the last class is outside as well)
        if k > 2:
            teacher[-1, 1] = -np.inf
    return rng, logits, ids, Operand(teacher, dtype)


def forward(logits, ids, teacher, temperature, reduction, dtype, upstream=None, grad=True):
    rows, classes = logits.shape
    loss, stats = Output(1, rows if reduction == 0 else 1, ACC[dtype]), Output(1, 3 * rows, ACC[dtype])
    out = Output(rows, classes, dtype) if grad else None
    capi.check(capi.lib().rp_hip_distillation_forward(loss.ptr, at(out), stats.ptr, logits.ptr, ints(ids).ptr, teacher.ptr, at(upstream), rows, classes, ids.shape[1], logits.rs, temperature,
                                                      reduction, dtype), "rp_hip_distillation_forward")
    return loss, out, stats


@pytest.mark.parametrize("dtype", ALL, ids=NAMES.get)
@pytest.mark.parametrize("rows,classes,k", SIZES)
def test_loss_and_gradient(rows, classes, k, dtype):
    temperature, reduction, u = (1.0, 1.5, 4.0)[k % 3], (rows + k) % 3, UNIT[dtype]
    rng, logits, ids, teacher = problem(rows, classes, k, dtype, classes + k, twice=k % 2 == 0)
    up = vector(rng.uniform(0.5, 2, rows if reduction == 0 else 1) * rows, ACC[dtype])
    want, grad, q, mass, f = distill_reference(logits.values, ids, teacher.values, temperature, reduction, up.values[0])
    loss, out, stats = forward(logits, ids, teacher, temperature, reduction, dtype, up)
    # a log sum: teams add fewer than 400 exponentials one after the other (longer rows 1024 threads walk), arguments are rounded to u of themselves
    steps = 400 + classes / 1024
    size = np.abs(logits.values).max(1) / temperature + np.abs(np.where(np.isfinite(teacher.values), teacher.values, 0.0)).max(1) / temperature
    lse_off = u * (steps + 8 * size)
    log_q_off = 2 * lse_off + 4 * u * size
    loss_off = temperature ** 2 * (2 * log_q_off + 64 * u * (size + 10) + k * u * (2 * size + 20))
    loss_off = loss_off if reduction == 0 else loss_off.sum() / (rows if reduction == 1 else 1)
    assert_within(loss.read()[0], want, loss_off + 2 * u * np.abs(want), "loss")
    off = np.abs(f)[:, None] * (q * 1.1 * (lse_off[:, None] + 16 * u * (1 + np.abs(np.log(np.maximum(q, 1e-300))))) + mass * (lse_off[:, None] + (k + 16) * u * (1 + 2 * size[:, None])) + 4 * u * (q + mass))
    assert_within(out.read(), grad, rounded(off, grad, dtype), "gradient")
    alone = Output(rows, classes, dtype)
    capi.check(capi.lib().rp_hip_distillation_backward(alone.ptr, stats.ptr, logits.ptr, ints(ids).ptr, teacher.ptr, up.ptr, rows, classes, k, logits.rs, temperature, reduction, dtype), "rp_hip_distillation_backward")
    assert np.array_equal(alone.bits(), out.bits())


@pytest.mark.parametrize("dtype", ALL, ids=NAMES.get)
def test_rows_without_entries_are_left_out(dtype):
    rng, logits, ids, teacher = problem(4, 300, 5, dtype, 1, padded=False)
    ids[1] = -1
    t = teacher.values.copy()
    t[2] = -np.inf
    teacher = Operand(t, dtype)
    loss, grad, _ = forward(logits, ids, teacher, 2.0, 0, dtype)
    assert np.all(loss.read()[0, [1, 2]] == 0) and np.all(grad.read()[[1, 2]] == 0)
    assert np.all(loss.read()[0, [0, 3]] > 0) and np.all(np.abs(grad.read()[[0, 3]]).sum(1) > 0)


def test_a_class_named_twice_counts_twice():
    logits, teacher = Operand(np.zeros((1, 8)), F32), Operand(np.zeros((1, 4)), F32)
    _, grad, _ = forward(logits, np.array([[2, 2, 5, 2]]), teacher, 1.0, 2, F32)
    want = np.full((1, 8), 1 / 8)
    want[0, 2] -= 3 / 4
    want[0, 5] -= 1 / 4
    assert_within(grad.read(), want, 8 * 2.0 ** -24, "gradient")


@pytest.mark.parametrize("dtype", ALL, ids=NAMES.get)
def test_infinite_and_missing_logits(dtype):
    """A class that the student excludes and the teacher wants has an infinite loss; NaN stays in its row."""
    rng, logits, ids, teacher = problem(4, 520, 6, dtype, 3, padded=False)
    v = logits.values.copy()
    v[0, ids[0, 2]] = -np.inf
    v[1, [k for k in range(520) if k not in ids[1]][:50]] = -np.inf
    v[2, 0] = np.nan
    logits = Operand(v, dtype)
    loss, grad, _ = forward(logits, ids, teacher, 1.0, 0, dtype)
    got, g = loss.read()[0], grad.read()
    assert got[0] == np.inf and np.isfinite(got[1]) and np.isnan(got[2]) and np.isfinite(got[3])
    assert np.all(np.isfinite(g[[0, 1, 3]])) and np.all(g[1][v[1] == -np.inf] == 0)


def test_gradient_agrees_with_differences():
    rng, logits, ids, teacher = problem(3, 13, 4, F64, 9)
    _, grad, _ = forward(logits, ids, teacher, 1.7, 1, F64)
    for i, j in ((0, 0), (1, 5), (2, int(ids[2, 0]))):
        e = np.zeros(logits.shape)
        e[i, j] = 1e-5
        plus, minus = (forward(Operand(logits.values + s * e, F64), ids, teacher, 1.7, 1, F64, grad=False)[0].read()[0, 0] for s in (1, -1))
        assert abs((plus - minus) / 2e-5 - grad.read()[i, j]) < 1e-8


def test_recorded_calls_replay_to_the_eager_result():
    for rows, classes in ((20, 1000), (3, 70001)):
        _, logits, ids, teacher = problem(rows, classes, 9, BF16, 4)
        idev, loss, grad, stats = ints(ids), Output(1, 1, F32), Output(rows, classes, BF16), Output(1, 3 * rows, F32)

        def step():
            capi.check(capi.lib().rp_hip_distillation_forward(loss.ptr, grad.ptr, stats.ptr, logits.ptr, idev.ptr, teacher.ptr, None, rows, classes, 9, logits.rs, 2.0, 1, BF16), "forward")

        with capi.Stream() as s:
            step()
            eager = [o.bits() for o in (loss, grad, stats)]
            with capi.Graph.capture() as graph:
                step()
            for _ in range(3):
                for o in (loss, grad, stats):
                    capi.check(capi.lib().rp_hip_memset(o.buf.ptr, 0, o.buf.nbytes), "memset")
                capi.synchronize()
                graph.launch()
                capi.check(capi.lib().rp_hip_stream_synchronize(), "sync")
                assert all(np.array_equal(a, o.bits()) for a, o in zip(eager, (loss, grad, stats)))
