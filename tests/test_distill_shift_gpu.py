"""Distillation of logits far from zero: their common offset changes neither loss nor gradient, and costs no digits of them."""
import numpy as np
import pytest

import test_distill_gpu as distill
from langhelp import *
from recpulse_amd import capi

pytestmark = pytest.mark.gpu

SHIFT = {F32: 4096.0, F64: 4096.0, F16: 1024.0, BF16: 256.0}
# (rows, classes, k): fewer classes than a vector, every way of holding a row, more entries than a small workgroup has threads
SIZES = [(40, 3, 2), (64, 1000, 10), (40, 1500, 300), (9, 9001, 20), (5, 33000, 64), (4, 70001, 5), (3, 140000, 6)]


def bounds(logits, ids, teacher, temperature, q, mass, f, want_log, dtype):
    """In units of the accumulate type's half step u.  A weight is 2 to (x s - b) with s = log2 e / T off by 3 of itself, so that of two classes that are D apart (in units of T) its logarithm is off by
    4 D, the exponential by 2; a sum adds classes / 256 of them one after the other and 40 more; a logarithm and a quotient are off by 2 of themselves.  None of it grows with the offset."""
    u, k = UNIT[dtype], ids.shape[1]
    apart = (logits.max(1, keepdims=True) - logits) / temperature
    apart_t = (teacher.max(1) - teacher.min(1)) / temperature
    steps = logits.shape[1] / 256 + 40
    log_q = u * (11 * apart.max(1) + steps + 50)
    log_p = u * (11 * apart_t + k + 60)
    loss = temperature ** 2 * (log_q + 2 * log_p + (2 * log_p + (k + 8) * u) * want_log)
    grad = np.abs(f)[:, None] * (q * u * (4 * apart + 4 * apart.max(1, keepdims=True) + steps + 14) + mass * u * (8 * apart_t[:, None] + 2 * k + 20) + 3 * u * (q + mass))
    return loss, grad


@pytest.mark.parametrize("dtype", ALL, ids=NAMES.get)
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("rows,classes,k", SIZES)
def test_logits_far_from_zero(rows, classes, k, sign, dtype):
    temperature, u = 2.0, UNIT[dtype]                            # (a power of two: the reference's quotients are exact)
    rng = np.random.default_rng(classes + k)
    logits = Operand(sign * (SHIFT[dtype] + rng.normal(2, 2, size=(rows, classes))), dtype, rs=classes + 1)
    teacher = Operand(sign * (SHIFT[dtype] + rng.normal(2, 2, size=(rows, k))), dtype)
    ids = np.stack([rng.choice(classes, k, replace=False) for _ in range(rows)]).astype(np.int32)
    want, grad, q, mass, f = distill_reference(logits.values, ids, teacher.values, temperature, 0, 1.0)
    log_q, t = np.log(q), teacher.values / temperature
    log_p = t - t.max(1, keepdims=True) - np.log(np.exp(t - t.max(1, keepdims=True)).sum(1, keepdims=True))
    loss_off, grad_off = bounds(logits.values, ids, teacher.values, temperature, q, mass, f, np.abs(log_p - np.take_along_axis(log_q, ids, 1)).max(1), dtype)
    loss, out, stats = distill.forward(logits, ids, teacher, temperature, 0, dtype)
    assert_within(loss.read()[0], want, loss_off + 4 * u * np.abs(want), "loss")
    assert_within(out.read(), grad, rounded(grad_off, grad, dtype), "gradient")
    loss, _, kept = distill.forward(logits, ids, teacher, temperature, 0, dtype, grad=False)
    assert_within(loss.read()[0], want, loss_off + 4 * u * np.abs(want), "loss alone")
    for st in (stats, kept):
        alone = Output(rows, classes, dtype)
        capi.check(capi.lib().rp_hip_distillation_backward(alone.ptr, st.ptr, logits.ptr, ints(ids).ptr, teacher.ptr, None, rows, classes, k, logits.rs, temperature, 0, dtype), "rp_hip_distillation_backward")
        assert_within(alone.read(), grad, rounded(grad_off, grad, dtype), "gradient alone")
