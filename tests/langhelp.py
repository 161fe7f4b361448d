"""Helpers for the tests of layer norm, gated layers, the loss of a large vocabulary and distillation: operands with any strides, outputs with gaps that have to
stay as they were, and bounds for the comparison with 64 bits."""
import numpy as np

import oracle
from recpulse_amd import capi

F32, F64, F16, BF16 = capi.F32, capi.F64, capi.F16, capi.BF16
ALL = [F32, F64, F16, BF16]
NAMES = {F32: "f32", F64: "f64", F16: "f16", BF16: "bf16"}
HALF = {F32: 2.0 ** -24, F64: 2.0 ** -53, F16: 2.0 ** -11, BF16: 2.0 ** -8}      # a rounding is off by at most this share of the value
TINY = {F32: 2.0 ** -150, F64: 0.0, F16: 2.0 ** -25, BF16: 2.0 ** -134}          # and, where the result is subnormal, by this much
ACC = {F32: F32, F64: F64, F16: F32, BF16: F32}
UNIT = {F32: 2.0 ** -24, F64: 2.0 ** -53, F16: 2.0 ** -24, BF16: 2.0 ** -24}     # half a step of the accumulate type
MARK = 17.0                                                                     # what outputs hold before a call


def storage(values, dtype):
    return oracle.to_storage(np.asarray(values, dtype=np.float64), dtype)


def f64(array, dtype):
    return oracle.to_f64(np.ascontiguousarray(array), dtype)


class Operand:
    """A [rows, cols] operand on the device with strides in elements: `lead` elements before it, rows `rs` apart, columns `cs`."""

    def __init__(self, values, dtype, rs=None, cs=1, lead=0):
        values = np.asarray(values, dtype=np.float64)
        rows, cols = values.shape
        self.shape, self.dtype, self.cs, self.lead = (rows, cols), dtype, cs, lead
        self.rs = rs if rs is not None else cols * cs
        size = lead + (rows - 1) * self.rs + (cols - 1) * cs + 1
        self.store = storage(np.full(size, MARK), dtype)
        self.at = lead + np.arange(rows)[:, None] * self.rs + np.arange(cols) * cs
        self.store[self.at] = storage(values, dtype)
        self.values = f64(self.store[self.at], dtype)          # what the device sees
        self.buf = capi.DeviceBuffer.from_numpy(self.store)

    @property
    def ptr(self):
        return self.buf.at(self.lead * capi.DTYPE_SIZE[self.dtype])


class Output(Operand):
    """The same for an output; what lies between its rows and columns has to stay as it was."""

    def __init__(self, rows, cols, dtype, rs=None, cs=1, lead=0, start=None):
        super().__init__(np.full((rows, cols), MARK) if start is None else start, dtype, rs, cs, lead)

    def read(self):
        capi.synchronize()
        got = self.buf.to_numpy(self.store.dtype, self.store.shape)
        outside = np.ones(got.shape, dtype=bool)
        outside[self.at] = False
        assert np.array_equal(got[outside], self.store[outside]), "written outside of the output"
        return f64(got[self.at], self.dtype)

    def bits(self):
        capi.synchronize()
        return self.buf.to_numpy(self.store.dtype, self.store.shape)[self.at]


def vector(values, dtype):
    return Operand(np.asarray(values, dtype=np.float64)[None], dtype)


def ints(values):
    return capi.DeviceBuffer.from_numpy(np.ascontiguousarray(values, dtype=np.int32))


def room(size):
    assert size >= 0
    return capi.DeviceBuffer(max(1, size))


def at(operand):
    return None if operand is None else operand.ptr


def rounded(bound, want, dtype):
    """The bound of an output that is rounded once to its type, of values that are off by `bound`."""
    return bound + HALF[dtype] * (np.abs(want) + bound) + TINY[dtype]


def assert_within(got, want, bound, what):
    got, want, bound = np.broadcast_arrays(np.asarray(got, dtype=np.float64), want, bound)
    assert np.array_equal(np.isnan(got), np.isnan(want)), f"{what}: NaN where there is none, or none where there is"
    fine = np.isfinite(want)
    assert np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)]), f"{what}: infinities"
    off = np.abs(got[fine] - want[fine])
    worst = np.argmax(off - bound[fine]) if off.size else 0
    assert np.all(off <= bound[fine]), f"{what}: off by {off[worst]:.3e}, allowed {bound[fine][worst]:.3e} at {want[fine][worst]:.6e} ({np.mean(off > bound[fine]):.3f} of the values)"


def norm_reference(x, w, b, eps):
    mean = x.mean(1, keepdims=True)
    r = 1.0 / np.sqrt(((x - mean) ** 2).mean(1, keepdims=True) + eps)
    h = (x - mean) * r
    return mean, r, h, h * (1.0 if w is None else w) + (0.0 if b is None else b)


GATES = {"silu": 0, "gelu": 1, "gelu_tanh": 2, "relu": 3, "sigmoid": 4}


def gate_reference(g, gate):
    """act(g) and its derivative in 64 bits."""
    from scipy.special import expit, ndtr
    if gate == "relu":
        return np.maximum(g, 0.0), (g > 0).astype(np.float64)
    if gate == "gelu":
        return g * ndtr(g), ndtr(g) + g * np.exp(-0.5 * g * g) / np.sqrt(2.0 * np.pi)
    if gate == "gelu_tanh":
        a = np.sqrt(2.0 / np.pi)
        s = expit(2.0 * a * (g + 0.044715 * g ** 3))
        return g * s, s + 2.0 * g * s * (1.0 - s) * a * (1.0 + 3.0 * 0.044715 * g * g)
    s = expit(g)
    return (s, s * (1.0 - s)) if gate == "sigmoid" else (g * s, s * (1.0 + g * (1.0 - s)))


def vocab_reference(x, w, bias, targets, reduction, upstream):
    """Result, log sums, and the gradient of the logits, in 64 bits."""
    z = x @ w + (0.0 if bias is None else bias)
    rows, classes = z.shape
    top = z.max(1, keepdims=True)
    lse = np.log(np.exp(z - top).sum(1)) + top[:, 0]
    held = (targets >= 0) & (targets < classes)
    safe = np.where(held, targets, 0)
    losses = np.where(held, lse - z[np.arange(rows), safe], 0.0)
    count = held.sum()
    result = losses if reduction == 0 else np.array([losses.sum() / (max(count, 1) if reduction == 1 else 1)])
    f = np.where(held, upstream, 0.0) / (max(count, 1) if reduction == 1 else 1)
    d = np.exp(z - lse[:, None])
    d[np.arange(rows), safe] -= 1.0
    return result, lse, d * f[:, None], f, np.exp(z - lse[:, None])


def distill_reference(logits, ids, teacher, temperature, reduction, upstream):
    rows, classes = logits.shape
    u = logits / temperature
    top = u.max(1, keepdims=True)
    log_q = u - top - np.log(np.exp(u - top).sum(1, keepdims=True))
    losses, grad, mass = np.zeros(rows), np.zeros_like(u), np.zeros_like(u)
    for i in range(rows):
        kept = [j for j in range(ids.shape[1]) if 0 <= ids[i, j] < classes and teacher[i, j] > -np.inf]
        if not kept:
            continue
        t = teacher[i, kept] / temperature
        log_p = t - t.max() - np.log(np.exp(t - t.max()).sum())
        for j, lp in zip(kept, log_p):
            p = np.exp(lp)
            if p > 0:
                losses[i] += p * (lp - log_q[i, ids[i, j]])
            mass[i, ids[i, j]] += p
        grad[i] = np.exp(log_q[i]) - mass[i]
    losses *= temperature ** 2
    f = temperature * np.asarray(upstream, dtype=np.float64) / (rows if reduction == 1 else 1) * np.ones(rows)
    result = losses if reduction == 0 else np.array([losses.sum() / (rows if reduction == 1 else 1)])
    return result, grad * f[:, None], np.exp(log_q), mass, f
