"""The loss of a large vocabulary, forward and backward, in a workspace of exactly the size that the question with strides names: nothing behind it is written, and results do not depend on what it held."""
import numpy as np
import pytest

import test_vocab_gpu as vocab
from langhelp import *
from recpulse_amd import capi

pytestmark = pytest.mark.gpu
GUARD = 1 << 16


class Guarded:
    """Device memory of `size` bytes between two guards, filled with `byte`."""

    def __init__(self, size, byte):
        self.size = size
        self.bytes = np.full(size + 2 * GUARD, byte, dtype=np.uint8)
        self.bytes[:GUARD] = self.bytes[GUARD + size:] = 91
        self.buf = capi.DeviceBuffer.from_numpy(self.bytes)

    @property
    def ptr(self):
        return self.buf.at(GUARD)

    def check(self):
        capi.synchronize()
        got = self.buf.to_numpy(np.uint8, self.bytes.shape)
        assert np.all(got[:GUARD] == 91) and np.all(got[GUARD + self.size:] == 91), "written outside of the workspace"


@pytest.mark.parametrize("dtype", ALL, ids=NAMES.get)
@pytest.mark.parametrize("lies", ["rows", "transposed", "strided"])
@pytest.mark.parametrize("rows,k,classes", [(1, 1, 1), (16, 256, 1031), (64, 520, 2050), (300, 72, 777), (1000, 520, 2056), (7, 5, 70000), (520, 1064, 3000)])
def test_workspaces_of_exactly_that_size(rows, k, classes, lies, dtype):
    rng, x, w, b, targets = vocab.problem(rows, k, classes, dtype, 8, lies == "transposed")
    if lies == "strided":
        w = Operand(w.values, dtype, rs=2 * classes + 1, cs=2, lead=1)
    size = [capi.lib().rp_hip_linear_cross_entropy_workspace_strided(rows, k, classes, backward, x.rs, x.cs, w.rs, w.cs, dtype) for backward in (0, 1)]
    assert 0 < size[0] <= size[1]
    up = vector([2.0], ACC[dtype])
    results = []
    for byte in (0, 255):                                       # (NaN in every type)
        space = Guarded(size[0], byte)
        loss, stats = vocab.forward(x, w, b, targets, dtype, 1, space)
        space.check()
        space = Guarded(size[1], byte)
        outs = dx, dw, db = Output(rows, k, dtype, k + 3), Output(k, classes, dtype), Output(1, classes, dtype)
        capi.check(capi.lib().rp_hip_linear_cross_entropy_backward(dx.ptr, dw.ptr, db.ptr, x.ptr, w.ptr, b.ptr, ints(targets).ptr, stats.ptr, up.ptr, space.ptr, rows, k, classes, 1,
                                                                   x.rs, x.cs, w.rs, w.cs, dx.rs, dw.rs, dw.cs, 0, 0, 0, dtype), "rp_hip_linear_cross_entropy_backward")
        space.check()
        for out in outs:
            out.read()
        results.append([o.bits() for o in (loss, stats) + outs])
    assert all(np.array_equal(p, q) for p, q in zip(*results))
    assert np.isfinite(f64(results[0][0], ACC[dtype])).all()
