"""Grouped and adapter layers on streams of their own and in graphs: nothing is shared with other streams' calls, and none needs a call before it is recorded."""
import ctypes

import numpy as np
import pytest

import oracle
from recpulse_amd import capi
from devhelp import BF16, F16, F32, F64, Dev
from test_grouped_gpu import Adapters, Grouped, call, ids_of, ptr

pytestmark = pytest.mark.gpu


def replayed(stream, record, outputs, check):
    """Recorded with nothing before it and no block in the pool, and replayed three times over cleared outputs."""
    capi.check(capi.lib().rp_hip_empty_cache(), "rp_hip_empty_cache")
    with capi.Graph.capture() as g:
        record()
    for _ in range(3):
        for o in outputs:
            call("rp_hip_memset", o.ptr, 0xff, o.buf.nbytes)
        g.launch()
        capi.check(capi.lib().rp_hip_stream_synchronize(), "rp_hip_stream_synchronize")
        check()


@pytest.mark.parametrize("dt", [BF16, F16], ids=ids_of)
def test_few_rows_recorded_without_a_call_before(dt):
    groups, rows, k, n = 2, 5, 4096, 512
    p = Grouped(dt, groups, rows, k, n, bias=False, nan=False)
    y = Dev.empty((rows, n), dt)

    def forward():
        call("rp_hip_grouped_linear_forward", y.ptr, p.dx.ptr, p.dw.ptr, None, p.do.ptr, groups, rows, k, n, k, 1, k * n, n, 1, n, dt)

    def check():
        p.check_forward(y)

    with capi.Stream() as stream:
        replayed(stream, forward, [y], check)
        forward()
        check()
        with capi.Graph.capture() as g:                        # (with a block for the shares of k now)
            forward()
        for _ in range(3):
            call("rp_hip_memset", y.ptr, 0xff, y.buf.nbytes)
            g.launch()
            check()


# a few rows; the term as a launch of its own (in one and in several parts of the rows); rows shared by workgroups in the gradients, beside dx's tiles and alone; products of float32 whose k
# is split on the null stream; widths and types that no kernel of the adapters' own takes
ADAPTERS = [(9, 4, 32, 4096, 512, 16, BF16), (90, 5, 300, 264, 136, 8, F16), (900, 5, 2500, 264, 2056, 8, BF16), (3, 2, 9000, 96, 200, 33, F16), (1, 1, 5000, 2048, 64, 16, BF16),
            (5, 3, 40, 2048, 256, 8, F32), (2, 2, 4, 4096, 2048, 8, F32), (4, 2, 60, 2000, 5, 4, BF16), (4, 2, 60, 1000, 130, 4, F64)]


class ForeignStream(capi.Stream):
    """A stream that the library did not make: it does not know when one ends, and keeps no memory for it."""

    def __init__(self):
        p = ctypes.c_void_p()
        assert capi.lib().hipStreamCreateWithFlags(ctypes.byref(p), 1) == 0          # (of the runtime that the library is linked to)
        self.ptr, self._prev = p.value, None

    def __del__(self):
        capi.lib().hipStreamDestroy(ctypes.c_void_p(self.ptr))


class Step:
    """A layer's forward and backward pass with outputs of its own."""

    def __init__(self, shape, seed):
        *sizes, dt = shape
        self.p = p = Adapters(dt, *sizes, behind=min(3, sizes[2] - 1), seed=seed)
        _, adapters, rows, k, n, rank = sizes
        p.y, p.h = Dev.empty((rows, n), dt), Dev.empty((rows, rank), p.acc)
        self.u, self.out = Dev.empty((rows, rank), p.acc), [Dev.empty(s, dt) for s in ((rows, k), (adapters, k, rank), (adapters, rank, n))]

    def run(self):
        p, d = self.p, self.p.d
        _, _, rows, k, n, rank = p.sizes
        call("rp_hip_adapter_linear_forward", p.y.ptr, p.h.ptr, d["x"].ptr, d["w"].ptr, ptr(d["bias"]), d["a"].ptr, d["b"].ptr, *p.plan(), k, 1, *p.w_st, n, p.dt)
        call("rp_hip_adapter_linear_backward", *[o.ptr for o in self.out], self.u.ptr, d["g"].ptr, d["x"].ptr, d["w"].ptr, d["a"].ptr, d["b"].ptr, p.h.ptr, *p.plan(),
             n, k, 1, *p.w_st, k, 0, 0, 0, p.dt)

    def clear(self):
        for o in self.results():
            call("rp_hip_memset", o.ptr, 0xff, o.buf.nbytes)
        h = np.full((self.p.sizes[2], self.p.sizes[5]), 3.0, dtype=capi.NP_STORAGE[self.p.acc])
        call("rp_hip_memcpy_h2d", self.p.h.ptr, h.ctypes.data, h.nbytes)

    def results(self):
        return [self.p.y, *self.out]

    def bits(self):
        return [o.numpy() for o in self.results()]

    def check(self):
        self.p.check_forward()
        self.p.check_backward(self.out)


@pytest.mark.parametrize("kind", [capi.Stream, ForeignStream], ids=["created", "foreign"])
@pytest.mark.parametrize("shape", ADAPTERS, ids=lambda s: "x".join(map(str, s[:6])) + ids_of(s[6]))
def test_adapters_on_two_streams_at_once_and_recorded(shape, kind):
    """Two layers' passes side by side, with a third on the null stream: each has the bits that it has alone.  Then the same recorded, with nothing before and with blocks in the
    pool, and two graphs replayed side by side."""
    steps = [Step(shape, seed) for seed in range(3)]
    streams = [kind(), kind()]
    alone = []
    for s, v in zip(streams + [None], steps):
        v.clear()
        if s is None:
            v.run()
        else:
            with s:
                v.run()
        capi.synchronize()
        v.check()
        alone.append(v.bits())
    for _ in range(4):
        for v in steps:
            v.clear()
        capi.synchronize()
        for s, v in zip(streams, steps):
            with s:
                v.run()
        steps[2].run()
        capi.synchronize()
        for v, want in zip(steps, alone):
            for a, b in zip(v.bits(), want):
                assert np.array_equal(a.view(np.uint8), b.view(np.uint8))
    with streams[0]:
        replayed(streams[0], steps[0].run, steps[0].results(), steps[0].check)
    graphs = []
    for s, v in zip(streams, steps):
        with s:
            v.run()
            with capi.Graph.capture() as g:
                v.run()
            v.clear()
            g.launch()
            capi.synchronize()
            v.check()
        graphs.append((s, g, v, v.bits()))
    for _ in range(3):
        for v in steps:
            v.clear()
        capi.synchronize()
        for s, g, v, _ in graphs:
            with s:
                g.launch()
        capi.synchronize()
        for _, _, v, want in graphs:
            for a, b in zip(v.bits(), want):
                assert np.array_equal(a.view(np.uint8), b.view(np.uint8))


def test_a_stream_with_memory_ends_while_another_is_recorded():
    """The memory is given back later: a recording allows no freeing."""
    steps = [Step((9, 4, 32, 4096, 512, 16, BF16), seed) for seed in range(2)]
    here, other = capi.Stream(), capi.Stream()
    for s, v in zip((here, other), steps):
        v.clear()
        with s:
            v.run()
        capi.synchronize()
        v.check()
    with here:
        with capi.Graph.capture() as g:
            steps[0].run()
            ended, other.ptr = other.ptr, None
            call("rp_hip_stream_destroy", ended)
            steps[0].run()
        for _ in range(3):
            steps[0].clear()
            g.launch()
            capi.synchronize()
            steps[0].check()
    with capi.Stream():                                        # (the next one frees it)
        steps[1].clear()
        steps[1].run()
        capi.synchronize()
        steps[1].check()


def test_memory_goes_with_the_streams():
    """Streams made and ended one after the other do not keep their memory."""
    v = Step((900, 5, 2500, 264, 2056, 8, BF16), 3)
    free, total = ctypes.c_size_t(), ctypes.c_size_t()
    left = []
    for _ in range(12):
        v.clear()
        with capi.Stream():
            v.run()
        capi.synchronize()
        v.check()
        assert capi.lib().hipMemGetInfo(ctypes.byref(free), ctypes.byref(total)) == 0
        left.append(free.value)
    assert left[-1] >= left[2] - (8 << 20)
