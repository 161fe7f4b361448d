"""Grouped and adapter layers on streams of their own and in graphs: nothing is shared with other streams' calls, and none needs a call before it is recorded."""
import numpy as np
import pytest

import oracle
from recpulse_amd import capi
from devhelp import BF16, F16, Dev
from test_grouped_gpu import Grouped, call, ids_of, ptr

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
