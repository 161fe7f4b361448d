"""Layer norm, gated layers, the loss of a large vocabulary and distillation on streams that nothing orders, on streams that the library did not make, and in graphs."""
import numpy as np
import pytest

import test_distill_gpu as distill
import test_gated_gpu as gated
import test_norm_gpu as norm
import test_vocab_gpu as vocab
from langhelp import *
from recpulse_amd import capi
from test_grouped_streams_gpu import ForeignStream

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ALL, ids=NAMES.get)
@pytest.mark.parametrize("tied", [False, True], ids=["rows", "transposed"])
def test_every_pass_on_a_stream_without_memory(tied, dtype):
    """... whose products are not split where that takes memory, within the same bounds."""
    with ForeignStream():
        for rows, k, n in ((16, 2048, 1032), (5, 1100, 72), (300, 72, 264), (700, 520, 264)):
            gated.test_forward(rows, k, n, tied, dtype)
            gated.test_backward(rows, k, n, tied, dtype)
        for rows, k, classes in ((16, 256, 1031), (64, 520, 2050), (257, 129, 1537)):
            vocab.test_forward(rows, k, classes, tied, dtype)
            vocab.test_backward(rows, k, classes, tied, dtype)
        norm.test_forward(37, 520, dtype)
        norm.test_backward(37, 520, dtype)
        distill.test_loss_and_gradient(21, 1000, 10, dtype)


class Step:
    """All four operators, forward and backward, on operands of its own."""

    def __init__(self, dtype, seed, rows, k, n, classes, entries, tied):
        rng = np.random.default_rng(seed)
        self.sizes, self.dtype, self.entries = (rows, k, n, classes), dtype, entries
        self.x, self.scale = Operand(rng.normal(size=(rows, k)), dtype), vector(rng.normal(size=k), dtype)
        v = rng.normal(0, k ** -0.5, size=(k, 2 * n))
        self.w = Operand(v, dtype, 1, k) if tied else Operand(v, dtype)
        v = rng.normal(0, n ** -0.5, size=(n, classes))
        self.head = Operand(v, dtype, 1, n) if tied else Operand(v, dtype)
        self.logits, self.teacher = Operand(rng.normal(size=(rows, classes)), dtype), Operand(rng.normal(size=(rows, entries)), dtype)
        self.ids, self.targets = ints(rng.integers(0, classes, (rows, entries))), ints(rng.integers(0, classes, rows))
        a = ACC[dtype]
        weights = lambda r, c: Output(r, c, dtype, 1, r) if tied else Output(r, c, dtype)
        self.outs = {"y": Output(rows, k, dtype), "norm": Output(rows, 2, a), "z": Output(rows, 2 * n, a), "h": Output(rows, n, dtype), "loss": Output(1, 1, a), "stats": Output(1, 2 * rows + 1, a),
                     "dh": Output(rows, n, dtype), "dhead": weights(n, classes), "dz": Output(rows, 2 * n, dtype), "dy": Output(rows, k, dtype), "dw": weights(k, 2 * n), "db": Output(1, 2 * n, dtype),
                     "dx": Output(rows, k, dtype), "dscale": Output(1, k, dtype), "kl": Output(1, 1, a), "kl_stats": Output(1, 3 * rows, a), "dlogits": Output(rows, classes, dtype)}
        lib = capi.lib()
        self.space = room(max(lib.rp_hip_linear_cross_entropy_workspace(rows, n, classes, 1, dtype), lib.rp_hip_layer_norm_workspace(rows, k, dtype)))

    def run(self):
        (rows, k, n, classes), t, lib, w, head, space = self.sizes, self.dtype, capi.lib(), self.w, self.head, self.space.ptr
        o = {name: out.ptr for name, out in self.outs.items()}
        dhead, dw = self.outs["dhead"], self.outs["dw"]
        for name, args in (("layer_norm_forward", (o["y"], o["norm"], self.x.ptr, self.scale.ptr, None, rows, k, k, k, 1e-5, t)),
                           ("gated_linear_forward", (o["h"], o["z"], o["y"], w.ptr, None, rows, k, n, 0, k, 1, w.rs, w.cs, n, t)),
                           ("linear_cross_entropy_forward", (o["loss"], o["stats"], o["h"], head.ptr, None, self.targets.ptr, space, rows, n, classes, 1, n, 1, head.rs, head.cs, t)),
                           ("linear_cross_entropy_backward", (o["dh"], o["dhead"], None, o["h"], head.ptr, None, self.targets.ptr, o["stats"], None, space, rows, n, classes, 1, n, 1,
                                                              head.rs, head.cs, n, dhead.rs, dhead.cs, 0, 0, 0, t)),
                           ("gated_linear_backward", (o["dy"], o["dw"], o["db"], o["dz"], o["dh"], o["z"], o["y"], w.ptr, rows, k, n, 0, n, k, 1, w.rs, w.cs, k, dw.rs, dw.cs, 0, 0, 0, t)),
                           ("layer_norm_backward", (o["dx"], o["dscale"], None, o["dy"], self.x.ptr, self.scale.ptr, o["norm"], space, rows, k, k, k, k, 0, 0, 0, t)),
                           ("distillation_forward", (o["kl"], o["dlogits"], o["kl_stats"], self.logits.ptr, self.ids.ptr, self.teacher.ptr, None, rows, classes, self.entries, classes, 2.0, 1, t))):
            capi.check(getattr(lib, "rp_hip_" + name)(*args), name)

    def bits(self):
        return {name: out.bits() for name, out in self.outs.items()}

    def clear(self):
        for out in self.outs.values():
            capi.check(capi.lib().rp_hip_memset(out.buf.ptr, 0, out.buf.nbytes), "memset")
        capi.check(capi.lib().rp_hip_memset(self.space.ptr, 255, self.space.nbytes), "memset")


SIZES = [(16, 1024, 2048, 4096, False), (16, 1024, 2048, 4096, True), (5, 520, 264, 1031, True), (600, 520, 264, 2056, False)]


def same(step, want, when):
    got = step.bits()
    assert [name for name in want if not np.array_equal(want[name], got[name])] == [], when


@pytest.mark.parametrize("kind", [capi.Stream, ForeignStream], ids=["created", "foreign"])
@pytest.mark.parametrize("dtype", [BF16, F32, F64], ids=NAMES.get)
@pytest.mark.parametrize("rows,k,n,classes,tied", SIZES)
def test_two_streams_at_a_time(rows, k, n, classes, tied, dtype, kind):
    """Steps on two streams that nothing orders leave what each leaves alone."""
    steps = [Step(dtype, seed, rows, k, n, classes, 10, tied) for seed in (1, 2)]
    streams = [kind(), kind()]
    alone = []
    for step, stream in zip(steps, streams):
        with stream:
            step.run()
        alone.append(step.bits())
    for step in steps:
        step.clear()
    capi.synchronize()
    for _ in range(12):
        for step, stream in zip(steps, streams):
            with stream:
                step.run()
    capi.synchronize()
    for step, want in zip(steps, alone):
        same(step, want, "both")


@pytest.mark.parametrize("dtype", [BF16, F32, F64], ids=NAMES.get)
@pytest.mark.parametrize("rows,k,n,classes,tied", SIZES)
def test_recorded_steps_side_by_side(rows, k, n, classes, tied, dtype):
    """Recorded with no block in the pool and with some, replayed over cleared outputs and workspaces while another graph runs, with eager work of the same kind between."""
    steps = [Step(dtype, seed, rows, k, n, classes, 10, tied) for seed in (1, 2, 3)]
    streams = [capi.Stream(), capi.Stream()]
    graphs = []
    for step, stream in zip(steps, streams):
        with stream:
            capi.check(capi.lib().rp_hip_empty_cache(), "rp_hip_empty_cache")
            with capi.Graph.capture() as bare:
                step.run()
            step.run()
            with capi.Graph.capture() as graph:
                step.run()
            for g in (bare, graph):
                step.clear()
                capi.synchronize()
                g.launch()
                want = step.bits()
                for _ in range(2):
                    step.clear()
                    capi.synchronize()
                    g.launch()
                    same(step, want, "replayed alone")
                graphs.append((stream, g, step, want))
    for first, second in ((0, 2), (1, 3)):
        for _ in range(3):
            for step in steps:
                step.clear()
            capi.synchronize()
            for stream, g, _, _ in (graphs[first], graphs[second]):
                with stream:
                    g.launch()
            steps[2].run()
            capi.synchronize()
            for at in (first, second):
                same(graphs[at][2], graphs[at][3], "replayed side by side")
