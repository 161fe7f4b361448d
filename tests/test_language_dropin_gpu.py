"""Layer norm, gated layers, the loss of a large vocabulary and distillation through the drop-in: values, gradients, refusals, and all of them in one training step."""
import numpy as np
import pytest

import recpulse_cuda as rp
from langhelp import GATES, distill_reference, gate_reference, norm_reference, vocab_reference
from recpulse.module import GatedFeedForward, LayerNorm, Linear, LinearCrossEntropy

pytestmark = pytest.mark.gpu
DTYPES = ["float64", "float32", "float16", "bfloat16"]
HALF_STEP = {"float64": 2.0 ** -53, "float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
UNIT = {"float64": 2.0 ** -53, "float32": 2.0 ** -24, "float16": 2.0 ** -24, "bfloat16": 2.0 ** -24}


def dev(arr, dtype="float64", grad=False):
    t = rp.from_numpy(np.ascontiguousarray(arr, dtype=np.float64)).to(device="cuda", dtype=dtype)
    return t.requires_grad_(True) if grad else t


def host(t):
    return t.to(device="cpu", dtype="float64").to_numpy()


def spread(rng, *shape):
    """Values that every dtype holds exactly."""
    return rng.integers(-64, 65, shape) / 32.0


def close(got, want, dtype, terms):
    """Against the largest value: `terms` products or sums in the accumulate type, and six roundings to the dtype on the way."""
    assert got.shape == want.shape
    bound = (8 * terms * UNIT[dtype] + 6 * HALF_STEP[dtype]) * np.max(np.abs(want))
    assert np.max(np.abs(got - want)) <= bound, (np.max(np.abs(got - want)), bound)


def weighed(y, c, dtype):
    """sum of y c as a scalar: the diagonal of products with c's columns, one at a time."""
    rows, cols = y.shape
    total = None
    for i in range(rows):
        part = y.slice([i, 0], [i + 1, cols]).op_matmul(dev(c[i][:, None], dtype)).op_sum_all()
        total = part if total is None else total.op_add(part)
    return total


def gate_and_gradients(x, w, bias, gate, c):
    n = w.shape[1] // 2
    z = x @ w + bias
    act, slope = gate_reference(z[:, :n], gate)
    dz = np.concatenate([c * z[:, n:] * slope, c * act], 1)
    return act * z[:, n:], dz @ w.T, x.T @ dz, dz.sum(0)


def norm_gradients(x, w, c, eps):
    mean, r, h, _ = norm_reference(x, w, None, eps)
    g = c * w
    return r * (g - g.mean(1, keepdims=True) - h * (g * h).mean(1, keepdims=True)), (c * h).sum(0), c.sum(0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_layer_norm(dtype):
    rng = np.random.default_rng(1)
    x, w, b, c = spread(rng, 5, 24), spread(rng, 24), spread(rng, 24), spread(rng, 5, 24)
    xd, wd, bd = dev(x, dtype, True), dev(w, dtype, True), dev(b, dtype, True)
    y = xd.op_layer_norm(wd, bd, 1e-3)
    close(host(y), norm_reference(x, w, b, 1e-3)[3], dtype, 40)
    weighed(y, c, dtype).backward()
    for t, want in zip((xd, wd, bd), norm_gradients(x, w, c, 1e-3)):
        close(host(t.grad), want, dtype, 80)
    bare = dev(x, dtype, True)
    y = bare.op_layer_norm()
    weighed(y, c, dtype).backward()
    close(host(bare.grad), norm_gradients(x, np.ones(24), c, 1e-5)[0], dtype, 80)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gate", sorted(GATES))
def test_gated_linear(gate, dtype):
    rng = np.random.default_rng(2)
    x, w, bias, c = spread(rng, 6, 20), spread(rng, 20, 32) / 4, spread(rng, 32), spread(rng, 6, 16)
    xd, wd, bd = dev(x, dtype, True), dev(w, dtype, True), dev(bias, dtype, True)
    y = xd.op_gated_linear(wd, bd, gate)
    want = gate_and_gradients(x, w, bias, gate, c)
    close(host(y), want[0], dtype, 60)
    weighed(y, c, dtype).backward()
    for t, v in zip((xd, wd, bd), want[1:]):
        close(host(t.grad), v, dtype, 120)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
def test_linear_cross_entropy(reduction, dtype):
    rng = np.random.default_rng(3)
    x, w, bias, targets = spread(rng, 7, 16), spread(rng, 16, 40) / 2, spread(rng, 40), [3, -1, 0, 39, 12, -1, 3]
    red = {"none": 0, "mean": 1, "sum": 2}[reduction]
    xd, wd, bd = dev(x, dtype, True), dev(w, dtype, True), dev(bias, dtype, True)
    loss = xd.op_linear_cross_entropy(wd, targets, bd, reduction)
    acc = "float64" if dtype == "float64" else "float32"
    assert loss.dtype == acc and loss.shape == ((7,) if red == 0 else (1,))
    want, _, d, _, _ = vocab_reference(x, w, bias, np.array(targets), red, 1.0)
    close(host(loss), want, acc, 200)
    loss.backward()                                             # (for 'none' of ones, one for each row)
    for t, v in zip((xd, wd, bd), (d @ w.T, x.T @ d, d.sum(0))):
        close(host(t.grad), v, dtype, 200)


def test_a_transposed_weight():
    """The embedding's rows as the last projection's columns: a view, and its gradient comes back through it."""
    rng = np.random.default_rng(4)
    x, table, targets = spread(rng, 9, 24), spread(rng, 50, 24) / 4, rng.integers(0, 50, 9)
    for dtype in DTYPES:
        xd, td = dev(x, dtype, True), dev(table, dtype, True)
        loss = xd.op_linear_cross_entropy(td.T, targets.tolist())
        want, _, d, _, _ = vocab_reference(x, table.T, None, targets, 1, 1.0)
        loss.backward()
        close(host(xd.grad), d @ table, dtype, 200)
        close(host(td.grad), d.T @ x, dtype, 200)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
def test_distillation_loss(reduction, dtype):
    rng = np.random.default_rng(5)
    logits, teacher = spread(rng, 5, 30), spread(rng, 5, 4)
    ids = np.stack([rng.choice(30, 4, replace=False) for _ in range(5)])
    ids[1] = -1
    red = {"none": 0, "mean": 1, "sum": 2}[reduction]
    xd, td = dev(logits, dtype, True), dev(teacher, dtype, True)
    loss = xd.op_distillation_loss(ids.tolist(), td, 2.0, reduction)
    want, grad, _, _, _ = distill_reference(logits, ids, teacher, 2.0, red, 1.0)
    close(host(loss), want, "float64" if dtype == "float64" else "float32", 200)
    loss.backward()
    close(host(xd.grad), grad, dtype, 200)
    assert not td.has_grad


def test_a_second_backward_adds():
    rng = np.random.default_rng(6)
    x, w, targets = spread(rng, 40, 16), spread(rng, 16, 64) / 4, rng.integers(0, 64, 40)
    for dtype in DTYPES:
        xd, wd = dev(x, dtype, True), dev(w, dtype, True)
        for _ in range(2):
            xd.op_linear_cross_entropy(wd, targets.tolist()).backward()
        _, _, d, _, _ = vocab_reference(x, w, None, targets, 1, 1.0)
        close(host(xd.grad), 2 * d @ w.T, dtype, 200)
        close(host(wd.grad), 2 * x.T @ d, dtype, 200)


def test_refusals():
    x, w = dev(np.ones((4, 6))), dev(np.ones((6, 8)))
    with pytest.raises(RuntimeError, match="weight \\[in_features"):
        x.op_gated_linear(dev(np.ones((5, 8))))
    with pytest.raises(RuntimeError, match="weight \\[in_features"):
        x.op_gated_linear(dev(np.ones((6, 7))))
    with pytest.raises(RuntimeError, match="dense vector of 8"):
        x.op_gated_linear(w, dev(np.ones(4)))
    with pytest.raises(RuntimeError, match="dense vector of 6"):
        x.op_layer_norm(dev(np.ones(5)))
    with pytest.raises(RuntimeError, match="eps"):
        x.op_layer_norm(eps=-1.0)
    with pytest.raises(RuntimeError, match="target out of range"):
        x.op_linear_cross_entropy(w, [0, 8, 0, 0])
    with pytest.raises(RuntimeError, match="target out of range"):
        x.op_linear_cross_entropy(w, [0, -2, 0, 0])
    with pytest.raises(RuntimeError, match="one target for each"):
        x.op_linear_cross_entropy(w, [0, 1, 2])
    with pytest.raises(RuntimeError, match="of x's dtype"):
        x.op_linear_cross_entropy(dev(np.ones((6, 8)), "float32"), [0, 1, 2, 3])
    with pytest.raises(RuntimeError, match="class out of range"):
        x.op_distillation_loss([[6]] * 4, dev(np.ones((4, 1))))
    with pytest.raises(RuntimeError, match="temperature"):
        x.op_distillation_loss([[0]] * 4, dev(np.ones((4, 1))), 0.0)
    with pytest.raises(RuntimeError, match="teacher \\[rows"):
        x.op_distillation_loss([[0]] * 3, dev(np.ones((3, 1))))


# ---- one step of a small language model: norm, gated block with a residual, norm, the vocabulary's loss, and the same logits against a teacher ----

def parameters(rng, features, hidden, classes):
    return {"first.weight": 1 + 0.1 * rng.normal(size=features), "first.bias": 0.1 * rng.normal(size=features), "up.weight": rng.normal(0, features ** -0.5, size=(features, 2 * hidden)),
            "up.bias": 0.1 * rng.normal(size=2 * hidden), "down.weight": rng.normal(0, hidden ** -0.5, size=(hidden, features)), "down.bias": 0.1 * rng.normal(size=features),
            "last.weight": 1 + 0.1 * rng.normal(size=features), "last.bias": 0.1 * rng.normal(size=features), "head.weight": rng.normal(0, features ** -0.5, size=(features, classes)),
            "head.bias": 0.1 * rng.normal(size=classes)}


def reference_step(p, x, targets, ids, teacher):
    h = norm_reference(x, p["first.weight"], p["first.bias"], 1e-5)[3]
    z = h @ p["up.weight"] + p["up.bias"]
    n = z.shape[1] // 2
    y = x + (gate_reference(z[:, :n], "silu")[0] * z[:, n:]) @ p["down.weight"] + p["down.bias"]
    out = norm_reference(y, p["last.weight"], p["last.bias"], 1e-5)[3]
    logits = out @ p["head.weight"] + p["head.bias"]
    hard = vocab_reference(out, p["head.weight"], p["head.bias"], targets, 1, 1.0)[0][0]
    return hard + distill_reference(logits, ids, teacher, 2.0, 1, 1.0)[0][0]


class Model:
    def __init__(self, p, dtype, features, hidden, classes):
        self.first, self.block, self.last, self.head, self.loss = LayerNorm(features), GatedFeedForward(features, hidden), LayerNorm(features), Linear(features, classes), LinearCrossEntropy(features, classes)
        self.tensors = {name: dev(v, dtype, True) for name, v in p.items()}
        t = self.tensors
        self.first.weight, self.first.bias, self.last.weight, self.last.bias = t["first.weight"], t["first.bias"], t["last.weight"], t["last.bias"]
        self.block.up.weight, self.block.up.bias, self.block.down.weight, self.block.down.bias = t["up.weight"], t["up.bias"], t["down.weight"], t["down.bias"]
        self.head.weight, self.head.bias, self.loss.weight, self.loss.bias = t["head.weight"], t["head.bias"], t["head.weight"], t["head.bias"]

    def step(self, x, targets, ids, teacher):
        y = x.op_add(self.block(self.first(x)))
        out = self.last(y)
        hard = self.loss(out, targets)
        soft = self.head(out).op_distillation_loss(ids, teacher, 2.0)
        total = hard.op_add(soft)
        total.backward()
        return total


def test_training_step_agrees_with_differences():
    rng = np.random.default_rng(7)
    rows, features, hidden, classes = 6, 12, 10, 18
    p = parameters(rng, features, hidden, classes)
    x, teacher, targets = rng.normal(size=(rows, features)), rng.normal(size=(rows, 3)), np.array([0, 17, -1, 4, 4, 9])
    ids = np.stack([rng.choice(classes, 3, replace=False) for _ in range(rows)])
    model, xd = Model(p, "float64", features, hidden, classes), dev(x, "float64", True)
    total = model.step(xd, targets.tolist(), ids.tolist(), dev(teacher))
    assert abs(host(total)[0] - reference_step(p, x, targets, ids, teacher)) < 1e-11
    for name in list(p) + ["x"]:
        array = x if name == "x" else p[name]
        got = host(xd.grad if name == "x" else model.tensors[name].grad).reshape(-1)
        for i in np.linspace(0, array.size - 1, 5).astype(int):
            value = []
            for sign in (1e-5, -1e-5):
                moved = array.copy()
                moved.reshape(-1)[i] += sign
                value.append(reference_step({**p, **({} if name == "x" else {name: moved})}, moved if name == "x" else x, targets, ids, teacher))
            # (third derivatives below 100: step^2 / 6 of them, and 1e-15 / step)
            assert abs((value[0] - value[1]) / 2e-5 - got[i]) < 3e-8, name


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_training_step_in_few_bits(dtype):
    """The same step at sizes that the tiled kernels take, its gradients beside those in 64 bits: about a dozen roundings lie between them, each of at most half a step of a value of the size of its row."""
    rng = np.random.default_rng(8)
    rows, features, hidden, classes = 192, 128, 256, 1000
    p = parameters(rng, features, hidden, classes)
    x, teacher, targets = rng.normal(size=(rows, features)), rng.normal(size=(rows, 8)), rng.integers(-1, classes, rows)
    ids = np.stack([rng.choice(classes, 8, replace=False) for _ in range(rows)])
    results = {}
    for dt in ("float64", dtype):
        as_is = {k: host(dev(v, dtype)) for k, v in p.items()}      # both from the same numbers
        xd, td = dev(host(dev(x, dtype)), dt, True), dev(host(dev(teacher, dtype)), dt)
        model = Model(as_is, dt, features, hidden, classes)
        total = model.step(xd, targets.tolist(), ids.tolist(), td)
        results[dt] = {"total": host(total), "x": host(xd.grad), **{k: host(t.grad) for k, t in model.tensors.items()}}
    for name, want in results["float64"].items():
        off = np.linalg.norm(results[dtype][name] - want) / np.linalg.norm(want)
        assert off <= 12 * HALF_STEP[dtype] + 2000 * UNIT[dtype], (name, off)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_one_tensor_as_several_inputs(dtype):
    """... whose gradients add up, those of a second pass to those of the first."""
    rng = np.random.default_rng(11)
    x, w = spread(rng, 300, 24), spread(rng, 24)
    xd, wd = dev(x, dtype), dev(w, dtype, True)
    for _ in range(2):
        xd.op_layer_norm(wd, wd, 1e-3).op_sum_all().backward()
    _, dw, db = norm_gradients(x, w, np.ones((300, 24)), 1e-3)
    close(host(wd.grad), 2 * (dw + db), dtype, 400)
    k = 544
    x = spread(rng, k, k) / 16
    xd = dev(x, dtype, True)
    for _ in range(2):
        xd.op_gated_linear(xd, None, "sigmoid").op_sum_all().backward()
    _, dx, dw, _ = gate_and_gradients(x, x, np.zeros(k), "sigmoid", np.ones((k, k // 2)))
    close(host(xd.grad), 2 * (dx + dw), dtype, 2 * k)
