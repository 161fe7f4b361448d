"""The ops and modules whose weight depends on the row, through the drop-in (`recpulse_cuda`, `recpulse.module`) on the GPU.

Gradients are of loss = r . y . c with vectors r and c, so that every row and column has another gradient, against the formula's in
float64 and against differences.  Tolerances: an output's error is counted against the largest magnitude in it.  A chain here has at most
six products of at most 64 terms and a few roundings in the tensor type between them, so it is off by less than 6 (64 + 8) u + 24 h times
the products' magnitudes, with u the accumulate type's and h the tensor type's half step; the magnitudes' sum is within 8 times the
largest entry, the square root of 64 terms whose signs vary.
"""
import numpy as np
import pytest

import recpulse_cuda as rp
from recpulse.module import AdapterLinear, ExpertLinear, Linear, MixtureOfExperts, Module

pytestmark = pytest.mark.gpu
DTYPES = ["float32", "float64", "float16", "bfloat16"]
HALF_STEP = {"float32": 2.0 ** -24, "float64": 2.0 ** -53, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
UNIT = {"float32": 2.0 ** -24, "float64": 2.0 ** -52, "float16": 2.0 ** -24, "bfloat16": 2.0 ** -24}


def dev(arr, dtype="float64", grad=False):
    t = rp.from_numpy(np.ascontiguousarray(arr, dtype=np.float64 if dtype == "float64" else np.float32)).to(device="cuda", dtype=dtype)
    return t.requires_grad_(True) if grad else t


def host(t):
    return t.to(device="cpu", dtype="float64").to_numpy()


def close(got, want, dtype):
    assert got.shape == want.shape
    bound = 8 * (6 * 72 * UNIT[dtype] + 24 * HALF_STEP[dtype]) * np.max(np.abs(want), initial=0.0)
    assert np.max(np.abs(got - want), initial=0.0) <= bound


def weighed(y, r, c, dtype):
    return dev(r[None, :], dtype).op_matmul(y).op_matmul(dev(c[:, None], dtype)).op_sum_all()


def difference(fn, arrays, at, eps=1e-5):
    """Central differences of fn by arrays[at] at some of its entries: (flat indexes, values)."""
    flat = np.linspace(0, arrays[at].size - 1, 12).astype(int)
    out = []
    for i in flat:
        moved = []
        for sign in (eps, -eps):
            copy = [a.copy() for a in arrays]
            copy[at].reshape(-1)[i] += sign
            moved.append(fn(copy))
        out.append((moved[0] - moved[1]) / (2 * eps))
    return flat, np.array(out)


def spread(rng, *shape):
    """Values that every dtype holds exactly."""
    return rng.integers(-64, 65, shape) / 32.0


def softmax_at(logits, experts, normalize):
    e = np.exp(logits - logits.max(1, keepdims=True))
    picked = np.take_along_axis(e, experts, 1)
    return picked / (picked if normalize else e).sum(1, keepdims=True)


# ---- routing ----
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("normalize", [True, False])
def test_route(normalize, dtype):
    rng = np.random.default_rng(1)
    logits = np.stack([rng.permutation(12) for _ in range(33)]) / 4.0
    x = dev(logits, dtype, grad=True)
    weights, routing = x.op_route(3, normalize)
    assert weights.shape == (33, 3) and weights.dtype == ("float64" if dtype == "float64" else "float32")
    assert (routing.tokens, routing.k, routing.groups) == (33, 3, 12)
    experts = np.argsort(-logits, 1)[:, :3]
    assert np.array_equal(routing.experts, experts)
    order = np.argsort(experts.reshape(-1), kind="stable")
    assert np.array_equal(routing.order, order) and np.array_equal(routing.position.reshape(-1)[order], np.arange(99))
    assert np.array_equal(routing.offsets, np.concatenate([[0], np.cumsum(np.bincount(experts.reshape(-1), minlength=12))]))
    wdt = weights.dtype
    close(host(weights), softmax_at(logits, experts, normalize), wdt)
    r, c = rng.normal(0, 1, 33), np.array([1.0, -2.0, 0.5])
    weighed(weights, r, c, wdt).backward()
    fn = lambda a: float(r @ softmax_at(a[0], experts, normalize) @ c)
    flat, want = difference(fn, [logits], 0)
    assert x.grad.dtype == dtype
    assert np.max(np.abs(host(x.grad).reshape(-1)[flat] - want)) <= max(1e-8, 4 * HALF_STEP[dtype], 200 * UNIT[dtype])   # differences: eps^2 and u / eps in float64


def test_group_rows():
    ids = [2, -1, 0, 2, 7, 1, 0]
    routing = rp.group_rows(ids, 3, "cuda")
    assert (routing.tokens, routing.k, routing.groups) == (7, 1, 3)
    assert np.array_equal(routing.offsets, [0, 2, 3, 5]) and np.array_equal(routing.order, [2, 6, 5, 0, 3, -1, -1])
    assert np.array_equal(routing.position[:, 0], [3, -1, 0, 4, -1, 2, 1])


# ---- exchange and grouped linear, a chain: dispatch, grouped linear, combine ----
def chain_want(x, w, b, weights, ids, out_rows):
    y = np.zeros((len(ids), w.shape[2]))
    for i, g in enumerate(ids):
        if 0 <= g < w.shape[0]:
            y[i] = weights[i, 0] * (x[i] @ w[g] + b[g])
    return y


@pytest.mark.parametrize("dtype", DTYPES)
def test_dispatch_grouped_linear_combine(dtype):
    rng = np.random.default_rng(2)
    rows, k, n, groups = 45, 40, 24, 5
    ids = rng.integers(-1, groups, rows)
    ids[ids == 3] = -1                                                        # a group without rows, and rows without a group
    assert (ids == -1).sum() > 5
    x, w, b, weights = spread(rng, rows, k), spread(rng, groups, k, n), spread(rng, groups, n), spread(rng, rows, 1)
    r, c = spread(rng, rows), spread(rng, n)
    wdt = "float64" if dtype == "float64" else "float32"
    routing = rp.group_rows(ids.tolist(), groups, "cuda")
    dx, dw, db, dweights = dev(x, dtype, True), dev(w, dtype, True), dev(b, dtype, True), dev(weights, wdt, True)
    y = dx.op_dispatch(routing).op_grouped_linear(dw, routing, db).op_combine(dweights, routing)
    assert y.shape == (rows, n) and y.dtype == dtype
    close(host(y), chain_want(x, w, b, weights, ids, rows), dtype)
    weighed(y, r, c, dtype).backward()
    dy = np.outer(r, c)
    want = [np.zeros_like(x), np.zeros_like(w), np.zeros_like(b), np.zeros_like(weights)]
    for i, g in enumerate(ids):
        if g < 0:
            continue
        want[0][i] = weights[i, 0] * (w[g] @ dy[i])
        want[1][g] += weights[i, 0] * np.outer(x[i], dy[i])
        want[2][g] += weights[i, 0] * dy[i]
        want[3][i, 0] = dy[i] @ (x[i] @ w[g] + b[g])
    for t, v in zip((dx, dw, db, dweights), want):
        close(host(t.grad), v, dtype)
    if dtype == "float64":
        fn = lambda a: float(r @ chain_want(*a, ids, rows) @ c)
        for at, t in enumerate((dx, dw, db, dweights)):
            flat, num = difference(fn, [x, w, b, weights], at)
            assert np.max(np.abs(host(t.grad).reshape(-1)[flat] - num)) <= 1e-5      # values to 1e3 with u / eps = 1e-11 each
    first = [host(t.grad) for t in (dx, dw, db, dweights)]
    again = dx.op_dispatch(routing).op_grouped_linear(dw, routing, db).op_combine(dweights, routing)
    weighed(again, r, c, dtype).backward()                                    # added to what is there, and the same bits
    for t, v in zip((dx, dw, db, dweights), first):
        assert np.array_equal(host(t.grad), 2 * v)


def test_rows_of_no_group_are_zero_in_ops():
    rng = np.random.default_rng(3)
    routing = rp.group_rows([-1, 1, -1, 0, -1], 2, "cuda")
    x = dev(rng.normal(0, 1, (5, 8)), "float32", True)
    w = dev(rng.normal(0, 1, (2, 8, 6)), "float32", True)
    for _ in range(3):                                                        # blocks of the pool that held other values
        rp.ones([5, 8], device="cuda"); rp.ones([5, 6], device="cuda")
        rows = x.op_dispatch(routing)
        y = rows.op_grouped_linear(w, routing)
        assert np.all(host(rows)[2:] == 0) and np.all(host(y)[2:] == 0)
        x.zero_grad()
        y.op_sum_all().backward()
        assert np.all(host(x.grad)[[0, 2, 4]] == 0) and np.all(host(x.grad)[[1, 3]] != 0)


def test_grouped_linear_strided_operands():
    rng = np.random.default_rng(4)
    routing = rp.group_rows([0, 0, 1, 1, 1], 2, "cuda")
    x, w = rng.normal(0, 1, (8, 5)), rng.normal(0, 1, (2, 6, 8))
    dx, dw = dev(x, grad=True), dev(w, grad=True)
    y = dx.transpose(0, 1).op_grouped_linear(dw.transpose(1, 2), routing)     # rows already in the order of their groups
    want = np.concatenate([x.T[:2] @ w[0].T, x.T[2:] @ w[1].T])
    close(host(y), want, "float64")
    y.op_sum_all().backward()
    ones = np.ones((5, 6))
    close(host(dx.grad), np.concatenate([ones[:2] @ w[0], ones[2:] @ w[1]]).T, "float64")
    close(host(dw.grad), np.stack([ones[:2].T @ x.T[:2], ones[2:].T @ x.T[2:]]), "float64")


# ---- adapters ----
def adapter_rows(ids, lengths, rows):
    out = np.full(rows, -1)
    out[:sum(lengths)] = np.repeat(ids, lengths)
    return out


def adapter_want(x, w, bias, a, b, scales, which):
    y = x @ w + bias
    for i, s in enumerate(which):
        if s >= 0:
            y[i] += scales[s] * (x[i] @ a[s]) @ b[s]
    return y


@pytest.mark.parametrize("dtype", DTYPES)
def test_adapter_linear(dtype):
    rng = np.random.default_rng(5)
    rows, k, n, rank, adapters = 50, 48, 40, 4, 3
    ids, lengths = [2, -1, 0, 2, 0], [7, 5, 0, 20, 9]                         # an adapter twice, one that none uses, an empty segment, rows behind the last
    which = adapter_rows(ids, lengths, rows)
    scales = [0.5, 2.0, -1.0]
    arrays = [spread(rng, rows, k), spread(rng, k, n), spread(rng, n), spread(rng, adapters, k, rank), spread(rng, adapters, rank, n)]
    x, w, bias, a, b = (dev(v, dtype, True) for v in arrays)
    y = x.op_adapter_linear(w, a, b, ids, lengths, bias, scales)
    close(host(y), adapter_want(*arrays, scales, which), dtype)
    r, c = spread(rng, rows), spread(rng, n)
    weighed(y, r, c, dtype).backward()
    vx, vw, _, va, vb = arrays
    dy = np.outer(r, c)
    want = [dy @ vw.T, vx.T @ dy, dy.sum(0), np.zeros_like(va), np.zeros_like(vb)]
    for i, s in enumerate(which):
        if s >= 0:
            want[0][i] += scales[s] * (dy[i] @ vb[s].T) @ va[s].T
            want[3][s] += scales[s] * np.outer(vx[i], dy[i] @ vb[s].T)
            want[4][s] += scales[s] * np.outer(vx[i] @ va[s], dy[i])
    for t, v in zip((x, w, bias, a, b), want):
        close(host(t.grad), v, dtype)
    if dtype == "float64":
        fn = lambda v: float(r @ adapter_want(*v, scales, which) @ c)
        for at, t in enumerate((x, w, bias, a, b)):
            flat, num = difference(fn, arrays, at)
            assert np.max(np.abs(host(t.grad).reshape(-1)[flat] - num)) <= 1e-4      # values to 1e5 with u / eps = 1e-11 each
    only = dev(vx, dtype, True)                                               # no gradient but x's, no bias, scales of one
    y = only.op_adapter_linear(dev(vw, dtype), dev(va, dtype), dev(vb, dtype), ids, lengths)
    close(host(y), adapter_want(vx, vw, 0, va, vb, [1, 1, 1], which), dtype)
    y.op_sum_all().backward()
    assert only.has_grad


def test_adapter_linear_refusals():
    x, w, a, b = (dev(np.ones(s)) for s in ((6, 4), (4, 5), (2, 4, 3), (2, 3, 5)))
    bad = [(dict(ids=[0], lengths=[7]), "longer than the 6 rows"), (dict(ids=[2], lengths=[6]), "below 2"), (dict(ids=[-2], lengths=[6]), "below 2"),
           (dict(ids=[0, 1], lengths=[6]), "one length for each segment"), (dict(ids=[0], lengths=[-1]), "not negative"),
           (dict(ids=[], lengths=[]), "at least one segment"), (dict(ids=[0], lengths=[6], scales=[1.0]), "one scale for each adapter")]
    for kw, word in bad:
        with pytest.raises(RuntimeError, match=word):
            x.op_adapter_linear(w, a, b, **kw)
    with pytest.raises(RuntimeError, match="of x's dtype and device"):
        x.op_adapter_linear(w, b, a, ids=[0], lengths=[6])


def test_routed_refusals():
    routing = rp.group_rows([0, 1, 1], 2, "cuda")
    x, w = dev(np.ones((3, 4))), dev(np.ones((2, 4, 5)))
    for call, word in ((lambda: dev(np.ones((4, 4))).op_dispatch(routing), "3 rows"), (lambda: x.op_combine(dev(np.ones((3, 2))), routing), "weights"),
                       (lambda: x.op_combine(dev(np.ones((3, 1)), "float32"), routing), "weights"), (lambda: x.op_grouped_linear(dev(np.ones((3, 4, 5))), routing), "groups"),
                       (lambda: x.op_grouped_linear(w, routing, dev(np.ones((2, 4)))), "bias"), (lambda: x.op_route(5), "4 experts"), (lambda: x.op_route(0), "4 experts"),
                       (lambda: rp.group_rows([], 2, "cuda"), "at least one row"), (lambda: rp.group_rows([0], 2000, "cuda"), "1024 groups")):
        with pytest.raises(RuntimeError, match=word):
            call()


# ---- modules ----
def test_modules():
    moe = MixtureOfExperts(16, 32, 6, 2)
    assert sorted(moe.tracked) == ["down.bias", "down.weight", "router.weight", "up.bias", "up.weight"]
    assert moe.up.weight.shape == (6, 16, 32) and moe.down.bias.shape == (6, 16) and len(moe.parameters()) == 5
    layer = AdapterLinear(16, 8, 3, 2)
    assert sorted(layer.learnable()) == ["a", "b"] and sorted(layer.frozen()) == ["bias", "weight"]
    layer.to(device="cuda")
    x = dev(np.ones((5, 16)), "float32")
    plain = x.op_linear(layer.weight, layer.bias)
    assert np.array_equal(host(layer(x, [1], [5])), host(plain))              # an untrained adapter changes nothing
    assert ExpertLinear(2, 3, 4, bias=False).bias is None


@pytest.mark.parametrize("normalize", [True, False])
def test_mixture_of_experts(normalize):
    """A network: a linear layer, the mixture, a layer with adapters; values and every gradient in float64."""
    class Net(Module):
        def __init__(self):
            super().__init__()
            self.first = Linear(12, 16)
            self.mix = MixtureOfExperts(16, 24, 5, 2, normalize)
            self.last = AdapterLinear(16, 8, 2, 3, scale=0.5, train_shared=True)

        def forward(self, x):
            return self.last(self.mix(self.first(x)), [1, 0, -1], [20, 10, 4])

    rp.manual_seed(7)
    rng = np.random.default_rng(7)
    net = Net().to(device="cuda", dtype="float64")
    names = sorted(net.tracked)
    shapes = {name: net.tracked[name].shape for name in names}
    values = {name: rng.normal(0, 0.4, shapes[name]) for name in names}
    net.load_state({name: dev(values[name]) for name in names})
    x = rng.normal(0, 1, (40, 12))
    which = adapter_rows([1, 0, -1], [20, 10, 4], 40)
    r, c = rng.normal(0, 1, 40), rng.normal(0, 1, 8)

    def want(arrays):
        v = dict(zip(names, arrays))
        h = x @ v["first.weight"] + v["first.bias"]
        logits = h @ v["mix.router.weight"]
        experts = np.argsort(-logits, 1)[:, :2]
        weights = softmax_at(logits, experts, normalize)
        y = np.zeros_like(h)
        for t in range(40):
            for j, e in enumerate(experts[t]):
                y[t] += weights[t, j] * (np.maximum(h[t] @ v["mix.up.weight"][e] + v["mix.up.bias"][e], 0) @ v["mix.down.weight"][e] + v["mix.down.bias"][e])
        return adapter_want(y, v["last.weight"], v["last.bias"], v["last.a"], v["last.b"], [0.5, 0.5], which)

    arrays = [values[name] for name in names]
    y = net(dev(x))
    close(host(y), want(arrays), "float64")
    weighed(y, r, c, "float64").backward()
    scale = float(np.abs(want(arrays)).max())
    for at, name in enumerate(names):
        flat, num = difference(lambda a: float(r @ want(a) @ c), arrays, at, eps=1e-6)
        got = host(net.tracked[name].grad).reshape(-1)[flat]
        # third derivatives times eps^2 / 6 = 2e-13 and u / eps = 1e-10 of a sum of 320 values; 1e-6 leaves both far behind
        assert np.max(np.abs(got - num)) <= 1e-6 * max(1.0, scale, np.abs(num).max()), name


def test_training_steps_run():
    rng = np.random.default_rng(8)
    moe = MixtureOfExperts(32, 64, 8, 2).to(device="cuda", dtype="bfloat16")
    x = dev(rng.normal(0, 1, (100, 32)), "bfloat16")
    for _ in range(3):
        moe.zero_grad()
        moe(x).op_mean_all().backward()
        assert all(np.all(np.isfinite(host(p.grad))) and p.grad.shape == p.shape for p in moe.parameters())
