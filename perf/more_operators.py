"""What stands around the products of a language model, as cases for timing and for comparing results: layer norm, the gated
linear layer, the cross entropy of a large vocabulary from the hidden rows, and distillation from a teacher's top logits.

A case is a dict of plain values with an "op" and its sizes; `listed()` holds the fixed ones, `draw(rng)` makes others of
the same ranges.  With `own` false `run` computes plain torch operations in float32, with `own` true it calls the C ABI
through `recpulse_amd.capi` on the same tensors.

  norm      y = (x - mean) / sqrt(variance + eps) w + b of each row; with backward dx, dw and db.
  gated     h = act(x.Wg + bg) (x.Wu + bu) with W = [Wg | Wu]; with backward dx, dW and db.
  vocab     mean over the rows with a target of log sum exp(x.W + b) - (x.W + b)[target]; with backward dx, dW and db.
  distill   mean over the rows of T^2 sum p (log p - log q) with p the teacher's softmax among its entries and q the
            student's among all classes, both at temperature T; with backward the gradient of the student's logits.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
CODES = {"f32": 0, "f16": 2, "bf16": 3}                      # recpulse_amd.capi's dtype codes
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
GATES = {"silu": 0, "gelu": 1, "gelu_tanh": 2, "relu": 3, "sigmoid": 4}
EPS = 1e-5
MOST_FLOPS = 6 * 8192 * 4096 * 32768                         # of the largest listed case


def listed():
    return [
        # one decoding step of a few requests: nothing but latency
        dict(name="norm-decode", op="norm", dtype="bf16", rows=16, width=4096, affine=True, backward=False),
        # rows that come from data, in float32
        dict(name="norm-odd", op="norm", dtype="f32", rows=1999, width=1031, affine=True, backward=True),
        # a training step's batch
        dict(name="norm-train", op="norm", dtype="bf16", rows=16384, width=4096, affine=True, backward=True),
        # decoding: the weights are read once
        dict(name="gated-decode", op="gated", dtype="bf16", rows=16, inner=4096, hidden=8192, act="silu", bias=False, backward=False),
        # training, sizes that come from data
        dict(name="gated-odd", op="gated", dtype="f16", rows=1999, inner=519, hidden=1031, act="gelu", bias=True, backward=True),
        # training
        dict(name="gated-train", op="gated", dtype="bf16", rows=8192, inner=4096, hidden=8192, act="silu", bias=False, backward=True),
        # scoring the continuations of a prompt: few rows, the weights are read once
        dict(name="vocab-score", op="vocab", dtype="bf16", rows=64, inner=4096, classes=32768, bias=False, tied=False, without=0, backward=False),
        # fine-tuning, a vocabulary of odd size, the embedding's rows as weights, one row in eight without a target
        dict(name="vocab-odd", op="vocab", dtype="f16", rows=1000, inner=520, classes=10007, bias=True, tied=True, without=8, backward=True),
        # training, the largest
        dict(name="vocab-train", op="vocab", dtype="bf16", rows=8192, inner=4096, classes=32768, bias=False, tied=False, without=0, backward=True),
        # the framework's small classifier against a larger one, in float32
        dict(name="distill-small", op="distill", dtype="f32", rows=256, classes=1000, k=10, temperature=2.0, padded=False, backward=True),
        # scoring a student on rows of odd length, one in eight padding
        dict(name="distill-odd", op="distill", dtype="f16", rows=777, classes=50021, k=20, temperature=1.0, padded=True, backward=False),
        # training
        dict(name="distill-train", op="distill", dtype="bf16", rows=4096, classes=65536, k=64, temperature=1.5, padded=False, backward=True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _width(rng, low, high):
    """A width: mostly whole vectors, now and then any number."""
    n = _log(rng, low, high)
    unit = rng.choice([1, 8, 64])
    return max(low, min(high, n // unit * unit))


def draw(rng):
    op = rng.choice(["norm", "gated", "vocab", "distill"])
    backward = rng.random() < 0.6
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "norm":
        return dict(op=op, dtype=dtype, rows=_log(rng, 1, 16384), width=_width(rng, 64, 8192), affine=rng.random() < 0.8, backward=backward)
    if op == "gated":
        return dict(op=op, dtype=dtype, rows=_log(rng, 1, 8192 if dtype != "f32" else 2048), inner=_width(rng, 64, 4096), hidden=_width(rng, 64, 8192),
                    act=rng.choice(sorted(GATES)), bias=rng.random() < 0.5, backward=backward)
    if op == "vocab":
        inner, classes = _width(rng, 64, 4096), _width(rng, 1000, 131072)
        most = MOST_FLOPS // (6 * inner * classes) // (8 if dtype == "f32" else 1)
        return dict(op=op, dtype=dtype, rows=_log(rng, 1, max(1, min(8192, most))), inner=inner, classes=classes, bias=rng.random() < 0.5, tied=rng.random() < 0.5,
                    without=rng.choice([0, 0, 2, 8]), backward=backward)
    classes = _width(rng, 100, 131072)
    return dict(op=op, dtype=dtype, rows=_log(rng, 1, min(8192, (1 << 28) // classes)), classes=classes, k=rng.randint(1, 64), temperature=rng.choice([1.0, 1.5, 2.0, 4.0]),
                padded=rng.random() < 0.3, backward=backward)


# ---- inputs ------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    c, t = dict(case), DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, dtype=t):
        out = torch.empty(*shape, device="cuda", dtype=dtype)
        return out.normal_(0.0, scale, generator=gen)

    def zeros(*shape, dtype=t):
        return torch.zeros(*shape, device="cuda", dtype=dtype)

    s = {"case": c, "code": CODES[case["dtype"]], "room": {}}
    if c["op"] == "norm":
        rows, width = c["rows"], c["width"]
        s["x"] = normal(rows, width) * (0.5 + torch.rand(rows, 1, device="cuda", generator=gen)).to(t) + normal(rows, 1)
        s["w"] = 1.0 + normal(width, scale=0.2) if c["affine"] else None
        s["b"] = normal(width, scale=0.2) if c["affine"] else None
        s["y"], s["stats"] = zeros(rows, width), zeros(rows, 2, dtype=torch.float32)
        if c["backward"]:
            s["grad_y"], s["grad_x"] = normal(rows, width), zeros(rows, width)
            s["grad_w"], s["grad_b"] = (zeros(width), zeros(width)) if c["affine"] else (None, None)
    elif c["op"] == "gated":
        rows, inner, hidden = c["rows"], c["inner"], c["hidden"]
        s["x"], s["w"] = normal(rows, inner), normal(inner, 2 * hidden, scale=inner ** -0.5)
        s["bias"] = normal(2 * hidden, scale=0.1) if c["bias"] else None
        s["h"] = zeros(rows, hidden)
        if c["backward"]:
            s["z"], s["grad_z"] = zeros(rows, 2 * hidden, dtype=torch.float32), zeros(rows, 2 * hidden)
            s["grad_h"], s["grad_x"], s["grad_w"] = normal(rows, hidden), zeros(rows, inner), zeros(inner, 2 * hidden)
            s["grad_bias"] = zeros(2 * hidden) if c["bias"] else None
    elif c["op"] == "vocab":
        rows, inner, classes = c["rows"], c["inner"], c["classes"]
        s["x"] = normal(rows, inner)
        table = normal(classes, inner, scale=2.0 * inner ** -0.5) if c["tied"] else normal(inner, classes, scale=2.0 * inner ** -0.5)
        s["w"] = table.t() if c["tied"] else table            # [inner, classes] either way
        s["bias"] = normal(classes, scale=0.5) if c["bias"] else None
        # frequent and rare words
        s["targets"] = (classes * torch.rand(rows, device="cuda", generator=gen) ** 3).int().clamp(max=classes - 1)
        if c["without"]:
            s["targets"][torch.rand(rows, device="cuda", generator=gen) < 1.0 / c["without"]] = -1
        s["loss"], s["stats"] = zeros(1, dtype=torch.float32), zeros(2 * rows + 1, dtype=torch.float32)
        if c["backward"]:
            s["upstream"] = zeros(1, dtype=torch.float32) + 64.0
            s["grad_x"] = zeros(rows, inner)
            s["grad_w"] = zeros(classes, inner).t() if c["tied"] else zeros(inner, classes)
            s["grad_bias"] = zeros(classes) if c["bias"] else None
    else:
        rows, classes, k = c["rows"], c["classes"], c["k"]
        s["logits"] = normal(rows, classes, scale=2.0)
        # the teacher's largest: no class twice
        start = torch.randint(0, classes, (rows, 1), device="cuda", generator=gen)
        s["ids"] = ((start + (classes // k) * torch.arange(k, device="cuda")) % classes).int()
        s["teacher"] = (normal(rows, k, scale=2.0, dtype=torch.float32) + 3.0).sort(1, descending=True).values.to(t)
        if c["padded"]:                                       # rows of padding, and lists that end early
            s["ids"][torch.rand(rows, device="cuda", generator=gen) < 0.125] = -1
            s["ids"][:, k // 2:][torch.rand(rows, device="cuda", generator=gen) < 0.125] = -1
        s["upstream"] = zeros(1, dtype=torch.float32) + float(rows)
        s["loss"], s["stats"] = zeros(1, dtype=torch.float32), zeros(3 * rows, dtype=torch.float32)
        s["grad_logits"] = zeros(rows, classes) if c["backward"] else None
    return s


# ---- the plain forms ---------------------------------------------------------------------------------------------

def _norm_plain(s, c):
    t, x = s["x"].dtype, s["x"].float()
    mean = x.mean(1, keepdim=True)
    r = torch.rsqrt(((x - mean) ** 2).mean(1, keepdim=True) + EPS)
    h = (x - mean) * r
    out = {"y": (h * s["w"].float() + s["b"].float() if c["affine"] else h).to(t)}
    if c["backward"]:
        dy = s["grad_y"].float()
        g = dy * s["w"].float() if c["affine"] else dy
        out["grad_x"] = (r * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True))).to(t)
        if c["affine"]:
            out["grad_w"], out["grad_b"] = (dy * h).sum(0).to(t), dy.sum(0).to(t)
    return out


def _gate(g, act):
    """act(g) and its derivative."""
    if act == "relu":
        return g.clamp(min=0.0), (g > 0).to(g.dtype)
    if act == "gelu":
        cdf = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
        return g * cdf, cdf + g * torch.exp(-0.5 * g * g) / math.sqrt(2.0 * math.pi)
    if act == "gelu_tanh":
        a = math.sqrt(2.0 / math.pi)
        th = torch.tanh(a * (g + 0.044715 * g ** 3))
        return 0.5 * g * (1.0 + th), 0.5 * (1.0 + th) + 0.5 * g * (1.0 - th * th) * a * (1.0 + 3.0 * 0.044715 * g * g)
    sig = 1.0 / (1.0 + torch.exp(-g))
    if act == "sigmoid":
        return sig, sig * (1.0 - sig)
    return g * sig, sig * (1.0 + g * (1.0 - sig))


def _gated_plain(s, c):
    t, n = s["x"].dtype, c["hidden"]
    x, w = s["x"].float(), s["w"].float()
    z = torch.mm(x, w)
    if c["bias"]:
        z = z + s["bias"].float()
    a, slope = _gate(z[:, :n], c["act"])
    out = {"h": (a * z[:, n:]).to(t)}
    if c["backward"]:
        dh = s["grad_h"].float()
        dz = torch.cat([dh * z[:, n:] * slope, dh * a], 1)
        out["grad_x"], out["grad_w"] = torch.mm(dz, w.t()).to(t), torch.mm(x.t(), dz).to(t)
        if c["bias"]:
            out["grad_bias"] = dz.sum(0).to(t)
    return out


def _vocab_plain(s, c):
    t = s["x"].dtype
    x, w = s["x"].float(), s["w"].float()
    z = torch.mm(x, w)
    if c["bias"]:
        z = z + s["bias"].float()
    there, target = s["targets"] >= 0, s["targets"].clamp(min=0).long()[:, None]
    most = z.max(1, keepdim=True).values
    e = torch.exp(z - most)
    total = e.sum(1, keepdim=True)
    loss = torch.where(there, (torch.log(total) + most - z.gather(1, target))[:, 0], 0.0)
    count = there.sum().clamp(min=1)
    out = {"loss": (loss.double().sum() / count).float().reshape(1)}
    if c["backward"]:
        d = e / total
        d.scatter_add_(1, target, torch.full_like(target, -1.0, dtype=torch.float32))
        d = d * torch.where(there, s["upstream"] / count, 0.0)[:, None]
        out["grad_x"], out["grad_w"] = torch.mm(d, w.t()).to(t), (torch.mm(d.t(), x).t() if c["tied"] else torch.mm(x.t(), d)).to(t)
        if c["bias"]:
            out["grad_bias"] = d.sum(0).to(t)
    return out


def _distill_plain(s, c):
    t, rows, scale = s["logits"].dtype, c["rows"], 1.0 / c["temperature"]
    z = s["logits"].float() * scale
    most = z.max(1, keepdim=True).values
    e = torch.exp(z - most)
    total = e.sum(1, keepdim=True)
    there, ids = s["ids"] >= 0, s["ids"].clamp(min=0).long()
    u = torch.where(there, s["teacher"].float() * scale, -math.inf)
    top = torch.where(there[:, :1], u.max(1, keepdim=True).values, 0.0)
    p = torch.exp(u - top)
    mass = p.sum(1, keepdim=True)
    some = mass > 0
    log_mass = torch.log(torch.where(some, mass, 1.0))
    p = p / torch.where(some, mass, 1.0)
    log_ratio = torch.where(there, u - top - log_mass, 0.0) - (z.gather(1, ids) - most - torch.log(total))
    loss = (p * log_ratio).sum(1) * c["temperature"] ** 2
    out = {"loss": (loss.double().sum() / rows).float().reshape(1)}
    if c["backward"]:
        d = torch.where(some, e / total, 0.0)
        d.scatter_add_(1, ids, -p)
        out["grad_logits"] = (d * (c["temperature"] / rows * s["upstream"])).to(t)
    return out


# ---- the framework's calls -----------------------------------------------------------------------------------------

def _at(tensor):
    return None if tensor is None else tensor.data_ptr()


def _room(s, name, size):
    """Room for what a call leaves between its launches, kept with the state as a training program keeps it."""
    if name not in s["room"]:
        s["room"][name] = torch.empty(max(1, size), device="cuda", dtype=torch.uint8)
    return s["room"][name].data_ptr()


def _own(s, c):
    from recpulse_amd import capi
    lib, code = capi.lib(), s["code"]
    lib.rp_hip_set_stream(torch.cuda.current_stream().cuda_stream)
    if c["op"] == "norm":
        rows, width = c["rows"], c["width"]
        capi.check(lib.rp_hip_layer_norm_forward(_at(s["y"]), _at(s["stats"]) if c["backward"] else None, _at(s["x"]), _at(s["w"]), _at(s["b"]), rows, width, width, width,
                                                 EPS, code), "rp_hip_layer_norm_forward")
        out = {"y": s["y"]}
        if c["backward"]:
            room = _room(s, "norm", lib.rp_hip_layer_norm_workspace(rows, width, code)) if c["affine"] else None
            capi.check(lib.rp_hip_layer_norm_backward(_at(s["grad_x"]), _at(s["grad_w"]), _at(s["grad_b"]), _at(s["grad_y"]), _at(s["x"]), _at(s["w"]), _at(s["stats"]), room,
                                                      rows, width, width, width, width, 0, 0, 0, code), "rp_hip_layer_norm_backward")
            out["grad_x"] = s["grad_x"]
            if c["affine"]:
                out.update(grad_w=s["grad_w"], grad_b=s["grad_b"])
        return out
    if c["op"] == "gated":
        rows, inner, hidden, gate = c["rows"], c["inner"], c["hidden"], GATES[c["act"]]
        capi.check(lib.rp_hip_gated_linear_forward(_at(s["h"]), _at(s["z"]) if c["backward"] else None, _at(s["x"]), _at(s["w"]), _at(s["bias"]), rows, inner, hidden, gate,
                                                   inner, 1, 2 * hidden, 1, hidden, code), "rp_hip_gated_linear_forward")
        out = {"h": s["h"]}
        if c["backward"]:
            capi.check(lib.rp_hip_gated_linear_backward(_at(s["grad_x"]), _at(s["grad_w"]), _at(s["grad_bias"]), _at(s["grad_z"]), _at(s["grad_h"]), _at(s["z"]), _at(s["x"]),
                                                        _at(s["w"]), rows, inner, hidden, gate, hidden, inner, 1, 2 * hidden, 1, inner, 2 * hidden, 1, 0, 0, 0, code),
                       "rp_hip_gated_linear_backward")
            out.update(grad_x=s["grad_x"], grad_w=s["grad_w"])
            if c["bias"]:
                out["grad_bias"] = s["grad_bias"]
        return out
    if c["op"] == "vocab":
        rows, inner, classes, lies = c["rows"], c["inner"], c["classes"], s["w"].stride()
        room = _room(s, "vocab", lib.rp_hip_linear_cross_entropy_workspace(rows, inner, classes, int(c["backward"]), code))
        capi.check(lib.rp_hip_linear_cross_entropy_forward(_at(s["loss"]), _at(s["stats"]), _at(s["x"]), _at(s["w"]), _at(s["bias"]), _at(s["targets"]), room,
                                                           rows, inner, classes, 1, inner, 1, *lies, code), "rp_hip_linear_cross_entropy_forward")
        out = {"loss": s["loss"]}
        if c["backward"]:
            capi.check(lib.rp_hip_linear_cross_entropy_backward(_at(s["grad_x"]), _at(s["grad_w"]), _at(s["grad_bias"]), _at(s["x"]), _at(s["w"]), _at(s["bias"]), _at(s["targets"]),
                                                                _at(s["stats"]), _at(s["upstream"]), room, rows, inner, classes, 1, inner, 1, *lies,
                                                                inner, *s["grad_w"].stride(), 0, 0, 0, code), "rp_hip_linear_cross_entropy_backward")
            out.update(grad_x=s["grad_x"], grad_w=s["grad_w"])
            if c["bias"]:
                out["grad_bias"] = s["grad_bias"]
        return out
    capi.check(lib.rp_hip_distillation_forward(_at(s["loss"]), _at(s["grad_logits"]), _at(s["stats"]), _at(s["logits"]), _at(s["ids"]), _at(s["teacher"]), _at(s["upstream"]),
                                               c["rows"], c["classes"], c["k"], c["classes"], c["temperature"], 1, code), "rp_hip_distillation_forward")
    out = {"loss": s["loss"]}
    if c["backward"]:
        out["grad_logits"] = s["grad_logits"]
    return out


def run(s):
    c = s["case"]
    if own:
        return _own(s, c)
    return {"norm": _norm_plain, "gated": _gated_plain, "vocab": _vocab_plain, "distill": _distill_plain}[c["op"]](s, c)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------

def work(c):
    es, ways = SIZE[c["dtype"]], 3 if c["backward"] else 1
    if c["op"] == "norm":
        cells, columns = c["rows"] * c["width"], c["width"] * (2 if c["affine"] else 0)
        return {"bytes": es * ((4 if c["backward"] else 2) * cells + (2 if c["backward"] else 1) * columns), "flops": (20 if c["backward"] else 8) * cells}
    if c["op"] == "gated":
        rows, inner, hidden = c["rows"], c["inner"], c["hidden"]
        data = rows * (inner + hidden) + 2 * inner * hidden
        return {"bytes": es * data * (2 if c["backward"] else 1), "flops": 4 * rows * inner * hidden * ways}
    if c["op"] == "vocab":
        rows, inner, classes = c["rows"], c["inner"], c["classes"]
        data = rows * inner + inner * classes
        return {"bytes": es * data * (2 if c["backward"] else 1) + 4 * rows, "flops": 2 * rows * inner * classes * ways}
    cells = c["rows"] * c["classes"]
    return {"bytes": es * cells * (2 if c["backward"] else 1) + c["rows"] * c["k"] * (es + 4), "flops": 6 * cells}


# ---- from the definitions, in 64 bits --------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    c, back = s["case"], case["backward"]
    if c["op"] == "norm":
        x = s["x"].double()
        var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
        h = (x - mean) / torch.sqrt(var + EPS)
        w = s["w"].double() if c["affine"] else torch.ones(c["width"], device="cuda", dtype=torch.float64)
        out = {"y": h * w + (s["b"].double() if c["affine"] else 0.0)}
        if back:
            dy = s["grad_y"].double()
            g, n = dy * w, c["width"]
            # h is orthogonal to ones and of squared length n var / (var + eps)
            out["grad_x"] = (g - g.sum(1, keepdim=True) / n - h * ((g * h).sum(1, keepdim=True) / n)) / torch.sqrt(var + EPS)
            if c["affine"]:
                out["grad_w"], out["grad_b"] = (dy * h).sum(0), dy.sum(0)
        return out
    if c["op"] == "gated":
        x, w, n = s["x"].double(), s["w"].double(), c["hidden"]
        bias = s["bias"].double() if c["bias"] else torch.zeros(2 * n, device="cuda", dtype=torch.float64)
        gate, up = x @ w[:, :n] + bias[:n], x @ w[:, n:] + bias[n:]
        bell = torch.exp(-gate ** 2 / 2) / math.sqrt(2 * math.pi)
        if c["act"] == "relu":
            act, slope = torch.where(gate > 0, gate, 0.0), torch.where(gate > 0, 1.0, 0.0).double()
        elif c["act"] == "gelu":
            below = torch.special.ndtr(gate)
            act, slope = gate * below, below + gate * bell
        elif c["act"] == "gelu_tanh":
            a, b = math.sqrt(2 / math.pi), 0.044715
            half = torch.sigmoid(2 * a * (gate + b * gate ** 3))          # (1 + tanh v) / 2
            act, slope = gate * half, half + gate * 2 * half * (1 - half) * a * (1 + 3 * b * gate ** 2)
        else:
            half = torch.sigmoid(gate)
            act, slope = (half, half * (1 - half)) if c["act"] == "sigmoid" else (gate * half, half + gate * half * (1 - half))
        out = {"h": act * up}
        if back:
            dh = s["grad_h"].double()
            dg, du = dh * up * slope, dh * act
            out["grad_x"] = dg @ w[:, :n].t() + du @ w[:, n:].t()
            out["grad_w"] = torch.cat([x.t() @ dg, x.t() @ du], 1)
            if c["bias"]:
                out["grad_bias"] = torch.cat([dg.sum(0), du.sum(0)])
        return out
    if c["op"] == "vocab":
        rows, classes = c["rows"], c["classes"]
        x, held = s["x"].double(), s["targets"] >= 0
        count, step = max(1, int(held.sum())), 8192
        pieces = [(v, min(classes, v + step)) for v in range(0, classes, step)]

        def logits(lo, hi):
            return x @ s["w"][:, lo:hi].double() + (s["bias"][lo:hi].double() if c["bias"] else 0.0)

        lse = torch.full((rows,), -math.inf, device="cuda", dtype=torch.float64)
        at = torch.zeros(rows, device="cuda", dtype=torch.float64)
        for lo, hi in pieces:
            z = logits(lo, hi)
            lse = torch.logaddexp(lse, torch.logsumexp(z, 1))
            inside = ((s["targets"] >= lo) & (s["targets"] < hi)).nonzero()[:, 0]
            at[inside] = z[inside, s["targets"][inside].long() - lo]
        out = {"loss": ((lse - at)[held].sum() / count).reshape(1)}
        if back:
            f = torch.where(held, float(s["upstream"]) / count, 0.0).double()
            dx, dw, db = torch.zeros_like(x), [], []
            for lo, hi in pieces:
                d = torch.exp(logits(lo, hi) - lse[:, None])
                inside = ((s["targets"] >= lo) & (s["targets"] < hi)).nonzero()[:, 0]
                d[inside, s["targets"][inside].long() - lo] -= 1.0
                d *= f[:, None]
                dx += d @ s["w"][:, lo:hi].double().t()
                dw.append(x.t() @ d)
                db.append(d.sum(0))
            out["grad_x"], out["grad_w"] = dx, torch.cat(dw, 1)
            if c["bias"]:
                out["grad_bias"] = torch.cat(db)
        return out
    rows, temp = c["rows"], c["temperature"]
    log_q = torch.log_softmax(s["logits"].double() / temp, 1)
    listed_ids = s["ids"].long()
    here = listed_ids >= 0
    u = torch.where(here, s["teacher"].double() / temp, -math.inf)
    kept = here.any(1)
    log_p = torch.where(here & kept[:, None], u - torch.logsumexp(u, 1, keepdim=True), -math.inf)
    p = torch.exp(log_p)
    terms = torch.where(here, p * (log_p - log_q.gather(1, listed_ids.clamp(min=0))), 0.0)
    out = {"loss": (temp ** 2 * terms.sum() / rows).reshape(1)}
    if back:
        target = torch.zeros_like(log_q).scatter_add_(1, listed_ids.clamp(min=0), p)
        out["grad_logits"] = (torch.exp(log_q) * kept[:, None] - target) * (temp / rows * float(s["upstream"]))
    return out
