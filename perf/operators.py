"""Layers whose weight depends on the row, as cases for timing and for comparing results: routing of tokens to experts,
the exchange of rows between tokens and groups, the experts' products, and low-rank adapters beside a shared projection.

A case is a dict of plain values with an "op" and its sizes; `listed()` holds the fixed ones, `draw(rng)` makes others of
the same ranges.  With `own` false `run` computes plain torch operations in float32, with `own` true it calls the C ABI
through `recpulse_amd.capi` on the same tensors.

  route      the k largest of each token's logits, their softmax weights, and the slots sorted by expert; with backward
             the gradient of the logits.  Padding tokens have logits of -inf and are sent nowhere.
  exchange   rows copied from tokens to their experts' groups, and the groups' results added up per token with the
             routing weights; with backward the gradients of both.
  experts    y = x.W + b with one weight for each group of rows, groups of any size; with backward dx, dW and db.
  adapters   y = x.W + b + scale (x.A).B where W is shared and A, B belong to the row's request; with backward dx, dA, dB.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
CODES = {"f32": 0, "f16": 2, "bf16": 3}                      # recpulse_amd.capi's dtype codes
SIZE = {"bf16": 2, "f16": 2, "f32": 4}


def listed():
    return [
        # one decoding step of a few requests: nothing but latency
        dict(name="route-decode", op="route", dtype="bf16", tokens=16, experts=64, k=6, normalize=True, padded=False, backward=False),
        # a training step's batch, one token in eight padding
        dict(name="route-train", op="route", dtype="f32", tokens=16384, experts=128, k=8, normalize=False, padded=True, backward=True),
        dict(name="exchange-decode", op="exchange", dtype="bf16", tokens=16, k=2, d=4096, padded=False, backward=False),
        dict(name="exchange-train", op="exchange", dtype="bf16", tokens=8192, k=2, d=4096, padded=True, backward=True),
        # decoding: a few rows for each expert, the weights are read once
        dict(name="experts-decode", op="experts", dtype="bf16", rows=16, groups=8, inner=4096, outer=4096, bias=False, backward=False),
        # a prompt
        dict(name="experts-prompt", op="experts", dtype="f16", rows=4096, groups=8, inner=1024, outer=4096, bias=True, backward=False),
        # training, sizes that come from data
        dict(name="experts-odd", op="experts", dtype="bf16", rows=1999, groups=6, inner=519, outer=1031, bias=True, backward=True),
        # training at the sizes of the framework's small network, in float32
        dict(name="experts-mlp", op="experts", dtype="f32", rows=1024, groups=4, inner=784, outer=256, bias=True, backward=True),
        # training, the largest
        dict(name="experts-train", op="experts", dtype="bf16", rows=16384, groups=16, inner=4096, outer=4096, bias=True, backward=True),
        # decoding: every request a single row with an adapter of its own
        dict(name="adapters-decode", op="adapters", dtype="bf16", rows=32, segments=32, adapters=32, inner=4096, outer=4096, rank=16, without=0, bias=False, backward=False),
        # prompts of several requests, one of them without an adapter
        dict(name="adapters-prompt", op="adapters", dtype="bf16", rows=4096, segments=7, adapters=4, inner=4096, outer=4096, rank=32, without=1, bias=True, backward=False),
        # fine-tuning
        dict(name="adapters-train", op="adapters", dtype="f16", rows=2048, segments=5, adapters=3, inner=1024, outer=2048, rank=8, without=0, bias=True, backward=True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _width(rng, low, high):
    """A width: mostly whole vectors, now and then any number."""
    n = _log(rng, low, high)
    unit = rng.choice([1, 8, 64])
    return max(low, min(high, n // unit * unit))


def draw(rng):
    op = rng.choice(["route", "exchange", "experts", "experts", "adapters", "adapters"])
    backward = rng.random() < 0.5
    if op == "route":
        experts = rng.randint(4, 256)
        return dict(op=op, dtype=rng.choice(["bf16", "f16", "f32"]), tokens=_log(rng, 1, 32768), experts=experts, k=rng.randint(1, min(8, experts)),
                    normalize=rng.random() < 0.5, padded=rng.random() < 0.5, backward=backward)
    if op == "exchange":
        return dict(op=op, dtype=rng.choice(["bf16", "f16", "f32"]), tokens=_log(rng, 1, 8192), k=rng.randint(1, 6), d=_width(rng, 64, 4096),
                    padded=rng.random() < 0.5, backward=backward)
    if op == "experts":
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        return dict(op=op, dtype=dtype, rows=_log(rng, 1, 16384 if dtype != "f32" else 4096), groups=rng.randint(1, 16), inner=_width(rng, 64, 4096),
                    outer=_width(rng, 64, 4096), bias=rng.random() < 0.5, backward=backward)
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    rows = _log(rng, 1, 8192 if dtype != "f32" else 2048)
    segments = rng.randint(1, min(rows, 48))
    return dict(op=op, dtype=dtype, rows=rows, segments=segments, adapters=rng.randint(1, 32), inner=_width(rng, 64, 4096), outer=_width(rng, 64, 4096),
                rank=rng.choice([4, 8, 16, 16, 32, 64]), without=rng.randint(0, segments // 4), bias=rng.random() < 0.5, backward=backward)


# ---- inputs ------------------------------------------------------------------------------------------------------

def _cut(gen, rows, parts, empty):
    """`parts` sizes that add up to `rows`, uneven; with `empty` some may be zero, otherwise none is."""
    if empty:
        share = torch.exp(0.4 * torch.randn(parts, generator=gen))
        at = torch.multinomial(share, rows, replacement=True, generator=gen)
        return torch.bincount(at, minlength=parts).tolist()
    cuts = torch.randperm(rows - 1, generator=gen)[:parts - 1].sort().values + 1
    ends = [0] + cuts.tolist() + [rows]
    return [b - a for a, b in zip(ends, ends[1:])]


def _offsets(sizes):
    return torch.tensor([0] + sizes).cumsum(0).to(torch.int32).cuda()


def prepare(case, seed):
    gen = torch.Generator().manual_seed(seed)
    dev = torch.Generator(device="cuda").manual_seed(seed)
    c, t = dict(case), DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, dtype=t):
        return (torch.randn(*shape, device="cuda", generator=dev) * scale).to(dtype)

    def zeros(*shape, dtype=t):
        return torch.zeros(*shape, device="cuda", dtype=dtype)

    s = {"case": c, "code": CODES[case["dtype"]]}
    if c["op"] == "route":
        tokens, experts, k = c["tokens"], c["experts"], c["k"]
        s["logits"] = normal(tokens, experts, scale=2.0)
        if c["padded"]:
            s["logits"][torch.rand(tokens, device="cuda", generator=dev) < 0.125] = -math.inf
        s["grad_weights"] = normal(tokens, k, dtype=torch.float32)
        s["weights"] = zeros(tokens, k, dtype=torch.float32)
        s["experts"], s["order"], s["position"] = (zeros(*shape, dtype=torch.int32) for shape in ((tokens, k), (tokens * k,), (tokens * k,)))
        s["offsets"] = zeros(experts + 1, dtype=torch.int32)
        s["grad_logits"] = zeros(tokens, experts)
    elif c["op"] == "exchange":
        tokens, k, d = c["tokens"], c["k"], c["d"]
        place = torch.randperm(tokens * k, generator=gen).to(torch.int32).reshape(tokens, k)
        if c["padded"]:
            place[torch.rand(tokens, generator=gen) < 0.125] = -1
        s["position"] = place.cuda()
        s["weights"] = torch.softmax(normal(tokens, k, dtype=torch.float32), 1)
        s["x"], s["z"] = normal(tokens, d), normal(tokens * k, d)
        s["grad_y"], s["grad_rows"] = normal(tokens, d), normal(tokens * k, d)
        s["rows"], s["y"] = zeros(tokens * k, d), zeros(tokens, d)
        s["grad_z"], s["grad_x"] = zeros(tokens * k, d), zeros(tokens, d)
        s["grad_weights"] = zeros(tokens, k, dtype=torch.float32)
    elif c["op"] == "experts":
        rows, groups, inner, outer = c["rows"], c["groups"], c["inner"], c["outer"]
        sizes = _cut(gen, rows, groups, True)
        s["offsets"], s["most"] = _offsets(sizes), max(sizes)
        s["x"], s["w"] = normal(rows, inner), normal(groups, inner, outer, scale=inner ** -0.5)
        s["bias"] = normal(groups, outer, scale=0.1) if c["bias"] else None
        s["y"] = zeros(rows, outer)
        if c["backward"]:
            s["grad_y"] = normal(rows, outer)
            s["grad_x"], s["grad_w"] = zeros(rows, inner), zeros(groups, inner, outer)
            s["grad_bias"] = zeros(groups, outer) if c["bias"] else None
    else:
        rows, segments, adapters, inner, outer, rank = (c[name] for name in ("rows", "segments", "adapters", "inner", "outer", "rank"))
        sizes = _cut(gen, rows, segments, False)
        s["offsets"], s["most"] = _offsets(sizes), max(sizes)
        ids = torch.randperm(segments, generator=gen) % adapters
        ids[torch.randperm(segments, generator=gen)[:c["without"]]] = -1
        s["ids"] = ids.to(torch.int32).cuda()
        s["x"], s["w"] = normal(rows, inner), normal(inner, outer, scale=inner ** -0.5)
        s["a"], s["b"] = normal(adapters, inner, rank, scale=inner ** -0.5), normal(adapters, rank, outer, scale=rank ** -0.5)
        s["scales"] = (0.5 + torch.rand(adapters, generator=gen)).cuda()
        s["bias"] = normal(outer, scale=0.1) if c["bias"] else None
        s["y"], s["low"] = zeros(rows, outer), zeros(rows, rank, dtype=torch.float32)
        if c["backward"]:
            s["grad_y"] = normal(rows, outer)
            s["grad_x"], s["grad_a"], s["grad_b"] = zeros(rows, inner), zeros(adapters, inner, rank), zeros(adapters, rank, outer)
            s["grad_low"] = zeros(rows, rank, dtype=torch.float32)
    return s


# ---- the plain forms ---------------------------------------------------------------------------------------------

def _route_plain(s, c):
    tokens, experts, k = c["tokens"], c["experts"], c["k"]
    logits = s["logits"].float()
    best, ids = torch.sort(logits, dim=1, descending=True, stable=True)
    best, ids = best[:, :k], ids[:, :k]
    picked = best > -math.inf
    top = torch.where(picked[:, :1], best[:, :1], 0.0)
    e = torch.exp(best - top)
    p = torch.exp(logits - top)
    total = (e if c["normalize"] else p).sum(1, keepdim=True)
    total = torch.where(total > 0, total, 1.0)
    weights = e / total
    flat = torch.where(picked, ids, experts).reshape(-1)
    ordered, order = torch.sort(flat, stable=True)
    bounds = torch.searchsorted(ordered, torch.arange(experts + 1, device="cuda"))
    count = torch.arange(tokens * k, device="cuda")
    position = torch.empty_like(count)
    position[order] = count
    out = {"weights": weights, "experts": torch.where(picked, ids, -1).int(), "offsets": bounds.int(),
           "order": torch.where(count < bounds[-1], order, -1).int(), "position": torch.where(picked.reshape(-1), position, -1).int()}
    if c["backward"]:
        g = torch.where(picked, s["grad_weights"], 0.0)
        mean = (weights * g).sum(1, keepdim=True)
        grad = torch.zeros_like(logits) if c["normalize"] else -(p / total) * mean
        grad.scatter_add_(1, ids, weights * (g - mean) if c["normalize"] else weights * g)
        out["grad_logits"] = grad.to(s["logits"].dtype)
    return out


def _exchange_plain(s, c):
    t = s["x"].dtype
    tokens, k, d = c["tokens"], c["k"], c["d"]
    there = (s["position"] >= 0)[..., None]
    at = torch.where(there[..., 0], s["position"], tokens * k).long()

    def spread(values):                                        # [tokens, k, d] to the rows of the groups
        rows = torch.zeros(tokens * k + 1, d, device="cuda")
        rows[at.reshape(-1)] = values.reshape(-1, d)
        return rows[:-1].to(t)

    def gather(rows):
        return torch.where(there, rows.float()[at.clamp(max=tokens * k - 1)], 0.0)

    z = gather(s["z"])
    out = {"rows": spread(s["x"].float()[:, None].expand(tokens, k, d)), "y": (s["weights"][..., None] * z).sum(1).to(t)}
    if c["backward"]:
        g = s["grad_y"].float()[:, None]
        out["grad_z"] = spread(s["weights"][..., None] * g)
        out["grad_weights"] = (g * z).sum(2)
        out["grad_x"] = gather(s["grad_rows"]).sum(1).to(t)
    return out


def _padded(s):
    """Rows of each group side by side: their indices [groups, most], which of them are there, and each row's place."""
    begin, end = s["offsets"][:-1].long(), s["offsets"][1:].long()
    at = begin[:, None] + torch.arange(s["most"], device="cuda")
    row = torch.arange(s["case"]["rows"], device="cuda")
    group = torch.searchsorted(end, row, right=True)
    return at.clamp(max=s["case"]["rows"] - 1), (at < end[:, None])[..., None], group * s["most"] + row - begin[group]


def _experts_plain(s, c):
    t = s["x"].dtype
    at, there, place = _padded(s)
    x, w = torch.where(there, s["x"].float()[at], 0.0), s["w"].float()
    y = torch.bmm(x, w)
    if c["bias"]:
        y = y + s["bias"].float()[:, None]
    out = {"y": y.reshape(-1, c["outer"])[place].to(t)}
    if c["backward"]:
        g = torch.where(there, s["grad_y"].float()[at], 0.0)
        out["grad_x"] = torch.bmm(g, w.transpose(1, 2)).reshape(-1, c["inner"])[place].to(t)
        out["grad_w"] = torch.bmm(x.transpose(1, 2), g).to(t)
        if c["bias"]:
            out["grad_bias"] = g.sum(1).to(t)
    return out


def _adapters_plain(s, c):
    t = s["x"].dtype
    at, there, place = _padded(s)
    ids = s["ids"].long().clamp(min=0)
    scale = torch.where(s["ids"] >= 0, s["scales"][ids], 0.0)[:, None, None]
    a, b = s["a"].float()[ids], s["b"].float()[ids]
    x = s["x"].float()
    xs = torch.where(there, x[at], 0.0)
    low = scale * torch.bmm(xs, a)
    y = torch.mm(x, s["w"].float()) + torch.bmm(low, b).reshape(-1, c["outer"])[place]
    if c["bias"]:
        y = y + s["bias"].float()
    out = {"y": y.to(t)}
    if c["backward"]:
        g = s["grad_y"].float()
        gs = torch.where(there, g[at], 0.0)
        grad_low = scale * torch.bmm(gs, b.transpose(1, 2))
        out["grad_x"] = (torch.mm(g, s["w"].float().t()) + torch.bmm(grad_low, a.transpose(1, 2)).reshape(-1, c["inner"])[place]).to(t)
        out["grad_a"] = torch.zeros_like(s["a"], dtype=torch.float32).index_add_(0, ids, torch.bmm(xs.transpose(1, 2), grad_low)).to(t)
        out["grad_b"] = torch.zeros_like(s["b"], dtype=torch.float32).index_add_(0, ids, torch.bmm(low.transpose(1, 2), gs)).to(t)
    return out


# ---- the framework's calls -----------------------------------------------------------------------------------------

def _at(tensor):
    return None if tensor is None else tensor.data_ptr()


def _own(s, c):
    from recpulse_amd import capi
    lib, code = capi.lib(), s["code"]
    lib.rp_hip_set_stream(torch.cuda.current_stream().cuda_stream)
    if c["op"] == "route":
        tokens, experts, k = c["tokens"], c["experts"], c["k"]
        out = {name: s[name] for name in ("weights", "experts", "offsets", "order", "position")}
        capi.check(lib.rp_hip_route_forward(_at(s["weights"]), _at(s["experts"]), _at(s["offsets"]), _at(s["order"]), _at(s["position"]), _at(s["logits"]),
                                            experts, tokens, experts, k, c["normalize"], code), "rp_hip_route_forward")
        if c["backward"]:
            capi.check(lib.rp_hip_route_backward(_at(s["grad_logits"]), _at(s["grad_weights"]), _at(s["weights"]), _at(s["experts"]), _at(s["logits"]),
                                                 experts, tokens, experts, k, c["normalize"], code), "rp_hip_route_backward")
            out["grad_logits"] = s["grad_logits"]
        return out
    if c["op"] == "exchange":
        tokens, k, d = c["tokens"], c["k"], c["d"]
        where = _at(s["position"])
        capi.check(lib.rp_hip_dispatch_rows(_at(s["rows"]), _at(s["x"]), where, tokens, k, d, d, d, code), "rp_hip_dispatch_rows")
        capi.check(lib.rp_hip_combine_forward(_at(s["y"]), _at(s["z"]), _at(s["weights"]), where, tokens, k, d, d, d, code), "rp_hip_combine_forward")
        out = {"rows": s["rows"], "y": s["y"]}
        if c["backward"]:
            capi.check(lib.rp_hip_combine_backward(_at(s["grad_z"]), _at(s["grad_weights"]), _at(s["grad_y"]), _at(s["z"]), _at(s["weights"]), where,
                                                   tokens, k, d, d, d, d, code), "rp_hip_combine_backward")
            capi.check(lib.rp_hip_combine_forward(_at(s["grad_x"]), _at(s["grad_rows"]), None, where, tokens, k, d, d, d, code), "rp_hip_combine_forward")
            out.update(grad_z=s["grad_z"], grad_weights=s["grad_weights"], grad_x=s["grad_x"])
        return out
    rows, inner, outer = c["rows"], c["inner"], c["outer"]
    if c["op"] == "experts":
        groups = c["groups"]
        capi.check(lib.rp_hip_grouped_linear_forward(_at(s["y"]), _at(s["x"]), _at(s["w"]), _at(s["bias"]), _at(s["offsets"]), groups, rows, inner, outer,
                                                     inner, 1, inner * outer, outer, 1, outer, code), "rp_hip_grouped_linear_forward")
        out = {"y": s["y"]}
        if c["backward"]:
            capi.check(lib.rp_hip_grouped_linear_backward(_at(s["grad_x"]), _at(s["grad_w"]), _at(s["grad_bias"]), _at(s["grad_y"]), _at(s["x"]), _at(s["w"]),
                                                          _at(s["offsets"]), groups, rows, inner, outer, outer, inner, 1, inner * outer, outer, 1, inner,
                                                          0, 0, 0, code), "rp_hip_grouped_linear_backward")
            out.update(grad_x=s["grad_x"], grad_w=s["grad_w"])
            if c["bias"]:
                out["grad_bias"] = s["grad_bias"]
        return out
    plan = (_at(s["scales"]), _at(s["ids"]), _at(s["offsets"]), c["segments"], c["adapters"], rows, inner, outer, c["rank"])
    capi.check(lib.rp_hip_adapter_linear_forward(_at(s["y"]), _at(s["low"]), _at(s["x"]), _at(s["w"]), _at(s["bias"]), _at(s["a"]), _at(s["b"]), *plan,
                                                 inner, 1, outer, 1, outer, code), "rp_hip_adapter_linear_forward")
    out = {"y": s["y"]}
    if c["backward"]:
        capi.check(lib.rp_hip_adapter_linear_backward(_at(s["grad_x"]), _at(s["grad_a"]), _at(s["grad_b"]), _at(s["grad_low"]), _at(s["grad_y"]), _at(s["x"]),
                                                      _at(s["w"]), _at(s["a"]), _at(s["b"]), _at(s["low"]), *plan, outer, inner, 1, outer, 1, inner,
                                                      0, 0, 0, code), "rp_hip_adapter_linear_backward")
        out.update(grad_x=s["grad_x"], grad_a=s["grad_a"], grad_b=s["grad_b"])
    return out


def run(s):
    c = s["case"]
    if own:
        return _own(s, c)
    return {"route": _route_plain, "exchange": _exchange_plain, "experts": _experts_plain, "adapters": _adapters_plain}[c["op"]](s, c)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------

def work(c):
    es = SIZE[c["dtype"]]
    if c["op"] == "route":
        slots, cells = c["tokens"] * c["k"], c["tokens"] * c["experts"]
        data = cells * es + slots * 16 + 4 * (c["experts"] + 1)
        if c["backward"]:
            data += slots * 4 + cells * es
        return {"bytes": data, "flops": 4 * cells}
    if c["op"] == "exchange":
        t, r = c["tokens"] * c["d"] * es, c["tokens"] * c["k"] * c["d"] * es
        slots = c["tokens"] * c["k"]
        data, flops = 2 * t + 2 * r + 8 * slots, 2 * slots * c["d"]
        if c["backward"]:
            data += 2 * t + 2 * r + 4 * slots
            flops += 4 * slots * c["d"]
        return {"bytes": data, "flops": flops}
    rows, inner, outer = c["rows"], c["inner"], c["outer"]
    ways = 3 if c["backward"] else 1
    if c["op"] == "experts":
        used = c["groups"] * (1 - (1 - 1 / c["groups"]) ** rows)
        data = es * (rows * (inner + outer) + used * inner * outer)
        if c["backward"]:
            data += es * (rows * (inner + outer) + c["groups"] * inner * outer)
        return {"bytes": data, "flops": 2 * rows * inner * outer * ways}
    used = min(c["segments"] - c["without"], c["adapters"])
    data = es * (rows * (inner + outer) + inner * outer + used * c["rank"] * (inner + outer))
    flops = 2 * rows * (inner * outer + c["rank"] * (inner + outer))
    if c["backward"]:
        data += es * (rows * (inner + outer) + c["adapters"] * c["rank"] * (inner + outer))
        flops += 2 * rows * (inner * outer + 3 * c["rank"] * (inner + outer))
    return {"bytes": data, "flops": flops}


# ---- from the definitions, in 64 bits --------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    if c["op"] == "route":
        logits = s["logits"].double()
        tokens, experts, k = c["tokens"], c["experts"], c["k"]
        rest, chosen, live = logits.clone(), [], []
        for _ in range(k):                                      # the first of the largest, taken out, k times
            most = rest.max(1, keepdim=True).values
            first = (rest == most).int().argmax(1, keepdim=True)
            chosen.append(first)
            live.append(most > -math.inf)
            rest.scatter_(1, first, -math.inf)
        ids, picked = torch.cat(chosen, 1), torch.cat(live, 1)
        p = torch.nan_to_num(torch.softmax(logits, 1), nan=0.0)
        weights = torch.where(picked, p.gather(1, ids), 0.0)
        if c["normalize"]:
            own_logits = torch.where(picked, logits.gather(1, ids), -math.inf)
            weights = torch.nan_to_num(torch.softmax(own_logits, 1), nan=0.0)
        ids = torch.where(picked, ids, -1)
        order, position, offsets, flat = [], [-1] * (tokens * k), [0], ids.reshape(-1).tolist()
        lists = [[] for _ in range(experts)]
        for slot, e in enumerate(flat):
            if e >= 0:
                lists[e].append(slot)
        for one in lists:
            for slot in one:
                position[slot] = len(order)
                order.append(slot)
            offsets.append(len(order))
        order += [-1] * (tokens * k - len(order))
        out = {"weights": weights, "experts": ids.int(), "offsets": torch.tensor(offsets, dtype=torch.int32),
               "order": torch.tensor(order, dtype=torch.int32), "position": torch.tensor(position, dtype=torch.int32)}
        if c["backward"]:
            hot = torch.zeros_like(logits)
            given = torch.where(picked, s["grad_weights"].double(), 0.0)
            hot.scatter_add_(1, ids.clamp(min=0), given)
            among = torch.zeros_like(logits).scatter_add_(1, ids.clamp(min=0), weights) if c["normalize"] else p
            out["grad_logits"] = among * (hot - (among * hot).sum(1, keepdim=True))
        return out
    if c["op"] == "exchange":
        place, k = s["position"].tolist(), c["k"]
        zero = torch.zeros(1, c["d"], device="cuda", dtype=torch.float64)
        z, back = torch.cat([s["z"].double(), zero]), torch.cat([s["grad_rows"].double(), zero])
        source, owner = [-1] * (c["tokens"] * k), [0.0] * (c["tokens"] * k)
        w = s["weights"].double().tolist()
        for t, row in enumerate(place):
            for j, at in enumerate(row):
                if at >= 0:
                    source[at], owner[at] = t, w[t][j]
        source, owner = torch.tensor(source, device="cuda"), torch.tensor(owner, device="cuda", dtype=torch.float64)
        x, g = torch.cat([s["x"].double(), zero]), torch.cat([s["grad_y"].double(), zero])
        at = s["position"].long()                               # -1 is the row of zeros at the end
        out = {"rows": x[source], "y": sum(s["weights"][:, j:j + 1].double() * z[at[:, j]] for j in range(k))}
        if c["backward"]:
            out["grad_z"] = owner[:, None] * g[source]
            out["grad_weights"] = torch.stack([(g[:-1] * z[at[:, j]]).sum(1) for j in range(k)], 1)
            out["grad_x"] = sum(back[at[:, j]] for j in range(k))
        return out
    ends = s["offsets"].tolist()
    spans = list(zip(ends, ends[1:]))
    x = s["x"].double()
    g = s["grad_y"].double() if c["backward"] else None
    if c["op"] == "experts":
        y, out = torch.zeros(c["rows"], c["outer"], device="cuda", dtype=torch.float64), {}
        dx, dw, db = torch.zeros_like(x), [], []
        for e, (lo, hi) in enumerate(spans):
            w = s["w"][e].double()
            y[lo:hi] = x[lo:hi] @ w + (s["bias"][e].double() if c["bias"] else 0.0)
            if c["backward"]:
                dx[lo:hi] = g[lo:hi] @ w.t()
                dw.append(x[lo:hi].t() @ g[lo:hi])
                db.append(g[lo:hi].sum(0))
        out["y"] = y
        if c["backward"]:
            out["grad_x"], out["grad_w"] = dx, torch.stack(dw)
            if c["bias"]:
                out["grad_bias"] = torch.stack(db)
        return out
    w = s["w"].double()
    y = x @ w + (s["bias"].double() if c["bias"] else 0.0)
    dx = g @ w.t() if c["backward"] else None
    da, db = torch.zeros_like(s["a"], dtype=torch.float64), torch.zeros_like(s["b"], dtype=torch.float64)
    for (lo, hi), e in zip(spans, s["ids"].tolist()):
        if e < 0:
            continue
        a, b, scale = s["a"][e].double(), s["b"][e].double(), float(s["scales"][e])
        low = scale * (x[lo:hi] @ a)
        y[lo:hi] += low @ b
        if c["backward"]:
            grad_low = scale * (g[lo:hi] @ b.t())
            dx[lo:hi] += grad_low @ a.t()
            da[e] += x[lo:hi].t() @ grad_low
            db[e] += low.t() @ g[lo:hi]
    return {"y": y, "grad_x": dx, "grad_a": da, "grad_b": db} if c["backward"] else {"y": y}
