"""Measured cases of the operators that train routed experts, through the public entry points, from one
decoded token to a training batch.

Every case is a dict of plain values; ``op`` names the operator:

* ``product``     rows sorted by expert times that expert's bf16 matrix [n, k]; ``form`` "forward" (x W^T),
  "by_input" (dy W) or "by_weight" (dy^T x of each expert's rows).
* ``activation``  the gradient of the gated activation between an expert's products, with the routing weights:
  by gate and up, by the weights, and the weighted activation that the down matrix's gradient reads.
* ``norm``        the residual's addition and RMS norm, with an output in bf16, in E4M3 with a scale per 128
  columns, or both; ``norm_gradient`` its backward pass.

Inputs have the distributions that the path meets: activations N(0, 1) with a few columns 20 times as
large, gradients N(0, 1e-3), weights N(0, 0.02), rows per expert from top-k routing by scores with a Zipf or
a uniform bias.
"""
import math

import torch

own = False

HIDDEN, EXPERT_HIDDEN, LATENT, EXPERTS, TOP_K = 7168, 2048, 3584, 896, 16   # the benchmark layer and the latent shape
BLOCK, LARGEST, SMALLEST = 128, 448.0, 2.0 ** -126                     # block, largest E4M3 value, smallest scale
BETA, LINEAR_BETA, ROUTE_SCALE, TINY, EPSILON = 4.0, 25.0, 2.5, 1e-20, 1e-5


def _product(name, form, tokens, experts, top_k, n, k, out, bias):
    return {"name": name, "op": "product", "form": form, "tokens": tokens, "experts": experts, "top_k": top_k, "n": n, "k": k,
            "out": out, "bias": bias}


def listed():
    return [
        # gate of the experts of one decoded token: most groups are empty, the others have one row
        _product("product_token", "forward", 1, 64, TOP_K, EXPERT_HIDDEN, HIDDEN, "bf16", "uniform"),
        # down of a decode batch, loads uneven
        _product("product_batch", "forward", 61, 64, 8, HIDDEN, EXPERT_HIDDEN, "bf16", "zipf"),
        # up of a training batch
        _product("product_4096", "forward", 4096, 64, 8, EXPERT_HIDDEN, HIDDEN, "bf16", "uniform"),
        # the gradient by the input of a prompt of odd length at the latent shape, in f32 as sums of two matrices' are kept
        _product("by_input_1021", "by_input", 1021, 48, 6, EXPERT_HIDDEN, LATENT, "f32", "zipf"),
        # the gradient by the weight of a training batch
        _product("by_weight_4096", "by_weight", 4096, 32, 8, EXPERT_HIDDEN, HIDDEN, "f32", "uniform"),
        # of many small experts, some of them without a row
        _product("by_weight_small", "by_weight", 733, EXPERTS, 4, 264, 520, "bf16", "zipf"),
        # a short prompt's routes, with rows of odd length
        {"name": "activation_77", "op": "activation", "tokens": 77, "top_k": 3, "columns": 1023, "form": "situ"},
        # a training batch
        {"name": "activation_4096", "op": "activation", "tokens": 4096, "top_k": 8, "columns": EXPERT_HIDDEN, "form": "swiglu"},
        # one decoded token in front of 8-bit products
        {"name": "norm_token", "op": "norm", "rows": 1, "columns": HIDDEN, "type": "bf16", "residual": True, "out": "codes"},
        # a prefill batch whose rows go to the router in bf16 and to the experts in 8 bits
        {"name": "norm_8192", "op": "norm", "rows": 8192, "columns": HIDDEN, "type": "bf16", "residual": True, "out": "both"},
        # the backward pass over a residual stream kept in f32, odd sizes
        {"name": "norm_gradient_1021", "op": "norm_gradient", "rows": 1021, "columns": 3583, "type": "f32", "residual": True},
        # of a training batch
        {"name": "norm_gradient_8192", "op": "norm_gradient", "rows": 8192, "columns": HIDDEN, "type": "bf16", "residual": True},
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choices(["product", "activation", "norm", "norm_gradient"], [6, 2, 3, 2])[0]
    if op == "product":
        form = rng.choice(["forward", "by_input", "by_weight"])
        experts = _log_int(rng, 1, EXPERTS)
        narrow, wide = 8 * _log_int(rng, 1, EXPERT_HIDDEN // 8), 8 * _log_int(rng, 1, HIDDEN // 8)
        most = 32 * EXPERT_HIDDEN * HIDDEN               # elements of all experts' matrices
        while experts * narrow * wide > most:
            experts = max(1, experts // 2)
        top_k = rng.randint(1, min(8, experts))
        n, k = (narrow, wide) if rng.random() < 0.5 else (wide, narrow)
        return {"op": op, "form": form, "tokens": _log_int(rng, 1, 4096), "experts": experts, "top_k": top_k, "n": n, "k": k,
                "out": rng.choice(["bf16", "f32"]), "bias": rng.choice(["uniform", "zipf"])}
    if op == "activation":
        return {"op": op, "tokens": _log_int(rng, 1, 4096), "top_k": rng.randint(1, 8), "columns": _log_int(rng, 1, EXPERT_HIDDEN),
                "form": rng.choice(["swiglu", "situ"])}
    case = {"op": op, "rows": _log_int(rng, 1, 8192), "columns": _log_int(rng, 16, HIDDEN), "type": rng.choice(["bf16", "f32"]),
            "residual": rng.random() < 0.7}
    if case["type"] == "f32":
        case["rows"] = max(1, case["rows"] // 2)         # the bytes of the largest listed case
    if op == "norm":
        case["out"] = rng.choice(["bf16", "codes", "both"])
    return case


# ------------------------------------------------------------------------------------------ inputs
_TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _normal(g, *shape, scale=1.0, dtype=torch.bfloat16):
    return (torch.randn(*shape, generator=g, device="cuda", dtype=dtype) * scale).to(dtype)


def _activations(g, rows, columns, dtype=torch.bfloat16):
    x = _normal(g, rows, columns, dtype=dtype)
    x[:, ::97] *= 20                                     # the columns that stand out
    return x


def _blocks(n):
    return (n + BLOCK - 1) // BLOCK


def _routing(g, tokens, experts, top_k, bias):
    """Ids of each token's experts, and the expert offsets of the rows in their grouped order."""
    logits = torch.randn(tokens, experts, generator=g, device="cuda")
    if bias == "zipf":
        logits -= torch.log(torch.arange(1, experts + 1, device="cuda").float())
    ids = torch.topk(logits, top_k, dim=1).indices
    counts = torch.bincount(ids.reshape(-1), minlength=experts)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)
    return logits, ids, offsets


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, s = case["op"], {"case": case}
    if op == "product":
        rows, n, k = case["tokens"] * case["top_k"], case["n"], case["k"]
        _, _, s["offsets"] = _routing(g, case["tokens"], case["experts"], case["top_k"], case["bias"])
        if case["form"] != "by_input":
            s["x"] = _activations(g, rows, k)
        if case["form"] != "forward":
            s["dy"] = _normal(g, rows, n, scale=1e-3)
        if case["form"] != "by_weight":
            s["w"] = _normal(g, case["experts"], n, k, scale=0.02)
    elif op == "activation":
        rows, columns, k = case["tokens"] * case["top_k"], case["columns"], case["top_k"]
        logits, ids, _ = _routing(g, case["tokens"], max(64, k), k, "zipf")
        chosen = torch.sigmoid(torch.gather(logits, 1, ids))
        s["weights"] = (chosen / (TINY + chosen.sum(1, keepdim=True)) * ROUTE_SCALE).contiguous()
        s["routes"] = torch.argsort(ids.reshape(-1), stable=True).to(torch.int32)
        s["gate"], s["up"] = _normal(g, rows, columns, scale=1.7), _normal(g, rows, columns, scale=1.7)
        s["d_out"] = _normal(g, rows, columns, scale=1e-3)
    else:
        kind = _TYPES[case["type"]]
        s["weight"] = _normal(g, case["columns"], scale=0.1) + 1
        s["x"] = _activations(g, case["rows"], case["columns"], kind)
        if op == "norm":
            s["residual"] = _normal(g, case["rows"], case["columns"], scale=3.0, dtype=kind) if case["residual"] else None
        else:
            s["rstd"] = torch.rsqrt(s["x"].double().square().mean(1) + EPSILON).float()
            s["dy"] = _normal(g, case["rows"], case["columns"], scale=1e-3)
            s["d_sum"] = _normal(g, case["rows"], case["columns"], scale=1e-3, dtype=kind) if case["residual"] else None
    if own:
        s["call"] = _handle(s)
    return s


# ------------------------------------------------------------------------------------------ the framework's calls
def _handle(s):
    """What a program keeps from call to call: the objects that hold weights and workspaces."""
    from moonshine_b200 import grouped, norm
    case = s["case"]
    if case["op"] == "product":
        if case["form"] == "by_weight":
            return grouped.GroupedWeightGradient(case["experts"], case["n"], case["k"])
        return grouped.GroupedProduct(s["w"])
    if case["op"] == "activation":
        return grouped.GatedActivation(case["form"], beta=BETA, linear_beta=LINEAR_BETA)
    return norm.RmsNorm(s["weight"], epsilon=EPSILON)


def _run_own(s):
    case, call = s["case"], s["call"]
    op = case["op"]
    if op == "product":
        kind = _TYPES[case["out"]]
        if case["form"] == "forward":
            return call.forward(s["x"], s["offsets"], dtype=kind)
        if case["form"] == "by_input":
            return call.by_input(s["dy"], s["offsets"], dtype=kind)
        return call.forward(s["dy"], s["x"], s["offsets"], dtype=kind)
    if op == "activation":
        d_gate, d_up, scaled, d_weights = call.backward(s["d_out"], s["gate"], s["up"], s["weights"], s["routes"])
        return {"d_gate": d_gate, "d_up": d_up, "scaled": scaled, "d_weights": d_weights}
    if op == "norm":
        r = call.forward(s["x"], s["residual"], y=case["out"] != "codes", codes=case["out"] != "bf16")
        out = {"rstd": r.rstd}
        if s["residual"] is not None:
            out["sum"] = r.sum
        if r.y is not None:
            out["y"] = r.y
        if r.codes is not None:
            out["codes"], out["scales"] = r.codes[:, :case["columns"]], r.scales[:, :_blocks(case["columns"])]
        return out
    dx, d_weight = call.backward(s["dy"], s["x"], s["rstd"], s["d_sum"])
    return {"dx": dx, "d_weight": d_weight}


# ------------------------------------------------------------------------------------------ the plain form, in 32 bits
def _run_product(s):
    case, form = s["case"], s["case"]["form"]
    cuts = s["offsets"].tolist()
    kind, rows = _TYPES[case["out"]], case["tokens"] * case["top_k"]
    if form == "by_weight":
        out = torch.zeros(case["experts"], case["n"], case["k"], device="cuda", dtype=kind)
        for e in range(case["experts"]):
            if cuts[e + 1] > cuts[e]:
                out[e] = (s["dy"][cuts[e]:cuts[e + 1]].float().t() @ s["x"][cuts[e]:cuts[e + 1]].float()).to(kind)
        return out
    out = torch.empty(rows, case["n"] if form == "forward" else case["k"], device="cuda", dtype=kind)
    for e in range(case["experts"]):
        if cuts[e + 1] > cuts[e]:
            w = s["w"][e].float()
            if form == "forward":
                out[cuts[e]:cuts[e + 1]] = (s["x"][cuts[e]:cuts[e + 1]].float() @ w.t()).to(kind)
            else:
                out[cuts[e]:cuts[e + 1]] = (s["dy"][cuts[e]:cuts[e + 1]].float() @ w).to(kind)
    return out


def _run_activation(s):
    gate, up, u = s["gate"].float(), s["up"].float(), s["d_out"].float()
    routes = s["routes"].long()
    w = s["weights"].reshape(-1)[routes].unsqueeze(1)
    sig, rest = torch.sigmoid(gate), torch.sigmoid(-gate)              # rest: 1 - sig without cancellation
    if s["case"]["form"] == "swiglu":
        left, d_left = gate * sig, sig * (1 + gate * rest)
        right, d_right = up, torch.ones_like(up)
    else:
        tg, tu = torch.tanh(gate / BETA), torch.tanh(up / LINEAR_BETA)
        left = BETA * tg * sig
        d_left = (1 - tg) * (1 + tg) * sig + left * rest
        right, d_right = LINEAR_BETA * tu, (1 - tu) * (1 + tu)
    act = left * right
    d_act = w * u
    d_weights = torch.zeros_like(s["weights"]).reshape(-1)
    d_weights[routes] = (u * act).sum(1)
    return {"d_gate": (d_act * right * d_left).to(torch.bfloat16), "d_up": (d_act * left * d_right).to(torch.bfloat16),
            "scaled": (w * act).to(torch.bfloat16), "d_weights": d_weights.reshape(s["weights"].shape)}


def _quantize(y):
    """[rows, columns] -> E4M3 values and scales per 128 columns."""
    rows, columns = y.shape
    padded = torch.nn.functional.pad(y, (0, _blocks(columns) * BLOCK - columns)).reshape(rows, _blocks(columns), BLOCK)
    scales = torch.clamp(padded.abs().amax(2) / LARGEST, min=SMALLEST)
    q = (padded / scales.unsqueeze(2)).to(torch.float8_e4m3fn)
    return q.reshape(rows, -1)[:, :columns].contiguous(), scales


def _run_norm(s):
    case, kind = s["case"], _TYPES[s["case"]["type"]]
    total = s["x"] if s["residual"] is None else (s["x"].float() + s["residual"].float()).to(kind)
    h = total.float()
    rstd = torch.rsqrt((h * h).mean(1) + EPSILON)
    y = h * rstd.unsqueeze(1) * s["weight"].float()
    out = {"rstd": rstd}
    if s["residual"] is not None:
        out["sum"] = total
    if case["out"] != "codes":
        out["y"] = y.to(torch.bfloat16)
    if case["out"] != "bf16":
        out["codes"], out["scales"] = _quantize(y)
    return out


def _run_norm_gradient(s):
    h, dy, rstd = s["x"].float(), s["dy"].float(), s["rstd"].unsqueeze(1)
    wdy = dy * s["weight"].float()
    dx = rstd * wdy - h * (rstd * rstd * rstd / h.shape[1] * (wdy * h).sum(1, keepdim=True))
    if s["d_sum"] is not None:
        dx = dx + s["d_sum"].float()
    return {"dx": dx.to(s["x"].dtype), "d_weight": (dy * h * rstd).sum(0)}


def run(s):
    if own:
        return _run_own(s)
    return {"product": _run_product, "activation": _run_activation, "norm": _run_norm,
            "norm_gradient": _run_norm_gradient}[s["case"]["op"]](s)


# ------------------------------------------------------------------------------------------ what a pass needs
def work(case):
    op = case["op"]
    if op == "product":
        rows, n, k, e = case["tokens"] * case["top_k"], case["n"], case["k"], case["experts"]
        size = 2 if case["out"] == "bf16" else 4
        touched = e * (1 - (1 - case["top_k"] / e) ** case["tokens"])  # experts that some token selects, for a uniform choice
        moved = {"forward": 2 * rows * k + 2 * touched * n * k + size * rows * n,
                 "by_input": 2 * rows * n + 2 * touched * n * k + size * rows * k,
                 "by_weight": 2 * rows * (n + k) + size * e * n * k}[case["form"]]
        return {"bytes": int(moved), "flops": 2 * rows * n * k}
    if op == "activation":
        routes, columns = case["tokens"] * case["top_k"], case["columns"]
        return {"bytes": 12 * routes * columns + 12 * routes, "flops": 30 * routes * columns}
    rows, columns, size = case["rows"], case["columns"], 2 if case["type"] == "bf16" else 4
    if op == "norm":
        moved = rows * columns * (size * (3 if case["residual"] else 1)) + 4 * rows + 2 * columns
        moved += 2 * rows * columns if case["out"] != "codes" else 0
        moved += rows * (columns + 4 * _blocks(columns)) if case["out"] != "bf16" else 0
        return {"bytes": moved, "flops": 8 * rows * columns}
    return {"bytes": rows * columns * (2 + size * (3 if case["residual"] else 2)) + 4 * rows + 6 * columns, "flops": 10 * rows * columns}


# ------------------------------------------------------------------------------------------ the definition, in 64 bits
def _exact_product(s):
    case, form = s["case"], s["case"]["form"]
    offsets = s["offsets"].long()
    rows = torch.arange(case["tokens"] * case["top_k"], device="cuda")
    group = torch.searchsorted(offsets[1:].contiguous(), rows, right=True)
    if form == "by_weight":
        out = torch.empty(case["experts"], case["n"], case["k"], device="cuda", dtype=torch.float64)
        for e in range(case["experts"]):
            at = (group == e).nonzero().reshape(-1)
            out[e] = torch.einsum("rn,rk->nk", s["dy"][at].double(), s["x"][at].double())
        return out
    left, rule = (s["x"], "rk,nk->rn") if form == "forward" else (s["dy"], "rn,nk->rk")
    out = torch.empty(rows.numel(), case["n"] if form == "forward" else case["k"], device="cuda", dtype=torch.float64)
    for e in group.unique().tolist():
        at = (group == e).nonzero().reshape(-1)
        out[at] = torch.einsum(rule, left[at].double(), s["w"][e].double())
    return out


def _exact_activation(s):
    """The derivatives by differentiating ln: d(g s(g)) = s(g) + g s(g) s(-g), d tanh = 1 / cosh^2."""
    case = s["case"]
    gate, up, u = s["gate"].double(), s["up"].double(), s["d_out"].double()
    flat = s["weights"].double().reshape(-1)
    w = flat[s["routes"].long()][:, None]
    sig, rest = 1 / (1 + torch.exp(-gate)), 1 / (1 + torch.exp(gate))
    if case["form"] == "swiglu":
        a, da, b, db = gate * sig, sig + gate * sig * rest, up, 1.0
    else:
        a = BETA * torch.tanh(gate / BETA) * sig
        da = sig / torch.cosh(gate / BETA) ** 2 + BETA * torch.tanh(gate / BETA) * sig * rest
        b, db = LINEAR_BETA * torch.tanh(up / LINEAR_BETA), 1 / torch.cosh(up / LINEAR_BETA) ** 2
    d_weights = torch.empty_like(flat)
    d_weights[s["routes"].long()] = torch.einsum("rc,rc->r", u, a * b)
    return {"d_gate": u * w * b * da, "d_up": u * w * a * db, "scaled": w * a * b, "d_weights": d_weights.view(s["weights"].shape)}


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "product":
        return _exact_product(s)
    if op == "activation":
        return _exact_activation(s)
    weight, rows, columns = s["weight"].double(), case["rows"], case["columns"]
    if op == "norm_gradient":
        # by the chain rule through z = h rstd: the part of w dy that changes the row's length falls out
        h, dy, rstd = s["x"].double(), s["dy"].double(), s["rstd"].double()[:, None]
        z, by_z = h * rstd, dy * weight
        dx = (by_z - z * torch.einsum("rc,rc->r", by_z, z)[:, None] / columns) * rstd
        if s["d_sum"] is not None:
            dx = dx + s["d_sum"].double()
        return {"dx": dx, "d_weight": torch.einsum("rc,rc->c", dy, z)}
    total = s["x"].double() if s["residual"] is None else s["x"].double() + s["residual"].double()
    h = total.to(_TYPES[case["type"]]).double()          # the norm is that of the sum as it is kept
    rstd = 1 / torch.sqrt(torch.einsum("rc,rc->r", h, h) / columns + EPSILON)
    y = h * rstd[:, None] * weight
    out = {"rstd": rstd}
    if s["residual"] is not None:
        out["sum"] = total
    if case["out"] != "codes":
        out["y"] = y
    if case["out"] != "bf16":
        scales = torch.empty(rows, _blocks(columns), dtype=torch.float64, device="cuda")
        codes = torch.empty(rows, columns, dtype=torch.float64, device="cuda")
        for b in range(_blocks(columns)):
            part = y[:, b * BLOCK:(b + 1) * BLOCK]
            scales[:, b] = (part.abs().amax(1) / LARGEST).clamp(min=SMALLEST)
            codes[:, b * BLOCK:(b + 1) * BLOCK] = (part / scales[:, b:b + 1]).float().to(torch.float8_e4m3fn).double()
        out["codes"], out["scales"] = codes, scales
    return out
