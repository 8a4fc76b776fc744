"""Measured cases of the 8-bit block-scaled operators and of the router's balance loss, through the
public entry points, from one decoded token to a prefill or training batch.

Every case is a dict of plain values; ``op`` names the operator:

* ``quantize``   a matrix to E4M3 with one f32 scale per block of 128: of a row's columns (activations),
  of a column's rows, transposed (both operands of a weight gradient), or of 128 x 128 (weights).
* ``linear``     y = x W^T with x bf16, quantised by rows within the call, and W held in 128 x 128 blocks.
* ``gradients``  that product's gradients: by its input, from W laid out transposed, and by its weight.
* ``experts``    the routed experts on such tables: gate, up, activation, down, weighted sum, for
  given expert ids and weights.
* ``balance``    counts per expert, balance loss and mean scores of ragged sequences, and the gradient of
  loss and routing weights by the router's logits.

Inputs have the distributions that the path meets: activations N(0, 1) with a few columns 20 times as
large, gradients N(0, 1e-3), weights N(0, 0.02), routing by scores with a Zipf or a uniform bias.
"""
import math

import torch

own = False

HIDDEN, EXPERT_HIDDEN, LATENT, EXPERTS, TOP_K = 7168, 2048, 3584, 896, 16   # the benchmark layer and the latent shape
BLOCK, LARGEST, SMALLEST = 128, 448.0, 2.0 ** -126                     # block, largest E4M3 value, smallest scale
BETA, LINEAR_BETA, ROUTE_SCALE, TINY = 4.0, 25.0, 2.5, 1e-20
COEFFICIENT = 1e-2


def listed():
    return [
        # the activations of a prefill batch before its products
        {"name": "quantize_rows_8192", "op": "quantize", "form": "rows", "rows": 8192, "columns": HIDDEN, "type": "bf16"},
        # one operand of a weight gradient over an odd number of tokens
        {"name": "quantize_columns_1021", "op": "quantize", "form": "columns", "rows": 1021, "columns": LATENT, "type": "bf16"},
        # a projection of one decoded token
        {"name": "linear_1", "op": "linear", "tokens": 1, "rows": LATENT, "columns": HIDDEN},
        # the shared expert's down projection of a decode batch
        {"name": "linear_47", "op": "linear", "tokens": 47, "rows": HIDDEN, "columns": EXPERT_HIDDEN},
        # a latent projection of a prompt of odd length
        {"name": "linear_1021", "op": "linear", "tokens": 1021, "rows": LATENT, "columns": HIDDEN},
        # a square projection of a large prefill
        {"name": "linear_8192", "op": "linear", "tokens": 8192, "rows": HIDDEN, "columns": HIDDEN},
        # the backward pass of a projection in a training step
        {"name": "gradients_4096", "op": "gradients", "tokens": 4096, "rows": EXPERT_HIDDEN, "columns": HIDDEN},
        # the routed experts of one decoded token
        {"name": "experts_1", "op": "experts", "tokens": 1, "hidden": HIDDEN, "expert_hidden": EXPERT_HIDDEN,
         "experts": 64, "top_k": TOP_K, "bias": "uniform", "form": "swiglu"},
        # of a decode batch
        {"name": "experts_61", "op": "experts", "tokens": 61, "hidden": HIDDEN, "expert_hidden": EXPERT_HIDDEN,
         "experts": 64, "top_k": 8, "bias": "zipf", "form": "situ"},
        # of a prefill
        {"name": "experts_4096", "op": "experts", "tokens": 4096, "hidden": HIDDEN, "expert_hidden": EXPERT_HIDDEN,
         "experts": 64, "top_k": TOP_K, "bias": "uniform", "form": "swiglu"},
        # a few short sequences of odd lengths, softmax scores
        {"name": "balance_257", "op": "balance", "tokens": 257, "sequences": 5, "experts": 160, "top_k": 6, "score": "softmax"},
        # a training batch at the router's full width
        {"name": "balance_32768", "op": "balance", "tokens": 32768, "sequences": 16, "experts": EXPERTS, "top_k": TOP_K,
         "score": "sigmoid"},
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choices(["quantize", "linear", "gradients", "experts", "balance"], [3, 5, 2, 5, 4])[0]
    if op == "quantize":
        return {"op": op, "form": rng.choice(["rows", "columns", "blocks"]), "rows": _log_int(rng, 1, 8192),
                "columns": _log_int(rng, 16, HIDDEN), "type": rng.choice(["bf16", "f32"])}
    if op == "linear":
        return {"op": op, "tokens": _log_int(rng, 1, 8192), "rows": _log_int(rng, 16, HIDDEN), "columns": _log_int(rng, 16, HIDDEN)}
    if op == "gradients":
        return {"op": op, "tokens": _log_int(rng, 1, 4096), "rows": _log_int(rng, 16, EXPERT_HIDDEN), "columns": _log_int(rng, 16, HIDDEN)}
    if op == "experts":
        experts = _log_int(rng, 4, 64)
        return {"op": op, "tokens": _log_int(rng, 1, 4096), "hidden": 16 * _log_int(rng, 8, HIDDEN // 16),
                "expert_hidden": 16 * _log_int(rng, 4, EXPERT_HIDDEN // 16), "experts": experts,
                "top_k": rng.randint(1, min(TOP_K, experts)), "bias": rng.choice(["uniform", "zipf"]),
                "form": rng.choice(["swiglu", "situ"])}
    experts, tokens = _log_int(rng, 4, 1024), _log_int(rng, 1, 32768)
    return {"op": op, "tokens": tokens, "sequences": _log_int(rng, 1, 32), "experts": experts,
            "top_k": rng.randint(1, min(32, experts)), "score": rng.choice(["sigmoid", "softmax"])}


# ------------------------------------------------------------------------------------------ inputs
def _normal(g, *shape, scale=1.0, dtype=torch.bfloat16):
    return (torch.randn(*shape, generator=g, device="cuda", dtype=dtype) * scale).to(dtype)


def _activations(g, rows, columns, dtype=torch.bfloat16):
    x = _normal(g, rows, columns, dtype=dtype)
    x[:, ::97] *= 20                                     # the columns that stand out
    return x


def _pitch(n):
    return (n + 15) // 16 * 16


def _blocks(n):
    return (n + BLOCK - 1) // BLOCK


def _table(g, *shape):
    """E4M3 values of a weight table, rows padded to 16 bytes with zeros, and its scales per 128 x 128."""
    *lead, rows, columns = shape
    q = torch.zeros(*lead, rows, _pitch(columns), device="cuda", dtype=torch.float8_e4m3fn)
    q.view(torch.uint8)[..., :columns] = _normal(g, *lead, rows, columns, scale=110.0).clamp_(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    scales = (0.5 + torch.rand(*lead, _blocks(rows), _blocks(columns), generator=g, device="cuda")) * (0.02 / 110.0)
    return q, scales


def _transposed(q, scales, rows, columns):
    """The same table with rows and columns exchanged."""
    t = torch.zeros(columns, _pitch(rows), device="cuda", dtype=torch.float8_e4m3fn)
    t.view(torch.uint8)[:, :rows] = q.view(torch.uint8)[:, :columns].t()
    return t, scales.t().contiguous()


def _routes(g, tokens, experts, top_k, bias):
    logits = torch.randn(tokens, experts, generator=g, device="cuda")
    if bias == "zipf":
        logits -= torch.log(torch.arange(1, experts + 1, device="cuda").float())
    return logits, torch.topk(logits, top_k, dim=1).indices.to(torch.int32).contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, s = case["op"], {"case": case}
    if op == "quantize":
        kind = torch.bfloat16 if case["type"] == "bf16" else torch.float32
        s["x"] = _activations(g, case["rows"], case["columns"], kind)
    elif op == "linear":
        s["x"] = _activations(g, case["tokens"], case["columns"])
        s["w"], s["w_scales"] = _table(g, case["rows"], case["columns"])
    elif op == "gradients":
        s["x"] = _activations(g, case["tokens"], case["columns"])
        s["dy"] = _normal(g, case["tokens"], case["rows"], scale=1e-3)
        w, scales = _table(g, case["rows"], case["columns"])
        s["wt"], s["wt_scales"] = _transposed(w, scales, case["rows"], case["columns"])
    elif op == "experts":
        d, i, e = case["hidden"], case["expert_hidden"], case["experts"]
        s["x"] = _activations(g, case["tokens"], d)
        for name, rows, columns in (("w1", i, d), ("w3", i, d), ("w2", d, i)):
            s[name], s[name + "_scales"] = _table(g, e, rows, columns)
        logits, s["ids"] = _routes(g, case["tokens"], e, case["top_k"], case["bias"])
        chosen = torch.sigmoid(torch.gather(logits, 1, s["ids"].long()))
        s["weights"] = (chosen / chosen.sum(1, keepdim=True) * ROUTE_SCALE).contiguous()
    else:
        t, n = case["tokens"], case["sequences"]
        logits, s["ids"] = _routes(g, t, case["experts"], case["top_k"], "zipf")
        s["logits"] = logits.contiguous()
        cuts = torch.randint(0, t + 1, (n - 1,), generator=g, device="cuda").sort().values
        s["offsets"] = torch.cat([cuts.new_zeros(1), cuts, cuts.new_full((1,), t)]).to(torch.int32)
        s["d_loss"] = torch.rand(n, generator=g, device="cuda") + 0.5
        s["d_weights"] = torch.randn(t, case["top_k"], generator=g, device="cuda") * 1e-3
    if own:
        s["call"] = _handle(s)
    return s


# ------------------------------------------------------------------------------------------ the framework's calls
def _handle(s):
    """What a program keeps from call to call: the objects that hold tables and workspaces."""
    from moonshine_b200 import balance, fp8
    case = s["case"]
    op = case["op"]
    if op == "quantize":
        return getattr(fp8, "quantize_" + case["form"])
    if op == "linear":
        return fp8.Fp8Linear(s["w"], s["w_scales"], case["rows"], case["columns"])
    if op == "gradients":
        return fp8.Fp8LinearGradient(s["wt"], s["wt_scales"], case["rows"], case["columns"])
    if op == "experts":
        return fp8.Fp8Experts(s["w1"], s["w1_scales"], s["w3"], s["w3_scales"], s["w2"], s["w2_scales"], top_k=case["top_k"],
                              activation=case["form"], beta=BETA, linear_beta=LINEAR_BETA)
    return balance.RouterBalance(case["experts"], case["top_k"], score=case["score"], coefficient=COEFFICIENT,
                                 route_scale=ROUTE_SCALE)


def _run_own(s):
    op, call = s["case"]["op"], s["call"]
    if op == "quantize":
        q, scales = call(s["x"])
        rows, columns = s["x"].shape
        if s["case"]["form"] == "columns":
            return {"q": q[:, :rows], "scales": scales[:, :_blocks(rows)]}
        return {"q": q[:, :columns], "scales": scales[:, :_blocks(columns)]}
    if op == "linear":
        return call.forward(s["x"])
    if op == "gradients":
        return {"dx": call.by_input(s["dy"]), "dw": call.by_weight(s["dy"], s["x"])}
    if op == "experts":
        return call.forward(s["x"], s["ids"], s["weights"])
    counts, loss, means = call.forward(s["logits"], s["ids"], s["offsets"])
    d_logits = call.backward(s["logits"], s["ids"], counts, s["offsets"], s["d_loss"], s["d_weights"])
    return {"counts": counts, "loss": loss, "means": means, "d_logits": d_logits}


# ------------------------------------------------------------------------------------------ the plain form, in 32 bits
def _scale_of(largest):
    scale = torch.maximum(largest / torch.full_like(largest, LARGEST), torch.full_like(largest, SMALLEST))
    return torch.where(torch.isfinite(largest), scale, torch.full_like(scale, math.nan))


def _quantize(x):
    """[..., columns] -> E4M3 values and scales per 128 columns."""
    columns = x.shape[-1]
    padded = torch.nn.functional.pad(x.float(), (0, _blocks(columns) * BLOCK - columns))
    padded = padded.reshape(*x.shape[:-1], _blocks(columns), BLOCK)
    scales = _scale_of(padded.abs().amax(-1))
    q = (padded / scales.unsqueeze(-1)).to(torch.float8_e4m3fn)
    return q.reshape(*x.shape[:-1], -1)[..., :columns].contiguous(), scales


def _quantize_blocks(x):
    rows, columns = x.shape
    padded = torch.nn.functional.pad(x.float(), (0, _blocks(columns) * BLOCK - columns, 0, _blocks(rows) * BLOCK - rows))
    tiles = padded.reshape(_blocks(rows), BLOCK, _blocks(columns), BLOCK)
    scales = _scale_of(tiles.abs().amax((1, 3)))
    q = (tiles / scales[:, None, :, None]).to(torch.float8_e4m3fn)
    return q.reshape(padded.shape)[:rows, :columns].contiguous(), scales


def _values(q, scales):
    """What E4M3 rows with scales per 128 columns stand for."""
    return q.float() * scales.repeat_interleave(BLOCK, -1)[..., :q.shape[-1]]


def _table_values(q, scales, columns):
    full = scales.repeat_interleave(BLOCK, -2)[..., :q.shape[-2], :].repeat_interleave(BLOCK, -1)[..., :columns]
    return q[..., :columns].float() * full


def _activation(gate, up, form):
    if form == "swiglu":
        return gate * torch.sigmoid(gate) * up
    return BETA * torch.tanh(gate / BETA) * torch.sigmoid(gate) * (LINEAR_BETA * torch.tanh(up / LINEAR_BETA))


def _run_experts(s):
    case, e, k = s["case"], s["case"]["experts"], s["case"]["top_k"]
    x = _values(*_quantize(s["x"]))
    ids = s["ids"].long().reshape(-1)
    order = torch.argsort(ids, stable=True)
    counts = torch.bincount(ids, minlength=e)
    first = torch.cumsum(counts, 0) - counts
    expert = ids[order]
    place = torch.arange(ids.numel(), device=ids.device) - first[expert]
    rows = x.new_zeros(e, int(counts.max()), x.shape[1])
    rows[expert, place] = x[order // k]
    gate = torch.bmm(rows, _table_values(s["w1"], s["w1_scales"], case["hidden"]).transpose(1, 2))
    up = torch.bmm(rows, _table_values(s["w3"], s["w3_scales"], case["hidden"]).transpose(1, 2))
    act = _values(*_quantize(_activation(gate, up, case["form"])))
    down = torch.bmm(act, _table_values(s["w2"], s["w2_scales"], case["expert_hidden"]).transpose(1, 2))
    routed = torch.empty(ids.numel(), x.shape[1], device=x.device)
    routed[order] = down[expert, place]
    return (routed.reshape(-1, k, x.shape[1]) * s["weights"].unsqueeze(-1)).sum(1).to(torch.bfloat16)


def _scores(logits, score):
    """Scores of each expert, and what a token's scores are divided by in the balance loss."""
    if score == "sigmoid":
        p = torch.sigmoid(logits)
        return p, TINY + p.sum(1, keepdim=True)
    e = torch.exp(logits - logits.amax(1, keepdim=True))
    return e / e.sum(1, keepdim=True), logits.new_ones(logits.shape[0], 1)


def _balance(logits, ids, offsets, d_loss, d_weights, case):
    t, e, k, n = case["tokens"], case["experts"], case["top_k"], case["sequences"]
    sequence = torch.searchsorted(offsets[1:].long().contiguous(), torch.arange(t, device=logits.device), right=True)
    length = (offsets[1:] - offsets[:-1]).to(logits.dtype).clamp(min=1)
    counts = torch.bincount((sequence.unsqueeze(1) * e + ids.long()).reshape(-1), minlength=n * e).reshape(n, e)
    p, total = _scores(logits, case["score"])
    member = (sequence.unsqueeze(0) == torch.arange(n, device=logits.device).unsqueeze(1)).to(logits.dtype)
    means = (member @ (p / total)) / length.unsqueeze(1)
    share = counts.to(logits.dtype) * (e / k) / length.unsqueeze(1)
    loss = COEFFICIENT * (share * means).sum(1)
    # by the scores: of the loss, then of the routing weights scale * s_i / (tiny + sum of the chosen)
    f, c = share[sequence], (COEFFICIENT * d_loss.to(logits.dtype) / length)[sequence].unsqueeze(1)
    d_p = c * (f - (f * p / total).sum(1, keepdim=True)) / total if case["score"] == "sigmoid" else c * f
    chosen = torch.gather(p, 1, ids.long())
    under = TINY + chosen.sum(1, keepdim=True)
    dw = d_weights.to(logits.dtype)
    d_p = d_p.scatter_add(1, ids.long(), ROUTE_SCALE * (dw - (dw * chosen / under).sum(1, keepdim=True)) / under)
    d_logits = d_p * p * (1 - p) if case["score"] == "sigmoid" else p * (d_p - (d_p * p).sum(1, keepdim=True))
    return {"counts": counts.to(torch.int32), "loss": loss, "means": means, "d_logits": d_logits}


def run(s):
    if own:
        return _run_own(s)
    case = s["case"]
    op = case["op"]
    if op == "quantize":
        if case["form"] == "blocks":
            q, scales = _quantize_blocks(s["x"])
        else:
            q, scales = _quantize(s["x"].t() if case["form"] == "columns" else s["x"])
        return {"q": q, "scales": scales}
    if op == "linear":
        return (_values(*_quantize(s["x"])) @ _table_values(s["w"], s["w_scales"], case["columns"]).t()).to(torch.bfloat16)
    if op == "gradients":
        dx = _values(*_quantize(s["dy"])) @ _table_values(s["wt"], s["wt_scales"], case["rows"]).t()
        dw = _values(*_quantize(s["dy"].t())) @ _values(*_quantize(s["x"].t())).t()
        return {"dx": dx.to(torch.bfloat16), "dw": dw}
    if op == "experts":
        return _run_experts(s)
    return _balance(s["logits"], s["ids"], s["offsets"], s["d_loss"], s["d_weights"], case)


# ------------------------------------------------------------------------------------------ what a pass needs
def work(case):
    op = case["op"]
    if op == "quantize":
        r, c = case["rows"], case["columns"]
        across = {"rows": r * _blocks(c), "columns": c * _blocks(r), "blocks": _blocks(r) * _blocks(c)}[case["form"]]
        return {"bytes": r * c * (3 if case["type"] == "bf16" else 5) + 4 * across, "flops": 3 * r * c}
    if op == "linear":
        t, n, k = case["tokens"], case["rows"], case["columns"]
        return {"bytes": 2 * t * k + n * k + 4 * _blocks(n) * _blocks(k) + 2 * t * n, "flops": 2 * t * n * k}
    if op == "gradients":
        t, n, k = case["tokens"], case["rows"], case["columns"]
        return {"bytes": 2 * t * n + 2 * t * k + n * k + 4 * _blocks(n) * _blocks(k) + 2 * t * k + 4 * n * k, "flops": 4 * t * n * k}
    if op == "experts":
        t, d, i, e, k = case["tokens"], case["hidden"], case["expert_hidden"], case["experts"], case["top_k"]
        touched = e * (1 - (1 - k / e) ** t)             # experts that some token selects, for a uniform choice
        return {"bytes": int(touched * 3 * d * i + 4 * t * d + 8 * t * k), "flops": 6 * t * k * d * i}
    t, e, k, n = case["tokens"], case["experts"], case["top_k"], case["sequences"]
    return {"bytes": 8 * t * e + 8 * t * k + 8 * n * e + 12 * n, "flops": 20 * t * e}


# ------------------------------------------------------------------------------------------ the definition, in 64 bits
def _exact_blocks(x, rows_of):
    """The values that blocks of rows_of x 128 of x stand for after quantisation, their codes and scales."""
    rows, columns = x.shape
    up, across = -(-rows // rows_of), _blocks(columns)
    full = torch.zeros(up * rows_of, across * BLOCK, dtype=torch.float64, device=x.device)
    full[:rows, :columns] = x.double()
    tiles = full.view(up, rows_of, across, BLOCK)
    scales = (tiles.abs().amax((1, 3)) / LARGEST).clamp(min=SMALLEST)
    per = scales[:, None, :, None]
    codes = (tiles / per).float().to(torch.float8_e4m3fn).double()
    cut = lambda v: v.reshape(full.shape)[:rows, :columns]  # noqa: E731
    return cut(codes * per), cut(codes), scales


def _exact_table(q, scales, columns):
    out = q[:, :columns].double()
    for r in range(scales.shape[0]):
        out[r * BLOCK:(r + 1) * BLOCK] *= scales[r].double().repeat_interleave(BLOCK)[:columns]
    return out


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        x = s["x"].t() if case["form"] == "columns" else s["x"]
        _, codes, scales = _exact_blocks(x, BLOCK if case["form"] == "blocks" else 1)
        return {"q": codes, "scales": scales}
    if op == "linear":
        return _exact_blocks(s["x"], 1)[0] @ _exact_table(s["w"], s["w_scales"], case["columns"]).t()
    if op == "gradients":
        dx = _exact_blocks(s["dy"], 1)[0] @ _exact_table(s["wt"], s["wt_scales"], case["rows"]).t()
        dw = _exact_blocks(s["dy"].t(), 1)[0] @ _exact_blocks(s["x"].t(), 1)[0].t()
        return {"dx": dx, "dw": dw}
    if op == "experts":
        x = _exact_blocks(s["x"], 1)[0]
        out = torch.zeros_like(x)
        for e in range(case["experts"]):
            token, rank = (s["ids"] == e).nonzero(as_tuple=True)
            if token.numel() == 0:
                continue
            gate = x[token] @ _exact_table(s["w1"][e], s["w1_scales"][e], case["hidden"]).t()
            up = x[token] @ _exact_table(s["w3"][e], s["w3_scales"][e], case["hidden"]).t()
            sig = 1 / (1 + torch.exp(-gate))
            if case["form"] == "swiglu":
                act = gate * sig * up
            else:
                act = BETA * torch.tanh(gate / BETA) * sig * LINEAR_BETA * torch.tanh(up / LINEAR_BETA)
            down = _exact_blocks(act, 1)[0] @ _exact_table(s["w2"][e], s["w2_scales"][e], case["expert_hidden"]).t()
            out.index_add_(0, token, down * s["weights"][token, rank].double().unsqueeze(1))
        return out
    # balance: sequence by sequence, the gradient from the definition's quotient and product rules
    n, e, k = case["sequences"], case["experts"], case["top_k"]
    loss, means = s["logits"].new_zeros(n, dtype=torch.float64), s["logits"].new_zeros(n, e, dtype=torch.float64)
    d_logits = torch.zeros_like(s["logits"], dtype=torch.float64)
    cuts = s["offsets"].tolist()
    for q in range(n):
        begin, end = cuts[q], cuts[q + 1]
        if begin == end:
            continue
        logits, ids = s["logits"][begin:end].double(), s["ids"][begin:end].long()
        share = torch.zeros(e, dtype=torch.float64, device=logits.device)
        share.index_add_(0, ids.reshape(-1), torch.ones(ids.numel(), dtype=torch.float64, device=logits.device))
        share *= e / (k * (end - begin))
        p = torch.sigmoid(logits) if case["score"] == "sigmoid" else torch.softmax(logits, 1)
        z = p.sum(1, keepdim=True) + TINY if case["score"] == "sigmoid" else torch.ones_like(p[:, :1])
        means[q] = (p / z).mean(0)
        loss[q] = COEFFICIENT * (share * means[q]).sum()
        by = torch.zeros_like(p) + COEFFICIENT * s["d_loss"][q].double() / (end - begin) * share
        if case["score"] == "sigmoid":
            by = by / z - (by * p).sum(1, keepdim=True) / (z * z)
        chosen, dw = p.gather(1, ids), s["d_weights"][begin:end].double()
        d = chosen.sum(1, keepdim=True) + TINY
        by.scatter_add_(1, ids, ROUTE_SCALE * (dw / d - (dw * chosen).sum(1, keepdim=True) / (d * d)))
        d_logits[begin:end] = by * p * (1 - p) if case["score"] == "sigmoid" else p * by - p * (p * by).sum(1, keepdim=True)
    return {"counts": None, "loss": loss, "means": means, "d_logits": d_logits}
