"""The feed-forward half of a layer, as cases that can be timed and compared: products with bias, activation, gate and residual in their epilogue and
their gradients, the same grouped by expert with ragged numbers of rows, the router that makes the groups, and the rows' way back to their tokens.

`listed()` names the cases, `draw()` gives further ones of the same ranges, `prepare()` makes what a program holds before the call,
`run()` is one call: through the package where `own` is true, in elementary torch operations in 32 bits where it is not.
"""
import math

import torch

own = False

TORCH = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"f16": 2, "bf16": 2, "f32": 4}
SCRATCH = 64 << 20  # bytes of workspace that a program keeps for all its calls


def _linear(name, dtype, out, rows, n, k, act="none", bias=False, gate=False, residual=False, keep=False, groups=1, gather=False):
    return {"name": name, "op": "linear", "dtype": dtype, "out": out, "rows": rows, "n": n, "k": k, "act": act, "bias": bias, "gate": gate,
            "residual": residual, "keep": keep, "groups": groups, "gather": gather}


def _backward(name, dtype, grad, rows, n, k, act="none", bias=False, gate=False, groups=1):
    return {"name": name, "op": "backward", "dtype": dtype, "grad": grad, "rows": rows, "n": n, "k": k, "act": act, "bias": bias, "gate": gate,
            "groups": groups}


def _route(name, dtype, tokens, experts, top, score, chosen_only, bias=False, backward=False):
    return {"name": name, "op": "route_backward" if backward else "route", "dtype": dtype, "tokens": tokens, "experts": experts, "top": top,
            "score": score, "chosen_only": chosen_only, "bias": bias, "scale": 2.5 if score == "sigmoid" else 1.0}


def _rows(name, op, dtype, tokens, top, width, weighted=True, residual=False):
    return {"name": name, "op": op, "dtype": dtype, "tokens": tokens, "top": top, "width": width, "weighted": weighted, "residual": residual}


def listed():
    return [
        # one token through a small layer: latency and host time are what count
        _linear("linear_1_small", "bf16", "bf16", 1, 1024, 2048, act="gelu", bias=True),
        # a batch in training, the wide layer: bias and activation in the epilogue, its argument kept for the gradient
        _linear("linear_train", "bf16", "bf16", 4000, 8192, 4096, act="gelu_tanh", bias=True, keep=True),
        # a ragged batch through a ragged layer, summed with the residual in 32 bits
        _linear("linear_ragged_f32", "f16", "f32", 1003, 4618, 3080, bias=True, residual=True),
        # the gradient of a gated layer: of its input, weights, bias and gate
        _backward("linear_backward", "bf16", "bf16", 4099, 4096, 4096, act="silu", bias=True, gate=True),
        # a step of eight tokens with two experts each out of 32: the bytes of the weights of those that are met
        _linear("experts_step", "bf16", "bf16", 16, 4096, 4096, act="silu", gate=True, groups=32, gather=True),
        # a prompt over 64 experts of uneven load
        _linear("experts_prompt", "f16", "f16", 16384, 2048, 2048, act="silu", gate=True, groups=64, gather=True),
        # the gradient of the experts' second product, weights' gradients in 32 bits
        _backward("experts_backward", "f16", "f32", 8195, 4096, 1536, groups=16),
        # the router for a step: latency
        _route("route_step", "bf16", 8, 64, 6, "softmax", True),
        # the router for a prompt over many experts, with the bias that evens out their load
        _route("route_prompt", "f32", 16384, 256, 8, "sigmoid", True, bias=True),
        # its gradient
        _route("route_backward", "bf16", 16001, 128, 4, "softmax", False, backward=True),
        # the experts' results put together with the residual
        _rows("combine_prompt", "combine", "bf16", 8192, 8, 4096, residual=True),
        # the gradient of that: of every expert's rows and of the router's weights
        _rows("combine_backward", "dispatch", "f16", 4099, 2, 2832),
    ]


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 100)


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _one(rng):
    op = rng.choice(["linear", "linear", "experts", "experts", "backward", "experts_backward", "route", "route_backward", "combine", "dispatch"])
    dtype = rng.choice(["f16", "bf16"])
    act = rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"])
    gate = act != "none" and rng.random() < 0.4
    groups = 1 if op in ("linear", "backward") else rng.choice([4, 8, 16, 32, 64, 128])
    if op in ("linear", "experts"):
        return _linear("", dtype, rng.choice([dtype, dtype, "f32"]), _log(rng, 1, 16384), _log(rng, 100, 8192), 8 * _log(rng, 32, 1024), act, rng.random() < 0.5,
                       gate, not gate and rng.random() < 0.3, rng.random() < 0.3, groups, groups > 1 and rng.random() < 0.5)
    if op in ("backward", "experts_backward"):  # (what the activation's gradient is rounded to is 16 bits: gradients in 32 bits where there is none)
        return _backward("", dtype, rng.choice([dtype, "f32"]) if act == "none" else dtype, _log(rng, 16, 16384), 8 * _log(rng, 32, 1024), 8 * _log(rng, 32, 1024), act,
                         rng.random() < 0.5, gate, groups)
    if op in ("route", "route_backward"):
        experts = rng.choice([8, 16, 40, 64, 128, 160, 256])
        return _route("", rng.choice([dtype, "f32"]), _log(rng, 1, 32768), experts, rng.choice([1, 2, 4, 6, 8]), rng.choice(["softmax", "sigmoid"]), rng.random() < 0.5,
                      op == "route" and rng.random() < 0.3, op == "route_backward")
    return _rows("", op, dtype, _log(rng, 1, 16384), rng.choice([1, 2, 4, 6, 8]), 8 * _log(rng, 32, 1024), rng.random() < 0.7, op == "combine" and rng.random() < 0.5)


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        case = _one(rng)
        del case["name"]
        # (the plain form keeps the weights of all groups in 32 bits)
        if _cost(case) <= most and case.get("groups", 1) * case.get("n", 0) * case.get("k", 0) <= 64 * 4096 * 4096:
            return case


def _sizes(case):
    """Rows of each group, uneven, and some with none: what the experts of a prompt or a step get."""
    groups, rows = case["groups"], case["rows"]
    share = [0.1 + ((g + 1) * 0.618033989) % 1 for g in range(groups)]
    upto = [int(rows * sum(share[: g + 1]) / sum(share) + 0.5) for g in range(groups)]
    return [b - a for a, b in zip([0] + upto, upto)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    t = TORCH[case["dtype"]]
    s = dict(case)
    s["scratch"] = torch.empty(SCRATCH, dtype=torch.uint8, device="cuda")
    if case["op"] in ("linear", "backward"):
        rows, n, k, groups = case["rows"], case["n"], case["k"], case["groups"]
        order = torch.randperm(groups, generator=g, device="cuda").tolist()  # which expert has how many rows
        sizes = [_sizes(case)[i] for i in order]
        s["most"] = max(sizes)
        s["offsets"] = torch.tensor([sum(sizes[:i]) for i in range(groups + 1)], dtype=torch.int32).cuda() if groups > 1 else None
        s["w"] = torch.empty(groups, n, k, dtype=t, device="cuda").normal_(0.0, 1.0 / math.sqrt(k), generator=g)
        s["bias"] = normal(groups, n).to(t) if case["bias"] else None
        s["gate"] = normal(rows, n).to(t) if case["gate"] else None
        if case["op"] == "linear":
            x_rows = max(1, rows // 2) if case["gather"] else rows
            s["x"] = normal(x_rows, k).to(t)
            s["source"] = torch.randint(0, x_rows, (rows,), generator=g, device="cuda", dtype=torch.int32) if case["gather"] else None
            s["c"] = normal(rows, n).to(TORCH[case["out"]]) if case["residual"] else None
            return s
        s["x"] = normal(rows, k).to(t)
        s["dy"] = normal(rows, n).to(t)
        s["z"] = normal(rows, n).to(t) if case["act"] != "none" else None  # what the forward call kept
        return s
    if case["op"] in ("route", "route_backward"):
        s["logits"] = (normal(case["tokens"], case["experts"]) * 1.5).to(t)
        s["bias"] = normal(case["experts"]) * 0.1 if case["bias"] else None
        if case["op"] == "route_backward":
            s["chosen"] = torch.sort(s["logits"].float(), dim=1, descending=True, stable=True)[1][:, : case["top"]].to(torch.int32).contiguous()
            s["dweights"] = normal(case["tokens"], case["top"])
        return s
    tokens, top, width = case["tokens"], case["top"], case["width"]
    s["place"] = torch.randperm(tokens * top, generator=g, device="cuda").to(torch.int32).view(tokens, top)
    s["weights"] = torch.rand(tokens, top, generator=g, device="cuda") if case["weighted"] else None
    s["values"] = normal(tokens * top, width).to(t)  # the experts' results
    s["x"] = normal(tokens, width).to(t)  # the residual, or the gradient of the sum
    return s


def run(s):
    return {"linear": _run_linear, "backward": _run_backward, "route": _run_route, "route_backward": _run_route_backward, "combine": _run_combine,
            "dispatch": _run_dispatch}[s["op"]](s)


def _activation(z, act):
    if act == "relu":
        return torch.where(z > 0, z, 0.0)
    if act == "gelu":
        return z * 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return z * 0.5 * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))
    return z * torch.sigmoid(z) if act == "silu" else z


def _slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    if act == "gelu_tanh":
        th = torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z))
        return 0.5 * (1.0 + th) + 0.5 * z * (1.0 - th * th) * math.sqrt(2.0 / math.pi) * (1.0 + 0.134145 * z * z)
    p = torch.sigmoid(z)
    return p * (1.0 + z * (1.0 - p)) if act == "silu" else torch.ones_like(z)


def _groups_of(s):
    """Of every row: its group, and its place among the rows of all groups, each filled up to the longest."""
    row = torch.arange(s["rows"], device="cuda")
    group = torch.bucketize(row, s["offsets"][1:].long(), right=True)
    return group, group * s["most"] + row - s["offsets"].long()[group]


def _filled(a, at, s):
    """The rows of a as a batch of groups, filled up with zeros"""
    b = torch.zeros(s["groups"] * s["most"], a.shape[1], device="cuda")
    b[at] = a
    return b.view(s["groups"], s["most"], a.shape[1])


def _run_linear(s):
    rows, n, k, groups, act = s["rows"], s["n"], s["k"], s["groups"], s["act"]
    if own:
        import rocwmma_amd as R

        types = {"f16": R.F16, "bf16": R.BF16, "f32": R.F32}
        y = torch.empty(rows, n, dtype=TORCH[s["out"]], device="cuda")
        z = torch.empty(rows, n, dtype=s["x"].dtype, device="cuda") if s["keep"] else None
        R.linear(types[s["dtype"]], types[s["out"]], rows, n, k, s["x"], s["w"], y, bias=s["bias"], activation=getattr(R, "ACT_" + act.upper()), gate=s["gate"],
                 c=s["c"], z=z, groups=groups, offsets=s["offsets"], source=s["source"], x_rows=s["x"].shape[0], workspace=s["scratch"])
        return [y, z] if s["keep"] else y
    x = s["x"].float()
    if s["gather"]:
        x = x[s["source"].long()]
    if groups == 1:
        z = x @ s["w"][0].float().t()
        group = torch.zeros(rows, dtype=torch.int64, device="cuda")
    else:
        group, at = _groups_of(s)
        z = (_filled(x, at, s) @ s["w"].float().transpose(1, 2)).view(-1, n)[at]
    if s["bias"] is not None:
        z = z + s["bias"].float()[group]
    y = _activation(z, act)
    if s["gate"] is not None:
        y = y * s["gate"].float()
    if s["c"] is not None:
        y = y + s["c"].float()
    y = y.to(TORCH[s["out"]])
    return [y, z.to(s["x"].dtype)] if s["keep"] else y


def _run_backward(s):
    rows, n, k, groups, act, t = s["rows"], s["n"], s["k"], s["groups"], s["act"], s["x"].dtype
    if own:
        import rocwmma_amd as R

        types = {"f16": R.F16, "bf16": R.BF16, "f32": R.F32}
        dx = torch.empty(rows, k, dtype=t, device="cuda")
        dw = torch.empty(groups, n, k, dtype=TORCH[s["grad"]], device="cuda")
        dbias = torch.empty(groups, n, dtype=torch.float32, device="cuda") if s["bias"] is not None else None
        dgate = torch.empty(rows, n, dtype=t, device="cuda") if s["gate"] is not None else None
        dz = torch.empty(rows, n, dtype=t, device="cuda") if act != "none" else None
        R.linear_backward(types[s["dtype"]], types[s["grad"]], rows, n, k, s["dy"], s["x"], s["w"], dx=dx, dw=dw, dbias=dbias, z=s["z"],
                          activation=getattr(R, "ACT_" + act.upper()), gate=s["gate"], dgate=dgate, dz=dz, groups=groups, offsets=s["offsets"], workspace=s["scratch"])
        return {"dx": dx, "dw": dw, "dbias": dbias, "dgate": dgate}
    dz, x, dgate, dbias = s["dy"].float(), s["x"].float(), None, None
    if act != "none":
        z = s["z"].float()
        if s["gate"] is not None:
            dgate = (dz * _activation(z, act)).to(t)
            dz = dz * s["gate"].float()
        dz = dz * _slope(z, act)
    if groups == 1:
        dx, dw = dz @ s["w"][0].float(), (dz.t() @ x)[None]
        sums = dz.sum(0, keepdim=True)
    else:
        _, at = _groups_of(s)
        filled = _filled(dz, at, s)
        dx = (filled @ s["w"].float()).view(-1, k)[at]
        dw = filled.transpose(1, 2) @ _filled(x, at, s)
        sums = filled.sum(1)
    if s["bias"] is not None:
        dbias = sums
    return {"dx": dx.to(t), "dw": dw.to(TORCH[s["grad"]]), "dbias": dbias, "dgate": dgate}


def _run_route(s):
    tokens, experts, top = s["tokens"], s["experts"], s["top"]
    if own:
        import rocwmma_amd as R

        weights = torch.empty(tokens, top, dtype=torch.float32, device="cuda")
        chosen, place = (torch.empty(tokens, top, dtype=torch.int32, device="cuda") for _ in range(2))
        source, offsets = torch.empty(tokens * top, dtype=torch.int32, device="cuda"), torch.empty(experts + 1, dtype=torch.int32, device="cuda")
        R.route({"f16": R.F16, "bf16": R.BF16, "f32": R.F32}[s["dtype"]], tokens, experts, top, s["logits"], weights, chosen, place, source, offsets,
                score=R.ROUTE_SOFTMAX if s["score"] == "softmax" else R.ROUTE_SIGMOID, chosen_only=s["chosen_only"], scale=s["scale"], bias=s["bias"],
                workspace=s["scratch"])
        return [weights, chosen, place, source, offsets]
    x = s["logits"].float()
    by = x if s["bias"] is None else x + s["bias"]
    chosen = torch.sort(by, dim=1, descending=True, stable=True)[1][:, :top]  # of equal ones the lowest first
    p = _scores(x, s["score"])
    w = p.gather(1, chosen)
    if s["chosen_only"]:
        w = w / w.sum(1, keepdim=True)
    flat = chosen.reshape(-1)
    order = torch.sort(flat, stable=True)[1]
    place = torch.empty_like(flat)
    place[order] = torch.arange(tokens * top, device="cuda")
    count = torch.zeros(experts + 1, dtype=torch.int64, device="cuda")
    count.index_add_(0, flat + 1, torch.ones_like(flat))
    return [w * s["scale"], chosen.to(torch.int32), place.view(tokens, top).to(torch.int32), (order // top).to(torch.int32), count.cumsum(0).to(torch.int32)]


def _scores(x, score):
    if score == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-x))
    e = torch.exp(x - x.amax(1, keepdim=True))
    return e / e.sum(1, keepdim=True)


def _run_route_backward(s):
    tokens, experts, top = s["tokens"], s["experts"], s["top"]
    if own:
        import rocwmma_amd as R

        dlogits = torch.empty_like(s["logits"])
        R.route_backward({"f16": R.F16, "bf16": R.BF16, "f32": R.F32}[s["dtype"]], tokens, experts, top, s["logits"], s["chosen"], s["dweights"], dlogits,
                         score=R.ROUTE_SOFTMAX if s["score"] == "softmax" else R.ROUTE_SIGMOID, chosen_only=s["chosen_only"], scale=s["scale"])
        return dlogits
    x, chosen = s["logits"].float(), s["chosen"].long()
    p = _scores(x, s["score"])
    g = s["dweights"] * s["scale"]
    if s["chosen_only"]:  # of w / sum w
        w = p.gather(1, chosen)
        total = w.sum(1, keepdim=True)
        g = (g - (g * w / total).sum(1, keepdim=True)) / total
    dp = torch.zeros_like(p).scatter_(1, chosen, g)
    if s["score"] == "sigmoid":
        d = dp * p * (1.0 - p)
    else:
        d = p * (dp - (dp * p).sum(1, keepdim=True))
    return d.to(s["logits"].dtype)


def _run_combine(s):
    tokens, top, width, t = s["tokens"], s["top"], s["width"], s["values"].dtype
    c = s["x"] if s["residual"] else None
    if own:
        import rocwmma_amd as R

        y = torch.empty(tokens, width, dtype=t, device="cuda")
        R.combine({"f16": R.F16, "bf16": R.BF16}[s["dtype"]], tokens, top, width, s["values"], tokens * top, s["place"], y, weights=s["weights"], c=c)
        return y
    v = s["values"].float()[s["place"].long()]
    y = (v * s["weights"][..., None]).sum(1) if s["weighted"] else v.sum(1)
    return (y if c is None else y + c.float()).to(t)


def _run_dispatch(s):
    tokens, top, width, t = s["tokens"], s["top"], s["width"], s["values"].dtype
    if own:
        import rocwmma_amd as R

        rows = torch.empty(tokens * top, width, dtype=t, device="cuda")
        dweights = torch.empty(tokens, top, dtype=torch.float32, device="cuda") if s["weighted"] else None
        R.dispatch({"f16": R.F16, "bf16": R.BF16}[s["dtype"]], tokens, top, width, s["x"], rows, tokens * top, s["place"], weights=s["weights"],
                   values=s["values"] if s["weighted"] else None, dweights=dweights)
        return [rows, dweights] if s["weighted"] else rows
    x, at = s["x"].float(), s["place"].long()
    rows = torch.zeros(tokens * top, width, dtype=t, device="cuda")
    rows[at] = ((x[:, None] * s["weights"][..., None]) if s["weighted"] else x[:, None].expand(tokens, top, width)).to(t)
    return [rows, (s["values"].float()[at] * x[:, None]).sum(2)] if s["weighted"] else rows


def work(case):
    e = BYTES[case["dtype"]]
    if case["op"] in ("linear", "backward"):
        rows, n, k = case["rows"], case["n"], case["k"]
        met = sum(v > 0 for v in _sizes(case))
        if case["op"] == "linear":
            x_rows = max(1, rows // 2) if case["gather"] else rows
            each = BYTES[case["out"]] * (2 if case["residual"] else 1) + e * (case["gate"] + case["keep"])
            index = (4 * rows if case["gather"] else 0) + (4 * case["groups"] if case["groups"] > 1 else 0)
            return {"bytes": x_rows * k * e + met * n * k * e + rows * n * each + (met * n * e if case["bias"] else 0) + index, "flops": 2.0 * rows * n * k}
        each = e * (1 + (case["act"] != "none") + 2 * case["gate"])
        return {"bytes": rows * n * each + 2 * rows * k * e + met * n * k * e + case["groups"] * n * (k * BYTES[case["grad"]] + (4 if case["bias"] else 0)),
                "flops": 4.0 * rows * n * k}
    if case["op"] in ("route", "route_backward"):
        tokens, experts, top = case["tokens"], case["experts"], case["top"]
        if case["op"] == "route":
            return {"bytes": tokens * (experts * e + 16 * top) + 4 * experts * (2 if case["bias"] else 1), "flops": 4.0 * tokens * experts}
        return {"bytes": tokens * (2 * experts * e + 8 * top), "flops": 6.0 * tokens * experts}
    tokens, top, width = case["tokens"], case["top"], case["width"]
    index = tokens * top * (8 if case["weighted"] else 4)
    if case["op"] == "combine":
        return {"bytes": tokens * width * e * (top + 1 + case["residual"]) + index, "flops": 2.0 * tokens * top * width}
    return {"bytes": tokens * width * e * (1 + top * (2 if case["weighted"] else 1)) + index + (tokens * top * 4 if case["weighted"] else 0),
            "flops": (3.0 if case["weighted"] else 1.0) * tokens * top * width}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("linear", "backward"):
        start = s["offsets"].tolist() if case["groups"] > 1 else [0, case["rows"]]
        f = lambda name, a, b: None if s[name] is None else s[name][a:b].double()  # noqa: E731
        parts = []
        for e in range(case["groups"]):
            a, b = start[e], start[e + 1]
            w, z = s["w"][e].double(), None
            if case["op"] == "linear":
                x = s["x"].double()[s["source"][a:b].long()] if case["gather"] else s["x"][a:b].double()
                z = torch.addmm(torch.zeros((), dtype=torch.float64, device="cuda") if s["bias"] is None else s["bias"][e].double(), x, w.t())
                y, gate, c = _in_64(z, case["act"])[0], f("gate", a, b), f("c", a, b)
                parts.append((y * (1.0 if gate is None else gate) + (0.0 if c is None else c), z))
                continue
            dy, gate, x = f("dy", a, b), f("gate", a, b), f("x", a, b)
            value, slope = (None, 1.0) if case["act"] == "none" else _in_64(f("z", a, b), case["act"])
            dz = dy * slope * (1.0 if gate is None else gate)
            parts.append((dz @ w, (x.t() @ dz).t(), dz.sum(0) if case["bias"] else None, None if gate is None else dy * value))
        if case["op"] == "linear":
            y, z = (torch.cat([p[i] for p in parts]) for i in range(2))
            return [y, z] if case["keep"] else y
        return {"dx": torch.cat([p[0] for p in parts]), "dw": torch.stack([p[1] for p in parts]), "dbias": torch.stack([p[2] for p in parts]) if case["bias"] else None,
                "dgate": torch.cat([p[3] for p in parts]) if case["gate"] else None}
    if case["op"] in ("route", "route_backward"):
        x, top = s["logits"].double(), case["top"]
        if case["op"] == "route":  # (the choice goes by sums in 32 bits, where the bias is added)
            by = (s["logits"].float() + (0.0 if s["bias"] is None else s["bias"])).cpu().numpy()
            chosen = torch.from_numpy((-by).argsort(axis=1, kind="stable")[:, :top].copy()).cuda()
        else:
            chosen = s["chosen"].long()
        logw = torch.log_softmax(x, 1) if case["score"] == "softmax" else torch.nn.functional.logsigmoid(x)
        picked = logw.gather(1, chosen)
        w = (torch.softmax(picked, 1) if case["chosen_only"] else picked.exp()) * case["scale"]
        if case["op"] == "route":
            return [w, None, None, None, None]
        # d w_j / d x_i = w_j (d log w_j / d x_i): of the logarithm of a score 1 - s_i for sigmoid (its own), delta_ij - p_i for softmax
        g = s["dweights"].double() * w
        if case["chosen_only"]:
            g = g - w / case["scale"] * g.sum(1, keepdim=True)
        d = torch.zeros_like(x)
        if case["score"] == "sigmoid":
            return d.scatter_(1, chosen, g * torch.sigmoid(-x).gather(1, chosen))
        return d.scatter_(1, chosen, g) - g.sum(1, keepdim=True) * logw.exp()
    tokens, top = case["tokens"], case["top"]
    weights = s["weights"].double() if case["weighted"] else torch.ones(tokens, top, dtype=torch.float64, device="cuda")
    at, x = s["place"].long(), s["x"].double()
    if case["op"] == "combine":
        y = x.clone() if case["residual"] else torch.zeros_like(x)
        for j in range(top):
            y += weights[:, j, None] * s["values"][at[:, j]].double()
        return y
    rows = torch.empty(tokens * top, case["width"], dtype=torch.float64, device="cuda")
    for j in range(top):
        rows[at[:, j]] = weights[:, j, None] * x
    if not case["weighted"]:
        return rows
    return [rows, torch.stack([(x * s["values"][at[:, j]].double()).sum(1) for j in range(top)], 1)]


def _in_64(z, act):
    """The activation and its derivative"""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        return z.clamp(min=0.0), torch.heaviside(z, torch.zeros_like(z))
    if act == "gelu":
        cdf = torch.special.ndtr(z)
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / (2 * math.pi) ** 0.5
    u = z if act == "silu" else (8 / math.pi) ** 0.5 * (z + 0.044715 * z ** 3)  # (1 + tanh(u / 2)) / 2 is the sigmoid of u
    du = 1.0 if act == "silu" else (8 / math.pi) ** 0.5 * (1 + 3 * 0.044715 * z ** 2)
    p = torch.sigmoid(u)
    return z * p, p + z * p * (1 - p) * du
