"""One decoding step that verifies a tree of drafted tokens, as cases that can be timed and compared: the products with 4-bit weights,
the rotary positions with the append to the cache, and the attention of the drafted tokens over a paged cache.

`listed()` names the cases, `draw()` gives further ones of the same ranges, `prepare()` makes what a program holds before the call,
`run()` is one call: through the package where `own` is true, in elementary torch operations in 32 bits where it is not.
"""
import math

import numpy as np
import torch

own = False

TORCH = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"f16": 2, "bf16": 2, "f32": 4}
SCRATCH = 64 << 20  # bytes of workspace that a program keeps for all its calls


def _w4(name, dtype, out, tokens, n, k, group, zeros=False, residual=False):
    return {"name": name, "op": "w4", "dtype": dtype, "out": out, "tokens": tokens, "n": n, "k": k, "group": group, "zeros": zeros,
            "residual": residual}


def _rope(name, dtype, tokens, heads, kv_heads, dim, rotary, layout="half", append=True, inverse=False, first=0, base=10000.0, factor=1.0):
    return {"name": name, "op": "rope", "dtype": dtype, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "rotary": rotary, "layout": layout, "append": append, "inverse": inverse, "first": first, "base": base, "factor": factor}


def _tree(name, dtype, batch, nodes, kv, heads, kv_heads, dim, page=16):
    return {"name": name, "op": "tree", "dtype": dtype, "batch": batch, "nodes": nodes, "kv": kv, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "page": page}


def listed():
    return [
        # the smallest product, one token through a narrow layer: latency and host time are what count
        _w4("w4_1_small", "bf16", "bf16", 1, 1024, 2048, 128),
        # one token through a wide layer, with zero points: the bytes of the weights
        _w4("w4_1_wide", "f16", "f16", 1, 16384, 8192, 128, zeros=True),
        # a tree of drafted tokens through a ragged layer with small groups and zero points, sums kept in 32 bits for what adds them up
        _w4("w4_24_ragged", "bf16", "f32", 24, 10250, 4168, 32, zeros=True),
        # a prompt's tokens, residual added: the matrix cores
        _w4("w4_prompt", "bf16", "bf16", 1000, 8192, 4096, 64, residual=True),
        # a step of eight sequences: query and key heads rotated, keys and values written to their places in the cache
        _rope("rope_step", "bf16", 8, 32, 8, 128, 128, first=1900),
        # a prompt of the same
        _rope("rope_prompt", "f16", 8192, 32, 8, 128, 128),
        # neighbouring pairs, a quarter of each head, far positions with lengthened wavelengths, in single precision
        _rope("rope_far_f32", "f32", 3001, 12, 12, 96, 24, layout="interleaved", append=False, first=900001, base=500000.0, factor=8.0),
        # the gradient of a training step: rotated back
        _rope("rope_backward", "bf16", 4099, 24, 24, 64, 64, layout="interleaved", append=False, inverse=True),
        # one token of one sequence with a short cache: latency
        _tree("tree_1_short", "bf16", 1, 1, 700, 32, 8, 128),
        # one token each of a ragged batch: the bytes of the cache
        _tree("tree_1_batch", "bf16", 32, 1, 8192, 32, 8, 128),
        # drafted trees of a ragged batch
        _tree("tree_48_batch", "f16", 8, 48, 4099, 24, 4, 64, page=32),
        # the largest trees over a long cache: both the cache's bytes and the matrix cores
        _tree("tree_64_long", "bf16", 2, 64, 65600, 32, 8, 128, page=64),
    ]


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _one(rng):
    op = rng.choice(["w4", "rope", "tree"])
    dtype = rng.choice(["f16", "bf16"])
    if op == "w4":
        return _w4("", dtype, rng.choice([dtype, "f32"]), _log(rng, 1, 1024), _log(rng, 200, 16384), 8 * _log(rng, 64, 2048),
                   rng.choice([32, 64, 128]), rng.random() < 0.5, rng.random() < 0.5)
    if op == "rope":
        kv = rng.choice([1, 2, 4, 8, 12])
        dim = rng.choice([64, 80, 96, 128, 192, 256])
        return _rope("", rng.choice([dtype, "f32"]), _log(rng, 1, 16384), kv * rng.choice([1, 2, 4, 8]), kv, dim, rng.choice([dim, dim // 2, dim // 4]),
                     rng.choice(["half", "interleaved"]), rng.random() < 0.5, rng.random() < 0.3, _log(rng, 1, 1000000), rng.choice([10000.0, 500000.0]),
                     rng.choice([1.0, 4.0]))
    kv = rng.choice([1, 2, 4, 8])
    nodes = rng.choice([1, _log(rng, 2, 128)])
    return _tree("", dtype, _log(rng, 1, 32), nodes, nodes + _log(rng, 20, 65536), kv * rng.randint(1, 8), kv, rng.choice([64, 128, 256]), rng.choice([16, 32, 64]))


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        case = _one(rng)
        del case["name"]
        if case["op"] == "rope" and case["append"]:
            case["inverse"] = False
        # (the plain attention writes its scores out: as many of them as of the largest case at most)
        fits = case["op"] != "tree" or case["batch"] * case["heads"] * case["nodes"] * case["kv"] <= 2 * 32 * 64 * 65600
        if _cost(case) <= most and fits:
            return case


def _lengths(case):
    """Drafted tokens and cached positions (the drafted among them) of each sequence of a ragged batch."""
    b = np.arange(case["batch"])
    nodes = 1 + ((case["nodes"] - 1) * np.where(b == 0, 1.0, (b * 0.754877666) % 1)).astype(np.int64)
    kv = np.maximum(nodes + 1, (case["kv"] * np.where(b == 0, 1.0, 0.1 + 0.9 * ((b * 0.618033989) % 1))).astype(np.int64))
    return nodes, kv


def _frequencies(case):
    """Radians per position of each pair, in 64 bits: base^(-2 i / r); wavelengths that turn less than once in 8192 / 4 positions are
    lengthened by `factor`, those that turn more than four times as often kept, and those between are blended."""
    i = torch.arange(case["rotary"] // 2, dtype=torch.float64)
    f = case["base"] ** (-2.0 * i / case["rotary"])
    if case["factor"] == 1.0:
        return f
    keep = ((8192.0 * f / (2 * math.pi) - 1.0) / 3.0).clamp(0.0, 1.0)
    return f * (keep + (1.0 - keep) / case["factor"])


def _pack(nibbles):
    """The storage that the kernels read: blocks of 16 rows x 128 k, zeros past the edges (the layout is written out in the package's header)."""
    n, k = nibbles.shape
    full = torch.zeros((n + 15) // 16 * 16, (k + 127) // 128 * 128, dtype=torch.uint8, device=nibbles.device)
    full[:n, :k] = nibbles
    e = full.view(full.shape[0] // 16, 16, full.shape[1] // 128, 4, 4, 8).permute(0, 2, 4, 1, 3, 5)
    return (e[..., [0, 4, 1, 5]] | (e[..., [2, 6, 3, 7]] << 4)).contiguous().view(-1)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    t = TORCH[case["dtype"]]
    s = dict(case)
    if case["op"] == "w4":
        n, k, groups = case["n"], case["k"], -(-case["k"] // case["group"])
        s["rows"] = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device="cuda", generator=g)  # two weights a byte, the even k low
        s["packed"] = _pack(torch.stack([s["rows"] & 15, s["rows"] >> 4], -1).view(n, k))
        s["scales"] = ((0.5 + torch.rand(groups, n, generator=g, device="cuda")) * 0.2 / math.sqrt(k)).to(t)
        s["zero_points"] = torch.randint(5, 11, (groups, n), dtype=torch.uint8, device="cuda", generator=g) if case["zeros"] else None
        s["x"] = normal(case["tokens"], k).to(t)
        s["c"] = normal(case["tokens"], n).to(TORCH[case["out"]]) if case["residual"] else None
        return s
    if case["op"] == "rope":
        tokens, h, kv, d = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        s["qkv"] = normal(tokens, h + 2 * kv, d).to(t)  # what one product for all three leaves
        s["q_in"], s["k_in"], s["v_in"] = s["qkv"].split([h, kv, kv], 1)
        s["positions"] = (torch.arange(tokens, device="cuda") + case["first"]).to(torch.int32)
        turns = (_frequencies(case) / (2 * math.pi)).tolist()
        s["turns"] = torch.tensor([(v + 2 ** 63) % 2 ** 64 - 2 ** 63 for v in (int(x * 2.0 ** 64) for x in turns)], dtype=torch.int64).cuda()
        s["scale"] = 1.0 if case["factor"] == 1.0 else 0.1 * math.log(case["factor"]) + 1.0
        if case["append"]:
            s["slots"] = torch.randperm(tokens + 64, generator=g, device="cuda")[:tokens].to(torch.int32)
            s["k_cache"], s["v_cache"] = (torch.zeros(tokens + 64, kv, d, dtype=t, device="cuda") for _ in range(2))
        return s
    nodes, kv = _lengths(case)
    batch, page, d = case["batch"], case["page"], case["dim"]
    pages = -(-kv // page)
    order = torch.randperm(int(pages.sum()), generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(batch, int(pages.max()), dtype=torch.int32, device="cuda")
    at = 0
    for b in range(batch):
        table[b, : pages[b]] = order[at: at + pages[b]]
        at += int(pages[b])
    words = -(-case["nodes"] // 64)
    seen = np.zeros((int(nodes.sum()), words * 64), dtype=np.uint8)
    r, row = np.random.RandomState(seed % 2 ** 32), 0
    for b in range(batch):  # a token's parent is one of the few before it; it sees itself and what its parent sees
        for j in range(nodes[b]):
            if j:
                seen[row + j] = seen[row + max(0, j - 1 - int(r.exponential(3.0)))]
            seen[row + j, j] = 1
        row += int(nodes[b])
    s["mask"] = torch.from_numpy(np.packbits(seen, axis=1, bitorder="little").view(np.int64)).cuda()
    s["q_start"] = torch.from_numpy(np.concatenate([[0], np.cumsum(nodes)]).astype(np.int32)).cuda()
    s["kv_len"] = torch.from_numpy(kv.astype(np.int32)).cuda()
    s["table"], s["words"] = table, words
    s["q"] = (normal(int(nodes.sum()), case["heads"], d) * 2.0).to(t)
    s["k_cache"], s["v_cache"] = (torch.empty(int(pages.sum()) * page, case["kv_heads"], d, dtype=t, device="cuda").normal_(generator=g) for _ in range(2))
    s["most_kv"] = int(kv.max())
    s["scratch"] = torch.empty(SCRATCH, dtype=torch.uint8, device="cuda")
    return s


def run(s):
    return {"w4": _run_w4, "rope": _run_rope, "tree": _run_tree}[s["op"]](s)


def _run_w4(s):
    tokens, n, k, group = s["tokens"], s["n"], s["k"], s["group"]
    if own:
        import rocwmma_amd as R

        types = {"f16": R.F16, "bf16": R.BF16, "f32": R.F32}
        y = torch.empty(tokens, n, dtype=TORCH[s["out"]], device="cuda")
        R.w4_matmul(types[s["dtype"]], types[s["out"]], tokens, n, k, group, s["x"], s["packed"], s["scales"], y, zeros=s["zero_points"],
                    c=s["c"], beta=1.0 if s["residual"] else 0.0)
        return y
    q = torch.stack([s["rows"] & 15, s["rows"] >> 4], -1).view(n, k).float()
    of = torch.arange(k, device="cuda") // group
    zero = 8.0 if s["zero_points"] is None else s["zero_points"].float().t()[:, of]
    y = s["x"].float() @ ((q - zero) * s["scales"].float().t()[:, of]).t()
    if s["residual"]:
        y = y + s["c"].float()
    return y.to(TORCH[s["out"]])


def _run_rope(s):
    tokens, h, kv, d, r = s["tokens"], s["heads"], s["kv_heads"], s["dim"], s["rotary"]
    qkv, append = s["qkv"], s["append"]
    if own:
        import rocwmma_amd as R

        row = (h + 2 * kv) * d
        q = torch.empty(tokens, h, d, dtype=qkv.dtype, device="cuda")
        k = s["k_cache"] if append else torch.empty(tokens, kv, d, dtype=qkv.dtype, device="cuda")
        parts = [R.rope_part(s["q_in"], q, h, (row, d), (h * d, d)),
                 R.rope_part(s["k_in"], k, kv, (row, d), (kv * d, d), to_slots=append)]
        if append:
            parts.append(R.rope_part(s["v_in"], s["v_cache"], kv, (row, d), (kv * d, d), rotate=False, to_slots=True))
        R.rope({"f16": R.F16, "bf16": R.BF16, "f32": R.F32}[s["dtype"]], R.ROPE_HALF if s["layout"] == "half" else R.ROPE_INTERLEAVED, tokens, d, r,
               parts, s["positions"], s["turns"], scale=s["scale"], inverse=s["inverse"], slots=s["slots"] if append else None,
               slot_count=tokens + 64 if append else 0)
        return [q, k, s["v_cache"]] if append else [q, k]
    x = qkv[:, : h + kv].float()
    turn = ((s["positions"].long()[:, None] * s["turns"]) >> 32).float() * 2.0 ** -32  # the product wraps around with the turns
    cos, sin = (f(turn * (2 * math.pi))[:, None, :] * s["scale"] for f in (torch.cos, torch.sin))
    if s["inverse"]:
        sin = -sin
    if s["layout"] == "half":
        a, b = x[..., : r // 2], x[..., r // 2: r]
        y = torch.cat([a * cos - b * sin, a * sin + b * cos, x[..., r:]], -1)
    else:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        y = torch.cat([torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2), x[..., r:]], -1)
    y = y.to(qkv.dtype)
    if not append:
        return [y[:, :h].contiguous(), y[:, h:].contiguous()]
    at = s["slots"].long()
    s["k_cache"][at] = y[:, h:]
    s["v_cache"][at] = qkv[:, h + kv:]
    return [y[:, :h].contiguous(), s["k_cache"], s["v_cache"]]


def _run_tree(s):
    q, batch, h, kv, d, nodes = s["q"], s["batch"], s["heads"], s["kv_heads"], s["dim"], s["nodes"]
    total, group, scale = q.shape[0], h // kv, 1.0 / math.sqrt(d)
    if own:
        import rocwmma_amd as R

        out = torch.empty_like(q)
        lse = torch.empty(total, h, dtype=torch.float32, device="cuda")
        R.tree_attention({"f16": R.F16, "bf16": R.BF16}[s["dtype"]], batch, total, h, kv, d, q, s["k_cache"], s["v_cache"], out, s["table"],
                         s["page"], s["k_cache"].shape[0] // s["page"], s["q_start"], s["kv_len"], nodes, s["most_kv"], mask=s["mask"],
                         mask_words=s["words"], lse=lse, scale=scale, workspace=s["scratch"])
        return [out, lse]
    start = s["q_start"].long()
    count, node = start[1:] - start[:-1], torch.arange(nodes, device="cuda")
    row = torch.minimum(start[:-1, None] + node, start[-1] - 1)  # [batch, nodes]
    pos = torch.arange(s["most_kv"], device="cuda")
    slot = s["table"].long()[:, pos // s["page"]] * s["page"] + pos % s["page"]
    past = pos - (s["kv_len"].long() - count)[:, None]  # which drafted token a position holds; negative: the prefix
    bits = ((s["mask"][row][..., None] >> torch.arange(64, device="cuda")) & 1).flatten(-2).bool()
    at = past.clamp(0, nodes - 1)[:, None, :].expand(batch, nodes, -1)
    sees = (past < 0)[:, None, :] | ((past < count[:, None])[:, None, :] & bits.gather(2, at))
    score = q[row].float().view(batch, nodes, kv, group, d).permute(0, 2, 1, 3, 4).reshape(batch, kv, nodes * group, d) @ s["k_cache"][slot].float().permute(0, 2, 3, 1)
    score = (score * scale).view(batch, kv, nodes, group, -1).masked_fill(~sees[:, None, :, None, :], -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp(score - top)
    sums = p.sum(-1, keepdim=True)
    o = (p.view(batch, kv, nodes * group, -1) @ s["v_cache"][slot].float().permute(0, 2, 1, 3)).view(batch, kv, nodes, group, d)
    o = torch.where(sums > 0, o / sums, 0.0).permute(0, 2, 1, 3, 4).reshape(batch, nodes, h, d)
    lse = (top + torch.log(sums)).squeeze(-1).permute(0, 2, 1, 3).reshape(batch, nodes, h)
    token = torch.arange(total, device="cuda")
    seq = torch.bucketize(token, start[1:], right=True)
    return [o[seq, token - start[seq]].to(q.dtype), lse[seq, token - start[seq]]]


def work(case):
    e = BYTES[case["dtype"]]
    if case["op"] == "w4":
        t, n, k, groups = case["tokens"], case["n"], case["k"], -(-case["k"] // case["group"])
        o = BYTES[case["out"]]
        return {"bytes": n * k // 2 + groups * n * (e + (1 if case["zeros"] else 0)) + t * k * e + t * n * o * (2 if case["residual"] else 1),
                "flops": 2.0 * t * n * k}
    if case["op"] == "rope":
        heads = case["heads"] + case["kv_heads"]
        moved = heads + (case["kv_heads"] if case["append"] else 0)
        return {"bytes": 2 * case["tokens"] * moved * case["dim"] * e + case["tokens"] * 4 + case["rotary"] * 4,
                "flops": 3.0 * case["tokens"] * heads * case["rotary"]}
    nodes, kv = _lengths(case)
    rows = int(nodes.sum()) * case["heads"]
    seen = float((nodes * (kv - nodes) + nodes * (nodes + 1) / 2).sum()) * case["heads"]  # at most: a chain sees this many
    return {"bytes": int(kv.sum()) * case["kv_heads"] * case["dim"] * 2 * e + rows * (2 * case["dim"] * e + 4), "flops": 4.0 * case["dim"] * seen}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "w4":
        n, k, group = case["n"], case["k"], case["group"]
        w = torch.empty(n, k, dtype=torch.float64, device="cuda")
        w[:, 0::2], w[:, 1::2] = (s["rows"] % 16).double(), (s["rows"] // 16).double()
        y = torch.zeros(case["tokens"], n, dtype=torch.float64, device="cuda")
        for g in range(-(-k // group)):  # group by group: (sum of x q - z sum of x) s
            x = s["x"][:, g * group: (g + 1) * group].double()
            z = 8.0 if s["zero_points"] is None else s["zero_points"][g].double()
            y += (x @ w[:, g * group: (g + 1) * group].t() - z * x.sum(1, keepdim=True)) * s["scales"][g].double()
        return y + s["c"].double() if case["residual"] else y
    if case["op"] == "rope":
        h, kv, r = case["heads"], case["kv_heads"], case["rotary"]
        x = s["qkv"].double()
        angle = s["positions"].double()[:, None] * _frequencies(case).cuda() * (-1.0 if case["inverse"] else 1.0)
        wave = torch.polar(torch.full_like(angle, s["scale"]), angle)[:, None, :]
        y = x[:, : h + kv].clone()
        first, second = (slice(0, r // 2), slice(r // 2, r)) if case["layout"] == "half" else (slice(0, r, 2), slice(1, r, 2))
        z = torch.complex(x[:, : h + kv, first], x[:, : h + kv, second]) * wave
        y[..., first], y[..., second] = z.real, z.imag
        if not case["append"]:
            return [y[:, :h], y[:, h:]]
        at = s["slots"].long()
        k_cache, v_cache = s["k_cache"].double(), s["v_cache"].double()
        k_cache[at], v_cache[at] = y[:, h:], x[:, h + kv:]
        return [y[:, :h], k_cache, v_cache]
    nodes, kv = _lengths(case)
    group, page, start = case["heads"] // case["kv_heads"], case["page"], s["q_start"].tolist()
    seen = np.unpackbits(s["mask"].cpu().numpy().view(np.uint8), axis=1, bitorder="little")
    out, lse = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), torch.zeros(s["q"].shape[:2], dtype=torch.float64, device="cuda")
    for b in range(case["batch"]):
        n, length = int(nodes[b]), int(kv[b])
        at = (s["table"][b].long()[:, None] * page + torch.arange(page, device="cuda")).flatten()[:length]
        left = torch.zeros(n, length, dtype=torch.float64, device="cuda")
        left[:, length - n:] = torch.from_numpy(np.where(seen[start[b]: start[b] + n, :n] > 0, 0.0, -np.inf)).cuda()
        for head in range(case["heads"]):
            score = s["q"][start[b]: start[b + 1], head].double() @ s["k_cache"][at, head // group].double().t() / math.sqrt(case["dim"]) + left
            lse[start[b]: start[b + 1], head] = torch.logsumexp(score, -1)
            out[start[b]: start[b + 1], head] = torch.softmax(score, -1) @ s["v_cache"][at, head // group].double()
    return [out, lse]
