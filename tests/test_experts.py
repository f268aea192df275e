"""The router, the rows' way to the experts and back, and the gradients of both, against 64 bits.

Bounds, eps = 2^-24.  Weights: the exponentials are off by (|argument| + 2) eps, a sum of E of them by E eps more, quotient and scale by 3; a logarithm of a score by 4 eps of its size.
With arguments up to a = max |x - max x| that is (2 a + E + 12) eps relative to the weight (each of two exponentials).  Rows: sums of `top` products, (top + 2) eps sum |w v|."""
import math

import pytest

import rocwmma_amd as R

EPS = 2.0 ** -24
HALF = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": EPS}
TINY = {"f16": 2.0 ** -25, "bf16": 2.0 ** -134, "f32": 2.0 ** -126}
TYPES = {"f16": R.F16, "bf16": R.BF16, "f32": R.F32}
SCORES = {"softmax": R.ROUTE_SOFTMAX, "sigmoid": R.ROUTE_SIGMOID}


def _torch(name):
    import torch

    return {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}[name]


def _weights64(x, chosen, score, chosen_only, scale):
    import torch

    logw = torch.log_softmax(x, 1) if score == "softmax" else torch.nn.functional.logsigmoid(x)
    picked = logw.gather(1, chosen)
    w = torch.softmax(picked, 1) if chosen_only else picked.exp()
    return w * scale


def _run(logits, top, dtype, score="softmax", chosen_only=False, scale=1.0, bias=None, pad=0, offset=0):
    """route() of these logits; returns what it writes, checked against a stable sort and 64 bits where the logits are finite"""
    import torch

    tokens, experts = logits.shape
    buffer = torch.full((offset + tokens * (experts + pad) + 8,), float("nan"), dtype=_torch(dtype), device="cuda")
    buffer[offset: offset + tokens * (experts + pad)].view(tokens, experts + pad)[:, :experts] = logits.to(_torch(dtype))
    x = buffer[offset: offset + tokens * (experts + pad)].view(tokens, experts + pad)[:, :experts].float()
    full = lambda *shape: torch.full(shape, -7, dtype=torch.int32, device="cuda")  # noqa: E731
    weights, chosen, place, source, offsets = torch.full((tokens + 1, top), -7.0, device="cuda"), full(tokens + 1, top), full(tokens + 1, top), full(tokens * top + 1), full(experts + 2)
    need = R.route_workspace_bytes(tokens, experts, top)
    scratch = torch.full((need + 64,), 0xFF, dtype=torch.uint8, device="cuda")
    R.route(TYPES[dtype], tokens, experts, top, buffer[offset:], weights, chosen, place, source, offsets, score=SCORES[score], chosen_only=chosen_only, scale=scale, bias=bias,
            ldl=experts + pad, workspace=scratch if need else None, workspace_bytes=need)
    torch.cuda.synchronize()
    assert (scratch[need:] == 0xFF).all()
    for t in (weights[tokens:], chosen[tokens:], place[tokens:], source[tokens * top:], offsets[experts + 1:]):
        assert (t == -7).all()
    weights, chosen, place, source, offsets = weights[:tokens], chosen[:tokens], place[:tokens], source[: tokens * top], offsets[: experts + 1]
    by = x if bias is None else x + bias
    order = torch.where(torch.isnan(by), torch.full_like(by, -math.inf), by)
    # a stable sort by NaN last, then by value
    rank = torch.sort(order.cpu().double() + 0.0, dim=1, descending=True, stable=True)[1]
    is_nan = torch.isnan(by).cpu().gather(1, rank)
    want = rank.gather(1, torch.sort(is_nan.int(), dim=1, stable=True)[1])[:, :top]
    assert torch.equal(chosen.cpu().long(), want)
    flat = chosen.reshape(-1).long()
    perm = torch.sort(flat, stable=True)[1]
    inverse = torch.empty_like(perm)
    inverse[perm] = torch.arange(tokens * top, device="cuda")
    assert torch.equal(place.reshape(-1).long(), inverse) and torch.equal(source.long(), perm // top)
    assert torch.equal(offsets.long().cpu(), torch.cat([torch.zeros(1, dtype=torch.int64), torch.bincount(flat.cpu(), minlength=experts).cumsum(0)]))
    if torch.isfinite(x).all():
        exact = _weights64(x.double(), chosen.long(), score, chosen_only, scale)
        a = (x.amax(1, keepdim=True) - x.amin(1, keepdim=True)).double() + x.abs().amax(1, keepdim=True).double()
        assert ((weights - exact).abs() <= (2 * a + experts + 12) * EPS * exact + TINY["f32"]).all(), ((weights - exact).abs() / exact / EPS).max()
    return weights, chosen, place, source, offsets


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("tokens,experts,top", [(1, 1, 1), (1, 8, 2), (7, 64, 6), (64, 65, 8), (65, 128, 4), (100, 200, 32), (1000, 256, 8), (333, 1024, 3), (17, 300, 17), (5000, 16, 2)])
def test_route(dtype, tokens, experts, top):
    import torch

    torch.manual_seed(tokens + experts)
    x = torch.randn(tokens, experts, device="cuda") * 2
    for score in ("softmax", "sigmoid"):
        for chosen_only in (False, True):
            _run(x, top, dtype, score, chosen_only, scale=2.5 if chosen_only else 1.0)
    _run(x, top, dtype, bias=torch.randn(experts, device="cuda"), pad=3, offset=1)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 63, 64, 65, 79, 80, 81, 4097, 40001])
def test_route_numbers_of_tokens(tokens):
    import torch

    _run(torch.randn(tokens, 40, device="cuda"), 4, "bf16")


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,experts", [(3, 8), (70, 32), (40, 3)])
def test_route_to_every_expert(tokens, experts):
    import torch

    for score in ("softmax", "sigmoid"):
        _run(torch.randn(tokens, experts, device="cuda"), experts, "f16", score, True, bias=torch.randn(experts, device="cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("experts", [1, 8, 1000])
def test_route_of_no_tokens(experts):
    """Every expert's rows begin and end at 0"""
    import torch

    offsets = torch.full((experts + 2,), -7, dtype=torch.int32, device="cuda")
    R.route(R.F16, 0, experts, 1, None, None, None, None, None, offsets)
    assert (offsets[:-1] == 0).all() and offsets[-1] == -7


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [5, 200])
@pytest.mark.parametrize("top", [2, 8])
def test_route_ties_infinities_and_nan(tokens, top):
    """Equal logits, zeros of both signs, rows of -infinity, experts masked by the type's lowest value, infinities, NaN"""
    import torch

    torch.manual_seed(top)
    x = torch.randint(-2, 3, (tokens, 70), device="cuda").float()
    x[0, ::2] = -0.0
    _run(x, top, "f32")
    _run(torch.zeros(tokens, 70, device="cuda"), top, "bf16")
    low = x.clone()
    low[:, 5:] = torch.finfo(torch.float16).min
    _run(low, top, "f16", chosen_only=True)
    masked = x.clone()
    masked[:, 3:] = -math.inf
    masked[1] = -math.inf
    for score in ("softmax", "sigmoid"):
        for chosen_only in (False, True):
            w, chosen, *_ = _run(masked, top, "f32", score, chosen_only)
            assert (w[1] == 0).all() and torch.isfinite(w).all() and (w[0][chosen[0] >= 3] == 0).all()
            if chosen_only:
                assert ((w[0].sum() - 1).abs() < 1e-6).all()
    bad = x.clone()
    bad[2, 10], bad[2, 20], bad[3], bad[4, 0] = math.nan, -math.nan, math.nan, math.inf
    w, chosen, *_ = _run(bad, top, "f32", "sigmoid")
    assert not (chosen[2] == 10).any() and torch.equal(chosen[3].cpu(), torch.arange(top, dtype=torch.int32)) and chosen[4, 0] == 0 and w[4, 0] == 1
    assert torch.isfinite(w[[0, 1, 2]]).all()


@pytest.mark.gpu
def test_route_far_logits():
    """Scores that 32 bits cannot hold, by their ratios"""
    import torch

    x = torch.linspace(-300, -200, 64, device="cuda").repeat(3, 1)
    for score in ("softmax", "sigmoid"):
        w, *_ = _run(x, 4, "f32", score, True)
        assert (w > 0).all()
    _run(-x, 4, "f32", "softmax", False)
    bias = torch.linspace(200, 0, 64, device="cuda")
    w, chosen, *_ = _run(torch.linspace(0, 100, 64, device="cuda").repeat(70, 1), 4, "f32", "softmax", True, bias=bias)
    assert (w > 0).all() and (chosen[:, 0] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("chosen_only", [False, True])
@pytest.mark.parametrize("dtype,tokens,experts,top", [("f32", 1, 1, 1), ("bf16", 9, 64, 6), ("f16", 130, 100, 8), ("f32", 301, 256, 32), ("f32", 5, 1000, 4)])
def test_route_backward(score, chosen_only, dtype, tokens, experts, top):
    import torch

    torch.manual_seed(experts)
    t = _torch(dtype)
    x = (torch.randn(tokens, experts, device="cuda") * 2).to(t)
    chosen = torch.sort(x.float(), dim=1, descending=True, stable=True)[1][:, :top].to(torch.int32).contiguous()
    dw = torch.randn(tokens, top, device="cuda")
    d = torch.full((tokens + 1, experts + 3), float("nan"), dtype=t, device="cuda")
    R.route_backward(TYPES[dtype], tokens, experts, top, x, chosen, dw, d, score=SCORES[score], chosen_only=chosen_only, scale=1.5, ldd=experts + 3)
    assert torch.isnan(d[:, experts:]).all() and torch.isnan(d[tokens:]).all()
    leaf = x.double().cpu().requires_grad_()
    (_weights64(leaf, chosen.long().cpu(), score, chosen_only, 1.5) * dw.double().cpu()).sum().backward()
    w = _weights64(x.double(), chosen.long(), score, False, 1.5)
    a = 2 * (x.amax(1, keepdim=True) - x.amin(1, keepdim=True)).double() + x.abs().amax(1, keepdim=True).double()
    # every term is a product of dw, weights and scores, each within the bound of a weight; their sums add up to (1.5 max |dw|) top of them
    most = (dw.double().abs() * (1.5 if chosen_only else w)).sum(1, keepdim=True)
    want = leaf.grad.cuda()
    bound = 3 * (2 * a + experts + 12) * EPS * most
    assert ((d[:tokens, :experts].double() - want).abs() <= bound + HALF[dtype] * (want.abs() + bound) + TINY[dtype]).all()
    # against differences, in 64 bits, of the formula that the kernel's weights were held to
    if dtype == "f32":
        step, h = torch.randn(tokens, experts, device="cuda").double(), 1e-4
        f = lambda s: (_weights64(x.double() + s * h * step, chosen.long(), score, chosen_only, 1.5) * dw.double()).sum().item()  # noqa: E731
        slope = (want * step).sum().item()
        assert abs((f(1) - f(-1)) / (2 * h) - slope) <= 1e-6 * (most.sum().item() * experts + 1)


@pytest.mark.gpu
def test_route_backward_of_experts_that_are_not_there_or_twice():
    import torch

    x = torch.randn(3, 8, device="cuda")
    chosen = torch.tensor([[1, 9], [-1, 2], [4, 4]], dtype=torch.int32).cuda()
    dw = torch.ones(3, 2, device="cuda")
    d = torch.empty(3, 8, device="cuda")
    R.route_backward(R.F32, 3, 8, 2, x, chosen, dw, d, score=R.ROUTE_SIGMOID)
    s = torch.sigmoid(x)
    want = torch.zeros(3, 8, device="cuda")
    want[0, 1], want[1, 2], want[2, 4] = (s * (1 - s))[0, 1], (s * (1 - s))[1, 2], 2 * (s * (1 - s))[2, 4]
    assert torch.allclose(d, want, atol=1e-6)
    x[1] = -math.inf
    R.route_backward(R.F32, 3, 8, 2, x, chosen, dw, d, chosen_only=True)
    assert torch.isfinite(d).all() and (d[1] == 0).all()


def _rows(dtype, tokens, top, width, rows=None, pad=0, offset=0, seed=0, drop=()):
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)
    t, rows = _torch(dtype), tokens * top if rows is None else rows
    place = torch.randperm(rows, generator=g, device="cuda")[: tokens * top].to(torch.int32).view(tokens, top)
    for at, value in drop:
        place.view(-1)[at] = value
    made = []
    for n in (rows, tokens, tokens):
        buffer = torch.full((offset + n * (width + pad) + 8,), float("nan"), dtype=t, device="cuda")
        view = buffer[offset: offset + n * (width + pad)].view(n, width + pad)
        view[:, :width] = torch.randn(n, width, generator=g, device="cuda").to(t)
        made += [buffer[offset:], view]
    return place, torch.rand(tokens, top, generator=g, device="cuda") - 0.3, made


ROWS = [(1, 1, 8, 0, 0), (3, 2, 40, 0, 0), (5, 3, 129, 0, 0), (70, 8, 512, 0, 0), (33, 9, 1032, 8, 0), (20, 32, 264, 0, 0), (10, 2, 4104, 0, 0), (9, 4, 96, 3, 1), (300, 1, 2048, 0, 0)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("tokens,top,width,pad,offset", ROWS)
def test_combine(dtype, tokens, top, width, pad, offset):
    import torch

    slots = tokens * top
    place, weights, (values, vview, c, cview, y, yview) = _rows(dtype, tokens, top, width, slots + 5, pad, offset, drop=((0, -1), (slots // 2, slots + 5)) if slots > 3 else ())
    for w, residual, in_place in ((weights, True, False), (None, False, False), (weights, True, True)):
        yview.fill_(float("nan"))
        R.combine(TYPES[dtype], tokens, top, width, values, slots + 5, place, c if in_place else y, weights=w, c=c if residual else None, ldv=width + pad, ldc=width + pad, ldy=width + pad)
        in_, at = ((place >= 0) & (place < slots + 5)), place.long().clamp(0, slots + 4)
        terms = torch.where(in_[..., None], vview.double()[at][..., :width] * (1.0 if w is None else w.double()[..., None]), 0.0)
        base = before if in_place else cview[:, :width].double() if residual else 0.0
        if not in_place:
            before = cview[:, :width].double().clone()
        want = terms.sum(1) + base
        bound = (top + 2) * EPS * (terms.abs().sum(1) + (abs(base) if residual else 0.0))
        got = (cview if in_place else yview)
        assert ((got[:, :width].double() - want).abs() <= bound + HALF[dtype] * (want.abs() + bound) + TINY[dtype]).all()
        assert torch.isnan(got[:, width:]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("tokens,top,width,pad,offset", ROWS)
def test_dispatch(dtype, tokens, top, width, pad, offset):
    import torch

    slots = tokens * top
    place, weights, (values, vview, x, xview, _, _) = _rows(dtype, tokens, top, width, slots + 5, pad, offset, drop=((0, -1), (slots // 2, slots + 5)) if slots > 3 else ())
    in_, at = (place >= 0) & (place < slots + 5), place.long().clamp(0, slots + 4)
    for w, dots, rows in ((None, False, True), (weights, True, True), (weights, True, False), (None, True, True)):
        out = torch.full((offset + (slots + 5) * (width + pad) + 8,), float("nan"), dtype=_torch(dtype), device="cuda")
        dw = torch.full((tokens + 1, top), float("nan"), device="cuda")
        R.dispatch(TYPES[dtype], tokens, top, width, x, out[offset:] if rows else None, slots + 5, place, weights=w, values=values if dots else None, dweights=dw if dots else None,
                   ldx=width + pad, ldv=width + pad, ldo=width + pad)
        oview = out[offset: offset + (slots + 5) * (width + pad)].view(slots + 5, width + pad)
        terms = xview[:, None, :width].double() * (torch.ones_like(weights) if w is None else w).double()[..., None]
        if rows:
            assert ((oview[at[in_]][:, :width].double() - terms[in_]).abs() <= HALF[dtype] * terms[in_].abs() + TINY[dtype] + (0 if w is None else EPS * terms[in_].abs())).all()
            untouched = torch.ones(slots + 5, dtype=torch.bool, device="cuda")
            untouched[at[in_]] = False
            assert torch.isnan(oview[untouched]).all() and torch.isnan(oview[:, width:]).all()
        if dots:
            products = torch.where(in_[..., None], xview[:, None, :width].double() * vview.double()[at][..., :width], 0.0)
            want = products.sum(2)
            assert ((dw[:tokens].double() - want).abs() <= (width + 8) * EPS * products.abs().sum(2) + EPS * want.abs()).all()
            assert torch.isnan(dw[tokens:]).all()


@pytest.mark.gpu
def test_each_is_the_others_gradient():
    """<combine(v), dy> = <v, dispatch(dy)> and its derivative along the weights is dweights, in values that 16 bits hold exactly"""
    import torch

    tokens, top, width = 40, 3, 72
    place = torch.randperm(tokens * top, device="cuda").to(torch.int32).view(tokens, top)
    small = lambda *shape: torch.randint(-4, 5, shape, device="cuda").bfloat16()  # noqa: E731
    v, dy, w = small(tokens * top, width), small(tokens, width), torch.randint(-2, 3, (tokens, top), device="cuda").float()
    y, dv, dw = torch.empty(tokens, width, dtype=torch.bfloat16, device="cuda"), torch.empty_like(v), torch.empty(tokens, top, device="cuda")
    R.combine(R.BF16, tokens, top, width, v, tokens * top, place, y, weights=w)
    R.dispatch(R.BF16, tokens, top, width, dy, dv, tokens * top, place, weights=w, values=v, dweights=dw)
    inner = (y.double() * dy.double()).sum()
    assert inner == (v.double() * dv.double()).sum() and inner == (w.double() * dw.double()).sum()


@pytest.mark.gpu
def test_more_rows_than_the_caches_keep():
    """In values that 16 bits hold exactly"""
    import torch

    tokens, top, width = 3000, 8, 2104
    rows = tokens * top
    place = torch.randperm(rows, device="cuda").to(torch.int32).view(tokens, top)
    place[5, 2], place[2999, 7] = -1, rows
    small = lambda *shape: torch.randint(-3, 4, shape, device="cuda").bfloat16()  # noqa: E731
    v, x, w = small(rows, width), small(tokens, width), torch.randint(-1, 2, (tokens, top), device="cuda").float()
    y, out, dw = torch.empty_like(x), torch.full_like(v, float("nan")), torch.empty(tokens, top, device="cuda")
    R.combine(R.BF16, tokens, top, width, v, rows, place, y, weights=w, c=x)
    R.dispatch(R.BF16, tokens, top, width, x, out, rows, place, weights=w, values=v, dweights=dw)
    there = (place >= 0) & (place < rows)
    at = torch.where(there, place, 0).long()
    total = x.float()
    for j in range(top):
        total += torch.where(there[:, j, None], v[at[:, j]].float() * w[:, j, None], 0.0)
        assert torch.equal(out[at[:, j]][there[:, j]].float(), (x.float() * w[:, j, None])[there[:, j]])
        assert torch.equal(dw[:, j], torch.where(there[:, j], (x.float() * v[at[:, j]].float()).sum(1), 0.0))
    assert torch.equal(y.float(), total) and torch.isnan(out).any(1).sum() == 2


@pytest.mark.gpu
def test_long_rows():
    """Rows past 2^31 bytes"""
    import torch

    tokens, width, rows = 4, 4096, 300000
    values = torch.zeros(rows, width, dtype=torch.bfloat16, device="cuda")
    place = torch.tensor([[0, 299999], [262143, 262144], [262145, 1], [2, 3]], dtype=torch.int32).cuda()
    x = torch.randn(tokens, width, device="cuda").bfloat16()
    R.dispatch(R.BF16, tokens, 2, width, x, values, rows, place)
    assert torch.equal(values[place.long()], x[:, None].expand(4, 2, width))
    y = torch.empty_like(x)
    R.combine(R.BF16, tokens, 2, width, values, rows, place, y)
    assert torch.equal(y, x * 2)


@pytest.mark.gpu
def test_graph():
    """The router recorded with both its forms, replayed with new logits, the program's eager work between"""
    import torch

    for tokens in (20, 700):
        x = torch.randn(tokens, 64, device="cuda")
        make = lambda: (torch.zeros(tokens, 4, device="cuda"), *(torch.zeros(tokens, 4, dtype=torch.int32, device="cuda") for _ in range(2)),  # noqa: E731
                        torch.zeros(tokens * 4, dtype=torch.int32, device="cuda"), torch.zeros(65, dtype=torch.int32, device="cuda"))
        out, eager = make(), make()
        scratch = torch.empty(max(16, R.route_workspace_bytes(tokens, 64, 4)), dtype=torch.uint8, device="cuda")
        other = torch.empty_like(scratch)
        R.route(R.F32, tokens, 64, 4, x, *eager, workspace=other)
        torch.cuda.synchronize()
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(graph, stream=side):
            R.route(R.F32, tokens, 64, 4, x, *out, workspace=scratch, stream=torch.cuda.current_stream())
        for _ in range(4):
            x.normal_()
            graph.replay()
            R.route(R.F32, tokens, 64, 4, x, *eager, workspace=other)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, eager))


def _set(a, change):
    for name, value in change.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("change,code", [
    (dict(type=R.E4M3), -2), (dict(score=2), -1), (dict(experts=0), -1), (dict(top=0), -1), (dict(top=9), -1), (dict(experts=2000, ldl=2000), -3), (dict(top=33, experts=64, ldl=64), -3),
    (dict(tokens=2 ** 30), -3), (dict(ldl=7), -1), (dict(logits=None), -1), (dict(weights=None), -1), (dict(chosen=None), -1), (dict(place=None), -1), (dict(source=None), -1),
    (dict(offsets=None), -1), (dict(logits=0x1001), -4), (dict(weights=0x2001), -4), (dict(offsets=0x6002), -4), (dict(bias=0x7002), -4), (dict(tokens=1000), -3),
    (dict(tokens=1000, workspace=0x8000, workspace_bytes=64), -3), (dict(tokens=1000, workspace=0x8008, workspace_bytes=1 << 20), -4),
])
def test_route_refusals(change, code):
    import ctypes

    a = R.RouteArgs(R.BF16, R.ROUTE_SOFTMAX, 0, 4, 8, 2, 8, 0x1000, None, 0x2000, 0x3000, 0x4000, 0x5000, 0x6000, 1.0, None, 0)
    assert R.lib().r355_route(ctypes.byref(_set(a, change)), None) == code and R.lib().r355_last_error()
    assert R.lib().r355_route(None, None) == -1


@pytest.mark.parametrize("change,code", [
    (dict(type=R.I8), -2), (dict(score=-1), -1), (dict(top=9), -1), (dict(ldl=7), -1), (dict(ldd=7), -1), (dict(logits=None), -1), (dict(chosen=None), -1), (dict(dweights=None), -1),
    (dict(dlogits=None), -1), (dict(dlogits=0x4001), -4), (dict(chosen=0x2002), -4), (dict(tokens=2 ** 29), -3),
])
def test_route_backward_refusals(change, code):
    import ctypes

    a = R.RouteBackwardArgs(R.BF16, R.ROUTE_SOFTMAX, 0, 4, 8, 2, 8, 8, 0x1000, 0x2000, 0x3000, 0x4000, 1.0)
    assert R.lib().r355_route_backward(ctypes.byref(_set(a, change)), None) == code and R.lib().r355_last_error()


@pytest.mark.parametrize("change,code", [
    (dict(type=R.F32), -2), (dict(top=0), -1), (dict(width=0), -1), (dict(tokens=2 ** 30), -3), (dict(rows=2 ** 31), -3), (dict(width=2 ** 24 + 8), -3), (dict(place=None), -1),
    (dict(place=0x3002), -4), (dict(weights=0x4002), -4),
])
def test_rows_refusals(change, code):
    import ctypes

    combine = R.CombineArgs(R.BF16, 4, 2, 8, 8, 0x1000, 0x3000, None, None, 0x2000, 8, 8, 8)
    dispatch = R.DispatchArgs(R.BF16, 4, 2, 8, 8, 0x1000, 0x3000, None, None, 0x2000, None, 8, 8, 8)
    assert R.lib().r355_combine(ctypes.byref(_set(combine, change)), None) == code
    assert R.lib().r355_dispatch(ctypes.byref(_set(dispatch, change)), None) == code


def test_rows_refusals_of_each():
    import ctypes

    for change, code in ((dict(values=None), -1), (dict(y=None), -1), (dict(ldv=7), -1), (dict(ldy=7), -1), (dict(c=0x5000, ldc=7), -1), (dict(y=0x2001), -4), (dict(tokens=2 ** 28, width=2 ** 20, ldv=2 ** 20, ldy=2 ** 20), -3)):
        a = R.CombineArgs(R.BF16, 4, 2, 8, 8, 0x1000, 0x3000, None, None, 0x2000, 8, 8, 8)
        assert R.lib().r355_combine(ctypes.byref(_set(a, change)), None) == code, change
    for change, code in ((dict(x=None), -1), (dict(out=None), -1), (dict(dweights=0x5000), -1), (dict(ldx=7), -1), (dict(ldo=7), -1), (dict(dweights=0x5000, values=0x6000, ldv=7), -1), (dict(out=0x2001), -4)):
        a = R.DispatchArgs(R.BF16, 4, 2, 8, 8, 0x1000, 0x3000, None, None, 0x2000, None, 8, 8, 8)
        assert R.lib().r355_dispatch(ctypes.byref(_set(a, change)), None) == code, change
    assert R.lib().r355_combine(None, None) == -1 and R.lib().r355_dispatch(None, None) == -1


def test_arrays_are_checked():
    import torch

    i32, f32 = torch.zeros(8, dtype=torch.int32), torch.zeros(8)
    with pytest.raises(ValueError):
        R.route(R.F32, 4, 8, 2, 0x1000, f32.double(), 0x2000, 0x3000, 0x4000, 0x5000)
    with pytest.raises(ValueError):
        R.route(R.F32, 4, 8, 2, 0x1000, 0x1000, i32.long(), 0x3000, 0x4000, 0x5000)
    with pytest.raises(ValueError):
        R.combine(R.BF16, 4, 2, 8, 0x1000, 8, i32, 0x2000, weights=f32)
    with pytest.raises(ValueError):
        R.dispatch(R.BF16, 4, 2, 8, 0x1000, 0x2000, 8, i32.long())


@pytest.mark.parametrize("top", [1, 6, 32])
def test_route_workspace_for_more_tokens_serves_fewer(top):
    """(blocks of 16 tokens up to 16384 of them, of 20 from the next one on)"""
    need = [R.route_workspace_bytes(tokens, 40, top) for tokens in [*range(1, 400), *range(16300, 16500), 20000, 32768, 32769, 65536, 65537, 2 ** 25]]
    assert need == sorted(need) and need[-1] > 0


def test_argument_structures(tmp_path):
    """What Python writes against what the compiler makes of the header"""
    import ctypes

    import test_argument_bytes as B

    for kind, name in ((R.RouteArgs, "route"), (R.RouteBackwardArgs, "route_backward"), (R.CombineArgs, "combine"), (R.DispatchArgs, "dispatch"), (R.LinearArgs, "linear"),
                       (R.LinearBackwardArgs, "linear_backward")):
        names = [f for f, _ in kind._fields_]
        layout, size = B._layout(tmp_path, "r355_%s_args" % name, names)
        packed = getattr(R, "_%s_ARGS" % name.upper())
        assert ctypes.sizeof(kind) == size == packed.size
        # every value that is packed, made one at a time not zero, is the structure's field of that place; what is left over is padding
        fields = iter(names)
        letters = packed.format.lstrip("=")
        for i, letter in enumerate(letters):
            values = [0.0 if c == "d" else 0 for c in letters]
            values[i] = 1.5 if letter == "d" else 3
            a = kind.from_buffer_copy(packed.pack(*values))
            held = [f for f in names if getattr(a, f)]
            assert held == ([next(fields)] if held else []) and (not held or getattr(a, held[0]) == values[i]), (name, i)
        assert next(fields, None) is None
        assert {n: (getattr(kind, n).offset, getattr(kind, n).size) for n in names} == layout
