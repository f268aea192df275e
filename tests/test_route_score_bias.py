"""The router's choice by score plus bias (ROUTE_SCORE_BIAS), against 64 bits; the weights and the order of the rows are test_experts.py's.

eps = 2^-24.  A score is off by (2 a + E + 12) eps of itself (test_experts.py: a the largest argument of an exponential, E the experts of a softmax's sum), its sum with the bias by half a step of
the result, eps of |score| + |bias|.  Experts whose sums are further apart than what both are off by have to come in the order of the sums."""
import ctypes
import math

import pytest

import rocwmma_amd as R

EPS = 2.0 ** -24
SCORES = {"softmax": R.ROUTE_SOFTMAX, "sigmoid": R.ROUTE_SIGMOID}


def _route(x, top, dtype, score, bias, chosen_only=False, scale=1.0, stream=None, out=None, scratch=None):
    import torch

    tokens, experts = x.shape
    empty = lambda *shape: torch.full(shape, -7, dtype=torch.int32, device="cuda")  # noqa: E731
    out = out or (torch.full((tokens, top), -7.0, device="cuda"), empty(tokens, top), empty(tokens, top), empty(tokens * top), empty(experts + 1))
    need = R.route_workspace_bytes(tokens, experts, top)
    scratch = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda") if scratch is None else scratch
    R.route(dtype, tokens, experts, top, x, *out, score=score, chosen_only=chosen_only, scale=scale, bias=bias, workspace=scratch, stream=stream)
    return out


def _weights64(x, chosen, score, chosen_only, scale):
    import torch

    logw = torch.log_softmax(x, 1) if score == "softmax" else torch.nn.functional.logsigmoid(x)
    picked = logw.gather(1, chosen)
    return (torch.softmax(picked, 1) if chosen_only else picked.exp()) * scale


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype,tokens,experts,top", [("f32", 1, 2, 1), ("bf16", 7, 64, 6), ("f16", 100, 100, 8), ("f32", 1000, 256, 8), ("bf16", 333, 1024, 3), ("f32", 40, 8, 8), ("f16", 2000, 160, 6)])
def test_choice(score, dtype, tokens, experts, top):
    import torch

    g = torch.Generator(device="cuda").manual_seed(experts + top)
    x = (torch.randn(tokens, experts, generator=g, device="cuda") * 2).to({"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}[dtype])
    bias = torch.randn(experts, generator=g, device="cuda") * (0.3 if score == "sigmoid" else 2.0 / experts)
    xd = x.double()
    s = torch.softmax(xd, 1) if score == "softmax" else torch.sigmoid(xd)
    a = (x.amax(1, keepdim=True) - x.amin(1, keepdim=True)).double() + xd.abs().amax(1, keepdim=True)
    value, off = s + bias.double(), (2 * a + experts + 12) * EPS * s + EPS * (s + bias.double().abs())
    for chosen_only in (False, True):
        w, chosen, place, source, offsets = _route(x, top, getattr(R, dtype.upper()), SCORES[score] | R.ROUTE_SCORE_BIAS, bias, chosen_only, 2.5)
        chosen = chosen.long()
        assert (torch.sort(chosen, dim=1)[0].diff(dim=1) > 0).all()
        got, far = value.gather(1, chosen), off.gather(1, chosen)
        assert (got[:, :-1] - got[:, 1:] >= -(far[:, :-1] + far[:, 1:])).all()  # in their order
        others = value.scatter(1, chosen, -math.inf)  # none that is left out is larger
        assert ((others - off).amax(1) <= (got + far)[:, -1]).all()
        want = _weights64(xd, chosen, score, chosen_only, 2.5)
        assert ((w - want).abs() <= (2 * a + experts + 12) * EPS * want).all()
        flat = chosen.reshape(-1)
        perm = torch.sort(flat, stable=True)[1]
        assert torch.equal(source.long(), perm // top) and torch.equal(place.reshape(-1).long()[perm], torch.arange(tokens * top, device="cuda"))
        assert torch.equal(offsets[1:].long(), torch.bincount(flat, minlength=experts).cumsum(0))
        # nearly every token's choice is decided by more than that
        top_ = torch.sort(value, dim=1, descending=True)[0][:, : top + 1]
        clear = ((top_[:, :-1] - top_[:, 1:]) > 2 * off.amax(1, keepdim=True)).all(1)
        assert clear.double().mean() > 0.9 and torch.equal(chosen[clear], torch.sort(value, dim=1, descending=True)[1][clear][:, :top])


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [3, 70])
def test_by_the_score_and_not_by_the_logit(tokens):
    """sigma(3) + 0.05 = 1.0026 is more than sigma(5) = 0.9933, 3.05 is less than 5"""
    import torch

    x = torch.tensor([[3.0, 5.0, -9.0]], device="cuda").repeat(tokens, 1)
    bias = torch.tensor([0.05, 0.0, 0.0], device="cuda")
    by_score = _route(x, 1, R.F32, R.ROUTE_SIGMOID | R.ROUTE_SCORE_BIAS, bias)
    by_logit = _route(x, 1, R.F32, R.ROUTE_SIGMOID, bias)
    assert (by_score[1] == 0).all() and (by_logit[1] == 1).all()
    assert torch.allclose(by_score[0], torch.sigmoid(x[:, :1]), rtol=1e-6)  # (the weight is the score alone)
    # without a bias the flag changes nothing
    assert all(torch.equal(a, b) for a, b in zip(_route(x, 2, R.F32, R.ROUTE_SOFTMAX | R.ROUTE_SCORE_BIAS, None), _route(x, 2, R.F32, R.ROUTE_SOFTMAX, None)))


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("tokens", [5, 100])
def test_ties_infinities_and_nan(score, tokens):
    import torch

    x, bias = torch.zeros(tokens, 70, device="cuda"), torch.zeros(70, device="cuda")
    flag = SCORES[score] | R.ROUTE_SCORE_BIAS
    bias[::2] = -0.0
    assert torch.equal(_route(x, 4, R.F32, flag, bias)[1].cpu(), torch.arange(4, dtype=torch.int32).repeat(tokens, 1))
    bias[50], bias[60], bias[10] = 0.25, 0.25, math.nan
    assert torch.equal(_route(x, 4, R.F32, flag, bias)[1].cpu(), torch.tensor([50, 60, 0, 1], dtype=torch.int32).repeat(tokens, 1))
    x[0, 5:] = -math.inf  # scores of 0, which a bias can lift: their weight is 0
    x[1] = -math.inf
    w, chosen, *_ = _route(x, 4, R.F32, flag, bias, True)
    assert torch.isfinite(w).all() and (w[1] == 0).all() and (w[0][chosen[0] >= 5] == 0).all()
    if score == "sigmoid":
        x[2, 7], x[2, 8], x[2, 9] = math.nan, math.inf, 40.0  # (sigma of both is 1 in f32: the lower expert first)
        w, chosen, *_ = _route(x, 4, R.F32, flag, torch.zeros(70, device="cuda"))
        assert chosen[2].tolist() == [8, 9, 0, 1] and w[2].tolist() == [1.0, 1.0, 0.5, 0.5]
        every = _route(x[2:3].contiguous(), 32, R.F32, flag, torch.where(torch.arange(70, device="cuda") < 32, 4.0, 0.0))[1]
        assert 7 not in every[0].tolist()


@pytest.mark.gpu
def test_gradient_takes_the_same_scores():
    import torch

    x, dw = torch.randn(50, 40, device="cuda"), torch.randn(50, 4, device="cuda")
    for score in SCORES.values():
        chosen = _route(x, 4, R.F32, score | R.ROUTE_SCORE_BIAS, torch.randn(40, device="cuda"))[1]
        a, b = torch.empty_like(x), torch.empty_like(x)
        R.route_backward(R.F32, 50, 40, 4, x, chosen, dw, a, score=score | R.ROUTE_SCORE_BIAS)
        R.route_backward(R.F32, 50, 40, 4, x, chosen, dw, b, score=score)
        assert torch.equal(a, b) and a.abs().sum() > 0


@pytest.mark.gpu
def test_graph():
    import torch

    for tokens in (20, 700):
        x, bias = torch.randn(tokens, 64, device="cuda"), torch.randn(64, device="cuda") * 0.2
        flag = R.ROUTE_SIGMOID | R.ROUTE_SCORE_BIAS
        scratch = torch.empty(max(16, R.route_workspace_bytes(tokens, 64, 4)), dtype=torch.uint8, device="cuda")
        out = _route(x, 4, R.F32, flag, bias, scratch=scratch)
        torch.cuda.synchronize()
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(graph, stream=side):
            _route(x, 4, R.F32, flag, bias, out=out, scratch=scratch, stream=torch.cuda.current_stream())
        for _ in range(4):
            x.normal_()
            graph.replay()
            eager = _route(x, 4, R.F32, flag, bias)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, eager))


@pytest.mark.parametrize("score,code", [(2, -1), (R.ROUTE_SCORE_BIAS | 2, -1), (512, -1), (-1, -1), (R.ROUTE_SCORE_BIAS | R.ROUTE_SIGMOID, -4), (R.ROUTE_SCORE_BIAS, -4)])
def test_scores(score, code):
    """What is no score is refused; what is one gets as far as the alignment of the logits"""
    route = R.RouteArgs(R.BF16, score, 0, 4, 8, 2, 8, 0x1001, None, 0x2000, 0x3000, 0x4000, 0x5000, 0x6000, 1.0, None, 0)
    back = R.RouteBackwardArgs(R.BF16, score, 0, 4, 8, 2, 8, 8, 0x1001, 0x2000, 0x3000, 0x4000, 1.0)
    assert R.lib().r355_route(ctypes.byref(route), None) == R.lib().r355_route_backward(ctypes.byref(back), None) == code
