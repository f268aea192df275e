"""Rotary positions against the formula in 64 bits (the angle from integers, modulo a turn).

Bound of the error: the angle, within an eighth of a turn, is rounded twice (2 pi/4 2^-24), the sums of sine and cosine are within 4e-8 and
their evaluation rounds by 2^-23; with the scale that is under 3.5e-7, and the two products and their sum add 1.5 2^-23: under 6e-7
(|a| + |b|) scale, before the one rounding to the result's type."""
import numpy as np
import pytest

import rocwmma_amd as R

HALF_ULP = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}
TYPES = {"f16": R.F16, "bf16": R.BF16, "f32": R.F32}
LAYOUT = {"half": R.ROPE_HALF, "interleaved": R.ROPE_INTERLEAVED}


def _torch_type(name):
    import torch

    return {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}[name]


def _pairs(layout, rotary):
    i = np.arange(rotary // 2)
    return (i, i + rotary // 2) if layout == "half" else (2 * i, 2 * i + 1)


def _want(x, layout, rotary, positions, turns, scale, inverse):
    """(result, |a| + |b| of each element's pair) of x [tokens][heads][dim] in float64."""
    parts = np.array([[(int(p) * int(t)) % 2 ** 64 for t in turns] for p in positions], dtype=object)
    angle = (parts / 2.0 ** 64).astype(np.float64)[:, None, :] * 2.0 * np.pi * (-1.0 if inverse else 1.0)
    a, b = _pairs(layout, rotary)
    y, size = x.copy(), np.zeros_like(x)
    y[..., a] = scale * (x[..., a] * np.cos(angle) - x[..., b] * np.sin(angle))
    y[..., b] = scale * (x[..., a] * np.sin(angle) + x[..., b] * np.cos(angle))
    size[..., a] = size[..., b] = np.abs(x[..., a]) + np.abs(x[..., b])
    return y, size


def _dev_turns(turns):
    import torch

    return torch.from_numpy(turns.view(np.int64)).cuda()


def _check(got, want, size, dtype, scale=1.0):
    bound = 6e-7 * abs(scale) * size + HALF_ULP[dtype] * np.abs(want) * (1 + 1e-6) + (2.0 ** -25 if dtype == "f16" else 0.0)
    assert np.all(np.abs(got - want) <= bound), np.max(np.abs(got - want) - bound)


def _case(dtype, layout, tokens, heads, dim, rotary, first=0, inverse=False, scale=1.0, base=10000.0, pad=0, head_pad=0, offset=0, in_place=False):
    import torch

    rng = np.random.RandomState(tokens + heads + dim)
    t = _torch_type(dtype)
    positions = (first + rng.permutation(tokens)).astype(np.int32)
    turns = R.rope_turns(rotary, base)
    hs = dim + head_pad
    ts = heads * hs + pad
    buf = torch.full((offset + tokens * ts + 16,), float("nan"), dtype=t, device="cuda")
    view = buf[offset: offset + tokens * ts].view(tokens, ts)[:, : heads * hs].view(tokens, heads, hs)[..., :dim]
    x = torch.from_numpy(rng.randn(tokens, heads, dim)).to(t)
    view.copy_(x.cuda())
    out = buf if in_place else torch.full_like(buf, float("nan"))
    R.rope(TYPES[dtype], LAYOUT[layout], tokens, dim, rotary, [R.rope_part(buf[offset:], out[offset:], heads, (ts, hs), (ts, hs))],
           torch.from_numpy(positions).cuda(), _dev_turns(turns), scale=scale, inverse=inverse)
    got = out[offset: offset + tokens * ts].view(tokens, ts)[:, : heads * hs].view(tokens, heads, hs)
    assert torch.isnan(got[..., dim:]).all()
    want, size = _want(x.double().numpy(), layout, rotary, positions, turns, scale, inverse)
    got = got[..., :dim].double().cpu().numpy()
    _check(got, want, size, dtype, scale)
    assert np.array_equal(got[..., rotary:], x.double().numpy()[..., rotary:])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("tokens,heads,dim,rotary", [(1, 1, 64, 64), (5, 3, 128, 128), (33, 7, 96, 24), (4, 2, 80, 80), (300, 8, 128, 64), (7, 5, 10, 6), (2, 33, 256, 2)])
def test_rope_vs_formula(dtype, layout, tokens, heads, dim, rotary):
    _case(dtype, layout, tokens, heads, dim, rotary)
    _case(dtype, layout, tokens, heads, dim, rotary, first=1000003, inverse=True, scale=1.25, base=500000.0)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rope_positions_to_the_ends_of_the_type(layout):
    for first in (-40, 2 ** 31 - 64, -2 ** 31):
        _case("f32", layout, 40, 2, 64, 64, first=first)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("in_place", [False, True])
def test_rope_strides_alignment_in_place(layout, in_place):
    _case("bf16", layout, 9, 4, 64, 32, pad=24, head_pad=8, in_place=in_place)
    _case("bf16", layout, 9, 4, 64, 32, pad=4, head_pad=4, in_place=in_place)
    _case("f16", layout, 9, 4, 64, 32, pad=3, head_pad=5, offset=1, in_place=in_place)
    _case("f32", layout, 9, 4, 64, 32, pad=3, in_place=in_place)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 70, 9000])
def test_rope_parts_and_slots(tokens):
    """Queries beside, rotated keys and plain values into their rows of a cache, one launch; slots outside the cache are left out."""
    import torch

    rng = np.random.RandomState(3)
    h, kv, d, r, slots = 6, 2, 64, 32, tokens + 9
    x = torch.from_numpy(rng.randn(tokens, h + 2 * kv, d)).bfloat16()
    turns, positions = R.rope_turns(r), np.arange(tokens).astype(np.int32) + 77
    slot = rng.permutation(slots)[:tokens].astype(np.int32)
    if tokens > 2:
        slot[1], slot[2] = -1, slots
    dev = x.cuda()
    q = torch.empty(tokens, h, d, dtype=torch.bfloat16, device="cuda")
    k, v = (torch.full((slots, kv, d), 3.0, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    row = (h + 2 * kv) * d
    R.rope(R.BF16, R.ROPE_HALF, tokens, d, r,
           [R.rope_part(dev, q, h, (row, d), (h * d, d)), R.rope_part(dev[:, h:], k, kv, (row, d), (kv * d, d), to_slots=True),
            R.rope_part(dev[:, h + kv:], v, kv, (row, d), (kv * d, d), rotate=False, to_slots=True)],
           torch.from_numpy(positions).cuda(), _dev_turns(turns), slots=torch.from_numpy(slot).cuda(), slot_count=slots)
    xd = x.double().numpy()
    want, size = _want(xd[:, : h + kv], "half", r, positions, turns, 1.0, False)
    _check(q.double().cpu().numpy(), want[:, :h], size[:, :h], "bf16")
    inside = (slot >= 0) & (slot < slots)
    wk, wv, ws = np.full((slots, kv, d), 3.0), np.full((slots, kv, d), 3.0), np.zeros((slots, kv, d))
    wk[slot[inside]], wv[slot[inside]], ws[slot[inside]] = want[inside, h:], xd[inside, h + kv:], size[inside, h:]
    _check(k.double().cpu().numpy(), wk, ws, "bf16")
    assert np.array_equal(v.double().cpu().numpy(), wv)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rope_inverse_is_the_gradient(layout):
    """<g, rope(x + h e) - rope(x - h e)> / 2 h of the map in f32 against the element of inverse(g): the map is linear, so the difference is
    exact but for the rounding of its two values (6e-7 of their size, over 2 h = 2)."""
    import torch

    rng = np.random.RandomState(8)
    tokens, heads, d, r = 3, 2, 16, 12
    turns, positions = _dev_turns(R.rope_turns(r)), torch.tensor([5, 70001, 12], dtype=torch.int32, device="cuda")
    st = (heads * d, d)

    def call(x, inverse):
        y = torch.empty_like(x)
        R.rope(R.F32, LAYOUT[layout], tokens, d, r, [R.rope_part(x, y, heads, st, st)], positions, turns, scale=1.5, inverse=inverse)
        return y.double().cpu().numpy()

    x, g = (torch.from_numpy(rng.randn(tokens, heads, d).astype(np.float32)).cuda() for _ in range(2))
    grad, gd = call(g, True), g.double().cpu().numpy()
    for t, h, e in [(0, 0, 0), (1, 1, 5), (1, 0, 6), (2, 1, 11), (2, 0, 12), (0, 1, 15)]:
        up, down = x.clone(), x.clone()
        up[t, h, e] += 1.0
        down[t, h, e] -= 1.0
        step = float(up[t, h, e].double() - down[t, h, e].double())
        slope = np.sum(gd[t, h] * (call(up, False)[t, h] - call(down, False)[t, h])) / step
        # one element moves two results, each within 6e-7 * 1.5 * (|a| + |b|) <= 6e-6 at these inputs
        assert abs(slope - grad[t, h, e]) <= 2 * 6e-6 * np.max(np.abs(gd[t, h])) + 6e-6


@pytest.mark.gpu
def test_rope_backward_of_rotation_returns_the_input():
    import torch

    x = torch.randn(64, 4, 64, device="cuda")
    y, z = torch.empty_like(x), torch.empty_like(x)
    turns, positions = _dev_turns(R.rope_turns(64)), torch.arange(64, dtype=torch.int32, device="cuda") * 999983
    for a, b, inverse in ((x, y, False), (y, z, True)):
        R.rope(R.F32, R.ROPE_HALF, 64, 64, 64, [R.rope_part(a, b, 4, (256, 64), (256, 64))], positions, turns, inverse=inverse)
    pair = x.abs() + x.abs().roll(32, -1)
    assert torch.all((z - x).abs() <= 3 * 6e-7 * pair)  # two rotations, the second of values up to sqrt(2) as large


def test_rope_turns():
    def holds(turns, f):  # whole steps of 2^-64 of a turn, of a frequency in double
        return np.all(np.abs(turns.astype(np.float64) - f * 2.0 ** 64) <= 1.0 + 1e-14 * f * 2.0 ** 64)

    for rotary, base in ((64, 10000.0), (24, 500000.0), (2, 10000.0)):
        f = base ** (-2.0 * np.arange(rotary // 2) / rotary) / (2 * np.pi)
        assert holds(R.rope_turns(rotary, base), f)
        assert holds(R.rope_turns(rotary, base, factor=4.0), f / 4.0)
        turned = 8192 * f
        keep = np.clip((turned - 1.0) / 3.0, 0.0, 1.0)
        assert holds(R.rope_turns(rotary, base, factor=8.0, original_length=8192), f * (keep + (1 - keep) / 8.0))
    # a pair that turns more than once a position keeps the fraction
    assert holds(R.rope_turns(2, 10000.0, factor=0.1), np.array([10.0 / (2 * np.pi) - 1.0]))


def _refused(code, **change):
    a = dict(dtype=R.F16, layout=R.ROPE_HALF, tokens=4, head_dim=64, rotary_dim=64, parts=[R.rope_part(0x1000, 0x2000, 2, (128, 64), (128, 64))],
             positions=0x3000, turns=0x4000)
    a.update(change)
    with pytest.raises(R.R355Error) as e:
        R.rope(**a)
    assert e.value.code == code, str(e.value)


def test_rope_refusals():
    st = (128, 64)
    _refused(-1, turns=None)
    _refused(-1, positions=None)
    _refused(-1, layout=2)
    _refused(-1, parts=[R.rope_part(None, 0x2000, 2, st, st)])
    _refused(-1, parts=[R.rope_part(0x1000, None, 2, st, st)])
    _refused(-1, parts=[R.rope_part(0x1000, 0x2000, 2, st, st, to_slots=True)])
    _refused(-2, dtype=R.I8)
    _refused(-3, rotary_dim=63)
    _refused(-3, rotary_dim=66)
    _refused(-3, rotary_dim=0)
    _refused(-3, head_dim=4098)
    _refused(-3, parts=[R.rope_part(0x1000, 0x2000, 0, st, st)])
    _refused(-4, parts=[R.rope_part(0x1001, 0x2000, 2, st, st)])
    _refused(-4, turns=0x4004)
    for n in (0, 4):
        with pytest.raises(ValueError):
            R.rope(R.F16, R.ROPE_HALF, 4, 64, 64, [R.rope_part(0x1000, 0x2000, 2, st, st)] * n, 0x3000, 0x4000)
    for bad in (dict(rotary_dim=3), dict(rotary_dim=0), dict(base=0.0), dict(factor=0.0), dict(original_length=8192, slow=4.0, fast=4.0)):
        with pytest.raises(R.R355Error):
            R.rope_turns(**{"rotary_dim": 8, **bad})
    R.rope(R.F16, R.ROPE_HALF, 0, 64, 64, [R.rope_part(None, None, 2, st, st)], None, 0x4000)  # no tokens: nothing to do
