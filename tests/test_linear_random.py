"""Calls of linear() and linear_backward() drawn over what their documentation allows (sizes, groups, rows by their numbers, strides, alignment, parts of the epilogue, workspaces of any size), against
64 bits (linearlib.py)."""
import math
import random

import pytest


def _log(rng, least, most):
    return int(round(math.exp(rng.uniform(math.log(least), math.log(most)))))


def _sizes(rng):
    """rows, n, k, groups and offsets of a call that is quickly checked; half of them with lengths in multiples of 8"""
    while True:
        even = rng.random() < 0.6
        rows = _log(rng, 1, 9000)
        n, k = (8 * _log(rng, 1, 700), 8 * _log(rng, 1, 500)) if even else (_log(rng, 1, 3000), _log(rng, 1, 2500))
        groups = rng.choice([1, 1, 1, 2, 5, 8, 16, 40, 70])
        if rows * n * k <= 3e10 and groups * n * k <= 3e8:
            break
    offsets = None
    if groups > 1:
        offsets = sorted(rng.randint(0, rows) for _ in range(groups + 1))
        if rng.random() < 0.6:
            offsets[0], offsets[-1] = 0, rows
        if rng.random() < 0.3:  # groups without rows
            at = rng.randrange(groups)
            offsets[at: at + 3] = [offsets[at]] * len(offsets[at: at + 3])
    elif rng.random() < 0.1:
        first = rng.randint(0, rows)
        offsets = [first, rng.randint(first, rows)]
    return even, rows, n, k, groups, offsets


def _common(rng, scratch):
    dtype = rng.choice(["f16", "bf16"])
    return dtype, rng.choice([dtype, "f32"]), dict(act=rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"]), gate=rng.random() < 0.4, offset=rng.choice([0, 0, 0, 8, 1, 3]),
                                                   workspace=rng.choice([None, scratch, scratch, scratch[: 16 * rng.randint(1, 1 << 16)]]), seed=rng.randrange(10 ** 6))


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(16))
def test_forward(seed):
    import torch

    import linearlib

    rng, scratch = random.Random(seed), torch.full((1 << 26,), 0xFF, dtype=torch.uint8, device="cuda")
    for _ in range(25):
        even, rows, n, k, groups, offsets = _sizes(rng)
        dtype, out, kw = _common(rng, scratch)
        source = x_rows = None
        if rng.random() < 0.3:
            x_rows = rng.randint(1, rows)
            source = [rng.randint(-1, x_rows) if rng.random() < 0.05 else rng.randrange(x_rows) for _ in range(rows)]
        c = rng.random() < 0.4
        kw.update(bias=rng.random() < 0.5, c=c, in_place=c and rng.random() < 0.4, keep=rng.random() < 0.4, pad=tuple(rng.choice([0, 0, 8, 64] if even else [0, 0, 8, 16, 1, 5]) for _ in range(6)))
        print(dtype, out, rows, n, k, groups, offsets, x_rows, {name: value for name, value in kw.items() if name != "workspace"}, flush=True)
        linearlib.run_linear(dtype, out, rows, n, k, groups=groups, offsets=offsets, source=source, x_rows=x_rows, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(16))
def test_backward(seed):
    import torch

    import linearlib

    rng, scratch = random.Random(100 + seed), torch.full((1 << 26,), 0xFF, dtype=torch.uint8, device="cuda")
    for _ in range(25):
        even, rows, n, k, groups, offsets = _sizes(rng)
        dtype, grad, kw = _common(rng, scratch)
        kw.update(accumulate=rng.random() < 0.3, want=rng.choice([("dx", "dw", "dbias"), ("dx",), ("dw",), ("dx", "dw"), ("dw", "dbias")]), pad=rng.choice([0, 0, 8, 64] if even else [0, 0, 8, 1, 5]))
        print(dtype, grad, rows, n, k, groups, offsets, {name: value for name, value in kw.items() if name != "workspace"}, flush=True)
        linearlib.run_backward(dtype, grad, rows, n, k, groups=groups, offsets=offsets, **kw)
