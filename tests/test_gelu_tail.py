"""GELU where its values are small: relative to themselves, of every kernel that takes the activation.

z are the 16-bit values given (one product of one with z).  The distribution function is off by eps = 2^-24 times: 0.8 (the polynomial), 6 (t: two roundings, times what t P(t) makes of them), 4
(its steps), 2 (the exponential) and 2.2 z^2 / 2 (its argument: z^2 and the product with log2 e are rounded), less than 1.5 z^2 + 14 in all; with z and the result's rounding 1.5 z^2 + 16."""
import pytest

import rocwmma_amd as R

EPS = 2.0 ** -24


def _cdf(z):
    """By erfc, which keeps the lower tail (torch.special.ndtr does not: in 64 bits it is 0 from -8.3 on)"""
    import torch

    return 0.5 * torch.special.erfc(-z * 0.5 ** 0.5)


def _points(n):
    """From -13 to 8, as f16 has them, n times over"""
    import torch

    return torch.cat([torch.linspace(-13, 0, 6 * n // 8, device="cuda"), torch.linspace(0, 8, n - 6 * n // 8, device="cuda")]).half()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,k,space", [(1, 8, 0), (2, 8, 0), (16, 8, 0), (200, 8, 0), (200, 7, 0), (200, 4096, 1 << 24)])
def test_values(rows, k, space):
    """Dot products, few rows, tiles, single elements, a split sum"""
    import torch

    n = 1024
    z = _points(n)
    x, w = torch.zeros(rows, k, device="cuda").half(), torch.zeros(n, k, device="cuda").half()
    x[:, k - 1], w[:, k - 1] = 1.0, z
    y = torch.full((rows, n), float("nan"), device="cuda")
    workspace = torch.empty(space, dtype=torch.uint8, device="cuda") if space else None
    if space:
        assert R.linear_launch_plan(R.linear_args(R.F16, R.F32, rows, n, k, x, w, y, activation=R.ACT_GELU, workspace=workspace)).splits > 1
    R.linear(R.F16, R.F32, rows, n, k, x, w, y, activation=R.ACT_GELU, workspace=workspace)
    zd = z.double()
    want = zd * _cdf(zd)
    off = (y.double() - want).abs()
    far = (1.5 * zd * zd + 16) * EPS * want.abs() + zd.abs() * 2.0 ** -126  # (what is flushed)
    assert (off <= far).all(), (off / far).max().item()


@pytest.mark.gpu
def test_slopes():
    """Of one row, by the bias's gradient, which no rounding to 16 bits comes before: Phi(z) + z phi(z), each of the two within the bound, and their sum"""
    import torch

    n = 2048
    z = _points(n).view(1, n)
    dy, db, dz = torch.ones(1, n, device="cuda").half(), torch.empty(n, device="cuda"), torch.empty(1, n, device="cuda").half()
    R.linear_backward(R.F16, R.F16, 1, n, 8, dy, None, None, dbias=db, z=z, activation=R.ACT_GELU, dz=dz)
    zd = z[0].double()
    cdf, density = _cdf(zd), torch.exp(-zd * zd / 2) / (2 * torch.pi) ** 0.5
    off, far = (db.double() - (cdf + zd * density)).abs(), (1.5 * zd * zd + 18) * EPS * (cdf + (zd * density).abs()) + (1 + zd.abs()) * 2.0 ** -126
    assert (off <= far).all(), (off / far).max().item()
