"""Products with 4-bit weights at the ends of what their arguments may be (bounds: tests/test_w4.py)."""
import pytest

import rocwmma_amd as R
from test_w4 import _case, _refused


@pytest.mark.gpu
@pytest.mark.parametrize("group", [1 << 31, 2 ** 32 - 128])
@pytest.mark.parametrize("tokens,n", [(1, 40), (20, 24590), (97, 24590)])
def test_w4_one_group_however_long(group, tokens, n):
    """A group far longer than k: k plus its length passes 32 bits."""
    _case("f16", "f32", tokens, n, 1032, group, zeros=True, seed=n)
    _case("bf16", "bf16", tokens, n, 129, group, seed=tokens)


@pytest.mark.parametrize("n,tokens", [(128256, 8400), (28672, 38000), (152064, 65536), (1 << 24, 1023), (32768, (1 << 19) - 1), (1, 1 << 19)])
def test_w4_sizes_are_taken(n, tokens):
    """(as far as the check of the pointers)"""
    _refused(-1, n=n, tokens=tokens, x=None)


def test_w4_more_results_than_that_are_refused():
    _refused(-3, n=1 << 15, tokens=1 << 19)
    _refused(-3, n=(1 << 24) - 15, tokens=1025)


@pytest.mark.gpu
def test_w4_in_several_launches():
    """More tiles than a launch has workgroups: x off the vectors (16 rows x 32 tokens a tile), the result in the place of c."""
    import torch

    n, k, tokens, group = 1 << 22, 4, 1100, 32
    g = torch.Generator(device="cuda").manual_seed(1)
    rows = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device="cuda", generator=g)
    packed = torch.empty(R.w4_packed_bytes(n, k), dtype=torch.uint8, device="cuda")
    R.w4_pack(rows, n, k, packed)
    x, s = torch.randn(tokens, k, device="cuda", generator=g).half(), (0.5 + torch.rand(1, n, device="cuda", generator=g)).half()
    y = torch.empty(tokens, n, dtype=torch.float16, device="cuda")
    y.copy_(torch.arange(tokens, device="cuda").half()[:, None].expand(tokens, n) / 128)
    c = torch.arange(tokens, device="cuda").half().double() / 128
    R.w4_matmul(R.F16, R.F16, tokens, n, k, group, x, packed, s, y, c=y, beta=1.0)
    q = torch.stack([rows & 15, rows >> 4], -1).view(n, k).double()

    def check(got, x, q, s, c):
        want = x.double() @ ((q - 8.0) * s.double()[:, None]).t() + c[:, None]
        spread = x.double().abs() @ ((40.0 + q) * s.double()[:, None]).t()
        bound = (32 + 1 + 16) * 2.0 ** -24 * spread + (2.0 ** -11 + 2.0 ** -22) * want.abs() + 2.0 ** -23 * c[:, None] + 1e-7
        assert torch.all((got.double() - want).abs() <= bound)

    for t in (0, 31, 500, 960, 991, 992, 1023, 1024, tokens - 1):
        check(y[t: t + 1], x[t: t + 1], q, s[0], c[t: t + 1])
    for r in (0, 16, n // 2 - 5, n - 33):
        check(y[:, r: r + 33], x, q[r: r + 33], s[0, r: r + 33], c)
