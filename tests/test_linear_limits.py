"""Sizes at which a kernel's launch ends: another kernel takes them, or the call is refused before anything is launched."""
import pytest

import rocwmma_amd as R

AT = 0x100000
MOST = 2 ** 24 - 8  # workgroups of 256 threads


def _forward(rows, n, k, groups=1, **kw):
    return R.linear_args(R.BF16, R.BF16, rows, n, k, AT, AT, AT, groups=groups, offsets=AT if groups > 1 else None, **kw)


def _tiles(rows, n, groups, edge, across):
    """That any division of the rows into groups fits in"""
    whole = min(rows // edge + groups, rows) if groups > 1 else -(-rows // edge)
    return whole * -(-n // across)


@pytest.mark.parametrize("rows,n,groups", [(5184, 99568, 1024), (5184, 99552, 1024), (1024, 131072, 1024), (1024, 131056, 1024), (5184, 99504, 1024), (1024, 130928, 1024)])
def test_few_rows_of_many_groups(rows, n, groups):
    """Workgroups of 512 threads, as many for each XCD: 1348 x 6223 tiles are 4 fewer than 2^23, which rounded up are 2^32 threads"""
    plan = R.linear_launch_plan(_forward(rows, n, 8, groups))
    edge = 1 if rows <= groups else 16
    rounded = -(-_tiles(rows, n, groups, edge, 16) // 8) * 8
    if rounded > MOST // 2:
        assert plan.kernel == R.LINEAR_TILES
    else:
        assert plan.kernel == (R.LINEAR_DOTS if rows <= groups else R.LINEAR_FEW)


@pytest.mark.parametrize("rows,n,groups", [(2 ** 30, 8, 1), (2 ** 30, 64, 1), (2 ** 29, 200, 1), (2 ** 30, 8, 1000), (1024, 2 ** 21, 1024)])
def test_tiles_that_a_launch_holds(rows, n, groups):
    plan = R.linear_launch_plan(_forward(rows, n, 8, groups))
    assert plan.kernel == R.LINEAR_TILES and 0 < -(-_tiles(plan.first_rows or rows, n, groups, plan.tile_rows, plan.tile_cols) // 8) * 8 <= MOST
    dx, _ = R.linear_backward_launch_plan(R.linear_backward_args(R.BF16, R.BF16, rows, 8, n, AT, AT, AT, dx=AT, groups=groups, offsets=AT if groups > 1 else None))
    assert dx.kernel == R.LINEAR_TILES and 0 < -(-_tiles(dx.first_rows or rows, n, groups, dx.tile_rows, dx.tile_cols) // 8) * 8 <= MOST


def test_gradients_of_large_weights():
    args = R.linear_backward_args(R.BF16, R.BF16, 64, 2 ** 18, 2 ** 18, AT, AT, AT, dw=AT)
    _, dw = R.linear_backward_launch_plan(args)
    assert dw.kernel == R.LINEAR_TILES and dw.tile_rows * dw.tile_cols > 64 * 64
    assert R.linear_backward_launch_plan(R.linear_backward_args(R.BF16, R.BF16, 64, 2 ** 18, 2 ** 18, AT, AT, AT, dx=AT, dw=AT))[1].together == 0


@pytest.mark.parametrize("call", ["forward", "dx", "dw"])
def test_refused_before_anything_is_launched(call):
    """Results that no tiles cover in one launch: an error from the plan and from the call, which writes nothing (the addresses are nobody's)"""
    import ctypes

    most = 2 ** 22 - 8
    if call == "forward":
        a, lib = _forward(2 ** 30, most, 8), R.lib().r355_linear
        plan = lambda: R.linear_launch_plan(a)  # noqa: E731
    else:
        kw = dict(dx=AT) if call == "dx" else dict(dw=AT)
        rows, n, groups = (2 ** 30, 8, 1) if call == "dx" else (8, most, 1024)
        a, lib = R.linear_backward_args(R.BF16, R.BF16, rows, n, most, AT, AT, AT, groups=groups, offsets=AT if groups > 1 else None, z=AT, dz=AT, activation=R.ACT_SILU, **kw), R.lib().r355_linear_backward
        plan = lambda: R.linear_backward_launch_plan(a)  # noqa: E731
    with pytest.raises(R.R355Error) as refused:
        plan()
    assert refused.value.code == -3
    assert lib(ctypes.byref(a), None) == -3


@pytest.mark.gpu
def test_a_billion_rows():
    """2^30 rows of 8 elements, more tiles of 64 rows than a launch holds; in values that 16 bits hold exactly"""
    import torch

    rows, n = 2 ** 30, 8
    x = torch.empty(rows, 8, dtype=torch.bfloat16, device="cuda")
    piece = torch.randint(-3, 4, (1 << 20, 8), device="cuda").bfloat16()
    x.view(1024, 1 << 20, 8)[:] = piece
    x.view(1024, 1 << 20, 8)[:, 0, 0] = torch.arange(1024, device="cuda").bfloat16()  # (to 8 bits)
    w = torch.randint(-2, 3, (n, 8), device="cuda").bfloat16()
    y = torch.full((rows, n), float("nan"), dtype=torch.bfloat16, device="cuda")
    R.linear(R.BF16, R.BF16, rows, n, 8, x, w, y)
    torch.cuda.synchronize()
    for at in range(0, 1024, 31):
        rows_ = slice(at << 20, at + 1 << 20)
        assert torch.equal(y[rows_], (x[rows_].float() @ w.float().t()).bfloat16()), at
