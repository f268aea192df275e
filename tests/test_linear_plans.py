"""What the calls of a layer's products launch (r355_linear_launch_plan, r355_linear_backward_launch_plan), on the host, and every kernel in every form that can be launched,
against 64 bits (linearlib.py)."""
import ctypes

import pytest

import rocwmma_amd as R

AT = 0x100000  # an address that nothing reads
TILES = [(256, 256), (192, 256), (256, 128), (192, 128), (128, 256), (128, 128), (64, 64)]
SCRATCH = 1 << 26

# rows, n, k, groups, whether there is a workspace -> the tile
FORWARD = [
    (2154, 5880, 272, 1, True, (256, 256)), (2156, 3856, 32, 1, True, (192, 256)), (1938, 3288, 1280, 1, True, (256, 128)), (661, 6000, 144, 1, True, (192, 128)),
    (1081, 6880, 1288, 1, False, (128, 256)), (8376, 480, 32, 1, True, (128, 128)), (19, 16, 32, 1, False, (64, 64)),
    (31, 7824, 96, 16, False, (256, 256)), (2557, 3160, 32, 4, False, (192, 256)), (37, 6128, 2168, 16, True, (256, 128)), (1780, 2424, 136, 4, True, (192, 128)),
    (644, 6296, 1160, 4, False, (128, 256)), (19, 6744, 352, 16, True, (128, 128)), (43, 16, 32, 4, True, (64, 64)),
]
DX = [
    (6803, 272, 2112, 1, False, (256, 256)), (5742, 16, 1520, 1, False, (192, 256)), (8394, 1288, 696, 1, False, (256, 128)), (2123, 136, 1944, 1, False, (192, 128)),
    (2394, 3216, 3256, 1, True, (128, 256)), (7144, 16, 616, 1, False, (128, 128)), (1, 16, 32, 1, True, (64, 64)),
    (509, 16, 4296, 16, False, (256, 256)), (5497, 16, 1360, 16, False, (192, 256)), (8343, 1560, 592, 16, True, (256, 128)), (6262, 144, 592, 16, True, (192, 128)),
    (1190, 1480, 3576, 16, True, (128, 256)), (3, 2608, 4720, 4, True, (128, 128)), (1, 16, 32, 4, True, (64, 64)),
]
DW = [
    (322, 6448, 1992, 1, False, (256, 256)), (1, 7096, 1176, 1, True, (192, 256)), (1156, 1664, 3744, 1, False, (256, 128)), (141, 2552, 1632, 1, False, (192, 128)),
    (1255, 2832, 2712, 1, False, (128, 256)), (1, 4536, 944, 1, True, (128, 128)), (1, 16, 32, 1, True, (64, 64)),
    (4484, 3336, 208, 16, True, (256, 256)), (1, 152, 3000, 16, True, (192, 256)), (5140, 840, 1544, 4, False, (256, 128)), (2134, 912, 264, 16, False, (192, 128)),
    (6641, 1064, 3456, 4, False, (128, 256)), (1, 2192, 88, 16, False, (128, 128)), (1, 16, 32, 4, True, (64, 64)),
]


def _forward(dtype, rows, n, k, groups, space, **kw):
    kw = {"workspace": AT if space else None, "workspace_bytes": SCRATCH if space else 0, **kw}
    return R.linear_args(dtype, dtype, rows, n, k, AT, AT, AT, groups=groups, offsets=AT if groups > 1 else None, **kw)


def _backward(dtype, rows, n, k, groups, space, want, **kw):
    kw = {"workspace": AT if space else None, "workspace_bytes": SCRATCH if space else 0, **kw}
    return R.linear_backward_args(dtype, dtype, rows, n, k, AT, AT, AT, dx=AT if "dx" in want else None, dw=AT if "dw" in want else None, groups=groups,
                                  offsets=AT if groups > 1 else None, **kw)


def _tile(plan):
    return plan.tile_rows, plan.tile_cols


def _offsets(rows, groups):
    """Uneven, the first and the last group without rows where there are more than two"""
    if groups == 1:
        return None
    share = [0.0 if groups > 2 and g in (0, groups - 1) else 0.3 + (g * 0.618033989) % 1 for g in range(groups)]
    return [int(rows * sum(share[:g]) / sum(share) + 0.5) for g in range(groups + 1)]


def test_every_tile_in_every_form():
    """The sizes below take each tile in each form, of one matrix of weights and of groups"""
    for dtype in (R.F16, R.BF16):
        for cases, plan in ((FORWARD, lambda *c: R.linear_launch_plan(_forward(dtype, *c))), (DX, lambda *c: R.linear_backward_launch_plan(_backward(dtype, *c, ("dx",)))[0]),
                            (DW, lambda *c: R.linear_backward_launch_plan(_backward(dtype, *c, ("dw",)))[1])):
            for *case, tile in cases:
                p = plan(*case)
                assert (p.kernel, _tile(p)) == (R.LINEAR_TILES, tile), case
            for grouped in (False, True):
                assert {c[5] for c in cases if (c[3] > 1) == grouped} == set(TILES)


@pytest.mark.gpu
@pytest.mark.parametrize("at", range(len(FORWARD)))
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_forward(dtype, at):
    import torch

    import linearlib

    rows, n, k, groups, space, _ = FORWARD[at]
    linearlib.run_linear(dtype, dtype if at % 2 else "f32", rows, n, k, act="silu", bias=True, gate=True, c=True, keep=True, groups=groups, offsets=_offsets(rows, groups),
                         workspace=torch.full((SCRATCH,), 0xFF, dtype=torch.uint8, device="cuda") if space else None, seed=at)


@pytest.mark.gpu
@pytest.mark.parametrize("at", range(len(DX)))
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("want", ["dx", "dw"])
def test_backward(want, dtype, at):
    import torch

    import linearlib

    rows, n, k, groups, space, _ = (DX if want == "dx" else DW)[at]
    linearlib.run_backward(dtype, dtype if at % 2 else "f32", rows, n, k, groups=groups, offsets=_offsets(rows, groups), accumulate=at % 3 == 0, want=(want,),
                           workspace=torch.full((SCRATCH,), 0xFF, dtype=torch.uint8, device="cuda") if space else None, seed=at)


def test_other_kernels():
    plan = R.linear_launch_plan(_forward(R.BF16, 1, 1024, 2048, 1, True))
    assert (plan.kernel, plan.tile_rows, plan.splits) == (R.LINEAR_DOTS, 0, 0)
    assert R.linear_launch_plan(_forward(R.BF16, 30, 1024, 2048, 32, True)).kernel == R.LINEAR_DOTS
    assert R.linear_launch_plan(_forward(R.F16, 16, 1024, 2048, 1, True)).kernel == R.LINEAR_FEW
    assert R.linear_launch_plan(_forward(R.F16, 12, 1024, 1024, 4, True)).kernel == R.LINEAR_FEW
    plan = R.linear_launch_plan(_forward(R.F16, 1, 1024, 2047, 1, False))
    assert (plan.kernel, _tile(plan)) == (R.LINEAR_ELEMENTS, (64, 64))
    assert R.linear_launch_plan(_forward(R.BF16, 0, 64, 64, 1, True)).kernel == R.LINEAR_NONE
    for want, which in (("dx", 0), ("dw", 1)):
        plans = R.linear_backward_launch_plan(_backward(R.BF16, 100, 45, 67, 1, False, (want,)))
        assert (plans[which].kernel, _tile(plans[which])) == (R.LINEAR_ELEMENTS, (64, 64)) and plans[1 - which].kernel == R.LINEAR_NONE


def test_splits_copies_rests_and_both_in_one():
    plan = R.linear_launch_plan(_forward(R.BF16, 100, 512, 8192, 1, True))
    assert plan.kernel == R.LINEAR_TILES and plan.splits > 1 and R.linear_launch_plan(_forward(R.BF16, 100, 512, 8192, 1, False)).splits == 1
    plan = R.linear_launch_plan(_forward(R.BF16, 1500, 1496, 1500, 1, True))
    assert (plan.kernel, plan.copies) == (R.LINEAR_TILES, 2) and R.linear_launch_plan(_forward(R.BF16, 1500, 1496, 1500, 1, False)).kernel == R.LINEAR_ELEMENTS
    dx, dw = R.linear_backward_launch_plan(_backward(R.BF16, 4099, 4096, 4096, 1, True, ("dx", "dw")))
    assert (_tile(dx), dx.first_rows, dx.together, _tile(dw)) == ((256, 256), 4096, 0, (256, 256))
    dx, dw = R.linear_backward_launch_plan(_backward(R.BF16, 2048, 1024, 1024, 1, True, ("dx", "dw")))
    assert dx.together == dw.together == 1 and _tile(dx) == _tile(dw) == (64, 64) and dx.splits >= 1 and dw.splits >= 1
    dx, dw = R.linear_backward_launch_plan(_backward(R.BF16, 0, 1024, 1024, 1, True, ("dx", "dw")))
    assert dx.kernel == R.LINEAR_NONE and dw.kernel == R.LINEAR_TILES


def test_what_is_refused_has_no_plan():
    a = _forward(R.BF16, 4, 8, 16, 1, False)
    a.ldx = 15
    with pytest.raises(R.R355Error):
        R.linear_launch_plan(a)
    a = _backward(R.BF16, 4, 8, 16, 1, False, ("dx",))
    a.lddx = 15
    with pytest.raises(R.R355Error):
        R.linear_backward_launch_plan(a)
    plan = R.LinearPlan()
    assert R.lib().r355_linear_launch_plan(None, ctypes.byref(plan)) == -1 and R.lib().r355_linear_launch_plan(ctypes.byref(_forward(R.BF16, 4, 8, 16, 1, False)), None) == -1
    assert R.lib().r355_linear_backward_launch_plan(ctypes.byref(_backward(R.BF16, 4, 8, 16, 1, False, ("dx",))), None, ctypes.byref(plan)) == -1
