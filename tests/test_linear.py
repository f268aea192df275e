"""Products with bias, activation, gate and residual in their epilogue, for one matrix of weights and grouped by expert, against 64 bits (linearlib.py has the bounds)."""
import pytest

import rocwmma_amd as R


def _run(*args, **kw):
    import linearlib

    return linearlib.run_linear(*args, **kw)


def _offsets(sizes):
    at = [0]
    for s in sizes:
        at.append(at[-1] + s)
    return at


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("rows,n,k", [(1, 1, 8), (1, 64, 64), (3, 40, 136), (16, 17, 512), (17, 64, 72), (33, 130, 264), (64, 64, 128), (65, 72, 1000), (130, 257, 392), (300, 264, 8)])
def test_sizes(dtype, rows, n, k):
    _run(dtype, dtype, rows, n, k, act="silu", bias=True, seed=rows + n)
    _run(dtype, "f32", rows, n, k, c=True, keep=True, seed=rows + n + 1)


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("rows,n", [(2, 48), (70, 96), (70, 91)])
def test_epilogue(act, rows, n):
    _run("bf16", "bf16", rows, n, 256, act=act, bias=True, gate=True, c=True, keep=True, scale=3.0)
    _run("f16", "f32", rows, n, 256, act=act, gate=True, scale=8.0)
    _run("f16", "f16", rows, n, 256, act=act, bias=True, c=True, in_place=True)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n,k", [(3000, 4500, 72), (2500, 3584, 192), (5000, 5000, 24), (1024, 2048, 320), (700, 1300, 200)])
def test_many_tiles(rows, n, k):
    _run("bf16", "bf16", rows, n, k, act="gelu_tanh", bias=True, keep=True)
    _run("f16", "f32", rows, n, k, gate=True, c=True)


@pytest.mark.gpu
@pytest.mark.parametrize("k", [8, 56, 64, 72, 120, 128, 136, 184, 192, 248, 320, 448, 1032])
def test_lengths_of_the_sum(k):
    """Every number of stages around those that the loops request ahead, in each tile"""
    _run("f16", "f16", 2300, 6200, k, bias=True)
    _run("bf16", "f32", 1100, 1600, k)
    _run("bf16", "bf16", 100, 200, k)
    _run("f16", "f32", 9, 100, k)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,out", [("f16", "f16"), ("bf16", "f32")])
@pytest.mark.parametrize("rows,n,k", [(5, 33, 67), (70, 129, 45), (200, 65, 1001), (1, 7, 1), (64, 64, 64)])
def test_any_alignment(dtype, out, rows, n, k):
    """Odd lengths, rows an odd number of elements apart, first elements off every boundary but their own"""
    _run(dtype, out, rows, n, k, act="silu", bias=True, gate=True, c=True, keep=True, pad=(1, 3, 5, 2, 7, 1), offset=1)
    _run(dtype, out, rows, n, k, groups=3, offsets=_offsets([rows // 2, 0, rows - rows // 2]), pad=(0, 1, 0, 0, 0, 0), source=[(7 * r) % rows for r in range(rows)])


@pytest.mark.gpu
@pytest.mark.parametrize("pad", [(8, 0, 0, 0, 0, 0), (0, 16, 0, 0, 0, 0), (0, 0, 8, 8, 8, 8), (0, 0, 1, 0, 0, 0), (0, 0, 0, 0, 1, 0), (0, 0, 0, 3, 0, 5)])
def test_strides(pad):
    _run("bf16", "bf16", 150, 136, 128, act="gelu", bias=True, gate=True, c=True, keep=True, pad=pad)
    _run("f16", "f32", 10, 136, 128, act="relu", bias=True, gate=True, c=True, keep=True, pad=pad)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("sizes", [[0, 5, 0, 0, 40], [1] * 70, [0] * 64 + [3, 0, 130], [300, 1, 0, 64], [16, 17, 15, 33, 0, 2], [0, 0, 0], [513, 1700, 0, 900], [0] * 1000 + [77] * 24])
def test_groups(dtype, sizes):
    rows = sum(sizes) or 4
    source = [(13 * r + 5) % max(1, rows // 2) for r in range(rows)]
    _run(dtype, dtype, rows, 136 if len(sizes) < 100 else 24, 64, act="silu", bias=True, gate=True, groups=len(sizes), offsets=_offsets(sizes))
    _run(dtype, "f32", rows, 33, 72, bias=True, c=True, keep=True, groups=len(sizes), offsets=_offsets(sizes), source=source, x_rows=max(1, rows // 2))


@pytest.mark.gpu
@pytest.mark.parametrize("k", [64, 200, 328])
def test_groups_on_large_tiles(k):
    """Last tiles of 1 to 255 rows beside whole ones"""
    sizes = [2300, 1, 64, 0, 65, 128, 129, 192, 193, 255, 256, 300, 100, 1500]
    _run("bf16", "bf16", sum(sizes), 4000, k, act="silu", bias=True, gate=True, groups=len(sizes), offsets=_offsets(sizes))
    _run("f16", "f32", sum(sizes), 4001, k, c=True, keep=True, groups=len(sizes), offsets=_offsets(sizes), source=[(13 * r + 5) % 999 for r in range(sum(sizes))], x_rows=999)


@pytest.mark.gpu
def test_groups_of_some_rows():
    """Offsets that begin after the first row and end before the last; a slice of the offsets is some of the experts"""
    _run("bf16", "bf16", 500, 72, 64, bias=True, groups=3, offsets=[17, 100, 100, 450], c=True, in_place=True)
    _run("bf16", "bf16", 40, 72, 64, bias=True, groups=4, offsets=[3, 3, 9, 20, 31])


@pytest.mark.gpu
@pytest.mark.parametrize("offsets", [[0, 900, 950, 1000], [-5, 10, 50, 60], [50, 20, 60, 60], [-2 ** 31, -1, 2 ** 31 - 1, 60]])
@pytest.mark.parametrize("k", [64, 65])
def test_offsets_beyond_the_rows_are_cut_off(offsets, k):
    import linearlib

    if sorted(offsets) == offsets:
        _run("f16", "f16", 60, 40, k, groups=3, offsets=offsets)
    else:  # (what groups that overlap leave is not said, where they write is)
        import torch

        x, w = torch.randn(60, k, device="cuda").half(), torch.randn(3, 40, k, device="cuda").half()
        y, view = linearlib.matrix(torch.zeros(60, 40, device="cuda"), torch.float16, 44)
        R.linear(R.F16, R.F16, 60, 40, k, x, w, y, groups=3, offsets=torch.tensor(offsets, dtype=torch.int32).cuda(), ldy=44)
        assert torch.isnan(view[0, :, 40:]).all() and torch.isnan(y[60 * 44:]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,groups", [(200, 300), (2000, 300), (5000, 130)])
def test_groups_that_are_no_division_of_the_rows(rows, groups):
    """Every other group claims all rows: more tiles than a launch has workgroups for.  Every row that is written is one of the groups' results"""
    import linearlib
    import torch

    n, k = 40, 64
    x, w = torch.randint(-2, 3, (rows, k), device="cuda").half(), torch.randint(-2, 3, (1, n, k), device="cuda").half().expand(groups, n, k).contiguous()
    offsets = torch.tensor([0, rows] * (groups // 2 + 1), dtype=torch.int32)[: groups + 1].cuda()
    y, view = linearlib.matrix(torch.zeros(rows, n, device="cuda"), torch.float16, n + 4)
    y.fill_(float("nan"))
    R.linear(R.F16, R.F16, rows, n, k, x, w, y, groups=groups, offsets=offsets, ldy=n + 4)
    assert torch.isnan(view[0, :, n:]).all() and torch.isnan(y[rows * (n + 4):]).all()
    want = x.float() @ w[0].float().t()
    got = view[0, :, :n].float()
    assert (torch.isnan(got) | (got == want)).all() and (got == want).any()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,k", [(6, 64), (300, 72), (30, 65)])
def test_source_rows_that_are_not_there_read_as_zeros(rows, k):
    source = [(r * 7) % 11 for r in range(rows)]
    source[1], source[rows // 2], source[-1] = -1, 11, 2 ** 31 - 1
    _run("bf16", "bf16", rows, 40, k, bias=True, source=source, x_rows=11)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,k", [(6, 64), (300, 64), (300, 63)])
def test_infinities_and_nan_stay_in_their_rows_and_columns(rows, k):
    import torch

    x, w = torch.randn(rows, k, device="cuda").bfloat16(), torch.randn(40, k, device="cuda").bfloat16()
    x[2, 5], x[rows - 1, k - 1], w[7, 3] = float("inf"), float("nan"), float("nan")
    y = torch.zeros(rows, 40, dtype=torch.bfloat16, device="cuda")
    R.linear(R.BF16, R.BF16, rows, 40, k, x, w, y)
    bad = ~torch.isfinite(y)
    want = torch.zeros_like(bad)
    want[2], want[-1], want[:, 7] = True, True, True
    assert torch.equal(bad, want)


@pytest.mark.gpu
def test_activations_at_their_ends():
    """Far arguments, infinities and NaN of the activations; one product of one element each, so that the argument is exact"""
    import torch

    values = [0.0, -0.0, 1e-3, -1e-3, 20.0, -20.0, 100.0, -100.0, 3e4, -3e4, float("inf"), float("nan")]
    x = torch.zeros(len(values), 8, dtype=torch.float16, device="cuda")
    x[:, 0] = torch.tensor(values)
    w = torch.zeros(8, 8, dtype=torch.float16, device="cuda")
    w[:, 0] = 1.0
    for act, f in (("RELU", torch.relu), ("GELU", torch.nn.functional.gelu), ("GELU_TANH", lambda v: torch.nn.functional.gelu(v, approximate="tanh")), ("SILU", torch.nn.functional.silu)):
        y = torch.empty(len(values), 8, dtype=torch.float32, device="cuda")
        R.linear(R.F16, R.F32, len(values), 8, 8, x[:], w, y, activation=getattr(R, "ACT_" + act))
        want = f(torch.tensor(values, dtype=torch.float16).double())
        got = y[:, 0].cpu().double()
        assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.isinf(got), torch.isinf(want)), act
        fine = torch.isfinite(want)
        assert ((got - want)[fine].abs() <= 2.0 ** -18 * want[fine].abs() + 2.0 ** -22 * torch.tensor(values)[fine].abs().clamp(max=20.0)).all(), act


@pytest.mark.gpu
def test_long_matrices():
    """Operands and results past 2^31 bytes; rows and weights from their far ends"""
    import torch

    n, k, rows = 2048, 2048, 600000
    x = torch.zeros(rows, k, dtype=torch.bfloat16, device="cuda")
    w = torch.randn(n, k, device="cuda").bfloat16()
    at = [0, 299999, 524288, rows - 1]
    x[at] = torch.randn(4, k, device="cuda").bfloat16()
    y = torch.empty(rows, n, dtype=torch.bfloat16, device="cuda")
    R.linear(R.BF16, R.BF16, rows, n, k, x, w, y)
    want = x[at].double() @ w.double().t()
    assert ((y[at].double() - want).abs() <= 2.0 ** -7 * want.abs() + 1e-3).all()
    assert (y[1:1000] == 0).all() and (y[-1000:-1] == 0).all()


@pytest.mark.gpu
def test_streams_and_graph():
    """On a stream of its own; recorded with new offsets and values at every replay, the eager work of the program between them"""
    import linearlib
    import torch

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    _run("bf16", "bf16", 100, 72, 128, act="silu", bias=True, stream=None)
    rows, n, k, groups = 90, 136, 128, 5
    x, w = torch.randn(rows, k, device="cuda").bfloat16(), torch.randn(groups, n, k, device="cuda").bfloat16()
    offsets = torch.zeros(groups + 1, dtype=torch.int32, device="cuda")
    y, eager = (torch.zeros(rows, n, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    call = lambda to, s: R.linear(R.BF16, R.BF16, rows, n, k, x, w, to, activation=R.ACT_SILU, groups=groups, offsets=offsets, stream=s)  # noqa: E731
    call(y, None)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        call(y, torch.cuda.current_stream())
    for step, at in enumerate([[0, 10, 10, 50, 60, 90], [0, 0, 0, 0, 90, 90], [0, 1, 2, 3, 4, 90], [5, 20, 30, 40, 50, 60]]):
        offsets.copy_(torch.tensor(at, dtype=torch.int32))
        x.copy_(torch.randn(rows, k, device="cuda"))
        y.zero_(), eager.zero_()
        graph.replay()
        call(eager, None)
        torch.cuda.synchronize()
        assert torch.equal(y, eager) and eager.abs().sum() > 0
    assert linearlib.EPS


def _workspace_bytes(rows, n, k, **kw):
    return R.linear_workspace_bytes(R.linear_args(R.BF16, R.BF16, rows, n, k, 0x1000, 0x2000, 0x3000, **kw))


def _scratch(nbytes):
    import torch

    return torch.full((nbytes,), 255, dtype=torch.uint8, device="cuda")  # (NaN, whatever is read of it before it is written)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n,k,pad", [(100, 200, 4096, 0), (65, 129, 2056, 3), (300, 70, 1999, 1), (17, 513, 8192, 0)])
def test_sums_split_over_workgroups(rows, n, k, pad):
    """With a workspace and few tiles: the whole epilogue after the shares are added, c in place, both types of the result, a workspace for fewer shares, one that is too small for any"""
    need = _workspace_bytes(rows, n, k, ldx=k + pad)
    assert need > 0
    for size in (need, need // 2 // 16 * 16, 16):
        _run("bf16", "bf16", rows, n, k, act="gelu", bias=True, gate=True, c=True, keep=True, pad=(pad, 0, pad, pad, pad, pad), workspace=_scratch(size))
        _run("f16", "f32", rows, n, k, act="silu", bias=True, c=True, in_place=True, pad=(pad, 0, 0, 0, 0, 0), workspace=_scratch(size))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n,k,groups,pad,offset,gather", [(700, 1000, 999, 1, 0, 0, False), (600, 1100, 1024, 1, 3, 1, True), (1000, 600, 1003, 3, 1, 1, True), (1500, 700, 520, 4, 4, 0, False)])
def test_operands_laid_out_anew(rows, n, k, groups, pad, offset, gather):
    """Rows off 16-byte boundaries, or that end inside 16 bytes, with a workspace that holds them evenly; NaN behind every row and beside the operands"""
    offsets = None if groups == 1 else _offsets([rows // 2, 0] + [rows // 8] * (groups - 2))
    a = R.linear_args(R.BF16, R.BF16, rows, n, k, 0x1000 + 2 * offset, 0x2000 + 2 * offset, 0x3000, groups=groups, offsets=0x4000 if groups > 1 else None, ldx=k + pad, ldw=k + pad,
                      source=0x5000 if gather else None, x_rows=rows // 3 if gather else None)
    eights = (k + 7) // 8 * 8
    need = R.linear_workspace_bytes(a)
    assert need >= 2 * eights * groups * n
    kw = dict(groups=groups, offsets=offsets, pad=(pad, pad, 0, 0, 0, 0), offset=offset)
    if gather:
        kw.update(source=[(13 * r + 5) % (rows // 3) for r in range(rows)], x_rows=rows // 3)
    for size in (need, 2 * eights * groups * n // 2):
        _run("bf16", "bf16", rows, n, k, act="silu", bias=True, gate=True, keep=True, workspace=_scratch(size), **kw)
        _run("f16", "f32", rows, n, k, c=True, workspace=_scratch(size), **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("offsets,rows,n,k", [([0, 30, 30, 58, 60], 60, 200, 4096), ([3, 20, 50], 64, 1030, 2056), ([0] * 70 + [40] + [90] * 60, 97, 33, 1999), ([5, 90], 100, 72, 2048),
                                                ([3, 20, 50], 64, 1030, 8200), ([5, 90], 100, 72, 8192), ([0] * 70 + [40] + [90] * 60, 97, 33, 5999)])
def test_sums_of_groups_split_over_workgroups(offsets, rows, n, k):
    """Rows before, between and behind the groups are left as they were, also by what adds the shares"""
    groups = len(offsets) - 1
    need = _workspace_bytes(rows, n, k, groups=groups, offsets=0x4000)
    assert need > 0 or k < 4096  # (short sums are left whole)
    need = need or 1 << 16
    _run("bf16", "bf16", rows, n, k, act="gelu", bias=True, gate=True, keep=True, groups=groups, offsets=offsets, workspace=_scratch(need))
    _run("f16", "f32", rows, n, k, bias=True, c=True, in_place=True, groups=groups, offsets=offsets, workspace=_scratch(need // 2 // 16 * 16))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n,k", [(4099, 4096, 1544), (2600, 8192, 1600)])
def test_rows_past_whole_rounds_of_tiles(rows, n, k):
    """The rows that whole rounds of large tiles leave go out on tiles of their own, all operands with them, split along the sum where there is a workspace"""
    _run("bf16", "bf16", rows, n, k, act="silu", bias=True, gate=True, c=True, keep=True, pad=(0, 0, 8, 16, 24, 32))
    _run("f16", "f32", rows, n, k, c=True, in_place=True, source=[(13 * r + 5) % 2000 for r in range(rows)], x_rows=2000, workspace=_scratch(1 << 24))


@pytest.mark.gpu
@pytest.mark.parametrize("sizes,n,k", [([1] * 32, 2048, 1024), ([4] * 16, 2048, 2048), ([5, 0, 0, 1, 0, 0, 0, 0, 2, 0], 80, 1032), ([3, 0, 9, 0, 20], 100, 2056), ([0, 1], 72, 64)])
def test_few_rows_of_each_group(sizes, n, k):
    """The kernels for few rows, with weights that the caches hold and that they do not, with several of their tiles to a group"""
    _run("bf16", "bf16", sum(sizes), n, k, act="silu", bias=True, gate=True, groups=len(sizes), offsets=_offsets(sizes))
    _run("f16", "f32", sum(sizes), n, k, c=True, keep=True, groups=len(sizes), offsets=_offsets(sizes), source=[(3 * r) % 5 for r in range(sum(sizes))], x_rows=5)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [2, 12, 70, 900])
def test_one_group_with_offsets(rows):
    _run("bf16", "bf16", rows, 72, 128, bias=True, act="relu", groups=1, offsets=[rows // 3, rows - 1], c=True, in_place=True)


@pytest.mark.gpu
@pytest.mark.parametrize("pad,offset", [(0, 0), (64, 0), (8, 0), (0, 32)])
def test_rows_of_results_on_and_off_cache_lines(pad, offset):
    """Results whose rows begin with a cache line are written past the caches, others not: what lies between the rows stays, in either case"""
    _run("bf16", "bf16", 300, 256, 128, act="silu", keep=True, pad=(0, 0, 0, 0, pad, 64 - pad % 64), offset=offset)
    _run("f16", "f32", 300, 256, 128, c=True, in_place=True, pad=(0, 0, 0, 0, pad, 0), offset=offset)


@pytest.mark.gpu
def test_two_calls_at_once():
    """On two streams, each with a workspace of its own, against the same calls one after the other"""
    import torch

    rows, n, k = 100, 200, 4096
    a = [torch.randn(rows, k, device="cuda").bfloat16() for _ in range(2)]
    w = [torch.randn(n, k, device="cuda").bfloat16() for _ in range(2)]
    streams, need = [torch.cuda.Stream() for _ in range(2)], _workspace_bytes(rows, n, k)
    scratch = [_scratch(need) for _ in range(2)]
    alone, both = ([torch.empty(rows, n, dtype=torch.bfloat16, device="cuda") for _ in range(2)] for _ in range(2))
    for i in range(2):
        R.linear(R.BF16, R.BF16, rows, n, k, a[i], w[i], alone[i], workspace=scratch[0])
    torch.cuda.synchronize()
    for _ in range(20):
        for i in range(2):
            R.linear(R.BF16, R.BF16, rows, n, k, a[i], w[i], both[i], workspace=scratch[i], stream=streams[i])
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(alone, both))


def test_workspace_bytes():
    assert _workspace_bytes(100, 200, 4096) >= 2 * 100 * 200 * 4
    assert _workspace_bytes(2, 4096, 4096) == 0 and _workspace_bytes(4096, 4096, 4096) == 0 and _workspace_bytes(0, 8, 8) == 0
    assert _workspace_bytes(100, 200, 4096, groups=2, offsets=0x4000) >= 2 * 100 * 200 * 4


def _args(**change):
    a = R.linear_args(R.BF16, R.BF16, 4, 8, 16, 0x1000, 0x2000, 0x3000)
    for name, value in change.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("change,code", [
    (dict(in_type=R.F32), -2), (dict(out_type=R.F16), -2), (dict(activation=9), -1), (dict(activation=-1), -1), (dict(n=0), -1), (dict(k=0), -1), (dict(groups=0), -1),
    (dict(groups=2), -1), (dict(groups=2000, offsets=0x4000), -3), (dict(rows=2 ** 30 + 1), -3), (dict(n=2 ** 22, ldy=2 ** 22), -3), (dict(x=None), -1), (dict(w=None), -1), (dict(y=None), -1),
    (dict(ldx=15), -1), (dict(ldw=8), -1), (dict(ldy=7), -1), (dict(gate=0x5000, ldg=4), -1), (dict(c=0x5000, ldc=4), -1), (dict(z=0x5000, ldz=4), -1), (dict(ldx=2 ** 22), -1),
    (dict(x=0x1001), -4), (dict(y=0x3001), -4), (dict(bias=0x5001), -4), (dict(offsets=0x4002), -4), (dict(source=0x4001), -4), (dict(out_type=R.F32, y=0x3002), -4),
    (dict(groups=2, offsets=0x4000, w_stride=100), -1), (dict(groups=2, offsets=0x4000, w_stride=-200), -1), (dict(source=0x4000, x_rows=0), -3),
    (dict(source=0x4000, x_rows=2 ** 27), -3), (dict(rows=2 ** 30, n=2 ** 21, ldy=2 ** 21), -3),
])
def test_refusals(change, code):
    import ctypes

    assert R.lib().r355_linear(ctypes.byref(_args(**change)), None) == code
    assert R.lib().r355_last_error()


def test_no_rows_is_nothing_to_do():
    import ctypes

    assert R.lib().r355_linear(ctypes.byref(_args(rows=0, x=None, y=None)), None) == 0
    assert R.lib().r355_linear(None, None) == -1


def test_index_arrays_are_checked():
    import torch

    for kw in (dict(offsets=torch.zeros(2, dtype=torch.int64)), dict(offsets=torch.zeros(1, dtype=torch.int32)), dict(source=torch.zeros(4, dtype=torch.float32)),
               dict(source=torch.zeros(4, dtype=torch.int32))):
        with pytest.raises(ValueError):
            R.linear(R.BF16, R.BF16, 4, 8, 16, 0x1000, 0x2000, 0x3000, **kw)
