"""The gradients of a layer's products against 64 bits (linearlib.py has the bounds) and against differences of the forward call."""
import pytest

import rocwmma_amd as R


def _run(*args, **kw):
    import linearlib

    return linearlib.run_backward(*args, **kw)


def _offsets(sizes):
    at = [0]
    for s in sizes:
        at.append(at[-1] + s)
    return at


def _scratch(n=1 << 22):
    import torch

    return torch.full((n,), 0xFF, dtype=torch.uint8, device="cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("rows,n,k", [(1, 8, 8), (3, 40, 136), (17, 64, 72), (64, 64, 128), (65, 72, 1000), (130, 264, 392), (1001, 136, 200)])
def test_sizes(dtype, rows, n, k):
    _run(dtype, dtype, rows, n, k, act="silu", gate=True, workspace=_scratch(), seed=rows)
    _run(dtype, "f32", rows, n, k, seed=rows + 1)


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("n", [48, 45])
def test_activations(act, gate, n):
    _run("bf16", "bf16", 150, n, 128, act=act, gate=gate, workspace=_scratch())
    _run("f16", "f32", 150, n, 128, act=act, gate=gate, accumulate=True)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 8, 63, 64, 65, 128, 129, 200, 1000])
def test_lengths_of_the_sum_over_rows(rows):
    _run("bf16", "f32", rows, 72, 136)
    _run("f16", "f16", rows, 72, 136, groups=3, offsets=_offsets([rows // 3, 0, rows - rows // 3]))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n,k", [(500, 4096, 3584), (3000, 72, 4200), (1500, 2048, 1024), (4000, 3500, 200)])
def test_many_tiles(rows, n, k):
    _run("bf16", "bf16", rows, n, k, act="gelu_tanh", workspace=_scratch(1 << 26))
    _run("f16", "f32", rows, n - n % 8, k, accumulate=True, workspace=_scratch(1 << 26))


@pytest.mark.gpu
@pytest.mark.parametrize("sizes", [[0, 5, 0, 0, 40], [1] * 70, [300, 1, 0, 64], [0, 0, 0], [513, 1700, 0, 900], [0] * 200 + [7] * 9])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_groups(dtype, sizes):
    rows = sum(sizes) or 4
    _run(dtype, dtype, rows, 136 if len(sizes) < 100 else 24, 64, act="silu", gate=True, groups=len(sizes), offsets=_offsets(sizes), workspace=_scratch())
    _run(dtype, "f32", rows, 40, 72, groups=len(sizes), offsets=_offsets(sizes), accumulate=True)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [64, 200, 328])
def test_groups_on_large_tiles(n):
    """Last tiles of 1 to 255 rows beside whole ones"""
    sizes = [2300, 1, 64, 0, 65, 128, 129, 192, 193, 255, 256, 300, 100, 1500]
    _run("bf16", "bf16", sum(sizes), n, 4000, act="silu", groups=len(sizes), offsets=_offsets(sizes), want=("dx",))
    _run("f16", "f32", sum(sizes), n, 3000, groups=len(sizes), offsets=_offsets(sizes), workspace=_scratch())


@pytest.mark.gpu
def test_groups_of_some_rows():
    _run("bf16", "bf16", 500, 72, 64, act="relu", groups=3, offsets=[17, 100, 100, 450])


@pytest.mark.gpu
@pytest.mark.parametrize("pad,offset", [(8, 0), (1, 0), (0, 1), (5, 3)])
@pytest.mark.parametrize("rows,n,k", [(70, 48, 72), (33, 45, 67)])
def test_strides_and_any_alignment(pad, offset, rows, n, k):
    _run("bf16", "bf16", rows, n, k, act="gelu", gate=True, pad=pad, offset=offset, workspace=_scratch())
    _run("f16", "f32", rows, n, k, accumulate=True, pad=pad, offset=offset, groups=2, offsets=[0, 20, rows])


@pytest.mark.gpu
@pytest.mark.parametrize("want", [("dx",), ("dw",), ("dbias",), ("dx", "dbias"), ()])
def test_parts_of_the_gradient(want):
    _run("bf16", "bf16", 100, 64, 72, act="silu", want=want)
    if want:
        _run("bf16", "bf16", 100, 64, 72, want=want)


@pytest.mark.gpu
@pytest.mark.parametrize("grad", ["bf16", "f32"])
@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("rows,n,k,sizes,pad", [(4096, 72, 136, None, 0), (90, 4096, 72, None, 0), (3000, 100, 45, None, 1), (4000, 40, 72, [3000, 0, 1000], 0)])
def test_sums_split_over_workgroups(rows, n, k, sizes, pad, accumulate, grad):
    """With a workspace and few tiles, dx and dw: whole, for fewer shares, and too small for any"""
    groups, offsets = (1, None) if sizes is None else (len(sizes), _offsets(sizes))
    a = R.linear_backward_args(R.BF16, R.F32, rows, n, k, 0x1000, 0x2000, 0x3000, dx=0x4000, dw=0x5000, groups=groups, offsets=None if sizes is None else 0x6000)
    need = R.linear_backward_workspace_bytes(a)
    assert need > 0
    for size in (need, need // 2 // 16 * 16, 16):
        _run("bf16", grad, rows, n, k, act="gelu", groups=groups, offsets=offsets, accumulate=accumulate, pad=pad, workspace=_scratch(size))


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["none", "silu"])
@pytest.mark.parametrize("rows,n,k,sizes,pad,offset", [(1100, 1003, 520, None, 0, 0), (900, 1000, 603, None, 0, 1), (1000, 700, 999, [500, 0, 300, 150], 1, 0), (1200, 1001, 512, [200, 1000], 7, 1)])
def test_operands_laid_out_anew(rows, n, k, sizes, pad, offset, act):
    """Rows off 16-byte boundaries, or that end inside 16 bytes, with a workspace that holds them evenly; NaN behind every row and beside the operands"""
    groups, offsets = (1, None) if sizes is None else (len(sizes), _offsets(sizes))
    a = R.linear_backward_args(R.BF16, R.BF16, rows, n, k, 0x1000 + 2 * offset, 0x2000 + 2 * offset, 0x3000 + 2 * offset, dx=0x4000, dw=0x5000, groups=groups,
                               offsets=None if sizes is None else 0x6000, lddy=n + pad, ldx=k + pad, ldw=k + pad)
    need, eights = R.linear_backward_workspace_bytes(a), (n + 7) // 8 * 8
    assert need >= 2 * eights * (groups * k + rows)
    for size in (need, need // 3 // 16 * 16):
        _run("bf16", "bf16", rows, n, k, act=act, groups=groups, offsets=offsets, pad=pad, offset=offset, workspace=_scratch(size))
    _run("f16", "f32", rows, n, k, act=act, groups=groups, offsets=offsets, pad=pad, offset=offset, accumulate=True, workspace=_scratch(need), want=("dw",))
    _run("f16", "f16", rows, n, k, act=act, groups=groups, offsets=offsets, pad=pad, offset=offset, workspace=_scratch(need), want=("dx", "dbias"))


@pytest.mark.gpu
@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("act", ["none", "silu"])
@pytest.mark.parametrize("k", [72, 45])
def test_no_rows(accumulate, act, k):
    """The weights' and the bias's gradient are zeros, or what was there"""
    import torch

    dw, db = torch.full((40, k), 3.0, device="cuda"), torch.full((40,), 5.0, device="cuda")
    R.linear_backward(R.F16, R.F32, 0, 40, k, None, None, None, dx=0x1000, dw=dw, dbias=db, activation=R.ACT_SILU if act == "silu" else R.ACT_NONE, dz=0x1000, accumulate=accumulate,
                      workspace=_scratch())
    assert (dw == (3.0 if accumulate else 0.0)).all() and (db == (5.0 if accumulate else 0.0)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [2, 70, 900])
def test_one_group_with_offsets(rows):
    _run("bf16", "f32", rows, 72, 136, act="relu", gate=True, groups=1, offsets=[rows // 3, rows - 1])


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n,k", [(4099, 1544, 4096)])
def test_rows_past_whole_rounds_of_tiles(rows, n, k):
    _run("bf16", "bf16", rows, n, k, act="silu", gate=True, pad=8, workspace=_scratch(1 << 24))


@pytest.mark.gpu
def test_infinities_and_nan_stay_in_their_rows_and_columns():
    import torch

    rows, n, k = 200, 72, 136
    x, w, dy = torch.randn(rows, k, device="cuda").bfloat16(), torch.randn(n, k, device="cuda").bfloat16(), torch.randn(rows, n, device="cuda").bfloat16()
    x[3, 5], w[7, 9], dy[rows - 1, n - 1] = float("nan"), float("inf"), float("nan")
    dx, dw, db = torch.empty_like(x), torch.empty(n, k, device="cuda"), torch.empty(n, device="cuda")
    R.linear_backward(R.BF16, R.F32, rows, n, k, dy, x, w, dx=dx, dw=dw, dbias=db)
    bad = torch.zeros(rows, k, dtype=torch.bool, device="cuda")
    bad[-1], bad[:, 9] = True, True
    assert torch.equal(~torch.isfinite(dx), bad)
    bad = torch.zeros(n, k, dtype=torch.bool, device="cuda")
    bad[-1], bad[:, 5] = True, True
    assert torch.equal(~torch.isfinite(dw), bad)
    assert torch.equal(~torch.isfinite(db), torch.arange(n, device="cuda") == n - 1)


@pytest.mark.gpu
def test_graph():
    """Recorded on a stream of its own with other values and offsets at every replay, the program's eager work between them"""
    import torch

    rows, n, k, groups = 300, 72, 136, 3
    make = lambda *shape: torch.randn(*shape, device="cuda").bfloat16()  # noqa: E731
    x, w, dy, z, gate = make(rows, k), make(groups, n, k), make(rows, n), make(rows, n), make(rows, n)
    offsets = torch.zeros(groups + 1, dtype=torch.int32, device="cuda")
    scratch = [_scratch() for _ in range(2)]

    def results():
        return [torch.zeros(rows, k, dtype=torch.bfloat16, device="cuda"), torch.zeros(groups, n, k, device="cuda"), torch.zeros(groups, n, device="cuda"),
                torch.zeros_like(z), torch.zeros_like(z)]

    def call(to, workspace, stream):
        dx, dw, db, dg, dz = to
        R.linear_backward(R.BF16, R.F32, rows, n, k, dy, x, w, dx=dx, dw=dw, dbias=db, z=z, activation=R.ACT_SILU, gate=gate, dgate=dg, dz=dz, accumulate=True, groups=groups,
                          offsets=offsets, workspace=workspace, stream=stream)

    recorded, eager = results(), results()
    call(eager, scratch[1], None)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        call(recorded, scratch[0], torch.cuda.current_stream())
    for at in ([0, 100, 100, 300], [0, 0, 0, 300], [10, 20, 250, 260]):
        offsets.copy_(torch.tensor(at, dtype=torch.int32))
        dy.copy_(torch.randn(rows, n, device="cuda"))
        for a, b in zip(recorded, eager):
            a.zero_(), b.zero_()
        graph.replay()
        call(eager, scratch[1], None)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(recorded, eager)) and eager[1].abs().sum() > 0


@pytest.mark.gpu
@pytest.mark.parametrize("over", ["dy", "z"])
def test_dz_in_the_place_of_what_it_is_made_of(over):
    import torch

    rows, n, k = 100, 64, 72
    make = lambda *shape: torch.randn(*shape, device="cuda").half()  # noqa: E731
    x, w, dy, z, gate = make(rows, k), make(n, k), make(rows, n), make(rows, n), make(rows, n)
    results = []
    for dz in (torch.empty_like(dy), dy.clone() if over == "dy" else z.clone()):
        dx, dw, db, dg = torch.empty_like(x), torch.empty_like(w), torch.empty(n, device="cuda"), torch.empty_like(dy)
        here = dict(dy=dz if over == "dy" and results else dy, z=dz if over == "z" and results else z)
        R.linear_backward(R.F16, R.F16, rows, n, k, here["dy"], x, w, dx=dx, dw=dw, dbias=db, z=here["z"], activation=R.ACT_SILU, gate=gate, dgate=dg, dz=dz)
        results.append((dx, dw, db, dg, dz))
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.gpu
def test_the_result_does_not_depend_on_scheduling_and_little_on_the_workspace():
    import torch

    a, b = (_run("bf16", "f32", 3000, 264, 72, act="silu", gate=True, workspace=_scratch()) for _ in range(2))
    assert all(torch.equal(a[name], b[name]) for name in a)
    _run("bf16", "f32", 3000, 264, 72, act="silu", gate=True)
    _run("bf16", "f32", 3000, 264, 72, act="silu", gate=True, workspace=_scratch(264 * 4 * 3))


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "gelu_tanh", "silu"])
def test_against_differences(act):
    """dL of L = sum y r for steps of x, w, bias and gate along random directions, of calls in f32 results.  A central difference is off by
    h^2 / 6 times the third derivative along the step, here |act'''| <= 1 times the cube of the argument's change; roundings of y in f32 and of the operands (the steps are made of
    16-bit values) by 2^-24 sum |y r| / h.  dz is rounded to 16 bits."""
    import torch

    rows, n, k, h = 24, 32, 64, 2.0 ** -5
    g = torch.Generator(device="cuda").manual_seed(3)
    normal = lambda *shape: (torch.randn(*shape, generator=g, device="cuda") * 64).round() / 64  # noqa: E731
    quarter = lambda *shape: torch.randint(-1, 2, shape, generator=g, device="cuda").float()  # noqa: E731
    t = torch.float16
    x, w, b, gate, r = normal(rows, k), normal(n, k) / 8, normal(n), normal(rows, n), normal(rows, n)
    ax = {"relu": R.ACT_RELU, "gelu": R.ACT_GELU, "gelu_tanh": R.ACT_GELU_TANH, "silu": R.ACT_SILU, "none": R.ACT_NONE}[act]

    def loss(x, w, b, gate):
        y = torch.empty(rows, n, device="cuda")
        R.linear(R.F16, R.F32, rows, n, k, x.to(t), w.to(t), y, bias=b.to(t), activation=ax, gate=gate.to(t))
        return (y.double() * r.double()).sum().item(), (y.double() * r.double()).abs().sum().item()

    z = torch.empty(rows, n, dtype=t, device="cuda")
    y = torch.empty(rows, n, device="cuda")
    R.linear(R.F16, R.F32, rows, n, k, x.to(t), w.to(t), y, bias=b.to(t), z=z)
    dx, dw, db, dgate, dz = torch.empty(rows, k, dtype=t, device="cuda"), torch.empty(n, k, device="cuda"), torch.empty(n, device="cuda"), torch.empty_like(z), torch.empty_like(z)
    R.linear_backward(R.F16, R.F32, rows, n, k, r.to(t), x.to(t), w.to(t), dx=dx, dw=dw, dbias=db, z=z, activation=ax, gate=gate.to(t), dgate=dgate, dz=dz)
    for name, at, grad in (("x", x, dx), ("w", w, dw), ("b", b, db), ("gate", gate, dgate)):
        step = quarter(*at.shape)
        if name == "w":
            step = step / 8
        values = dict(x=x, w=w, b=b, gate=gate)
        up, size = loss(**{**values, name: at + h * step})
        down, _ = loss(**{**values, name: at - h * step})
        analytic = (grad.double() * step.double()).sum().item()
        spread = (grad.double() * step.double()).abs().sum().item()
        # curvature, as above (six times as much); relu has a kink: a result whose argument passes zero on the way is off by half of its change
        dzs = (x.double() @ step.double().t()) if name == "w" else (step.double() @ w.double().t()) if name == "x" else step.double().expand(rows, n) if name == "b" else torch.zeros(rows, n, device="cuda").double()
        rg = (r * gate).double().abs()
        curved = 0.0 if act == "none" else (rg * dzs.abs() * (z.double().abs() <= h * dzs.abs() + 2.0 ** -8)).sum().item() if act == "relu" else (rg * dzs.abs() ** 3).sum().item() * h * h
        bound = curved + 2.0 ** -22 * size / h + 2.0 ** -9 * spread + 2.0 ** -9 * (rg * dzs.abs() * (1 + z.double().abs())).sum().item()
        assert abs((up - down) / (2 * h) - analytic) <= bound, (name, (up - down) / (2 * h), analytic, bound)


def _args(**change):
    a = R.linear_backward_args(R.BF16, R.BF16, 4, 8, 16, 0x1000, 0x2000, 0x3000, dx=0x4000, dw=0x5000)
    for name, value in change.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("change,code", [
    (dict(in_type=R.F32), -2), (dict(grad_type=R.F16), -2), (dict(activation=9), -1), (dict(n=0), -1), (dict(k=0), -1), (dict(groups=0), -1), (dict(groups=2), -1),
    (dict(groups=2000, offsets=0x6000), -3), (dict(dy=None), -1), (dict(w=None), -1), (dict(x=None), -1), (dict(activation=R.ACT_SILU, dz=0x7000), -1),
    (dict(activation=R.ACT_SILU, z=0x7000), -1), (dict(gate=0x7000), -1), (dict(dgate=0x7000), -1), (dict(dgate=0x7000, gate=0x8000, dz=0x9000), -1), (dict(lddy=7), -1), (dict(ldx=15), -1),
    (dict(ldw=15), -1), (dict(lddx=15), -1), (dict(lddw=15), -1), (dict(dy=0x1001), -4), (dict(dx=0x4001), -4), (dict(dbias=0x6002), -4), (dict(grad_type=R.F32, dw=0x5002), -4),
    (dict(groups=2, offsets=0x6000, w_stride=100), -1), (dict(groups=2, offsets=0x6000, dw_stride=100), -1), (dict(rows=2 ** 30 + 1), -3),
])
def test_refusals(change, code):
    import ctypes

    assert R.lib().r355_linear_backward(ctypes.byref(_args(**change)), None) == code
    assert R.lib().r355_last_error()


def test_workspace_bytes():
    a = R.linear_backward_args(R.BF16, R.BF16, 4000, 264, 72, 0x1000, 0x2000, 0x3000, dbias=0x4000)
    assert R.linear_backward_workspace_bytes(a) % (264 * 4) == 0 and R.linear_backward_workspace_bytes(a) > 0
    a.dbias, a.n = None, 0
    assert R.linear_backward_workspace_bytes(a) == 0
