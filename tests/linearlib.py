"""A layer's products and their gradients in 64 bits, with the bounds that rounding leaves, for the tests of linear() and linear_backward().

Bounds, eps = 2^-24.  A sum of k products in f32, in any order: (k + 8) eps sum |x w|.  The bias adds one rounding of the result.  Activations: e^-z as 2^(z log2 e) is off by
(|z| + 2) eps relative, so sigma by (|u| + 6) eps at most (u its argument, whose own roundings are 4 eps |u|); erf by 2 eps absolute.  So act(z) is off by
(|act| (5 |u| + 8) + 2 |z|) eps, its slope by (1 + |z|) (10 |u| + 16) eps, and both pass an error of z on with a factor of at most 1.13 (the slope: 1)."""
import math

import torch

import rocwmma_amd as R

EPS = 2.0 ** -24
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: EPS}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -126}  # half of the smallest steps (f32: what is flushed)
TORCH = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
TYPES = {"f16": R.F16, "bf16": R.BF16, "f32": R.F32}
ACTS = {"none": R.ACT_NONE, "relu": R.ACT_RELU, "gelu": R.ACT_GELU, "gelu_tanh": R.ACT_GELU_TANH, "silu": R.ACT_SILU}


def act64(z, act):
    """Value, slope, and the argument of the sigmoid that bounds their errors"""
    one = torch.ones_like(z)
    if act == "none":
        return z, one, 0 * z
    if act == "relu":
        return z.clamp(min=0), (z > 0).double(), 0 * z
    if act == "gelu":
        cdf = torch.special.ndtr(z)
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi), z * z / 2
    u = z if act == "silu" else math.sqrt(8 / math.pi) * (z + 0.044715 * z ** 3)
    du = one if act == "silu" else math.sqrt(8 / math.pi) * (1 + 3 * 0.044715 * z * z)
    s = torch.sigmoid(u)
    return z * s, s + z * s * (1 - s) * du, u.abs()


def act_bound(z, act):
    if act in ("none", "relu"):
        return 0 * z
    value, _, u = act64(z, act)
    return (value.abs() * (5 * u + 8) + 2 * z.abs()) * EPS


def slope_bound(z, act):
    if act in ("none", "relu"):
        return 0 * z
    return (1 + z.abs()) * (10 * act64(z, act)[2] + 16) * EPS


def rounded(want, err, dtype):
    """Bound of the error of a value that is `want` within `err` before it is rounded to a type"""
    return err + HALF[dtype] * (want.abs() + err) + TINY[dtype]


def matrix(values, dtype, ld=None, offset=0):
    """(the tensor to hand over, its view of the values): rows `ld` elements apart that begin `offset` elements into their buffer, NaN around them"""
    rows, cols = values.shape[-2:]
    groups = values.shape[0] if values.dim() == 3 else 1
    ld = ld or cols
    buffer = torch.full((offset + groups * rows * ld + 8,), float("nan"), dtype=dtype, device="cuda")
    view = buffer[offset: offset + groups * rows * ld].view(groups, rows, ld)
    view[:, :, :cols] = values.reshape(groups, rows, cols).to(dtype)
    return buffer[offset:], view


def span(groups, rows, offsets):
    """First row and the row past the last of every group, cut off at the rows"""
    if offsets is None:
        return [(0, rows)]
    at = [min(max(o, 0), rows) for o in offsets]
    return [(a, max(a, b)) for a, b in zip(at[:-1], at[1:])]


def run_linear(dtype, out, rows, n, k, act="none", bias=False, gate=False, c=False, keep=False, groups=1, offsets=None, source=None, x_rows=None, pad=(0, 0, 0, 0, 0, 0), offset=0,
               in_place=False, workspace=None, seed=0, scale=1.0, stream=None):
    """linear() against 64 bits.  pad: what is added to the leading dimensions of x, w, gate, c, y, z; offset: elements that every operand is off its buffer's start.  Returns y, z."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    t, o = TORCH[dtype], TORCH[out]
    x_rows = rows if x_rows is None else x_rows
    xv, wv = (normal(x_rows, k) * scale).to(t), (normal(groups, n, k) / math.sqrt(k)).to(t)
    bv, gv, cv = normal(groups, n).to(t), normal(rows, n).to(t), normal(rows, n).to(o)
    x, w = matrix(xv, t, k + pad[0], offset)[0], matrix(wv, t, k + pad[1], offset)[0]
    gt, ct = matrix(gv, t, n + pad[2], offset)[0], matrix(cv, o, n + pad[3], offset)[0]
    y, yview = matrix(torch.full((rows, n), float("nan"), device="cuda"), o, n + pad[4], offset)
    if in_place:
        y, yview = matrix(cv, o, n + pad[4], offset)
        ct = y
    z, zview = matrix(torch.full((rows, n), float("nan"), device="cuda"), t, n + pad[5], offset)
    bt = matrix(bv, t, None, offset)[0]
    off = None if offsets is None else torch.tensor(offsets, dtype=torch.int32).cuda()
    src = None if source is None else torch.tensor(source, dtype=torch.int32).cuda()
    R.linear(TYPES[dtype], TYPES[out], rows, n, k, x, w, y, bias=bt if bias else None, activation=ACTS[act], gate=gt if gate else None, c=ct if c else None, z=z if keep else None,
             groups=groups, offsets=off, source=src, x_rows=x_rows, ldx=k + pad[0], ldw=k + pad[1], ldg=n + pad[2], ldc=n + (pad[4] if in_place else pad[3]), ldy=n + pad[4],
             ldz=n + pad[5], workspace=workspace, stream=stream)
    torch.cuda.synchronize()
    got, got_z = yview[0].double(), zview[0].double()
    assert torch.isnan(got[:, n:]).all() and torch.isnan(got_z[:, n:]).all()  # nothing is written between the rows
    written = torch.zeros(rows, dtype=torch.bool, device="cuda")
    for e, (a, b) in enumerate(span(groups, rows, offsets)):
        if a == b:
            continue
        written[a:b] = True
        xs = xv[a:b].double()
        if source is not None:
            s = torch.tensor(source[a:b])
            good = (s >= 0) & (s < x_rows)
            xs = torch.where(good[:, None].cuda(), xv.double()[torch.where(good, s, 0).cuda()], 0.0)
        zs, err = xs @ wv[e].double().t(), (k + 8) * EPS * (xs.abs() @ wv[e].double().abs().t())
        if bias:
            zs = zs + bv[e].double()
            err = err + EPS * (zs.abs() + err)
        value, _, _ = act64(zs, act)
        want, far = value, 1.13 * err + act_bound(zs, act)
        if gate:
            want, far = want * gv[a:b].double(), far * gv[a:b].double().abs() + EPS * (want * gv[a:b].double()).abs()
        if c:
            want = want + cv[a:b].double()
            far = far + EPS * (want.abs() + far)
        far = rounded(want, far, o)
        off_by = (got[a:b, :n] - want).abs()
        assert (off_by <= far).all(), (e, (off_by / far).max().item())
        if keep:
            far = rounded(zs, err, t)
            assert ((got_z[a:b, :n] - zs).abs() <= far).all(), ((got_z[a:b, :n] - zs).abs() / far).max().item()
    untouched = cv.double() if in_place else torch.full_like(got[:, :n], float("nan"))
    assert torch.equal(torch.nan_to_num(got[~written, :n], 7.0), torch.nan_to_num(untouched[~written], 7.0))  # rows of no group
    if not keep:
        assert torch.isnan(got_z).all()
    return y, z


def run_backward(dtype, grad, rows, n, k, act="none", gate=False, groups=1, offsets=None, accumulate=False, want=("dx", "dw", "dbias"), pad=0, offset=0, workspace=None, seed=0,
                 stream=None):
    """linear_backward() against 64 bits.  pad, offset: of every matrix.  Returns what was written."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    t, o = TORCH[dtype], TORCH[grad]
    xv, wv, dyv, zv, gv = normal(rows, k).to(t), (normal(groups, n, k) / math.sqrt(n)).to(t), normal(rows, n).to(t), (normal(rows, n) * 1.5).to(t), normal(rows, n).to(t)
    dwv, dbv = normal(groups, n, k).to(o), normal(groups, n)
    nan = lambda *shape: torch.full(shape, float("nan"), device="cuda")  # noqa: E731
    x, w, dy, z, gt = (matrix(v, t, v.shape[-1] + pad, offset)[0] for v in (xv, wv, dyv, zv, gv))
    dz, dzview = matrix(nan(rows, n), t, n + pad, offset)
    dgate, dgview = matrix(nan(rows, n), t, n + pad, offset)
    dx, dxview = matrix(nan(rows, k), t, k + pad, offset)
    dw, dwview = matrix(dwv if accumulate else nan(groups, n, k), o, k + pad, offset)
    db = dbv.clone() if accumulate else nan(groups, n)
    off = None if offsets is None else torch.tensor(offsets, dtype=torch.int32).cuda()
    element = act != "none" or gate
    dgate_wanted = gate and act != "none"
    R.linear_backward(TYPES[dtype], TYPES[grad], rows, n, k, dy, x, w, dx=dx if "dx" in want else None, dw=dw if "dw" in want else None, dbias=db if "dbias" in want else None,
                      z=z if act != "none" else None, activation=ACTS[act], gate=gt if gate else None, dgate=dgate if dgate_wanted else None, dz=dz if element else None,
                      accumulate=accumulate, groups=groups, offsets=off, lddy=n + pad, ldx=k + pad, ldw=k + pad, ldz=n + pad, ldg=n + pad, lddz=n + pad, lddg=n + pad, lddx=k + pad,
                      lddw=k + pad, workspace=workspace, stream=stream)
    torch.cuda.synchronize()
    for view, cols in ((dzview, n), (dgview, n), (dxview, k), (dwview, k)):
        assert torch.isnan(view[:, :, cols:]).all()
    written = torch.zeros(rows, dtype=torch.bool, device="cuda")

    def near(got, want_, far):
        assert ((got.double() - want_).abs() <= far).all(), ((got.double() - want_).abs() / far).max().item()

    for e, (a, b) in enumerate(span(groups, rows, offsets)):
        written[a:b] = True
        dys, xs, ws = dyv[a:b].double(), xv[a:b].double(), wv[e].double()
        value, slope, _ = act64(zv[a:b].double(), act)
        gs = gv[a:b].double() if gate else torch.ones_like(dys)
        exact, err = dys * gs * slope, (dys * gs).abs() * (slope_bound(zv[a:b].double(), act) + 2 * EPS * slope.abs())
        off_by = rounded(exact, err, t) if element else 0 * exact  # of the dz that the products take
        if element:
            near(dzview[0, a:b, :n], exact, off_by)
        if dgate_wanted:
            near(dgview[0, a:b, :n], dys * value, rounded(dys * value, dys.abs() * act_bound(zv[a:b].double(), act) + EPS * (dys * value).abs(), t))
        if "dx" in want:
            want_ = exact @ ws
            near(dxview[0, a:b, :k], want_, rounded(want_, off_by @ ws.abs() + (n + 8) * EPS * ((exact.abs() + off_by) @ ws.abs()), t))
        if "dw" in want:
            want_ = exact.t() @ xs
            far = off_by.t() @ xs.abs() + (b - a + 8) * EPS * ((exact.abs() + off_by).t() @ xs.abs())
            if accumulate:
                want_ = want_ + dwv[e].double()
                far = far + EPS * (want_.abs() + far)
            near(dwview[e, :, :k], want_, rounded(want_, far, o))
        if "dbias" in want:
            want_ = exact.sum(0)
            far = err.sum(0) + (b - a + 8) * EPS * (exact.abs() + err).sum(0)
            if accumulate:
                want_ = want_ + dbv[e].double()
                far = far + EPS * (want_.abs() + far)
            near(db[e], want_, far + TINY[torch.float32])
    for view, cols in ((dxview, k), (dzview, n), (dgview, n)):
        assert torch.isnan(view[0, ~written]).all()
    return {"dx": dxview[0, :, :k], "dw": dwview[:, :, :k], "dbias": db, "dgate": dgview[0, :, :n]}
