"""Products with 4-bit weights and group scales against the formula in 64 bits.

Bound of the error: the kernel sums x (16 + q) and x over a stretch of min(group, 128) k in f32, takes their difference times the scale, and
adds up one such term per 128 k (or group) and per wave.  Each of these additions rounds by at most 2^-24 of what has been summed, so the
error is at most (stretch + stretches + 16) 2^-24 of the sum of |x| (16 + q + 16 + z) |s|, and the result is rounded once to its type."""
import numpy as np
import pytest

import rocwmma_amd as R

HALF_ULP = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}
TYPES = {"f16": R.F16, "bf16": R.BF16, "f32": R.F32}


def _torch_type(name):
    import torch

    return {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}[name]


def _case(dtype, out, tokens, n, k, group, zeros=False, alpha=1.0, beta=0.0, ldx=None, ldc=None, ldy=None, offset=0, seed=0, in_place=False):
    """Runs one product; x starts `offset` elements into its buffer and what lies between its rows, and past them, is NaN."""
    import torch

    rng = np.random.RandomState(seed)
    ldx, ldc, ldy = ldx or k, ldc or n, ldy or n
    if in_place:
        ldc = ldy
    groups = -(-k // group)
    q = rng.randint(0, 16, (n, k)).astype(np.uint8)
    z = rng.randint(0, 16, (groups, n)).astype(np.uint8) if zeros else np.full((groups, n), 8, np.uint8)
    padded = np.concatenate([q, np.full((n, k % 2), 9, np.uint8)], 1)
    rows = torch.from_numpy(padded[:, 0::2] | (padded[:, 1::2] << 4)).cuda()
    packed = torch.full((R.w4_packed_bytes(n, k),), 0xFF, dtype=torch.uint8, device="cuda")
    R.w4_pack(rows, n, k, packed)
    t, o = _torch_type(dtype), _torch_type(out)
    x = torch.from_numpy(rng.randn(tokens, k)).to(t)
    s = torch.from_numpy((0.25 + rng.rand(groups, n)) / np.sqrt(k)).to(t)
    c = torch.from_numpy(rng.randn(tokens, n)).to(o)
    xbuf = torch.full((offset + tokens * ldx + 8,), float("nan"), dtype=t, device="cuda")
    xbuf[offset: offset + tokens * ldx].view(tokens, ldx)[:, :k] = x.cuda()
    cbuf = torch.full((tokens, ldc), float("nan"), dtype=o, device="cuda")
    cbuf[:, :n] = c.cuda()
    y = cbuf if in_place else torch.full((tokens, ldy), float("nan"), dtype=o, device="cuda")
    args = dict(zeros=torch.from_numpy(z).cuda() if zeros else None, c=cbuf if beta else None, alpha=alpha, beta=beta, ldx=ldx, ldc=ldc, ldy=ldy)
    R.w4_matmul(TYPES[dtype], TYPES[out], tokens, n, k, group, xbuf[offset:], packed, s.cuda(), y, **args)
    got = y.double().cpu().numpy()
    assert np.all(np.isnan(got[:, n:]))  # nothing is written between the rows
    of = np.arange(k) // group
    xd, sd, qd, zd = x.double().numpy(), s.double().numpy().T[:, of], q.astype(np.float64), z.astype(np.float64).T[:, of]
    want = alpha * (xd @ ((qd - zd) * sd).T) + beta * c.double().numpy()
    stretch = min(group, 128)
    spread = np.abs(xd) @ ((32.0 + qd + zd) * np.abs(sd)).T
    bound = abs(alpha) * (stretch + k / stretch + 16) * 2.0 ** -24 * spread + (HALF_ULP[out] + 2.0 ** -22) * np.abs(want) + 2.0 ** -23 * abs(beta) * np.abs(c.double().numpy()) + 1e-7
    assert np.all(np.abs(got[:, :n] - want) <= bound), np.max(np.abs(got[:, :n] - want) / bound)
    return y


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("group", [32, 64, 128, 256])
@pytest.mark.parametrize("tokens,n,k", [(1, 16, 128), (1, 1, 8), (3, 33, 264), (16, 70, 1000), (17, 260, 520), (65, 96, 2048), (130, 257, 392)])
def test_w4_vs_formula(dtype, group, tokens, n, k):
    _case(dtype, dtype, tokens, n, k, group, zeros=(n + group) % 3 == 0, seed=n + k)
    _case(dtype, "f32", tokens, n, k, group, zeros=True, alpha=-1.5, beta=0.5, seed=n + k + 1)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 2, 7, 16, 32, 33, 48, 64, 100, 256, 300])
def test_w4_tokens(tokens):
    _case("bf16", "bf16", tokens, 512, 1536, 128, zeros=True, beta=1.0, seed=tokens)
    _case("f16", "f32", tokens, 516, 1096, 64, seed=tokens)


@pytest.mark.gpu
@pytest.mark.parametrize("n,k", [(4096, 4096), (16, 32768), (20000, 256), (1024, 11008 + 8)])
def test_w4_shapes(n, k):
    _case("f16", "f16", 1, n, k, 128, seed=1)
    _case("bf16", "f32", 5, n, k, 32, zeros=True, seed=2)


@pytest.mark.gpu
@pytest.mark.parametrize("k", [1, 7, 31, 129, 1001])
def test_w4_k_off_the_vectors(k):
    """(k = 1001 with groups of 384 and of more than k as well)"""
    _case("f16", "f16", 3, 36, 8 * k, 384, zeros=True, seed=k)
    _case("bf16", "f32", 70, 36, 8 * k, 1 << 20, seed=k)
    _case("bf16", "bf16", 5, 40, k, 32, seed=k)
    _case("f16", "f32", 20, 41, k, 128, zeros=True, seed=k)


@pytest.mark.gpu
def test_w4_strides_and_alignment():
    _case("bf16", "bf16", 9, 64, 256, 64, ldx=264, ldc=68, ldy=72, beta=2.0)
    _case("bf16", "f32", 9, 64, 256, 64, ldx=257, ldc=65, ldy=67, beta=2.0)
    _case("f16", "f16", 30, 66, 256, 32, ldx=259, offset=1)
    _case("f16", "f16", 30, 64, 256, 32, offset=3)
    _case("bf16", "bf16", 12, 48, 384, 128, ldy=52, beta=1.0, in_place=True)


@pytest.mark.gpu
def test_w4_same_bits_again_and_with_other_tokens_beside():
    import torch

    a = _case("bf16", "f32", 24, 200, 2056, 64, zeros=True, seed=5)
    b = _case("bf16", "f32", 24, 200, 2056, 64, zeros=True, seed=5)
    assert torch.equal(a, b)


@pytest.mark.gpu
def test_w4_no_tokens_and_other_stream():
    import torch

    R.w4_matmul(R.F16, R.F16, 0, 16, 128, 128, None, None, None, None)
    n, k = 256, 1024
    rows = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device="cuda")
    packed = torch.empty(R.w4_packed_bytes(n, k), dtype=torch.uint8, device="cuda")
    R.w4_pack(rows, n, k, packed)
    x, s = torch.randn(2, k, device="cuda").half(), torch.rand(k // 128, n, device="cuda").half()
    y, z = torch.empty(2, n, dtype=torch.float32, device="cuda"), torch.empty(2, n, dtype=torch.float32, device="cuda")
    R.w4_matmul(R.F16, R.F32, 2, n, k, 128, x, packed, s, y)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    R.w4_matmul(R.F16, R.F32, 2, n, k, 128, x, packed, s, z, stream=side)
    side.synchronize()
    assert torch.equal(y, z)


def _refused(code, **change):
    a = dict(in_type=R.F16, out_type=R.F16, tokens=4, n=64, k=256, group=64, x=0x1000, w=0x2000, scales=0x3000, y=0x4000)
    a.update(change)
    with pytest.raises(R.R355Error) as e:
        R.w4_matmul(**a)
    assert e.value.code == code, str(e.value)


def test_w4_refusals():
    for name in ("x", "w", "scales", "y"):
        _refused(-1, **{name: None})
    _refused(-1, n=0)
    _refused(-1, k=0)
    _refused(-1, beta=1.0)
    _refused(-1, ldx=255)
    _refused(-1, ldy=63)
    _refused(-1, beta=1.0, c=0x5000, ldc=63)
    _refused(-2, in_type=R.F32)
    _refused(-2, out_type=R.BF16)
    _refused(-3, group=0)
    _refused(-3, group=96)
    _refused(-3, group=16)
    _refused(-3, n=(1 << 24) + 1)
    _refused(-3, tokens=(1 << 19) + 1)
    _refused(-3, k=(1 << 22) + 128)
    _refused(-3, n=1 << 24, tokens=1 << 10)
    _refused(-4, w=0x2008)
    _refused(-4, x=0x1001)
    _refused(-4, out_type=R.F32, y=0x4002)
    for bad, code in ((dict(q=None), -1), (dict(packed=None), -1), (dict(n=0), -1), (dict(ldq=3), -1), (dict(packed=0x1004), -4), (dict(n=(1 << 24) + 1), -3)):
        a = dict(q=0x1000, n=16, k=8, packed=0x2000)
        a.update(bad)
        with pytest.raises(R.R355Error) as e:
            R.w4_pack(**a)
        assert e.value.code == code
    assert R.w4_packed_bytes(1, 1) == 1024 and R.w4_packed_bytes(17, 129) == 4096
