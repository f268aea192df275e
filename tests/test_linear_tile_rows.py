"""Tiles of 192 rows: sizes of gradients for which the plan takes them for the weights' product, whose operands are not contiguous along the sum, against 64 bits (linearlib.py)."""
import pytest


def _offsets(sizes):
    at = [0]
    for s in sizes:
        at.append(at[-1] + s)
    return at


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,grad", [("bf16", "bf16"), ("f16", "f32")])
@pytest.mark.parametrize("rows,n,k,sizes", [
    (4096, 2880, 2880, None), (1024, 1536, 8192, None), (3339, 1664, 5048, None), (1000, 2872, 2888, None), (65, 1536, 8192, None),
    (8192, 1536, 4096, [2000, 3000, 192, 3000]), (8840, 536, 3552, [2210, 1, 4419, 2210]), (3994, 1624, 384, [500, 0, 1000, 7, 993, 64, 930, 500]),
])
def test_weights_gradient(dtype, grad, rows, n, k, sizes):
    import torch

    import linearlib

    groups, offsets = (1, None) if sizes is None else (len(sizes), _offsets(sizes))
    for accumulate, workspace in ((False, None), (True, torch.full((1 << 26,), 0xFF, dtype=torch.uint8, device="cuda"))):
        linearlib.run_backward(dtype, grad, rows, n, k, groups=groups, offsets=offsets, accumulate=accumulate, workspace=workspace, want=("dw", "dbias"))
