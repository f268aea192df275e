"""Products with 4-bit weights: what a token gives does not depend on the tokens beside it, nor on how many there are while the same tile is taken."""
import numpy as np
import pytest

import rocwmma_amd as R


@pytest.mark.gpu
@pytest.mark.parametrize("counts,n", [((5, 9, 16), 200), ((17, 24, 32), 200), ((98, 111, 128), 24590)])
def test_w4_same_bits_beside_other_tokens(counts, n):
    import torch

    k, group = 1032, 64
    g = torch.Generator(device="cuda").manual_seed(n)
    rows = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device="cuda", generator=g)
    packed = torch.empty(R.w4_packed_bytes(n, k), dtype=torch.uint8, device="cuda")
    R.w4_pack(rows, n, k, packed)
    scales = torch.rand(-(-k // group), n, device="cuda", generator=g).half()
    first = torch.randn(counts[0], k, device="cuda", generator=g).half()
    want = None
    for tokens in counts:
        x = torch.randn(tokens, k, device="cuda", generator=g).half()  # (others each time)
        x[: counts[0]] = first
        y = torch.empty(tokens, n, dtype=torch.float32, device="cuda")
        R.w4_matmul(R.F16, R.F32, tokens, n, k, group, x, packed, scales, y)
        got = y[: counts[0]].cpu().numpy()
        assert want is None or np.array_equal(got, want)
        want = got
