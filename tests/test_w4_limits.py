"""Products with 4-bit weights at the ends of what their arguments may be (bounds: tests/test_w4.py)."""
import pytest

from test_w4 import _case


@pytest.mark.gpu
@pytest.mark.parametrize("group", [1 << 31, 2 ** 32 - 128])
@pytest.mark.parametrize("tokens,n", [(1, 40), (20, 24590), (97, 24590)])
def test_w4_one_group_however_long(group, tokens, n):
    """A group far longer than k: k plus its length passes 32 bits."""
    _case("f16", "f32", tokens, n, 1032, group, zeros=True, seed=n)
    _case("bf16", "bf16", tokens, n, 129, group, seed=tokens)
