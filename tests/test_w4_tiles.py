"""Products with 4-bit weights at sizes for which each of the tiles is taken, none of them whole at the end of the rows, the tokens or k (bounds: tests/test_w4.py)."""
import pytest

from test_w4 import _case

# (tokens, rows): one to four blocks of 16 rows with up to 16 and up to 32 tokens, then 128 x 32, 64 x 64, 128 x 64, 128 x 128 and 256 x 128
SIZES = [(3, 100), (2, 4100), (3, 8200), (7, 12300), (4099, 15), (81, 2699), (24, 8201), (24, 12299), (20, 24590), (161, 5390), (40, 24590), (97, 24590), (193, 24590)]


@pytest.mark.gpu
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("tokens,n", SIZES)
def test_w4_every_tile(tokens, n, group):
    _case("f16", "f16", tokens, n, 1032, group, zeros=group == 64, seed=n)
    _case("bf16", "f32", tokens, n, 904, group, zeros=group != 64, alpha=0.75, beta=0.5, seed=tokens)
