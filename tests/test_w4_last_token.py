"""Products with 4-bit weights on the ring of LDS buffers where the last tile holds a single token and the waves that share k run past its last block: what they load
there lies outside of x by every way of counting it (bounds: tests/test_w4.py)."""
import pytest

from test_w4 import _case

# (group, tokens, rows): tiles of 64 x 32 (groups of 32), 128 x 32 and 128 x 64
SIZES = [(32, 33, 6210), (32, 33, 12354), (64, 33, 12353), (128, 33, 12357), (64, 65, 13121), (128, 65, 13122)]


@pytest.mark.gpu
@pytest.mark.parametrize("k", [8, 264, 1032])
@pytest.mark.parametrize("group,tokens,n", SIZES)
def test_w4_one_token_in_the_last_tile(group, tokens, n, k):
    _case("f16", "f16", tokens, n, k, group, zeros=True, seed=n)
    _case("bf16", "f32", tokens, n, k, group, ldx=k + 8, beta=0.5, seed=k)
