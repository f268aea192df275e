"""Index arrays off the alignment of their elements (scalar loads would drop the low bits of such an address) are refused at the C entries."""
import pytest

import rocwmma_amd as R
from test_rope import _refused as rope_refused
from test_tree_attention import _refused as tree_refused


@pytest.mark.parametrize("name", ["table", "q_start", "kv_len"])
def test_tree_attention(name):
    tree_refused(-4, **{name: 0x5002})


def test_rope():
    part = R.rope_part(0x1000, 0x2000, 2, (128, 64), (128, 64), to_slots=True)
    rope_refused(-4, positions=0x3002, slots=0x5000, parts=[part])
    rope_refused(-4, slots=0x5001, parts=[part])
