"""The static checks of the generated code (tests/test_isa_hazards.py) for the operators of a decoding step, and: no kernel of theirs spills registers
or keeps anything in scratch memory, whose loads would wait for the direct loads in flight."""
import os
import re

import pytest

from rocwmma_amd import build as B
from test_isa_hazards import WIDE_STORE_SCALAR_OFFSET, _asm, _early_overwrites, _stale_matrix_operands


@pytest.mark.skipif(not os.path.exists(B.HIPCC), reason="hipcc not installed")
@pytest.mark.parametrize("source", ["w4.hip", "rope.hip", "tree_attention.hip"])
def test_generated_code(source):
    text = _asm((source, []))
    assert not _stale_matrix_operands(text)
    assert not _early_overwrites(text)
    assert not WIDE_STORE_SCALAR_OFFSET.search(text)
    sizes = re.findall(r"\.private_segment_fixed_size:\s*(\d+)", text)
    spills = re.findall(r"\.vgpr_spill_count:\s*(\d+)", text)
    assert sizes and spills
    assert all(int(n) == 0 for n in spills), spills
    assert all(int(n) == 0 for n in sizes), sizes
    assert not re.search(r"v_pk_(add|mul|fma)_f32", text)
