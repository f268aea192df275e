"""Static checks of the generated gfx950 code of the layers' products and the router (no GPU needed): the hazards of test_isa_hazards.py, that nothing spills in the loops over the
sum, and that their matrix instructions keep the accumulators in place."""
import os
import re

import pytest

from rocwmma_amd import build as B
from test_isa_hazards import WIDE_STORE_SCALAR_OFFSET, _asm, _early_overwrites, _stale_matrix_operands

UNITS = [("linear_tiles.hip", []), ("linear_tiles.hip", ["-DR355_LINEAR_BF16"]), ("linear.hip", []), ("experts.hip", [])]
_TEXTS = {}


def _texts():
    if not _TEXTS:
        from concurrent.futures import ThreadPoolExecutor

        with ThreadPoolExecutor(max_workers=len(UNITS)) as pool:
            for unit, text in zip(UNITS, pool.map(_asm, UNITS)):
                _TEXTS[(unit[0], tuple(unit[1]))] = text
    return _TEXTS


@pytest.mark.skipif(not os.path.exists(B.HIPCC), reason="hipcc not installed")
def test_hazards():
    matrix = stores = 0
    for unit, text in _texts().items():
        assert not _stale_matrix_operands(text), (unit, _stale_matrix_operands(text)[:3])
        assert not _early_overwrites(text), (unit, _early_overwrites(text)[:3])
        assert not WIDE_STORE_SCALAR_OFFSET.findall(text), unit
        matrix += len(re.findall(r"^\s*v_mfma_", text, flags=re.M))
        stores += len(re.findall(r"buffer_store_dwordx[34]", text))
    assert matrix > 5000 and stores > 1000  # the scans are looking at the kernels' instructions (the loops are one stage long)


@pytest.mark.skipif(not os.path.exists(B.HIPCC), reason="hipcc not installed")
def test_no_packed_f32_and_no_spills_to_memory():
    for unit, text in _texts().items():
        assert not re.findall(r"v_pk_(add|mul|fma)_f32", text), unit
        assert not re.findall(r"\.vgpr_spill_count:\s+[1-9]", text), unit
        assert not re.findall(r"\.private_segment_fixed_size:\s+[1-9]", text), unit


@pytest.mark.skipif(not os.path.exists(B.HIPCC), reason="hipcc not installed")
def test_loops_over_the_sum_only_multiply_read_and_load():
    """The blocks with the most matrix instructions: no accumulator is moved, and per matrix instruction there is less than one other vector instruction"""
    found = 0
    for (source, _), text in _texts().items():
        if source != "linear_tiles.hip":
            continue
        for block in re.split(r"^\.LBB\S+:.*$|^\s*s_cbranch\S* .*$", text, flags=re.M):
            ins = [l.strip() for l in block.splitlines()]
            matrix = sum(i.startswith("v_mfma") for i in ins)
            if matrix < 30:
                continue
            found += 1
            assert not any(i.startswith(("v_accvgpr_read", "v_accvgpr_write", "scratch_", "v_readlane")) for i in ins)
            assert sum(i.startswith("v_") and not i.startswith("v_mfma") for i in ins) < matrix
    assert found >= 40
