"""Attention of more sequences than a wave has lanes, the long ones beyond the first 64: which share of whose positions a workgroup takes, and which of them are joined, is counted
over all of them (bounds: tests/test_tree_attention.py)."""
import numpy as np
import pytest

from test_tree_attention import Problem


def _lengths(batch, tokens, long):
    """(tokens, positions): short ones, some without positions or without tokens, `long` ones from the 65th on"""
    lengths = []
    for b in range(batch):
        n = 1 + (b * 7) % tokens
        lengths.append((n, n + (b * 37) % 90))
        if b % 11 == 4:
            lengths[-1] = (n, 0)
        if b % 13 == 5:
            lengths[-1] = (0, 60)
    for i, l in enumerate(long):
        b = 64 + i * (batch - 64) // len(long)
        lengths[b] = (tokens, l)
    lengths[3] = (tokens, 700)
    return lengths


@pytest.mark.gpu
@pytest.mark.parametrize("batch,long", [(65, [5000]), (130, [3000, 257, 1500, 2100])])
@pytest.mark.parametrize("tokens,heads,kv_heads,dim", [(1, 4, 1, 64), (6, 4, 1, 128), (12, 4, 1, 64), (30, 4, 1, 64), (3, 2, 1, 256)])  # 16, 32, 64, 128 rows a workgroup, wide heads
def test_more_sequences_than_lanes(batch, long, tokens, heads, kv_heads, dim):
    p = Problem("bf16", _lengths(batch, tokens, long), heads, kv_heads, dim, seed=batch + tokens)
    a = p.check()
    share = p.max_tokens * heads * (dim + 2) * 4
    assert p.need // share > batch  # split
    b = p.check(workspace=(batch + 9) * share)  # ... into fewer
    c = p.check(workspace=0)  # ... not at all
    again = p.run(workspace=(batch + 9) * share)
    assert np.array_equal(b[0], again[0]) and np.array_equal(b[1], again[1])
    assert not np.array_equal(a[0], c[0])  # (the sums are split, which the last bits show)
