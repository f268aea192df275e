"""Attention of drafted tokens where the caller allows for a long cache (the kernel of eight waves is chosen by that, not by the lengths on the device, so
small lengths reach it): bounds as in tests/test_tree_attention.py."""
import numpy as np
import pytest

from test_tree_attention import Problem

pytestmark = pytest.mark.gpu
LONG = 1 << 20  # positions allowed for: 256 MiB and more of keys and values with two key heads of 32 and more


def _allow(p):
    """A table wide enough for LONG positions, of which the pages that there are come first."""
    wide = np.full((p.batch, LONG // p.page), -1, np.int32)
    wide[:, : p.table.shape[1]] = p.table
    p.table = wide
    return p


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("past", [0, 1, 31, 32, 58, 65, 190, 500])
def test_tree_long_vs_formula(dtype, dim, past):
    _allow(Problem(dtype, [(70, 70 + past), (45, 45 + 2 * past)], 6, 2, dim, seed=dim + past)).check(extra_kv=LONG)


@pytest.mark.parametrize("workspace", ["asked", 0])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_tree_long_split(dim, workspace):
    p = _allow(Problem("bf16", [(50, 3000), (7, 1111), (33, 40)], 8, 2, dim, page=32, seed=dim))
    a = p.check(extra_kv=LONG, workspace=workspace)
    b = p.run(extra_kv=LONG, workspace=workspace)
    assert p.need > 0
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])


def test_tree_long_chain():
    _allow(Problem("f16", [(150, 150), (1, 77), (65, 400)], 6, 3, 64, seen=None, seed=4)).check(extra_kv=LONG)


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("dim", [64, 128])
def test_tree_long_what_is_not_seen_does_not_count(bad, dim):
    p = _allow(Problem("bf16", [(40, 150), (40, 56)], 12, 2, dim, seed=9))
    want, bound, wl, bl = p.want(dim ** -0.5)
    used = np.concatenate([p.slots(b) for b in range(2)])
    spare = np.setdiff1d(np.arange(p.pages * p.page), used)
    p.k[spare], p.v[spare] = bad, bad
    victim = 3
    for b in range(2):
        p.v[p.slots(b)[p.lengths[b][1] - 40 + victim], :, 5] = bad
    out, lse = p.run(extra_kv=LONG)
    sees = np.concatenate([p.seen[b][:, victim] for b in range(2)])
    assert sees.any() and not sees.all()
    assert np.all(np.abs(out - want)[~sees] <= bound[~sees]) and np.all(np.abs(lse - wl) <= bl)
    assert not np.isfinite(out[sees][..., 5]).any()


@pytest.mark.parametrize("lengths", [[(1, 900)], [(1, 3000), (1, 100), (3, 700)], [(4, 6000)], [(1, 10 + 97 * i) for i in range(40)]])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 1, 128), (8, 2, 64), (16, 8, 256)])
def test_tree_one_workgroup_a_cu_and_several(lengths, heads, kv_heads, dim):
    """Shares of one sequence, of several with eight shares each and more, and of more sequences than that."""
    p = Problem("bf16", lengths, heads, kv_heads, dim, seed=len(lengths))
    p.check()
    _allow(p).check(extra_kv=LONG)
