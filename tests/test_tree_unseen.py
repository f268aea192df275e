"""Attention over drafted tokens whose values hold infinities and NaN: they reach the elements of the rows that see them, and nothing else.  Elements that they do not reach are held
against the formula in 64 bits without them (bounds: tests/test_tree_attention.py)."""
import numpy as np
import pytest

from test_tree_attention import Problem
from test_tree_long_caches import LONG, _allow

INF, NAN = float("inf"), float("nan")


def _check(p, bad, **kw):
    """bad: (drafted token, element of the head, value), the same in every sequence and key head"""
    want, bound, want_lse, lse_bound = p.want(p.dim ** -0.5)
    plus, minus = np.zeros((2, p.total, p.dim), bool)
    first = 0
    for b, (n, l) in enumerate(p.lengths):
        for token, d, value in bad:
            p.v[p.slots(b)[l - n + token], :, d] = value
            plus[first: first + n, d] |= p.seen[b][:, token] & (value != -INF)
            minus[first: first + n, d] |= p.seen[b][:, token] & (value != INF)
        first += n
    out, lse = p.run(**kw)
    plus, minus = (np.broadcast_to(x[:, None], out.shape) for x in (plus, minus))
    clean = ~plus & ~minus
    assert plus.any() and minus.any() and (plus & minus).any() and clean[plus.any(2)].any()
    assert np.all(np.abs(out - want)[clean] <= bound[clean]) and np.all(np.abs(lse - want_lse) <= lse_bound)
    assert np.all(out[plus & ~minus] == INF) and np.all(out[minus & ~plus] == -INF) and np.all(np.isnan(out[plus & minus]))


def _some(b, n):
    """every row sees itself and about half of the others"""
    seen = np.random.RandomState(b).rand(n, n) < 0.5
    np.fill_diagonal(seen, True)
    return seen


BAD = [(0, 1, INF), (1, 5, NAN), (2, 5, INF), (2, 7, -INF), (3, 7, INF), (3, 8, -INF), (4, 30, NAN)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [32, 64, 128, 256])
@pytest.mark.parametrize("n,heads,kv_heads", [(7, 2, 2), (9, 6, 2), (30, 4, 2), (45, 6, 2)])  # up to 16, 32, 64 and 128 rows a workgroup (heads of 256: 16 and 64)
def test_tree_reaches_those_that_see_it(dtype, dim, n, heads, kv_heads):
    _check(Problem(dtype, [(n, n + 150), (n, n)], heads, kv_heads, dim, seen=_some, seed=dim + n), BAD)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_tree_reaches_those_that_see_it_long(dtype, dim):
    p = Problem(dtype, [(45, 45 + 150), (45, 45)], 6, 2, dim, seen=_some, seed=dim)
    _check(_allow(p), BAD, extra_kv=LONG)
