"""Attention of the chunk of a prompt: many tokens, each seeing those up to itself.  A sample of the rows is held against the formula in 64 bits; bounds as in
tests/test_tree_attention.py."""
import numpy as np
import pytest

import rocwmma_amd as R
from test_tree_attention import U, Problem, _refused


def _check(p, sample):
    """rows `sample` of every sequence, at the first and the last head of every key head"""
    out, lse = p.run()
    assert np.isfinite(out).all() and np.isfinite(lse).all()
    q, k, v = (x.double().numpy() for x in (p.q, p.k, p.v))
    first, u, scale, group = 0, U[p.dtype], p.dim ** -0.5, p.heads // p.kv
    for b, (n, l) in enumerate(p.lengths):
        for kv in range(p.kv):
            ks, vs = k[p.slots(b), kv], v[p.slots(b), kv]
            for i in sorted({min(i, n - 1) for i in sample}):
                seen = l - n + i + 1
                for h in sorted({kv * group, kv * group + group - 1}):
                    row = q[first + i, h]
                    x = ks[:seen] @ row * scale
                    e = (p.dim + 4) * 2.0 ** -24 * scale * np.max(np.abs(ks[:seen]) @ np.abs(row))
                    w = np.exp(x - x.max())
                    want_lse = x.max() + np.log(w.sum())
                    w /= w.sum()
                    want = w @ vs[:seen]
                    small = seen * np.abs(vs[:seen]).max() * 2.0 ** -35 if p.dtype == "f16" else 0.0
                    bound = (u + 2 * e + 2.0 ** -21 + (seen + 64) * 2.0 ** -24) * (w @ np.abs(vs[:seen])) * (1 + 4 * u) + u * np.abs(want) + small + 1e-7
                    assert np.all(np.abs(out[first + i, h] - want) <= bound), (b, i, h)
                    assert abs(lse[first + i, h] - want_lse) <= 2 * e + (seen + 64) * 2.0 ** -24 + 2.0 ** -21 * (1 + abs(want_lse)), (b, i, h)
        first += n


SAMPLE = [0, 1, 15, 16, 31, 63, 64, 127, 128, 255, 256, 511, 700, 1023, 1024, 2047, 2048, 3000, 4091, 4095, 10 ** 9]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,lengths,heads,kv_heads,dim", [
    ("bf16", [(4096, 4096)], 32, 8, 128), ("f16", [(2048, 5000)], 64, 8, 64), ("bf16", [(512, 512)], 32, 1, 128), ("f16", [(1025, 1100), (3, 2000)], 32, 1, 64),
    ("bf16", [(2100, 2100)], 16, 2, 256), ("f16", [(8192, 8192)], 4, 2, 64), ("bf16", [(1000, 1000)] * 3 + [(5, 9)], 24, 4, 96)])
def test_chunk_of_a_prompt(dtype, lengths, heads, kv_heads, dim):
    _check(Problem(dtype, lengths, heads, kv_heads, dim, page=32, seen=None, seed=heads + dim), SAMPLE)


@pytest.mark.parametrize("tokens,heads,kv_heads", [(4096, 32, 8), (2048, 64, 8), (512, 32, 1), (1024, 32, 1), (131072, 32, 8), (1 << 20, 8, 8)])
def test_sizes_of_prompts_are_taken(tokens, heads, kv_heads):
    """(as far as the check of the pointers)"""
    for dim in (64, 128, 256):
        _refused(-1, q=None, batch=1, total_tokens=tokens, max_tokens=tokens, max_kv=tokens, table_stride=tokens // 16, heads=heads, kv_heads=kv_heads, head_dim=dim)


def test_more_workgroups_than_a_launch_has_are_refused():
    sizes = dict(batch=65535, total_tokens=1 << 20, max_kv=16, table_stride=1, heads=256, kv_heads=256)
    _refused(-1, q=None, max_tokens=1, **sizes)
    _refused(-3, max_tokens=129, **sizes)  # two tiles of rows
    _refused(-3, max_tokens=1, **{**sizes, "heads": 1 << 30, "kv_heads": 1 << 30})
    _refused(-3, max_tokens=1, **{**sizes, "batch": 65536})
    _refused(-3, max_tokens=(1 << 28) + 1, batch=1, total_tokens=1 << 30, max_kv=16, table_stride=1, heads=4, kv_heads=1)
    assert R.lib().r355_last_error()
