"""Attention of drafted tokens over a paged cache against the formula in 64 bits.

Bound of the error of an element, with A = sum_j p_j |v_j| and u the largest relative rounding of the type (2^-11 f16, 2^-8 bf16):
a score is a sum of d products in f32 and one scaling, off by at most e = (d + 4) 2^-24 scale sum |q| |k| (the largest of the row), which
changes a weight by 2 e of itself (numerator and sum); the weight is rounded (u) and its exponential is within 2^-21; f32 sums over n positions add
(n + 64) 2^-24; a weight under the type's normal numbers is off by half its smallest step (bf16: none; f16: 2^-25 of 2^10, n |v| of
that); and the result is rounded (u)."""
import numpy as np
import pytest

import rocwmma_amd as R

TYPES = {"f16": R.F16, "bf16": R.BF16}
U = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def _torch_type(name):
    import torch

    return {"f16": torch.float16, "bf16": torch.bfloat16}[name]


def _tree(rng, n):
    seen = np.zeros((n, n), bool)
    for j in range(n):
        if j:
            seen[j] = seen[max(0, j - 1 - int(rng.exponential(2.0)))]
        seen[j, j] = True
    return seen


class Problem:
    """A batch: `lengths` of (drafted tokens, cached positions).  seen: per sequence the drafted tokens that each row sees (None: chain)."""

    def __init__(self, dtype, lengths, heads, kv_heads, dim, page=16, seed=0, seen="tree", loud=1.0, spare=3):
        import torch

        rng = np.random.RandomState(seed)
        self.dtype, self.lengths, self.heads, self.kv, self.dim, self.page = dtype, lengths, heads, kv_heads, dim, page
        self.total, self.batch = sum(n for n, _ in lengths), len(lengths)
        self.max_tokens, self.max_kv = max(n for n, _ in lengths), max(l for _, l in lengths)
        pages = [-(-l // page) for _, l in lengths]
        self.pages = sum(pages) + spare
        order = rng.permutation(self.pages).astype(np.int32)
        self.table = np.full((self.batch, max(max(pages), 1)), -1, np.int32)
        at = 0
        for b, m in enumerate(pages):
            self.table[b, :m] = order[at: at + m]
            at += m
        t = _torch_type(dtype)
        self.q = torch.from_numpy(rng.randn(self.total, heads, dim) * loud).to(t)
        self.k, self.v = (torch.from_numpy(rng.randn(self.pages * page, kv_heads, dim)).to(t) for _ in range(2))
        self.seen = [None if seen is None else _tree(rng, n) if isinstance(seen, str) else seen(b, n) for b, (n, _) in enumerate(lengths)]

    def slots(self, b):
        l = self.lengths[b][1]
        return (self.table[b][:, None] * self.page + np.arange(self.page)).reshape(-1)[:l]

    def mask(self, words):
        bits = np.zeros((self.total, words * 64), np.uint8)
        row = 0
        for (n, _), s in zip(self.lengths, self.seen):
            bits[row: row + n, :n] = s
            row += n
        return np.packbits(bits, axis=1, bitorder="little").view(np.int64)

    def want(self, scale):
        """(out, bound of its error, lse, bound of its error)"""
        out, bound = np.zeros((self.total, self.heads, self.dim)), np.zeros((self.total, self.heads, self.dim))
        lse, lbound = np.zeros((self.total, self.heads)), np.zeros((self.total, self.heads))
        q, k, v = (x.double().numpy() for x in (self.q, self.k, self.v))
        row, u = 0, U[self.dtype]
        for b, (n, l) in enumerate(self.lengths):
            vis = np.ones((n, l), bool)
            drafted = np.tril(np.ones((n, n), bool)) if self.seen[b] is None else self.seen[b]
            keep = min(n, l)  # (drafted tokens beyond the cache: the last ones are there)
            vis[:, l - keep:] = drafted[:, n - keep:]
            for h in range(self.heads):
                ks, vs = k[self.slots(b), h // (self.heads // self.kv)], v[self.slots(b), h // (self.heads // self.kv)]
                for i in range(n):
                    m = vis[i]
                    if not m.any():
                        lse[row + i, h] = -np.inf
                        continue
                    x = ks[m] @ q[row + i, h] * scale
                    e = (self.dim + 4) * 2.0 ** -24 * abs(scale) * np.max(np.abs(ks[m]) @ np.abs(q[row + i, h]))
                    top = x.max()
                    p = np.exp(x - top)
                    lse[row + i, h] = top + np.log(p.sum())
                    p /= p.sum()
                    out[row + i, h] = p @ vs[m]
                    a = p @ np.abs(vs[m])
                    small = m.sum() * np.abs(vs[m]).max() * 2.0 ** -35 if self.dtype == "f16" else 0.0
                    bound[row + i, h] = (u + 2 * e + 2.0 ** -21 + (m.sum() + 64) * 2.0 ** -24) * a * (1 + 4 * u) + u * np.abs(out[row + i, h]) + small + 1e-7
                    lbound[row + i, h] = 2 * e + (m.sum() + 64) * 2.0 ** -24 + 2.0 ** -21 + 2.0 ** -21 * abs(lse[row + i, h])
            row += n
        return out, bound, lse, lbound

    def run(self, scale=None, workspace="asked", chain=False, stream=None, extra_kv=0):
        import torch

        scale = self.dim ** -0.5 if scale is None else scale
        out = torch.full(self.q.shape, float("nan"), dtype=self.q.dtype, device="cuda")
        lse = torch.full((self.total, self.heads), float("nan"), dtype=torch.float32, device="cuda")
        start = np.concatenate([[0], np.cumsum([n for n, _ in self.lengths])]).astype(np.int32)
        dev = [torch.from_numpy(x).cuda() for x in (self.table, start, np.array([l for _, l in self.lengths], np.int32))]
        words = -(-self.max_tokens // 64)
        mask = None if chain or self.seen[0] is None else torch.from_numpy(self.mask(words)).cuda()
        q, k, v = self.q.cuda(), self.k.cuda(), self.v.cuda()
        args = [TYPES[self.dtype], self.batch, self.total, self.heads, self.kv, self.dim, q, k, v, out, dev[0], self.page, self.pages, dev[1], dev[2],
                self.max_tokens, min(self.max_kv + extra_kv, self.table.shape[1] * self.page)]
        kw = dict(mask=mask, mask_words=words if mask is not None else 0, lse=lse, scale=scale)
        need = R.tree_attention_workspace_bytes(R.tree_attention_args(*args, **kw))
        size = need if workspace == "asked" else workspace
        ws = torch.full((max(size, 16),), 0xFF, dtype=torch.uint8, device="cuda") if size else None
        self.need = need
        R.tree_attention(*args, **kw, workspace=ws, stream=stream)
        torch.cuda.synchronize()
        return out.double().cpu().numpy(), lse.double().cpu().numpy()

    def check(self, scale=None, **kw):
        out, lse = self.run(scale, **kw)
        want, bound, wl, bl = self.want(self.dim ** -0.5 if scale is None else scale)
        assert np.all(np.abs(out - want) <= bound), np.max(np.abs(out - want) / np.maximum(bound, 1e-30))
        empty = np.isinf(wl)
        assert np.array_equal(lse[empty], wl[empty])
        assert np.all(np.abs(lse[~empty] - wl[~empty]) <= bl[~empty])
        return out, lse


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128, 256, 8, 72, 96, 192])
@pytest.mark.parametrize("heads,kv_heads,n", [(4, 4, 1), (12, 2, 4), (6, 1, 9), (8, 2, 30), (6, 2, 70)])
def test_tree_vs_formula(dtype, dim, heads, kv_heads, n):
    Problem(dtype, [(n, n + 100), (max(1, n - 3), n + 31)], heads, kv_heads, dim, seed=dim + n).check()


@pytest.mark.gpu
@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 31, 32, 33, 127, 128, 129, 255, 256, 257, 383, 384, 385, 513, 1000])
def test_tree_lengths(length):
    Problem("bf16", [(1, length)], 4, 2, 64, page=32, seed=length).check()
    Problem("f16", [(min(length, 5), length)], 10, 1, 128, seed=length).check()
    Problem("bf16", [(min(length, 40), length)], 8, 2, 128, seed=length).check()


@pytest.mark.gpu
@pytest.mark.parametrize("page", [16, 32, 48, 64, 256])
def test_tree_pages(page):
    Problem("f16", [(3, 300), (2, 61), (5, 500)], 4, 2, 64, page=page, seed=page).check()


@pytest.mark.gpu
@pytest.mark.parametrize("n,heads,kv_heads", [(1, 8, 2), (20, 4, 1), (50, 8, 2)])
def test_tree_split_over_workgroups(n, heads, kv_heads):
    """More positions than one workgroup takes: with the workspace asked for, with a third of it, with none; the same result within
    the bound each time and the same bits on the same workspace."""
    p = Problem("bf16", [(n, 5000), (max(1, n // 2), 2600), (n, 300)], heads, kv_heads, 128, page=32, seed=n)
    a = p.check()
    assert p.need > 0
    b = p.run()
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])
    p.check(workspace=p.need // 3)
    p.check(workspace=0)


@pytest.mark.gpu
def test_tree_chain():
    """Without a mask a row sees up to itself: chunks of a prompt, whole prompts, single tokens."""
    for lengths in ([(200, 200), (1, 77), (65, 400)], [(1, 1), (1, 900)], [(33, 33)]):
        Problem("bf16", lengths, 6, 3, 64, seen=None, seed=4).check()


@pytest.mark.gpu
def test_tree_rows_that_see_nothing_or_only_themselves():
    # no prefix: an empty mask row leaves nothing; a prefix: the row sees only that
    def some(b, n):
        s = np.zeros((n, n), bool)
        s[0, 0] = s[2, 1] = True
        return s

    out, lse = Problem("f16", [(4, 4), (4, 20), (3, 3)], 4, 2, 64, seen=some, seed=1).check()
    assert np.all(out[1] == 0) and np.all(np.isneginf(lse[1])) and np.all(out[3] == 0)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 20, 40])
def test_tree_sequences_without_tokens_or_positions(n):
    p = Problem("bf16", [(n, 70), (0, 50), (n, n), (2, 0), (0, 0), (3, 1)], 8, 2, 64, seed=2, seen=None)
    out, lse = p.run()
    want, bound, wl, bl = p.want(64 ** -0.5)
    rows = [0] * n + [2] * n + [3] * 2 + [5] * 3
    keep = np.array([r not in (3, 5) for r in rows])
    assert np.all(np.abs(out - want)[keep] <= bound[keep])
    assert np.all(out[~keep][:2] == 0) and np.all(np.isneginf(lse[~keep][:2]))
    # three drafted tokens over one position: it is the last of them, and only that row sees it
    assert np.all(out[-3:-1] == 0) and np.all(np.isneginf(lse[-3:-1]))
    assert np.all(np.abs(out - want)[-1] <= bound[-1])


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("n,heads", [(6, 2), (6, 12), (30, 12)])
def test_tree_what_is_not_seen_does_not_count(bad, n, heads):
    """Drafted tokens and slots that a row does not see hold infinities and NaN; rows that see them are not finite, the others as without."""
    import torch

    p = Problem("bf16", [(n, 150), (n, n + 16)], heads, 2, 64, seed=9)
    want, bound, wl, bl = p.want(0.125)
    used = np.concatenate([p.slots(b) for b in range(2)])
    spare = np.setdiff1d(np.arange(p.pages * p.page), used)
    p.k[spare], p.v[spare] = bad, bad
    victim = 3
    for b in range(2):
        p.v[p.slots(b)[p.lengths[b][1] - n + victim], :, 5] = bad
        p.k[p.slots(b)[p.lengths[b][1] - n + victim]] = float("nan") if bad != bad else p.k[p.slots(b)[p.lengths[b][1] - n + victim]]
    out, lse = p.run(0.125)
    sees = np.concatenate([p.seen[b][:, victim] for b in range(2)])
    assert sees.any() and not sees.all()
    assert np.all(np.abs(out - want)[~sees] <= bound[~sees]) and np.all(np.abs(lse - wl)[~sees] <= bl[~sees])
    assert not np.isfinite(out[sees][..., 5]).any()


@pytest.mark.gpu
def test_tree_loud_scores_and_scales():
    """Scores of hundreds: the running maximum moves, weights underflow."""
    Problem("f16", [(7, 700), (3, 40)], 4, 2, 64, seed=3, loud=20.0).check(scale=0.5)
    Problem("bf16", [(40, 700)], 8, 2, 128, seed=3, loud=10.0).check(scale=-0.25)
    Problem("bf16", [(4, 300)], 4, 2, 64, seed=3).check(scale=0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [2, 60])
def test_tree_strides(n):
    """q and out as slices of wider rows, k and v interleaved in one cache, a wider table, no lse."""
    import torch

    p = Problem("f16", [(n, 200), (n, 90)], 8, 2, 64, seed=6)
    want, bound, _, _ = p.want(0.125)
    wide = torch.full((p.total, 12, 80), float("nan"), dtype=torch.float16, device="cuda")
    wide[:, 2:10, :64] = p.q.cuda()
    both = torch.full((p.pages * p.page, 2, 2, 72), float("nan"), dtype=torch.float16, device="cuda")
    both[:, 0, :, :64], both[:, 1, :, :64] = p.k.cuda(), p.v.cuda()
    out = torch.full((p.total, 9, 68), float("nan"), dtype=torch.float16, device="cuda")
    table = torch.full((p.batch, p.table.shape[1] + 5), -7, dtype=torch.int32, device="cuda")
    table[:, : p.table.shape[1]] = torch.from_numpy(p.table).cuda()
    R.tree_attention(R.F16, 2, p.total, 8, 2, 64, wide[:, 2:], both, both[:, 1:], out[:, 1:], table, p.page, p.pages,
                     torch.tensor([0, n, 2 * n], dtype=torch.int32, device="cuda"), torch.tensor([200, 90], dtype=torch.int32, device="cuda"), n, 200,
                     mask=torch.from_numpy(p.mask(1)).cuda(), mask_words=1, q_strides=(960, 80), k_strides=(288, 72), v_strides=(288, 72),
                     out_strides=(612, 68))
    got = out.double().cpu().numpy()
    assert np.all(np.abs(got[:, 1:, :64] - want) <= bound)
    assert np.isnan(got[:, 0]).all() and np.isnan(got[..., 64:]).all()


@pytest.mark.gpu
def test_tree_bounds_hold_against_the_arrays():
    """Lengths over the bounds given, pages outside the cache: left out and zeros, nothing else."""
    import torch

    p = Problem("bf16", [(4, 100)], 4, 2, 64, seed=7, seen=None)
    q, k, v = p.q.cuda(), p.k.cuda(), p.v.cuda()
    out = torch.full(p.q.shape, float("nan"), dtype=p.q.dtype, device="cuda")
    lse = torch.full((4, 4), float("nan"), device="cuda")
    start, table = torch.tensor([0, 9], dtype=torch.int32, device="cuda"), torch.from_numpy(p.table).cuda()

    def call(length, max_kv, table):
        R.tree_attention(R.BF16, 1, 4, 4, 2, 64, q, k, v, out, table, p.page, p.pages, start, torch.tensor([length], dtype=torch.int32, device="cuda"), 4, max_kv, lse=lse)
        return out.double().cpu().numpy(), lse.double().cpu().numpy()

    want, bound, wl, bl = p.want(0.125)
    got, gl = call(10 ** 9, 100, table)  # held to max_kv = 100, and the nine tokens to the four that there are
    assert np.all(np.abs(got - want) <= bound) and np.all(np.abs(gl - wl) <= bl)
    away = table.clone()
    away[0, 2] = p.pages
    p.k[p.slots(0)[32:48]], p.v[p.slots(0)[32:48]] = 0, 0
    want, bound, wl, bl = p.want(0.125)
    got, gl = call(100, 100, away)
    assert np.all(np.abs(got - want) <= bound) and np.all(np.abs(gl - wl) <= bl)


@pytest.mark.gpu
def test_tree_cache_beyond_4_gib():
    """Offsets past 32 bits: the pages of a short sequence lie at the end of a cache of 5 GiB."""
    import torch

    p = Problem("f16", [(3, 90)], 4, 2, 64, seed=5)
    slots = (5 << 30) // (2 * 64 * 2)
    k, v = (torch.empty(slots, 2, 64, dtype=torch.float16, device="cuda") for _ in range(2))
    shift = slots // 16 - p.pages
    k[shift * 16:], v[shift * 16:] = p.k.cuda(), p.v.cuda()
    out = torch.empty(p.q.shape, dtype=torch.float16, device="cuda")
    R.tree_attention(R.F16, 1, 3, 4, 2, 64, p.q.cuda(), k, v, out, torch.from_numpy(p.table + shift).cuda(), 16, slots // 16,
                     torch.tensor([0, 3], dtype=torch.int32, device="cuda"), torch.tensor([90], dtype=torch.int32, device="cuda"), 3, 90,
                     mask=torch.from_numpy(p.mask(1)).cuda(), mask_words=1)
    want, bound, _, _ = p.want(0.125)
    assert np.all(np.abs(out.double().cpu().numpy() - want) <= bound)


@pytest.mark.gpu
def test_tree_on_another_stream():
    import torch

    p = Problem("bf16", [(2, 3000)], 4, 2, 64, seed=5)
    a = p.run()
    b = p.run(stream=torch.cuda.Stream())
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])


def _args(**change):
    a = dict(dtype=R.F16, batch=2, total_tokens=4, heads=8, kv_heads=2, head_dim=64, q=0x1000, k=0x2000, v=0x3000, out=0x4000, table=0x5000, page_size=16,
             pages=32, q_start=0x6000, kv_len=0x7000, max_tokens=2, max_kv=256, table_stride=16)
    a.update(change)
    return R.tree_attention_args(**a)


def _refused(code, **change):
    a = _args(**change)
    import ctypes

    assert R.lib().r355_tree_attention(ctypes.byref(a), None) == code, (change, R.lib().r355_last_error())


def test_tree_refusals():
    for name in ("q", "k", "v", "out", "table", "q_start", "kv_len"):
        _refused(-1, **{name: None})
    for name in ("heads", "kv_heads", "head_dim", "page_size"):
        _refused(-1, **{name: 0}, **({"scale": 1.0} if name == "head_dim" else {}))
    _refused(-2, dtype=R.F32)
    _refused(-3, heads=7)
    _refused(-3, head_dim=60)
    _refused(-3, head_dim=264)
    _refused(-3, page_size=24)
    _refused(-3, mask=0x8000, mask_words=0)
    _refused(-3, max_kv=257)
    _refused(-3, max_kv=(1 << 30) + 1)
    _refused(-3, k_strides=(1 << 26, 64))
    _refused(-3, v_strides=(56, 64))
    _refused(-3, pages=1 << 31, page_size=48)
    _refused(-3, batch=1 << 24)
    _refused(-4, q=0x1008)
    _refused(-4, k=0x2008)
    _refused(-4, v=0x3008)
    _refused(-4, out=0x4004)
    _refused(-4, q_strides=(516, 64))
    _refused(-4, out_strides=(514, 64))
    _refused(-4, mask=0x8004, mask_words=1)
    _refused(-4, workspace=0x9008, workspace_bytes=1 << 20)
    for nothing in (dict(batch=0), dict(total_tokens=0), dict(max_tokens=0)):
        _refused(0, q=None, **nothing)
        assert R.tree_attention_workspace_bytes(_args(**nothing)) == 0


def test_tree_workspace_is_for_long_sequences():
    assert R.tree_attention_workspace_bytes(_args(max_kv=200, table_stride=100)) == 0
    need = R.tree_attention_workspace_bytes(_args(max_kv=16384, table_stride=1024))
    assert need > 0 and need % (4 * 8 * (64 + 2) * 4) == 0
    assert R.tree_attention_workspace_bytes(_args(heads=7)) == 0


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), 1e300])
def test_tree_refuses_a_scale_that_is_not_finite(scale):
    _refused(-1, scale=scale)
