"""The three operators together: the attention half of a decoding step, each of its stages against the formula in 64 bits of what the stage before it wrote, and the
whole of it from a graph.

Bounds of the errors, u being the type's largest relative rounding: those of each operator's own tests (tests/test_w4.py, test_rope.py, test_tree_attention.py).  A product
adds (stretch + stretches + 16) 2^-24 of the sum of |x| (32 + q + z) |s| to its one rounding; a rotation 6e-7 (|a| + |b|) to its; in the attention a score is off
by e = (d + 4) 2^-24 scale sum |q| |k|, a weight by 2 e of itself, its rounding u and 2^-21, the sums by (n + 64) 2^-24, and the result is rounded."""
import numpy as np
import pytest

import rocwmma_amd as R
from rocwmma_amd import decode_step as D

pytestmark = pytest.mark.gpu
U = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def _product(layer, x, weights, u, c=0.0):
    """(x w^T + c, bound of the error of the one that the kernel makes)"""
    rows, _, scales = weights
    q = rows.cpu().numpy()
    q = np.stack([q & 15, q >> 4], axis=2).reshape(q.shape[0], -1).astype(np.float64)
    s = np.repeat(scales.double().cpu().numpy(), layer.group, axis=0)[: q.shape[1]].T
    want, stretch = x @ ((q - 8.0) * s).T + c, min(layer.group, 128)
    bound = (stretch + q.shape[1] / stretch + 16) * 2.0 ** -24 * (np.abs(x) @ ((40.0 + q) * np.abs(s)).T)
    return want, bound + (u + 2.0 ** -22) * np.abs(want) + 2.0 ** -23 * np.abs(c) + 1e-7


def _rotated(layer, x, positions, u):
    turns, half = layer.turns.cpu().numpy().view(np.uint64), layer.head_dim // 2
    angle = np.array([[(int(p) * int(t)) % 2 ** 64 / 2.0 ** 64 for t in turns] for p in positions])[:, None, :] * 2 * np.pi
    a, b = x[..., :half], x[..., half:]
    want = np.concatenate([a * np.cos(angle) - b * np.sin(angle), a * np.sin(angle) + b * np.cos(angle)], axis=2)
    return want, 6e-7 * np.tile(np.abs(a) + np.abs(b), 2) + u * np.abs(want) * (1 + 1e-6) + 2.0 ** -25


def _attended(layer, q, k, v, step, lengths, u):
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    bits = np.unpackbits(step["mask"].view(np.uint8), axis=1, bitorder="little").astype(bool)
    row, scale = 0, layer.head_dim ** -0.5
    for seq, (n, before) in enumerate(lengths):
        place = np.arange(before + n)
        slots = step["table"][seq, place // layer.page_size] * layer.page_size + place % layer.page_size
        for i in range(row, row + n):
            seen = np.concatenate([np.ones(before, bool), bits[i, :n]])
            for h in range(layer.heads):
                ks, vs = (m[slots, h // (layer.heads // layer.kv_heads)][seen] for m in (k, v))
                x = ks @ q[i, h] * scale
                e = (layer.head_dim + 4) * 2.0 ** -24 * scale * np.max(np.abs(ks) @ np.abs(q[i, h]))
                p = np.exp(x - x.max())
                p /= p.sum()
                out[i, h] = p @ vs
                small = seen.sum() * np.abs(vs).max() * 2.0 ** -35
                bound[i, h] = (u + 2 * e + 2.0 ** -21 + (seen.sum() + 64) * 2.0 ** -24) * (p @ np.abs(vs)) * (1 + 4 * u) + u * np.abs(out[i, h]) + small + 1e-7
        row += n
    return out, bound


def _close(got, want, bound):
    error = np.abs(got - want)
    assert np.all(error <= bound), np.max(error / bound)


@pytest.mark.parametrize("dtype,lengths,group", [("f16", [(1, 37), (1, 0), (1, 300)], 128), ("bf16", [(9, 70), (1, 5), (17, 0)], 64), ("f16", [(33, 260), (5, 16)], 32)])
def test_step_vs_formula_and_from_a_graph(dtype, lengths, group):
    import torch

    page, pages = 16, 64
    layer = D.AttentionLayer(512, 8, 2, 64, pages, page, group=group, dtype=dtype, seed=len(lengths))
    layer.k.normal_()
    layer.v.normal_()
    before = [m.double().cpu().numpy() for m in (layer.k, layer.v)]
    host = D.draft(lengths, page, pages, seed=3)
    step = {name: torch.from_numpy(a).cuda() for name, a in host.items()}
    tokens = sum(n for n, _ in lengths)
    layer.reserve(tokens, max(n for n, _ in lengths), max(sum(l) for l in lengths), len(lengths), step["table"].shape[1])
    x = torch.randn(tokens, 512, device="cuda").to(layer.torch_type)
    y = layer.step(x, **step)
    x_, y_, qkv, q, k, v, attended = (m.double().cpu().numpy() for m in (x, y, layer.qkv, layer.q, layer.k, layer.v, layer.attended))
    u = U[dtype]
    _close(qkv.reshape(tokens, -1), *_product(layer, x_, layer.wqkv, u))
    _close(q, *_rotated(layer, qkv[:, :8], host["positions"], u))
    _close(k[host["slots"]], *_rotated(layer, qkv[:, 8:10], host["positions"], u))
    assert np.array_equal(v[host["slots"]], qkv[:, 10:])
    _close(attended, *_attended(layer, q, k, v, host, lengths, u))
    _close(y_, *_product(layer, attended.reshape(tokens, -1), layer.wo, u, c=x_))
    others = np.setdiff1d(np.arange(pages * page), host["slots"])
    for m, was in zip((layer.k, layer.v), before):  # nothing but the tokens' slots is written
        assert np.array_equal(m.double().cpu().numpy()[others], was[others])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        layer.step(x, **step, stream=torch.cuda.current_stream())
    for replay in range(3):
        for buffer in (layer.qkv, layer.q, layer.attended, layer.y):
            buffer.fill_(float("nan"))
        layer.workspace.fill_(0xFF)
        layer.k[step["slots"].long()] = float("nan")
        layer.v[step["slots"].long()] = float("nan")
        x.add_(1.0)  # the program's own eager work between replays, and other inputs
        eager = layer.step(x, **step).clone()
        layer.y.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(layer.y, eager), replay


def test_draft_is_refused_without_pages():
    with pytest.raises(ValueError):
        D.draft([(4, 100)], 16, 6)
