"""The attention half of a decoding step with drafted tokens, out of this library's operators: one product with 4-bit weights for queries, keys and
values, one launch that rotates queries and keys and appends keys and values to a paged cache, attention of every token over its
sequence's cache and its ancestors in the draft, and a second 4-bit product that adds the residual.

    python -m rocwmma_amd.decode_step [--sequences 8] [--drafted 48] [--cached 4000] [--hidden 4096] [--heads 32] [--kv-heads 8] [--head-dim 128]

times such a step over random weights and a random cache, launched one by one and replayed from a graph.  With --experts (and --top, --width) the feed-forward
half follows, expert_layer.py's."""
import argparse


class AttentionLayer:
    """Packed weights, a paged cache and the buffers of one layer; step() only launches kernels, so it can be recorded into a graph."""

    def __init__(self, hidden, heads, kv_heads, head_dim, pages, page_size, group=128, dtype="bf16", base=10000.0, seed=0):
        import torch

        import rocwmma_amd as R

        if hidden % group or heads * head_dim % group:
            raise ValueError("AttentionLayer: hidden and heads * head_dim must be multiples of the group")
        self.hidden, self.heads, self.kv_heads, self.head_dim = hidden, heads, kv_heads, head_dim
        self.pages, self.page_size, self.group = pages, page_size, group
        self.dtype, self.torch_type = {"bf16": (R.BF16, torch.bfloat16), "f16": (R.F16, torch.float16)}[dtype]
        self.qkv_heads = heads + 2 * kv_heads
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.wqkv = self._weights(self.qkv_heads * head_dim, hidden, gen)
        self.wo = self._weights(hidden, heads * head_dim, gen)
        self.k, self.v = (torch.zeros((pages * page_size, kv_heads, head_dim), dtype=self.torch_type, device="cuda") for _ in range(2))
        self.turns = torch.from_numpy(R.rope_turns(head_dim, base).view("int64")).cuda()

    def _weights(self, n, k, gen):
        """(rows of nibbles, packed, scales) of a random matrix whose product keeps the size of its input"""
        import torch

        import rocwmma_amd as R

        rows = torch.randint(0, 256, (n, (k + 1) // 2), dtype=torch.uint8, device="cuda", generator=gen)
        packed = torch.empty(R.w4_packed_bytes(n, k), dtype=torch.uint8, device="cuda")
        R.w4_pack(rows, n, k, packed)
        scales = ((0.75 + 0.5 * torch.rand((-(-k // self.group), n), device="cuda", generator=gen)) * 0.2 / k ** 0.5).to(self.torch_type)
        return rows, packed, scales

    def reserve(self, total_tokens, max_tokens, max_kv, batch, table_stride):
        """The buffers of steps of up to that size, kept for all of them: tokens in all, drafted tokens of a sequence, cached positions of one (those of the
        step among them), sequences and entries of a row of the table."""
        import torch

        import rocwmma_amd as R

        empty = lambda *shape, dtype=self.torch_type: torch.empty(shape, dtype=dtype, device="cuda")
        self.qkv = empty(total_tokens, self.qkv_heads, self.head_dim)
        self.q, self.attended = empty(total_tokens, self.heads, self.head_dim), empty(total_tokens, self.heads, self.head_dim)
        self.y = empty(total_tokens, self.hidden)
        self.total_tokens, self.batch, self.max_tokens, self.max_kv = total_tokens, batch, max_tokens, max_kv
        sizes = R.tree_attention_args(self.dtype, batch, total_tokens, self.heads, self.kv_heads, self.head_dim, None, None, None, None, None,
                                      self.page_size, self.pages, None, None, max_tokens, max_kv, table_stride=table_stride)
        self.workspace = empty(max(R.tree_attention_workspace_bytes(sizes), 16), dtype=torch.uint8)

    def _holds(self, x, positions, slots, table, q_start, kv_len, mask):
        """ValueError unless the step is one that the buffers of reserve() and the kernels' strides were made for"""
        tokens, batch = x.shape[0], table.shape[0]
        if tokens > self.total_tokens or batch > self.batch:
            raise ValueError("step: %d tokens of %d sequences, reserved are %d of %d" % (tokens, batch, self.total_tokens, self.batch))
        if tuple(x.shape) != (tokens, self.hidden) or x.dtype != self.torch_type or not x.is_contiguous():
            raise ValueError("step: x must be contiguous rows of %d %s, got %s of %s" % (self.hidden, self.torch_type, tuple(x.shape), x.dtype))
        if positions.numel() != tokens or slots.numel() != tokens:
            raise ValueError("step: %d tokens, but %d positions and %d slots" % (tokens, positions.numel(), slots.numel()))
        if q_start.numel() <= batch or kv_len.numel() < batch:
            raise ValueError("step: %d sequences, but q_start has %d elements and kv_len %d" % (batch, q_start.numel(), kv_len.numel()))
        if mask is not None and (mask.dim() != 2 or mask.shape[0] < tokens):
            raise ValueError("step: the mask needs a row of words for each of the %d tokens, got %s" % (tokens, tuple(mask.shape)))

    def step(self, x, positions, slots, table, q_start, kv_len, mask=None, stream=None):
        """x [tokens][hidden] -> x + attention(x) W_o^T.  positions, slots: of every token, its place in the sequence and in the cache; table, q_start,
        kv_len (which counts the tokens of this step), mask: as of tree_attention().  What q_start and kv_len hold stays in device memory and is not looked at here:
        a sequence has at most reserve()'s max_tokens of the step's tokens and max_kv positions (of one with more, the rows of the result mean nothing)."""
        import rocwmma_amd as R

        self._holds(x, positions, slots, table, q_start, kv_len, mask)
        tokens, batch, d, f = x.shape[0], table.shape[0], self.head_dim, self.qkv_heads * self.head_dim
        R.w4_matmul(self.dtype, self.dtype, tokens, f, self.hidden, self.group, x, self.wqkv[1], self.wqkv[2], self.qkv, stream=stream)
        keys, values = self.qkv[:, self.heads:], self.qkv[:, self.heads + self.kv_heads:]
        token, row, slot = (f, d), (self.heads * d, d), (self.kv_heads * d, d)
        R.rope(self.dtype, R.ROPE_HALF, tokens, d, d,
               [R.rope_part(self.qkv, self.q, self.heads, token, row), R.rope_part(keys, self.k, self.kv_heads, token, slot, to_slots=True),
                R.rope_part(values, self.v, self.kv_heads, token, slot, rotate=False, to_slots=True)],
               positions, self.turns, slots=slots, slot_count=self.pages * self.page_size, stream=stream)
        R.tree_attention(self.dtype, batch, tokens, self.heads, self.kv_heads, d, self.q, self.k, self.v, self.attended, table, self.page_size, self.pages,
                         q_start, kv_len, self.max_tokens, self.max_kv, mask=mask, mask_words=0 if mask is None else mask.shape[1],
                         workspace=self.workspace, stream=stream)
        R.w4_matmul(self.dtype, self.dtype, tokens, self.hidden, self.heads * d, self.group, self.attended, self.wo[1], self.wo[2], self.y, c=x, beta=1.0,
                    stream=stream)
        return self.y[:tokens]


def draft(lengths, page_size, pages, seed=0):
    """A step's host arrays (numpy) for `lengths` of (drafted tokens, positions cached before them): random trees, pages in random order.  Tokens
    of one depth share a position; each has a slot of its own behind the prefix."""
    import numpy as np

    rng = np.random.RandomState(seed)
    need = [-(-(n + before) // page_size) for n, before in lengths]
    if sum(need) > pages:
        raise ValueError("draft: %d pages are needed, there are %d" % (sum(need), pages))
    order, at = rng.permutation(pages).astype(np.int32), 0
    table = np.full((len(lengths), max(need)), -1, np.int32)
    most = max(n for n, _ in lengths)
    mask = np.zeros((sum(n for n, _ in lengths), -(-most // 64) * 64), np.uint8)
    positions, slots, row = [], [], 0
    for b, (n, before) in enumerate(lengths):
        table[b, : need[b]] = order[at: at + need[b]]
        at += need[b]
        depth = np.zeros(n, np.int32)
        for j in range(n):
            if j:
                parent = max(0, j - 1 - int(rng.exponential(2.0)))
                depth[j] = depth[parent] + 1
                mask[row + j] = mask[row + parent]
            mask[row + j, j] = 1
        place = before + np.arange(n)
        positions.append(before + depth)
        slots.append(table[b, place // page_size] * page_size + place % page_size)
        row += n
    start = np.concatenate([[0], np.cumsum([n for n, _ in lengths])]).astype(np.int32)
    return {"positions": np.concatenate(positions).astype(np.int32), "slots": np.concatenate(slots).astype(np.int32), "table": table, "q_start": start,
            "kv_len": np.array([n + before for n, before in lengths], np.int32), "mask": np.packbits(mask, axis=1, bitorder="little").view(np.int64)}


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--sequences", type=int, default=8)
    ap.add_argument("--drafted", type=int, default=48)
    ap.add_argument("--cached", type=int, default=4000)
    ap.add_argument("--hidden", type=int, default=4096)
    ap.add_argument("--heads", type=int, default=32)
    ap.add_argument("--kv-heads", type=int, default=8)
    ap.add_argument("--head-dim", type=int, default=128)
    ap.add_argument("--page-size", type=int, default=16)
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--experts", type=int, default=0, help="a feed-forward half of so many experts (0: none)")
    ap.add_argument("--top", type=int, default=4, help="experts of a token")
    ap.add_argument("--width", type=int, default=1024, help="of an expert")
    args = ap.parse_args()

    import torch

    lengths = [(args.drafted, args.cached)] * args.sequences
    pages = args.sequences * -(-(args.drafted + args.cached) // args.page_size)
    layer = AttentionLayer(args.hidden, args.heads, args.kv_heads, args.head_dim, pages, args.page_size)
    layer.k.normal_()
    layer.v.normal_()
    step = {name: torch.from_numpy(a).cuda() for name, a in draft(lengths, args.page_size, pages).items()}
    tokens = args.sequences * args.drafted
    layer.reserve(tokens, args.drafted, args.drafted + args.cached, args.sequences, step["table"].shape[1])
    x = torch.randn(tokens, args.hidden, device="cuda").to(layer.torch_type)
    whole = layer.step
    if args.experts:
        from rocwmma_amd.expert_layer import ExpertLayer

        experts = ExpertLayer(args.hidden, args.width, args.experts, args.top)
        experts.reserve(tokens)

        def whole(x, stream=None, **step):
            return experts.forward(layer.step(x, stream=stream, **step), stream=stream)

    whole(x, **step)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        whole(x, **step, stream=torch.cuda.current_stream())
    for name, fn in (("launched", lambda: whole(x, **step)), ("replayed", graph.replay)):
        for _ in range(20):
            fn()
        begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        begin.record()
        for _ in range(args.steps):
            fn()
        end.record()
        end.synchronize()
        us = begin.elapsed_time(end) * 1e3 / args.steps
        print("%s: %.1f us a step, %d tokens, %.0f tokens/ms" % (name, us, tokens, tokens / us * 1e3))


if __name__ == "__main__":
    main()
