"""The feed-forward half of a layer with experts, out of this library's operators: a product for the router's logits, the router, three products grouped by
expert (gate and value straight from the tokens' rows, the third back to the layer's width) and the rows' way back to their tokens, with the residual; and all its gradients.

    python -m rocwmma_amd.expert_layer [--tokens 4096] [--hidden 2048] [--width 1024] [--experts 64] [--top 6] [--dtype bf16]

times a forward pass, launched call by call and replayed from a graph, and a forward pass with its gradients, over random weights."""
import argparse


def _on(stream):
    """torch's own kernels on the stream that a call of the library takes (None: the default stream)"""
    import torch

    if stream is None:
        stream = torch.cuda.default_stream()
    return torch.cuda.stream(stream if isinstance(stream, torch.cuda.Stream) else torch.cuda.ExternalStream(getattr(stream, "cuda_stream", stream)))


class ExpertLayer:
    """y = x + sum over the chosen experts e of w_e (silu(x G_e^T) * (x U_e^T)) D_e^T.  forward() and backward() only launch kernels into the buffers of reserve(), so they
    can be recorded into a graph."""

    def __init__(self, hidden, width, experts, top, dtype="bf16", score="softmax", seed=0):
        import torch

        import rocwmma_amd as R

        if hidden % 8 or width % 8:
            raise ValueError("ExpertLayer: hidden and width must be multiples of 8")
        if not 0 < top <= experts:
            raise ValueError("ExpertLayer: of %d experts %d cannot be chosen" % (experts, top))
        self.hidden, self.width, self.experts, self.top = hidden, width, experts, top
        self.dtype, self.torch_type = {"bf16": (R.BF16, torch.bfloat16), "f16": (R.F16, torch.float16)}[dtype]
        self.score = {"softmax": R.ROUTE_SOFTMAX, "sigmoid": R.ROUTE_SIGMOID}[score]
        gen = torch.Generator(device="cuda").manual_seed(seed)
        weights = lambda *shape: torch.empty(shape, dtype=self.torch_type, device="cuda").normal_(0.0, shape[-1] ** -0.5, generator=gen)  # noqa: E731
        self.router = weights(experts, hidden)
        self.gate, self.up, self.down = weights(experts, width, hidden), weights(experts, width, hidden), weights(experts, hidden, width)
        self.tokens = self.trained = 0
        self.kept = None  # tokens of the pass whose buffers backward() can take

    def reserve(self, tokens, training=False):
        """The buffers of passes of up to that many tokens, kept for all of them (a pass that was kept is gone)."""
        import torch

        import rocwmma_amd as R

        empty = lambda *shape, dtype=self.torch_type: torch.empty(shape, dtype=dtype, device="cuda")  # noqa: E731
        rows, i32, f32 = tokens * self.top, torch.int32, torch.float32
        self.tokens, self.trained, self.kept = tokens, tokens if training else 0, None
        self.logits, self.y = empty(tokens, self.experts), empty(tokens, self.hidden)
        self.weights, self.chosen, self.place = empty(tokens, self.top, dtype=f32), empty(tokens, self.top, dtype=i32), empty(tokens, self.top, dtype=i32)
        self.source, self.offsets = empty(rows, dtype=i32), empty(self.experts + 1, dtype=i32)
        self.u, self.h, self.out = empty(rows, self.width), empty(rows, self.width), empty(rows, self.hidden)
        need = [R.route_workspace_bytes(tokens, self.experts, self.top)]
        for m in {min(1 << i, tokens) for i in range(tokens.bit_length() + 1)}:  # (few tokens may make use of more than many)
            for m_, n, k, groups in ((m, self.experts, self.hidden, 1), (m * self.top, self.width, self.hidden, self.experts), (m * self.top, self.hidden, self.width, self.experts)):
                need.append(R.linear_workspace_bytes(R.linear_args(self.dtype, self.dtype, m_, n, k, self.router, self.router, self.router, groups=groups,
                                                                   offsets=self.offsets if groups > 1 else None)))
        if training:
            self.z, self.xs = empty(rows, self.width), empty(rows, self.hidden)
            self.dout = empty(rows, self.hidden)
            # the parts of dx: the rows of both products and the router's; and which of them are of which token, so that one sum rounds them once
            self.parts, self.terms = empty(2 * rows + tokens, self.hidden), empty(tokens, 2 * self.top + 1, dtype=i32)
            self.dxs, self.dxs2, self.dx_router = self.parts[:rows], self.parts[rows: 2 * rows], self.parts[2 * rows:]
            self.terms[:, -1] = torch.arange(2 * rows, 2 * rows + tokens, dtype=i32, device="cuda")
            self.dh, self.dz, self.du = empty(rows, self.width), empty(rows, self.width), empty(rows, self.width)
            self.dweights, self.dlogits, self.dx = empty(tokens, self.top, dtype=f32), empty(tokens, self.experts), empty(tokens, self.hidden)
            self.gradients = {name: torch.empty_like(getattr(self, name)) for name in ("router", "gate", "up", "down")}
            for n, k, groups, m in ((self.hidden, self.width, self.experts, rows), (self.width, self.hidden, self.experts, rows), (self.experts, self.hidden, 1, tokens)):
                a = R.linear_backward_args(self.dtype, self.dtype, m, n, k, self.xs, self.xs, self.xs, dx=self.xs, dw=self.xs, groups=groups, offsets=self.offsets if groups > 1 else None)
                need.append(R.linear_backward_workspace_bytes(a))
        self.workspace = empty(max(need + [16]), dtype=torch.uint8)

    def _rows(self, x, most):
        tokens = x.shape[0]
        if x.dim() != 2 or x.shape[1] != self.hidden or x.dtype != self.torch_type or not x.is_contiguous():
            raise ValueError("ExpertLayer: rows of %d %s are needed, contiguous, got %s of %s" % (self.hidden, self.torch_type, tuple(x.shape), x.dtype))
        if tokens > most:
            raise ValueError("ExpertLayer: %d tokens, reserved are %d" % (tokens, most))
        return tokens, tokens * self.top

    def forward(self, x, keep=False, stream=None):
        """x [tokens][hidden] -> y.  keep: what backward() needs stays in the buffers (reserved with training=True) until the next pass."""
        import rocwmma_amd as R

        t, e = self.dtype, self.experts
        tokens, rows = self._rows(x, self.trained if keep else self.tokens)
        self.kept = None  # (every pass writes to the buffers of the last one)
        grouped = dict(groups=e, offsets=self.offsets, workspace=self.workspace, stream=stream)
        R.linear(t, t, tokens, e, self.hidden, x, self.router, self.logits, workspace=self.workspace, stream=stream)
        R.route(t, tokens, e, self.top, self.logits, self.weights, self.chosen, self.place, self.source, self.offsets, score=self.score, chosen_only=True, workspace=self.workspace,
                stream=stream)
        R.linear(t, t, rows, self.width, self.hidden, x, self.up, self.u, source=self.source, x_rows=tokens, **grouped)
        R.linear(t, t, rows, self.width, self.hidden, x, self.gate, self.h, activation=R.ACT_SILU, gate=self.u, z=self.z if keep else None, source=self.source, x_rows=tokens, **grouped)
        R.linear(t, t, rows, self.hidden, self.width, self.h, self.down, self.out, **grouped)
        R.combine(t, tokens, self.top, self.hidden, self.out, rows, self.place, self.y, weights=self.weights, c=x, stream=stream)
        self.kept = tokens if keep else None
        return self.y[:tokens]

    def backward(self, x, dy, stream=None):
        """dL/dx for dL/dy of the forward(x, keep=True) before it, with no other pass between (of recorded passes a replay is one, which is not seen here); the weights' gradients are left
        in self.gradients."""
        import torch

        import rocwmma_amd as R

        t, e, g = self.dtype, self.experts, self.gradients
        tokens, rows = self._rows(x, self.trained)
        if dy.shape != x.shape or dy.dtype != x.dtype or not dy.is_contiguous():
            raise ValueError("ExpertLayer: dy must be as x, got %s of %s" % (tuple(dy.shape), dy.dtype))
        if self.kept != tokens:
            raise ValueError("ExpertLayer: backward() of %d tokens needs the forward(keep=True) of them just before, %s" % (
                tokens, "the buffers hold none" if self.kept is None else "it was of %d" % self.kept))
        grouped = dict(groups=e, offsets=self.offsets, workspace=self.workspace, stream=stream)
        R.dispatch(t, tokens, self.top, self.hidden, dy, self.dout, rows, self.place, weights=self.weights, values=self.out, dweights=self.dweights, stream=stream)
        R.dispatch(t, tokens, self.top, self.hidden, x, self.xs, rows, self.place, stream=stream)
        R.linear_backward(t, t, rows, self.hidden, self.width, self.dout, self.h, self.down, dx=self.dh, dw=g["down"], **grouped)
        R.linear_backward(t, t, rows, self.width, self.hidden, self.dh, self.xs, self.gate, dx=self.dxs, dw=g["gate"], z=self.z, activation=R.ACT_SILU, gate=self.u, dgate=self.du,
                          dz=self.dz, **grouped)
        R.linear_backward(t, t, rows, self.width, self.hidden, self.du, self.xs, self.up, dx=self.dxs2, dw=g["up"], **grouped)
        R.route_backward(t, tokens, e, self.top, self.logits, self.chosen, self.dweights, self.dlogits, score=self.score, chosen_only=True, stream=stream)
        R.linear_backward(t, t, tokens, e, self.hidden, self.dlogits, x, self.router, dx=self.dx_router, dw=g["router"], workspace=self.workspace, stream=stream)
        # the residual's gradient, the rows' of both products, the router's
        with _on(stream):
            place, terms = self.place[:tokens], self.terms[:tokens]
            terms[:, : self.top].copy_(place)
            torch.add(place, len(self.dxs), out=terms[:, self.top: 2 * self.top])
        R.combine(t, tokens, 2 * self.top + 1, self.hidden, self.parts, len(self.parts), self.terms, self.dx, c=dy, stream=stream)
        return self.dx[:tokens]


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--tokens", type=int, default=4096)
    ap.add_argument("--hidden", type=int, default=2048)
    ap.add_argument("--width", type=int, default=1024)
    ap.add_argument("--experts", type=int, default=64)
    ap.add_argument("--top", type=int, default=6)
    ap.add_argument("--dtype", choices=["bf16", "f16"], default="bf16")
    ap.add_argument("--steps", type=int, default=50)
    args = ap.parse_args()

    import torch

    layer = ExpertLayer(args.hidden, args.width, args.experts, args.top, args.dtype)
    layer.reserve(args.tokens, training=True)
    x, dy = (torch.randn(args.tokens, args.hidden, device="cuda").to(layer.torch_type) for _ in range(2))
    layer.forward(x)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        layer.forward(x, stream=torch.cuda.current_stream())

    def train():
        layer.forward(x, keep=True)
        layer.backward(x, dy)

    products = 6.0 * args.tokens * args.top * args.hidden * args.width  # operations of the experts' three products
    for name, fn, times in (("forward, launched", lambda: layer.forward(x), 1), ("forward, replayed", graph.replay, 1), ("forward and backward", train, 3)):
        for _ in range(5):
            fn()
        begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        begin.record()
        for _ in range(args.steps):
            fn()
        end.record()
        end.synchronize()
        us = begin.elapsed_time(end) * 1e3 / args.steps
        print("%s: %.1f us, %d tokens, %.0f TFLOP/s of the experts' products" % (name, us, args.tokens, times * products / us / 1e6))


if __name__ == "__main__":
    main()
