"""A gated feed-forward block in MXFP4, as a program would use it: training steps with bfloat16 master weights, then
single tokens from a captured graph.

    python examples/mxfp4_feed_forward.py [--tokens 512] [--hidden 1024] [--inner 2816] [--steps 30]

Forward, of x [m, hidden] with weights gate and up [inner, hidden] and down [hidden, inner]:
    h = silu(x gate^T) * (x up^T)     one kernel, h leaves it in MXFP4
    y = h down^T
The backward pass needs the quantised x and h and no other result of the forward pass.
"""
import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))
import int4linear_amd as lib  # noqa: E402


class Mx:
    """A matrix in MXFP4."""

    def __init__(self, rows: int, k: int):
        self.rows, self.k = rows, k
        self.codes = torch.empty(lib.mxfp4_code_bytes(rows, k), dtype=torch.uint8, device="cuda")
        self.scales = torch.empty(lib.mxfp4_scale_bytes(rows, k), dtype=torch.uint8, device="cuda")

    def take(self, x: torch.Tensor) -> "Mx":
        lib.mxfp4_quantize(x, self.codes, self.scales, self.rows, self.k)
        return self

    def __iter__(self):
        return iter((self.codes, self.scales))


class FeedForward:
    """All buffers for up to `tokens` rows are made once; the calls allocate nothing."""

    def __init__(self, tokens: int, hidden: int, inner: int, seed: int = 0):
        self.hidden, self.inner = hidden, inner
        gen = torch.Generator("cuda").manual_seed(seed)
        self.weights = [torch.randn(n, k, device="cuda", generator=gen).div_(k**0.5).bfloat16()
                        for n, k in ((inner, hidden), (inner, hidden), (hidden, inner))]
        self.q = [Mx(*w.shape) for w in self.weights]
        self.xq, self.hq = Mx(tokens, hidden), Mx(tokens, inner)
        self.y = torch.empty(tokens, hidden, dtype=torch.bfloat16, device="cuda")
        self.dh = torch.empty(tokens, inner, dtype=torch.bfloat16, device="cuda")
        self.dx = torch.empty(tokens, hidden, dtype=torch.bfloat16, device="cuda")
        self.grads = [torch.empty(w.shape, device="cuda") for w in self.weights]
        self.work = torch.empty(max(lib.mxfp4_gated_backward_bytes(tokens, inner, hidden),
                                    lib.mxfp4_linear_backward_bytes(tokens, hidden, inner)), dtype=torch.uint8, device="cuda")
        self.quantize()

    def quantize(self) -> None:
        for q, w in zip(self.q, self.weights):
            q.take(w)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        m = x.shape[0]
        lib.mxfp4_quantize(x, *self.xq, m, self.hidden)
        gate, up, down = self.q
        lib.mxfp4_gated_quantized(*self.xq, *gate, *up, *self.hq, m, self.inner, self.hidden)
        lib.mxfp4_linear(*self.hq, *down, None, self.y, "bf16", m, self.hidden, self.inner)
        return self.y[:m]

    def backward(self, dy: torch.Tensor) -> torch.Tensor:
        """Gradients of the last forward call's result: into self.grads; returns that of x."""
        m = dy.shape[0]
        gate, up, down = self.q
        lib.mxfp4_linear_backward(dy, *self.hq, *down, self.dh, self.grads[2], "f32", None, self.work, m, self.hidden, self.inner)
        lib.mxfp4_gated_backward(self.dh, *self.xq, *gate, *up, self.dx, self.grads[0], self.grads[1], "f32", self.work, m,
                                 self.inner, self.hidden)
        return self.dx[:m]


def train(block: FeedForward, x: torch.Tensor, target: torch.Tensor, steps: int, rate: float) -> list[float]:
    """Mean squared error; the weights move by `rate` times their own size along the normalised gradient."""
    masters = [w.float() for w in block.weights]
    losses = []
    for _ in range(steps):
        error = block.forward(x).float() - target
        losses.append(error.square().mean().item())
        block.backward((error / error.numel()).mul_(2 * 2**10).bfloat16())  # (a loss scale: the direction alone is used)
        for master, w, g in zip(masters, block.weights, block.grads):
            master.sub_(g, alpha=rate * float(master.norm() / g.norm().clamp(min=1e-30)))
            w.copy_(master)
        block.quantize()
    return losses


def main() -> None:
    p = argparse.ArgumentParser()
    for name, value in (("tokens", 512), ("hidden", 1024), ("inner", 2816), ("steps", 30)):
        p.add_argument(f"--{name}", type=int, default=value)
    a = p.parse_args()
    lib.init()
    x = torch.randn(a.tokens, a.hidden, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).bfloat16()
    target = FeedForward(a.tokens, a.hidden, a.inner, seed=2).forward(x).float()
    block = FeedForward(a.tokens, a.hidden, a.inner)
    losses = train(block, x, target, a.steps, 0.02)
    print(f"{a.steps} steps, {a.tokens} tokens: loss {losses[0]:.4f} -> {losses[-1]:.4f}")

    # one token at a time: the block's three calls as one graph
    token = x[:1].clone()
    block.forward(token)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = block.forward(token)
    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    for i in range(a.tokens):
        if i == a.tokens // 2:
            start.record()
        token.copy_(x[i : i + 1])
        graph.replay()
    end.record()
    torch.cuda.synchronize()
    eager = block.forward(x[-1:].clone()).clone()
    graph.replay()
    print(f"{start.elapsed_time(end) * 1e3 / (a.tokens - a.tokens // 2):.1f} us per token from a graph; same result as eager: "
          f"{torch.equal(y, eager)}")


if __name__ == "__main__":
    main()
