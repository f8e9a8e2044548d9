"""A norm and an 8-bit linear layer behind it, as a program would use them: training steps with float master weights, then single
tokens from a captured graph.

    python examples/int8_norm_linear.py [--tokens 512] [--hidden 1024] [--out 2816] [--steps 30]

Forward, of the residual stream x [m, hidden] in float with a weight [out, hidden]:
    h = norm(x) gamma + beta     one pass, h leaves it in 8 bits with a scale for each token
    y = h weight^T + bias        weight: 8 bits with a scale for each output channel
The backward pass needs x and the quantised h and no other result of the forward pass.
"""
import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))
import int4linear_amd as lib  # noqa: E402


class Int8:
    """A matrix in 8 bits."""

    def __init__(self, rows: int, k: int):
        self.rows, self.k = rows, k
        self.codes = torch.empty(rows, lib.int8_code_bytes(1, k), dtype=torch.int8, device="cuda")
        self.scales = torch.empty(rows, device="cuda")

    def take(self, x: torch.Tensor) -> "Int8":
        lib.int8_quantize(x, self.codes, self.scales, self.rows, self.k, in_type="f32")
        return self

    def __iter__(self):
        return iter((self.codes, self.scales))


class NormLinear:
    """All buffers for up to `tokens` rows are made once; the calls allocate nothing."""

    def __init__(self, tokens: int, hidden: int, out: int, seed: int = 0):
        self.hidden, self.out = hidden, out
        gen = torch.Generator("cuda").manual_seed(seed)
        self.weight = torch.randn(out, hidden, device="cuda", generator=gen).div_(hidden**0.5)
        self.bias, self.beta = torch.zeros(out, device="cuda"), torch.zeros(hidden, device="cuda")
        self.gamma = torch.ones(hidden, device="cuda")
        self.parameters = (self.weight, self.bias, self.gamma, self.beta)
        self.grads = [torch.empty_like(p) for p in self.parameters]
        self.wq, self.hq = Int8(out, hidden), Int8(tokens, hidden)
        self.y = torch.empty(tokens, out, dtype=torch.bfloat16, device="cuda")
        self.dh = torch.empty(tokens, hidden, dtype=torch.bfloat16, device="cuda")
        self.dx = torch.empty(tokens, hidden, device="cuda")
        self.work = torch.empty(max(lib.int8_linear_backward_bytes(tokens, out, hidden, "f32"),
                                    lib.layer_norm_backward_bytes(tokens, hidden)), dtype=torch.uint8, device="cuda")
        self.quantize()

    def quantize(self) -> None:
        self.wq.take(self.weight)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        m = x.shape[0]
        lib.layer_norm_int8(x, self.gamma, self.beta, *self.hq, m, self.hidden, in_type="f32")
        lib.int8_linear(*self.hq, *self.wq, self.bias, self.y, "bf16", m, self.out, self.hidden)
        return self.y[:m]

    def backward(self, x: torch.Tensor, dy: torch.Tensor) -> torch.Tensor:
        """Gradients of the last forward call's result: into self.grads; returns that of x."""
        m = dy.shape[0]
        dw, dbias, dgamma, dbeta = self.grads
        lib.int8_linear_backward(dy, *self.hq, *self.wq, self.dh, dw, "f32", dbias, self.work, m, self.out, self.hidden)
        lib.layer_norm_backward(self.dh, x, self.gamma, self.dx, dgamma, dbeta, self.work, m, self.hidden, dy_type="bf16", in_type="f32")
        return self.dx[:m]


def train(layer: NormLinear, x: torch.Tensor, target: torch.Tensor, steps: int, rate: float) -> list[float]:
    """Mean squared error by gradient descent; the weight moves by `rate` times its own size along its normalised gradient, the
    vectors by `rate` along theirs."""
    losses = []
    for _ in range(steps):
        error = layer.forward(x).float() - target
        losses.append(error.square().mean().item())
        layer.backward(x, (error / error.numel()).mul_(2 * 2**10).bfloat16())  # (a loss scale: the direction alone is used)
        for p, g in zip(layer.parameters, layer.grads):
            size = p.norm() if p.dim() > 1 else 1.0
            p.sub_(g * (rate * size / g.norm().clamp(min=1e-30)))
        layer.quantize()
    return losses


def main() -> None:
    p = argparse.ArgumentParser()
    for name, value in (("tokens", 512), ("hidden", 1024), ("out", 2816), ("steps", 30)):
        p.add_argument(f"--{name}", type=int, default=value)
    a = p.parse_args()
    lib.init()
    x = torch.randn(a.tokens, a.hidden, device="cuda", generator=torch.Generator("cuda").manual_seed(1)) * 3 + 1
    target = NormLinear(a.tokens, a.hidden, a.out, seed=2).forward(x).float()
    layer = NormLinear(a.tokens, a.hidden, a.out)
    losses = train(layer, x, target, a.steps, 0.02)
    print(f"{a.steps} steps, {a.tokens} tokens: loss {losses[0]:.4f} -> {losses[-1]:.4f}")

    # one token at a time: both calls as one graph
    token = x[:1].clone()
    layer.forward(token)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer.forward(token)
    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    for i in range(a.tokens):
        if i == a.tokens // 2:
            start.record()
        token.copy_(x[i : i + 1])
        graph.replay()
    end.record()
    torch.cuda.synchronize()
    eager = layer.forward(x[-1:].clone()).clone()
    graph.replay()
    print(f"{start.elapsed_time(end) * 1e3 / (a.tokens - a.tokens // 2):.1f} us per token from a graph; same result as eager: "
          f"{torch.equal(y, eager)}")


if __name__ == "__main__":
    main()
