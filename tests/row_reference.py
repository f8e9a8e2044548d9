"""8-bit matrices and layer norms in float64, from their definitions, and bounds on what their float32 arithmetic may add.  Matrices are
torch tensors, on any device."""
from __future__ import annotations

import torch

DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = 2.0 ** -24  # one rounding to float32, relative


def up(a: int, b: int) -> int:
    return (a + b - 1) // b * b


def encode(x: torch.Tensor):
    """(codes as int8 with their padding, scales as float32).  A quotient of two floats is further than 2^-26 of itself from the middle of
    two whole numbers or right on it, so float64 decides as the definition does."""
    rows, k = x.shape
    v = x.double()
    bad = ~torch.isfinite(v).all(1)
    v = torch.where(bad[:, None], torch.zeros_like(v), v)
    scale = (v.abs().amax(1).float() / torch.tensor(127.0, device=x.device)).clamp(min=2.0**-100)
    codes = torch.zeros(rows, up(k, 128), dtype=torch.int8, device=x.device)
    codes[:, :k] = torch.round(v / scale.double()[:, None]).to(torch.int8)
    return codes, torch.where(bad, torch.full_like(scale, float("nan")), scale)


def decode(codes: torch.Tensor, scales: torch.Tensor, k: int) -> torch.Tensor:
    return codes[:, :k].double() * scales.double()[:, None]


def rounding(y: torch.Tensor, out: str) -> torch.Tensor:
    """Half a unit in the last place of the output type, at most."""
    if out == "f32":
        return y.abs() * 2.0**-24 + 2.0**-150
    return y.abs() * 2.0**-11 + 2.0**-25 if out == "f16" else y.abs() * 2.0**-8 + 2.0**-134


def check(got: torch.Tensor, want: torch.Tensor, error, out: str):
    bound = error + rounding(want.abs() + error, out)
    off = (got.double().to(want.device) - want).abs()
    assert bool((off <= bound).all()), f"off by up to {(off / bound).max().item():.3g} bounds, {int((off > bound).sum())} elements"


def normalised(x: torch.Tensor, eps: float):
    """h = (x - mean) / sqrt(variance + eps), its factor r, and what h is off at most: differences of x and two roundings of the mean
    (each U of itself), a mean and a variance whose sums are `depth` additions deep (at least 64 lanes share a row, 8 values at a time), a
    root and a quotient."""
    v = x.double()
    d = v - v.mean(1, keepdim=True)
    r = 1.0 / torch.sqrt((d * d).mean(1, keepdim=True) + eps)
    h = d * r
    depth = x.shape[1] / 64 + 24
    # (what is centred on is the mean to within depth * U of the values' size, and what is left of that is taken off again)
    left = depth * U * v.abs().mean(1, keepdim=True)
    return h, r, U * ((depth / 2 + 16) * h.abs() + (2 * depth + 8) * r * (d.abs().mean(1, keepdim=True) + left) + 4 * r * left)


def norm(x, gamma, beta, eps):
    """y and its error."""
    h, _, error = normalised(x, eps)
    g = torch.ones_like(h[0]) if gamma is None else gamma.double()
    b = torch.zeros_like(h[0]) if beta is None else beta.double()
    y = h * g + b
    return y, error * g.abs() + U * (2 * (h * g).abs() + y.abs())


def norm_gradients(dy, x, gamma, eps):
    """(dx, dgamma, dbeta), each with its error."""
    h, r, eh = normalised(x, eps)
    rows, n = x.shape
    dy = dy.double()
    g = dy if gamma is None else dy * gamma.double()
    depth = n / 64 + 24
    mean, mean_h = g.mean(1, keepdim=True), (g * h).mean(1, keepdim=True)
    e_mean = (depth + 2) * U * g.abs().mean(1, keepdim=True)
    e_mean_h = (depth + 6) * U * (g * h).abs().mean(1, keepdim=True) + (g.abs() * eh).mean(1, keepdim=True)
    inner = g - mean - h * mean_h
    e_inner = U * (4 * g.abs() + 4 * mean.abs() + 4 * (h * mean_h).abs()) + e_mean + h.abs() * e_mean_h + eh * (mean_h.abs() + e_mean_h)
    e_r = (depth / 2 + 16) * U
    dx = r * inner, r * (e_inner + e_r * inner.abs())
    # rows are added in any order
    dgamma = (dy * h).sum(0), (rows + 2) * U * (dy * h).abs().sum(0) + 1.01 * (dy.abs() * eh).sum(0)
    dbeta = dy.sum(0), (rows + 2) * U * dy.abs().sum(0)
    return dx, dgamma, dbeta
