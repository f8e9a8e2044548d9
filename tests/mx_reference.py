"""MXFP4 operators in float64 on the CPU, from their definitions, and bounds on what float32 sums and one
rounding may add.  Matrices are torch tensors."""
from __future__ import annotations

import math

import torch

GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U32 = 2.0 ** -23  # a float32 addition, truncated or rounded


def up(a: int, b: int) -> int:
    return (a + b - 1) // b * b


def code_stride(k: int) -> int:
    return up(k, 256) // 2


def scale_stride(k: int) -> int:
    return up(k, 512) // 32


def encode(x: torch.Tensor):
    """(codes, scales) as uint8 matrices with their padding, block by block."""
    rows, k = x.shape
    v = torch.zeros(rows, up(k, 512), dtype=torch.float64)
    v[:, :k] = x.double()
    b = v.reshape(rows, -1, 32)
    bad = ~torch.isfinite(b).all(2)
    b = torch.where(bad.unsqueeze(2), torch.zeros_like(b), b)
    big = b.abs().amax(2)
    e = torch.where(big > 0, torch.frexp(big).exponent.long() - 3, torch.full_like(big, -127, dtype=torch.long)).clamp(min=-127)
    a = torch.ldexp(b.abs(), -e.unsqueeze(2))
    dist = (a.unsqueeze(3) - GRID).abs()
    best = dist.min(3, keepdim=True).values
    even_first = torch.tensor([0, 2, 4, 6, 1, 3, 5, 7])  # of two nearest the even code
    code = even_first[(dist[..., even_first] == best).to(torch.uint8).argmax(3)]
    code = (code + 8 * torch.signbit(b).long()).reshape(rows, -1)
    keep = 2 * code_stride(k)
    codes = (code[:, :keep:2] + 16 * code[:, 1:keep:2]).to(torch.uint8)
    scales = torch.where(bad, torch.full_like(e, 255), e + 127).to(torch.uint8)
    return codes, scales


def decode(codes: torch.Tensor, scales: torch.Tensor, k: int) -> torch.Tensor:
    rows = codes.shape[0]
    n = torch.stack((codes & 15, codes >> 4), 2).reshape(rows, -1).long()
    v = GRID[n & 7] * torch.where(n >= 8, -1.0, 1.0).double()
    s = scales.long()
    f = torch.where(s == 255, torch.full_like(s, 0, dtype=torch.float64) * math.nan, torch.ldexp(torch.ones_like(s, dtype=torch.float64), s - 127))
    return (v * f.repeat_interleave(32, 1)[:, : v.shape[1]])[:, :k]


def act(g: torch.Tensor, kind: str):
    """Value, slope, and the argument of the exponential inside."""
    if kind == "silu":
        s = torch.sigmoid(g)
        return g * s, s + g * s * torch.sigmoid(-g), g
    r, a = 2.0 * math.sqrt(2.0 / math.pi), 0.044715
    z = r * (g + a * g ** 3)
    s = torch.sigmoid(z)
    return g * s, s + g * s * torch.sigmoid(-z) * r * (1.0 + 3.0 * a * g * g), z


def rounding(y: torch.Tensor, out: str) -> torch.Tensor:
    """Half a unit in the last place of the output type, at most."""
    if out == "f32":
        return y.abs() * 2.0 ** -24 + 2.0 ** -150
    return y.abs() * 2.0 ** -11 + 2.0 ** -25 if out == "f16" else y.abs() * 2.0 ** -8 + 2.0 ** -134


def product(x: torch.Tensor, w: torch.Tensor):
    """x w^T and what float32 sums in any order are off at most."""
    return x @ w.T, x.shape[1] * U32 * (x.abs() @ w.abs().T)


def gated(x, wg, wu, kind):
    """h and its error in float32: sums, the activation's argument (a few roundings of |z|) and the products."""
    (g, eg), (u, eu) = product(x, wg), product(x, wu)
    a, slope, z = act(g, kind)
    ea = 1.2 * eg + a.abs() * (16.0 + 16.0 * z.abs()) * U32  # |act'| < 1.2
    return a * u, ea * u.abs() + a.abs() * eu + ea * eu + 4 * U32 * (a * u).abs()


def gated_gradients(dh, x, wg, wu, kind):
    """dg, du and their errors: as above, and one rounding to bfloat16."""
    (g, eg), (u, eu) = product(x, wg), product(x, wu)
    a, slope, z = act(g, kind)
    ea = 1.2 * eg + a.abs() * (16.0 + 16.0 * z.abs()) * U32
    es = 1.2 * eg + (32.0 + 32.0 * z.abs() * (1.0 + g.abs())) * U32  # |act''| < 1.2
    dg, du = dh * u * slope, dh * a
    edg = dh.abs() * (eu * slope.abs() + (u.abs() + eu) * es) + 8 * U32 * dg.abs()
    edu = dh.abs() * ea + 4 * U32 * du.abs()
    return dg, edg + rounding(dg.abs() + edg, "bf16"), du, edu + rounding(du.abs() + edu, "bf16")
