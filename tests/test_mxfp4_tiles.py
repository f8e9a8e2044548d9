"""MXFP4 products at sizes where each tile of the GEMM is the one that runs, several to a workgroup, with an odd and an even number of
stages and ragged ends, against float64; and the streaming kernel in the form it takes for wide weights."""
import math

import pytest
import torch

import int4linear_amd as lib
from tests import line_tiles
from tests import mx_reference as ref
from tests.test_mxfp4 import guarded, untouched

#: workgroups of a tile that run at once on 256 CUs, 4-bit operands
PLACES = {(256, 256): 256, (128, 128): 512, (64, 128): 256, (64, 64): 512}

# (tile, m, n, k): k in stages of 256, begun
LINEAR = [
    ((256, 256), 8190, 8180, 500), ((256, 256), 8190, 8180, 700), ((256, 256), 8190, 4090, 1000), ((256, 256), 8150, 4095, 1150),
    ((256, 256), 8190, 4088, 1300), ((256, 256), 16380, 16376, 250),
    ((128, 128), 4250, 4500, 500), ((128, 128), 4250, 4504, 700), ((128, 128), 4233, 4501, 1000), ((128, 128), 4250, 4504, 1150),
    ((128, 128), 4250, 4500, 1300),
    ((64, 128), 4250, 4504, 250), ((64, 128), 2200, 4204, 500), ((64, 128), 900, 4104, 700), ((64, 128), 900, 4101, 1000), ((64, 128), 890, 4104, 1150),
    ((64, 128), 900, 4100, 1300),
    ((64, 64), 2200, 4204, 250), ((64, 64), 1100, 2104, 700), ((64, 64), 1090, 2101, 1300)]

# n: columns of each of the two matrices
GATED = [
    ((256, 256), 8190, 2040, 1000), ((256, 256), 8150, 2043, 1150), ((256, 256), 8190, 1900, 1300), ((256, 256), 8190, 4088, 700),
    ((128, 128), 4250, 2248, 500), ((128, 128), 4233, 2250, 700), ((128, 128), 4250, 2255, 1000), ((128, 128), 4250, 2100, 1150),
    ((64, 128), 4250, 2250, 250), ((64, 128), 900, 2052, 700), ((64, 128), 890, 2055, 1000), ((64, 128), 900, 2048, 1150)]

STREAMED = [(3, 8200, 300), (5, 8203, 700), (16, 8200, 1300), (17, 8192, 515), (32, 8205, 2050)]


def tiles_of(tile, m, columns):
    return math.ceil(m / tile[0]) * math.ceil(columns / tile[1])


@pytest.mark.parametrize("tile, m, n, k", LINEAR)
def test_the_tile_of_a_linear_case(tile, m, n, k):
    assert line_tiles.tile(m, n, k) == tile and tiles_of(tile, m, n) > PLACES[tile]


@pytest.mark.parametrize("tile, m, n, k", GATED)
def test_the_tile_of_a_gated_case(tile, m, n, k):
    """With h as floats and in MXFP4, whose rows are padded to 256."""
    for columns in (n, ref.up(n, 256)):
        assert line_tiles.tile(m, columns, k, pair=True) == tile and tiles_of(tile, m, 2 * columns) > PLACES[tile]


def test_the_cases_reach_every_tile_with_odd_and_even_numbers_of_stages():
    for cases, tiles in ((LINEAR, line_tiles.TILES), (GATED, line_tiles.TILES[:3])):
        for tile in tiles:
            stages = {math.ceil(k / 256) for t, _, _, k in cases if t == tile}
            assert any(s % 2 for s in stages - {1}) and any(s % 2 == 0 for s in stages), (tile, stages)
            assert {n % 8 == 0 for t, _, n, _ in cases if t == tile} == {True, False}


# ---- on the device --------------------------------------------------------------------------------


def operand(seed, rows, k, low):
    """A random MXFP4 matrix and its values in float64, both on the device.  Every code occurs; a block's scale is 2^low, 2^(low + 1) or
    2^(low + 2), so that a scale read from a neighbouring block or stage shows."""
    gen = torch.Generator("cuda").manual_seed(seed)
    codes = torch.randint(0, 256, (rows, ref.code_stride(k)), dtype=torch.uint8, device="cuda", generator=gen)
    scales = torch.randint(127 + low, 130 + low, (rows, ref.scale_stride(k)), dtype=torch.uint8, device="cuda", generator=gen)
    codes[:, (k + 1) // 2 :] = 0
    if k % 2:
        codes[:, k // 2] &= 15
    scales[:, (k + 31) // 32 :] = 0
    grid = ref.GRID.cuda()
    nibbles = torch.stack((codes & 15, codes >> 4), 2).view(rows, -1)[:, :k].long()
    values = grid[nibbles & 7] * torch.where(nibbles >= 8, -1.0, 1.0).double()
    return (codes, scales), values * torch.exp2(scales.double() - 127.0).repeat_interleave(32, 1)[:, :k]


def check(got, want, error, out):
    bound = error + ref.rounding(want.abs() + error, out)
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), f"off by up to {(off / bound).max().item():.3g} bounds, {int((off > bound).sum())} elements"


@pytest.mark.gpu
@pytest.mark.parametrize("m, n, k", [c[1:] for c in LINEAR] + STREAMED)
def test_linear(gpu, m, n, k):
    """Every term is a multiple of 2^-6 and every sum below 2^24 of them: exact in any order."""
    (xq, x), (wq, w) = operand(m + k, m, k, -2), operand(n + k, n, k, -2)
    bias = torch.randint(-4096, 4096, (n,), generator=torch.Generator("cuda").manual_seed(n), device="cuda").float() / 64
    want = x @ w.T
    assert 36 * 2.0**6 * k < 2.0**24 - 4096
    for out, b in (("bf16", None), ("f32", bias), ("f16", bias)):
        dtype = ref.DTYPE[out]
        raw, y = guarded(m * n * dtype.itemsize)
        lib.mxfp4_linear(*xq, *wq, b, y, out, m, n, k)
        torch.cuda.synchronize()
        assert untouched(raw)
        exact = want if b is None else want + b.double()
        assert torch.equal(y.view(dtype).view(m, n), exact.float().to(dtype)), out


def gated_operands(m, n, k):
    """The gate's and the other projection's results are about 1 in size."""
    low = -1 - round(math.log2(8.6 * math.sqrt(k)))
    return operand(m + k, m, k, -1), operand(n + k, n, k, low), operand(n + k + 1, n, k, low)


def check_quantized(codes, scales, want, error):
    """Each value is one that some h within the error rounds to, and what is behind the rows is zero."""
    m, n = want.shape
    blocks = ref.up(n, 32) // 32
    assert not codes[:, blocks * 16 :].any() and not scales[:, blocks:].any()
    h, slack = (torch.zeros(m, blocks * 32, dtype=torch.float64, device="cuda") for _ in range(2))
    h[:, :n], slack[:, :n] = want, error + 2.0**-140
    size = h.abs().view(m, -1, 32)
    lowest = torch.frexp((size - slack.view(m, -1, 32)).clamp(min=0).amax(2)).exponent.long() - 3
    highest = torch.frexp((size + slack.view(m, -1, 32)).amax(2)).exponent.long() - 3
    s = scales[:, :blocks].long() - 127
    assert bool(((s >= lowest.clamp(min=-127)) & (s <= highest.clamp(min=-127))).all())
    unit = torch.exp2(s.double()).repeat_interleave(32, 1)
    nibbles = torch.stack((codes & 15, codes >> 4), 2).view(m, -1)[:, : blocks * 32].long()
    got = ref.GRID.cuda()[nibbles & 7] * torch.where(nibbles >= 8, -1.0, 1.0).double() * unit
    a = (h.abs() / unit).clamp(max=8)
    step = torch.where(a <= 2, 0.5, torch.where(a <= 4, 1.0, 2.0))
    assert bool(((got - h).abs() <= (step / 2 + (a > 6) * (a - 6).clamp(min=0)) * unit + 2 * slack).all())
    assert not got[:, n:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["silu", "gelu"])
@pytest.mark.parametrize("m, n, k", [c[1:] for c in GATED] + STREAMED)
def test_gated(gpu, m, n, k, kind):
    (xq, x), (gq, wg), (uq, wu) = gated_operands(m, n, k)
    want, error = ref.gated(x, wg, wu, kind)
    for out in ("bf16", "f32", "f16"):
        raw, h = guarded(m * n * ref.DTYPE[out].itemsize)
        lib.mxfp4_gated(*xq, *gq, *uq, h, out, m, n, k, activation=kind)
        torch.cuda.synchronize()
        assert untouched(raw)
        check(h.view(ref.DTYPE[out]).view(m, n), want, error, out)
    raw_c, codes = guarded(lib.mxfp4_code_bytes(m, n))
    raw_s, scales = guarded(lib.mxfp4_scale_bytes(m, n))
    lib.mxfp4_gated_quantized(*xq, *gq, *uq, codes, scales, m, n, k, activation=kind)
    torch.cuda.synchronize()
    assert untouched(raw_c) and untouched(raw_s)
    check_quantized(codes.view(m, -1), scales.view(m, -1), want, error)


@pytest.mark.gpu
@pytest.mark.parametrize("few", [False, True])
@pytest.mark.parametrize("m, n, k", [c[1:] for c in GATED])
def test_gated_backward(gpu, m, n, k, few):
    """`few`: about 32 of the elements of a column of dh are not zero: what rounding may add up to is then so
    little that a single wrong element of dg or du, or one in a wrong place, exceeds it."""
    kind, dw_type = "silu" if k % 100 else "gelu", "f32" if n % 8 else "bf16"
    (xq, x), (gq, wg), (uq, wu) = gated_operands(m, n, k)
    gen = torch.Generator("cuda").manual_seed(k)
    dh = torch.randn(m, n, generator=gen, device="cuda").bfloat16()
    if few:
        dh = torch.where(torch.rand(m, n, generator=gen, device="cuda") < 32 / m, dh, torch.zeros_like(dh))
    dg, edg, du, edu = ref.gated_gradients(dh.double(), x, wg, wu, kind)
    size = lib.mxfp4_gated_backward_bytes(m, n, k)
    raw, work = guarded(size + 256)
    work = work[-work.data_ptr() % 256 :][:size]
    (raw_x, dx), (raw_g, dwg), (raw_u, dwu) = guarded(2 * m * k), *(guarded(ref.DTYPE[dw_type].itemsize * n * k) for _ in range(2))
    lib.mxfp4_gated_backward(dh, *xq, *gq, *uq, dx, dwg, dwu, dw_type, work, m, n, k, activation=kind)
    torch.cuda.synchronize()
    assert untouched(raw) and untouched(raw_x) and untouched(raw_g) and untouched(raw_u)
    (a, ea), (b, eb) = ref.product(dg, wg.T), ref.product(du, wu.T)
    check(dx.view(torch.bfloat16).view(m, k), a + b, 2 * (ea + eb) + 1.01 * (edg @ wg.abs() + edu @ wu.abs()), "bf16")
    for got, d, e in ((dwg, dg, edg), (dwu, du, edu)):
        want, error = ref.product(d.T, x.T)
        check(got.view(ref.DTYPE[dw_type]).view(n, k), want, error + 1.01 * (e.T @ x.abs()), dw_type)


@pytest.mark.gpu
@pytest.mark.parametrize("m, n, k", [(70, 900, 520), (2500, 40, 72)])
def test_results_repeat_whatever_slice_arrives_first(gpu, m, n, k):
    """The products of a small backward pass whose sums are long (dx over 2 n, the weights' over m) are made in slices that meet through
    atomic counters; what is added up, and in which order, is not left to them: the same bits from call to call, with other work on
    the device and on any stream."""
    (xq, _), (gq, _), (uq, _) = gated_operands(m, n, k)
    dh = torch.randn(m, n, generator=torch.Generator("cuda").manual_seed(1), device="cuda").bfloat16()
    first, busy = None, torch.randn(2048, 2048, device="cuda")
    streams = [torch.cuda.current_stream(), torch.cuda.Stream(), torch.cuda.Stream()]
    other = torch.cuda.Stream()
    for i in range(12):
        stream = streams[i % 3]
        stream.wait_stream(torch.cuda.current_stream())
        other.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(other):
            for _ in range(i % 4):
                busy = torch.nn.functional.normalize(busy @ busy)
        with torch.cuda.stream(stream):
            got = [torch.empty(m, k, dtype=torch.bfloat16, device="cuda"), *torch.empty(2, n, k, device="cuda")]
            work = torch.empty(lib.mxfp4_gated_backward_bytes(m, n, k), dtype=torch.uint8, device="cuda")
            lib.mxfp4_gated_backward(dh, *xq, *gq, *uq, *got, "f32", work, m, n, k)
        torch.cuda.synchronize()
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(first, got))
