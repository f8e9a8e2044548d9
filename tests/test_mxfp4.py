"""MXFP4 operators: refusals and sizes (CPU), and their results on the device against float64."""
import math
from pathlib import Path

import pytest
import torch

import int4linear_amd as lib
from int4linear_amd import _lib
from tests import mx_reference as ref

OK, SHAPE, NULL, ALIGN, UNSUPPORTED, SCRATCH = 0, 1, 2, 3, 5, 7


# ---- without a device ---------------------------------------------------------------------------


@pytest.mark.parametrize("rows, k", [(0, 0), (1, 1), (3, 256), (3, 257), (5, 512), (7, 513), (2, 14336), (1 << 20, 1 << 20)])
def test_sizes(rows, k):
    assert lib.mxfp4_code_bytes(rows, k) == rows * ((k + 255) // 256) * 128
    assert lib.mxfp4_scale_bytes(rows, k) == rows * ((k + 511) // 512) * 16
    assert lib.mxfp4_code_bytes(-1, k) == 0 and lib.mxfp4_scale_bytes(rows, -1) == 0


def test_refusals():
    L = _lib.load()
    A, odd = 4096, 4104  # an aligned and a misaligned address; nothing is read
    q = L.int4linear_mxfp4_quantize
    assert q(A, 3, 8, A, A, -1, 8, None) == SHAPE and q(A, 3, 7, A, A, 1, 8, None) == SHAPE
    assert q(A, 0, 8, A, A, 1, 8, None) == UNSUPPORTED and q(A, 4, 8, A, A, 1, 8, None) == UNSUPPORTED
    assert q(None, 3, 8, A, A, 1, 8, None) == NULL and q(A, 3, 8, None, A, 1, 8, None) == NULL
    assert q(A, 3, 8, odd, A, 1, 8, None) == ALIGN and q(A, 3, 8, A, odd, 1, 8, None) == ALIGN
    assert q(A + 1, 3, 8, A, A, 1, 8, None) == ALIGN and q(A + 2, 1, 8, A, A, 1, 8, None) == ALIGN
    assert q(A, 3, 1 << 31, A, A, 1, (1 << 30) + 1, None) == UNSUPPORTED
    assert q(None, 3, 0, None, None, 5, 0, None) == OK and q(None, 3, 8, None, None, 0, 8, None) == OK
    d = L.int4linear_mxfp4_dequantize
    assert d(A, A, A, 3, 8, 1, -8, None) == SHAPE and d(A, A, A, 9, 8, 1, 8, None) == UNSUPPORTED
    assert d(A, A, None, 3, 8, 1, 8, None) == NULL and d(A, odd, A, 3, 8, 1, 8, None) == ALIGN
    lin = L.int4linear_mxfp4_linear
    assert lin(A, A, A, A, None, A, 3, 1, -1, 8, None) == SHAPE and lin(A, A, A, A, None, A, 0, 1, 1, 8, None) == UNSUPPORTED
    assert lin(A, A, A, A, None, None, 3, 1, 1, 8, None) == NULL and lin(A, None, A, A, None, A, 3, 1, 1, 8, None) == NULL
    assert lin(A, A, odd, A, None, A, 3, 1, 1, 8, None) == ALIGN and lin(A, A, A, A, A + 2, A, 3, 1, 1, 8, None) == ALIGN
    assert lin(A, A, A, A, None, odd, 3, 1, 1, 8, None) == ALIGN
    assert lin(None, None, None, None, None, None, 3, 0, 5, 8, None) == OK and lin(None, None, None, None, None, None, 3, 5, 0, 8, None) == OK
    g = L.int4linear_mxfp4_gated
    assert g(A, A, A, A, A, A, 2, A, 3, 1, 1, 8, None) == UNSUPPORTED and g(A, A, A, A, A, A, 0, A, 0, 1, 1, 8, None) == UNSUPPORTED
    assert g(A, A, A, A, None, A, 0, A, 3, 1, 1, 8, None) == NULL and g(A, A, A, A, A, odd, 1, A, 3, 1, 1, 8, None) == ALIGN
    gq = L.int4linear_mxfp4_gated_quantized
    assert gq(A, A, A, A, A, A, -1, A, A, 1, 1, 8, None) == UNSUPPORTED and gq(A, A, A, A, A, A, 0, A, None, 1, 1, 8, None) == NULL
    assert gq(A, A, A, A, A, A, 0, odd, A, 1, 1, 8, None) == ALIGN and gq(A, A, A, A, A, A, 0, A, A, -1, 1, 8, None) == SHAPE


def test_refusals_of_the_gradients():
    L = _lib.load()
    A, odd, big = 4096, 4104, 1 << 40
    b = L.int4linear_mxfp4_linear_backward
    need = lib.mxfp4_linear_backward_bytes(10, 20, 30)
    assert need > 0 and need % 256 == 0 and lib.mxfp4_linear_backward_bytes(-1, 2, 3) == 0
    assert b(A, A, A, A, A, A, A, 3, A, A, need - 1, 10, 20, 30, None) == SCRATCH
    assert b(A, A, A, A, A, A, A, 3, A, None, need, 10, 20, 30, None) == NULL
    assert b(A, A, A, A, A, A, A, 3, A, A + 16, need, 10, 20, 30, None) == ALIGN
    assert b(None, A, A, A, A, A, A, 3, A, A, big, 10, 20, 30, None) == NULL
    assert b(A, A, A, A, None, A, A, 3, A, A, big, 10, 20, 30, None) == NULL
    assert b(odd, A, A, A, A, A, A, 3, A, A, big, 10, 20, 30, None) == ALIGN
    assert b(A, A, A, A, A, A, A, 2, A, A, big, 10, 20, 30, None) == UNSUPPORTED
    assert b(A, A, A, A, A, A, A, 3, A, A, big, 10, -20, 30, None) == SHAPE
    assert b(A, A, A, A, A, None, None, 3, None, None, 0, 10, 20, 30, None) == OK   # nothing is wanted
    gb = L.int4linear_mxfp4_gated_backward
    need = lib.mxfp4_gated_backward_bytes(10, 20, 30)
    assert need > 0 and need % 256 == 0 and lib.mxfp4_gated_backward_bytes(1, 2, -3) == 0
    assert gb(A, A, A, A, A, A, A, 0, A, A, A, 3, A, need - 1, 10, 20, 30, None) == SCRATCH
    assert gb(A, A, A, A, A, A, A, 0, A, A, None, 3, A, need, 10, 20, 30, None) == NULL
    assert gb(A, A, A, A, A, A, A, 5, A, A, A, 3, A, need, 10, 20, 30, None) == UNSUPPORTED
    assert gb(A, A, A, A, A, A, A, 0, A, A, A, 2, A, need, 10, 20, 30, None) == UNSUPPORTED
    assert gb(A, A, A, A, A, A, A, 0, A, A, odd, 3, A, need, 10, 20, 30, None) == ALIGN
    assert gb(A, A, A, A, A, A, A, 0, None, None, None, 3, None, 0, 10, 20, 30, None) == OK


def test_the_reference_gradients_against_differences():
    """The formulas that the device's gradients are compared with, against central differences."""
    gen = torch.Generator().manual_seed(5)
    m, n, k = 5, 7, 11
    dh, x, wg, wu = (torch.randn(*s, generator=gen, dtype=torch.float64) for s in ((m, n), (m, k), (n, k), (n, k)))
    for kind in ("silu", "gelu"):
        dg, _, du, _ = ref.gated_gradients(dh, x, wg, wu, kind)
        grads = (dg @ wg + du @ wu, dg.T @ x, du.T @ x)
        for which, grad in enumerate(grads):
            v = torch.randn(grad.shape, generator=gen, dtype=torch.float64)
            eps = 1e-5
            values = []
            for sign in (eps, -eps):
                args = [x, wg, wu]
                args[which] = args[which] + sign * v
                values.append((dh * ref.gated(*args, kind)[0]).sum())
            assert math.isclose((values[0] - values[1]).item() / (2 * eps), (grad * v).sum().item(), rel_tol=1e-7)


# ---- on the device --------------------------------------------------------------------------------

GUARD = 4096


def guarded(nbytes):
    """A device buffer between two guard zones, everything 0xA5."""
    raw = torch.full((nbytes + 2 * GUARD,), 0xA5, dtype=torch.uint8, device="cuda")
    return raw, raw[GUARD : GUARD + nbytes]


def untouched(raw):
    return bool((raw[:GUARD] == 0xA5).all()) and bool((raw[-GUARD:] == 0xA5).all())


def quantize(x, k=None, kind="bf16"):
    """A device matrix -> guarded codes and scales, checked for writes outside."""
    rows, ld = x.shape[0], x.stride(0)
    k = x.shape[1] if k is None else k
    raw_c, codes = guarded(lib.mxfp4_code_bytes(rows, k))
    raw_s, scales = guarded(lib.mxfp4_scale_bytes(rows, k))
    lib.mxfp4_quantize(x, codes, scales, rows, k, in_type=kind, ld=ld)
    torch.cuda.synchronize()
    assert untouched(raw_c) and untouched(raw_s)
    return codes.view(rows, -1), scales.view(rows, -1)


def matrix(seed, rows, k, scale=1.0, wide=6):
    """A random MXFP4 matrix: its operands on the device and its values in float64.  Block scales vary by
    2^`wide`, so that sums meet terms of very different size."""
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, k, generator=gen, dtype=torch.float64) * scale
    x = x * torch.exp2(-wide * torch.rand(rows, ref.up(k, 32) // 32, generator=gen, dtype=torch.float64)).repeat_interleave(32, 1)[:, :k]
    codes, scales = ref.encode(x)
    return (codes.cuda(), scales.cuda()), ref.decode(codes, scales, k)


SPECIAL = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, 6.0, 7.9, -0.25, -0.75, -5.0, -7.5, 0.2499, 0.2501, 4.9999, 5.0001, -0.0, 0.0]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows, k, ld", [(1, 1, 1), (1, 31, 31), (2, 32, 40), (3, 33, 33), (5, 255, 256), (4, 256, 256), (7, 513, 515),
                                         (33, 1000, 1001), (16, 4096, 4096), (130, 777, 784)])
def test_quantize_is_the_formula(gpu, kind, rows, k, ld):
    gen = torch.Generator().manual_seed(rows * 1000 + k)
    x = torch.randn(rows, ld, generator=gen) * torch.exp2(20 * torch.rand(rows, 1, generator=gen) - 10)
    x = x.to(ref.DTYPE[kind])
    if k >= 64:
        x[0, 32 : 32 + len(SPECIAL)] = torch.tensor(SPECIAL).to(x.dtype)  # ties and ends of the grid
        x[0, 32 + len(SPECIAL) : 64] = 1.0
        x[rows - 1, :32] = 0.0
    codes, scales = quantize(x.cuda(), k, kind)
    want_c, want_s = ref.encode(x[:, :k])
    assert torch.equal(scales.cpu(), want_s) and torch.equal(codes.cpu(), want_c)
    for out in ("f32", "f16", "bf16"):
        raw, y = guarded(rows * ld * ref.DTYPE[out].itemsize)
        lib.mxfp4_dequantize(codes, scales, y, rows, k, out_type=out, ld=ld)
        y = y.view(ref.DTYPE[out]).view(rows, ld).cpu()
        assert untouched(raw) and torch.equal(y[:, :k], ref.decode(want_c, want_s, k).to(ref.DTYPE[out]))
        assert (y[:, k:].contiguous().view(torch.uint8) == 0xA5).all()


@pytest.mark.gpu
def test_quantize_every_exponent_and_every_bf16(gpu):
    """Blocks whose largest value runs over all floats' exponents, denormals among them, and every finite
    bfloat16 next to a largest value of its own size."""
    e = torch.arange(-149, 128).double()
    x = torch.zeros(277, 64, dtype=torch.float32)
    x[:, 0], x[:, 1], x[:, 2], x[:, 40] = torch.exp2(e), -0.75 * torch.exp2(e), 0.3 * torch.exp2(e), 1.5 * torch.exp2(e - 1)
    codes, scales = quantize(x.cuda(), 64, "f32")
    want_c, want_s = ref.encode(x)
    assert torch.equal(scales.cpu(), want_s) and torch.equal(codes.cpu(), want_c)
    bits = torch.arange(0x10000, dtype=torch.int32)
    v = (bits << 16).view(torch.float32)
    v = v[torch.isfinite(v)].view(-1, 32)
    codes, scales = quantize(v.bfloat16().cuda(), 32, "bf16")
    want_c, want_s = ref.encode(v)
    assert torch.equal(scales.cpu(), want_s) and torch.equal(codes.cpu(), want_c)


@pytest.mark.gpu
def test_infinities_and_nans_make_their_block_nan_and_no_other(gpu):
    x = torch.ones(4, 96)
    x[0, 40], x[1, 0], x[2, 95] = math.inf, -math.inf, math.nan
    (codes, scales), y = quantize(x.cuda(), 96, "f32"), torch.empty(4, 96, device="cuda")
    assert scales.cpu()[:, :3].tolist() == [[125, 255, 125], [255, 125, 125], [125, 125, 255], [125, 125, 125]]
    lib.mxfp4_dequantize(codes, scales, y, 4, 96, out_type="f32")
    assert torch.equal(torch.isnan(y.cpu()), (torch.tensor([[0, 1, 0], [1, 0, 0], [0, 0, 1], [0, 0, 0]]) == 1).repeat_interleave(32, 1))
    # ... and a product its rows
    z = torch.empty(4, 4, device="cuda")
    lib.mxfp4_linear(codes, scales, codes, scales, None, z, "f32", 4, 4, 96)
    want = torch.full((4, 4), math.nan)
    want[3, 3] = 96.0
    assert torch.equal(torch.isnan(z.cpu()), torch.isnan(want)) and z[3, 3].item() == 96.0


@pytest.mark.gpu
def test_quantize_of_a_view_that_is_aligned_to_its_element_only(gpu):
    x = torch.randn(9, 300, generator=torch.Generator().manual_seed(2)).bfloat16()
    on = x.cuda()
    codes, scales = quantize(on[2:, 7:], 290)
    want = ref.encode(x[2:, 7:297])
    assert torch.equal(codes.cpu(), want[0]) and torch.equal(scales.cpu(), want[1])


def check(got, want, error, out):
    bound = error + ref.rounding(want.abs() + error, out)
    off = (got.double().cpu() - want).abs()
    assert bool((off <= bound).all()), f"off by up to {(off / bound).max().item():.3g} bounds"


LINEAR = [(1, 1, 1), (1, 100, 64), (2, 33, 257), (5, 64, 512), (16, 130, 1000), (17, 256, 256), (31, 31, 31), (32, 500, 4096), (33, 129, 515),
          (64, 96, 768), (65, 200, 300), (128, 128, 256), (129, 257, 511), (200, 300, 1024), (257, 513, 640), (300, 700, 2050)]


@pytest.mark.gpu
@pytest.mark.parametrize("m, n, k", LINEAR)
@pytest.mark.parametrize("out", ["f32", "f16", "bf16"])
def test_linear(gpu, m, n, k, out):
    (xq, x), (wq, w) = matrix(m + 7 * n, m, k), matrix(n + k, n, k)
    bias = torch.randn(n, generator=torch.Generator().manual_seed(3))
    want, error = ref.product(x, w)
    for b in (None, bias):
        raw, y = guarded(m * n * ref.DTYPE[out].itemsize)
        lib.mxfp4_linear(*xq, *wq, None if b is None else b.cuda(), y, out, m, n, k)
        torch.cuda.synchronize()
        assert untouched(raw)
        total = want if b is None else want + b.double()
        check(y.view(ref.DTYPE[out]).view(m, n), total, error + ref.U32 * total.abs(), out)


@pytest.mark.gpu
def test_linear_without_k_and_without_rows(gpu):
    bias, y = torch.randn(40, device="cuda"), torch.full((3, 40), 7.0, device="cuda")
    lib.mxfp4_linear(None, None, None, None, bias, y, "f32", 3, 40, 0)
    assert torch.equal(y, bias.expand(3, 40))
    lib.mxfp4_linear(None, None, None, None, None, y, "f32", 3, 40, 0)
    assert not y.any()
    lib.mxfp4_linear(None, None, None, None, None, y, "f32", 0, 40, 8)


@pytest.mark.gpu
def test_integers_come_out_exactly(gpu):
    """Small integers with scales of 1: every sum is an exact float, whatever the order of k."""
    gen = torch.Generator().manual_seed(11)
    k = 777
    x, w = (torch.randint(-4, 5, (r, k), generator=gen).double() for r in (70, 90))
    x[:, ::32], w[:, ::32] = 4.0, -4.0  # scales of 1
    (xc, xs), (wc, ws) = ref.encode(x), ref.encode(w)
    y = torch.empty(70, 90, device="cuda")
    lib.mxfp4_linear(xc.cuda(), xs.cuda(), wc.cuda(), ws.cuda(), None, y, "f32", 70, 90, k)
    assert torch.equal(ref.decode(xc, xs, k), x) and torch.equal(y.double().cpu(), x @ w.T)


GATED = [(1, 64, 256), (1, 33, 40), (3, 100, 300), (16, 260, 512), (33, 64, 1000), (64, 500, 256), (70, 129, 257), (130, 300, 768), (257, 200, 520)]


@pytest.mark.gpu
@pytest.mark.parametrize("m, n, k", GATED)
@pytest.mark.parametrize("kind", ["silu", "gelu"])
def test_gated(gpu, m, n, k, kind):
    (xq, x), (gq, wg), (uq, wu) = matrix(m, m, k), matrix(n, n, k, 2.0 / math.sqrt(k), 2), matrix(k, n, k, 2.0 / math.sqrt(k), 2)
    want, error = ref.gated(x, wg, wu, kind)
    for out in ("f32", "f16", "bf16"):
        raw, h = guarded(m * n * ref.DTYPE[out].itemsize)
        lib.mxfp4_gated(*xq, *gq, *uq, h, out, m, n, k, activation=kind)
        torch.cuda.synchronize()
        assert untouched(raw)
        check(h.view(ref.DTYPE[out]).view(m, n), want, error, out)
    # in MXFP4: each value is one that some h within the error rounds to
    raw_c, codes = guarded(lib.mxfp4_code_bytes(m, n))
    raw_s, scales = guarded(lib.mxfp4_scale_bytes(m, n))
    lib.mxfp4_gated_quantized(*xq, *gq, *uq, codes, scales, m, n, k, activation=kind)
    torch.cuda.synchronize()
    assert untouched(raw_c) and untouched(raw_s)
    codes, scales = codes.view(m, -1).cpu(), scales.view(m, -1).cpu()
    blocks = ref.up(n, 32) // 32
    assert not codes[:, blocks * 16 :].any() and not scales[:, blocks:].any()
    padded = torch.zeros(m, blocks * 32, dtype=torch.float64)
    padded[:, :n], slack = want, torch.zeros(m, blocks * 32, dtype=torch.float64)
    slack[:, :n] = error + 2.0 ** -140
    top = padded.abs().view(m, -1, 32)
    lowest = torch.frexp((top - slack.view(m, -1, 32)).clamp(min=0).amax(2)).exponent.long() - 3
    highest = torch.frexp((top + slack.view(m, -1, 32)).amax(2)).exponent.long() - 3
    s = scales[:, :blocks].long() - 127
    assert bool(((s >= lowest.clamp(min=-127)) & (s <= highest.clamp(min=-127))).all())
    unit = torch.ldexp(torch.ones(m, blocks, dtype=torch.float64), s).repeat_interleave(32, 1)
    got = ref.decode(codes, scales, 32 * blocks)
    a = (padded.abs() / unit).clamp(max=8)
    step = torch.where(a <= 2, 0.5, torch.where(a <= 4, 1.0, 2.0))
    assert bool(((got - padded).abs() <= (step / 2 + (a > 6) * (a - 6).clamp(min=0)) * unit + 2 * slack).all())
    assert torch.equal(got[:, n:], torch.zeros(m, 32 * blocks - n, dtype=torch.float64))


BACKWARD = [(70, 5, 40), (75, 15, 40), (1000, 64, 64), (2500, 40, 72), (64, 2000, 64), (700, 130, 40), (40, 900, 520), (1, 1, 1), (1, 64, 256), (3, 65, 40), (16, 128, 300), (64, 64, 64), (65, 130, 257), (100, 300, 100), (130, 257, 515), (192, 320, 512)]


@pytest.mark.gpu
@pytest.mark.parametrize("m, n, k", BACKWARD)
@pytest.mark.parametrize("dw_type", ["f32", "bf16"])
def test_linear_backward(gpu, m, n, k, dw_type):
    (xq, x), (wq, w) = matrix(m + 1, m, k), matrix(n + 2, n, k)
    dy = torch.randn(m, n, generator=torch.Generator().manual_seed(m * n)).bfloat16()
    raw, work = guarded(lib.mxfp4_linear_backward_bytes(m, n, k) + 256)
    work = work[-work.data_ptr() % 256 :][: lib.mxfp4_linear_backward_bytes(m, n, k)]
    raw_x, dx = guarded(2 * m * k)
    raw_w, dw = guarded(ref.DTYPE[dw_type].itemsize * n * k)
    raw_b, db = guarded(4 * n)
    lib.mxfp4_linear_backward(dy.cuda(), *xq, *wq, dx, dw, dw_type, db, work, m, n, k)
    torch.cuda.synchronize()
    assert untouched(raw) and untouched(raw_x) and untouched(raw_w) and untouched(raw_b)
    d = dy.double()
    check(dx.view(torch.bfloat16).view(m, k), *ref.product(d, w.T), "bf16")
    check(dw.view(ref.DTYPE[dw_type]).view(n, k), *ref.product(d.T, x.T), dw_type)
    check(db.view(torch.float32), d.sum(0), m * ref.U32 * d.abs().sum(0), "f32")
    # each output alone is the same
    parts = (torch.empty_like(dx), torch.empty_like(dw), torch.empty_like(db))
    for i in range(3):
        args = [p if j == i else None for j, p in enumerate(parts)]
        lib.mxfp4_linear_backward(dy.cuda(), *xq, *wq, args[0], args[1], dw_type, args[2], work, m, n, k)
    assert all(torch.equal(a, b) for a, b in zip(parts, (dx, dw, db)))


@pytest.mark.gpu
def test_gradients_read_every_scale_and_code(gpu):
    """dx = I w: every value that a code and a scale from 2^-127 to 2^125 stand for is a bfloat16 number and comes out."""
    n = 253
    codes, scales = torch.zeros(n, 128, dtype=torch.uint8), torch.zeros(n, 16, dtype=torch.uint8)
    codes[:, :16] = torch.tensor([16 * (i % 8 * 2 + 1) + i % 8 * 2 for i in range(16)], dtype=torch.uint8)
    scales[:, 0] = torch.arange(n)
    size = lib.mxfp4_linear_backward_bytes(n, n, 32)
    work, dx = torch.empty(size, dtype=torch.uint8, device="cuda"), torch.empty(n, 32, dtype=torch.bfloat16, device="cuda")
    args = (torch.eye(n, dtype=torch.bfloat16).cuda(), codes.cuda(), scales.cuda(), codes.cuda(), scales.cuda())
    lib.mxfp4_linear_backward(*args, dx, None, "f32", None, work, n, n, 32)
    assert torch.equal(dx.cpu().double(), ref.decode(codes, scales, 32))
    args[4][7, 0] = 255
    lib.mxfp4_linear_backward(*args, dx, None, "f32", None, work, n, n, 32)
    assert bool(torch.isnan(dx).all())


@pytest.mark.gpu
@pytest.mark.parametrize("m, n, k", [(6390, 4090, 4860), (6390, 2800, 2810), (2810, 6390, 2800), (4096, 2048, 2816), (1000, 2000, 1990), (1030, 2000, 1990)])
def test_gradients_of_large_layers_with_integers(gpu, m, n, k):
    """Sums of integers below 2^24 are exact in any order: whole tiles, shared ones and both float outputs have to hit them."""
    r = torch.Generator().manual_seed(m + n + k)
    value = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], device="cuda") * 2

    def integers(rows):
        codes, scales = torch.zeros(rows, ref.code_stride(k), dtype=torch.uint8), torch.zeros(rows, ref.scale_stride(k), dtype=torch.uint8)
        codes[:, : k // 2] = torch.randint(0, 256, (rows, k // 2), generator=r, dtype=torch.uint8)
        scales[:, : (k + 31) // 32] = 128
        codes, scales = codes.cuda(), scales.cuda()
        low, high = codes[:, : k // 2].long() & 15, codes[:, : k // 2].long() >> 4
        return (codes, scales), value[torch.stack([low, high], 2).view(rows, k)]

    (xq, x), (wq, w) = integers(m), integers(n)
    dy = torch.randint(-8, 9, (m, n), generator=r).float().cuda()
    work = torch.empty(lib.mxfp4_linear_backward_bytes(m, n, k), dtype=torch.uint8, device="cuda")
    for _ in range(2):
        dx, dw = torch.empty(m, k, dtype=torch.bfloat16, device="cuda"), torch.empty(n, k, device="cuda")
        db = torch.empty(n, device="cuda")
        lib.mxfp4_linear_backward(dy.bfloat16(), *xq, *wq, dx, dw, "f32", db, work, m, n, k)
        assert torch.equal(dw, dy.T.contiguous() @ x)
        assert torch.equal(dx, (dy @ w).bfloat16())
        assert torch.equal(db, dy.sum(0))
        dw16 = torch.empty(n, k, dtype=torch.bfloat16, device="cuda")
        lib.mxfp4_linear_backward(dy.bfloat16(), *xq, *wq, None, dw16, "bf16", None, work, m, n, k)
        assert torch.equal(dw16, dw.bfloat16())


@pytest.mark.gpu
@pytest.mark.parametrize("m, n, k", BACKWARD)
@pytest.mark.parametrize("kind", ["silu", "gelu"])
def test_gated_backward(gpu, m, n, k, kind):
    (xq, x), (gq, wg), (uq, wu) = matrix(m, m, k), matrix(n, n, k, 2.0 / math.sqrt(k), 2), matrix(k, n, k, 2.0 / math.sqrt(k), 2)
    dh = torch.randn(m, n, generator=torch.Generator().manual_seed(m * n)).bfloat16()
    dg, edg, du, edu = ref.gated_gradients(dh.double(), x, wg, wu, kind)
    size = lib.mxfp4_gated_backward_bytes(m, n, k)
    for dw_type in ("bf16", "f32"):
        raw, work = guarded(size + 256)
        work = work[-work.data_ptr() % 256 :][:size]
        (raw_x, dx), (raw_g, dwg), (raw_u, dwu) = guarded(2 * m * k), *(guarded(ref.DTYPE[dw_type].itemsize * n * k) for _ in range(2))
        lib.mxfp4_gated_backward(dh.cuda(), *xq, *gq, *uq, dx, dwg, dwu, dw_type, work, m, n, k, activation=kind)
        torch.cuda.synchronize()
        assert untouched(raw) and untouched(raw_x) and untouched(raw_g) and untouched(raw_u)
        (a, ea), (b, eb) = ref.product(dg, wg.T), ref.product(du, wu.T)
        # (the two products are one sum of 2 n terms)
        check(dx.view(torch.bfloat16).view(m, k), a + b, 2 * (ea + eb) + 1.01 * (edg @ wg.abs() + edu @ wu.abs()), "bf16")
        for got, d, e in ((dwg, dg, edg), (dwu, du, edu)):
            want, error = ref.product(d.T, x.T)
            check(got.view(ref.DTYPE[dw_type]).view(n, k), want, error + 1.01 * (e.T @ x.abs()), dw_type)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["silu", "gelu"])
def test_gated_gradients_against_differences(gpu, kind):
    """The device's gradients along random directions against differences of the forward pass in float64."""
    m, n, k = 40, 96, 160
    (xq, x), (gq, wg), (uq, wu) = matrix(1, m, k), matrix(2, n, k, 0.2, 1), matrix(3, n, k, 0.2, 1)
    dh = torch.randn(m, n, generator=torch.Generator().manual_seed(4)).bfloat16()
    dx, dwg, dwu = (torch.empty(*s, dtype=d, device="cuda") for s, d in (((m, k), torch.bfloat16), ((n, k), torch.float32), ((n, k), torch.float32)))
    work = torch.empty(lib.mxfp4_gated_backward_bytes(m, n, k), dtype=torch.uint8, device="cuda")
    lib.mxfp4_gated_backward(dh.cuda(), *xq, *gq, *uq, dx, dwg, dwu, "f32", work, m, n, k, activation=kind)
    gen = torch.Generator().manual_seed(6)
    for which, grad in enumerate((dx, dwg, dwu)):
        v = torch.randn(grad.shape, generator=gen, dtype=torch.float64)
        values = []
        for eps in (1e-5, -1e-5):
            args = [x, wg, wu]
            args[which] = args[which] + eps * v
            values.append((dh.double() * ref.gated(*args, kind)[0]).sum().item())
        slope, got = (values[0] - values[1]) / 2e-5, (grad.double().cpu() * v).sum().item()
        # 2^-8 of a sum of terms of random sign, each rounded twice to bfloat16
        assert abs(got - slope) <= 2.0 ** -8 * (grad.double().cpu() * v).norm().item() * 4 + 1e-5 * abs(slope)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["silu", "gelu"])
def test_gated_at_gates_whose_square_is_no_float(gpu, kind):
    """g = 2^65, 0 and -2^65: act is g, 0 and 0, its slope 1, 1/2 and 0."""
    x, wg, wu = torch.zeros(1, 32).double(), torch.zeros(3, 32).double(), torch.full((3, 32), 3.0).double()
    x[0, 0], wg[0, 0], wg[2, 0] = 1.0, 2.0**65, -(2.0**65)
    (xq, gq, uq) = ([t.cuda() for t in ref.encode(v)] for v in (x, wg, wu))
    h, dh = torch.empty(1, 3, device="cuda"), torch.ones(1, 3, dtype=torch.bfloat16, device="cuda")
    lib.mxfp4_gated(*xq, *gq, *uq, h, "f32", 1, 3, 32, activation=kind)
    assert h.tolist() == [[3 * 2.0**65, 0.0, 0.0]]
    dx, dwg, dwu = torch.empty(1, 32, dtype=torch.bfloat16, device="cuda"), *torch.empty(2, 3, 32, device="cuda")
    work = torch.empty(lib.mxfp4_gated_backward_bytes(1, 3, 32), dtype=torch.uint8, device="cuda")
    lib.mxfp4_gated_backward(dh, *xq, *gq, *uq, dx, dwg, dwu, "f32", work, 1, 3, 32, activation=kind)
    assert dwg[:, 0].tolist() == [3.0, 1.5, 0.0] and dwu[:, 0].tolist() == [2.0**65, 0.0, 0.0]
    assert not dwg[:, 1:].any() and not dwu[:, 1:].any()
    # (the columns behind the first: du wu alone)
    assert dx[0, 0].item() == 6 * 2.0**65 and bool((dx[0, 1:] == 3 * 2.0**65).all())


@pytest.mark.gpu
def test_gradients_of_empty_sums(gpu):
    (xq, _), (wq, _) = matrix(1, 5, 40), matrix(2, 6, 40)
    dw, db = torch.full((6, 40), 7.0, device="cuda"), torch.full((6,), 7.0, device="cuda")
    work = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
    lib.mxfp4_linear_backward(None, None, None, *wq, None, dw, "f32", db, work, 0, 6, 40)
    assert not dw.any() and not db.any()
    dx = torch.full((5, 40), 7.0, dtype=torch.bfloat16, device="cuda")
    lib.mxfp4_linear_backward(None, *xq, None, None, dx, None, "f32", None, work, 5, 0, 40)
    assert not dx.any()
    dx.fill_(7.0)
    lib.mxfp4_gated_backward(None, *xq, None, None, None, None, dx, None, None, "f32", work, 5, 0, 40)
    assert not dx.any()
    dwu = torch.full((6, 40), 7.0, device="cuda")
    dw.fill_(7.0)
    lib.mxfp4_gated_backward(None, None, None, *wq, *wq, None, dw, dwu, "f32", work, 0, 6, 40)
    assert not dw.any() and not dwu.any()


@pytest.mark.gpu
def test_large_offsets(gpu):
    """Rows of w whose codes begin beyond 4 GiB, and an output beyond 2^31 elements."""
    n, k = (1 << 16) + 5, 1 << 17
    gen = torch.Generator(device="cuda").manual_seed(1)
    codes = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device="cuda", generator=gen)
    scales = torch.full((n, k // 32), 127, dtype=torch.uint8, device="cuda")
    (xq, x) = matrix(4, 3, k, 1.0, 0)
    y = torch.empty(3, n, device="cuda")
    lib.mxfp4_linear(*xq, codes, scales, None, y, "f32", 3, n, k)
    for r in (0, 1, n - 6, n - 1):
        w = ref.decode(codes[r : r + 1].cpu(), scales[r : r + 1].cpu(), k)
        check(y[:, r : r + 1], *ref.product(x, w), "f32")
    del codes, scales, y
    m, n, k = 1 << 16, (1 << 15) + 64, 32
    (xq, x), (wq, w) = matrix(5, m, k, 1.0, 0), matrix(6, n, k, 1.0, 0)
    y = torch.zeros(m, n, dtype=torch.bfloat16, device="cuda")
    lib.mxfp4_linear(*xq, *wq, None, y, "bf16", m, n, k)
    for r in (0, m - 2, m - 1):
        check(y[r : r + 1], *ref.product(x[r : r + 1], w), "bf16")


@pytest.mark.gpu
def test_conversion_of_very_many_rows(gpu):
    """More rows than one axis of a launch holds; every value is represented exactly."""
    rows, k = (1 << 28) + 5, 3
    x = torch.randint(0, 4, (rows, k), dtype=torch.int8, device="cuda").bfloat16()
    x = torch.where(x == 3, 4.0, x).bfloat16()
    codes = torch.full((lib.mxfp4_code_bytes(rows, k),), 0x77, dtype=torch.uint8, device="cuda")
    scales = torch.full((lib.mxfp4_scale_bytes(rows, k),), 0x77, dtype=torch.uint8, device="cuda")
    lib.mxfp4_quantize(x, codes, scales, rows, k)
    y = torch.empty_like(x)
    lib.mxfp4_dequantize(codes, scales, y, rows, k)
    assert torch.equal(x, y)
    assert not codes.view(rows, -1)[-3:, 2:].any() and not scales.view(rows, -1)[-3:, 1:].any()


@pytest.mark.gpu
def test_results_do_not_change_from_call_to_call(gpu):
    """No atomics, no order that depends on timing: the same bits every time, on any stream."""
    m, n, k = 130, 300, 1100
    (xq, _), (gq, _), (uq, _) = matrix(1, m, k), matrix(2, n, k), matrix(3, n, k)
    dh = torch.randn(m, n, device="cuda").bfloat16()
    first = None
    for stream in (torch.cuda.current_stream(), torch.cuda.Stream(), torch.cuda.Stream()):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            y = torch.empty(m, n, device="cuda")
            h, dx, dwg, dwu = torch.empty(m, n, device="cuda"), torch.empty(m, k, dtype=torch.bfloat16, device="cuda"), *torch.empty(2, n, k, device="cuda")
            work = torch.empty(lib.mxfp4_gated_backward_bytes(m, n, k), dtype=torch.uint8, device="cuda")
            lib.mxfp4_linear(*xq, *gq, None, y, "f32", m, n, k)
            lib.mxfp4_gated(*xq, *gq, *uq, h, "f32", m, n, k)
            lib.mxfp4_gated_backward(dh, *xq, *gq, *uq, dx, dwg, dwu, "f32", work, m, n, k)
        torch.cuda.synchronize()
        got = (y, h, dx, dwg, dwu)
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(first, got))


@pytest.mark.gpu
def test_a_block_captured_into_a_graph(gpu):
    """Quantise, gate, multiply: captured once, replayed on new activations."""
    m, n, k = 20, 320, 512
    (gq, _), (uq, _), (dq, _) = matrix(2, n, k, 0.1), matrix(3, n, k, 0.1), matrix(4, k, n, 0.1)
    x, y = torch.zeros(m, k, dtype=torch.bfloat16, device="cuda"), torch.empty(m, k, dtype=torch.bfloat16, device="cuda")
    xq = [torch.empty(f(m, k), dtype=torch.uint8, device="cuda") for f in (lib.mxfp4_code_bytes, lib.mxfp4_scale_bytes)]
    hq = [torch.empty(f(m, n), dtype=torch.uint8, device="cuda") for f in (lib.mxfp4_code_bytes, lib.mxfp4_scale_bytes)]

    def block():
        lib.mxfp4_quantize(x, *xq, m, k)
        lib.mxfp4_gated_quantized(*xq, *gq, *uq, *hq, m, n, k)
        lib.mxfp4_linear(*hq, *dq, None, y, "bf16", m, k, n)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        block()
    for seed in range(4):
        x.copy_(torch.randn(m, k, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        got = y.clone()
        y.zero_()
        block()
        torch.cuda.synchronize()
        assert got.any() and torch.equal(got, y)


@pytest.mark.gpu
def test_gradients_captured_into_a_graph(gpu):
    """Long sums in slices, whose counters every call clears: each replay gives the eager call's bits."""
    m, n, k = 70, 900, 520
    (xq, _), (gq, _), (uq, _), (wq, _) = matrix(1, m, k), matrix(2, n, k, 0.1), matrix(3, n, k, 0.1), matrix(4, n, k, 0.1)
    dh = torch.zeros(m, n, dtype=torch.bfloat16, device="cuda")
    bytes_needed = lib.mxfp4_linear_backward_bytes(m, n, k), lib.mxfp4_gated_backward_bytes(m, n, k)
    work = torch.full((max(bytes_needed),), 0xFF, dtype=torch.uint8, device="cuda")
    outs = [torch.empty(m, k, dtype=torch.bfloat16, device="cuda") for _ in range(2)] + [torch.empty(n, k, device="cuda") for _ in range(3)]
    outs.append(torch.empty(n, device="cuda"))

    def step():
        lib.mxfp4_linear_backward(dh, *xq, *wq, outs[0], outs[2], "f32", outs[5], work, m, n, k)
        lib.mxfp4_gated_backward(dh, *xq, *gq, *uq, outs[1], outs[3], outs[4], "f32", work, m, n, k)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for seed in range(4):
        dh.copy_(torch.randn(m, n, generator=torch.Generator().manual_seed(seed)))
        work.fill_(0xFF)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in outs]
        for t in outs:
            t.zero_()
        step()
        torch.cuda.synchronize()
        assert all(bool(a.any()) and torch.equal(a, b) for a, b in zip(got, outs))


@pytest.mark.gpu
def test_the_example_learns_and_serves(gpu):
    import importlib.util

    spec = importlib.util.spec_from_file_location("mxfp4_feed_forward", Path(__file__).resolve().parent.parent / "examples" / "mxfp4_feed_forward.py")
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    x = torch.randn(96, 128, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).bfloat16()
    target = example.FeedForward(96, 128, 320, seed=2).forward(x).float()
    block = example.FeedForward(96, 128, 320)
    losses = example.train(block, x, target, 40, 0.02)
    assert losses[-1] < losses[0] / 2
    token = x[:1].clone()
    want = [block.forward(x[i : i + 1].contiguous()).clone() for i in range(4)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = block.forward(token)
    for i in range(4):
        token.copy_(x[i : i + 1])
        graph.replay()
        assert torch.equal(y, want[i])
        block.forward(x)  # eager work between the replays
        torch.cuda.synchronize()
