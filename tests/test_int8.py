"""8-bit linear layers: refusals and sizes (CPU), and their results on the device against float64."""
import math

import pytest
import torch

import int4linear_amd as lib
from int4linear_amd import _lib
from tests import row_reference as ref
from tests.test_mxfp4 import guarded, untouched

OK, SHAPE, NULL, ALIGN, UNSUPPORTED, SCRATCH = 0, 1, 2, 3, 5, 7


# ---- without a device ---------------------------------------------------------------------------


@pytest.mark.parametrize("rows, k", [(0, 0), (1, 1), (3, 128), (3, 129), (2, 14336), (1 << 20, 1 << 20)])
def test_sizes(rows, k):
    assert lib.int8_code_bytes(rows, k) == rows * ((k + 127) // 128) * 128
    assert lib.int8_code_bytes(-1, k) == 0 and lib.int8_code_bytes(rows, -1) == 0


def test_refusals():
    L = _lib.load()
    A, odd = 4096, 4104  # an aligned and a misaligned address; nothing is read
    q = L.int4linear_int8_quantize
    assert q(A, 3, 8, A, A, -1, 8, None) == SHAPE and q(A, 3, 7, A, A, 1, 8, None) == SHAPE and q(A, 3, 8, A, A, 1, -8, None) == SHAPE
    assert q(A, 0, 8, A, A, 1, 8, None) == UNSUPPORTED and q(A, 4, 8, A, A, 1, 8, None) == UNSUPPORTED
    assert q(None, 3, 8, A, A, 1, 8, None) == NULL and q(A, 3, 8, None, A, 1, 8, None) == NULL and q(A, 3, 8, A, None, 1, 8, None) == NULL
    assert q(A, 3, 8, odd, A, 1, 8, None) == ALIGN and q(A, 3, 8, A, A + 2, 1, 8, None) == ALIGN
    assert q(A + 1, 3, 8, A, A, 1, 8, None) == ALIGN and q(A + 2, 1, 8, A, A, 1, 8, None) == ALIGN
    assert q(A, 3, 1 << 31, A, A, 1, (1 << 30) + 1, None) == UNSUPPORTED and q(A, 3, 8, A, A, (1 << 30) + 1, 8, None) == UNSUPPORTED
    assert q(None, 3, 0, None, None, 5, 0, None) == OK and q(None, 3, 8, None, None, 0, 8, None) == OK
    d = L.int4linear_int8_dequantize
    assert d(A, A, A, 3, 8, 1, -8, None) == SHAPE and d(A, A, A, 9, 8, 1, 8, None) == UNSUPPORTED and d(A, A, A, 3, 7, 1, 8, None) == SHAPE
    assert d(A, A, None, 3, 8, 1, 8, None) == NULL and d(A, A + 1, A, 3, 8, 1, 8, None) == ALIGN and d(odd, A, A, 3, 8, 1, 8, None) == ALIGN
    lin = L.int4linear_int8_linear
    assert lin(A, A, A, A, None, A, 3, 1, -1, 8, None) == SHAPE and lin(A, A, A, A, None, A, 0, 1, 1, 8, None) == UNSUPPORTED
    assert lin(A, A, A, A, None, A, 3, 1, 1, 1 << 17, None) == UNSUPPORTED and lin(A, A, A, A, None, A, 3, (1 << 30) + 1, 1, 8, None) == UNSUPPORTED
    assert lin(A, A, A, A, None, None, 3, 1, 1, 8, None) == NULL and lin(A, None, A, A, None, A, 3, 1, 1, 8, None) == NULL
    assert lin(A, A, odd, A, None, A, 3, 1, 1, 8, None) == ALIGN and lin(A, A, A, A, A + 2, A, 3, 1, 1, 8, None) == ALIGN
    assert lin(A, A, A, A + 2, None, A, 3, 1, 1, 8, None) == ALIGN and lin(A, A, A, A, None, odd, 3, 1, 1, 8, None) == ALIGN
    assert lin(None, None, None, None, None, None, 3, 0, 5, 8, None) == OK and lin(None, None, None, None, None, None, 3, 5, 0, 8, None) == OK


def test_refusals_of_the_gradients():
    L = _lib.load()
    A, odd, big = 4096, 4104, 1 << 40
    b = L.int4linear_int8_linear_backward
    need, need32 = (lib.int8_linear_backward_bytes(10, 20, 30, t) for t in ("bf16", "f32"))
    assert 0 < need < need32 and need % 256 == 0 and need32 % 256 == 0 and lib.int8_linear_backward_bytes(-1, 2, 3, "f32") == 0
    assert b(A, A, A, A, A, A, A, 3, A, A, need - 1, 10, 20, 30, None) == SCRATCH
    assert b(A, A, A, A, A, A, A, 1, A, A, need32 - 1, 10, 20, 30, None) == SCRATCH
    assert b(A, A, A, A, A, A, A, 3, A, None, need, 10, 20, 30, None) == NULL
    assert b(A, A, A, A, A, A, A, 3, A, A + 16, need, 10, 20, 30, None) == ALIGN
    assert b(None, A, A, A, A, A, A, 3, A, A, big, 10, 20, 30, None) == NULL and b(A, A, None, A, A, A, A, 3, A, A, big, 10, 20, 30, None) == NULL
    assert b(A, A, A, A, None, A, A, 3, A, A, big, 10, 20, 30, None) == NULL and b(odd, A, A, A, A, A, A, 3, A, A, big, 10, 20, 30, None) == ALIGN
    assert b(A, A, A + 2, A, A, A, A, 3, A, A, big, 10, 20, 30, None) == ALIGN
    assert b(A, A, A, A, A, A, A, 2, A, A, big, 10, 20, 30, None) == UNSUPPORTED
    assert b(A, A, A, A, A, A, A, 3, A, A, big, 10, -20, 30, None) == SHAPE
    assert b(A, A, A, A, A, None, None, 3, None, None, 0, 10, 20, 30, None) == OK  # nothing is wanted
    most = (1 << 22) - 64
    for sizes, status in (((most, 1, 1), SCRATCH), ((1, most, 1), SCRATCH), ((1, 1, most), SCRATCH), ((most + 1, 1, 1), UNSUPPORTED),
                          ((1, most + 1, 1), UNSUPPORTED), ((1, 1, most + 1), UNSUPPORTED)):
        assert b(A, A, A, A, A, A, A, 3, A, A, 0, *sizes, None) == status
    for m, status in ((1 << 21, SCRATCH), ((1 << 21) + 1, UNSUPPORTED)):  # in three pieces
        assert b(A, A, A, A, A, A, A, 1, A, A, 0, m, 1, 1, None) == status
        assert b(A, A, A, A, A, A, None, 1, A, A, 0, m, 1, 1, None) == SCRATCH


@pytest.mark.parametrize("wrong", [b"sixteen bytes...", "text", [1, 2], 4096.0])
def test_objects_without_an_address_are_refused(wrong):
    A = 4096
    for call in (lambda: lib.int8_quantize(wrong, A, A, 1, 8, stream=0), lambda: lib.int8_linear(A, A, A, wrong, None, A, "f32", 1, 1, 8, stream=0),
                 lambda: lib.int8_dequantize(A, wrong, A, 1, 8, stream=0),
                 lambda: lib.int8_linear_backward(A, A, A, A, A, wrong, A, "f32", None, None, 1, 1, 8, stream=0)):
        with pytest.raises(AttributeError, match="data_ptr"):
            call()


def test_the_reference_rounds_by_its_definition():
    """Codes of whole multiples and halves of a scale, by hand."""
    x = torch.tensor([[127.0, 0.5, 1.5, -0.5, -1.5, 2.5, 126.5, -126.5], [0.0] * 8, [254.0, 1.0, 3.0, 0.9999, 1.0001, -1.0, 5.0, -254.0]])
    codes, scales = ref.encode(x)
    assert codes[:, :8].tolist() == [[127, 0, 2, 0, -2, 2, 126, -126], [0] * 8, [127, 0, 2, 0, 1, 0, 2, -127]]
    assert scales.tolist() == [1.0, 2.0**-100, 2.0] and not codes[:, 8:].any()


# ---- on the device --------------------------------------------------------------------------------


def quantize(x, k=None, kind="bf16"):
    """A device matrix -> guarded codes and scales, checked for writes outside."""
    rows, ld = x.shape[0], x.stride(0)
    k = x.shape[1] if k is None else k
    raw_c, codes = guarded(lib.int8_code_bytes(rows, k))
    raw_s, scales = guarded(4 * rows)
    lib.int8_quantize(x, codes, scales, rows, k, in_type=kind, ld=ld)
    torch.cuda.synchronize()
    assert untouched(raw_c) and untouched(raw_s)
    return codes.view(torch.int8).view(rows, -1), scales.view(torch.float32)


def same(got, want):
    """Codes and scales, NaN for NaN."""
    return torch.equal(got[0].cpu(), want[0].cpu()) and torch.equal(got[1].cpu().view(torch.int32) & 0x7FFFFFFF, want[1].cpu().view(torch.int32) & 0x7FFFFFFF)


def matrix(seed, rows, k, scale=1.0):
    """A random 8-bit matrix: its operands on the device and its values in float64.  Rows differ by up to 2^6 in size, every code occurs."""
    gen = torch.Generator().manual_seed(seed)
    codes = torch.zeros(rows, ref.up(k, 128), dtype=torch.int8)
    codes[:, :k] = torch.randint(-128, 128, (rows, k), generator=gen, dtype=torch.int8)
    scales = (torch.exp2(-6 * torch.rand(rows, generator=gen)) * scale / 127).float()
    return (codes.cuda(), scales.cuda()), ref.decode(codes, scales, k)


ROWS = [(1, 1, 1), (1, 31, 31), (300, 64, 64), (77, 129, 130), (50, 256, 256), (2, 32, 40), (3, 33, 33), (5, 127, 128), (4, 128, 128), (7, 513, 515), (3, 1024, 1024), (6, 2049, 2060), (33, 1000, 1001),
        (16, 4096, 4096), (130, 777, 784), (5, 8200, 8200), (3, 16384, 16384), (2, 32800, 32801), (2, 70001, 70001)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows, k, ld", ROWS)
def test_quantize_is_the_formula(gpu, kind, rows, k, ld):
    gen = torch.Generator().manual_seed(rows * 1000 + k)
    x = torch.randn(rows, ld, generator=gen) * torch.exp2(20 * torch.rand(rows, 1, generator=gen) - 10)
    x = x.to(ref.DTYPE[kind])
    if k >= 64:  # ties: the scale is 2^-3
        x[0] = 0
        x[0, :40] = torch.arange(-20, 20) / 16.0
        x[0, 41] = 127 / 8
        x[rows - 1, :k] = 0 if rows > 1 else x[0, :k]
    codes, scales = quantize(x.cuda(), k, kind)
    want = ref.encode(x[:, :k].float())
    assert same((codes, scales), want)
    for out in ("f32", "f16", "bf16"):
        raw, y = guarded(rows * ld * ref.DTYPE[out].itemsize)
        lib.int8_dequantize(codes, scales, y, rows, k, out_type=out, ld=ld)
        torch.cuda.synchronize()
        y = y.view(ref.DTYPE[out]).view(rows, ld).cpu()
        # one float product, rounded once more
        value = (want[0][:, :k].float() * want[1][:, None]).to(ref.DTYPE[out])
        assert untouched(raw) and torch.equal(y[:, :k], value)
        assert (y[:, k:].contiguous().view(torch.uint8) == 0xA5).all()


@pytest.mark.gpu
def test_quantize_next_to_every_border(gpu):
    """For scales of many bits, the floats around each (n + 1/2) * scale."""
    gen = torch.Generator().manual_seed(7)
    top = (1 + torch.rand(4000, 1, generator=gen)) * torch.exp2(torch.randint(-90, 100, (4000, 1), generator=gen).float())
    scale = (top / 127.0).double()
    half = torch.arange(-126, 126).double() + 0.5
    x = (half * scale).float()
    step = torch.randint(-2, 3, x.shape, generator=gen, dtype=torch.int32)
    x = (x.view(torch.int32) + step).view(torch.float32)
    x = torch.cat([top, x], 1)
    assert same(quantize(x.cuda(), kind="f32"), ref.encode(x))


@pytest.mark.gpu
def test_quantize_rows_of_every_size(gpu):
    """Rows whose largest value runs over all floats' exponents, denormals among them, and the largest floats of each type."""
    e = torch.arange(-149, 128).double()
    x = torch.zeros(277, 64)
    x[:, 0], x[:, 1], x[:, 2], x[:, 40] = torch.exp2(e), -0.75 * torch.exp2(e), 0.3 * torch.exp2(e), 1.5 * torch.exp2(e - 1)
    assert same(quantize(x.cuda(), kind="f32"), ref.encode(x))
    for kind in ("f32", "bf16", "f16"):
        big = torch.finfo(ref.DTYPE[kind]).max
        x = torch.tensor([[big, -big, big / 2, big / 300, 0.0], [-big, 1.0, 0.0, 0.0, 2.0]], dtype=torch.float64).to(ref.DTYPE[kind])
        assert same(quantize(x.cuda(), kind=kind), ref.encode(x.float()))


@pytest.mark.gpu
@pytest.mark.parametrize("k", [96, 3000, 40000])
def test_infinities_and_nans_make_their_row_nan_and_no_other(gpu, k):
    x = torch.ones(4, k)
    x[0, 40], x[1, 0], x[2, k - 1] = math.inf, -math.inf, math.nan
    codes, scales = quantize(x.cuda(), kind="f32")
    assert torch.isnan(scales).tolist() == [True, True, True, False] and not codes[:3].any() and bool((codes[3, :k] == 127).all())
    y, z = torch.empty(4, k, device="cuda"), torch.empty(4, 4, device="cuda")
    lib.int8_dequantize(codes, scales, y, 4, k, out_type="f32")
    assert bool(torch.isnan(y[:3]).all()) and bool((y[3] == 127 * scales[3]).all())
    lib.int8_linear(codes, scales, codes, scales, None, z, "f32", 4, 4, k)  # ... and a product its rows and columns
    want = torch.full((4, 4), True)
    want[3, 3] = False
    assert torch.equal(torch.isnan(z.cpu()), want) and abs(z[3, 3].item() - k) < k * 2.0**-21


@pytest.mark.gpu
def test_quantize_of_a_view_that_is_aligned_to_its_element_only(gpu):
    x = torch.randn(9, 300, generator=torch.Generator().manual_seed(2)).bfloat16()
    assert same(quantize(x.cuda()[2:, 7:], 290), ref.encode(x[2:, 7:297].float()))


LINEAR = [(1, 1, 1), (1, 100, 64), (2, 33, 257), (5, 64, 512), (16, 130, 1000), (17, 256, 256), (31, 31, 31), (32, 500, 4096), (33, 129, 515),
          (64, 96, 768), (65, 200, 300), (128, 128, 256), (129, 257, 511), (200, 300, 1024), (257, 513, 640), (300, 700, 2050), (1, 8200, 300),
          (3, 8203, 2050), (16, 8200, 1300), (20, 8192, 5000), (48, 4100, 1000), (4250, 4504, 130), (2200, 4201, 400), (2, 5, 14336), (3, 130, 700),
          (4, 301, 1300), (4, 8195, 2050), (7, 50, 1025), (33, 8193, 515), (49, 5000, 700), (50, 8192, 300), (64, 8192, 1300), (64, 8193, 520), (64, 31, 4000), (65, 1, 1), (70, 3, 129),
          (66, 8, 128), (129, 12, 200), (65, 8193, 130), (100, 8200, 260),
          (900, 3904, 2100), (897, 3901, 2050), (330, 14336, 2100), (331, 14330, 2100),
          (500, 11008, 2100), (510, 10950, 2050), (2800, 2880, 2700), (2700, 2890, 2701)]


def product(x, w, bias=None):
    """x w^T + bias, and what a conversion of an exact sum, two products and a sum in float are off at most.  (And what float64 is: a
    product of two values has 62 bits, so k terms and their sums are off by 2^-53 each, all that is left where a sum is zero.)"""
    y = x @ w.T
    total = y if bias is None else y + bias.double().to(y.device)
    return total, ref.U * (3 * y.abs() + total.abs()) + 2 * x.shape[1] * 2.0**-53 * (x.abs() @ w.abs().T)


@pytest.mark.gpu
@pytest.mark.parametrize("m, n, k", LINEAR)
@pytest.mark.parametrize("out", ["f32", "f16", "bf16"])
def test_linear(gpu, m, n, k, out):
    (xq, x), (wq, w) = matrix(m + 7 * n, m, k), matrix(n + k, n, k)
    x, w = x.cuda(), w.cuda()
    bias = torch.randn(n, generator=torch.Generator().manual_seed(3)).cuda()
    for b in (None, bias):
        raw, y = guarded(m * n * ref.DTYPE[out].itemsize)
        lib.int8_linear(*xq, *wq, b, y, out, m, n, k)
        torch.cuda.synchronize()
        assert untouched(raw)
        ref.check(y.view(ref.DTYPE[out]).view(m, n), *product(x, w, b), out)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 40])
def test_sums_at_the_largest_k_are_exact(gpu, m):
    """Every product is 2^14 and k is 2^17 - 1: the sum is the largest 32-bit number that is reached."""
    n, k = 48, (1 << 17) - 1
    x, w = torch.zeros(m, k + 1, dtype=torch.int8, device="cuda"), torch.zeros(n, k + 1, dtype=torch.int8, device="cuda")
    x[:, :k], w[:, :k] = -128, -128
    one, y = torch.ones(max(m, n), device="cuda"), torch.empty(m, n, device="cuda")
    lib.int8_linear(x, one, w, one, None, y, "f32", m, n, k)
    assert bool((y == float(k << 14)).all())
    w[:, 0] = 127
    lib.int8_linear(x, one, w, one, None, y, "f32", m, n, k)
    assert bool((y == float((k - 1 << 14) - 128 * 127)).all())


@pytest.mark.gpu
def test_linear_without_k_and_without_rows(gpu):
    bias, y = torch.randn(40, device="cuda"), torch.full((3, 40), 7.0, device="cuda")
    lib.int8_linear(None, None, None, None, bias, y, "f32", 3, 40, 0)
    assert torch.equal(y, bias.expand(3, 40))
    lib.int8_linear(None, None, None, None, None, y, "f32", 3, 40, 0)
    assert not y.any()
    lib.int8_linear(None, None, None, None, None, y, "f32", 0, 40, 8)


BACKWARD = [(1, 1, 1), (2, 33, 65), (5, 7, 300), (16, 130, 1000), (64, 64, 64), (65, 129, 257), (130, 1001, 515), (300, 200, 333), (70, 900, 520),
            (1000, 2000, 1990), (2816, 2050, 2800), (2000, 2040, 1904), (1990, 2033, 1901), (2800, 2760, 2808)]


@pytest.mark.gpu
@pytest.mark.parametrize("m, n, k", BACKWARD)
@pytest.mark.parametrize("dw_type", ["bf16", "f32"])
def test_linear_backward(gpu, m, n, k, dw_type):
    (xq, x), (wq, w) = matrix(m, m, k), matrix(n, n, k, 1.0 / math.sqrt(k))
    x, w = x.cuda(), w.cuda()
    dy = torch.randn(m, n, generator=torch.Generator().manual_seed(m * n)).bfloat16().cuda()
    size = lib.int8_linear_backward_bytes(m, n, k, dw_type)
    raw, work = guarded(size + 256)
    work = work[-work.data_ptr() % 256 :][:size]
    (raw_x, dx), (raw_w, dw), (raw_b, db) = guarded(2 * m * k), guarded(ref.DTYPE[dw_type].itemsize * n * k), guarded(4 * n)
    lib.int8_linear_backward(dy, *xq, *wq, dx, dw, dw_type, db, work, m, n, k)
    torch.cuda.synchronize()
    assert untouched(raw) and untouched(raw_x) and untouched(raw_w) and untouched(raw_b)
    d = dy.double()
    # float sums of n (m) terms, each with one factor rounded to bfloat16 or, in three pieces of a float, 3 m of them
    size_x, size_w = d.abs() @ w.abs(), d.abs().T @ x.abs()
    got_x, got_w, got_b = dx.view(torch.bfloat16).view(m, k), dw.view(ref.DTYPE[dw_type]).view(n, k), db.view(torch.float32)
    ref.check(got_x, d @ w, (2.0**-8 + n * 2.0**-23) * size_x, "bf16")
    ref.check(got_w, d.T @ x, ((2.0**-8 if dw_type == "bf16" else 2.0**-24) + 3 * m * 2.0**-23) * size_w, dw_type)
    ref.check(got_b, d.sum(0), m * 2.0**-23 * d.abs().sum(0), "f32")
    # any of them alone: the same bits
    for which in range(3):
        alone = [torch.empty_like(t) if i == which else None for i, t in enumerate((got_x, got_w, got_b))]
        lib.int8_linear_backward(dy, *xq, *wq, alone[0], alone[1], dw_type, alone[2], work, m, n, k)
        assert torch.equal(alone[which], (got_x, got_w, got_b)[which])


@pytest.mark.gpu
@pytest.mark.parametrize("m, n, k", [(1000, 1000, 1000), (1000, 2000, 1990), (200, 5000, 4000), (4000, 300, 500)])
def test_input_gradients_do_not_depend_on_the_weights(gpu, m, n, k):
    """dx has the same bits beside dw in either type and without it."""
    (xq, _), (wq, _) = matrix(m, m, k), matrix(n, n, k, 1.0 / math.sqrt(k))
    dy = torch.randn(m, n, generator=torch.Generator().manual_seed(m * n)).bfloat16().cuda()
    results = []
    for dw_type in ("bf16", "f32", None):
        dw = torch.empty(n, k, dtype=ref.DTYPE[dw_type], device="cuda") if dw_type else None
        work = torch.empty(lib.int8_linear_backward_bytes(m, n, k, dw_type or "bf16"), dtype=torch.uint8, device="cuda")
        results.append(torch.empty(m, k, dtype=torch.bfloat16, device="cuda"))
        lib.int8_linear_backward(dy, *xq, *wq, results[-1], dw, dw_type or "bf16", None, work, m, n, k)
    assert torch.equal(results[0], results[1]) and torch.equal(results[0], results[2])


@pytest.mark.gpu
def test_gradients_as_floats_keep_the_values_bits(gpu):
    """One token with dy = 1: dw is X itself as a float, to the last bit."""
    k = 300
    codes = torch.randint(-128, 128, (1, 384), dtype=torch.int8, generator=torch.Generator().manual_seed(1)).cuda()
    codes[:, k:] = 0
    dy, work = torch.ones(1, 8, dtype=torch.bfloat16, device="cuda"), torch.empty(1 << 25, dtype=torch.uint8, device="cuda")
    for scale in (0.7310586, 0.75):
        dw = torch.empty(8, k, device="cuda")
        s = torch.tensor([scale], device="cuda")
        lib.int8_linear_backward(dy, codes, s, None, None, None, dw, "f32", None, work, 1, 8, k)
        assert torch.equal(dw, (codes[:, :k].float() * s).expand(8, k))


@pytest.mark.gpu
def test_gradients_against_differences(gpu):
    """The device's gradients along random directions against differences of the forward pass in float64."""
    m, n, k = 40, 96, 160
    (xq, x), (wq, w) = matrix(1, m, k), matrix(2, n, k, 0.2)
    dy = torch.randn(m, n, generator=torch.Generator().manual_seed(4)).bfloat16()
    dx, dw, db = torch.empty(m, k, dtype=torch.bfloat16, device="cuda"), torch.empty(n, k, device="cuda"), torch.empty(n, device="cuda")
    work = torch.empty(lib.int8_linear_backward_bytes(m, n, k, "f32"), dtype=torch.uint8, device="cuda")
    lib.int8_linear_backward(dy.cuda(), *xq, *wq, dx, dw, "f32", db, work, m, n, k)
    gen = torch.Generator().manual_seed(6)
    for which, grad in enumerate((dx, dw, db)):
        v = torch.randn(grad.shape, generator=gen, dtype=torch.float64)
        values = []
        for eps in (1e-3, -1e-3):  # (the forward pass is linear in each: no step is too long)
            args = [x, w, torch.zeros(n, dtype=torch.float64)]
            args[which] = args[which] + eps * v
            values.append((dy.double() * (args[0] @ args[1].T + args[2])).sum().item())
        slope, got = (values[0] - values[1]) / 2e-3, (grad.double().cpu() * v).sum().item()
        # 2^-8 of a sum of terms of random sign, each rounded twice to bfloat16
        assert abs(got - slope) <= 2.0**-8 * (grad.double().cpu() * v).norm().item() * 4 + 1e-9 * abs(slope)


@pytest.mark.gpu
def test_gradients_of_empty_sums(gpu):
    (xq, _), (wq, _) = matrix(1, 5, 40), matrix(2, 6, 40)
    work = torch.empty(1 << 25, dtype=torch.uint8, device="cuda")
    for dw_type in ("f32", "bf16"):
        dw, db = torch.full((6, 40), 7.0, device="cuda").to(ref.DTYPE[dw_type]), torch.full((6,), 7.0, device="cuda")
        lib.int8_linear_backward(None, None, None, *wq, None, dw, dw_type, db, work, 0, 6, 40)
        assert not dw.any() and not db.any()
    dx = torch.full((5, 40), 7.0, dtype=torch.bfloat16, device="cuda")
    lib.int8_linear_backward(None, *xq, None, None, dx, None, "f32", None, work, 5, 0, 40)
    assert not dx.any()


@pytest.mark.gpu
def test_large_offsets(gpu):
    """Rows of w and of an output beyond 4 GiB."""
    n, k = (1 << 16) + 5, (1 << 16) + 128
    gen = torch.Generator(device="cuda").manual_seed(1)
    codes = torch.randint(-127, 128, (n, k), dtype=torch.int8, device="cuda", generator=gen)
    scales = torch.rand(n, device="cuda", generator=gen)
    for m in (3, 70):
        (xq, x) = matrix(4, m, k)
        y = torch.empty(m, n, device="cuda")
        lib.int8_linear(*xq, codes, scales, None, y, "f32", m, n, k)
        at = torch.tensor([0, 1, n - 6, n - 1], device="cuda")
        ref.check(y[:, at], *product(x.cuda(), ref.decode(codes[at], scales[at], k)), "f32")
    del codes, y
    m, n, k = 1 << 16, (1 << 15) + 64, 32
    (xq, x), (wq, w) = matrix(5, m, k), matrix(6, n, k)
    y = torch.zeros(m, n, dtype=torch.bfloat16, device="cuda")
    lib.int8_linear(*xq, *wq, None, y, "bf16", m, n, k)
    for r in (0, m - 2, m - 1):
        ref.check(y[r : r + 1], *product(x[r : r + 1].cuda(), w.cuda()), "bf16")


@pytest.mark.gpu
def test_conversion_of_very_many_rows(gpu):
    """More rows than one axis of a launch holds; every value is represented exactly."""
    rows, k = (1 << 25) + 5, 3
    x = torch.randint(-1, 2, (rows, k), dtype=torch.int8, device="cuda").float() * 127
    codes = torch.full((rows, 128), 0x77, dtype=torch.int8, device="cuda")
    scales = torch.full((rows,), 7.0, device="cuda")
    lib.int8_quantize(x, codes, scales, rows, k, in_type="f32")
    assert not codes[:, k:].any()
    y = torch.empty_like(x)
    lib.int8_dequantize(codes, scales, y, rows, k, out_type="f32")
    assert torch.equal(x, y)


@pytest.mark.gpu
def test_a_layer_and_its_gradients_captured_into_a_graph(gpu):
    """Quantise, multiply, gradients: captured once, replayed on new activations with eager work on the same buffers in between; long sums
    meet through counters that every call clears."""
    m, n, k = 70, 900, 520
    (wq, _) = matrix(2, n, k, 0.1)
    x, dy = torch.zeros(m, k, dtype=torch.bfloat16, device="cuda"), torch.zeros(m, n, dtype=torch.bfloat16, device="cuda")
    xq = torch.empty(m, ref.up(k, 128), dtype=torch.int8, device="cuda"), torch.empty(m, device="cuda")
    work = torch.empty(lib.int8_linear_backward_bytes(m, n, k, "f32"), dtype=torch.uint8, device="cuda")
    outs = [torch.empty(m, n, device="cuda"), torch.empty(m, k, dtype=torch.bfloat16, device="cuda"), torch.empty(n, k, device="cuda"),
            torch.empty(n, device="cuda")]

    def step():
        lib.int8_quantize(x, *xq, m, k)
        lib.int8_linear(*xq, *wq, None, outs[0], "f32", m, n, k)
        lib.int8_linear_backward(dy, *xq, *wq, outs[1], outs[2], "f32", outs[3], work, m, n, k)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for seed in range(4):
        gen = torch.Generator().manual_seed(seed)
        x.copy_(torch.randn(m, k, generator=gen))
        dy.copy_(torch.randn(m, n, generator=gen))
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
def test_results_do_not_change_from_stream_to_stream(gpu):
    m, n, k = 130, 300, 1100
    (xq, _), (wq, _) = matrix(1, m, k), matrix(2, n, k)
    dy, first = torch.randn(m, n, device="cuda").bfloat16(), None
    for stream in (torch.cuda.current_stream(), torch.cuda.Stream(), torch.cuda.Stream()):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            y, dx, dw = torch.empty(m, n, device="cuda"), torch.empty(m, k, dtype=torch.bfloat16, device="cuda"), torch.empty(n, k, device="cuda")
            work = torch.empty(lib.int8_linear_backward_bytes(m, n, k, "f32"), dtype=torch.uint8, device="cuda")
            lib.int8_linear(*xq, *wq, None, y, "f32", m, n, k)
            lib.int8_linear_backward(dy, *xq, *wq, dx, dw, "f32", None, work, m, n, k)
        torch.cuda.synchronize()
        first = first or (y, dx, dw)
        assert all(torch.equal(a, b) for a, b in zip(first, (y, dx, dw)))


@pytest.mark.gpu
@pytest.mark.parametrize("m, n, k", [(3, 40, 70), (200, 130, 515)])
@pytest.mark.parametrize("dw_type", ["bf16", "f32"])
def test_gradients_at_the_largest_floats(gpu, m, n, k, dw_type):
    """Values above the largest bfloat16, which is 2^-8 below the largest float."""
    (xq, _), (wq, _) = matrix(m, m, k), matrix(n, n, k)
    top = torch.finfo(torch.float32).max
    for codes, scales in (xq, wq):
        codes[:, :k][codes[:, :k] == -128] = 127
        codes[:, 0], codes[:, k - 1] = 127, -127
        scales[:2] = top / 127 * (1 - 2.0**-23)  # (127 times the rounded quotient is no float)
    x, w = ref.decode(*xq, k), ref.decode(*wq, k)
    assert (x.abs() > 3.39e38).any() and x.abs().max().item() <= top and w.abs().max().item() <= top
    dy = (torch.randn(m, n, generator=torch.Generator().manual_seed(m * n)) * 2.0**-20).bfloat16().cuda()
    dx, dw = torch.empty(m, k, dtype=torch.bfloat16, device="cuda"), torch.empty(n, k, dtype=ref.DTYPE[dw_type], device="cuda")
    work = torch.empty(lib.int8_linear_backward_bytes(m, n, k, dw_type), dtype=torch.uint8, device="cuda")
    lib.int8_linear_backward(dy, *xq, *wq, dx, dw, dw_type, None, work, m, n, k)
    d = dy.double()
    # as in test_linear_backward: a factor above the largest bfloat16 is taken as that, which is off by 2^-8 of it
    ref.check(dx, d @ w, (2.0**-8 + n * 2.0**-23) * (d.abs() @ w.abs()), "bf16")
    ref.check(dw, d.T @ x, ((2.0**-8 if dw_type == "bf16" else 2.0**-24) + 3 * m * 2.0**-23) * (d.abs().T @ x.abs()), dw_type)


@pytest.mark.gpu
def test_gradients_as_floats_keep_the_bits_of_the_largest_values(gpu):
    """One token with dy = 1: dw is X itself, up to the largest float."""
    k = 256
    codes = torch.randint(-127, 128, (1, k), dtype=torch.int8, generator=torch.Generator().manual_seed(1)).cuda()
    codes[0, 0], codes[0, 1] = 127, -127
    dy, work = torch.ones(1, 8, dtype=torch.bfloat16, device="cuda"), torch.empty(1 << 25, dtype=torch.uint8, device="cuda")
    s = torch.tensor([torch.finfo(torch.float32).max / 127 * (1 - 2.0**-23)], device="cuda")
    dw = torch.empty(8, k, device="cuda")
    lib.int8_linear_backward(dy, codes, s, None, None, None, dw, "f32", None, work, 1, 8, k)
    want = codes.float() * s
    assert bool(torch.isfinite(want).all()) and torch.equal(dw, want.expand(8, k))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows, k", [(9000, 500), (5000, 1000), (1100, 2000), (1030, 4000), (1100, 4999), (1030, 8192), (1030, 12001), (1024, 16384)])
def test_quantize_of_many_rows(gpu, rows, k, kind):
    """The kernels that many rows choose, every code and scale against the formula."""
    gen = torch.Generator().manual_seed(rows + k)
    x = (torch.randn(rows, k, generator=gen) * torch.exp2(20 * torch.rand(rows, 1, generator=gen) - 10)).to(ref.DTYPE[kind])
    assert same(quantize(x.cuda(), kind=kind), ref.encode(x.float()))


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 2])
def test_one_and_two_rows_against_weights_beyond_4_gib(gpu, m):
    n, k = (1 << 16) + 5, (1 << 16) + 128
    gen = torch.Generator(device="cuda").manual_seed(1)
    codes = torch.randint(-127, 128, (n, k), dtype=torch.int8, device="cuda", generator=gen)
    scales = torch.rand(n, device="cuda", generator=gen)
    (xq, x) = matrix(4, m, k)
    y = torch.empty(m, n, device="cuda")
    lib.int8_linear(*xq, codes, scales, None, y, "f32", m, n, k)
    at = torch.tensor([0, 1, n // 2, n - 6, n - 1], device="cuda")
    ref.check(y[:, at], *product(x.cuda(), ref.decode(codes[at], scales[at], k)), "f32")


@pytest.mark.gpu
@pytest.mark.parametrize("m, n", [(1, (1 << 22) + 5), (2, (1 << 22) + 4097), (5, (1 << 25) + 37)])
def test_more_workgroups_than_one_axis_holds(gpu, m, n):
    """Streamed weights of very many short rows."""
    k = 20
    (xq, x) = matrix(1, m, k)
    gen = torch.Generator("cuda").manual_seed(n)
    codes = torch.randint(-128, 128, (n, 128), dtype=torch.int8, device="cuda", generator=gen)
    codes[:, k:] = 0
    scales = torch.rand(n, device="cuda", generator=gen)
    raw, y = guarded(m * n * 2)
    lib.int8_linear(*xq, codes, scales, None, y, "bf16", m, n, k)
    torch.cuda.synchronize()
    assert untouched(raw)
    y = y.view(torch.bfloat16).view(m, n)
    for at in range(0, n, 1 << 22):
        part = slice(at, min(n, at + (1 << 22)))
        ref.check(y[:, part], *product(x.cuda(), ref.decode(codes[part], scales[part], k)), "bf16")
