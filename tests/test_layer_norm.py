"""Layer norms: refusals (CPU), and their results and gradients on the device against float64."""
import math

import pytest
import torch

import int4linear_amd as lib
from int4linear_amd import _lib
from tests import row_reference as ref
from tests.test_int8 import matrix, product
from tests.test_mxfp4 import guarded, untouched

OK, SHAPE, NULL, ALIGN, UNSUPPORTED, SCRATCH = 0, 1, 2, 3, 5, 7
EPS = 1e-5


# ---- without a device ---------------------------------------------------------------------------


def test_refusals():
    L = _lib.load()
    A, odd, e = 4096, 4104, EPS
    f = L.int4linear_layer_norm
    assert f(A, 3, 8, A, A, e, A, 3, 8, -1, 8, None) == SHAPE and f(A, 3, 7, A, A, e, A, 3, 8, 1, 8, None) == SHAPE
    assert f(A, 3, 8, A, A, e, A, 3, 7, 1, 8, None) == SHAPE and f(A, 3, 8, A, A, e, A, 3, 8, 1, -8, None) == SHAPE
    assert f(A, 0, 8, A, A, e, A, 3, 8, 1, 8, None) == UNSUPPORTED and f(A, 3, 8, A, A, e, A, 4, 8, 1, 8, None) == UNSUPPORTED
    for eps in (-1e-5, math.inf, math.nan):
        assert f(A, 3, 8, A, A, eps, A, 3, 8, 1, 8, None) == UNSUPPORTED
    big = (1 << 22) + 1
    assert f(A, 3, big, A, A, e, A, 3, big, 1, big, None) == UNSUPPORTED and f(A, 3, 8, A, A, e, A, 3, 8, (1 << 30) + 1, 8, None) == UNSUPPORTED
    assert f(None, 3, 8, A, A, e, A, 3, 8, 1, 8, None) == NULL and f(A, 3, 8, A, A, e, None, 3, 8, 1, 8, None) == NULL
    assert f(A + 1, 3, 8, A, A, e, A, 3, 8, 1, 8, None) == ALIGN and f(A, 3, 8, A + 2, A, e, A, 3, 8, 1, 8, None) == ALIGN
    assert f(A, 3, 8, A, A + 1, e, A, 3, 8, 1, 8, None) == ALIGN and f(A, 3, 8, A, A, e, A + 2, 1, 8, 1, 8, None) == ALIGN
    assert f(None, 3, 8, None, None, e, None, 3, 8, 0, 8, None) == OK and f(None, 3, 0, None, None, e, None, 3, 0, 5, 0, None) == OK
    for g in (L.int4linear_layer_norm_int8, L.int4linear_layer_norm_mxfp4):
        assert g(A, 3, 7, A, A, e, A, A, 1, 8, None) == SHAPE and g(A, 7, 8, A, A, e, A, A, 1, 8, None) == UNSUPPORTED
        assert g(A, 3, 8, A, A, -1.0, A, A, 1, 8, None) == UNSUPPORTED and g(None, 3, 8, A, A, e, A, A, 1, 8, None) == NULL
        assert g(A, 3, 8, A, A, e, None, A, 1, 8, None) == NULL and g(A, 3, 8, A, A, e, A, None, 1, 8, None) == NULL
        assert g(A, 3, 8, A, A, e, odd, A, 1, 8, None) == ALIGN and g(A, 3, 8, A, A, e, A, A + 2, 1, 8, None) == ALIGN
        assert g(None, 3, 8, None, None, e, None, None, 0, 8, None) == OK
    assert L.int4linear_layer_norm_mxfp4(A, 3, 8, A, A, e, A, A + 4, 1, 8, None) == ALIGN


def test_refusals_of_the_gradients():
    L = _lib.load()
    A, e, big = 4096, EPS, 1 << 40
    b = L.int4linear_layer_norm_backward
    need = lib.layer_norm_backward_bytes(10, 20)
    assert need > 0 and need % 256 == 0 and lib.layer_norm_backward_bytes(-1, 2) == 0 and lib.layer_norm_backward_bytes(1, -2) == 0

    def call(dy=A, dy_type=3, ld_dy=20, x=A, kind=3, ld=20, gamma=A, eps=e, dx=A, ld_dx=20, dgamma=A, dbeta=A, work=A, size=big, rows=10, n=20):
        return b(dy, dy_type, ld_dy, x, kind, ld, gamma, eps, dx, ld_dx, dgamma, dbeta, work, size, rows, n, None)

    assert call(size=need - 1) == SCRATCH and call(work=None) == NULL and call(work=A + 16) == ALIGN
    assert call(rows=-1) == SHAPE and call(n=-1) == SHAPE and call(ld_dy=19) == SHAPE and call(ld=19) == SHAPE and call(ld_dx=19) == SHAPE
    assert call(dy_type=0) == UNSUPPORTED and call(kind=4) == UNSUPPORTED and call(eps=-1.0) == UNSUPPORTED and call(eps=math.nan) == UNSUPPORTED
    assert call(dy=None) == NULL and call(x=None) == NULL
    assert call(dy=A + 1) == ALIGN and call(x=A + 2, kind=1) == ALIGN and call(gamma=A + 2) == ALIGN and call(dx=A + 1) == ALIGN
    assert call(dgamma=A + 2) == ALIGN and call(dbeta=A + 2) == ALIGN
    long = (1 << 22) + 1
    assert call(n=long, ld=long, ld_dy=long, ld_dx=long) == UNSUPPORTED and call(rows=(1 << 30) + 1) == UNSUPPORTED
    assert call(dx=None, dgamma=None, dbeta=None, work=None, size=0) == OK  # nothing is wanted
    assert call(dx=None, ld_dx=0, size=need - 1) == SCRATCH                 # (the distance of rows that are not wanted is not looked at)
    assert call(n=0, ld=0, ld_dy=0, ld_dx=0, dy=None, x=None, work=None, size=0) == OK


@pytest.mark.parametrize("wrong", [b"sixteen bytes...", "text", [1, 2], 4096.0])
def test_objects_without_an_address_are_refused(wrong):
    A = 4096
    for call in (lambda: lib.layer_norm(wrong, A, A, A, 1, 8, stream=0), lambda: lib.layer_norm(A, wrong, None, A, 1, 8, stream=0),
                 lambda: lib.layer_norm_int8(A, None, None, wrong, A, 1, 8, stream=0),
                 lambda: lib.layer_norm_mxfp4(A, None, wrong, A, A, 1, 8, stream=0),
                 lambda: lib.layer_norm_backward(A, A, A, wrong, A, A, None, 1, 8, stream=0)):
        with pytest.raises(AttributeError, match="data_ptr"):
            call()
    with pytest.raises(TypeError, match="work_bytes"):
        lib.layer_norm_backward(A, A, A, A, A, A, A, 1, 8, stream=0)


def test_rows_a_negative_number_apart_are_refused():
    """(ctypes makes a size_t of it; rows would lie in front of the array.)"""
    A = 4096
    for call in (lambda: lib.layer_norm(A, A, A, A, 3, 8, ld=-8, stream=0), lambda: lib.layer_norm(A, A, A, A, 3, 8, ld_y=-8, stream=0),
                 lambda: lib.layer_norm_int8(A, A, A, A, A, 3, 8, ld=-8, stream=0), lambda: lib.layer_norm_mxfp4(A, A, A, A, A, 3, 8, ld=-1, stream=0),
                 lambda: lib.layer_norm_backward(A, A, A, A, A, A, A, 3, 8, ld=-8, work_bytes=1 << 30, stream=0),
                 lambda: lib.layer_norm_backward(A, A, A, A, A, A, A, 3, 8, ld_dy=-8, work_bytes=1 << 30, stream=0),
                 lambda: lib.layer_norm_backward(A, A, A, A, A, A, A, 3, 8, ld_dx=-8, work_bytes=1 << 30, stream=0),
                 lambda: lib.int8_quantize(A, A, A, 3, 8, ld=-8, stream=0), lambda: lib.int8_dequantize(A, A, A, 3, 8, ld=-8, stream=0),
                 lambda: lib.mxfp4_quantize(A, A, A, 3, 8, ld=-8, stream=0), lambda: lib.mxfp4_dequantize(A, A, A, 3, 8, ld=-8, stream=0)):
        with pytest.raises(lib.Int4LinearError) as refused:
            call()
        assert refused.value.status == SHAPE


def test_the_reference_gradients_against_differences():
    """The formulas that the device's gradients are compared with, against central differences."""
    gen = torch.Generator().manual_seed(5)
    dy, x, gamma, beta = (torch.randn(*s, generator=gen, dtype=torch.float64) for s in ((5, 11), (5, 11), (11,), (11,)))
    grads = [g[0] for g in ref.norm_gradients(dy, x, gamma, EPS)]
    for which, grad in enumerate(grads):
        v = torch.randn(grad.shape, generator=gen, dtype=torch.float64)
        values = []
        for step in (1e-5, -1e-5):
            args = [x, gamma, beta]
            args[which] = args[which] + step * v
            values.append((dy * ref.norm(*args, EPS)[0]).sum())
        assert math.isclose((values[0] - values[1]).item() / 2e-5, (grad * v).sum().item(), rel_tol=1e-7)


# ---- on the device --------------------------------------------------------------------------------


def rows_of(seed, rows, n, kind, spread=1.0, offset=1.0):
    """Rows of different size, on top of what a column has in all of them."""
    gen = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, n, generator=gen) + offset * torch.randn(1, n, generator=gen)) * torch.exp(spread * torch.randn(rows, 1, generator=gen))
    return x.to(ref.DTYPE[kind])


def vectors(seed, n):
    gen = torch.Generator().manual_seed(seed)
    return 1 + 0.3 * torch.randn(n, generator=gen), 0.3 * torch.randn(n, generator=gen)


#: rows, n: one lane's values, whole and ragged waves, rows of one wave, of several, of every number of eights a thread holds, and longer ones
SIZES = [(1, 1), (3, 2), (2, 7), (5, 8), (4, 63), (7, 64), (9, 500), (33, 65), (1000, 40), (70, 128), (19, 129), (5000, 3), (41, 200), (9, 256), (5, 257), (3, 512), (6, 513), (5, 1000), (4, 1024), (3, 1030), (130, 777), (3, 2048), (2, 2050),
         (16, 4096), (5, 4999), (3, 8192), (2, 8193), (2, 16384), (3, 16385), (2, 32768), (2, 32770), (3, 100001)]


@pytest.mark.gpu
@pytest.mark.parametrize("rows, n", SIZES)
@pytest.mark.parametrize("kind, out", [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "bf16"), ("bf16", "f32"), ("f16", "bf16")])
def test_norm(gpu, rows, n, kind, out):
    x = rows_of(rows + n, rows, n, kind).cuda()
    gamma, beta = (t.cuda() for t in vectors(n, n))
    for g, b in ((gamma, beta), (None, None), (gamma, None), (None, beta)):
        raw, y = guarded(rows * n * ref.DTYPE[out].itemsize)
        lib.layer_norm(x, g, b, y, rows, n, eps=EPS, in_type=kind, out_type=out)
        torch.cuda.synchronize()
        assert untouched(raw)
        ref.check(y.view(ref.DTYPE[out]).view(rows, n), *ref.norm(x, g, b, EPS), out)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [300, 3001, 40000])
def test_norm_of_views_and_in_place(gpu, n):
    """Distances between rows, bases aligned to the element only; what is behind a row stays as it was."""
    big = rows_of(1, 9, n + 21, "bf16").cuda()
    x = big[2:, 7 : 7 + n]
    gamma, beta = (torch.cat([torch.zeros(1), t])[1:].cuda() for t in vectors(2, n))
    out = torch.full((7, n + 5), 9.0, device="cuda")
    lib.layer_norm(x, gamma, beta, out[:, 3:], 7, n, out_type="f32", ld=n + 21, ld_y=n + 5)
    want, error = ref.norm(x, gamma, beta, EPS)
    ref.check(out[:, 3 : 3 + n], want, error, "f32")
    assert bool((out[:, :3] == 9).all()) and bool((out[:, 3 + n :] == 9).all())
    before = big.clone()
    lib.layer_norm(x, gamma, beta, x, 7, n, ld=n + 21, ld_y=n + 21)
    ref.check(x, want, error, "bf16")
    before[2:, 7 : 7 + n] = x
    assert torch.equal(big, before)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [96, 1500, 9000, 50000])
def test_rows_far_from_zero(gpu, n):
    """A mean 3000 times as large as what is normalised costs no digits of that."""
    x = (3000.0 + torch.randn(6, n, generator=torch.Generator().manual_seed(n))).cuda()
    y = torch.empty_like(x)
    lib.layer_norm(x, None, None, y, 6, n, eps=EPS, in_type="f32", out_type="f32")
    want, error = ref.norm(x, None, None, EPS)
    assert error.max().item() < 3e-4  # (a sum of x as it is may be off by 3000 * 2^-24 = 2e-4 with its last rounding alone)
    ref.check(y, want, error, "f32")


@pytest.mark.gpu
def test_constant_rows_and_one_column(gpu):
    """No variance: the shift alone; with eps = 0 a quotient 0 / 0."""
    x, (gamma, beta) = torch.full((3, 700), 5.0, device="cuda"), (t.cuda() for t in vectors(1, 700))
    y = torch.empty_like(x)
    lib.layer_norm(x, gamma, beta, y, 3, 700, in_type="f32", out_type="f32")
    assert torch.equal(y, beta.expand(3, 700))
    lib.layer_norm(x, gamma, beta, y, 3, 700, eps=0.0, in_type="f32", out_type="f32")
    assert bool(torch.isnan(y).all())
    x, y = torch.randn(50, 1, device="cuda"), torch.empty(50, 1, device="cuda")
    lib.layer_norm(x, gamma, beta, y, 50, 1, in_type="f32", out_type="f32")
    assert bool((y == beta[0]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("n", [100, 3000, 40000])
def test_infinities_and_nans_stay_in_their_row(gpu, n):
    x = rows_of(3, 5, n, "f32")
    x[0, 1], x[1, n - 1], x[3, 8] = math.inf, math.nan, -math.inf
    bad = torch.tensor([True, True, False, True, False])
    x, y = x.cuda(), torch.empty(5, n, device="cuda")
    gamma, beta = (t.cuda() for t in vectors(1, n))
    lib.layer_norm(x, gamma, beta, y, 5, n, in_type="f32", out_type="f32")
    assert torch.equal(torch.isnan(y).all(1).cpu(), bad) and torch.equal(torch.isnan(y).any(1).cpu(), bad)
    codes, scales = torch.empty(5, ref.up(n, 128), dtype=torch.int8, device="cuda"), torch.empty(5, device="cuda")
    lib.layer_norm_int8(x, gamma, beta, codes, scales, 5, n, in_type="f32")
    assert torch.equal(torch.isnan(scales).cpu(), bad) and not codes[bad.cuda()].any()
    c4, s4 = (torch.empty(f(5, n), dtype=torch.uint8, device="cuda") for f in (lib.mxfp4_code_bytes, lib.mxfp4_scale_bytes))
    lib.layer_norm_mxfp4(x, gamma, beta, c4, s4, 5, n, in_type="f32")
    assert torch.equal((s4.view(5, -1)[:, : (n + 31) // 32] == 255).all(1).cpu(), bad)
    dx, work = torch.empty(5, n, device="cuda"), torch.empty(lib.layer_norm_backward_bytes(5, n), dtype=torch.uint8, device="cuda")
    lib.layer_norm_backward(y.nan_to_num(), x, gamma, dx, None, None, work, 5, n, dy_type="f32", in_type="f32")
    assert torch.equal(torch.isnan(dx).all(1).cpu(), bad) and torch.equal(torch.isnan(dx).any(1).cpu(), bad)


@pytest.mark.gpu
def test_squares_beyond_a_float_give_the_shift(gpu):
    x = torch.tensor([[1e25, -1e25, 3e25, 0.0], [1.0, 2.0, 3.0, 4.0]], device="cuda")
    beta, y = torch.tensor([1.0, 2.0, 3.0, 4.0], device="cuda"), torch.empty(2, 4, device="cuda")
    lib.layer_norm(x, None, beta, y, 2, 4, in_type="f32", out_type="f32")
    assert torch.equal(y[0], beta) and bool(torch.isfinite(y).all()) and not torch.equal(y[1], beta)


@pytest.mark.gpu
@pytest.mark.parametrize("rows, n", SIZES)
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_quantised_norms_are_the_norm_quantised(gpu, rows, n, kind):
    """Bit for bit what the norm as floats gives after its quantisation."""
    x = rows_of(rows + n, rows, n, kind).cuda()
    gamma, beta = (t.cuda() for t in vectors(n, n))
    if rows > 2:
        x[1] = 0
    y = torch.empty(rows, n, device="cuda")
    for g, b in ((gamma, beta), (None, None)):
        lib.layer_norm(x, g, b, y, rows, n, in_type=kind, out_type="f32")
        for fused, apart, sizes in ((lib.layer_norm_int8, lib.int8_quantize, (lib.int8_code_bytes(rows, n), 4 * rows)),
                                    (lib.layer_norm_mxfp4, lib.mxfp4_quantize, (lib.mxfp4_code_bytes(rows, n), lib.mxfp4_scale_bytes(rows, n)))):
            (raw_c, codes), (raw_s, scales) = guarded(sizes[0]), guarded(sizes[1])
            want = [torch.empty(size, dtype=torch.uint8, device="cuda") for size in sizes]
            fused(x, g, b, codes, scales, rows, n, in_type=kind)
            apart(y, *want, rows, n, in_type="f32")
            torch.cuda.synchronize()
            assert untouched(raw_c) and untouched(raw_s) and torch.equal(codes, want[0]) and torch.equal(scales, want[1])


BACKWARD = [(1, 1), (2, 7), (3, 64), (17, 500), (5, 513), (257, 1000), (130, 2050), (64, 4096), (300, 4999), (19, 8193), (9, 16384), (6, 16390), (5, 32768),
            (4, 40001), (1500, 72), (5000, 33), (1030, 1030), (20000, 64), (7, 100), (3001, 128), (4500, 250), (100, 256), (5, 257)]


@pytest.mark.gpu
@pytest.mark.parametrize("rows, n", BACKWARD)
@pytest.mark.parametrize("kind, dy_kind", [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "bf16"), ("bf16", "f32"), ("f16", "bf16")])
def test_norm_backward(gpu, rows, n, kind, dy_kind):
    x = rows_of(rows + n, rows, n, kind, spread=0.5).cuda()
    dy = torch.randn(rows, n, generator=torch.Generator().manual_seed(rows)).to(ref.DTYPE[dy_kind]).cuda()
    gamma = vectors(n, n)[0].cuda()
    size = lib.layer_norm_backward_bytes(rows, n)
    for g in (gamma, None):
        raw, work = guarded(size + 256)
        work = work[-work.data_ptr() % 256 :][:size]
        (raw_x, dx), (raw_g, dgamma), (raw_b, dbeta) = guarded(rows * n * ref.DTYPE[kind].itemsize), guarded(4 * n), guarded(4 * n)
        lib.layer_norm_backward(dy, x, g, dx, dgamma, dbeta, work, rows, n, dy_type=dy_kind, in_type=kind)
        torch.cuda.synchronize()
        assert untouched(raw) and untouched(raw_x) and untouched(raw_g) and untouched(raw_b)
        got = dx.view(ref.DTYPE[kind]).view(rows, n), dgamma.view(torch.float32), dbeta.view(torch.float32)
        for value, (want, error), out in zip(got, ref.norm_gradients(dy, x, g, EPS), (kind, "f32", "f32")):
            ref.check(value, want, error, out)
        for which in range(3):  # any of them alone: the same bits
            alone = [torch.empty_like(t) if i == which else None for i, t in enumerate(got)]
            lib.layer_norm_backward(dy, x, g, *alone, work, rows, n, dy_type=dy_kind, in_type=kind)
            assert torch.equal(alone[which], got[which])


@pytest.mark.gpu
@pytest.mark.parametrize("n", [300, 3001, 40000])
def test_norm_backward_of_views(gpu, n):
    rows = 11
    big_x, big_dy = rows_of(1, rows + 2, n + 21, "f32").cuda(), rows_of(2, rows + 2, n + 9, "bf16").cuda()
    x, dy, out = big_x[2:, 7 : 7 + n], big_dy[1:-1, 3 : 3 + n], torch.full((rows, n + 5), 9.0, device="cuda")
    gamma = torch.cat([torch.zeros(1), vectors(2, n)[0]])[1:].cuda()
    dgamma, dbeta = torch.full((2, n + 2), 9.0, device="cuda")
    work = torch.empty(lib.layer_norm_backward_bytes(rows, n), dtype=torch.uint8, device="cuda")
    lib.layer_norm_backward(dy, x, gamma, out[:, 3:], dgamma[1:], dbeta[1:], work, rows, n, dy_type="bf16", in_type="f32", ld_dy=n + 9, ld=n + 21,
                            ld_dx=n + 5)
    for value, (want, error) in zip((out[:, 3 : 3 + n], dgamma[1 : n + 1], dbeta[1 : n + 1]), ref.norm_gradients(dy, x, gamma, EPS)):
        ref.check(value, want, error, "f32")
    assert bool((out[:, :3] == 9).all()) and bool((out[:, 3 + n :] == 9).all())
    assert all(t[0].item() == 9 and t[n + 1].item() == 9 for t in (dgamma, dbeta))


@pytest.mark.gpu
def test_gradients_against_differences(gpu):
    """The device's gradients along random directions against differences of the forward pass in float64."""
    rows, n = 40, 700
    x, dy, (gamma, beta) = rows_of(1, rows, n, "f32", 0.3), torch.randn(rows, n, generator=torch.Generator().manual_seed(4)), vectors(3, n)
    dx, dgamma, dbeta = torch.empty(rows, n, device="cuda"), torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    work = torch.empty(lib.layer_norm_backward_bytes(rows, n), dtype=torch.uint8, device="cuda")
    lib.layer_norm_backward(dy.cuda(), x.cuda(), gamma.cuda(), dx, dgamma, dbeta, work, rows, n, dy_type="f32", in_type="f32")
    gen = torch.Generator().manual_seed(6)
    for which, grad in enumerate((dx, dgamma, dbeta)):
        v = torch.randn(grad.shape, generator=gen, dtype=torch.float64)
        values = []
        for step in (1e-5, -1e-5):
            args = [x.double(), gamma.double(), beta.double()]
            args[which] = args[which] + step * v
            values.append((dy.double() * ref.norm(*args, EPS)[0]).sum().item())
        slope, got = (values[0] - values[1]) / 2e-5, (grad.double().cpu() * v).sum().item()
        # float roundings of terms of random sign, and the differences' own (step^2 and what is lost of the values)
        assert abs(got - slope) <= 1e-4 * (grad.double().cpu() * v).norm().item() + 1e-7 * abs(slope) + 1e-5


@pytest.mark.gpu
def test_gradients_without_rows(gpu):
    dgamma, dbeta = torch.full((2, 500), 7.0, device="cuda")
    work = torch.empty(256, dtype=torch.uint8, device="cuda")
    lib.layer_norm_backward(None, None, None, None, dgamma, dbeta, work, 0, 500)
    assert not dgamma.any() and not dbeta.any()


@pytest.mark.gpu
def test_large_offsets(gpu):
    """Rows that begin beyond 4 GiB, and more rows than one axis of a launch holds."""
    rows, n = (1 << 20) + 9, 2100
    x = torch.empty(rows, n, dtype=torch.bfloat16, device="cuda")
    for at in range(0, rows, 1 << 18):
        x[at : at + (1 << 18)].normal_(generator=torch.Generator("cuda").manual_seed(at))
    y, dx = torch.empty_like(x), torch.empty_like(x)
    dgamma, dbeta = torch.empty(2, n, device="cuda")
    work = torch.empty(lib.layer_norm_backward_bytes(rows, n), dtype=torch.uint8, device="cuda")
    gamma, beta = (t.cuda() for t in vectors(1, n))
    lib.layer_norm(x, gamma, beta, y, rows, n)
    lib.layer_norm_backward(x, x, gamma, dx, dgamma, dbeta, work, rows, n)
    for at in (slice(0, 2), slice(rows - 12, rows)):
        ref.check(y[at], *ref.norm(x[at], gamma, beta, EPS), "bf16")
        ref.check(dx[at], *ref.norm_gradients(x[at], x[at], gamma, EPS)[0], "bf16")
    # sums over a million rows: terms x^2 / sqrt(variance) about 1 (and of mean 1), float sums of strips
    want = torch.zeros(2, n, dtype=torch.float64, device="cuda")
    for at in range(0, rows, 1 << 16):
        v = x[at : at + (1 << 16)]
        h = ref.normalised(v, EPS)[0]
        want += torch.stack(((v.double() * h).sum(0), v.double().sum(0)))
    size = 1.1 * rows  # sums of |x h| and |x|, and what h is off
    assert (dgamma.double() - want[0]).abs().max().item() < size * (rows / 256 + 256) * ref.U
    assert (dbeta.double() - want[1]).abs().max().item() < size * (rows / 256 + 256) * ref.U


@pytest.mark.gpu
@pytest.mark.parametrize("rows, n", [(5, 40), (300, 1000), (70, 20000), (3, 40000)])
def test_results_do_not_change(gpu, rows, n):
    """The same bits on any stream and whatever the workspace held."""
    x, gamma = rows_of(1, rows, n, "bf16").cuda(), vectors(2, n)[0].cuda()
    dy, first = torch.randn(rows, n, device="cuda").bfloat16(), None
    for i, stream in enumerate((torch.cuda.current_stream(), torch.cuda.Stream(), torch.cuda.Stream())):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            dx, dgamma, dbeta = torch.empty_like(x), torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
            work = torch.full((lib.layer_norm_backward_bytes(rows, n),), 0x7F * i, dtype=torch.uint8, device="cuda")
            lib.layer_norm_backward(dy, x, gamma, dx, dgamma, dbeta, work, rows, n)
        torch.cuda.synchronize()
        first = first or (dx, dgamma, dbeta)
        assert all(torch.equal(a, b) for a, b in zip(first, (dx, dgamma, dbeta)))


@pytest.mark.gpu
@pytest.mark.parametrize("m, n, k", [(1, 300, 200), (20, 320, 512), (90, 777, 1030)])
def test_a_norm_and_its_layer(gpu, m, n, k):
    """Norm into 8 bits, product, and back: dx of the layer is dy of the norm.  Eager against float64, then captured and replayed."""
    (wq, w) = matrix(2, n, k, 1.0 / math.sqrt(k))
    w = w.cuda()
    gamma, beta = (t.cuda() for t in vectors(k, k))
    x, dy = torch.empty(m, k, device="cuda"), torch.empty(m, n, dtype=torch.bfloat16, device="cuda")
    hq = torch.empty(m, ref.up(k, 128), dtype=torch.int8, device="cuda"), torch.empty(m, device="cuda")
    y, dh, dw = torch.empty(m, n, device="cuda"), torch.empty(m, k, dtype=torch.bfloat16, device="cuda"), torch.empty(n, k, device="cuda")
    dx, dgamma, dbeta = torch.empty(m, k, device="cuda"), torch.empty(k, device="cuda"), torch.empty(k, device="cuda")
    work = torch.empty(max(lib.int8_linear_backward_bytes(m, n, k, "f32"), lib.layer_norm_backward_bytes(m, k)), dtype=torch.uint8, device="cuda")

    def step():
        lib.layer_norm_int8(x, gamma, beta, *hq, m, k, in_type="f32")
        lib.int8_linear(*hq, *wq, None, y, "f32", m, n, k)
        lib.int8_linear_backward(dy, *hq, *wq, dh, dw, "f32", None, work, m, n, k)
        lib.layer_norm_backward(dh, x, gamma, dx, dgamma, dbeta, work, m, k, dy_type="bf16", in_type="f32")

    outs = (y, dh, dw, dx, dgamma, dbeta)
    x.copy_(rows_of(5, m, k, "f32"))
    dy.copy_(torch.randn(m, n, generator=torch.Generator().manual_seed(1)))
    step()
    h, error = ref.norm(x, gamma, beta, EPS)
    got = ref.decode(*hq, k)
    scale = hq[1].double()[:, None]
    assert bool(((got - h).abs() <= error + scale * (0.5 + 127 * 2 * ref.U)).all())
    ref.check(y, *product(got, w), "f32")
    d = dy.double()
    ref.check(dh, d @ w, (2.0**-8 + n * 2.0**-23) * (d.abs() @ w.abs()), "bf16")
    ref.check(dw, d.T @ got, (2.0**-24 + 3 * m * 2.0**-23) * (d.abs().T @ got.abs()), "f32")
    for value, (want, e) in zip((dx, dgamma, dbeta), ref.norm_gradients(dh, x, gamma, EPS)):
        ref.check(value, want, e, "f32")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for seed in range(4):
        x.copy_(rows_of(seed, m, k, "f32"))
        dy.copy_(torch.randn(m, n, generator=torch.Generator().manual_seed(seed)))
        work.fill_(0xFF)
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in outs]
        for t in outs:
            t.zero_()
        step()
        torch.cuda.synchronize()
        assert all(bool(a.any()) and torch.equal(a, b) for a, b in zip(replayed, outs))


@pytest.mark.gpu
def test_the_example_runs_and_its_gradients(gpu):
    import importlib.util
    from pathlib import Path

    spec = importlib.util.spec_from_file_location("int8_norm_linear", Path(__file__).resolve().parent.parent / "examples" / "int8_norm_linear.py")
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    tokens, hidden, out = 96, 128, 320
    x = torch.randn(tokens, hidden, device="cuda", generator=torch.Generator("cuda").manual_seed(1)) * 2 + 1
    target = example.NormLinear(tokens, hidden, out, seed=2).forward(x).float()
    layer = example.NormLinear(tokens, hidden, out)
    assert all(math.isfinite(v) for v in example.train(layer, x, target, 5, 0.02))
    # gradients at the values that the quantised operands stand for
    layer.forward(x)
    dy = torch.randn(tokens, out, device="cuda").bfloat16()
    dx = layer.backward(x, dy)
    h, w, d = ref.decode(*layer.hq, hidden), ref.decode(*layer.wq, hidden), dy.double()
    dw, dbias, dgamma, dbeta = layer.grads
    ref.check(layer.dh, d @ w, (2.0**-8 + out * 2.0**-23) * (d.abs() @ w.abs()), "bf16")
    ref.check(dw, d.T @ h, (2.0**-24 + 3 * tokens * 2.0**-23) * (d.abs().T @ h.abs()), "f32")
    ref.check(dbias, d.sum(0), tokens * 2.0**-23 * d.abs().sum(0), "f32")
    for value, (want, e) in zip((dx, dgamma, dbeta), ref.norm_gradients(layer.dh, x, layer.gamma, EPS)):
        ref.check(value, want, e, "f32")
    # one token at a time from a graph, eager work between the replays
    token = x[:1].clone()
    want = [layer.forward(x[i : i + 1].contiguous()).clone() for i in range(4)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer.forward(token)
    for i in range(4):
        token.copy_(x[i : i + 1])
        graph.replay()
        assert torch.equal(y, want[i])
        layer.forward(x)
        torch.cuda.synchronize()


# ---- rows of very large values


def work_of(rows, n):
    return torch.empty(lib.layer_norm_backward_bytes(rows, n), dtype=torch.uint8, device="cuda")


def large_rows(n, kind):
    """Finite rows whose squares (of x - mean) add up to more than a float holds, and an ordinary one behind them: large values, one and two
    of the type's lowest among ordinary ones, sums and differences that are no float either, and a constant row whose mean is not met exactly."""
    gen = torch.Generator().manual_seed(n)
    z = torch.randn(11, n, generator=gen)
    top = torch.finfo(ref.DTYPE[kind]).max
    z[0] *= 1e27
    z[1] *= 1e29
    z[2] *= 1e31
    z[3] *= 1e37
    z[4, n // 2] = -top
    z[5, 0] = z[5, n - 1] = -top
    z[6] = top * (1 - 2 * (torch.arange(n) % 2))
    z[7] = top * torch.where(torch.arange(n) % 4 == 3, -1.0, 1.0)
    z[8, 1] = top
    z[9] = 0.97 * top
    z[9, 0] = 0.9 * top
    return z.to(ref.DTYPE[kind])


@pytest.mark.gpu
@pytest.mark.parametrize("n", [8, 64, 100, 250, 500, 1000, 2000, 3001, 5000, 9000, 16000, 40000])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("copies", [1, 110])
def test_finite_rows_without_a_variance_in_floats(gpu, n, kind, copies):
    """They give beta, in every form; their dx is zero, and of what is summed over rows they have a share of dbeta alone."""
    rows = 11 * copies
    x = large_rows(n, kind).repeat(copies, 1).cuda()
    gamma, beta = (t.cuda() for t in vectors(n, n))
    y, z = torch.empty(2, rows, n, device="cuda")
    lib.layer_norm(x, gamma, beta, y, rows, n, eps=EPS, in_type=kind, out_type="f32")
    flat = torch.arange(rows, device="cuda") % 11 < 10
    assert torch.equal(y[flat], beta.expand(10 * copies, n))
    ref.check(y[~flat], *ref.norm(x[~flat], gamma, beta, EPS), "f32")
    lib.layer_norm(x, None, None, z, rows, n, eps=EPS, in_type=kind, out_type="f32")
    assert not z[flat].any()
    for fused, apart, sizes in ((lib.layer_norm_int8, lib.int8_quantize, (lib.int8_code_bytes(rows, n), 4 * rows)),
                                (lib.layer_norm_mxfp4, lib.mxfp4_quantize, (lib.mxfp4_code_bytes(rows, n), lib.mxfp4_scale_bytes(rows, n)))):
        got, want = ([torch.empty(size, dtype=torch.uint8, device="cuda") for size in sizes] for _ in range(2))
        fused(x, gamma, beta, *got, rows, n, eps=EPS, in_type=kind)
        apart(y, *want, rows, n, in_type="f32")
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    dy = torch.randn(rows, n, generator=torch.Generator().manual_seed(1)).cuda()
    dx, dgamma, dbeta = torch.empty_like(x), torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    lib.layer_norm_backward(dy, x, gamma, dx, dgamma, dbeta, work_of(rows, n), rows, n, eps=EPS, dy_type="f32", in_type=kind)
    (want_dx, e_dx), (want_dgamma, e_dgamma), _ = ref.norm_gradients(dy[~flat], x[~flat], gamma, EPS)
    assert not dx[flat].any()
    ref.check(dx[~flat], want_dx, e_dx, kind)
    ref.check(dgamma, want_dgamma, e_dgamma, "f32")
    ref.check(dbeta, dy.double().sum(0), (rows + 2) * ref.U * dy.double().abs().sum(0), "f32")


#: what a constant row's values are: from where a rounding of the mean begins to count to where squares of what it leaves are no float
CONSTANTS = [1.1e7, 1.1e9, 1.3e10, 1.7e12, 1.1e15, 1.9e18, 1.3e20, 1.1e24, 1.7e27, 1.1e33]


@pytest.mark.gpu
@pytest.mark.parametrize("n", [7, 100, 250, 500, 700, 1000, 1500, 3001, 5000, 9001, 16001, 40001, 100001])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_constant_rows_of_any_size(gpu, n, kind):
    """Whatever a rounding of the mean leaves of x - mean, the same in every column, is no deviation: y is beta."""
    x = torch.tensor(CONSTANTS)[:, None].expand(-1, n).to(ref.DTYPE[kind]).contiguous().cuda()
    rows = len(CONSTANTS)
    y = torch.empty(rows, n, device="cuda")
    lib.layer_norm(x, None, None, y, rows, n, eps=EPS, in_type=kind, out_type="f32")
    # With d what is left, the same in all columns, h = (d - mean(d)) r: a mean of `depth` additions and two more roundings, each U of itself.
    # Either the row counts as one without deviations, or its variance is 2^-22 of mean(d)^2 at least and |mean(d)| r 2^11 at most.
    depth = n / 64 + 24
    assert y.abs().max().item() <= (depth + 4) * ref.U * 2.0**11
    dy = torch.randn(rows, n, generator=torch.Generator().manual_seed(1)).cuda()
    dx, dgamma = torch.empty(rows, n, device="cuda").to(ref.DTYPE[kind]), torch.empty(n, device="cuda")
    lib.layer_norm_backward(dy, x, None, dx, dgamma, None, work_of(rows, n), rows, n, eps=EPS, dy_type="f32", in_type=kind)
    assert bool(torch.isfinite(dx).all()) and bool((dgamma.abs() <= (depth + 4) * ref.U * 2.0**11 * dy.abs().sum(0)).all())


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1000, 16001, 100001])
def test_rows_that_are_constant_but_for_a_few_columns(gpu, n):
    """Deviations of one unit in the last place, that eps is large beside: they stay, as small as they are."""
    x = torch.tensor([1050.8, 1.3, 7777.7])[:, None].repeat(1, n)
    x[:, [1, n // 2, n - 1]] *= 1 + 2.0**-23
    x = x.cuda()
    gamma, beta = (t.cuda() for t in vectors(n, n))
    y, dx, dgamma = torch.empty(3, n, device="cuda"), torch.empty(3, n, device="cuda"), torch.empty(n, device="cuda")
    lib.layer_norm(x, gamma, beta, y, 3, n, eps=EPS, in_type="f32", out_type="f32")
    ref.check(y, *ref.norm(x, gamma, beta, EPS), "f32")
    dy = torch.randn(3, n, generator=torch.Generator().manual_seed(1)).cuda()
    lib.layer_norm_backward(dy, x, gamma, dx, dgamma, None, work_of(3, n), 3, n, eps=EPS, dy_type="f32", in_type="f32")
    for value, (want, error) in zip((dx, dgamma), ref.norm_gradients(dy, x, gamma, EPS)):
        ref.check(value, want, error, "f32")


# ---- kernels that stay for several rows, and those that many rows choose


#: rows, n: for every way in which rows are dealt to waves, three turns of a workgroup and more
TURNS = [(70000, 40), (70000, 64), (40000, 128), (20000, 250), (9000, 500), (9001, 1000), (7000, 2000), (2501, 4000), (1000, 3000), (2000, 8000),
         (1030, 8192), (1300, 4999), (1100, 12001), (600, 16384), (601, 9001)]


@pytest.mark.gpu
@pytest.mark.parametrize("rows, n", TURNS)
@pytest.mark.parametrize("kind, out", [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "bf16")])
def test_every_row_of_many(gpu, rows, n, kind, out):
    x = rows_of(rows + n, rows, n, kind).cuda()
    gamma, beta = (t.cuda() for t in vectors(n, n))
    raw, y = guarded(rows * n * ref.DTYPE[out].itemsize)
    lib.layer_norm(x, gamma, beta, y, rows, n, eps=EPS, in_type=kind, out_type=out)
    torch.cuda.synchronize()
    assert untouched(raw)
    ref.check(y.view(ref.DTYPE[out]).view(rows, n), *ref.norm(x, gamma, beta, EPS), out)


@pytest.mark.gpu
@pytest.mark.parametrize("rows, n", TURNS)
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_every_quantised_row_of_many(gpu, rows, n, kind):
    """Bit for bit what the norm as floats gives after its quantisation, which takes other kernels."""
    x = rows_of(rows + n, rows, n, kind).cuda()
    gamma, beta = (t.cuda() for t in vectors(n, n))
    y = torch.empty(rows, n, device="cuda")
    lib.layer_norm(x, gamma, beta, y, rows, n, in_type=kind, out_type="f32")
    ref.check(y, *ref.norm(x, gamma, beta, EPS), "f32")
    for fused, apart, sizes in ((lib.layer_norm_int8, lib.int8_quantize, (lib.int8_code_bytes(rows, n), 4 * rows)),
                                (lib.layer_norm_mxfp4, lib.mxfp4_quantize, (lib.mxfp4_code_bytes(rows, n), lib.mxfp4_scale_bytes(rows, n)))):
        (raw_c, codes), (raw_s, scales) = guarded(sizes[0]), guarded(sizes[1])
        want = [torch.empty(size, dtype=torch.uint8, device="cuda") for size in sizes]
        fused(x, gamma, beta, codes, scales, rows, n, in_type=kind)
        apart(y, *want, rows, n, in_type="f32")
        torch.cuda.synchronize()
        assert untouched(raw_c) and untouched(raw_s) and torch.equal(codes, want[0]) and torch.equal(scales, want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("rows, n", [(70000, 64), (40000, 128), (20000, 250), (9000, 500), (5001, 1000), (2500, 2000), (1100, 4000), (600, 8000),
                                     (600, 16384), (900, 9001), (300, 20000)])
@pytest.mark.parametrize("kind, dy_kind", [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "bf16"), ("bf16", "f32")])
def test_gradients_of_many_rows(gpu, rows, n, kind, dy_kind):
    x = rows_of(rows + n, rows, n, kind, spread=0.5).cuda()
    dy = torch.randn(rows, n, generator=torch.Generator().manual_seed(rows)).to(ref.DTYPE[dy_kind]).cuda()
    gamma = vectors(n, n)[0].cuda()
    (raw_x, dx), (raw_g, dgamma), (raw_b, dbeta) = guarded(rows * n * ref.DTYPE[kind].itemsize), guarded(4 * n), guarded(4 * n)
    lib.layer_norm_backward(dy, x, gamma, dx, dgamma, dbeta, work_of(rows, n), rows, n, dy_type=dy_kind, in_type=kind)
    torch.cuda.synchronize()
    assert untouched(raw_x) and untouched(raw_g) and untouched(raw_b)
    got = dx.view(ref.DTYPE[kind]).view(rows, n), dgamma.view(torch.float32), dbeta.view(torch.float32)
    for value, (want, error), out in zip(got, ref.norm_gradients(dy, x, gamma, EPS), (kind, "f32", "f32")):
        ref.check(value, want, error, out)


# ---- the ends of the ranges


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_the_longest_rows(gpu, kind):
    """2^22 columns, the last of them with the largest values: a plain sum of them would be 2^22 times what a float holds."""
    rows, n = 3, 1 << 22
    x = rows_of(5, rows, n, kind)
    x[2] = torch.finfo(ref.DTYPE[kind]).max
    x = x.cuda()
    gamma, beta = (t.cuda() for t in vectors(1, n))
    y = torch.empty(rows, n, device="cuda")
    lib.layer_norm(x, gamma, beta, y, rows, n, eps=EPS, in_type=kind, out_type="f32")
    ref.check(y[:2], *ref.norm(x[:2], gamma, beta, EPS), "f32")
    assert torch.equal(y[2], beta)
    dy = torch.randn(rows, n, generator=torch.Generator().manual_seed(2)).cuda()
    dx, dgamma, dbeta = torch.empty_like(x), torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    lib.layer_norm_backward(dy, x, gamma, dx, dgamma, dbeta, work_of(rows, n), rows, n, eps=EPS, dy_type="f32", in_type=kind)
    (want_dx, e_dx), (want_dgamma, e_dgamma), _ = ref.norm_gradients(dy[:2], x[:2], gamma, EPS)
    ref.check(dx[:2], want_dx, e_dx, kind)
    assert bool(torch.isfinite(dx[2]).all())
    ref.check(dgamma, want_dgamma, e_dgamma, "f32")
    ref.check(dbeta, dy.double().sum(0), (rows + 2) * ref.U * dy.double().abs().sum(0), "f32")


@pytest.mark.gpu
def test_very_many_short_rows(gpu):
    """2^25 rows and a few: beyond what one axis of a launch holds, in every form and back."""
    rows, n = (1 << 25) + 5, 3
    x = torch.randn(rows, n, generator=torch.Generator("cuda").manual_seed(1), device="cuda") + 2
    gamma, beta = (t.cuda() for t in vectors(1, n))
    y = torch.empty_like(x)
    lib.layer_norm(x, gamma, beta, y, rows, n, eps=EPS, in_type="f32", out_type="f32")
    ref.check(y, *ref.norm(x, gamma, beta, EPS), "f32")
    codes, scales = torch.empty(rows, 128, dtype=torch.int8, device="cuda"), torch.empty(rows, device="cuda")
    want = torch.empty_like(codes), torch.empty_like(scales)
    lib.layer_norm_int8(x, gamma, beta, codes, scales, rows, n, in_type="f32")
    lib.int8_quantize(y, *want, rows, n, in_type="f32")
    assert torch.equal(codes, want[0]) and torch.equal(scales, want[1])
    del codes, scales, want
    dx, dgamma, dbeta = torch.empty_like(x), torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    lib.layer_norm_backward(x, x, gamma, dx, dgamma, dbeta, work_of(rows, n), rows, n, eps=EPS, dy_type="f32", in_type="f32")
    for value, (want, error) in zip((dx, dgamma, dbeta), ref.norm_gradients(x, x, gamma, EPS)):
        ref.check(value, want, error, "f32")
