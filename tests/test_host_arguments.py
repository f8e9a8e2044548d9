"""What the Python mirror takes as an operand, without a device."""
import numpy as np
import pytest
import torch

import int4linear_amd as lib
from int4linear_amd import api


def test_addresses_of_operands():
    t, a = torch.zeros(4), np.zeros(4)
    assert api._ptr(t) == t.data_ptr() and api._ptr(a) == a.ctypes.data and api._ptr(4096) == 4096 and api._ptr(None) == 0
    assert api._ptr(torch.nn.Parameter(t)) == t.data_ptr()


@pytest.mark.parametrize("wrong", [b"sixteen bytes...", "text", [1, 2], 4096.0, object()])
def test_objects_without_an_address_are_refused(wrong):
    """bytes and str are pointers to host memory for ctypes: they must not get that far."""
    A = 4096
    calls = [lambda: lib.gemm_s4s4s32(wrong, A, A, 1, 1, 8, stream=0), lambda: lib.gemm_s4s4s32(A, wrong, A, 1, 1, 8, stream=0),
             lambda: lib.linear_s32(A, A, wrong, A, 1, 1, 8, stream=0), lambda: lib.mxfp4_quantize(wrong, A, A, 1, 8, stream=0),
             lambda: lib.mxfp4_linear(A, A, A, wrong, None, A, "f32", 1, 1, 8, stream=0),
             lambda: lib.mxfp4_linear_backward(A, A, A, A, A, wrong, A, "f32", None, None, 1, 1, 8, stream=0)]
    for call in calls:
        with pytest.raises(AttributeError, match="data_ptr"):
            call()


def test_a_workspace_may_be_an_address_with_its_size():
    """Each is refused by the library for what it is (2: null, 3: alignment, 7: too small), not by Python on the way."""
    A, need = 4096, lib.mxfp4_linear_backward_bytes(10, 20, 30)

    def linear(work, **size):
        lib.mxfp4_linear_backward(A, A, A, A, A, A, A, "f32", A, work, 10, 20, 30, stream=0, **size)

    def gated(work, **size):
        lib.mxfp4_gated_backward(A, A, A, A, A, A, A, A, A, A, "f32", work, 10, 20, 30, stream=0, **size)

    for call in (linear, gated):
        for work, size, status in ((A, 0, 7), (A + 16, 1 << 40, 3), (None, 0, 2)):
            with pytest.raises(lib.Int4LinearError, match=f"status {status}"):
                call(work, work_bytes=size)
        with pytest.raises(lib.Int4LinearError, match="status 2"):
            call(None)
        with pytest.raises(TypeError, match="work_bytes"):
            call(A)
    with pytest.raises(lib.Int4LinearError, match="status 7"):
        linear(A, work_bytes=need - 1)
    # a tensor says its size itself; a smaller one given for it is believed
    work = torch.empty(need + 512, dtype=torch.uint8)
    work = work[-work.data_ptr() % 256 :]
    assert api._work(work, None) == (work.data_ptr(), work.numel()) and api._work(work, 256) == (work.data_ptr(), 256)
    with pytest.raises(lib.Int4LinearError, match="status 7"):
        linear(work, work_bytes=need - 1)


def test_sizes_beyond_a_tiles_offsets_are_refused():
    """A product's k to 2^22, every size of a gradient to 2^22 - 64: there the offset of a tile's last row still fits 32 bits."""
    A, most = 4096, (1 << 22) - 64
    assert 255 * 4 * most + 128 <= 1 << 32 < 255 * 4 * (most + 64 * 300)
    with pytest.raises(lib.Int4LinearError, match="status 5"):
        lib.mxfp4_linear(A, A, A, A, None, A, "f32", 1, 1, (1 << 22) + 1, stream=0)
    for sizes, status in (((most, 1, 1), 7), ((1, most, 1), 7), ((1, 1, most), 7), ((most + 1, 1, 1), 5), ((1, most + 1, 1), 5), ((1, 1, most + 1), 5)):
        with pytest.raises(lib.Int4LinearError, match=f"status {status}"):
            lib.mxfp4_linear_backward(A, A, A, A, A, A, A, "f32", A, A, *sizes, work_bytes=0, stream=0)
        with pytest.raises(lib.Int4LinearError, match=f"status {status}"):
            lib.mxfp4_gated_backward(A, A, A, A, A, A, A, A, A, A, "f32", A, *sizes, work_bytes=0, stream=0)
