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
