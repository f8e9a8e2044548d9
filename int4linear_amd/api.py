"""Host-side mirror of the reference's interface, on top of the C ABI.

Names and argument meaning follow the reference:
  linear_vN_launch(x_packed_d, w_packed_d, y_d, m, n, k)   kernels/linear_v21.h:760 (and v0..v20)
  pack(src, dst, m, n) / unpack(src, dst, m, n)            utils/packer.h:5-6
Device operands are torch tensors on a ROCm device (torch is only the owner of the
device memory and the stream) or raw integer device addresses.
"""
from __future__ import annotations

import numpy as np

from . import _lib

KERNELS = {"auto": 0, "simple": 1, "mfma": 2, "skinny": 3, "fp6": 4, "mfma128": 5, "mfma256": 6}


_HOST_KINDS = (int, np.ndarray)


def _ptr(obj) -> int:
    """Device (or host) address of a torch tensor / numpy array / raw int."""
    if obj is None:
        return 0
    if isinstance(obj, _HOST_KINDS):  # (one check for both: a call asks for up to ten tensors, at 0.2 us each)
        return obj if isinstance(obj, int) else obj.ctypes.data
    return obj.data_ptr()  # torch.Tensor


def _current_stream() -> int:
    """The handle torch.cuda.current_stream().cuda_stream gives, asked for without the Stream object that
    call makes: 2.7 us, longer than the smallest kernels run and more than a third of a call's 7.4 us on
    the host, against 0.3.  (A torch without that private function is asked the long way.)"""
    import torch

    if torch.cuda.is_initialized():  # (else torch sets itself up, or says why it cannot)
        try:
            return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())
        except AttributeError:
            pass
    return torch.cuda.current_stream().cuda_stream


def init() -> None:
    """One-time device set-up (idempotent)."""
    lib = _lib.load()
    _lib.check(lib.int4linear_init())


def gemm_s4s4s32(a_packed_d, b_packed_d, c_d, m: int, n: int, k: int, *, kernel: str = "auto",
                 stream: int | None = None) -> None:
    """Asynchronous C = A * B^T on `stream` (default: torch's current stream)."""
    lib = _lib.load()
    if stream is None:
        stream = _current_stream()
    st = lib.int4linear_gemm_s4s4s32_ex(_ptr(a_packed_d), _ptr(b_packed_d), _ptr(c_d), m, n, k,
                                        KERNELS[kernel], stream)
    _lib.check(st)


STATIC_SCRATCH_BYTES = 128 << 20  # INT4LINEAR_STATIC_SCRATCH_BYTES


def gemm_s4s4s32_static(a_packed_d, b_packed_d, c_d, m: int, n: int, k: int, *, stream: int | None = None) -> None:
    """gemm_s4s4s32 with automatic dispatch on the library's fixed scratch array: allocates
    nothing; shapes that need more scratch than the array holds raise (status 7)."""
    lib = _lib.load()
    if stream is None:
        stream = _current_stream()
    _lib.check(lib.int4linear_gemm_s4s4s32_static(_ptr(a_packed_d), _ptr(b_packed_d), _ptr(c_d), m, n, k,
                                                  stream))


def linear_s32(x_packed_d, w_packed_d, bias_d, y_d, m: int, n: int, k: int, *, kernel: str = "auto",
               stream: int | None = None) -> None:
    """Y = X * W^T + bias (int32); bias_d may be None."""
    lib = _lib.load()
    if stream is None:
        stream = _current_stream()
    _lib.check(lib.int4linear_linear_s32(_ptr(x_packed_d), _ptr(w_packed_d), _ptr(bias_d), _ptr(y_d), m, n, k,
                                         KERNELS[kernel], stream))


def linear_f32(x_packed_d, w_packed_d, bias_d, row_scale_d, col_scale_d, y_d, m: int, n: int, k: int, *,
               kernel: str = "auto", stream: int | None = None) -> None:
    """Y (float32) = ((float)(X * W^T + bias) * row_scale[i]) * col_scale[j]; each of bias_d,
    row_scale_d, col_scale_d may be None."""
    lib = _lib.load()
    if stream is None:
        stream = _current_stream()
    _lib.check(lib.int4linear_linear_f32(_ptr(x_packed_d), _ptr(w_packed_d), _ptr(bias_d), _ptr(row_scale_d),
                                         _ptr(col_scale_d), _ptr(y_d), m, n, k, KERNELS[kernel],
                                         stream))


def linear_f16(x_packed_d, w_packed_d, bias_d, row_scale_d, col_scale_d, y_d, m: int, n: int, k: int, *,
               kernel: str = "auto", stream: int | None = None) -> None:
    """Y (float16) = the value of linear_f32 rounded to nearest even once more."""
    lib = _lib.load()
    if stream is None:
        stream = _current_stream()
    _lib.check(lib.int4linear_linear_f16(_ptr(x_packed_d), _ptr(w_packed_d), _ptr(bias_d), _ptr(row_scale_d),
                                         _ptr(col_scale_d), _ptr(y_d), m, n, k, KERNELS[kernel],
                                         stream))


def linear_bf16(x_packed_d, w_packed_d, bias_d, row_scale_d, col_scale_d, y_d, m: int, n: int, k: int, *,
                kernel: str = "auto", stream: int | None = None) -> None:
    """Y (bfloat16) = the value of linear_f32 rounded to nearest even once more."""
    lib = _lib.load()
    if stream is None:
        stream = _current_stream()
    _lib.check(lib.int4linear_linear_bf16(_ptr(x_packed_d), _ptr(w_packed_d), _ptr(bias_d), _ptr(row_scale_d),
                                          _ptr(col_scale_d), _ptr(y_d), m, n, k, KERNELS[kernel],
                                          stream))


def fp6_operand_bytes(rows: int, k: int) -> int:
    """Bytes of the converted (FP6) form of a rows x k operand; 0 if k is unsupported."""
    return int(_lib.load().int4linear_fp6_operand_bytes(rows, k))


def fp6_convert(packed_d, converted_d, rows: int, k: int, *, stream: int | None = None) -> None:
    """Packed s4 operand -> the FP6 kernel's own operand form (convert static weights once)."""
    lib = _lib.load()
    if stream is None:
        stream = _current_stream()
    _lib.check(lib.int4linear_fp6_convert(_ptr(packed_d), _ptr(converted_d), rows, k, stream))


def gemm_fp6_converted(a_conv_d, b_conv_d, c_d, m: int, n: int, k: int, *, stream: int | None = None) -> None:
    """C = A * B^T from two operands already converted with fp6_convert."""
    lib = _lib.load()
    if stream is None:
        stream = _current_stream()
    _lib.check(lib.int4linear_gemm_fp6_converted(_ptr(a_conv_d), _ptr(b_conv_d), _ptr(c_d), m, n, k,
                                                 stream))


OUT_TYPES = {"s32": 0, "f32": 1, "f16": 2, "bf16": 3}  # INT4LINEAR_OUT_*


def linear_fp6_converted(x_conv_d, w_conv_d, bias_d, row_scale_d, col_scale_d, y_d, out_type: str, m: int, n: int,
                         k: int, *, stream: int | None = None) -> None:
    """gemm_fp6_converted with the epilogue of linear_s32 / linear_f32 / linear_f16 / linear_bf16
    (out_type "s32", "f32", "f16" or "bf16"); bias_d and the scales may each be None."""
    lib = _lib.load()
    if stream is None:
        stream = _current_stream()
    _lib.check(lib.int4linear_linear_fp6_converted(_ptr(x_conv_d), _ptr(w_conv_d), _ptr(bias_d), _ptr(row_scale_d),
                                                   _ptr(col_scale_d), _ptr(y_d), OUT_TYPES[out_type], m, n, k,
                                                   stream))


ACTIVATIONS = {"silu": 0, "gelu": 1}  # INT4LINEAR_ACT_*


def mxfp4_code_bytes(rows: int, k: int) -> int:
    """Bytes of a rows x k matrix's codes in MXFP4 (a row: 128 per 256 k begun)."""
    return int(_lib.load().int4linear_mxfp4_code_bytes(rows, k))


def mxfp4_scale_bytes(rows: int, k: int) -> int:
    """Bytes of a rows x k matrix's scales in MXFP4 (a row: 16 per 512 k begun)."""
    return int(_lib.load().int4linear_mxfp4_scale_bytes(rows, k))


def mxfp4_quantize(x_d, codes_d, scales_d, rows: int, k: int, *, in_type: str = "bf16", ld: int | None = None,
                   stream: int | None = None) -> None:
    """x_d (rows x k of in_type "f32", "f16" or "bf16", ld elements between rows, k if None) -> MXFP4."""
    lib = _lib.load()
    if stream is None:
        stream = _current_stream()
    _lib.check(lib.int4linear_mxfp4_quantize(_ptr(x_d), OUT_TYPES[in_type], k if ld is None else ld, _ptr(codes_d),
                                             _ptr(scales_d), rows, k, stream))


def mxfp4_dequantize(codes_d, scales_d, y_d, rows: int, k: int, *, out_type: str = "bf16", ld: int | None = None,
                     stream: int | None = None) -> None:
    """MXFP4 -> y_d (rows x k of out_type, ld elements between rows, k if None)."""
    lib = _lib.load()
    if stream is None:
        stream = _current_stream()
    _lib.check(lib.int4linear_mxfp4_dequantize(_ptr(codes_d), _ptr(scales_d), _ptr(y_d), OUT_TYPES[out_type],
                                               k if ld is None else ld, rows, k, stream))


def mxfp4_linear(x_codes_d, x_scales_d, w_codes_d, w_scales_d, bias_d, y_d, out_type: str, m: int, n: int, k: int, *,
                 stream: int | None = None) -> None:
    """Y (m x n of out_type) = X * W^T + bias for MXFP4 operands; bias_d (n float32) may be None."""
    lib = _lib.load()
    if stream is None:
        stream = _current_stream()
    _lib.check(lib.int4linear_mxfp4_linear(_ptr(x_codes_d), _ptr(x_scales_d), _ptr(w_codes_d), _ptr(w_scales_d),
                                           _ptr(bias_d), _ptr(y_d), OUT_TYPES[out_type], m, n, k, stream))


def mxfp4_gated(x_codes_d, x_scales_d, wg_codes_d, wg_scales_d, wu_codes_d, wu_scales_d, h_d, out_type: str, m: int,
                n: int, k: int, *, activation: str = "silu", stream: int | None = None) -> None:
    """H (m x n of out_type) = act(X * Wg^T) * (X * Wu^T) in one kernel; activation "silu" or "gelu"."""
    lib = _lib.load()
    if stream is None:
        stream = _current_stream()
    _lib.check(lib.int4linear_mxfp4_gated(_ptr(x_codes_d), _ptr(x_scales_d), _ptr(wg_codes_d), _ptr(wg_scales_d),
                                          _ptr(wu_codes_d), _ptr(wu_scales_d), ACTIVATIONS[activation], _ptr(h_d),
                                          OUT_TYPES[out_type], m, n, k, stream))


def mxfp4_gated_quantized(x_codes_d, x_scales_d, wg_codes_d, wg_scales_d, wu_codes_d, wu_scales_d, h_codes_d,
                          h_scales_d, m: int, n: int, k: int, *, activation: str = "silu",
                          stream: int | None = None) -> None:
    """mxfp4_gated with H in MXFP4, the form the down projection takes."""
    lib = _lib.load()
    if stream is None:
        stream = _current_stream()
    _lib.check(lib.int4linear_mxfp4_gated_quantized(_ptr(x_codes_d), _ptr(x_scales_d), _ptr(wg_codes_d),
                                                    _ptr(wg_scales_d), _ptr(wu_codes_d), _ptr(wu_scales_d),
                                                    ACTIVATIONS[activation], _ptr(h_codes_d), _ptr(h_scales_d), m, n, k,
                                                    stream))


def _work(work_d, work_bytes: int | None) -> tuple[int, int]:
    """Address and bytes of a workspace: a tensor, None, or an address, which needs work_bytes."""
    if work_bytes is None:
        if isinstance(work_d, int):
            raise TypeError("a workspace given as an address needs work_bytes")
        work_bytes = 0 if work_d is None else work_d.numel() * work_d.element_size()
    return _ptr(work_d), work_bytes


def mxfp4_linear_backward_bytes(m: int, n: int, k: int) -> int:
    """Bytes of workspace mxfp4_linear_backward needs."""
    return int(_lib.load().int4linear_mxfp4_linear_backward_bytes(m, n, k))


def mxfp4_linear_backward(dy_d, x_codes_d, x_scales_d, w_codes_d, w_scales_d, dx_d, dw_d, dw_type: str, dbias_d, work_d,
                          m: int, n: int, k: int, *, work_bytes: int | None = None, stream: int | None = None) -> None:
    """dx (bfloat16) = dy W, dw (dw_type "bf16" or "f32") = dy^T X, dbias (float32) = column sums of dy
    (bfloat16); dx_d, dw_d and dbias_d may each be None.  work_d: a tensor of at least
    mxfp4_linear_backward_bytes(m, n, k) bytes, or a device address with its work_bytes."""
    lib = _lib.load()
    if stream is None:
        stream = _current_stream()
    _lib.check(lib.int4linear_mxfp4_linear_backward(_ptr(dy_d), _ptr(x_codes_d), _ptr(x_scales_d), _ptr(w_codes_d),
                                                    _ptr(w_scales_d), _ptr(dx_d), _ptr(dw_d), OUT_TYPES[dw_type],
                                                    _ptr(dbias_d), *_work(work_d, work_bytes), m, n, k, stream))


def mxfp4_gated_backward_bytes(m: int, n: int, k: int) -> int:
    """Bytes of workspace mxfp4_gated_backward needs."""
    return int(_lib.load().int4linear_mxfp4_gated_backward_bytes(m, n, k))


def mxfp4_gated_backward(dh_d, x_codes_d, x_scales_d, wg_codes_d, wg_scales_d, wu_codes_d, wu_scales_d, dx_d, dwg_d,
                         dwu_d, dw_type: str, work_d, m: int, n: int, k: int, *, activation: str = "silu",
                         work_bytes: int | None = None, stream: int | None = None) -> None:
    """Gradients of mxfp4_gated from dh (bfloat16): dx (bfloat16), dwg and dwu (dw_type "bf16" or "f32");
    dx_d, or dwg_d and dwu_d together, may be None.  work_d: a tensor of at least
    mxfp4_gated_backward_bytes(m, n, k) bytes, or a device address with its work_bytes."""
    lib = _lib.load()
    if stream is None:
        stream = _current_stream()
    _lib.check(lib.int4linear_mxfp4_gated_backward(_ptr(dh_d), _ptr(x_codes_d), _ptr(x_scales_d), _ptr(wg_codes_d),
                                                   _ptr(wg_scales_d), _ptr(wu_codes_d), _ptr(wu_scales_d),
                                                   ACTIVATIONS[activation], _ptr(dx_d), _ptr(dwg_d), _ptr(dwu_d),
                                                   OUT_TYPES[dw_type], *_work(work_d, work_bytes), m, n, k, stream))


def int8_code_bytes(rows: int, k: int) -> int:
    """Bytes of a rows x k matrix's codes in 8 bits (a row: a multiple of 128); its scales are rows float32."""
    return int(_lib.load().int4linear_int8_code_bytes(rows, k))


def int8_quantize(x_d, codes_d, scales_d, rows: int, k: int, *, in_type: str = "bf16", ld: int | None = None,
                  stream: int | None = None) -> None:
    """x_d (rows x k of in_type "f32", "f16" or "bf16", ld elements between rows, k if None) -> 8 bits with a scale a row."""
    lib = _lib.load()
    if stream is None:
        stream = _current_stream()
    _lib.check(lib.int4linear_int8_quantize(_ptr(x_d), OUT_TYPES[in_type], k if ld is None else ld, _ptr(codes_d),
                                            _ptr(scales_d), rows, k, stream))


def int8_dequantize(codes_d, scales_d, y_d, rows: int, k: int, *, out_type: str = "bf16", ld: int | None = None,
                    stream: int | None = None) -> None:
    """8 bits -> y_d (rows x k of out_type, ld elements between rows, k if None)."""
    lib = _lib.load()
    if stream is None:
        stream = _current_stream()
    _lib.check(lib.int4linear_int8_dequantize(_ptr(codes_d), _ptr(scales_d), _ptr(y_d), OUT_TYPES[out_type],
                                              k if ld is None else ld, rows, k, stream))


def int8_linear(x_codes_d, x_scales_d, w_codes_d, w_scales_d, bias_d, y_d, out_type: str, m: int, n: int, k: int, *,
                stream: int | None = None) -> None:
    """Y (m x n of out_type) = X * W^T + bias for 8-bit operands; bias_d (n float32) may be None."""
    lib = _lib.load()
    if stream is None:
        stream = _current_stream()
    _lib.check(lib.int4linear_int8_linear(_ptr(x_codes_d), _ptr(x_scales_d), _ptr(w_codes_d), _ptr(w_scales_d),
                                          _ptr(bias_d), _ptr(y_d), OUT_TYPES[out_type], m, n, k, stream))


def int8_linear_backward_bytes(m: int, n: int, k: int, dw_type: str) -> int:
    """Bytes of workspace int8_linear_backward needs."""
    return int(_lib.load().int4linear_int8_linear_backward_bytes(m, n, k, OUT_TYPES[dw_type]))


def int8_linear_backward(dy_d, x_codes_d, x_scales_d, w_codes_d, w_scales_d, dx_d, dw_d, dw_type: str, dbias_d, work_d,
                         m: int, n: int, k: int, *, work_bytes: int | None = None, stream: int | None = None) -> None:
    """dx (bfloat16) = dy W, dw (dw_type "bf16" or "f32") = dy^T X, dbias (float32) = column sums of dy
    (bfloat16); dx_d, dw_d and dbias_d may each be None.  work_d: a tensor of at least
    int8_linear_backward_bytes(m, n, k, dw_type) bytes, or a device address with its work_bytes."""
    lib = _lib.load()
    if stream is None:
        stream = _current_stream()
    _lib.check(lib.int4linear_int8_linear_backward(_ptr(dy_d), _ptr(x_codes_d), _ptr(x_scales_d), _ptr(w_codes_d),
                                                   _ptr(w_scales_d), _ptr(dx_d), _ptr(dw_d), OUT_TYPES[dw_type],
                                                   _ptr(dbias_d), *_work(work_d, work_bytes), m, n, k, stream))


def layer_norm(x_d, gamma_d, beta_d, y_d, rows: int, n: int, *, eps: float = 1e-5, in_type: str = "bf16",
               out_type: str = "bf16", ld: int | None = None, ld_y: int | None = None, stream: int | None = None) -> None:
    """y_d (rows x n of out_type) = (x - mean) / sqrt(variance + eps) * gamma + beta, row by row of x_d (rows x n of
    in_type); gamma_d and beta_d (n float32) may each be None.  ld, ld_y: elements between rows, n if None."""
    lib = _lib.load()
    if stream is None:
        stream = _current_stream()
    _lib.check(lib.int4linear_layer_norm(_ptr(x_d), OUT_TYPES[in_type], n if ld is None else ld, _ptr(gamma_d),
                                         _ptr(beta_d), eps, _ptr(y_d), OUT_TYPES[out_type], n if ld_y is None else ld_y,
                                         rows, n, stream))


def layer_norm_int8(x_d, gamma_d, beta_d, codes_d, scales_d, rows: int, n: int, *, eps: float = 1e-5,
                    in_type: str = "bf16", ld: int | None = None, stream: int | None = None) -> None:
    """layer_norm with the result in 8 bits, the form int8_linear takes."""
    lib = _lib.load()
    if stream is None:
        stream = _current_stream()
    _lib.check(lib.int4linear_layer_norm_int8(_ptr(x_d), OUT_TYPES[in_type], n if ld is None else ld, _ptr(gamma_d),
                                              _ptr(beta_d), eps, _ptr(codes_d), _ptr(scales_d), rows, n, stream))


def layer_norm_mxfp4(x_d, gamma_d, beta_d, codes_d, scales_d, rows: int, n: int, *, eps: float = 1e-5,
                     in_type: str = "bf16", ld: int | None = None, stream: int | None = None) -> None:
    """layer_norm with the result in MXFP4, the form the mxfp4 layers take."""
    lib = _lib.load()
    if stream is None:
        stream = _current_stream()
    _lib.check(lib.int4linear_layer_norm_mxfp4(_ptr(x_d), OUT_TYPES[in_type], n if ld is None else ld, _ptr(gamma_d),
                                               _ptr(beta_d), eps, _ptr(codes_d), _ptr(scales_d), rows, n, stream))


def layer_norm_backward_bytes(rows: int, n: int) -> int:
    """Bytes of workspace layer_norm_backward needs."""
    return int(_lib.load().int4linear_layer_norm_backward_bytes(rows, n))


def layer_norm_backward(dy_d, x_d, gamma_d, dx_d, dgamma_d, dbeta_d, work_d, rows: int, n: int, *, eps: float = 1e-5,
                        dy_type: str = "bf16", in_type: str = "bf16", ld_dy: int | None = None, ld: int | None = None,
                        ld_dx: int | None = None, work_bytes: int | None = None, stream: int | None = None) -> None:
    """Gradients of layer_norm from dy_d (rows x n of dy_type): dx_d (of x_d's in_type), dgamma_d and dbeta_d (n
    float32); each of the three may be None.  work_d: a tensor of at least layer_norm_backward_bytes(rows, n) bytes, or a
    device address with its work_bytes."""
    lib = _lib.load()
    if stream is None:
        stream = _current_stream()
    _lib.check(lib.int4linear_layer_norm_backward(_ptr(dy_d), OUT_TYPES[dy_type], n if ld_dy is None else ld_dy, _ptr(x_d),
                                                  OUT_TYPES[in_type], n if ld is None else ld, _ptr(gamma_d), eps,
                                                  _ptr(dx_d), n if ld_dx is None else ld_dx, _ptr(dgamma_d), _ptr(dbeta_d),
                                                  *_work(work_d, work_bytes), rows, n, stream))


def workspace_bytes(m: int, n: int, k: int) -> int:
    """Internal workspace the automatic dispatch would use for this shape."""
    return int(_lib.load().int4linear_workspace_bytes(m, n, k))


def set_workspace_limit(nbytes: int) -> None:
    _lib.load().int4linear_set_workspace_limit(nbytes)


def release_workspace() -> None:
    _lib.check(_lib.load().int4linear_release_workspace())


def kernel_for_shape(m: int, n: int, k: int) -> str:
    return _lib.load().int4linear_kernel_for_shape(m, n, k).decode()


def pack_device(src_d, dst_d, m: int, n: int, *, stream: int | None = None) -> None:
    lib = _lib.load()
    if stream is None:
        stream = _current_stream()
    _lib.check(lib.int4linear_pack_s32_to_s4(_ptr(src_d), _ptr(dst_d), m, n, stream))


def unpack_device(src_d, dst_d, m: int, n: int, *, stream: int | None = None) -> None:
    lib = _lib.load()
    if stream is None:
        stream = _current_stream()
    _lib.check(lib.int4linear_unpack_s4_to_s32(_ptr(src_d), _ptr(dst_d), m, n, stream))


def _launch(symbol: str, x_packed_d, w_packed_d, y_d, m: int, n: int, k: int) -> None:
    lib = _lib.load()
    getattr(lib, symbol)(_ptr(x_packed_d), _ptr(w_packed_d), _ptr(y_d), m, n, k)


# Blocking entry points with the reference's names: default stream, device-synchronised
# on return, no status (a failure prints one line to stderr).
def linear_v0_launch(x_packed_d, w_packed_d, y_d, m, n, k):
    _launch("_Z16linear_v0_launchPvS_S_iii", x_packed_d, w_packed_d, y_d, m, n, k)


def linear_v1_launch(x_packed_d, w_packed_d, y_d, m, n, k):
    _launch("_Z16linear_v1_launchPvS_S_iii", x_packed_d, w_packed_d, y_d, m, n, k)


def linear_v2_launch(x_packed_d, w_packed_d, y_d, m, n, k):
    _launch("_Z16linear_v2_launchPvS_S_iii", x_packed_d, w_packed_d, y_d, m, n, k)


def linear_v10_launch(x_packed_d, w_packed_d, y_d, m, n, k):
    _launch("_Z17linear_v10_launchPvS_S_iii", x_packed_d, w_packed_d, y_d, m, n, k)


def linear_v11_launch(x_packed_d, w_packed_d, y_d, m, n, k):
    _launch("_Z17linear_v11_launchPvS_S_iii", x_packed_d, w_packed_d, y_d, m, n, k)


def linear_v20_launch(x_packed_d, w_packed_d, y_d, m, n, k):
    _launch("_Z17linear_v20_launchPvS_S_iii", x_packed_d, w_packed_d, y_d, m, n, k)


def linear_v21_launch(x_packed_d, w_packed_d, y_d, m, n, k):
    _launch("_Z17linear_v21_launchPvS_S_iii", x_packed_d, w_packed_d, y_d, m, n, k)


def pack(src: np.ndarray, dst: np.ndarray, m: int, n: int) -> None:
    """Host packer: src is m*n int32 values, dst receives m*ceil(n/8) int32 words."""
    lib = _lib.load()
    assert src.dtype == np.int32 and dst.dtype == np.int32
    assert src.flags.c_contiguous and dst.flags.c_contiguous
    assert src.size >= m * n and dst.size >= m * ((n + 7) // 8)
    lib._Z4packPKiPiii(_ptr(src), _ptr(dst), m, n)


def unpack(src: np.ndarray, dst: np.ndarray, m: int, n: int) -> None:
    """Host unpacker: inverse of pack."""
    lib = _lib.load()
    assert src.dtype == np.int32 and dst.dtype == np.int32
    assert src.flags.c_contiguous and dst.flags.c_contiguous
    assert src.size >= m * ((n + 7) // 8) and dst.size >= m * n
    lib._Z6unpackPKiPiii(_ptr(src), _ptr(dst), m, n)


def pack_rows(values: np.ndarray) -> np.ndarray:
    """Convenience: pack a 2-D integer array (any int dtype, values in [-8, 7]) into the
    m x ceil(n/8) int32 word layout."""
    m, n = values.shape
    src = np.ascontiguousarray(values, dtype=np.int32)
    dst = np.empty((m, (n + 7) // 8), dtype=np.int32)
    pack(src, dst, m, n)
    return dst
