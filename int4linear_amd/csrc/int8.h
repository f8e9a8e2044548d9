// 8-bit matrices with a scale for each row, and the row passes that make them: the formats and the launchers between
// api_int8.hip and the kernel files.
//
// A matrix of rows x k is two arrays: codes, 8-bit whole numbers, row-major, every row padded with zeros to a multiple of
// 128 bytes (one line of the caches and one stage of the GEMM); and scales, a float for each row (a token of x, an output
// channel of w).  A value is code * scale.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "kernels.h"

namespace int4linear {

__host__ __device__ inline size_t int8_code_stride(int k) { return ((size_t)k + 127) / 128 * 128; }

struct Int8Matrix {
    const int8_t *codes;
    const float *scales;
    int rows;
};

// y = x w^T + bias.  bias: n floats or null; out: an OutKind other than kOutS32.
hipError_t launch_int8_linear(const Int8Matrix &x, const Int8Matrix &w, const float *bias, void *y, int out, int k, const DeviceInfo &dev,
                              hipStream_t stream);

// The same for up to 64 rows of x (k > 0): w is streamed (kernels_int8_skinny.hip).
hipError_t int8_skinny_init();
bool int8_skinny_preferred(int m, int n);
hipError_t launch_int8_skinny(const Int8Matrix &x, const Int8Matrix &w, const float *bias, void *y, int out, int k, hipStream_t stream);

// y (rows x k of `type`, ld elements between rows) = what q stands for.
hipError_t launch_int8_dequantize(const Int8Matrix &q, void *y, int type, size_t ld, int k, hipStream_t stream);

// The longest row of a norm: sums over it are those of at most as many floats.
constexpr int kMostNorm = 1 << 22;

// One pass over rows of x (rows x n of `type`, an OutKind other than kOutS32; ld elements between rows): as they are, or
// normalised, (x - mean) / sqrt(variance + eps) * gamma + beta (gamma and beta: n floats or null), into one of three forms.
enum RowResult : int { kRowTyped, kRowInt8, kRowMx };
struct RowPass {
    const void *x;
    int type;
    size_t ld;
    int rows, n;
    bool norm;
    const float *gamma, *beta;
    float eps;
    RowResult result;
    void *y;             // kRowTyped: rows x n of `out`, ld_y elements between rows; else the codes
    int out;
    size_t ld_y;
    void *scales;        // floats (kRowInt8), bytes (kRowMx)
};
hipError_t launch_rows(const RowPass &p, const DeviceInfo &dev, hipStream_t stream);

// Gradients of the norm: dx (of `type`) from dy (of dy_type), and the sums over rows dgamma of dy * (normalised x), dbeta of dy;
// each may be null.  work: layer_norm_work_bytes(), 256-byte aligned.
struct NormBackward {
    const void *dy;
    int dy_type;
    size_t ld_dy;
    const void *x;
    int type;
    size_t ld;
    const float *gamma;
    float eps;
    void *dx;
    size_t ld_dx;
    float *dgamma, *dbeta;
    int rows, n;
    void *work;
};
size_t layer_norm_work_bytes(int rows, int n);
hipError_t launch_norm_backward(const NormBackward &p, const DeviceInfo &dev, hipStream_t stream);

}  // namespace int4linear
