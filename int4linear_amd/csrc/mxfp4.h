// MXFP4 matrices: the format, and the launchers between api_mxfp4.hip and the kernel files.
//
// A row is cut into blocks of 32 values along k.  A block has one scale, 2^(s - 127) with s in 8
// bits (E8M0; s = 255: the block is NaN), and 32 values of 4 bits (E2M1: sign, two exponent bits, one
// mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6), two per byte, even k in the low nibble as in the packed
// s4 layout.  Codes and scales are two arrays, row-major, both padded at the end of each row with
// zeros: codes to 128 bytes (256 k, one line of the caches and one stage of the GEMM), scales to 16
// (512 k, one load of a lane for two stages).
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "kernels.h"

namespace int4linear {

constexpr int kMxBlock = 32;      // values that share a scale
constexpr int kLineBytes = 128;   // codes of 256 k
constexpr int kLineFp4 = 256;     // k in a line of 4-bit values
constexpr int kLineInt8 = 128;    // k in a line of 8-bit values
constexpr int kLineBf16 = 64;     // k in a line of bfloat16

inline size_t mx_code_stride(int k) { return ((size_t)k + 255) / 256 * 128; }
inline size_t mx_scale_stride(int k) { return ((size_t)k + 511) / 512 * 16; }

// A matrix in MXFP4 whose rows are `rows` x k values.
struct MxMatrix {
    const uint8_t *codes;
    const uint8_t *scales;
    int rows;
};

// act(g) * u; the gelu is its tanh form.
enum Activation : int { kSilu = 0, kGelu = 1 };

// x (rows x k of `type`, an OutKind other than kOutS32; ld elements between rows) -> codes, scales.
hipError_t launch_mx_quantize(const void *x, int type, size_t ld, uint8_t *codes, uint8_t *scales, int rows, int k,
                              hipStream_t stream);
// The way back: y = what codes and scales stand for.
hipError_t launch_mx_dequantize(const MxMatrix &q, void *y, int type, size_t ld, int k, hipStream_t stream);
// What a backward pass's products want of its operands, in one launch: words cleared; up to three matrices q dequantised and transposed,
// dst[c * ld + r] = q[r][c] in bfloat16 for c < k, r going on to the next multiple of 64 with zeros; and of dy (rows x cols
// bfloat16, contiguous), where they are not null, the transpose (cols x ld_t, zeros behind the rows), a copy whose rows
// are padded with zeros (rows x ld_p), and every column's sum over 64 rows at a time (partial: ceil(rows / 64) x cols).
// With `int8` the matrices are codes of 8 bits with a scale for each row (rows padded to 128 bytes), whose products are rounded to
// bfloat16; where `apart` is not 0 what the rounding took away, rounded too, goes that many elements further on, and what is left of
// that as far again.
struct BackwardOperand {
    MxMatrix q;
    const float *row_scales = nullptr;
};
struct Transposed {
    BackwardOperand of;
    uint16_t *dst;
    size_t ld, apart;
};
struct Prepared {
    Transposed matrix[3];
    int matrices, k;
    bool int8;
    const uint16_t *dy;
    int rows, cols;
    uint16_t *transposed, *padded;
    int copies;  // of the transpose, side by side: ld_t / copies elements between them
    size_t ld_t, ld_p;
    float *partial;
    unsigned *zeros;  // words to be cleared
    int zero_count;
};
hipError_t launch_prepare(const Prepared &p, hipStream_t stream);

// sums[c] = the sum of `parts` rows of partial sums of `columns` columns, added in order (sums null: nothing to do).
struct ColumnSums {
    float *sums;
    const float *partial;
    int parts, columns;
};
hipError_t launch_column_sums(const ColumnSums &s, hipStream_t stream);

hipError_t line_gemm_init(const DeviceInfo &dev);

// y = x w^T + bias.  bias: n floats or null; out: an OutKind other than kOutS32.
hipError_t launch_mx_linear(const MxMatrix &x, const MxMatrix &w, const float *bias, void *y, int out, int k, const DeviceInfo &dev,
                            hipStream_t stream);
// h = act(x wg^T) * (x wu^T), as an array of `out` ...
hipError_t launch_mx_gated(const MxMatrix &x, const MxMatrix &wg, const MxMatrix &wu, Activation act, void *h, int out, int k,
                           const DeviceInfo &dev, hipStream_t stream);
// ... or in MXFP4.
hipError_t launch_mx_gated_quantized(const MxMatrix &x, const MxMatrix &wg, const MxMatrix &wu, Activation act, uint8_t *codes,
                                     uint8_t *scales, int k, const DeviceInfo &dev, hipStream_t stream);
// The same for few rows of x (k > 0; any number is taken): w is streamed (kernels_mxfp4_skinny.hip).
hipError_t launch_mx_linear_skinny(const MxMatrix &x, const MxMatrix &w, const float *bias, void *y, int out, int k, hipStream_t stream);
hipError_t launch_mx_gated_skinny(const MxMatrix &x, const MxMatrix &wg, const MxMatrix &wu, Activation act, void *h, int out, int k,
                                  hipStream_t stream);
hipError_t launch_mx_gated_quantized_skinny(const MxMatrix &x, const MxMatrix &wg, const MxMatrix &wu, Activation act, uint8_t *codes,
                                            uint8_t *scales, int k, hipStream_t stream);
// Gradients of the two projections (k > 0) from dh (m x n bfloat16): d is m x 2 * ld_n, dg in columns 0 .. ld_n - 1 and du
// behind them, dt is 2 * n x ld_m, the transposes of both; bfloat16, padding written as zeros.
hipError_t launch_mx_gated_gradients(const MxMatrix &x, const MxMatrix &wg, const MxMatrix &wu, Activation act, const uint16_t *dh,
                                     uint16_t *d, size_t ld_n, uint16_t *dt, size_t ld_m, int k, const DeviceInfo &dev,
                                     hipStream_t stream);
// y = a b^T for bfloat16 operands of m and n rows of k values, padded with zeros to a multiple of 64; `ld` elements
// between rows of either, a multiple of 64.  out: kOutF32 or kOutBF16.
struct Bf16Product {
    const uint16_t *a;
    int m;
    const uint16_t *b;
    int n;
    size_t ld;
    int k;
    void *y;
    int out;
    int terms;  // by which slices are chosen: k, but not three times as many where k holds a float's pieces, since the slices of the
                // other products would depend on the type of this one, and with them their last bits
};
// Up to three of them, and the column sums.  Small ones are cut into slices of k, whose sums meet in `space`; with
// `slices_alone` also one with a long sum that leaves the device idle beside the others, in one launch or
// by itself.  One whose y is null is not wanted; results do not depend on which are.
constexpr int kMostSlices = 1024;  // tiles of 64 x 64, times the slices of each
struct SliceSpace {
    float *partial;      // kMostSlices * 64 * 64
    unsigned *arrivals;  // kMostSlices * 4, zeros
};
hipError_t launch_bf16_products(const Bf16Product *p, int count, bool slices_alone, const ColumnSums &sums, const SliceSpace &space,
                                const DeviceInfo &dev, hipStream_t stream);

// Between the files of the C ABI (api.hip): the current device's record, set up for work on `stream`, and a
// HIP error as the status of a call.  Both return an INT4LINEAR_* status.
int api_begin(hipStream_t stream, DeviceInfo *info);
int api_status(hipError_t e);

}  // namespace int4linear
