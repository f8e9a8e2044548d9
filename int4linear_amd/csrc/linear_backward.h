// Gradients of a linear layer whose operands are in MXFP4 or in 8 bits: the call behind both layers' entry points.
#pragma once
#include "api_checks.h"
#include "mxfp4.h"

namespace int4linear {

// The products of a backward pass are those of bfloat16 operands: rows of 2 bytes of any of its sizes, and of 4 of n where dg and
// du lie side by side, of 6 of m where x lies in pieces.  A tile's loads are a base and 32 bits of offset over at most 256 rows of
// an operand.
constexpr int kMostGradient = (1 << 22) - 64, kMostInPieces = 1 << 21;
static_assert(kMostGradient % 64 == 0 && 255ull * 4 * kMostGradient + 128 <= 1ull << 32 && 255ull * 6 * kMostInPieces + 128 <= 1ull << 32);

// A value of 8 bits and a float scale as a sum of bfloat16, 8 bits each: its rounding to float to the last bit.
constexpr int kPieces = 3;

SliceSpace slice_space(Parts &p, bool terms);

// dx (m x k, bfloat16) = dy w, dw (n x k, dw_type) = dy^T x, dbias = column sums of dy; each may be null.  `int8`: x and w
// have codes of 8 bits and row_scales; else they are in MXFP4.  pieces: kPieces with 8 bits and dw as float, else 1.
size_t linear_backward_bytes(int m, int n, int k, int pieces);
int linear_backward(const void *dy, const BackwardOperand &x, const BackwardOperand &w, bool int8, void *dx, void *dw, int dw_type,
                    float *dbias, void *work, size_t work_bytes, int m, int n, int k, hipStream_t stream);

}  // namespace int4linear
