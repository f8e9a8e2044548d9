// Gradients of a linear layer whose operands are in MXFP4 or in 8 bits: the call behind both layers' entry points.
#pragma once
#include "api_checks.h"
#include "mxfp4.h"

namespace int4linear {

// The products of a backward pass are those of bfloat16 operands: rows of 2 bytes of any of its sizes, and of 4 of n where dg and
// du lie side by side, of 4 of m where x is the sum of two bfloat16.  A tile's loads are a base and 32 bits of offset over at most
// 256 rows of an operand.
constexpr int kMostGradient = (1 << 22) - 64;
static_assert(kMostGradient % 64 == 0 && 255ull * 4 * kMostGradient + 128 <= 1ull << 32);

SliceSpace slice_space(Parts &p, bool terms);

// dx (m x k, bfloat16) = dy w, dw (n x k, dw_type) = dy^T x, dbias = column sums of dy; each may be null.  `int8`: x and w
// have codes of 8 bits and row_scales; else they are in MXFP4.  `split`: x is taken as the sum of two bfloat16 (8 bits, dw as float).
size_t linear_backward_bytes(int m, int n, int k, bool split);
int linear_backward(const void *dy, const BackwardOperand &x, const BackwardOperand &w, bool int8, void *dx, void *dw, int dw_type,
                    float *dbias, void *work, size_t work_bytes, int m, int n, int k, hipStream_t stream);

}  // namespace int4linear
