// Gradients of a linear layer whose operands are in MXFP4 or in 8 bits: checks, the caller's workspace, the order of launches.
#include "linear_backward.h"

namespace int4linear {

// Where slices of small products meet (of products that have terms at all).
SliceSpace slice_space(Parts &p, bool terms)
{
    SliceSpace s;
    s.partial = p.take<float>(terms ? (size_t)kMostSlices * 64 * 64 : 0);
    s.arrivals = p.take<unsigned>(terms ? kMostSlices * 4 : 0);
    return s;
}

namespace {

struct LinearBackwardParts {
    uint16_t *dy_t, *dy_padded, *x_t, *w_t;
    float *sums;
    SliceSpace slices;
    size_t ld_m, ld_n, bytes;
};

LinearBackwardParts linear_backward_parts(void *work, int m, int n, int k, int pieces)
{
    Parts p{(uint8_t *)work};
    LinearBackwardParts r{};
    r.ld_m = up((size_t)m, 64);
    r.ld_n = up((size_t)n, 64);
    r.dy_t = p.take<uint16_t>((size_t)n * r.ld_m * pieces);
    r.dy_padded = p.take<uint16_t>(n % 64 ? (size_t)m * r.ld_n : 0);
    r.x_t = p.take<uint16_t>((size_t)k * r.ld_m * pieces);
    r.w_t = p.take<uint16_t>((size_t)k * r.ld_n);
    r.sums = p.take<float>((size_t)n * (r.ld_m / 64));
    r.slices = slice_space(p, m > 0 && n > 0 && k > 0);
    r.bytes = p.used;
    return r;
}

}  // namespace

size_t linear_backward_bytes(int m, int n, int k, int pieces)
{
    return m < 0 || n < 0 || k < 0 ? 0 : linear_backward_parts(nullptr, m, n, k, pieces).bytes;
}

int linear_backward(const void *dy, const BackwardOperand &x, const BackwardOperand &w, bool int8, void *dx, void *dw, int dw_type,
                    float *dbias, void *work, size_t work_bytes, int m, int n, int k, hipStream_t stream)
{
    Checks ok;
    ok.sizes(m, n, k).that(m <= kMostGradient && n <= kMostGradient && k <= kMostGradient, INT4LINEAR_ERR_UNSUPPORTED);
    ok.that(!dw || dw_type == INT4LINEAR_OUT_F32 || dw_type == INT4LINEAR_OUT_BF16, INT4LINEAR_ERR_UNSUPPORTED);
    const bool want_dx = dx && m > 0 && k > 0, want_dw = dw && n > 0 && k > 0, want_sums = dbias && n > 0;
    if (!ok || (!want_dx && !want_dw && !want_sums))
        return ok.status;
    ok.optional(dx, 16).optional(dw, 16).optional(dbias, 4).array(dy, 16, m > 0 && n > 0);
    auto check = [&](const BackwardOperand &q) {
        const bool used = q.q.rows > 0 && k > 0;
        if (int8)
            ok.array(q.q.codes, 16, used).array(q.row_scales, 4, used);
        else
            ok.matrix(q.q.codes, q.q.scales, q.q.rows, k);
    };
    if (want_dw)
        check(x);
    if (want_dx)
        check(w);
    const int pieces = int8 && dw && dw_type == INT4LINEAR_OUT_F32 ? kPieces : 1;
    ok.that(pieces == 1 || m <= kMostInPieces, INT4LINEAR_ERR_UNSUPPORTED);
    if (!ok)
        return ok.status;
    const LinearBackwardParts p = linear_backward_parts(work, m, n, k, pieces);
    ok.array(work, 256, p.bytes > 0).that(work_bytes >= p.bytes, INT4LINEAR_ERR_SCRATCH);
    if (!ok)
        return ok.status;
    DeviceInfo info;
    const int st = api_begin(stream, &info);
    if (st != INT4LINEAR_OK)
        return st;
    const bool ragged = n % 64 != 0;
    const size_t ld_sum = p.ld_m * pieces;  // of what dw sums over
    Prepared prepared{};
    prepared.k = k;
    prepared.int8 = int8;
    prepared.zeros = p.slices.arrivals;
    prepared.zero_count = m > 0 && n > 0 && k > 0 ? kMostSlices * 4 : 0;
    if (want_dw && m > 0)
        prepared.matrix[prepared.matrices++] = {x, p.x_t, ld_sum, pieces > 1 ? p.ld_m : 0};
    if (want_dx && n > 0)
        prepared.matrix[prepared.matrices++] = {w, p.w_t, p.ld_n, 0};
    if (m > 0 && n > 0 && (want_dw || want_sums || ragged)) {
        prepared.dy = (const uint16_t *)dy;
        prepared.rows = m;
        prepared.cols = n;
        prepared.transposed = want_dw ? p.dy_t : nullptr;
        prepared.copies = pieces;
        prepared.ld_t = ld_sum;
        prepared.padded = want_dx && ragged ? p.dy_padded : nullptr;
        prepared.ld_p = p.ld_n;
        prepared.partial = want_sums ? p.sums : nullptr;
    }
    hipError_t e = launch_prepare(prepared, stream);
    const Bf16Product products[] = {
        {p.dy_t, n, p.x_t, k, ld_sum, pieces > 1 && m > 0 ? (int)ld_sum : m, want_dw ? dw : nullptr, dw_type, m},
        {ragged ? p.dy_padded : (const uint16_t *)dy, m, p.w_t, k, p.ld_n, n, want_dx ? dx : nullptr, kOutBF16, n}};
    const ColumnSums sums{want_sums ? dbias : nullptr, p.sums, (int)(p.ld_m / 64), n};
    if (e == hipSuccess)
        e = launch_bf16_products(products, 2, int8, sums, p.slices, info, stream);
    return api_status(e);
}

}  // namespace int4linear
