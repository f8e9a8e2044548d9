// C ABI of the MXFP4 operators: argument checks, the caller's workspace cut into its parts, and the
// order of launches.  Nothing here allocates, records events or looks at the library's workspace.
#include "../../include/int4linear.h"
#include "mxfp4.h"

#include <cstdint>

namespace {

using namespace int4linear;

// Row and column numbers are 32-bit in the kernels, rounded up to tiles; offsets are 64-bit.
constexpr int kMostRows = 1 << 30;
// A tile's loads are a base and 32 bits of offset over at most 256 rows of an operand.  The longest rows of a product are k / 2 bytes;
// those of a gradient's products are bfloat16, 2 bytes of any of its sizes, and 4 of n where dg and du lie side by side.
constexpr int kMostK = 1 << 22;
constexpr int kMostGradient = kMostK - 64;
static_assert(255ull * (kMostK / 2) + 128 <= 1ull << 32 && kMostGradient % 64 == 0 && 255ull * 4 * kMostGradient + 128 <= 1ull << 32);

bool aligned(const void *p, size_t bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }
bool is_type(int type) { return type == INT4LINEAR_OUT_F32 || type == INT4LINEAR_OUT_F16 || type == INT4LINEAR_OUT_BF16; }
size_t type_bytes(int type) { return type == INT4LINEAR_OUT_F32 ? 4 : 2; }
bool is_activation(int act) { return act == INT4LINEAR_ACT_SILU || act == INT4LINEAR_ACT_GELU; }

// A status for the first of some checks that fails.
struct Checks {
    int status = INT4LINEAR_OK;
    Checks &that(bool ok, int otherwise)
    {
        if (status == INT4LINEAR_OK && !ok)
            status = otherwise;
        return *this;
    }
    Checks &sizes(int a, int b, int c)
    {
        that(a >= 0 && b >= 0 && c >= 0, INT4LINEAR_ERR_SHAPE);
        return that(a <= kMostRows && b <= kMostRows && c <= kMostRows, INT4LINEAR_ERR_UNSUPPORTED);
    }
    // An array the call reads or writes; `used`: it has elements.
    Checks &array(const void *p, size_t alignment, bool used)
    {
        that(!used || p, INT4LINEAR_ERR_NULL);
        return that(!used || aligned(p, alignment), INT4LINEAR_ERR_ALIGN);
    }
    Checks &optional(const void *p, size_t alignment) { return that(!p || aligned(p, alignment), INT4LINEAR_ERR_ALIGN); }
    Checks &matrix(const void *codes, const void *scales, int rows, int k)
    {
        array(codes, 16, rows > 0 && k > 0);
        return array(scales, 16, rows > 0 && k > 0);
    }
    explicit operator bool() const { return status == INT4LINEAR_OK; }
};

MxMatrix matrix(const void *codes, const void *scales, int rows) { return {(const uint8_t *)codes, (const uint8_t *)scales, rows}; }

size_t up(size_t v, size_t to) { return (v + to - 1) / to * to; }

// The caller's workspace, handed out part by part in steps of 256 bytes; with a null base it only counts.
struct Parts {
    uint8_t *base;
    size_t used = 0;
    template <class T>
    T *take(size_t count)
    {
        T *p = base ? (T *)(base + used) : nullptr;
        used += up(count * sizeof(T), 256);
        return p;
    }
};

// Where slices of small products meet (of products that have terms at all).
SliceSpace slice_space(Parts &p, bool terms)
{
    SliceSpace s;
    s.partial = p.take<float>(terms ? (size_t)kMostSlices * 64 * 64 : 0);
    s.arrivals = p.take<unsigned>(terms ? kMostSlices * 4 : 0);
    return s;
}

struct LinearBackwardParts {
    uint16_t *dy_t, *dy_padded, *x_t, *w_t;
    float *sums;
    SliceSpace slices;
    size_t ld_m, ld_n, bytes;
};

LinearBackwardParts linear_backward_parts(void *work, int m, int n, int k)
{
    Parts p{(uint8_t *)work};
    LinearBackwardParts r{};
    r.ld_m = up((size_t)m, 64);
    r.ld_n = up((size_t)n, 64);
    r.dy_t = p.take<uint16_t>((size_t)n * r.ld_m);
    r.dy_padded = p.take<uint16_t>(n % 64 ? (size_t)m * r.ld_n : 0);
    r.x_t = p.take<uint16_t>((size_t)k * r.ld_m);
    r.w_t = p.take<uint16_t>((size_t)k * r.ld_n);
    r.sums = p.take<float>((size_t)n * (r.ld_m / 64));
    r.slices = slice_space(p, m > 0 && n > 0 && k > 0);
    r.bytes = p.used;
    return r;
}

struct GatedBackwardParts {
    uint16_t *d, *d_t, *x_t, *w_t;
    SliceSpace slices;
    size_t ld_m, ld_n, bytes;
};

GatedBackwardParts gated_backward_parts(void *work, int m, int n, int k)
{
    Parts p{(uint8_t *)work};
    GatedBackwardParts r{};
    r.ld_m = up((size_t)m, 64);
    r.ld_n = up((size_t)n, 64);
    r.d = p.take<uint16_t>((size_t)m * 2 * r.ld_n);
    r.d_t = p.take<uint16_t>(2 * (size_t)n * r.ld_m);
    r.x_t = p.take<uint16_t>((size_t)k * r.ld_m);
    r.w_t = p.take<uint16_t>((size_t)k * 2 * r.ld_n);
    r.slices = slice_space(p, m > 0 && n > 0 && k > 0);
    r.bytes = p.used;
    return r;
}

}  // namespace

extern "C" {

size_t int4linear_mxfp4_code_bytes(int rows, int k) { return rows < 0 || k < 0 ? 0 : (size_t)rows * mx_code_stride(k); }

size_t int4linear_mxfp4_scale_bytes(int rows, int k) { return rows < 0 || k < 0 ? 0 : (size_t)rows * mx_scale_stride(k); }

int int4linear_mxfp4_quantize(const void *x_d, int type, size_t ld, void *codes_d, void *scales_d, int rows, int k, void *stream)
{
    Checks ok;
    ok.sizes(rows, 0, k).that(ld >= (size_t)(k > 0 ? k : 0), INT4LINEAR_ERR_SHAPE).that(is_type(type), INT4LINEAR_ERR_UNSUPPORTED);
    ok.array(x_d, type_bytes(type), rows > 0 && k > 0).matrix(codes_d, scales_d, rows, k);
    if (!ok || rows == 0 || k == 0)
        return ok.status;
    DeviceInfo info;
    const int st = api_begin((hipStream_t)stream, &info);
    if (st != INT4LINEAR_OK)
        return st;
    return api_status(launch_mx_quantize(x_d, type, ld, (uint8_t *)codes_d, (uint8_t *)scales_d, rows, k, (hipStream_t)stream));
}

int int4linear_mxfp4_dequantize(const void *codes_d, const void *scales_d, void *y_d, int type, size_t ld, int rows, int k,
                                void *stream)
{
    Checks ok;
    ok.sizes(rows, 0, k).that(ld >= (size_t)(k > 0 ? k : 0), INT4LINEAR_ERR_SHAPE).that(is_type(type), INT4LINEAR_ERR_UNSUPPORTED);
    ok.array(y_d, type_bytes(type), rows > 0 && k > 0).matrix(codes_d, scales_d, rows, k);
    if (!ok || rows == 0 || k == 0)
        return ok.status;
    DeviceInfo info;
    const int st = api_begin((hipStream_t)stream, &info);
    if (st != INT4LINEAR_OK)
        return st;
    return api_status(launch_mx_dequantize(matrix(codes_d, scales_d, rows), y_d, type, ld, k, (hipStream_t)stream));
}

int int4linear_mxfp4_linear(const void *x_codes_d, const void *x_scales_d, const void *w_codes_d, const void *w_scales_d,
                            const float *bias_d, void *y_d, int out_type, int m, int n, int k, void *stream)
{
    Checks ok;
    ok.sizes(m, n, k).that(k <= kMostK && is_type(out_type), INT4LINEAR_ERR_UNSUPPORTED);
    if (!ok || m == 0 || n == 0)
        return ok.status;
    ok.array(y_d, 16, true).optional(bias_d, 4).matrix(x_codes_d, x_scales_d, m, k).matrix(w_codes_d, w_scales_d, n, k);
    if (!ok)
        return ok.status;
    DeviceInfo info;
    const int st = api_begin((hipStream_t)stream, &info);
    if (st != INT4LINEAR_OK)
        return st;
    return api_status(launch_mx_linear(matrix(x_codes_d, x_scales_d, m), matrix(w_codes_d, w_scales_d, n), bias_d, y_d, out_type, k,
                                       info, (hipStream_t)stream));
}

int int4linear_mxfp4_gated(const void *x_codes_d, const void *x_scales_d, const void *wg_codes_d, const void *wg_scales_d,
                           const void *wu_codes_d, const void *wu_scales_d, int activation, void *h_d, int out_type, int m, int n,
                           int k, void *stream)
{
    Checks ok;
    ok.sizes(m, n, k).that(k <= kMostK && is_type(out_type) && is_activation(activation), INT4LINEAR_ERR_UNSUPPORTED);
    if (!ok || m == 0 || n == 0)
        return ok.status;
    ok.array(h_d, 16, true).matrix(x_codes_d, x_scales_d, m, k);
    ok.matrix(wg_codes_d, wg_scales_d, n, k).matrix(wu_codes_d, wu_scales_d, n, k);
    if (!ok)
        return ok.status;
    DeviceInfo info;
    const int st = api_begin((hipStream_t)stream, &info);
    if (st != INT4LINEAR_OK)
        return st;
    return api_status(launch_mx_gated(matrix(x_codes_d, x_scales_d, m), matrix(wg_codes_d, wg_scales_d, n),
                                      matrix(wu_codes_d, wu_scales_d, n), (Activation)activation, h_d, out_type, k, info,
                                      (hipStream_t)stream));
}

int int4linear_mxfp4_gated_quantized(const void *x_codes_d, const void *x_scales_d, const void *wg_codes_d, const void *wg_scales_d,
                                     const void *wu_codes_d, const void *wu_scales_d, int activation, void *h_codes_d,
                                     void *h_scales_d, int m, int n, int k, void *stream)
{
    Checks ok;
    ok.sizes(m, n, k).that(k <= kMostK && is_activation(activation), INT4LINEAR_ERR_UNSUPPORTED);
    if (!ok || m == 0 || n == 0)
        return ok.status;
    ok.matrix(h_codes_d, h_scales_d, m, n).matrix(x_codes_d, x_scales_d, m, k);
    ok.matrix(wg_codes_d, wg_scales_d, n, k).matrix(wu_codes_d, wu_scales_d, n, k);
    if (!ok)
        return ok.status;
    DeviceInfo info;
    const int st = api_begin((hipStream_t)stream, &info);
    if (st != INT4LINEAR_OK)
        return st;
    return api_status(launch_mx_gated_quantized(matrix(x_codes_d, x_scales_d, m), matrix(wg_codes_d, wg_scales_d, n),
                                                matrix(wu_codes_d, wu_scales_d, n), (Activation)activation, (uint8_t *)h_codes_d,
                                                (uint8_t *)h_scales_d, k, info, (hipStream_t)stream));
}

size_t int4linear_mxfp4_linear_backward_bytes(int m, int n, int k)
{
    return m < 0 || n < 0 || k < 0 ? 0 : linear_backward_parts(nullptr, m, n, k).bytes;
}

int int4linear_mxfp4_linear_backward(const void *dy_d, const void *x_codes_d, const void *x_scales_d, const void *w_codes_d,
                                     const void *w_scales_d, void *dx_d, void *dw_d, int dw_type, float *dbias_d, void *work_d,
                                     size_t work_bytes, int m, int n, int k, void *stream_v)
{
    Checks ok;
    ok.sizes(m, n, k).that(m <= kMostGradient && n <= kMostGradient && k <= kMostGradient, INT4LINEAR_ERR_UNSUPPORTED);
    ok.that(!dw_d || dw_type == INT4LINEAR_OUT_F32 || dw_type == INT4LINEAR_OUT_BF16, INT4LINEAR_ERR_UNSUPPORTED);
    const bool want_dx = dx_d && m > 0 && k > 0, want_dw = dw_d && n > 0 && k > 0, want_sums = dbias_d && n > 0;
    if (!ok || (!want_dx && !want_dw && !want_sums))
        return ok.status;
    ok.optional(dx_d, 16).optional(dw_d, 16).optional(dbias_d, 4).array(dy_d, 16, m > 0 && n > 0);
    if (want_dw)
        ok.matrix(x_codes_d, x_scales_d, m, k);
    if (want_dx)
        ok.matrix(w_codes_d, w_scales_d, n, k);
    const LinearBackwardParts p = linear_backward_parts(work_d, m, n, k);
    ok.array(work_d, 256, p.bytes > 0).that(work_bytes >= p.bytes, INT4LINEAR_ERR_SCRATCH);
    if (!ok)
        return ok.status;
    hipStream_t stream = (hipStream_t)stream_v;
    DeviceInfo info;
    const int st = api_begin(stream, &info);
    if (st != INT4LINEAR_OK)
        return st;
    const bool ragged = n % 64 != 0;
    Prepared prepared{};
    prepared.k = k;
    prepared.zeros = p.slices.arrivals;
    prepared.zero_count = m > 0 && n > 0 && k > 0 ? kMostSlices * 4 : 0;
    if (want_dw && m > 0)
        prepared.matrix[prepared.matrices++] = {matrix(x_codes_d, x_scales_d, m), p.x_t, p.ld_m};
    if (want_dx && n > 0)
        prepared.matrix[prepared.matrices++] = {matrix(w_codes_d, w_scales_d, n), p.w_t, p.ld_n};
    if (m > 0 && n > 0 && (want_dw || want_sums || ragged)) {
        prepared.dy = (const uint16_t *)dy_d;
        prepared.rows = m;
        prepared.cols = n;
        prepared.transposed = want_dw ? p.dy_t : nullptr;
        prepared.ld_t = p.ld_m;
        prepared.padded = want_dx && ragged ? p.dy_padded : nullptr;
        prepared.ld_p = p.ld_n;
        prepared.partial = want_sums ? p.sums : nullptr;
    }
    hipError_t e = launch_prepare(prepared, stream);
    const Bf16Product products[] = {{p.dy_t, n, p.x_t, k, p.ld_m, m, want_dw ? dw_d : nullptr, dw_type},
                                    {ragged ? p.dy_padded : (const uint16_t *)dy_d, m, p.w_t, k, p.ld_n, n, want_dx ? dx_d : nullptr, kOutBF16}};
    const ColumnSums sums{want_sums ? dbias_d : nullptr, p.sums, (int)(p.ld_m / 64), n};
    if (e == hipSuccess)
        e = launch_bf16_products(products, 2, sums, p.slices, info, stream);
    return api_status(e);
}

size_t int4linear_mxfp4_gated_backward_bytes(int m, int n, int k)
{
    return m < 0 || n < 0 || k < 0 ? 0 : gated_backward_parts(nullptr, m, n, k).bytes;
}

int int4linear_mxfp4_gated_backward(const void *dh_d, const void *x_codes_d, const void *x_scales_d, const void *wg_codes_d,
                                    const void *wg_scales_d, const void *wu_codes_d, const void *wu_scales_d, int activation,
                                    void *dx_d, void *dwg_d, void *dwu_d, int dw_type, void *work_d, size_t work_bytes, int m, int n,
                                    int k, void *stream_v)
{
    Checks ok;
    ok.sizes(m, n, k).that(m <= kMostGradient && n <= kMostGradient && k <= kMostGradient, INT4LINEAR_ERR_UNSUPPORTED);
    ok.that(is_activation(activation), INT4LINEAR_ERR_UNSUPPORTED);
    ok.that(!dwg_d || dw_type == INT4LINEAR_OUT_F32 || dw_type == INT4LINEAR_OUT_BF16, INT4LINEAR_ERR_UNSUPPORTED);
    ok.that(!dwg_d == !dwu_d, INT4LINEAR_ERR_NULL);
    const bool want_dx = dx_d && m > 0 && k > 0, want_dw = dwg_d && n > 0 && k > 0;
    if (!ok || (!want_dx && !want_dw))
        return ok.status;
    ok.optional(dx_d, 16).optional(dwg_d, 16).optional(dwu_d, 16).array(dh_d, 16, m > 0 && n > 0);
    ok.matrix(x_codes_d, x_scales_d, m, k).matrix(wg_codes_d, wg_scales_d, n, k).matrix(wu_codes_d, wu_scales_d, n, k);
    const GatedBackwardParts p = gated_backward_parts(work_d, m, n, k);
    ok.array(work_d, 256, p.bytes > 0).that(work_bytes >= p.bytes, INT4LINEAR_ERR_SCRATCH);
    if (!ok)
        return ok.status;
    hipStream_t stream = (hipStream_t)stream_v;
    DeviceInfo info;
    const int st = api_begin(stream, &info);
    if (st != INT4LINEAR_OK)
        return st;
    const MxMatrix x = matrix(x_codes_d, x_scales_d, m);
    const MxMatrix wg = matrix(wg_codes_d, wg_scales_d, n), wu = matrix(wu_codes_d, wu_scales_d, n);
    hipError_t e = hipSuccess;
    if (m > 0 && n > 0)
        e = launch_mx_gated_gradients(x, wg, wu, (Activation)activation, (const uint16_t *)dh_d, p.d, p.ld_n, p.d_t, p.ld_m, k, info,
                                      stream);
    // wg and wu side by side: row c of w_t is column c of wg, then column c of wu
    Prepared prepared{};
    prepared.k = k;
    prepared.zeros = p.slices.arrivals;
    prepared.zero_count = m > 0 && n > 0 && k > 0 ? kMostSlices * 4 : 0;
    if (want_dw && m > 0)
        prepared.matrix[prepared.matrices++] = {x, p.x_t, p.ld_m};
    if (want_dx && n > 0) {
        prepared.matrix[prepared.matrices++] = {wg, p.w_t, 2 * p.ld_n};
        prepared.matrix[prepared.matrices++] = {wu, p.w_t + p.ld_n, 2 * p.ld_n};
    }
    if (e == hipSuccess)
        e = launch_prepare(prepared, stream);
    const Bf16Product products[] = {
        {p.d_t, n, p.x_t, k, p.ld_m, m, want_dw ? dwg_d : nullptr, dw_type},
        {p.d_t + (size_t)n * p.ld_m, n, p.x_t, k, p.ld_m, m, want_dw ? dwu_d : nullptr, dw_type},
        {p.d, m, p.w_t, k, 2 * p.ld_n, (int)(n > 0 ? 2 * p.ld_n : 0), want_dx ? dx_d : nullptr, kOutBF16}};
    if (e == hipSuccess)
        e = launch_bf16_products(products, 3, ColumnSums{}, p.slices, info, stream);
    return api_status(e);
}

}  // extern "C"
