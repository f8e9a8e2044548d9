// C ABI of the 8-bit linear layers and of the layer norms: argument checks.  Nothing here allocates, records events or looks at
// the library's workspace.
#include "api_checks.h"
#include "int8.h"
#include "linear_backward.h"
#include "mxfp4.h"

#include <cmath>

namespace {

using namespace int4linear;

// Sums of products of 8-bit numbers: k * 128 * 128 is below 2^31.
constexpr int kMostSummands = (1 << 17) - 1;

Int8Matrix matrix(const void *codes, const float *scales, int rows) { return {(const int8_t *)codes, scales, rows}; }

void check(Checks &ok, const void *codes, const float *scales, int rows, int k)
{
    ok.array(codes, 16, rows > 0 && k > 0).array(scales, 4, rows > 0 && k > 0);
}

// What the norms' forward calls have in common; `result` says what else.
int layer_norm(RowPass p, void *stream)
{
    const bool used = p.rows > 0 && p.n > 0;
    Checks ok;
    ok.sizes(p.rows, p.n, 0).apart(p.ld, p.n);
    if (p.result == kRowTyped)
        ok.apart(p.ld_y, p.n);
    ok.that(p.n <= kMostNorm && is_type(p.type) && p.eps >= 0.0f && std::isfinite(p.eps), INT4LINEAR_ERR_UNSUPPORTED);
    if (p.result == kRowTyped)
        ok.that(is_type(p.out), INT4LINEAR_ERR_UNSUPPORTED);
    if (!ok)
        return ok.status;
    ok.array(p.x, type_bytes(p.type), used).optional(p.gamma, 4).optional(p.beta, 4);
    ok.array(p.y, p.result == kRowTyped ? type_bytes(p.out) : 16, used);
    if (p.result != kRowTyped)
        ok.array(p.scales, p.result == kRowInt8 ? 4 : 16, used);
    if (!ok || !used)
        return ok.status;
    p.norm = true;
    DeviceInfo info;
    const int st = api_begin((hipStream_t)stream, &info);
    return st != INT4LINEAR_OK ? st : api_status(launch_rows(p, info, (hipStream_t)stream));
}

}  // namespace

extern "C" {

size_t int4linear_int8_code_bytes(int rows, int k) { return rows < 0 || k < 0 ? 0 : (size_t)rows * int8_code_stride(k); }

int int4linear_int8_quantize(const void *x_d, int type, size_t ld, void *codes_d, float *scales_d, int rows, int k, void *stream)
{
    Checks ok;
    ok.sizes(rows, 0, k).apart(ld, k).that(is_type(type), INT4LINEAR_ERR_UNSUPPORTED);
    if (!ok || rows == 0 || k == 0)
        return ok.status;
    ok.array(x_d, type_bytes(type), true);
    check(ok, codes_d, scales_d, rows, k);
    if (!ok)
        return ok.status;
    DeviceInfo info;
    const int st = api_begin((hipStream_t)stream, &info);
    if (st != INT4LINEAR_OK)
        return st;
    RowPass p{};
    p.x = x_d;
    p.type = type;
    p.ld = ld;
    p.rows = rows;
    p.n = k;
    p.result = kRowInt8;
    p.y = codes_d;
    p.scales = scales_d;
    return api_status(launch_rows(p, info, (hipStream_t)stream));
}

int int4linear_int8_dequantize(const void *codes_d, const float *scales_d, void *y_d, int type, size_t ld, int rows, int k, void *stream)
{
    Checks ok;
    ok.sizes(rows, 0, k).apart(ld, k).that(is_type(type), INT4LINEAR_ERR_UNSUPPORTED);
    if (!ok || rows == 0 || k == 0)
        return ok.status;
    ok.array(y_d, type_bytes(type), true);
    check(ok, codes_d, scales_d, rows, k);
    if (!ok)
        return ok.status;
    DeviceInfo info;
    const int st = api_begin((hipStream_t)stream, &info);
    if (st != INT4LINEAR_OK)
        return st;
    return api_status(launch_int8_dequantize(matrix(codes_d, scales_d, rows), y_d, type, ld, k, (hipStream_t)stream));
}

int int4linear_int8_linear(const void *x_codes_d, const float *x_scales_d, const void *w_codes_d, const float *w_scales_d,
                           const float *bias_d, void *y_d, int out_type, int m, int n, int k, void *stream)
{
    Checks ok;
    ok.sizes(m, n, k).that(k <= kMostSummands && is_type(out_type), INT4LINEAR_ERR_UNSUPPORTED);
    if (!ok || m == 0 || n == 0)
        return ok.status;
    ok.array(y_d, 16, true).optional(bias_d, 4);
    check(ok, x_codes_d, x_scales_d, m, k);
    check(ok, w_codes_d, w_scales_d, n, k);
    if (!ok)
        return ok.status;
    DeviceInfo info;
    const int st = api_begin((hipStream_t)stream, &info);
    if (st != INT4LINEAR_OK)
        return st;
    return api_status(launch_int8_linear(matrix(x_codes_d, x_scales_d, m), matrix(w_codes_d, w_scales_d, n), bias_d, y_d, out_type, k, info,
                                         (hipStream_t)stream));
}

size_t int4linear_int8_linear_backward_bytes(int m, int n, int k, int dw_type)
{
    return linear_backward_bytes(m, n, k, dw_type == INT4LINEAR_OUT_F32 ? kPieces : 1);
}

int int4linear_int8_linear_backward(const void *dy_d, const void *x_codes_d, const float *x_scales_d, const void *w_codes_d,
                                    const float *w_scales_d, void *dx_d, void *dw_d, int dw_type, float *dbias_d, void *work_d,
                                    size_t work_bytes, int m, int n, int k, void *stream)
{
    const BackwardOperand x{{(const uint8_t *)x_codes_d, nullptr, m}, x_scales_d}, w{{(const uint8_t *)w_codes_d, nullptr, n}, w_scales_d};
    return linear_backward(dy_d, x, w, true, dx_d, dw_d, dw_type, dbias_d, work_d, work_bytes, m, n, k, (hipStream_t)stream);
}

int int4linear_layer_norm(const void *x_d, int type, size_t ld, const float *gamma_d, const float *beta_d, float eps, void *y_d, int out_type,
                          size_t ld_y, int rows, int n, void *stream)
{
    return layer_norm({x_d, type, ld, rows, n, true, gamma_d, beta_d, eps, kRowTyped, y_d, out_type, ld_y, nullptr}, stream);
}

int int4linear_layer_norm_int8(const void *x_d, int type, size_t ld, const float *gamma_d, const float *beta_d, float eps, void *codes_d,
                               float *scales_d, int rows, int n, void *stream)
{
    return layer_norm({x_d, type, ld, rows, n, true, gamma_d, beta_d, eps, kRowInt8, codes_d, 0, 0, scales_d}, stream);
}

int int4linear_layer_norm_mxfp4(const void *x_d, int type, size_t ld, const float *gamma_d, const float *beta_d, float eps, void *codes_d,
                                void *scales_d, int rows, int n, void *stream)
{
    return layer_norm({x_d, type, ld, rows, n, true, gamma_d, beta_d, eps, kRowMx, codes_d, 0, 0, scales_d}, stream);
}

size_t int4linear_layer_norm_backward_bytes(int rows, int n) { return rows < 0 || n < 0 ? 0 : layer_norm_work_bytes(rows, n); }

int int4linear_layer_norm_backward(const void *dy_d, int dy_type, size_t ld_dy, const void *x_d, int type, size_t ld, const float *gamma_d,
                                   float eps, void *dx_d, size_t ld_dx, float *dgamma_d, float *dbeta_d, void *work_d, size_t work_bytes,
                                   int rows, int n, void *stream)
{
    Checks ok;
    ok.sizes(rows, n, 0).apart(ld_dy, n).apart(ld, n);
    if (dx_d)
        ok.apart(ld_dx, n);
    ok.that(n <= kMostNorm && is_type(dy_type) && is_type(type) && eps >= 0.0f && std::isfinite(eps), INT4LINEAR_ERR_UNSUPPORTED);
    const bool want_dx = dx_d && rows > 0;
    if (!ok || n == 0 || (!want_dx && !dgamma_d && !dbeta_d))
        return ok.status;
    ok.array(dy_d, type_bytes(dy_type), rows > 0).array(x_d, type_bytes(type), rows > 0).optional(gamma_d, 4);
    ok.optional(dx_d, type_bytes(type)).optional(dgamma_d, 4).optional(dbeta_d, 4);
    const size_t need = layer_norm_work_bytes(rows, n);
    ok.array(work_d, 256, need > 0).that(work_bytes >= need, INT4LINEAR_ERR_SCRATCH);
    if (!ok)
        return ok.status;
    DeviceInfo info;
    const int st = api_begin((hipStream_t)stream, &info);
    if (st != INT4LINEAR_OK)
        return st;
    const NormBackward p{dy_d, dy_type, ld_dy, x_d, type, ld, gamma_d, eps, want_dx ? dx_d : nullptr, ld_dx, dgamma_d, dbeta_d, rows, n, work_d};
    return api_status(launch_norm_backward(p, info, (hipStream_t)stream));
}

}  // extern "C"
