// The norm's gradients.  With h = (x - mean) r, r = 1 / sqrt(variance + eps), g = dy gamma, and means over a row:
//   dx = r (g - mean(g) - h mean(g h)),   dgamma = sum over rows of dy h,   dbeta = sum over rows of dy.
// The forward pass leaves nothing behind: a row's mean and r follow from x, which has to be read in any case.
#include "row_math.h"

#include <type_traits>

namespace int4linear {

namespace {

constexpr int kThreads = 256;
constexpr int kStrips = 256;  // rows are summed in as many strips at most, and the strips' sums then in order

template <int TYPE>
using Element = OutElement<TYPE>;

struct BackwardStatistics {
    float shift, delta, r, mean_g, mean_gh;
};

struct WorkParts {
    float *partial;             // strips x 2 n: dgamma's, dbeta's
    BackwardStatistics *rows;
    size_t bytes;
};

int strips_of(int rows) { return min(rows, kStrips); }

WorkParts parts(void *work, int rows, int n)
{
    const size_t partial = ((size_t)strips_of(rows) * 2 * n * sizeof(float) + 255) / 256 * 256;
    const size_t statistics = ((size_t)rows * sizeof(BackwardStatistics) + 255) / 256 * 256;
    return {(float *)work, (BackwardStatistics *)((uint8_t *)work + partial), partial + statistics};
}

// Rows of any length: a workgroup finds a row's means, reading it three times ...
template <int TYPE, int DY>
__global__ __launch_bounds__(kThreads) void norm_statistics_kernel(NormBackward p, BackwardStatistics *to)
{
    constexpr int kWaves = kThreads / 64;
    __shared__ float room[3][2 * kWaves];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (int row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const Element<TYPE> *x = (const Element<TYPE> *)p.x + (size_t)row * p.ld;
        const Element<DY> *dy = (const Element<DY> *)p.dy + (size_t)row * p.ld_dy;
        float v[8], g[8], w[8];
        float sum[1] = {};
        for (int c0 = threadIdx.x * 8; c0 < p.n; c0 += kThreads * 8) {
            load8(x, c0, p.n, v);
#pragma unroll
            for (int e = 0; e < 8; ++e)
                sum[0] += v[e];
        }
        group_all<Add>(sum, room[0], wave, kWaves);
        const float shift = sum[0] / (float)p.n;
        float two[2] = {};
        for (int c0 = threadIdx.x * 8; c0 < p.n; c0 += kThreads * 8) {
            load8(x, c0, p.n, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float d = c0 + e < p.n ? v[e] - shift : 0.0f;
                two[0] += d;
                two[1] += d * d;
            }
        }
        group_all<Add>(two, room[1], wave, kWaves);
        const RowStatistics s = RowStatistics::from(shift, two[0], two[1], p.n, p.eps);
        float means[2] = {};
        for (int c0 = threadIdx.x * 8; c0 < p.n; c0 += kThreads * 8) {
            load8(x, c0, p.n, v);
            load8(dy, c0, p.n, g);
            if (p.gamma)
                load8(p.gamma, c0, p.n, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float a = p.gamma ? g[e] * w[e] : g[e];
                if (c0 + e < p.n) {
                    means[0] += a;
                    means[1] += a * s.normalised(v[e]);
                }
            }
        }
        group_all<Add>(means, room[2], wave, kWaves);
        if (threadIdx.x == 0)
            to[row] = {s.shift, s.delta, s.r, means[0] / (float)p.n, means[1] / (float)p.n};
    }
}

// ... and a thread walks a column of a strip of rows.
template <int TYPE, int DY>
__global__ __launch_bounds__(kThreads) void norm_columns_kernel(NormBackward p, const BackwardStatistics *of, float *partial, int per_strip)
{
    const int c = blockIdx.x * kThreads + threadIdx.x, first = blockIdx.y * per_strip, last = min(first + per_strip, p.rows);
    if (c >= p.n)
        return;
    const float w = p.gamma ? p.gamma[c] : 1.0f;
    float dgamma = 0.0f, dbeta = 0.0f;
    for (int row = first; row < last; ++row) {
        const BackwardStatistics s = of[row];
        const float g = (float)((const Element<DY> *)p.dy)[(size_t)row * p.ld_dy + c];
        const float h = (((float)((const Element<TYPE> *)p.x)[(size_t)row * p.ld + c] - s.shift) - s.delta) * s.r;
        dgamma += g * h;
        dbeta += g;
        if (p.dx)
            ((Element<TYPE> *)p.dx)[(size_t)row * p.ld_dx + c] = (Element<TYPE>)(s.r * (g * w - s.mean_g - h * s.mean_gh));
    }
    float *to = partial + (size_t)blockIdx.y * 2 * p.n + c;
    to[0] = dgamma;
    to[p.n] = dbeta;
}

// dgamma and dbeta from the strips' sums, in their order.
__global__ __launch_bounds__(kThreads) void norm_sums_kernel(const float *partial, int strips, int n, float *dgamma, float *dbeta)
{
    const int c = blockIdx.x * kThreads + threadIdx.x;
    if (c >= 2 * n)
        return;
    float sum = 0.0f;
    for (int s = 0; s < strips; ++s)
        sum += partial[(size_t)s * 2 * n + c];
    if (c < n) {
        if (dgamma)
            dgamma[c] = sum;
    } else if (dbeta) {
        dbeta[c - n] = sum;
    }
}

template <int TYPE, int DY>
hipError_t launch(const NormBackward &p, hipStream_t stream)
{
    const WorkParts w = parts(p.work, p.rows, p.n);
    if (p.rows > 0) {
        norm_statistics_kernel<TYPE, DY><<<min(p.rows, 1 << 20), kThreads, 0, stream>>>(p, w.rows);
        const int strips = strips_of(p.rows), per = (p.rows + strips - 1) / strips;
        norm_columns_kernel<TYPE, DY><<<dim3((unsigned)((p.n + kThreads - 1) / kThreads), (unsigned)strips), kThreads, 0, stream>>>(p, w.rows, w.partial, per);
    }
    if (p.dgamma || p.dbeta)
        norm_sums_kernel<<<(2 * p.n + kThreads - 1) / kThreads, kThreads, 0, stream>>>(w.partial, strips_of(p.rows), p.n, p.dgamma, p.dbeta);
    return hipGetLastError();
}

template <int TYPE>
hipError_t by_dy(const NormBackward &p, hipStream_t stream)
{
    return p.dy_type == kOutF32   ? launch<TYPE, kOutF32>(p, stream)
           : p.dy_type == kOutF16 ? launch<TYPE, kOutF16>(p, stream)
                                  : launch<TYPE, kOutBF16>(p, stream);
}

}  // namespace

size_t layer_norm_work_bytes(int rows, int n) { return parts(nullptr, rows, n).bytes; }

hipError_t launch_norm_backward(const NormBackward &p, const DeviceInfo &, hipStream_t stream)
{
    return p.type == kOutF32 ? by_dy<kOutF32>(p, stream) : p.type == kOutF16 ? by_dy<kOutF16>(p, stream) : by_dy<kOutBF16>(p, stream);
}

}  // namespace int4linear
