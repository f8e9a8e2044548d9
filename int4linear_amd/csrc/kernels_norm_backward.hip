// The norm's gradients.  With h = (x - mean) r, r = 1 / sqrt(variance + eps), g = dy gamma, and means over a row:
//   dx = r (g - mean(g) - h mean(g h)),   dgamma = sum over rows of dy h,   dbeta = sum over rows of dy.
// The forward pass leaves nothing behind: a row's mean and r follow from x, which has to be read in any case.
#include "row_math.h"

#include <type_traits>

namespace int4linear {

namespace {

constexpr int kThreads = 256;
// Rows are summed in as many strips at most, and the strips' sums then in order.
constexpr int kStrips = 256, kLongStrips = 64;
constexpr int kMostInRegisters = 16384;  // columns; longer rows are read more than once

template <int TYPE>
using Element = OutElement<TYPE>;

struct BackwardStatistics {
    RowStatistics of;
    float mean_g, mean_gh;
};

struct WorkParts {
    float *partial;             // strips x 2 n: dgamma's, dbeta's
    BackwardStatistics *rows;
    size_t bytes;
};

int strips_of(int rows, int n) { return min(rows, n > kMostInRegisters ? kLongStrips : kStrips); }

WorkParts parts(void *work, int rows, int n)
{
    const size_t partial = ((size_t)strips_of(rows, n) * 2 * n * sizeof(float) + 255) / 256 * 256;
    const size_t statistics = ((n > kMostInRegisters ? (size_t)rows * sizeof(BackwardStatistics) : 0) + 255) / 256 * 256;
    return {(float *)work, (BackwardStatistics *)((uint8_t *)work + partial), partial + statistics};
}

// Rows of any length: a workgroup finds a row's means, reading x three times, from the caches but for the first, and dy once (2000 x 40000
// bf16: 138 us, 320 MB, 2.3 TB/s) ...
template <int TYPE, int DY>
__global__ __launch_bounds__(kThreads) void norm_statistics_kernel(NormBackward p, BackwardStatistics *to)
{
    constexpr int kWaves = kThreads / 64;
    __shared__ float room[3][2 * kWaves];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const float over_n = 1.0f / (float)p.n;
    for (int row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const Element<TYPE> *x = (const Element<TYPE> *)p.x + (size_t)row * p.ld;
        const Element<DY> *dy = (const Element<DY> *)p.dy + (size_t)row * p.ld_dy;
        float v[8], g[8], w[8];
        float sum[1] = {};
        for (int c0 = threadIdx.x * 8; c0 < p.n; c0 += kThreads * 8) {
            load8(x, c0, p.n, v);
#pragma unroll
            for (int e = 0; e < 8; ++e)
                add_part(sum[0], v[e]);
        }
        group_all<Add>(sum, room[0], wave, kWaves);
        const float shift = row_shift(sum[0], over_n);
        float two[2] = {};
        for (int c0 = threadIdx.x * 8; c0 < p.n; c0 += kThreads * 8) {
            load8(x, c0, p.n, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float d = c0 + e < p.n ? v[e] - shift : 0.0f;
                two[0] += d;
                two[1] = fmaf(d, d, two[1]);
            }
        }
        group_all<Add>(two, room[1], wave, kWaves);
        const RowStatistics s = RowStatistics::from(shift, two[0], two[1], over_n, p.eps);
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
                    means[1] = fmaf(a, s.of(v[e]), means[1]);
                }
            }
        }
        group_all<Add>(means, room[2], wave, kWaves);
        if (threadIdx.x == 0)
            to[row] = {s, means[0] * over_n, means[1] * over_n};
    }
}

// ... and a wave walks 512 columns of a strip of rows, eight a lane, reading x and dy again; a workgroup's waves take every fourth row each, and
// their sums are added in order (83 us there, 480 MB, 5.7 TB/s; with the strips' sums the whole call takes 230).
constexpr int kColumns = 64 * 8;

template <int TYPE, int DY>
__global__ __launch_bounds__(kThreads) void norm_columns_kernel(NormBackward p, const BackwardStatistics *of, float *partial, int per_strip)
{
    using X = Element<TYPE>;
    using D = Element<DY>;
    constexpr int kWaves = kThreads / 64, kAhead = 2;  // rows whose values are on their way together
    __shared__ float sums[kWaves - 1][2][kColumns];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c0 = blockIdx.x * kColumns + lane * 8;
    const int first = blockIdx.y * per_strip, last = min(first + per_strip, p.rows);
    float gamma[8], dgamma[8] = {}, dbeta[8] = {};
#pragma unroll
    for (int e = 0; e < 8; ++e)
        gamma[e] = 1.0f;
    if (p.gamma)
        load8(p.gamma, c0, p.n, gamma);
    for (int at = first + wave; at < last; at += kWaves * kAhead) {
        Eight<X> in_x[kAhead];
        Eight<D> in_dy[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int row = min(at + u * kWaves, last - 1);
            fetch8((const X *)p.x + (size_t)row * p.ld, c0, p.n, in_x[u]);
            fetch8((const D *)p.dy + (size_t)row * p.ld_dy, c0, p.n, in_dy[u]);
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int row = at + u * kWaves;
            if (row >= last)
                break;
            const BackwardStatistics s = of[row];
            const float less = -s.of.r * s.mean_g, along = -s.of.r * s.mean_gh;
            float x[8], dy[8], out[8];
            widen8<X>(in_x[u], c0, p.n, x);
            widen8<D>(in_dy[u], c0, p.n, dy);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float h = s.of.of(x[e]);
                out[e] = fmaf(h, along, fmaf(dy[e] * gamma[e], s.of.r, less));
                dgamma[e] = fmaf(dy[e], h, dgamma[e]);
                dbeta[e] += dy[e];
            }
            if (p.dx)
                store8((X *)p.dx + (size_t)row * p.ld_dx, c0, p.n, out);
        }
    }
    if (wave > 0) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            sums[wave - 1][0][e * 64 + lane] = dgamma[e];
            sums[wave - 1][1][e * 64 + lane] = dbeta[e];
        }
    }
    __syncthreads();
    if (wave > 0)
        return;
    for (int w = 0; w < kWaves - 1; ++w)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            dgamma[e] += sums[w][0][e * 64 + lane];
            dbeta[e] += sums[w][1][e * 64 + lane];
        }
    float *to = partial + (size_t)blockIdx.y * 2 * p.n;
    store8(to, c0, p.n, dgamma);
    store8(to + p.n, c0, p.n, dbeta);
}

// (128 registers for each of 1024 threads hold eight columns a lane, 256 for each of 512 two or four times as many; of four times, some
// are kept in memory: 60 to 212 bytes a lane.)
template <int C>
constexpr int most_threads = C == 1 ? 1024 : 512;

// Rows that fit registers, read once.  WAVES waves share a row, C times eight columns a lane (or LANES lanes of one wave, eight columns
// each, and the wave has 64 / LANES rows); a workgroup takes a row, or a wave's, for each of its blockDim.y groups at a time and stays:
// gamma and the columns' sums are in registers, the next rows' values on their way while these rows' sums are made.
// A row's four sums are made in two meetings, since g h summed over the row is r (sum of g d) + c (sum of g) with d = x - shift.  At
// the end the groups' columns' sums meet in LDS and are added in the groups' order.  x, dy and dx of 16384 x 4096 bf16 in 80 us, 5.0 TB/s,
// as a copy; 4096 x 16384 168 us, since it spills; 65536 x 128, eight rows a wave, 18.3 us (one row a wave 55.5).
template <int TYPE, int DY, int WAVES, int C, int LANES>
__global__ __launch_bounds__(most_threads<C>) void norm_backward_kernel(NormBackward p, float *partial)
{
    constexpr int kAcross = WAVES * 64 * 8;
    extern __shared__ float columns[];  // n for each group, where there is more than one (32 KiB at most)
    __shared__ float rooms[2][most_threads<C> / 64 * 5];
    using X = Element<TYPE>;
    using D = Element<DY>;
    static_assert(LANES == 64 || (WAVES == 1 && C == 1));
    constexpr int kRows = 64 / LANES;  // of a group
    const int group = threadIdx.y, groups = blockDim.y, first = (LANES < 64 ? threadIdx.x % LANES : threadIdx.x) * 8;
    const int wave = WAVES == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const float over_n = 1.0f / (float)p.n;
    Eight<X> in_x[C];
    Eight<D> in_dy[C];
    float gamma[C][8], dgamma[C][8] = {}, dbeta[C][8] = {};
    auto fetch = [&](int row) {
        const X *x = (const X *)p.x + (size_t)row * p.ld;
        const D *dy = (const D *)p.dy + (size_t)row * p.ld_dy;
#pragma unroll
        for (int i = 0; i < C; ++i) {
            fetch8(x, first + i * kAcross, p.n, in_x[i]);
            fetch8(dy, first + i * kAcross, p.n, in_dy[i]);
        }
    };
#pragma unroll
    for (int i = 0; i < C; ++i) {
        in_x[i] = (Eight<X>)(X)0.0f;
        in_dy[i] = (Eight<D>)(D)0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e)
            gamma[i][e] = 1.0f;
        if (p.gamma)
            load8(p.gamma, first + i * kAcross, p.n, gamma[i]);
    }
    const int by = gridDim.x * groups * kRows;
    int row = (blockIdx.x * groups + group) * kRows + (LANES < 64 ? (int)threadIdx.x / LANES : 0);
    if (row < p.rows)
        fetch(row);
    // (every group makes as many turns, for their meetings; one without a row has zeros)
    int turn = 0;
    for (int base = blockIdx.x * groups * kRows; base < p.rows; base += by, row += by, turn ^= 1) {
        float x[C][8], dy[C][8];
        const bool there = row < p.rows;
#pragma unroll
        for (int i = 0; i < C; ++i) {
            widen8<X>(in_x[i], first + i * kAcross, p.n, x[i]);
            widen8<D>(in_dy[i], first + i * kAcross, p.n, dy[i]);
        }
        if (!there) {
#pragma unroll
            for (int i = 0; i < C; ++i)
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    x[i][e] = dy[i][e] = 0.0f;
        }
        if (row + by < p.rows)
            fetch(row + by);
        float *room = rooms[turn] + group * WAVES * 5;
        float sum[1] = {}, four[4] = {};
#pragma unroll
        for (int i = 0; i < C; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e)
                add_part(sum[0], x[i][e]);
        group_all<Add, LANES>(sum, room, wave, WAVES);
        const float shift = row_shift(sum[0], over_n);
#pragma unroll
        for (int i = 0; i < C; ++i) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                x[i][e] -= shift;
            behind8(first + i * kAcross, p.n, 0.0f, x[i]);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float g = dy[i][e] * gamma[i][e];
                four[0] += x[i][e];
                four[1] = fmaf(x[i][e], x[i][e], four[1]);
                four[2] += g;
                four[3] = fmaf(g, x[i][e], four[3]);
            }
        }
        group_all<Add, LANES>(four, room + WAVES, wave, WAVES);
        const RowStatistics s = RowStatistics::from(shift, four[0], four[1], over_n, p.eps);
        if (s.flat) {  // rare
            four[3] = 0.0f;
#pragma unroll
            for (int i = 0; i < C; ++i)
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    x[i][e] = 0.0f;
        }
        const float mean_g = four[2] * over_n, mean_gh = fmaf(s.r, four[3], s.c * four[2]) * over_n;
        const float less = -s.r * mean_g, along = -s.r * mean_gh;
        X *dx = (X *)p.dx + (size_t)row * p.ld_dx;
#pragma unroll
        for (int i = 0; i < C; ++i) {
            float out[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float h = s.normalised(x[i][e]), g = dy[i][e] * gamma[i][e];
                out[e] = fmaf(h, along, fmaf(g, s.r, less));
                if (there) {
                    dgamma[i][e] = fmaf(dy[i][e], h, dgamma[i][e]);
                    dbeta[i][e] += dy[i][e];
                }
            }
            if (there && p.dx && first + i * kAcross < p.n)
                store8(dx, first + i * kAcross, p.n, out);
        }
    }
    if (!partial)
        return;
    if constexpr (LANES < 64) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            dgamma[0][e] = across_all<LANES>(dgamma[0][e], Add{});
            dbeta[0][e] = across_all<LANES>(dbeta[0][e], Add{});
        }
    }
    float *to = partial + (size_t)blockIdx.x * 2 * p.n;
    if (groups == 1) {
        if (LANES == 64 || threadIdx.x < LANES) {
#pragma unroll
            for (int i = 0; i < C; ++i) {
                store8(to, first + i * kAcross, p.n, dgamma[i]);
                store8(to + p.n, first + i * kAcross, p.n, dbeta[i]);
            }
        }
        return;
    }
    auto add_groups = [&](const float(&sums)[C][8], float *result) {
        if (LANES == 64 || threadIdx.x < LANES) {
#pragma unroll
            for (int i = 0; i < C; ++i)
                store8(columns + (size_t)group * p.n, first + i * kAcross, p.n, sums[i]);
        }
        __syncthreads();
        for (int c = group * WAVES * 64 + threadIdx.x; c < p.n; c += groups * WAVES * 64) {
            float sum = columns[c];
            for (int g = 1; g < groups; ++g)
                sum += columns[g * p.n + c];
            result[c] = sum;
        }
        __syncthreads();
    };
    add_groups(dgamma, to);
    add_groups(dbeta, to + p.n);
}

// dgamma and dbeta from the strips' sums: 64 columns to a workgroup, a wave to every sixteenth strip; the waves' sums in their order.
__global__ __launch_bounds__(1024) void norm_sums_kernel(const float *partial, int strips, int n, float *dgamma, float *dbeta)
{
    __shared__ float part[1024];
    const int c = blockIdx.x * 64 + (threadIdx.x & 63), wave = threadIdx.x >> 6;
    float sum = 0.0f;
    if (c < 2 * n) {
#pragma unroll 16
        for (int s = wave; s < strips; s += 16)
            sum += partial[(size_t)s * 2 * n + c];
    }
    part[threadIdx.x] = sum;
    __syncthreads();
    if (wave != 0 || c >= 2 * n)
        return;
    for (int w = 1; w < 16; ++w)
        sum += part[w * 64 + threadIdx.x];
    if (c < n) {
        if (dgamma)
            dgamma[c] = sum;
    } else if (dbeta) {
        dbeta[c - n] = sum;
    }
}

template <int TYPE, int DY>
hipError_t launch(const NormBackward &p, const DeviceInfo &dev, hipStream_t stream)
{
    const WorkParts w = parts(p.work, p.rows, p.n);
    const int cus = min(dev.cu_count > 0 ? dev.cu_count : kStrips, kStrips);
    int strips = 0;
    auto run = [&](auto waves, auto c, auto lanes) {
        constexpr int WAVES = decltype(waves)::value, C = decltype(c)::value, LANES = decltype(lanes)::value, kRows = 64 / LANES;
        const int waves_of_rows = (p.rows + kRows - 1) / kRows;
        const int groups = min((waves_of_rows + cus - 1) / cus, most_threads<C> / 64 / WAVES);
        strips = min((waves_of_rows + groups - 1) / groups, cus);
        norm_backward_kernel<TYPE, DY, WAVES, C, LANES><<<strips, dim3(WAVES * 64, (unsigned)groups), groups > 1 ? groups * p.n * sizeof(float) : 0, stream>>>(
            p, p.dgamma || p.dbeta ? w.partial : nullptr);
    };
#define I4L_LANES(WAVES, C, LANES) run(std::integral_constant<int, WAVES>{}, std::integral_constant<int, C>{}, std::integral_constant<int, LANES>{})
#define I4L_RUN(WAVES, C) I4L_LANES(WAVES, C, 64)
    if (p.rows > 0) {
        if (p.n <= 64)
            I4L_LANES(1, 1, 8);
        else if (p.n <= 128)
            I4L_LANES(1, 1, 16);
        else if (p.n <= 256)
            I4L_LANES(1, 1, 32);
        else if (p.n <= 512)
            I4L_RUN(1, 1);
        else if (p.n <= 1024)
            I4L_RUN(2, 1);
        else if (p.n <= 2048)
            I4L_RUN(2, 2);
        else if (p.n <= 4096)
            I4L_RUN(4, 2);
        else if (p.n <= 8192)
            I4L_RUN(8, 2);
        else if (p.n <= kMostInRegisters)
            I4L_RUN(8, 4);
        else {
            strips = strips_of(p.rows, p.n);
            norm_statistics_kernel<TYPE, DY><<<min(p.rows, 1 << 20), kThreads, 0, stream>>>(p, w.rows);
            norm_columns_kernel<TYPE, DY><<<dim3((unsigned)((p.n + kColumns - 1) / kColumns), (unsigned)strips), kThreads, 0, stream>>>(
                p, w.rows, w.partial, (p.rows + strips - 1) / strips);
        }
    }
#undef I4L_RUN
#undef I4L_LANES
    if (p.dgamma || p.dbeta)
        norm_sums_kernel<<<(2 * p.n + 63) / 64, 1024, 0, stream>>>(w.partial, strips, p.n, p.dgamma, p.dbeta);
    return hipGetLastError();
}

template <int TYPE>
hipError_t by_dy(const NormBackward &p, const DeviceInfo &dev, hipStream_t stream)
{
    return p.dy_type == kOutF32   ? launch<TYPE, kOutF32>(p, dev, stream)
           : p.dy_type == kOutF16 ? launch<TYPE, kOutF16>(p, dev, stream)
                                  : launch<TYPE, kOutBF16>(p, dev, stream);
}

}  // namespace

size_t layer_norm_work_bytes(int rows, int n) { return parts(nullptr, rows, n).bytes; }

hipError_t launch_norm_backward(const NormBackward &p, const DeviceInfo &dev, hipStream_t stream)
{
    return p.type == kOutF32   ? by_dy<kOutF32>(p, dev, stream)
           : p.type == kOutF16 ? by_dy<kOutF16>(p, dev, stream)
                               : by_dy<kOutBF16>(p, dev, stream);
}

}  // namespace int4linear
