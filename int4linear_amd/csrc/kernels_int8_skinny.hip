// Few rows of x against 8-bit weights: every byte of w is read once, and the stream of w is what bounds it.
//
// One and two rows, three and four against fewer than 8192 of w: two waves share the k of two rows of w, 16 bytes a lane, so that a load is 1 KB of
// one row, straight into registers; four products to an instruction (v_dot4_i32_i8) are enough for what arrives, and the lanes' sums meet
// once at the end, then those of the two waves in LDS.  8192 x 8192, one row, weights from HBM: 11.6 us = 5.8 TB/s; a kernel that does nothing but
// read as much takes 11.1.
// More: a workgroup takes 16 R rows of w and all of k, its waves split k line by line.  A wave's lines of w and x go straight to LDS
// (eight rows of 128 bytes an instruction), those of its next line while it multiplies this one's with v_mfma_i32_16x16x64_i8, and the
// waves' sums meet in LDS.  Workgroups begin at different lines: rows lie a power of two apart as often as not, and where all begin
// at line 0 all are at the same few memory channels all the time (16 rows against 8192 x 8192 20.0 us, so 13.7; against 28672 x 8192
// 56, 41 us = 5.7 TB/s).  Sums of whole numbers: nothing depends on who adds when, or where.
#include "int8.h"
#include "mxfp4_epilogue.h"

namespace int4linear {

namespace {

typedef int v4i __attribute__((ext_vector_type(4)));

struct SkinnyArgs {
    const uint8_t *x, *w;
    unsigned stride;
    const float *xs, *ws, *bias;
    void *y;
    int out, m, n;
};

template <int OUT>
__device__ __forceinline__ void store(void *y, size_t at, float v)
{
    ((OutElement<OUT> *)y)[at] = (OutElement<OUT>)v;
}

__device__ __forceinline__ void finish(const SkinnyArgs &g, int r, int c, int sum)
{
    const float v = (float)sum * g.xs[r] * g.ws[c] + (g.bias ? g.bias[c] : 0.0f);
    const size_t at = (size_t)r * g.n + c;
    if (g.out == kOutF32)
        store<kOutF32>(g.y, at, v);
    else if (g.out == kOutF16)
        store<kOutF16>(g.y, at, v);
    else
        store<kOutBF16>(g.y, at, v);
}

__device__ __forceinline__ int wave_sum(int v)
{
    v += __builtin_amdgcn_mov_dpp(v, 0xB1, 0xF, 0xF, true);   // lanes 1 0 3 2
    v += __builtin_amdgcn_mov_dpp(v, 0x4E, 0xF, 0xF, true);   // lanes 2 3 0 1
    v += __builtin_amdgcn_mov_dpp(v, 0x141, 0xF, 0xF, true);  // 7 .. 0
    v += __builtin_amdgcn_mov_dpp(v, 0x140, 0xF, 0xF, true);  // 15 .. 0
    const auto rows = __builtin_amdgcn_permlane16_swap((unsigned)v, (unsigned)v, false, false);
    v = (int)(rows[0] + rows[1]);
    const auto halves = __builtin_amdgcn_permlane32_swap((unsigned)v, (unsigned)v, false, false);
    return (int)(halves[0] + halves[1]);
}

// (A launch holds fewer than 2^32 threads along x.)
constexpr unsigned kMostAlongX = 1u << 20;
__device__ __forceinline__ int block_number() { return (int)(blockIdx.y * kMostAlongX + blockIdx.x); }
dim3 blocks(int count)
{
    return dim3(min((unsigned)count, kMostAlongX), ((unsigned)count + kMostAlongX - 1) / kMostAlongX);
}

// M rows of x; kDotShare waves take kDotRows rows of w and share k.  (us with one row of w a wave, two, four, and with two that two and
// four waves share: one row of x against 8192 x 8192 11.6, 12.9, 13.1, 11.7, 11.7; 14336 x 4096 10.4, 10.5, 13.0, 10.6, 10.7; 4096 x
// 14336 10.9, 10.7, 11.2, 10.6, 10.6; four rows against 8192 x 8192 19.3, 16.1, 15.3, 15.8, 17.2.)
constexpr int kDotWaves = 4, kDotShare = 2, kDotRows = 2, kDotBytes = 64 * 16, kDotAhead = 4;

template <int M>
__global__ __launch_bounds__(kDotWaves * 64) void int8_dot_kernel(SkinnyArgs g)
{
    constexpr int R = kDotRows, split = kDotShare;
    __shared__ int part[kDotWaves][R * M];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int group = wave / split, share = wave % split;
    const int row = (block_number() * (kDotWaves / split) + group) * R;
    const uint8_t *w[R];
#pragma unroll
    for (int r = 0; r < R; ++r)
        w[r] = uniform(g.w + (size_t)min(row + r, g.n - 1) * g.stride);
    int acc[R][M] = {};
    for (unsigned at = share * kDotBytes + lane * 16; at - lane * 16 < g.stride; at += split * kDotBytes * kDotAhead) {
        v4i a[kDotAhead][M] = {}, b[kDotAhead][R] = {};
#pragma unroll
        for (int u = 0; u < kDotAhead; ++u) {
            const unsigned o = at + u * split * kDotBytes;
            if (o < g.stride) {
#pragma unroll
                for (int r = 0; r < R; ++r)
                    b[u][r] = __builtin_nontemporal_load((const v4i *)(w[r] + o));
#pragma unroll
                for (int m = 0; m < M; ++m)
                    a[u][m] = *(const v4i *)(g.x + (size_t)m * g.stride + o);
            }
        }
#pragma unroll
        for (int u = 0; u < kDotAhead; ++u)
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int m = 0; m < M; ++m)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        acc[r][m] = __builtin_amdgcn_sdot4(b[u][r][e], a[u][m][e], acc[r][m], false);
    }
    int mine = 0;
#pragma unroll
    for (int i = 0; i < R * M; ++i) {
        const int sum = wave_sum(acc[i / M][i % M]);
        mine = lane == i ? sum : mine;
    }
    if (lane < R * M)
        part[wave][lane] = mine;
    __syncthreads();
    if (share == 0 && lane < R * M)
        for (int s = 1; s < split; ++s)
            mine += part[wave + s][lane];
    if (share == 0 && lane < R * M && row + lane / M < g.n)
        finish(g, lane % M, row + lane / M, mine);
}

#define I4L_LDS(p) ((__attribute__((address_space(3))) void *)(p))

constexpr int kRows = 16, kLine = 128, kTileBytes = kRows * kLine;

template <int R, int FM>
constexpr int wave_lds = 2 * (R + FM) * kTileBytes;

// R x FM fragments of w and x.
template <int R, int FM>
__global__ __launch_bounds__(512) void int8_skinny_kernel(SkinnyArgs g)
{
    constexpr int kLoads = 2 * (R + FM);
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int waves = blockDim.x >> 6;
    const int number = block_number(), n0 = number * R * kRows;
    if (n0 >= g.n)
        return;
    uint8_t *mine = lds + wave * wave_lds<R, FM>;
    const unsigned my_lds = __builtin_amdgcn_readfirstlane((int)(size_t)I4L_LDS(mine));
    // Rows behind a matrix: its last one again.  The chunk that lies at place p of row r is p ^ (r / 2 % 8).
    const uint8_t *w = uniform(g.w + (size_t)n0 * g.stride), *x = g.x;
    unsigned off[R + FM][2];
#pragma unroll
    for (int f = 0; f < R + FM; ++f)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = 8 * h + (lane >> 3), last = f < R ? g.n - 1 - n0 : g.m - 1;
            off[f][h] = (unsigned)min((f < R ? f : f - R) * kRows + r, last) * g.stride + (((lane & 7) ^ ((r >> 1) & 7)) << 4);
        }
    const int lines = (int)(g.stride / kLine);
    const int turned = (int)((size_t)number * (waves + 1) % lines);
    // The line that is number t of this workgroup's order into buffer b.  (Behind the last: that one again, into a buffer that nobody
    // reads.)
    auto load = [&](int t, int b) {
        const unsigned to = my_lds + b * (wave_lds<R, FM> / 2);
        int line = min(t, lines - 1) + turned;
        line = line >= lines ? line - lines : line;
        const size_t at = (size_t)line * kLine;
#pragma unroll
        for (int f = 0; f < R + FM; ++f)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (f < R)
                    dma16<true>(w + at, off[f][h], to + f * kTileBytes + h * 1024);
                else
                    dma16(x + at, off[f][h], to + f * kTileBytes + h * 1024);
            }
    };
    const int row = lane & 15, q = lane >> 4;
    v4i acc[R][FM] = {};
    load(wave, 0);
    for (int t = wave, b = 0; t < lines; t += waves, b ^= 1) {
        load(t + waves, b ^ 1);
        asm volatile("s_waitcnt vmcnt(%0)" : : "n"(kLoads) : "memory");
        const uint8_t *from = mine + b * (wave_lds<R, FM> / 2) + row * kLine;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int place = ((q + 4 * i) ^ ((row >> 1) & 7)) << 4;
            v4i xf[FM];
#pragma unroll
            for (int j = 0; j < FM; ++j)
                xf[j] = *(const v4i *)(from + (R + j) * kTileBytes + place);
#pragma unroll
            for (int f = 0; f < R; ++f) {
                const v4i wf = *(const v4i *)(from + f * kTileBytes + place);
#pragma unroll
                for (int j = 0; j < FM; ++j)
                    acc[f][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf, xf[j], acc[f][j], 0, 0, 0);
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // read before it is loaded again
    }
    // Element t of a lane: column n0 + 16 f + 4 (lane / 16) + t of row m0 + 16 j + lane % 16.  Every wave leaves its sums where its
    // lines were; then they are added up.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    v4i *sums = (v4i *)mine;
#pragma unroll
    for (int f = 0; f < R; ++f)
#pragma unroll
        for (int j = 0; j < FM; ++j)
            sums[(f * FM + j) * 64 + lane] = acc[f][j];
    __syncthreads();
    for (int i = wave; i < R * FM; i += waves) {
        const int f = i / FM, j = i % FM;
        const v4i *from = (const v4i *)lds + i * 64 + lane;
        v4i s = from[0];
        for (int o = 1; o < waves; ++o)
            s += from[o * (wave_lds<R, FM> / 16)];
        const int r = j * kRows + row, c = n0 + f * kRows + 4 * q;
        if (r < g.m) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (c + e < g.n)
                    finish(g, r, c + e, s[e]);
        }
    }
}

template <int M>
hipError_t launch_dot(const SkinnyArgs &g, hipStream_t stream)
{
    constexpr int kPer = kDotWaves / kDotShare * kDotRows;
    int8_dot_kernel<M><<<blocks((g.n + kPer - 1) / kPer), kDotWaves * 64, 0, stream>>>(g);
    return hipGetLastError();
}

template <int R, int FM>
hipError_t launch_mfma(const SkinnyArgs &g, int waves, hipStream_t stream)
{
    int8_skinny_kernel<R, FM><<<blocks((g.n + R * kRows - 1) / (R * kRows)), waves * 64, (size_t)waves * wave_lds<R, FM>, stream>>>(g);
    return hipGetLastError();
}

// Two fragments of w a workgroup from here on (512 workgroups of one): they read x half as often.
constexpr int kWide = 8192;
constexpr int kMostWaves = 8;

}  // namespace

// Where this kernel is quicker than tiles (of any size, those that have a CU to themselves among them).  us here and on tiles, weights from HBM:
//   rows of x            3            16           32           48           64
//   2048 x 2048          4.8, 5.5     5.1, 5.6     5.1, 5.7     5.7, 5.8     6.1, 5.8
//   4096 x 4096          6.3, 8.3     6.2, 8.3     7.0, 8.4     8.1, 8.5     8.7, 8.5
//   4096 x 14336         13.3, 29.9   13.5, 30.3   16.8, 31.4   20.4, 33.2   22.5, 36.3
//   1024 x 8192          4.7, 13.4    7.7, 13.5    9.8, 13.6    11.6, 13.6   12.8, 13.7
//   8192 x 8192          13.1, 19.9   13.5, 20.1   15.4, 20.7   17.5, 21.5   19.6, 23.1
//   14336 x 4096         11.7, 14.8   12.6, 15.2   14.8, 15.4   18.2, 15.6   23.0, 16.0
//   28672 x 8192         38.2, 51.0   40.6, 48.6   48.1, 51.8   55.3, 52.2   69.7, 52.6
// (It does not look at k: against short rows of w the tiles are 3 to 5 % quicker from 56 rows of x on.)
bool int8_skinny_preferred(int m, int n) { return m <= 32 || (m <= 64 && n <= kWide); }

hipError_t int8_skinny_init()
{
    hipError_t e = hipSuccess;
    auto allow = [&](const void *kernel, int bytes) {
        if (e == hipSuccess)
            e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    };
    allow((const void *)int8_skinny_kernel<1, 1>, kMostWaves * wave_lds<1, 1>);
    allow((const void *)int8_skinny_kernel<1, 2>, kMostWaves * wave_lds<1, 2>);
    allow((const void *)int8_skinny_kernel<1, 3>, kMostWaves * wave_lds<1, 3>);
    allow((const void *)int8_skinny_kernel<1, 4>, kMostWaves * wave_lds<1, 4>);
    allow((const void *)int8_skinny_kernel<2, 1>, kMostWaves / 2 * wave_lds<2, 1>);
    allow((const void *)int8_skinny_kernel<2, 2>, kMostWaves / 2 * wave_lds<2, 2>);
    allow((const void *)int8_skinny_kernel<2, 3>, kMostWaves / 2 * wave_lds<2, 3>);
    allow((const void *)int8_skinny_kernel<2, 4>, kMostWaves / 2 * wave_lds<2, 4>);
    return e;
}

// Four waves, or eight where few workgroups (and few rows of x, which every wave's lines come with) leave room for more loads: 16 rows
// against 4096 x 14336 14.7 us, so 13.6; 1024 x 8192 8.7, 7.9; 32 rows 16.9, 17.1 and 9.9, 10.0.
hipError_t launch_int8_skinny(const Int8Matrix &x, const Int8Matrix &w, const float *bias, void *y, int out, int k, hipStream_t stream)
{
    const SkinnyArgs g{(const uint8_t *)x.codes, (const uint8_t *)w.codes, (unsigned)int8_code_stride(k), x.scales, w.scales, bias, y, out, x.rows, w.rows};
    const bool wide = g.n >= kWide;
    switch (g.m) {
    case 1:
        return launch_dot<1>(g, stream);
    case 2:
        return launch_dot<2>(g, stream);
    case 3:
        if (!wide)
            return launch_dot<3>(g, stream);
        break;
    case 4:
        if (!wide)
            return launch_dot<4>(g, stream);
        break;
    }
    switch ((g.m + kRows - 1) / kRows) {
    case 1:
        return wide ? launch_mfma<2, 1>(g, kMostWaves / 2, stream) : launch_mfma<1, 1>(g, kMostWaves, stream);
    case 2:
        return wide ? launch_mfma<2, 2>(g, kMostWaves / 2, stream) : launch_mfma<1, 2>(g, kMostWaves / 2, stream);
    case 3:
        return wide ? launch_mfma<2, 3>(g, kMostWaves / 2, stream) : launch_mfma<1, 3>(g, kMostWaves / 2, stream);
    case 4:
        return wide ? launch_mfma<2, 4>(g, kMostWaves / 2, stream) : launch_mfma<1, 4>(g, kMostWaves / 2, stream);
    default:
        return hipErrorInvalidValue;
    }
}

}  // namespace int4linear
