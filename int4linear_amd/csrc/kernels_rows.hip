// Passes over rows: the norm y = (x - mean) / sqrt(variance + eps) * gamma + beta, and quantisation to 8 bits by row, alone or
// of what the norm gives.
#include "row_math.h"

#include <type_traits>

namespace int4linear {

namespace {

constexpr int kThreads = 256;
// Fewer rows than this are spread over more waves each.
constexpr int kFewRows = 1024;

template <int TYPE>
using Element = OutElement<TYPE>;

// The form a row leaves in.
template <int RESULT>
struct RowWriter {
    const RowPass &p;
    size_t code_stride, scale_stride;

    // Columns a pass has to cover: the padding of the codes and scales too.
    static __device__ int columns(int n) { return RESULT == kRowTyped ? n : RESULT == kRowInt8 ? (n + 127) / 128 * 128 : (n + 511) / 512 * 512; }

    __device__ __forceinline__ void write(int row, int c0, const float (&v)[8], const RowScale &s) const
    {
        if constexpr (RESULT == kRowTyped) {
            store8_as(p.out, (uint8_t *)p.y + (size_t)row * p.ld_y * (p.out == kOutF32 ? 4 : 2), c0, p.n, v);
        } else if constexpr (RESULT == kRowInt8) {
            row_v2i codes;
            encode_int8(v, s, codes);
            if ((size_t)c0 < code_stride)
                *(row_v2i *)((uint8_t *)p.y + (size_t)row * code_stride + c0) = codes;
            if (c0 == 0)
                ((float *)p.scales)[row] = s.scale;
        } else {
            // a block is a quad of lanes
            unsigned big = 0, code;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                big = max(big, __builtin_bit_cast(unsigned, v[e]) & 0x7FFFFFFFu);
            big = max(big, (unsigned)__builtin_amdgcn_mov_dpp((int)big, 0xB1, 0xF, 0xF, true));
            big = max(big, (unsigned)__builtin_amdgcn_mov_dpp((int)big, 0x4E, 0xF, 0xF, true));
            const unsigned bits = encode_block_part(v, big, code);
            if ((size_t)c0 < code_stride * 2)
                *(unsigned *)((uint8_t *)p.y + (size_t)row * code_stride + c0 / 2) = bits;
            if (c0 % kMxBlock == 0)
                ((uint8_t *)p.scales)[(size_t)row * scale_stride + c0 / kMxBlock] = (uint8_t)code;
        }
    }
};

// h gamma + beta of eight columns from d = x - shift; what is behind the row's end becomes 0.
__device__ __forceinline__ void normalise8(const RowStatistics &s, int c0, int n, const float (&g)[8], const float (&b)[8], float (&v)[8])
{
#pragma unroll
    for (int e = 0; e < 8; ++e)
        v[e] = fmaf(s.normalised(v[e]), g[e], b[e]);
    behind8(c0, n, 0.0f, v);
}

// Columns c0 .. of gamma and beta.
__device__ __forceinline__ void load_affine(const RowPass &p, int c0, float (&g)[8], float (&b)[8])
{
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        g[e] = 1.0f;
        b[e] = 0.0f;
    }
    if (p.gamma)
        load8(p.gamma, c0, p.n, g);
    if (p.beta)
        load8(p.beta, c0, p.n, b);
}

__device__ __forceinline__ void largest8(const float (&v)[8], unsigned &big)
{
#pragma unroll
    for (int e = 0; e < 8; ++e)
        big = max(big, __builtin_bit_cast(unsigned, v[e]) & 0x7FFFFFFFu);
}

// Eight d = x - shift, and their share of the row's sums.
__device__ __forceinline__ void centre8(float shift, int c0, int n, float (&v)[8], float (&two)[2])
{
#pragma unroll
    for (int e = 0; e < 8; ++e)
        v[e] -= shift;
    behind8(c0, n, 0.0f, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        two[0] += v[e];
        two[1] = fmaf(v[e], v[e], two[1]);
    }
}

// Rows of any length: a workgroup takes a row at a time and reads it again in every pass, from the caches: twice for its quantisation, three times
// for a norm, four for a norm into 8 bits (4096 x 28672 bf16 101 us = 3.5 TB/s, 155 = 3.0, 186 = 1.9; into MXFP4 134).
template <int TYPE, int RESULT, bool NORM>
__global__ __launch_bounds__(kThreads) void row_loop_kernel(RowPass p, size_t code_stride, size_t scale_stride)
{
    constexpr int kWaves = kThreads / 64;
    __shared__ float room[3][2 * kWaves];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const RowWriter<RESULT> writer{p, code_stride, scale_stride};
    const float over_n = 1.0f / (float)p.n;
    for (int row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const Element<TYPE> *x = (const Element<TYPE> *)p.x + (size_t)row * p.ld;
        RowStatistics s{};
        float v[8];
        // A pass over the row as it leaves: f(first column, eight values).  (Whole quads of lanes, for MXFP4's blocks.)
        auto pass = [&](int columns, auto &&f) {
            for (int c0 = threadIdx.x * 8; c0 < columns; c0 += kThreads * 8) {
                load8(x, c0, p.n, v);
                if constexpr (NORM) {
                    float g[8], b[8];
                    load_affine(p, c0, g, b);
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        v[e] = s.flat ? 0.0f : v[e] - s.shift;
                    normalise8(s, c0, p.n, g, b, v);
                }
                f(c0, v);
            }
        };
        if constexpr (NORM) {
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
                centre8(shift, c0, p.n, v, two);
            }
            group_all<Add>(two, room[1], wave, kWaves);
            s = RowStatistics::from(shift, two[0], two[1], over_n, p.eps);
        }
        RowScale scale{};
        if constexpr (RESULT == kRowInt8) {
            unsigned big[1] = {};
            pass(p.n, [&](int, const float(&w)[8]) { largest8(w, big[0]); });
            group_all<Larger>(big, (unsigned *)room[2], wave, kWaves);
            scale = RowScale::of(big[0]);
        }
        pass(writer.columns(p.n), [&](int c0, const float(&w)[8]) { writer.write(row, c0, w, scale); });
        if constexpr (!NORM)
            __syncthreads();  // (else the room of one row is used again behind two further meetings)
    }
}

// The same with a row in registers, read once: WAVES waves share it (1: LANES lanes of a wave have a row to themselves, a workgroup four
// rows or more), a lane holds C times eight values, those of chunk i * 64 * WAVES + (its number in the group).  With a norm workgroups
// stay: gamma and beta are read once, and the next row's values are on their way while this one's sums are made (16384 x 8192 bf16
// 145 us a row after the other, so 102 us = 5.2 TB/s, what a copy of 1 GiB runs at).  Without, there is nothing to stay for (8192 x
// 14336 into 8 bits 62 us = 5.7 TB/s; 71 where workgroups stay).
template <int C>
constexpr int waves_per_simd = C <= 2 ? 4 : 3;

template <int TYPE, int RESULT, bool NORM, int WAVES, int C, int LANES>
__global__ __launch_bounds__(WAVES == 1 ? kThreads : WAVES * 64, waves_per_simd<C>) void row_kernel(RowPass p, size_t code_stride, size_t scale_stride)
{
    static_assert(LANES == 64 || (WAVES == 1 && C == 1));
    constexpr int kAcross = WAVES * 64 * 8, kRows = WAVES == 1 ? kThreads / LANES : 1;
    __shared__ float room[2][3][2 * WAVES];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int in_row = WAVES == 1 ? 0 : wave, first = (WAVES == 1 ? threadIdx.x % LANES : threadIdx.x) * 8;
    const RowWriter<RESULT> writer{p, code_stride, scale_stride};
    const float over_n = 1.0f / (float)p.n;
    Eight<Element<TYPE>> in[C];
    auto fetch = [&](int row) {
        const Element<TYPE> *x = (const Element<TYPE> *)p.x + (size_t)row * p.ld;
#pragma unroll
        for (int i = 0; i < C; ++i)
            fetch8(x, first + i * kAcross, p.n, in[i]);
    };
    int row = blockIdx.x * kRows + (LANES < 64 ? (int)threadIdx.x / LANES : WAVES == 1 ? wave : 0), turn = 0;
    if (row >= p.rows)
        return;
    fetch(row);
    float g[C][8], b[C][8];
    if constexpr (NORM)
#pragma unroll
        for (int i = 0; i < C; ++i)
            load_affine(p, first + i * kAcross, g[i], b[i]);
    for (;; turn ^= 1) {
        const int next = row + gridDim.x * kRows;
        float v[C][8];
#pragma unroll
        for (int i = 0; i < C; ++i)
            widen8<Element<TYPE>>(in[i], first + i * kAcross, p.n, v[i]);
        if (next < p.rows)
            fetch(next);
        if constexpr (NORM) {
            float sum[1] = {}, two[2] = {};
#pragma unroll
            for (int i = 0; i < C; ++i)
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    add_part(sum[0], v[i][e]);
            group_all<Add, LANES>(sum, room[turn][0], in_row, WAVES);
            const float shift = row_shift(sum[0], over_n);
#pragma unroll
            for (int i = 0; i < C; ++i)
                centre8(shift, first + i * kAcross, p.n, v[i], two);
            group_all<Add, LANES>(two, room[turn][1], in_row, WAVES);
            const RowStatistics s = RowStatistics::from(shift, two[0], two[1], over_n, p.eps);
            if (s.flat) {  // rare
#pragma unroll
                for (int i = 0; i < C; ++i)
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        v[i][e] = 0.0f;
            }
#pragma unroll
            for (int i = 0; i < C; ++i)
                normalise8(s, first + i * kAcross, p.n, g[i], b[i], v[i]);
        }
        RowScale scale{};
        if constexpr (RESULT == kRowInt8) {
            unsigned big[1] = {};
#pragma unroll
            for (int i = 0; i < C; ++i)
                largest8(v[i], big[0]);
            group_all<Larger, LANES>(big, (unsigned *)room[turn][2], in_row, WAVES);
            scale = RowScale::of(big[0]);
        }
#pragma unroll
        for (int i = 0; i < C; ++i)
            if (first + i * kAcross < writer.columns(p.n))
                writer.write(row, first + i * kAcross, v[i], scale);
        row = next;
        if (row >= p.rows)
            break;
    }
}

// us for 1000 x 4999 f32 by waves and eights a lane: 4, 4 15.4; 8, 2 13.3; 16, 1 15.5; for 4096 x 4096 bf16 into 8 bits: 4, 2 16.6; 8, 1
// 20.5; for 65536 x 1024 bf16: 1, 2 52.
template <int TYPE, int RESULT, bool NORM>
hipError_t launch(const RowPass &p, const DeviceInfo &dev, hipStream_t stream)
{
    const size_t codes = RESULT == kRowInt8 ? int8_code_stride(p.n) : mx_code_stride(p.n), scales = mx_scale_stride(p.n);
    const int cus = dev.cu_count > 0 ? dev.cu_count : 256;
    auto run = [&](auto waves, auto c, auto lanes) {
        constexpr int WAVES = decltype(waves)::value, C = decltype(c)::value, LANES = decltype(lanes)::value, kRows = WAVES == 1 ? kThreads / LANES : 1;
        constexpr int kPlaces = 4 * waves_per_simd<C> / (WAVES == 1 ? kThreads / 64 : WAVES);  // workgroups of a CU
        const int groups = min((p.rows + kRows - 1) / kRows, NORM ? cus * kPlaces : 1 << 20);
        row_kernel<TYPE, RESULT, NORM, WAVES, C, LANES><<<groups, WAVES == 1 ? kThreads : WAVES * 64, 0, stream>>>(p, codes, scales);
        return hipGetLastError();
    };
#define I4L_LANES(WAVES, C, LANES) run(std::integral_constant<int, WAVES>{}, std::integral_constant<int, C>{}, std::integral_constant<int, LANES>{})
#define I4L_RUN(WAVES, C) I4L_LANES(WAVES, C, 64)
    // Rows of a head's size: several to a wave, with lanes for the padding of 8-bit codes (that of MXFP4 reaches 512 columns).
    if constexpr (RESULT == kRowTyped) {
        if (p.n <= 64)
            return I4L_LANES(1, 1, 8);
    }
    if constexpr (RESULT != kRowMx) {
        if (p.n <= 128)
            return I4L_LANES(1, 1, 16);
        if (p.n <= 256)
            return I4L_LANES(1, 1, 32);
    }
    if (p.n <= 512)
        return I4L_RUN(1, 1);
    if (p.n <= 1024)
        return I4L_RUN(1, 2);
    const bool few = p.rows < kFewRows;
    // (floats take twice the registers on their way: no more than two eights of them to a lane)
    if constexpr (TYPE != kOutF32) {
        if (!few && p.n <= 2048)
            return I4L_RUN(1, 4);
        if (!few && p.n > 4096 && p.n <= 8192)
            return I4L_RUN(4, 4);
        if (!few && p.n > 8192 && p.n <= 16384)
            return I4L_RUN(8, 4);
    }
    if (p.n <= 2048)
        return I4L_RUN(4, 1);
    if (p.n <= 4096)
        return few ? I4L_RUN(8, 1) : I4L_RUN(4, 2);
    if (p.n <= 8192)
        return I4L_RUN(8, 2);
    if (p.n <= 16384)
        return I4L_RUN(16, 2);
#undef I4L_RUN
#undef I4L_LANES
    row_loop_kernel<TYPE, RESULT, NORM><<<min(p.rows, 1 << 20), kThreads, 0, stream>>>(p, codes, scales);
    return hipGetLastError();
}

template <int TYPE>
hipError_t by_result(const RowPass &p, const DeviceInfo &dev, hipStream_t stream)
{
    if (!p.norm)
        return launch<TYPE, kRowInt8, false>(p, dev, stream);
    if (p.result == kRowTyped)
        return launch<TYPE, kRowTyped, true>(p, dev, stream);
    return p.result == kRowInt8 ? launch<TYPE, kRowInt8, true>(p, dev, stream) : launch<TYPE, kRowMx, true>(p, dev, stream);
}

// A thread takes eight values at a time.
template <int TYPE>
__global__ __launch_bounds__(kThreads) void int8_dequantize_kernel(Int8Matrix q, Element<TYPE> *y, size_t ld, int k, size_t chunks)
{
    const size_t stride = int8_code_stride(k), all = (size_t)q.rows * chunks;
    for (size_t at = (size_t)blockIdx.x * kThreads + threadIdx.x; at < all; at += (size_t)gridDim.x * kThreads) {
        const size_t row = at / chunks;
        const int c0 = (int)(at % chunks) * 8;
        const row_v2i codes = *(const row_v2i *)(q.codes + row * stride + c0);
        const float s = q.scales[row];
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            v[e] = (float)(int8_t)(codes[e / 4] >> 8 * (e % 4)) * s;
            asm("" : "+v"(v[e]));  // (a value is a float; in sight, the product would be rounded to float16 without that step)
        }
        store8(y + row * ld, c0, k, v);
    }
}

template <int TYPE>
hipError_t dequantize(const Int8Matrix &q, void *y, size_t ld, int k, hipStream_t stream)
{
    const size_t chunks = ((size_t)k + 7) / 8, groups = ((size_t)q.rows * chunks + kThreads - 1) / kThreads;
    int8_dequantize_kernel<TYPE><<<(unsigned)min(groups, (size_t)1 << 20), kThreads, 0, stream>>>(q, (Element<TYPE> *)y, ld, k, chunks);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_rows(const RowPass &p, const DeviceInfo &dev, hipStream_t stream)
{
    return p.type == kOutF32   ? by_result<kOutF32>(p, dev, stream)
           : p.type == kOutF16 ? by_result<kOutF16>(p, dev, stream)
                               : by_result<kOutBF16>(p, dev, stream);
}

hipError_t launch_int8_dequantize(const Int8Matrix &q, void *y, int type, size_t ld, int k, hipStream_t stream)
{
    return type == kOutF32   ? dequantize<kOutF32>(q, y, ld, k, stream)
           : type == kOutF16 ? dequantize<kOutF16>(q, y, ld, k, stream)
                             : dequantize<kOutBF16>(q, y, ld, k, stream);
}

}  // namespace int4linear
