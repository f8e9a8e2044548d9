// Passes over rows: the norm y = (x - mean) / sqrt(variance + eps) * gamma + beta, and quantisation to 8 bits by row, alone or
// of what the norm gives.
#include "row_math.h"

#include <type_traits>

namespace int4linear {

namespace {

constexpr int kThreads = 256;

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

// (x - mean) r gamma + beta of eight columns; what is behind the row's end stays 0.
__device__ __forceinline__ void normalise8(const RowPass &p, const RowStatistics &s, int c0, float (&v)[8])
{
    float g[8], b[8];
    if (p.gamma)
        load8(p.gamma, c0, p.n, g);
    if (p.beta)
        load8(p.beta, c0, p.n, b);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        float y = s.normalised(v[e]);
        if (p.gamma)
            y *= g[e];
        if (p.beta)
            y += b[e];
        v[e] = c0 + e < p.n ? y : 0.0f;
    }
}

// A workgroup takes a row at a time and reads it again in every pass, from the caches.
template <int TYPE, int RESULT, bool NORM>
__global__ __launch_bounds__(kThreads) void row_loop_kernel(RowPass p, size_t code_stride, size_t scale_stride)
{
    constexpr int kWaves = kThreads / 64;
    __shared__ float room[3][2 * kWaves];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const RowWriter<RESULT> writer{p, code_stride, scale_stride};
    for (int row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const Element<TYPE> *x = (const Element<TYPE> *)p.x + (size_t)row * p.ld;
        RowStatistics s{};
        float v[8];
        if constexpr (NORM) {
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
            s = RowStatistics::from(shift, two[0], two[1], p.n, p.eps);
        }
        RowScale scale{};
        if constexpr (RESULT == kRowInt8) {
            unsigned big[1] = {};
            for (int c0 = threadIdx.x * 8; c0 < p.n; c0 += kThreads * 8) {
                load8(x, c0, p.n, v);
                if constexpr (NORM)
                    normalise8(p, s, c0, v);
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    big[0] = max(big[0], __builtin_bit_cast(unsigned, v[e]) & 0x7FFFFFFFu);
            }
            group_all<Larger>(big, (unsigned *)room[2], wave, kWaves);
            scale = RowScale::of(big[0]);
        }
        // (whole quads of lanes, for MXFP4's blocks)
        for (int c0 = threadIdx.x * 8; c0 < writer.columns(p.n); c0 += kThreads * 8) {
            load8(x, c0, p.n, v);
            if constexpr (NORM)
                normalise8(p, s, c0, v);
            writer.write(row, c0, v, scale);
        }
        if constexpr (!NORM)
            __syncthreads();  // (else the room of one row is used again behind two further meetings)
    }
}

template <int TYPE, int RESULT, bool NORM>
hipError_t launch(const RowPass &p, hipStream_t stream)
{
    const size_t codes = RESULT == kRowInt8 ? int8_code_stride(p.n) : mx_code_stride(p.n);
    row_loop_kernel<TYPE, RESULT, NORM><<<min(p.rows, 1 << 20), kThreads, 0, stream>>>(p, codes, mx_scale_stride(p.n));
    return hipGetLastError();
}

template <int TYPE>
hipError_t by_result(const RowPass &p, hipStream_t stream)
{
    if (!p.norm)
        return launch<TYPE, kRowInt8, false>(p, stream);
    if (p.result == kRowTyped)
        return launch<TYPE, kRowTyped, true>(p, stream);
    return p.result == kRowInt8 ? launch<TYPE, kRowInt8, true>(p, stream) : launch<TYPE, kRowMx, true>(p, stream);
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
        for (int e = 0; e < 8; ++e)
            v[e] = (float)(int8_t)(codes[e / 4] >> 8 * (e % 4)) * s;
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

hipError_t launch_rows(const RowPass &p, hipStream_t stream)
{
    return p.type == kOutF32   ? by_result<kOutF32>(p, stream)
           : p.type == kOutF16 ? by_result<kOutF16>(p, stream)
                               : by_result<kOutBF16>(p, stream);
}

hipError_t launch_int8_dequantize(const Int8Matrix &q, void *y, int type, size_t ld, int k, hipStream_t stream)
{
    return type == kOutF32   ? dequantize<kOutF32>(q, y, ld, k, stream)
           : type == kOutF16 ? dequantize<kOutF16>(q, y, ld, k, stream)
                             : dequantize<kOutBF16>(q, y, ld, k, stream);
}

}  // namespace int4linear
