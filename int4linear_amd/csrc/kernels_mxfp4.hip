// Conversions to and from MXFP4 (mxfp4.h has the format), and the transposes that the gradients need.
//
// Quantisation of a block x[0..31]:
//   e = max(-127, floor(log2(max |x|)) - 2),  scale code e + 127,
//   value = x * 2^-e rounded to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 (ties to the even code,
//   beyond 6 to 6), sign kept.
// x * 2^-e is exact (a power of two; what falls below the smallest float is far below 0.25 and
// rounds to 0 in any case) and the rounding is the hardware's v_cvt_scalef32_pk_fp4_f32 with a scale of
// 1, so the result follows from the formula bit by bit.  floor(log2) is the exponent field: a
// denormal maximum has the field 0 and meets the lower bound.  A block that holds an infinity or a NaN gets
// the scale code 255 and stands for 32 NaNs.
#include "mxfp4.h"
#include "mxfp4_epilogue.h"

namespace int4linear {

namespace {

typedef int v2i __attribute__((ext_vector_type(2)));
typedef int v4i __attribute__((ext_vector_type(4)));
typedef unsigned short v8us __attribute__((ext_vector_type(8)));

constexpr int kThreads = 256;
constexpr int kSegment = 512;  // k that one wave converts at a time: 8 per lane
constexpr int kUnroll = 4;     // segments per wave: their loads are in flight together

template <int TYPE>
struct Element;
template <>
struct Element<kOutF32> {
    using T = float;
    static __device__ float widen(T v) { return v; }
    static __device__ T narrow(float v) { return v; }
};
template <>
struct Element<kOutF16> {
    using T = _Float16;
    static __device__ float widen(T v) { return (float)v; }
    static __device__ T narrow(float v) { return (T)v; }
};
template <>
struct Element<kOutBF16> {
    using T = __bf16;
    static __device__ float widen(T v) { return (float)v; }
    static __device__ T narrow(float v) { return (T)v; }
};

// 2^e for e in -127 .. 127.
__device__ __forceinline__ float power_of_two(int e)
{
    return e < -126 ? __builtin_bit_cast(float, 0x00400000) : __builtin_bit_cast(float, (e + 127) << 23);
}

// The largest bit pattern (magnitudes as integers order like the values, NaN above infinity) over the
// four lanes of a quad.
__device__ __forceinline__ unsigned quad_max(unsigned v)
{
    v = max(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, true));  // lanes 1 0 3 2
    v = max(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, true));  // lanes 2 3 0 1
    return v;
}

// A lane converts 8 values, a quad of lanes a block, a wave kUnroll segments of 512 k (wave w those
// numbered w, w + waves, ...).  VEC: every group of 8 values is 16-byte aligned (32 for floats).
// Bound by HBM: 2.53 bytes per bfloat16 value.
template <int TYPE, bool VEC>
__global__ __launch_bounds__(kThreads) void mx_quantize_kernel(const typename Element<TYPE>::T *__restrict__ x, size_t ld,
                                                               uint8_t *__restrict__ codes, uint8_t *__restrict__ scales,
                                                               int rows, int k, int segments, size_t code_stride,
                                                               size_t scale_stride)
{
    using E = Element<TYPE>;
    using T = typename E::T;
    typedef T v8t __attribute__((ext_vector_type(8)));
    const int lane = threadIdx.x & 63;
    const long items = (long)rows * segments;
    const long waves = (long)gridDim.x * (kThreads / 64);
    const long first = (long)blockIdx.x * (kThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    v8t in[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const long item = first + u * waves;
        const int row = (int)(item / segments), c0 = (int)(item % segments) * kSegment + lane * 8;
        in[u] = (v8t)(T)0.0f;
        if (item < items && c0 < k) {
            const T *src = x + (size_t)row * ld + c0;
            if (VEC && c0 + 8 <= k) {
                in[u] = *(const v8t *)src;
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (c0 + i < k)
                        in[u][i] = src[i];
            }
        }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const long item = first + u * waves;
        if (item >= items)
            break;
        const int row = (int)(item / segments), c0 = (int)(item % segments) * kSegment + lane * 8;
        float v[8];
        unsigned big = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            v[i] = E::widen(in[u][i]);
            big = max(big, __builtin_bit_cast(unsigned, v[i]) & 0x7FFFFFFFu);
        }
        big = quad_max(big);
        unsigned code;
        const unsigned bits = encode_block_part(v, big, code);
        if ((size_t)c0 < code_stride * 2)
            *(unsigned *)(codes + (size_t)row * code_stride + c0 / 2) = bits;
        if ((lane & 3) == 0)
            scales[(size_t)row * scale_stride + c0 / kMxBlock] = (uint8_t)code;
    }
}

// A lane's 8 values from 4 bytes of codes and their block's scale.
__device__ __forceinline__ void decode8(unsigned c, unsigned scale, float (&v)[8])
{
    const float s = scale == 255 ? __builtin_nanf("") : power_of_two((int)scale - 127);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const unsigned n = c >> (4 * i);
        // E2M1's magnitude bits on top of a float's: exponent field 126 + e, or the subnormal 0.5.
        const unsigned mag = n & 7u;
        const float a = mag < 2 ? 0.5f * (float)mag : __builtin_bit_cast(float, (mag << 22) + 0x3F000000u);
        v[i] = ((n & 8u) ? -a : a) * s;
    }
}

template <int TYPE, bool VEC>
__global__ __launch_bounds__(kThreads) void mx_dequantize_kernel(const uint8_t *__restrict__ codes,
                                                                 const uint8_t *__restrict__ scales,
                                                                 typename Element<TYPE>::T *__restrict__ y, size_t ld, int rows,
                                                                 int k, int segments, size_t code_stride, size_t scale_stride)
{
    using E = Element<TYPE>;
    using T = typename E::T;
    typedef T v8t __attribute__((ext_vector_type(8)));
    const int lane = threadIdx.x & 63;
    const long items = (long)rows * segments;
    const long waves = (long)gridDim.x * (kThreads / 64);
    const long first = (long)blockIdx.x * (kThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    unsigned c[kUnroll], s[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const long item = first + u * waves;
        const int row = (int)(item / segments), c0 = (int)(item % segments) * kSegment + lane * 8;
        c[u] = s[u] = 0;
        if (item < items && c0 < k) {
            c[u] = *(const unsigned *)(codes + (size_t)row * code_stride + c0 / 2);
            s[u] = scales[(size_t)row * scale_stride + c0 / kMxBlock];
        }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const long item = first + u * waves;
        const int row = (int)(item / segments), c0 = (int)(item % segments) * kSegment + lane * 8;
        if (item >= items || c0 >= k)
            continue;
        float v[8];
        decode8(c[u], s[u], v);
        T *dst = y + (size_t)row * ld + c0;
        v8t out;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            out[i] = E::narrow(v[i]);
        if (VEC && c0 + 8 <= k) {
            *(v8t *)dst = out;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (c0 + i < k)
                    dst[i] = out[i];
        }
    }
}

// 64 rows x 64 k of q -> 64 rows of dst, by way of LDS.  Values of E2M1 times a power of two down to
// 2^-126 are bfloat16 numbers; smaller ones are rounded.
constexpr int kTile = 64;
constexpr int kTileStride = kTile + 2;  // elements between rows in LDS: an odd number of words

__device__ __forceinline__ void transpose_matrix(uint16_t *tile, const Transposed &t, int k, size_t code_stride, size_t scale_stride)
{
    const int r0 = blockIdx.x * kTile, c0 = blockIdx.y * kTile;
    if (r0 >= t.q.rows || c0 >= k)
        return;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int i = threadIdx.x + h * kThreads;
        const int r = i >> 3, c = (i & 7) * 8;
        float v[8] = {};
        if (r0 + r < t.q.rows)
            decode8(*(const unsigned *)(t.q.codes + (size_t)(r0 + r) * code_stride + (c0 + c) / 2),
                    t.q.scales[(size_t)(r0 + r) * scale_stride + (c0 + c) / kMxBlock], v);
#pragma unroll
        for (int e = 0; e < 8; ++e)
            tile[(c + e) * kTileStride + r] = __builtin_bit_cast(uint16_t, (__bf16)v[e]);
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int i = threadIdx.x + h * kThreads;
        const int c = i >> 3, r = (i & 7) * 8;
        if (c0 + c >= k)
            continue;
        v8us out;
#pragma unroll
        for (int e = 0; e < 8; ++e)
            out[e] = tile[c * kTileStride + r + e];
        *(v8us *)(t.dst + (size_t)(c0 + c) * t.ld + r0 + r) = out;
    }
}

__device__ __forceinline__ void transpose_dy(uint16_t *tile, const Prepared &p)
{
    const int r0 = blockIdx.x * kTile, c0 = blockIdx.y * kTile;
    if (r0 >= p.rows || c0 >= p.cols)
        return;
#pragma unroll
    for (int h = 0; h < kTile * kTile / kThreads; ++h) {
        const int i = threadIdx.x + h * kThreads;
        const int r = i >> 6, c = i & 63;
        const uint16_t v = r0 + r < p.rows && c0 + c < p.cols ? p.dy[(size_t)(r0 + r) * p.cols + c0 + c] : (uint16_t)0;
        tile[c * kTileStride + r] = v;
        if (p.padded && r0 + r < p.rows && (size_t)(c0 + c) < p.ld_p)
            p.padded[(size_t)(r0 + r) * p.ld_p + c0 + c] = v;
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int i = threadIdx.x + h * kThreads;
        const int c = i >> 3, r = (i & 7) * 8;
        v8us out;
        float sum = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            out[e] = tile[c * kTileStride + r + e];
            sum += __builtin_bit_cast(float, (unsigned)out[e] << 16);
        }
        if (p.transposed && c0 + c < p.cols)
            *(v8us *)(p.transposed + (size_t)(c0 + c) * p.ld_t + r0 + r) = out;
        if (p.partial) {
#pragma unroll
            for (int s = 1; s < 8; s *= 2)
                sum += __shfl_xor(sum, s);
            if ((i & 7) == 0 && c0 + c < p.cols)
                p.partial[(size_t)blockIdx.x * p.cols + c0 + c] = sum;
        }
    }
}

// blockIdx.z: one of the matrices, or dy behind them.
__global__ __launch_bounds__(kThreads) void prepare_kernel(Prepared p, size_t code_stride, size_t scale_stride)
{
    __shared__ uint16_t tile[kTile * kTileStride];
    if (blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0)
        for (int i = threadIdx.x; i < p.zero_count; i += kThreads)
            p.zeros[i] = 0;
    if ((int)blockIdx.z < p.matrices)
        transpose_matrix(tile, p.matrix[blockIdx.z], p.k, code_stride, scale_stride);
    else
        transpose_dy(tile, p);
}

// 64 columns per workgroup; the waves take every fourth row each, and their sums are added in order.
__global__ __launch_bounds__(kThreads) void column_sums_kernel(ColumnSums s)
{
    __shared__ float part[kThreads];
    const int c = blockIdx.x * 64 + (threadIdx.x & 63);
    float sum = 0.0f;
    if (c < s.columns) {
#pragma unroll 8
        for (int i = threadIdx.x >> 6; i < s.parts; i += kThreads / 64)
            sum += s.partial[(size_t)i * s.columns + c];
    }
    part[threadIdx.x] = sum;
    __syncthreads();
    if (threadIdx.x < 64 && c < s.columns)
        s.sums[c] = ((part[threadIdx.x] + part[threadIdx.x + 64]) + part[threadIdx.x + 128]) + part[threadIdx.x + 192];
}

int conversion_grid(int rows, int segments)
{
    const size_t items = (size_t)rows * segments;
    const size_t per_group = (size_t)kUnroll * (kThreads / 64);
    return (int)((items + per_group - 1) / per_group);
}

template <int TYPE>
hipError_t quantize(const void *x, size_t ld, uint8_t *codes, uint8_t *scales, int rows, int k, hipStream_t stream)
{
    using T = typename Element<TYPE>::T;
    const int segments = (k + kSegment - 1) / kSegment;
    const bool vec = ((uintptr_t)x % (8 * sizeof(T))) == 0 && ld % 8 == 0;
    auto kernel = vec ? mx_quantize_kernel<TYPE, true> : mx_quantize_kernel<TYPE, false>;
    kernel<<<conversion_grid(rows, segments), kThreads, 0, stream>>>((const T *)x, ld, codes, scales, rows, k, segments,
                                                                    mx_code_stride(k), mx_scale_stride(k));
    return hipGetLastError();
}

template <int TYPE>
hipError_t dequantize(const MxMatrix &q, void *y, size_t ld, int k, hipStream_t stream)
{
    using T = typename Element<TYPE>::T;
    const int segments = (k + kSegment - 1) / kSegment;
    const bool vec = ((uintptr_t)y % (8 * sizeof(T))) == 0 && ld % 8 == 0;
    auto kernel = vec ? mx_dequantize_kernel<TYPE, true> : mx_dequantize_kernel<TYPE, false>;
    kernel<<<conversion_grid(q.rows, segments), kThreads, 0, stream>>>(q.codes, q.scales, (T *)y, ld, q.rows, k, segments,
                                                                      mx_code_stride(k), mx_scale_stride(k));
    return hipGetLastError();
}

}  // namespace

hipError_t launch_mx_quantize(const void *x, int type, size_t ld, uint8_t *codes, uint8_t *scales, int rows, int k,
                              hipStream_t stream)
{
    switch (type) {
    case kOutF32:
        return quantize<kOutF32>(x, ld, codes, scales, rows, k, stream);
    case kOutF16:
        return quantize<kOutF16>(x, ld, codes, scales, rows, k, stream);
    default:
        return quantize<kOutBF16>(x, ld, codes, scales, rows, k, stream);
    }
}

hipError_t launch_mx_dequantize(const MxMatrix &q, void *y, int type, size_t ld, int k, hipStream_t stream)
{
    switch (type) {
    case kOutF32:
        return dequantize<kOutF32>(q, y, ld, k, stream);
    case kOutF16:
        return dequantize<kOutF16>(q, y, ld, k, stream);
    default:
        return dequantize<kOutBF16>(q, y, ld, k, stream);
    }
}

hipError_t launch_prepare(const Prepared &p, hipStream_t stream)
{
    int rows = p.dy ? p.rows : 0, cols = p.dy ? p.cols : 0;
    for (int i = 0; i < p.matrices; ++i) {
        rows = max(rows, p.matrix[i].q.rows);
        cols = max(cols, p.k);
    }
    if (rows == 0 || cols == 0)
        return hipSuccess;
    const dim3 grid((unsigned)((rows + kTile - 1) / kTile), (unsigned)((cols + kTile - 1) / kTile), (unsigned)(p.matrices + (p.dy != nullptr)));
    prepare_kernel<<<grid, kThreads, 0, stream>>>(p, mx_code_stride(p.k), mx_scale_stride(p.k));
    return hipGetLastError();
}

hipError_t launch_column_sums(const ColumnSums &s, hipStream_t stream)
{
    column_sums_kernel<<<(s.columns + 63) / 64, kThreads, 0, stream>>>(s);
    return hipGetLastError();
}

}  // namespace int4linear
