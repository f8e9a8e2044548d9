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

#include <type_traits>

namespace int4linear {

namespace {

typedef unsigned v4u __attribute__((ext_vector_type(4)));

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
// numbered w, w + waves, ...).  Groups of 8 values are loaded and stored 16 bytes at a time, aligned to their element only: the
// hardware splits those that are not aligned to more.  Bound by HBM: 2.53 bytes per bfloat16 value.  (8192 rows of bfloat16, k =
// 5000: 17 us and 23 back, 6.0 and 4.5 TB/s; 5001: 20 and 24, one element at a time 48 and 58.)
template <int TYPE>
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
    const long waves = (long)gridDim.x * gridDim.y * (kThreads / 64);
    const long first = ((long)blockIdx.y * gridDim.x + blockIdx.x) * (kThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    v8t in[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const long item = first + u * waves;
        const int row = (int)(item / segments), c0 = (int)(item % segments) * kSegment + lane * 8;
        in[u] = (v8t)(T)0.0f;
        if (item < items && c0 < k) {
            const T *src = x + (size_t)row * ld + c0;
            if (c0 + 8 <= k) {
                __builtin_memcpy(&in[u], src, sizeof(v8t));
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

template <int TYPE>
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
    const long waves = (long)gridDim.x * gridDim.y * (kThreads / 64);
    const long first = ((long)blockIdx.y * gridDim.x + blockIdx.x) * (kThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
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
        if (c0 + 8 <= k) {
            __builtin_memcpy(dst, &out, sizeof(v8t));
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (c0 + i < k)
                    dst[i] = out[i];
        }
    }
}

// Transposes for the gradients.  A lane takes 8 x 8 values, 16-bit, whose rows are four registers each: a byte permutation of
// two rows' registers gives two values of one column, so 32 permutations turn the square and neither LDS nor other lanes
// take part (through LDS: 124 us for 91).  A wave takes 64 rows x 64 columns, eight lanes down and eight across: it stores whole 128-byte lines.  Values of
// E2M1 times a power of two from 2^-127 are bfloat16 numbers.
constexpr int kTile = 64;
constexpr int kTilesAcross = 4;  // a workgroup's: a whole line of codes

// The values at (row 8i + r, column 8j + c) of a wave's tile, i = lane % 8, j = lane / 8: rows[r] -> dst, from the tile's
// first column on.
__device__ __forceinline__ void store_transposed(const v4u (&rows)[8], uint16_t *dst, size_t ld, int columns)
{
    const int lane = threadIdx.x & 63, c0 = (lane >> 3) * 8;
#pragma unroll
    for (int c = 0; c < 8; ++c) {
        v4u out;
#pragma unroll
        for (int w = 0; w < 4; ++w)
            out[w] = __builtin_amdgcn_perm(rows[2 * w + 1][c / 2], rows[2 * w][c / 2], c & 1 ? 0x07060302u : 0x05040100u);
        if (c0 + c < columns)
            *(v4u *)(dst + (size_t)(c0 + c) * ld + (lane & 7) * 8) = out;
    }
}

template <int DOWN>
__device__ __forceinline__ void transpose_matrix(const Transposed &t, int k, size_t code_stride, size_t scale_stride)
{
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r0 = (blockIdx.x * DOWN + wave / kTilesAcross) * kTile, c0 = (blockIdx.y * kTilesAcross + wave % kTilesAcross) * kTile;
    if (r0 >= t.q.rows || c0 >= k)
        return;
    const int row = r0 + (lane & 7) * 8, col = c0 + (lane >> 3) * 8;
    unsigned codes[8], scales[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) {
        codes[r] = scales[r] = 0;
        if (row + r < t.q.rows) {
            codes[r] = *(const unsigned *)(t.q.codes + (size_t)(row + r) * code_stride + col / 2);
            scales[r] = t.q.scales[(size_t)(row + r) * scale_stride + col / kMxBlock];
        }
    }
    v4u rows[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) {
        const float scale = __builtin_bit_cast(float, scales[r] << 23);
        rows[r] = (v4u){__builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes[r], scale, 0)),
                        __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes[r], scale, 1)),
                        __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes[r], scale, 2)),
                        __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes[r], scale, 3))};
        if (scales[r] == 255)
            rows[r] = (v4u)0x7FC07FC0u;
    }
    store_transposed(rows, t.dst + (size_t)c0 * t.ld + r0, t.ld, k - c0);
}

template <int DPP>
__device__ __forceinline__ float lanes(float v)
{
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), DPP, 0xF, 0xF, true));
}

template <int DOWN>
__device__ __forceinline__ void transpose_dy(const Prepared &p)
{
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r0 = (blockIdx.x * DOWN + wave / kTilesAcross) * kTile, c0 = (blockIdx.y * kTilesAcross + wave % kTilesAcross) * kTile;
    if (r0 >= p.rows || c0 >= p.cols)
        return;
    const int row = r0 + (lane & 7) * 8, col = c0 + (lane >> 3) * 8;
    v4u rows[8];
    if (p.cols >= 8) {
        // Eight elements at once, aligned to the element only (the hardware splits such loads); at a row's end the row's last
        // eight, shifted to their places.
        const int over = max(col + 8 - p.cols, 0);
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            rows[r] = (v4u)0u;
            if (row + r < p.rows)
                __builtin_memcpy(&rows[r], p.dy + (size_t)(row + r) * p.cols + (col - over), 16);
        }
        if (over) {
#pragma unroll
            for (int r = 0; r < 8; ++r)
                rows[r] = over < 8 ? __builtin_bit_cast(v4u, __builtin_bit_cast(unsigned __int128, rows[r]) >> (16 * over)) : (v4u)0u;
        }
    } else {
        unsigned __int128 v[8] = {};
#pragma unroll 1
        for (int c = p.cols - 1; c >= 0 && col == 0; --c)
#pragma unroll
            for (int r = 0; r < 8; ++r)
                v[r] = v[r] << 16 | (row + r < p.rows ? p.dy[(size_t)(row + r) * p.cols + c] : (uint16_t)0);
#pragma unroll
        for (int r = 0; r < 8; ++r)
            rows[r] = __builtin_bit_cast(v4u, v[r]);
    }
    if (p.padded && (size_t)col < p.ld_p) {
#pragma unroll
        for (int r = 0; r < 8; ++r)
            if (row + r < p.rows)
                *(v4u *)(p.padded + (size_t)(row + r) * p.ld_p + col) = rows[r];
    }
    if (p.transposed)
        store_transposed(rows, p.transposed + (size_t)c0 * p.ld_t + r0, p.ld_t, p.cols - c0);
    if (p.partial) {
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            float sum = 0.0f;
#pragma unroll
            for (int r = 0; r < 8; ++r)
                sum += __builtin_bit_cast(float, c & 1 ? rows[r][c / 2] & 0xFFFF0000u : rows[r][c / 2] << 16);
            sum += lanes<0xB1>(sum);   // 1 0 3 2
            sum += lanes<0x4E>(sum);   // 2 3 0 1
            sum += lanes<0x141>(sum);  // 7 .. 0: the other quad's
            if ((lane & 7) == 0 && col + c < p.cols)
                p.partial[(size_t)(r0 / kTile) * p.cols + col + c] = sum;
        }
    }
}

// blockIdx.z: one of the matrices, or dy behind them.  A workgroup takes DOWN x kTilesAcross tiles.
template <int DOWN>
__global__ __launch_bounds__(DOWN *kTilesAcross * 64) void prepare_kernel(Prepared p, size_t code_stride, size_t scale_stride)
{
    if (blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0)
        for (int i = threadIdx.x; i < p.zero_count; i += DOWN * kTilesAcross * 64)
            p.zeros[i] = 0;
    if ((int)blockIdx.z < p.matrices)
        transpose_matrix<DOWN>(p.matrix[blockIdx.z], p.k, code_stride, scale_stride);
    else
        transpose_dy<DOWN>(p);
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

// (A launch holds fewer than 2^32 threads along x.)
dim3 conversion_grid(int rows, int segments)
{
    constexpr size_t kMostAlongX = 1 << 22;
    const size_t items = (size_t)rows * segments;
    const size_t per_group = (size_t)kUnroll * (kThreads / 64), groups = (items + per_group - 1) / per_group;
    return dim3((unsigned)min(groups, kMostAlongX), (unsigned)((groups + kMostAlongX - 1) / kMostAlongX));
}

template <int TYPE>
hipError_t quantize(const void *x, size_t ld, uint8_t *codes, uint8_t *scales, int rows, int k, hipStream_t stream)
{
    using T = typename Element<TYPE>::T;
    const int segments = (k + kSegment - 1) / kSegment;
    mx_quantize_kernel<TYPE><<<conversion_grid(rows, segments), kThreads, 0, stream>>>((const T *)x, ld, codes, scales, rows, k, segments,
                                                                    mx_code_stride(k), mx_scale_stride(k));
    return hipGetLastError();
}

template <int TYPE>
hipError_t dequantize(const MxMatrix &q, void *y, size_t ld, int k, hipStream_t stream)
{
    using T = typename Element<TYPE>::T;
    const int segments = (k + kSegment - 1) / kSegment;
    mx_dequantize_kernel<TYPE><<<conversion_grid(q.rows, segments), kThreads, 0, stream>>>(q.codes, q.scales, (T *)y, ld, q.rows, k, segments,
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

// From a tile of 256 x 256 for each CU on, workgroups of 16 waves, whose tiles' rows are written 512 bytes at a time; below, of 4,
// which come to more CUs.  (us, 4 waves or 16: x, w and dy of 4096 x 4096 x 14336 106, 91; two weights of 14336 x 4096 and x 106, 102-108;
// 257 x 1400 x 1000 6.2, 9.2; 130 x 1001 x 515 6.7, 9.)
constexpr long kLargeTranspose = 256l * 256 * 256;

hipError_t launch_prepare(const Prepared &p, hipStream_t stream)
{
    int rows = p.dy ? p.rows : 0, cols = p.dy ? p.cols : 0;
    for (int i = 0; i < p.matrices; ++i) {
        rows = max(rows, p.matrix[i].q.rows);
        cols = max(cols, p.k);
    }
    if (rows == 0 || cols == 0)
        return hipSuccess;
    auto run = [&](auto down) {
        constexpr int DOWN = decltype(down)::value, kSide = DOWN * kTile, kWide = kTilesAcross * kTile;
        const dim3 grid((unsigned)((rows + kSide - 1) / kSide), (unsigned)((cols + kWide - 1) / kWide), (unsigned)(p.matrices + (p.dy != nullptr)));
        prepare_kernel<DOWN><<<grid, DOWN * kTilesAcross * 64, 0, stream>>>(p, mx_code_stride(p.k), mx_scale_stride(p.k));
    };
    if ((long)rows * cols >= kLargeTranspose)
        run(std::integral_constant<int, 4>{});
    else
        run(std::integral_constant<int, 1>{});
    return hipGetLastError();
}

hipError_t launch_column_sums(const ColumnSums &s, hipStream_t stream)
{
    column_sums_kernel<<<(s.columns + 63) / 64, kThreads, 0, stream>>>(s);
    return hipGetLastError();
}

}  // namespace int4linear
