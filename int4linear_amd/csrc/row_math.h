// What the row passes share: eight values of a row at a time, sums over a row's lanes, and the 8-bit format's rounding.
#pragma once
#include "int8.h"
#include "mxfp4_epilogue.h"

namespace int4linear {

typedef int row_v2i __attribute__((ext_vector_type(2)));

// Values c0 .. c0 + 7 of a row of n as floats, zeros behind its end.  (16 bytes of 16-bit types at once, aligned to the element
// only: the hardware splits those that are not aligned to more.)
template <class T>
__device__ __forceinline__ void load8(const T *row, int c0, int n, float (&v)[8])
{
    typedef T v8t __attribute__((ext_vector_type(8)));
    v8t in = (v8t)(T)0.0f;
    if (c0 + 8 <= n) {
        __builtin_memcpy(&in, row + c0, sizeof(v8t));
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (c0 + e < n)
                in[e] = row[c0 + e];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
        v[e] = (float)in[e];
}

// The other way, rounded to T.
template <class T>
__device__ __forceinline__ void store8(T *row, int c0, int n, const float (&v)[8])
{
    typedef T v8t __attribute__((ext_vector_type(8)));
    v8t out;
#pragma unroll
    for (int e = 0; e < 8; ++e)
        out[e] = (T)v[e];
    if (c0 + 8 <= n) {
        __builtin_memcpy(row + c0, &out, sizeof(v8t));
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (c0 + e < n)
                row[c0 + e] = out[e];
    }
}

__device__ __forceinline__ void store8_as(int out, void *row, int c0, int n, const float (&v)[8])
{
    if (out == kOutF32)
        store8((float *)row, c0, n, v);
    else if (out == kOutF16)
        store8((_Float16 *)row, c0, n, v);
    else
        store8((__bf16 *)row, c0, n, v);
}

// Every lane's value combined with all others of the wave, the same bits in all of them: neighbours, pairs, quads and eights by
// lane permutations, rows of 16 and halves of the wave by swaps.
template <class T, class Op>
__device__ __forceinline__ T wave_all(T v, Op op)
{
    auto permuted = [](T x, auto ctrl) {
        return __builtin_bit_cast(T, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), decltype(ctrl)::value, 0xF, 0xF, true));
    };
    v = op(v, permuted(v, std::integral_constant<int, 0xB1>{}));   // lanes 1 0 3 2
    v = op(v, permuted(v, std::integral_constant<int, 0x4E>{}));   // lanes 2 3 0 1
    v = op(v, permuted(v, std::integral_constant<int, 0x141>{}));  // 7 .. 0
    v = op(v, permuted(v, std::integral_constant<int, 0x140>{}));  // 15 .. 0
    const unsigned a = __builtin_bit_cast(unsigned, v);
    const auto rows = __builtin_amdgcn_permlane16_swap(a, a, false, false);
    v = op(__builtin_bit_cast(T, (unsigned)rows[0]), __builtin_bit_cast(T, (unsigned)rows[1]));
    const unsigned b = __builtin_bit_cast(unsigned, v);
    const auto halves = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    return op(__builtin_bit_cast(T, (unsigned)halves[0]), __builtin_bit_cast(T, (unsigned)halves[1]));
}

struct Add {
    __device__ float operator()(float a, float b) const { return a + b; }
};
struct Larger {
    __device__ unsigned operator()(unsigned a, unsigned b) const { return max(a, b); }
};

// N values of every thread combined over the `waves` waves of a group, which all meet here.  `room` (N * waves words of LDS) may be
// used again once the group has met for another time.
template <class Op, class T, int N>
__device__ __forceinline__ void group_all(T (&v)[N], T *room, int wave, int waves)
{
#pragma unroll
    for (int i = 0; i < N; ++i)
        v[i] = wave_all(v[i], Op{});
    if (waves == 1)
        return;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            room[wave * N + i] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        T all = room[i];
        for (int w = 1; w < waves; ++w)
            all = Op{}(all, room[w * N + i]);
        v[i] = all;
    }
}

// A row's mean is `shift` + `delta` with shift a first sum's (rounded) mean, so that what is squared and summed next is centred: the
// variance is the mean of (x - shift)^2 less delta^2, a correction of the first sum's rounding and no cancellation.
struct RowStatistics {
    float shift, delta, r;  // r = 1 / sqrt(variance + eps)
    __device__ static RowStatistics from(float shift, float sum, float squares, int n, float eps)
    {
        const float delta = sum / (float)n;
        const float variance = fmaxf(squares / (float)n - delta * delta, 0.0f);
        // (fmaxf takes a NaN away: rows with infinities or NaNs become NaN)
        return {shift, delta, 1.0f / sqrtf((squares == squares ? variance : squares) + eps)};
    }
    __device__ __forceinline__ float normalised(float x) const { return ((x - shift) - delta) * r; }
};

// The 8-bit format's scale of a row whose largest magnitude has the bits `big` (NaN above infinity above all numbers), and what
// its values are multiplied with.  A row with an infinity or a NaN has the scale NaN and codes of zero.
struct RowScale {
    float scale, inverse;
    __device__ static RowScale of(unsigned big)
    {
        if (big >= 0x7F800000u)
            return {__builtin_nanf(""), 0.0f};
        const float s = fmaxf(__builtin_bit_cast(float, big) / 127.0f, 0x1p-100f);
        return {s, 1.0f / s};
    }
};

// v / scale to the nearest whole number, ties to the even one, decided exactly: the product with the rounded inverse is within
// 1e-4 of the quotient, and what is left of v is exact in one fused operation.  Beyond half a scale the neighbour is nearer, at
// half a scale the even one is taken.
__device__ __forceinline__ void encode_int8(const float (&v)[8], const RowScale &s, row_v2i &codes)
{
    float q[8], left[8], most = 0.0f;
    const float half = 0.5f * s.scale;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        q[e] = rintf(v[e] * s.inverse);
        left[e] = fmaf(-q[e], s.scale, v[e]);
        most = fmaxf(most, fabsf(left[e]));
    }
    if (most >= half) {  // rare
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float a = fabsf(left[e]);
            const bool odd = ((int)q[e] & 1) != 0;
            if (a > half || (a == half && odd))
                q[e] += left[e] > 0.0f ? 1.0f : -1.0f;
        }
    }
    unsigned bytes[2] = {};
#pragma unroll
    for (int e = 0; e < 8; ++e)
        bytes[e / 4] |= ((unsigned)(int)q[e] & 0xFFu) << (8 * (e % 4));
    codes = s.scale == s.scale ? (row_v2i){(int)bytes[0], (int)bytes[1]} : (row_v2i)0;
}

}  // namespace int4linear
