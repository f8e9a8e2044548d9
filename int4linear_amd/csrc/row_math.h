// What the row passes share: eight values of a row at a time, sums over a row's lanes, and the 8-bit format's rounding.
#pragma once
#include "int8.h"
#include "mxfp4_epilogue.h"

namespace int4linear {

typedef int row_v2i __attribute__((ext_vector_type(2)));

// Eight values of a row of n for columns c0 .. c0 + 7, on their way to a lane: at the row's end the row's last eight, to be brought to
// their places when they are used (a load that has not been waited for cannot be).  16 bytes of 16-bit types at once, aligned to the
// element only: the hardware splits those that are not aligned to more.
template <class T>
using Eight = T __attribute__((ext_vector_type(8)));

template <class T>
__device__ __forceinline__ void fetch8(const T *row, int c0, int n, Eight<T> &in)
{
    in = (Eight<T>)(T)0.0f;
    if (n >= 8) {
        if (c0 < n)
            __builtin_memcpy(&in, row + min(c0, n - 8), sizeof(in));
    } else if (c0 == 0) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            in[e] = row[min(e, n - 1)];
    }
}

// As floats, zeros behind the row's end.
template <class T>
__device__ __forceinline__ void widen8(const Eight<T> &in, int c0, int n, float (&v)[8])
{
#pragma unroll
    for (int e = 0; e < 8; ++e)
        v[e] = (float)in[e];
    if (c0 + 8 > n) {
        const int over = n >= 8 ? c0 + 8 - n : 0;  // (behind the end: zeros in any order)
#pragma unroll
        for (int by = 4; by > 0; by /= 2)
#pragma unroll
            for (int e = 0; e < 8; ++e)
                v[e] = over & by ? (e + by < 8 ? v[e + by] : 0.0f) : v[e];
        if (n < 8) {
#pragma unroll
            for (int e = 1; e < 8; ++e)
                v[e] = e < n ? v[e] : 0.0f;
        }
    }
}

template <class T>
__device__ __forceinline__ void load8(const T *row, int c0, int n, float (&v)[8])
{
    Eight<T> in;
    fetch8(row, c0, n, in);
    widen8<T>(in, c0, n, v);
}

// What is behind the row's end set to `value`.
__device__ __forceinline__ void behind8(int c0, int n, float value, float (&v)[8])
{
    if (c0 + 8 > n) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            v[e] = c0 + e < n ? v[e] : value;
    }
}

// The other way, rounded to T; what is left at the row's end in four, two and one.
template <class T>
__device__ __forceinline__ void store8(T *row, int c0, int n, const float (&v)[8])
{
    typedef T Four __attribute__((ext_vector_type(4)));
    typedef T Two __attribute__((ext_vector_type(2)));
    Eight<T> out;
#pragma unroll
    for (int e = 0; e < 8; ++e)
        out[e] = (T)v[e];
    if (c0 + 8 <= n) {
        __builtin_memcpy(row + c0, &out, sizeof(out));
    } else if (c0 < n) {
        const int left = n - c0;
        T *to = row + c0;
        const Four four = {out[0], out[1], out[2], out[3]};
        const Two two = left & 4 ? (Two){out[4], out[5]} : (Two){out[0], out[1]};
        const T one = left & 4 ? (left & 2 ? out[6] : out[4]) : (left & 2 ? out[2] : out[0]);
        if (left & 4)
            __builtin_memcpy(to, &four, sizeof(four));
        if (left & 2)
            __builtin_memcpy(to + (left & 4), &two, sizeof(two));
        if (left & 1)
            to[left & 6] = one;
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

// Every lane's value combined with those of the others of its LANES lanes (8, 16, 32 or the whole wave), the same bits in all of
// them: neighbours, pairs, quads and eights by lane permutations, rows of 16 and halves of the wave by swaps.
template <int LANES = 64, class T, class Op>
__device__ __forceinline__ T wave_all(T v, Op op)
{
    auto permuted = [](T x, auto ctrl) {
        return __builtin_bit_cast(T, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), decltype(ctrl)::value, 0xF, 0xF, true));
    };
    v = op(v, permuted(v, std::integral_constant<int, 0xB1>{}));   // lanes 1 0 3 2
    v = op(v, permuted(v, std::integral_constant<int, 0x4E>{}));   // lanes 2 3 0 1
    v = op(v, permuted(v, std::integral_constant<int, 0x141>{}));  // 7 .. 0
    if constexpr (LANES >= 16)
        v = op(v, permuted(v, std::integral_constant<int, 0x140>{}));  // 15 .. 0
    if constexpr (LANES >= 32) {
        const unsigned a = __builtin_bit_cast(unsigned, v);
        const auto rows = __builtin_amdgcn_permlane16_swap(a, a, false, false);
        v = op(__builtin_bit_cast(T, (unsigned)rows[0]), __builtin_bit_cast(T, (unsigned)rows[1]));
    }
    if constexpr (LANES == 64) {
        const unsigned b = __builtin_bit_cast(unsigned, v);
        const auto halves = __builtin_amdgcn_permlane32_swap(b, b, false, false);
        v = op(__builtin_bit_cast(T, (unsigned)halves[0]), __builtin_bit_cast(T, (unsigned)halves[1]));
    }
    return v;
}

// What lanes LANES apart hold, combined over the wave: the rest of wave_all.
template <int LANES, class T, class Op>
__device__ __forceinline__ T across_all(T v, Op op)
{
    if constexpr (LANES == 8)
        v = op(v, __builtin_bit_cast(T, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x128, 0xF, 0xF, true)));  // a row turned by 8
    if constexpr (LANES <= 16) {
        const unsigned a = __builtin_bit_cast(unsigned, v);
        const auto rows = __builtin_amdgcn_permlane16_swap(a, a, false, false);
        v = op(__builtin_bit_cast(T, (unsigned)rows[0]), __builtin_bit_cast(T, (unsigned)rows[1]));
    }
    if constexpr (LANES <= 32) {
        const unsigned b = __builtin_bit_cast(unsigned, v);
        const auto halves = __builtin_amdgcn_permlane32_swap(b, b, false, false);
        v = op(__builtin_bit_cast(T, (unsigned)halves[0]), __builtin_bit_cast(T, (unsigned)halves[1]));
    }
    return v;
}

struct Add {
    __device__ float operator()(float a, float b) const { return a + b; }
};
struct Larger {
    __device__ unsigned operator()(unsigned a, unsigned b) const { return max(a, b); }
};

// N values of every thread combined over the `waves` waves of a group, which all meet here.  `room` (N * waves words of LDS) may be
// used again once the group has met for another time.  With one wave, over LANES of its lanes.
template <class Op, int LANES = 64, class T, int N>
__device__ __forceinline__ void group_all(T (&v)[N], T *room, int wave, int waves)
{
#pragma unroll
    for (int i = 0; i < N; ++i)
        v[i] = wave_all<LANES>(v[i], Op{});
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

// A row's sum as one of small parts of its values: that of as many as a row may have is a float, whatever finite floats they are, so that a
// row whose sum is none has an infinity or a NaN.  (A power of two: the same bits as a sum of the values themselves.)
constexpr float kPart = 0x1p-23f;
static_assert(kMostNorm <= 1 << 22);
__device__ __forceinline__ void add_part(float &sum, float v) { sum = fmaf(v, kPart, sum); }

// What all values of a row are centred on, from the sum of their parts.  It has to be one number: left in sight, the product would be merged
// with some of the differences that take it and not with others, and so be rounded for these alone.
__device__ __forceinline__ float row_shift(float sum, float over_n)
{
    float shift = sum * (over_n * (1.0f / kPart));
    asm("" : "+v"(shift));
    return shift;
}

// A row's mean is `shift` + delta with shift a first sum's (rounded) mean, so that what is squared and summed next is centred: the
// variance is the mean of (x - shift)^2 less delta^2, a correction of the first sum's rounding and no cancellation.
// h = (x - mean) / sqrt(variance + eps) is d r + c with d = x - shift, one rounding.  In a `flat` row h is 0, and d has to be: some of its d
// may be infinite.
struct RowStatistics {
    float shift, r, c;
    bool flat;
    __device__ static RowStatistics from(float shift, float sum, float squares, float over_n, float eps)
    {
        // Finite values that lie too far apart have an infinite sum of squares.  With an infinity or a NaN among them it is a NaN: shift is one
        // too, or the same infinity, and so is what is left of that value.
        const bool far = squares == __builtin_inff();
        const float delta = far ? 0.0f : sum * over_n, square = delta * delta;
        // Of a constant row whose mean is not met exactly every d is the same but 0, and the difference of the two squares is nothing but their
        // roundings.  Where it and eps are below 2^-22 of them it counts as nothing: r would make values of 1e10 and more out of what delta is
        // off.  (Floats that are not all the same deviate by more: by n^-1/2 of a unit in the mean's last place, of which delta is a few.)
        const float spread = fmaf(squares, over_n, -square);
        const float variance = (spread < 0.0f ? 0.0f : spread) + eps;
        const bool constant = variance < square * 0x1p-22f;
        const float r = rsqrtf(constant ? eps : variance);
        return {shift, r, (constant ? 0.0f : -delta) * r, far || constant};
    }
    __device__ __forceinline__ float normalised(float d) const { return fmaf(d, r, c); }
    __device__ __forceinline__ float of(float x) const { return normalised(flat ? 0.0f : x - shift); }
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
// half a scale the even one is taken.  (Added to 1.5 * 2^23 a number is rounded to a whole one, whose low byte is then the code.)
__device__ __forceinline__ void encode_int8(const float (&v)[8], const RowScale &s, row_v2i &codes)
{
    constexpr float kWhole = 12582912.0f;
    float t[8], left[8], most = 0.0f;
    const float half = 0.5f * s.scale;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        t[e] = fmaf(v[e], s.inverse, kWhole);
        left[e] = fmaf(kWhole - t[e], s.scale, v[e]);
        most = fmaxf(most, fabsf(left[e]));
    }
    if (most >= half) {  // rare
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float a = fabsf(left[e]);
            const bool odd = (__builtin_bit_cast(unsigned, t[e]) & 1u) != 0;
            if (a > half || (a == half && odd))
                t[e] += left[e] > 0.0f ? 1.0f : -1.0f;
        }
    }
    unsigned bytes[2];
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        unsigned two[2];
#pragma unroll
        for (int h = 0; h < 2; ++h)
            two[h] = __builtin_amdgcn_perm(__builtin_bit_cast(unsigned, t[4 * w + 2 * h + 1]), __builtin_bit_cast(unsigned, t[4 * w + 2 * h]), 0x0C0C0400u);
        bytes[w] = two[0] | two[1] << 16;
    }
    codes = s.scale == s.scale ? (row_v2i){(int)bytes[0], (int)bytes[1]} : (row_v2i)0;
}

}  // namespace int4linear
