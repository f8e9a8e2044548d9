// What the MXFP4 product kernels share: addresses for their loads, and what they do with their sums (activations,
// types, blocks in MXFP4).
#pragma once
#include "mxfp4.h"

#include <type_traits>

namespace int4linear {

// An address that is the same in all lanes, in scalar registers.  The compiler multiplies 64 bits in vector registers, and
// what it then adds to in a loop would stay in them.
__device__ __forceinline__ const uint8_t *uniform(const uint8_t *p)
{
    const unsigned long long bits = (unsigned long long)p;
    const unsigned low = __builtin_amdgcn_readfirstlane((int)bits), high = __builtin_amdgcn_readfirstlane((int)(bits >> 32));
    return (const uint8_t *)(low | ((unsigned long long)high << 32));
}

// 16 bytes per lane from base + offset straight into LDS at to + 16 * lane (NT: read once).  A load may read a scalar
// register no sooner than five instructions after a vector instruction wrote it (a reload of a spilled one, say), which the
// compiler sees to for its own loads only: hence the long s_nop.  (M0 is reserved: the compiler keeps nothing there, refuses it
// among the clobbers, and has no instruction in these kernels that would read it.)
template <bool NT = false>
__device__ __forceinline__ void dma16(const void *base, unsigned offset, unsigned to)
{
    if constexpr (NT)
        asm volatile("s_mov_b32 m0, %2\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %0, %1 nt" : : "v"(offset), "s"(base), "s"(to) : "memory");
    else
        asm volatile("s_mov_b32 m0, %2\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(offset), "s"(base), "s"(to) : "memory");
}

// The same from an address of the lane's own.
__device__ __forceinline__ void dma16(const void *lane_address, unsigned to)
{
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(lane_address), "s"(to) : "memory");
}

template <int OUT>
using OutElement = std::conditional_t<OUT == kOutF32, float, std::conditional_t<OUT == kOutF16, _Float16, __bf16>>;

// act(g) and its slope.  The gelu's (1 + tanh z) / 2 is the logistic function of 2 z.
constexpr float kGeluScale = 1.5957691216057308f;  // 2 sqrt(2 / pi)
constexpr float kGeluCubic = 0.044715f;

__device__ __forceinline__ float logistic(float z) { return 1.0f / (1.0f + expf(-z)); }

__device__ __forceinline__ float activate(int act, float g)
{
    return g * logistic(act == kSilu ? g : kGeluScale * (g + kGeluCubic * g * g * g));
}

__device__ __forceinline__ void activate_with_slope(int act, float g, float &value, float &slope)
{
    const float s = logistic(act == kSilu ? g : kGeluScale * (g + kGeluCubic * g * g * g));
    value = g * s;
    // (g^2 stays finite: far out its factor s (1 - s) is 0)
    slope = s + g * s * (1.0f - s) * (act == kSilu ? 1.0f : kGeluScale * (1.0f + 3.0f * kGeluCubic * fminf(g * g, 1e30f)));
}

// Eight values as E2M1 codes, the first in the lowest four bits.  The hardware's conversion rounds to nearest
// even and takes what is beyond 6 to 6.
__device__ __forceinline__ unsigned encode8(const float (&v)[8])
{
    unsigned c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0], v[1], 1.0f, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], 1.0f, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], 1.0f, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], 1.0f, 3);
    return c;
}

// Eight values of a block whose largest magnitude has the bits `big` (NaN above infinity above all numbers), and
// the block's scale code.
__device__ __forceinline__ unsigned encode_block_part(const float (&v)[8], unsigned big, unsigned &code)
{
    const unsigned field = big >> 23;  // 255: an infinity or a NaN
    code = field == 255 ? 255 : field > 2 ? field - 2 : 0;
    const float inverse = __builtin_bit_cast(float, code >= 254 ? 0x00400000u : (254 - code) << 23);  // 2^(127 - code)
    float s[8];
#pragma unroll
    for (int e = 0; e < 8; ++e)
        s[e] = field == 255 ? 0.0f : v[e] * inverse;
    return encode8(s);
}

// The scale of the block at column c0 of a row of h whose codes take `code_stride` bytes.  With the last block of
// the codes the rest of the scales' 16 bytes is written too.
__device__ __forceinline__ void store_block_scale(uint8_t *row, int c0, size_t code_stride, unsigned code)
{
    uint8_t *to = row + c0 / kMxBlock;
    *to = (uint8_t)code;
    if ((size_t)c0 + kMxBlock == code_stride * 2 && code_stride % (2 * kLineBytes))
        *(unsigned long long *)(to + 1) = 0;
}

}  // namespace int4linear
