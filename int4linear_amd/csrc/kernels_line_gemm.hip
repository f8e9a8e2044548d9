// GEMM over lines of 128 bytes: MXFP4 operands (256 k per line, block scales applied by the matrix
// instruction) and bfloat16 operands (64 k per line), y = a b^T.
//
// Both element types share one kernel, because their matrix instructions take the same bytes from
// a lane: v_mfma_scale_f32_32x32x64_f8f6f4 on 4-bit operands and v_mfma_f32_32x32x16_bf16 both
// read 16 bytes of row lane % 32, and both run 32 cycles.  A stage is one line of every row of the tile; lane
// group lane / 32 takes chunk (16 bytes) 4 * (lane / 32) + j of its rows in step j = 0 .. 3, for a and b
// alike, which is all that a sum over k asks for.  With 4-bit operands a chunk is one block of 32, and the
// scales of the four chunks that a lane sees in a stage are the four bytes of one aligned dword.
//
// b's rows are the instruction's first operand: a lane then holds, for one row of a, four consecutive
// columns of y in each group of eight, and stores are wide.
#include "mxfp4.h"

#include <type_traits>
#include <utility>

namespace int4linear {

namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef __bf16 v4bf __attribute__((ext_vector_type(4)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v4h __attribute__((ext_vector_type(4)));

constexpr int kFrag = 32;

// Rows of an operand.  data[row * stride] starts a row of `stages` lines; scales likewise (4-bit only).
struct LineRows {
    const uint8_t *data;
    const uint8_t *scales;
    size_t stride;
    size_t scale_stride;
    int rows;
};

// ---- what happens to a tile's sums ------------------------------------------------------------
// An epilogue is called once per wave as ep(acc, row, col, lane): acc[j][i] is the 32 x 32 block at rows
// row + 32 j of a and columns col + 32 i of the product; element t of a lane is at row + 32 j + lane % 32
// and column col + 32 i + 8 (t / 4) + 4 (lane / 32) + t % 4.  kPair: two operands b share the
// tile, blocks i even of the first, odd of the second, each pair over the same 32 columns.

template <int OUT>
__device__ __forceinline__ void store4(void *y, size_t at, const float (&v)[4], int valid, bool vec)
{
    if constexpr (OUT == kOutF32) {
        float *dst = (float *)y + at;
        if (vec && valid == 4) {
            *(v4f *)dst = (v4f){v[0], v[1], v[2], v[3]};
            return;
        }
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (q < valid)
                dst[q] = v[q];
    } else {
        using T = std::conditional_t<OUT == kOutF16, _Float16, __bf16>;
        typedef T v4t __attribute__((ext_vector_type(4)));
        T *dst = (T *)y + at;
        if (vec && valid == 4) {
            *(v4t *)dst = (v4t){(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
            return;
        }
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (q < valid)
                dst[q] = (T)v[q];
    }
}

// y = sums + bias, rounded once to OUT.
template <int OUT>
struct PlainEpilogue {
    static constexpr bool kPair = false;
    void *y[2];  // by blockIdx.z
    const float *bias;
    size_t ld;
    int m, n;
    bool vec;  // four columns from a multiple of four on are aligned

    template <int FM, int FN>
    __device__ void operator()(v16f (&acc)[FM][FN], int row, int col, int lane) const
    {
        void *dst = y[blockIdx.z];
#pragma unroll
        for (int j = 0; j < FM; ++j) {
            const int r = row + kFrag * j + (lane & 31);
            if (r >= m)
                continue;
#pragma unroll
            for (int i = 0; i < FN; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int c = col + kFrag * i + 8 * q + 4 * (lane >> 5);
                    if (c >= n)
                        continue;
                    float v[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        v[e] = acc[j][i][4 * q + e] + (bias ? bias[min(c + e, n - 1)] : 0.0f);
                    store4<OUT>(dst, (size_t)r * ld + c, v, min(n - c, 4), vec);
                }
        }
    }
};

// act(g) and its slope.  The gelu's (1 + tanh z) / 2 is the logistic function of 2 z.
constexpr float kGeluScale = 1.5957691216057308f;  // 2 sqrt(2 / pi)
constexpr float kGeluCubic = 0.044715f;

__device__ __forceinline__ float logistic(float z) { return 1.0f / (1.0f + expf(-z)); }

__device__ __forceinline__ float activate(int act, float g)
{
    if (act == kSilu)
        return g * logistic(g);
    return g * logistic(kGeluScale * (g + kGeluCubic * g * g * g));
}

__device__ __forceinline__ void activate_with_slope(int act, float g, float &value, float &slope)
{
    if (act == kSilu) {
        const float s = logistic(g);
        value = g * s;
        slope = s * (1.0f + g * (1.0f - s));
    } else {
        const float s = logistic(kGeluScale * (g + kGeluCubic * g * g * g));
        value = g * s;
        slope = s + g * s * (1.0f - s) * kGeluScale * (1.0f + 3.0f * kGeluCubic * g * g);
    }
}

// h = act(g) * u, rounded once to OUT.
template <int OUT>
struct GatedEpilogue {
    static constexpr bool kPair = true;
    void *h;
    size_t ld;
    int m, n, act;
    bool vec;

    template <int FM, int FN>
    __device__ void operator()(v16f (&acc)[FM][FN], int row, int col, int lane) const
    {
#pragma unroll
        for (int j = 0; j < FM; ++j) {
            const int r = row + kFrag * j + (lane & 31);
            if (r >= m)
                continue;
#pragma unroll
            for (int i = 0; i < FN; i += 2)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int c = col + kFrag * (i / 2) + 8 * q + 4 * (lane >> 5);
                    if (c >= n)
                        continue;
                    float v[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        v[e] = activate(act, acc[j][i][4 * q + e]) * acc[j][i + 1][4 * q + e];
                    store4<OUT>(h, (size_t)r * ld + c, v, min(n - c, 4), vec);
                }
        }
    }
};

// The same in MXFP4: a block of 32 columns of a row sits in lanes l and l + 32.
struct GatedMxEpilogue {
    static constexpr bool kPair = true;
    uint8_t *codes, *scales;
    size_t code_stride, scale_stride;
    int m, n, act;

    template <int FM, int FN>
    __device__ void operator()(v16f (&acc)[FM][FN], int row, int col, int lane) const
    {
#pragma unroll
        for (int j = 0; j < FM; ++j) {
            const int r = row + kFrag * j + (lane & 31);
#pragma unroll
            for (int i = 0; i < FN; i += 2) {
                const int c0 = col + kFrag * (i / 2);
                float v[16];
                unsigned big = 0;
#pragma unroll
                for (int t = 0; t < 16; ++t) {
                    const int c = c0 + 8 * (t / 4) + 4 * (lane >> 5) + t % 4;
                    v[t] = c < n ? activate(act, acc[j][i][t]) * acc[j][i + 1][t] : 0.0f;
                    big = max(big, __builtin_bit_cast(unsigned, v[t]) & 0x7FFFFFFFu);
                }
                big = max(big, (unsigned)__shfl_xor((int)big, 32));
                const int field = (int)(big >> 23);
                const int code = field == 255 ? 255 : max(field - 2, 0);
                const float inverse = field == 255 ? 0.0f : __builtin_bit_cast(float, code == 254 ? 0x00400000 : (254 - code) << 23);
                if (r >= m || (size_t)c0 >= code_stride * 2)
                    continue;
                unsigned short *dst = (unsigned short *)(codes + (size_t)r * code_stride + c0 / 2) + (lane >> 5);
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    float s[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        s[e] = field == 255 ? 0.0f : v[4 * q + e] * inverse;
                    unsigned bits = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, s[0], s[1], 1.0f, 0);
                    bits = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(bits, s[2], s[3], 1.0f, 1);
                    dst[2 * q] = (unsigned short)bits;
                }
                if (lane < 32) {
                    uint8_t *to = scales + (size_t)r * scale_stride + c0 / kMxBlock;
                    *to = (uint8_t)code;
                    // the row's last line of codes; its scales go on for one more where they are not 16 yet
                    if ((size_t)c0 + kMxBlock == code_stride * 2 && code_stride % (2 * kLineBytes))
                        *(unsigned long long *)(to + 1) = 0;
                }
            }
        }
    }
};

// dg = dh * u * act'(g), du = dh * act(g), rounded to bfloat16: they are the operands of two more products
// on matrix cores that take 16 bits; the roundings of the terms (2^-8 at most, of random sign) add up to as much as
// the rounding of the result itself.
struct GradientEpilogue {
    static constexpr bool kPair = true;
    const __bf16 *dh;
    __bf16 *d, *dt;
    size_t ld_n, ld_m;
    int m, n, act;
    bool vec;

    template <int FM, int FN>
    __device__ void operator()(v16f (&acc)[FM][FN], int row, int col, int lane) const
    {
#pragma unroll
        for (int j = 0; j < FM; ++j) {
            const int r = row + kFrag * j + (lane & 31);
#pragma unroll
            for (int i = 0; i < FN; i += 2)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int c = col + kFrag * (i / 2) + 8 * q + 4 * (lane >> 5);
                    v4bf in = {};
                    if (r < m && c < n) {
                        const __bf16 *src = dh + (size_t)r * n + c;
                        if (vec && c + 4 <= n) {
                            in = *(const v4bf *)src;
                        } else {
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                if (c + e < n)
                                    in[e] = src[e];
                        }
                    }
                    v4bf dg = {}, du = {};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (r >= m || c + e >= n)
                            continue;  // padding: exact zeros, whatever the clamped rows gave
                        float value, slope;
                        activate_with_slope(act, acc[j][i][4 * q + e], value, slope);
                        const float up = acc[j][i + 1][4 * q + e], g = (float)in[e];
                        dg[e] = (__bf16)(g * up * slope);
                        du[e] = (__bf16)(g * value);
                    }
                    if (r < m && (size_t)c < ld_n) {
                        *(v4bf *)(d + (size_t)r * 2 * ld_n + c) = dg;
                        *(v4bf *)(d + (size_t)r * 2 * ld_n + ld_n + c) = du;
                    }
                    if ((size_t)r < ld_m) {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (c + e < n) {
                                dt[(size_t)(c + e) * ld_m + r] = dg[e];
                                dt[((size_t)n + c + e) * ld_m + r] = du[e];
                            }
                    }
                }
        }
    }
};

// ---- the kernel -------------------------------------------------------------------------------

template <int WAVES_M_, int WAVES_N_, int FM_, int FN_>
struct LineTile {
    static constexpr int WAVES_M = WAVES_M_, WAVES_N = WAVES_N_, FM = FM_, FN = FN_;
    static constexpr int NWAVES = WAVES_M * WAVES_N, THREADS = NWAVES * 64;
    static constexpr int BM = WAVES_M * FM * kFrag, BN = WAVES_N * FN * kFrag;
    static constexpr int STAGE = (BM + BN) * kLineBytes;
    static constexpr int LDS = 2 * STAGE;
    static constexpr int CHUNKS = STAGE / 1024 / NWAVES;  // 1-KiB loads per wave and stage
    static_assert(STAGE % (1024 * NWAVES) == 0);
};

// Order of tiles: workgroup ids go round-robin over the 8 XCDs; ids congruent mod 8 get consecutive
// positions of an order that walks groups of 8 tile rows column by column, so that concurrent tiles of one
// XCD share operand rows in its L2.
__device__ __forceinline__ void tile_coords(int v, int total, int tiles_m, int tiles_n, int &tm, int &tn)
{
    constexpr int kXcd = 8, kGroup = 8;
    const int x = v % kXcd, j = v / kXcd;
    const int cnt = total / kXcd, rem = total % kXcd;
    const int q = x * cnt + (x < rem ? x : rem) + j;
    const int per_group = kGroup * tiles_n;
    const int group = q / per_group;
    const int first_m = group * kGroup;
    const int gsz = (tiles_m - first_m < kGroup) ? (tiles_m - first_m) : kGroup;
    const int in_group = q % per_group;
    tm = first_m + in_group % gsz;
    tn = in_group / gsz;
}

#define I4L_LDS(p) ((__attribute__((address_space(3))) void *)(p))
#define I4L_GLOBAL(p) ((const __attribute__((address_space(1))) void *)(p))

template <bool FP4, class C, class Ep>
__global__ __launch_bounds__(C::THREADS) void line_gemm_kernel(LineRows a, LineRows b0, LineRows b1, size_t a_batch, int stages,
                                                               int tiles_m, int tiles_n, Ep ep)
{
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / C::WAVES_N, wn = wave % C::WAVES_N;
    int tm, tn;
    tile_coords(blockIdx.x, tiles_m * tiles_n, tiles_m, tiles_n, tm, tn);
    const int m0 = tm * C::BM;
    const int n0 = tn * (Ep::kPair ? C::BN / 2 : C::BN);  // column of y

    // Row of an LDS row of b's part of the tile, and its matrix.
    auto b_row = [&](int r, bool &second) {
        second = Ep::kPair && ((r / kFrag) & 1);
        const int c = n0 + (Ep::kPair ? r / (2 * kFrag) * kFrag + r % kFrag : r);
        return min(c, b0.rows - 1);
    };

    // Load c of a wave fills LDS rows 8 (c * NWAVES + wave) .. + 7 of a stage, lane l the 16 bytes at place l.
    // The chunk that lies at place p of row r is p ^ (r / 2 % 8): the 16 lanes that an LDS read serves together
    // then touch every bank once.
    const uint8_t *src[C::CHUNKS];
#pragma unroll
    for (int c = 0; c < C::CHUNKS; ++c) {
        const int r = (c * C::NWAVES + wave) * 8 + (lane >> 3);
        const int chunk = (lane & 7) ^ ((r >> 1) & 7);
        bool second = false;
        if (r < C::BM) {
            src[c] = a.data + blockIdx.z * a_batch + (size_t)min(m0 + r, a.rows - 1) * a.stride + chunk * 16;
        } else {
            const int br = b_row(r - C::BM, second);
            src[c] = (second ? b1.data : b0.data) + (size_t)br * b0.stride + chunk * 16;
        }
    }
    auto load_stage = [&](int s) {
#pragma unroll
        for (int c = 0; c < C::CHUNKS; ++c) {
            uint8_t *dst = lds + (s & 1) * C::STAGE + (c * C::NWAVES + wave) * 1024;
            __builtin_amdgcn_global_load_lds(I4L_GLOBAL(src[c] + (size_t)s * kLineBytes), I4L_LDS(dst), 16, 0, 0);
        }
    };

    // Scales: this lane's row of every fragment, the dword of its lane group.
    const uint8_t *a_scale[C::FM], *b_scale[C::FN];
    if constexpr (FP4) {
#pragma unroll
        for (int j = 0; j < C::FM; ++j)
            a_scale[j] = a.scales + (size_t)min(m0 + (wm * C::FM + j) * kFrag + (lane & 31), a.rows - 1) * a.scale_stride + 4 * (lane >> 5);
#pragma unroll
        for (int i = 0; i < C::FN; ++i) {
            bool second;
            const int r = b_row((wn * C::FN + i) * kFrag + (lane & 31), second);
            b_scale[i] = (second ? b1.scales : b0.scales) + (size_t)r * b0.scale_stride + 4 * (lane >> 5);
        }
    }

    v16f acc[C::FM][C::FN];
#pragma unroll
    for (int j = 0; j < C::FM; ++j)
#pragma unroll
        for (int i = 0; i < C::FN; ++i)
            acc[j][i] = (v16f)0.0f;

    const int swz = ((lane & 31) >> 1) & 7;
    const uint8_t *a_rd = lds + (wm * C::FM * kFrag + (lane & 31)) * kLineBytes;
    const uint8_t *b_rd = lds + (C::BM + wn * C::FN * kFrag + (lane & 31)) * kLineBytes;

    if (stages > 0)
        load_stage(0);
    for (int s = 0; s < stages; ++s) {
        int sa[C::FM], sb[C::FN];
        if constexpr (FP4) {
#pragma unroll
            for (int j = 0; j < C::FM; ++j)
                sa[j] = *(const int *)(a_scale[j] + 8 * (size_t)s);
#pragma unroll
            for (int i = 0; i < C::FN; ++i)
                sb[i] = *(const int *)(b_scale[i] + 8 * (size_t)s);
        }
        __syncthreads();  // stage s has landed (the barrier waits for loads), stage s - 1 has been read
        if (s + 1 < stages)
            load_stage(s + 1);
        const int buffer = (s & 1) * C::STAGE;
        [&]<int... J>(std::integer_sequence<int, J...>) {
            ([&] {
                const int at = buffer + ((4 * (lane >> 5) + J) ^ swz) * 16;
                v4i fa[C::FM], fb[C::FN];
#pragma unroll
                for (int j = 0; j < C::FM; ++j)
                    fa[j] = *(const v4i *)(a_rd + at + j * kFrag * kLineBytes);
#pragma unroll
                for (int i = 0; i < C::FN; ++i)
                    fb[i] = *(const v4i *)(b_rd + at + i * kFrag * kLineBytes);
#pragma unroll
                for (int j = 0; j < C::FM; ++j)
#pragma unroll
                    for (int i = 0; i < C::FN; ++i) {
                        if constexpr (FP4) {
                            const v8i wide_a = {fa[j][0], fa[j][1], fa[j][2], fa[j][3], 0, 0, 0, 0};
                            const v8i wide_b = {fb[i][0], fb[i][1], fb[i][2], fb[i][3], 0, 0, 0, 0};
                            acc[j][i] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wide_b, wide_a, acc[j][i], 4, 4, J, sb[i], J, sa[j]);
                        } else {
                            acc[j][i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, fb[i]),
                                                                               __builtin_bit_cast(v8bf, fa[j]), acc[j][i], 0, 0, 0);
                        }
                    }
            }(), ...);
        }(std::make_integer_sequence<int, 4>{});
    }
    ep(acc, m0 + wm * C::FM * kFrag, n0 + wn * C::FN * kFrag / (Ep::kPair ? 2 : 1), lane);
}

using Tile128 = LineTile<2, 2, 2, 2>;

template <bool FP4, class C, class Ep>
hipError_t launch(const LineRows &a, const LineRows &b0, const LineRows &b1, size_t a_batch, int batch, int stages, int n, const Ep &ep,
                  hipStream_t stream)
{
    const int bn = Ep::kPair ? C::BN / 2 : C::BN;
    const int tiles_m = (a.rows + C::BM - 1) / C::BM, tiles_n = (n + bn - 1) / bn;
    line_gemm_kernel<FP4, C, Ep><<<dim3((unsigned)(tiles_m * tiles_n), 1, (unsigned)batch), C::THREADS, C::LDS, stream>>>(
        a, b0, b1, a_batch, stages, tiles_m, tiles_n, ep);
    return hipGetLastError();
}

LineRows rows_of(const MxMatrix &q, int k) { return {q.codes, q.scales, mx_code_stride(k), mx_scale_stride(k), q.rows}; }

bool aligned(const void *p, size_t ld, int out)
{
    const size_t bytes = out == kOutF32 ? 16 : 8;
    return (uintptr_t)p % bytes == 0 && ld % 4 == 0;
}

// f(std::integral_constant<int, out>) for the output type of a call.
template <class F>
hipError_t by_type(int out, F &&f)
{
    switch (out) {
    case kOutF32:
        return f(std::integral_constant<int, kOutF32>{});
    case kOutF16:
        return f(std::integral_constant<int, kOutF16>{});
    default:
        return f(std::integral_constant<int, kOutBF16>{});
    }
}

}  // namespace

hipError_t line_gemm_init(const DeviceInfo &) { return hipSuccess; }

hipError_t launch_mx_linear(const MxMatrix &x, const MxMatrix &w, const float *bias, void *y, int out, int k, const DeviceInfo &,
                            hipStream_t stream)
{
    const int stages = (k + kLineFp4 - 1) / kLineFp4;
    return by_type(out, [&](auto type) {
        const PlainEpilogue<decltype(type)::value> ep{{y, nullptr}, bias, (size_t)w.rows, x.rows, w.rows, aligned(y, w.rows, out)};
        return launch<true, Tile128>(rows_of(x, k), rows_of(w, k), rows_of(w, k), 0, 1, stages, w.rows, ep, stream);
    });
}

hipError_t launch_mx_gated(const MxMatrix &x, const MxMatrix &wg, const MxMatrix &wu, Activation act, void *h, int out, int k,
                           const DeviceInfo &, hipStream_t stream)
{
    const int stages = (k + kLineFp4 - 1) / kLineFp4;
    return by_type(out, [&](auto type) {
        const GatedEpilogue<decltype(type)::value> ep{h, (size_t)wg.rows, x.rows, wg.rows, act, aligned(h, wg.rows, out)};
        return launch<true, Tile128>(rows_of(x, k), rows_of(wg, k), rows_of(wu, k), 0, 1, stages, wg.rows, ep, stream);
    });
}

hipError_t launch_mx_gated_quantized(const MxMatrix &x, const MxMatrix &wg, const MxMatrix &wu, Activation act, uint8_t *codes,
                                     uint8_t *scales, int k, const DeviceInfo &, hipStream_t stream)
{
    const int stages = (k + kLineFp4 - 1) / kLineFp4;
    const int n = wg.rows;
    const GatedMxEpilogue ep{codes, scales, mx_code_stride(n), mx_scale_stride(n), x.rows, n, act};
    // (the grid covers the padding at the end of h's rows)
    return launch<true, Tile128>(rows_of(x, k), rows_of(wg, k), rows_of(wu, k), 0, 1, stages, (int)(mx_code_stride(n) * 2), ep, stream);
}

hipError_t launch_mx_gated_gradients(const MxMatrix &x, const MxMatrix &wg, const MxMatrix &wu, Activation act, const uint16_t *dh,
                                     uint16_t *d, size_t ld_n, uint16_t *dt, size_t ld_m, int k, const DeviceInfo &,
                                     hipStream_t stream)
{
    const int stages = (k + kLineFp4 - 1) / kLineFp4;
    const GradientEpilogue ep{(const __bf16 *)dh, (__bf16 *)d, (__bf16 *)dt, ld_n, ld_m, x.rows, wg.rows, act,
                              aligned(dh, wg.rows, kOutBF16)};
    return launch<true, Tile128>(rows_of(x, k), rows_of(wg, k), rows_of(wu, k), 0, 1, stages, wg.rows, ep, stream);
}

hipError_t launch_bf16_gemm(const uint16_t *a, size_t ld_a, int m, const uint16_t *b, size_t ld_b, int n, int k, void *y0, void *y1,
                            int batch, int out, const DeviceInfo &, hipStream_t stream)
{
    const int stages = (k + kLineBf16 - 1) / kLineBf16;
    const LineRows ra{(const uint8_t *)a, nullptr, ld_a * 2, 0, m}, rb{(const uint8_t *)b, nullptr, ld_b * 2, 0, n};
    return by_type(out, [&](auto type) {
        const PlainEpilogue<decltype(type)::value> ep{{y0, y1}, nullptr, (size_t)n, m, n, aligned(y0, n, out) && (batch == 1 || aligned(y1, n, out))};
        return launch<false, Tile128>(ra, rb, rb, (size_t)m * ld_a * 2, batch, stages, n, ep, stream);
    });
}

}  // namespace int4linear
