// Few rows of x against MXFP4 weights: every byte of w is read once.
//
// A workgroup owns 16 R rows of w (of both matrices for the gated block) and all of k.  Its waves split k
// tile by tile of 256 (one 128-byte line of a row); a wave issues all loads of a tile at once, waits, multiplies
// with v_mfma_scale_f32_16x16x128_f8f6f4 and takes its next tile.  The waves' sums meet in LDS at the end.  (Runs of two or
// four tiles at once were slower at every size: they leave room for fewer workgroups on a CU.)
// Bound by the stream of w.  A load instruction moves whole lines of eight rows straight into LDS: in the matrix
// instruction's own pattern (64 bytes of each of sixteen rows, into registers) the same kernel read 31 MB in 10.8 us.
// x and the scales are small and come from the caches into registers: a lane takes row lane % 16 of a fragment and
// chunks (16 bytes, one block of 32) lane / 16 and 4 + lane / 16 of a line, so that the blocks' scales are byte
// lane / 16 of the two dwords that a row has for the line.
#include "mxfp4.h"
#include "mxfp4_epilogue.h"

namespace int4linear {

namespace {

typedef int v2i __attribute__((ext_vector_type(2)));
typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));

constexpr int kRows = 16;      // rows of a fragment
constexpr int kTileBytes = kRows * kLineBytes;

enum Mode : int { kPlain, kGated, kGatedMx };

struct SkinnyArgs {
    const uint8_t *x, *xs, *w0, *w0s, *w1, *w1s;
    size_t stride, scale_stride;
    const float *bias;
    void *y;           // codes for kGatedMx
    uint8_t *y_scales;
    size_t ld, ld_scales;  // elements (bytes for kGatedMx) between rows of y
    int m, n, lines, out, act;
};

__device__ __forceinline__ v8i wide(const v4i &v) { return (v8i){v[0], v[1], v[2], v[3], 0, 0, 0, 0}; }

// Four results of row r of y from column c on.
template <int OUT>
__device__ __forceinline__ void store4(const SkinnyArgs &g, int r, int c, const v4f &v)
{
    using T = OutElement<OUT>;
    typedef T v4t __attribute__((ext_vector_type(4)));
    T *dst = (T *)g.y + (size_t)r * g.ld + c;
    if (g.n % 4 == 0) {
        *(v4t *)dst = (v4t){(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (c + e < g.n)
                dst[e] = (T)v[e];
    }
}

#define I4L_LDS(p) ((__attribute__((address_space(3))) void *)(p))

// R x FM fragments of w (times two for the gated modes) and x; a wave's run is one tile of each fragment.
template <int MODE, int R, int FM>
__global__ __launch_bounds__(1024) void mx_skinny_kernel(SkinnyArgs g)
{
    constexpr int MATS = MODE == kPlain ? 1 : 2, FW = R * MATS;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int waves = blockDim.x >> 6;
    const int n0 = blockIdx.x * R * kRows, m0 = blockIdx.y * FM * kRows;
    uint8_t *mine = lds + wave * (FW * kTileBytes);
    const unsigned my_lds = (unsigned)(size_t)I4L_LDS(mine);

    // Rows behind the matrix: the last one again.  (h's padding may have workgroups of its own.)
    const int nb = min(n0, g.n - 1), last = g.n - 1 - nb;
    const uint8_t *w0 = uniform(g.w0 + (size_t)nb * g.stride), *w1 = MATS == 2 ? uniform(g.w1 + (size_t)nb * g.stride) : nullptr;
    unsigned off[R][2];
#pragma unroll
    for (int f = 0; f < R; ++f)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = 8 * h + (lane >> 3);
            off[f][h] = (unsigned)min(f * kRows + r, last) * (unsigned)g.stride + (((lane & 7) ^ ((r >> 1) & 7)) << 4);
        }
    const int row = lane & 15, q = lane >> 4;
    v4f acc[FW][FM];
#pragma unroll
    for (int f = 0; f < FW; ++f)
#pragma unroll
        for (int j = 0; j < FM; ++j)
            acc[f][j] = (v4f)0.0f;

    for (int t = wave; t < g.lines; t += waves) {
#pragma unroll
        for (int f = 0; f < FW; ++f)
#pragma unroll
            for (int h = 0; h < 2; ++h)
                dma16<true>((f % MATS ? w1 : w0) + (size_t)t * kLineBytes, off[f / MATS][h], my_lds + f * kTileBytes + h * 1024);
        v2i ws[FW], xs[FM];
        v4i x[FM][2];
#pragma unroll
        for (int f = 0; f < FW; ++f)
            ws[f] = *(const v2i *)((f % MATS ? g.w1s : g.w0s) + (size_t)(nb + min(f / MATS * kRows + row, last)) * g.scale_stride +
                                   (size_t)t * 8);
#pragma unroll
        for (int j = 0; j < FM; ++j) {
            const int r = m0 + j * kRows + row;
            xs[j] = (v2i){0, 0};
            x[j][0] = x[j][1] = (v4i){0, 0, 0, 0};
            if (r < g.m) {
                xs[j] = *(const v2i *)(g.xs + (size_t)r * g.scale_stride + (size_t)t * 8);
                const uint8_t *src = g.x + (size_t)r * g.stride + (size_t)t * kLineBytes + q * 16;
                x[j][0] = *(const v4i *)src;
                x[j][1] = *(const v4i *)(src + 64);
            }
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
        for (int f = 0; f < FW; ++f)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const v4i w = *(const v4i *)(mine + f * kTileBytes + row * kLineBytes + (((q + 4 * i) ^ ((row >> 1) & 7)) << 4));
#pragma unroll
                for (int j = 0; j < FM; ++j)
                    acc[f][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wide(w), wide(x[j][i]), acc[f][j], 4, 4, 0,
                                                                                (int)((unsigned)ws[f][i] >> (8 * q)), 0,
                                                                                (int)((unsigned)xs[j][i] >> (8 * q)));
            }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // read before it is loaded again
    }

    // Element t of a lane: column n0 + 16 f + 4 (lane / 16) + t of row m0 + 16 j + lane % 16.  Every wave leaves
    // its sums; then one wave per R fragments (of both matrices) of a row block j adds them up in order.
    static_assert(FM <= 2, "a wave's sums fit where its tiles were");
    v4f *sums = (v4f *)mine;
#pragma unroll
    for (int f = 0; f < FW; ++f)
#pragma unroll
        for (int j = 0; j < FM; ++j)
            sums[(f * FM + j) * 64 + lane] = acc[f][j];
    __syncthreads();
    auto total = [&](int f, int j) {
        const v4f *from = (const v4f *)lds + (f * FM + j) * 64 + lane;
        v4f s = from[0];
        for (int w = 1; w < waves; ++w)
            s += from[w * (FW * kTileBytes / 16)];
        return s;
    };
    if constexpr (MODE == kGatedMx) {
        static_assert(R == 2, "a block of 32 columns");
        for (int j = wave; j < FM; j += waves) {
            const int r = m0 + j * kRows + row;
            float v[8];
            unsigned big = 0;
#pragma unroll
            for (int f = 0; f < R; ++f) {
                const v4f gate = total(f * MATS, j), up = total(f * MATS + MATS - 1, j);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int c = n0 + f * kRows + 4 * q + e;
                    v[4 * f + e] = c < g.n ? activate(g.act, gate[e]) * up[e] : 0.0f;
                    big = max(big, __builtin_bit_cast(unsigned, v[4 * f + e]) & 0x7FFFFFFFu);
                }
            }
            big = max(big, (unsigned)__shfl_xor((int)big, 16));
            big = max(big, (unsigned)__shfl_xor((int)big, 32));
            unsigned code;
            const unsigned bits = encode_block_part(v, big, code);
            if (r < g.m) {
                unsigned short *dst = (unsigned short *)((uint8_t *)g.y + (size_t)r * g.ld + n0 / 2) + q;
                dst[0] = (unsigned short)bits;
                dst[4] = (unsigned short)(bits >> 16);
                if (q == 0)
                    store_block_scale(g.y_scales + (size_t)r * g.ld_scales, n0, g.ld, code);
            }
        }
    } else {
        for (int b = wave; b < R * FM; b += waves) {
            const int f = b / FM, j = b % FM;
            const int r = m0 + j * kRows + row, c = n0 + f * kRows + 4 * q;
            v4f v = total(f * MATS, j);
            if constexpr (MODE == kGated) {
                const v4f up = total(f * MATS + MATS - 1, j);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    v[e] = activate(g.act, v[e]) * up[e];
            } else if (g.bias) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    v[e] += g.bias[min(c + e, g.n - 1)];
            }
            if (r < g.m && c < g.n) {
                if (g.out == kOutF32)
                    store4<kOutF32>(g, r, c, v);
                else if (g.out == kOutF16)
                    store4<kOutF16>(g, r, c, v);
                else
                    store4<kOutBF16>(g, r, c, v);
            }
        }
    }
}

constexpr int kMaxLds = 64 * 1024;

// Waves: k in two passes over the workgroup's tiles, so that the second one's loads follow the first's while other
// workgroups compute, and at most 16 waves.  14336 x 4096, one row: 8 waves 9.0 us, 4 9.4, 16 9.2; 8192 x 8192: 16 waves
// 9.7 us, 8 10.2; 4096 x 14336: 14 waves (56 tiles in four full passes) 7.9 us, 16 8.2.
template <int MODE, int R, int FM>
hipError_t launch_kernel(const SkinnyArgs &g, int n, hipStream_t stream)
{
    constexpr int kWaveLds = R * (MODE == kPlain ? 1 : 2) * kTileBytes;
    const int passes = max(2, (g.lines + 15) / 16);
    const int waves = min((g.lines + passes - 1) / passes, kMaxLds / kWaveLds);
    const dim3 grid((unsigned)((n + R * kRows - 1) / (R * kRows)), (unsigned)((g.m + FM * kRows - 1) / (FM * kRows)));
    mx_skinny_kernel<MODE, R, FM><<<grid, waves * 64, (size_t)waves * kWaveLds, stream>>>(g);
    return hipGetLastError();
}

template <int MODE, int R>
hipError_t launch_rows(const SkinnyArgs &g, int n, hipStream_t stream)
{
    return g.m <= kRows ? launch_kernel<MODE, R, 1>(g, n, stream) : launch_kernel<MODE, R, 2>(g, n, stream);
}

// Fragments of w per workgroup: more of them read x less often, fewer make more workgroups.  One as long as two would
// leave CUs without a workgroup.  (us, weights from HBM, with 1, 2, 4: 14336 x 4096, 1 row 9.0, 8.3, 8.7; 16 rows 11.4, 9.8, 9.5; 32 rows 17.1,
// 12.9, 11.7; 8192 x 8192, 1 row 10.4, 9.9, 12.4; 4096 x 4096, 1 row 4.8, 5.2, 7.3.)  The gated block has two of each, and with
// few rows the smaller x in return: 14336 x 4096, 1 row 14.0, 14.3; 8 rows 15.1, 14.9; 16 rows 16.8, 15.9; 32 rows 22.4, 19.0.
bool two_fragments(int n) { return n >= 2 * kRows * 256; }

SkinnyArgs arguments(const MxMatrix &x, const MxMatrix &w0, const MxMatrix &w1, int k)
{
    SkinnyArgs g{};
    g.x = x.codes;
    g.xs = x.scales;
    g.w0 = w0.codes;
    g.w0s = w0.scales;
    g.w1 = w1.codes;
    g.w1s = w1.scales;
    g.stride = mx_code_stride(k);
    g.scale_stride = mx_scale_stride(k);
    g.m = x.rows;
    g.n = w0.rows;
    g.lines = (k + kLineFp4 - 1) / kLineFp4;
    return g;
}

}  // namespace

hipError_t launch_mx_linear_skinny(const MxMatrix &x, const MxMatrix &w, const float *bias, void *y, int out, int k, hipStream_t stream)
{
    SkinnyArgs g = arguments(x, w, w, k);
    g.bias = bias;
    g.y = y;
    g.ld = (size_t)w.rows;
    g.out = out;
    return two_fragments(g.n) ? launch_rows<kPlain, 2>(g, g.n, stream) : launch_rows<kPlain, 1>(g, g.n, stream);
}

hipError_t launch_mx_gated_skinny(const MxMatrix &x, const MxMatrix &wg, const MxMatrix &wu, Activation act, void *h, int out, int k,
                                  hipStream_t stream)
{
    SkinnyArgs g = arguments(x, wg, wu, k);
    g.y = h;
    g.ld = (size_t)wg.rows;
    g.out = out;
    g.act = act;
    return two_fragments(g.n) && g.m > 4 ? launch_rows<kGated, 2>(g, g.n, stream) : launch_rows<kGated, 1>(g, g.n, stream);
}

hipError_t launch_mx_gated_quantized_skinny(const MxMatrix &x, const MxMatrix &wg, const MxMatrix &wu, Activation act, uint8_t *codes,
                                            uint8_t *scales, int k, hipStream_t stream)
{
    SkinnyArgs g = arguments(x, wg, wu, k);
    g.y = codes;
    g.y_scales = scales;
    g.ld = mx_code_stride(wg.rows);
    g.ld_scales = mx_scale_stride(wg.rows);
    g.act = act;
    return launch_rows<kGatedMx, 2>(g, (int)(g.ld * 2), stream);  // the padding too
}

}  // namespace int4linear
