// GEMM over lines of 128 bytes: MXFP4 operands (256 k per line, block scales applied by the matrix
// instruction) and bfloat16 operands (64 k per line), y = a b^T.
//
// Both element types share one kernel, because their matrix instructions take the same bytes from
// a lane: v_mfma_scale_f32_32x32x64_f8f6f4 on 4-bit operands and v_mfma_f32_32x32x16_bf16 both
// read 16 bytes of row lane % 32, and both run 32 cycles.  A stage is one line of every row of the tile; lane
// group lane / 32 takes chunk (16 bytes) 4 * (lane / 32) + j of its rows in step j = 0 .. 3, for a and b
// alike, which is all that a sum over k asks for.  With 4-bit operands a chunk is one block of 32, and the
// scales of the four chunks that a lane sees in a stage are the four bytes of one aligned dword.
#include "line_tiles.h"
#include "mxfp4.h"
#include "mxfp4_epilogue.h"

#include <type_traits>
#include <utility>

namespace int4linear {

namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef __bf16 v4bf __attribute__((ext_vector_type(4)));
typedef unsigned v2u __attribute__((ext_vector_type(2)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v4h __attribute__((ext_vector_type(4)));

constexpr int kFrag = 32;

// The operands.  A row is `stages` lines, `stride` bytes from the next, and with 4-bit values its scales, scale_stride
// bytes from the next, for a and b alike.  The gated block's two matrices b have as many rows each.
struct LineOperands {
    const uint8_t *a, *b0, *b1;
    const uint8_t *a_scales, *b0_scales, *b1_scales;
    unsigned stride, scale_stride;
    int a_rows, b_rows, stages;
};

// ---- what happens to a tile's sums ------------------------------------------------------------
// An epilogue is called once per wave as ep(acc, row, col, lane): acc[j][i] is the 32 x 32 block at rows
// row + 32 j of a and columns col + 32 i of the product.  Which operand the matrix instruction takes first decides
// what a lane holds of it:
//   kColumns = false: row lane % 32; element t is column 8 (t / 4) + 4 (lane / 32) + t % 4;
//   kColumns = true:  column lane % 32; element t is row 8 (t / 4) + 4 (lane / 32) + t % 4.
// 16-bit outputs whose rows are multiples of 16 bytes take the first: two lanes swap halves and each stores 16
// bytes.  All others take the second: a store covers 32 neighbouring elements of two rows, wherever they begin.
// kPair: two operands b share the tile, blocks i even of the first, odd of the second, each pair over the same
// 32 columns.

// Elements 8 * half .. of a lane's 16 columns of a row (kColumns = false), rounded to 16 bits -> 8 columns from
// 16 * half + 8 * (lane / 32) on.
template <int OUT>
__device__ __forceinline__ v4i gather_row(const float *v)
{
    using T = OutElement<OUT>;
    typedef T v2t __attribute__((ext_vector_type(2)));
    int p[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
        p[e] = __builtin_bit_cast(int, (v2t){(T)v[2 * e], (T)v[2 * e + 1]});
    const auto x = __builtin_amdgcn_permlane32_swap(p[0], p[2], false, false);
    const auto y = __builtin_amdgcn_permlane32_swap(p[1], p[3], false, false);
    return (v4i){(int)x[0], (int)y[0], (int)x[1], (int)y[1]};
}

// The 16 results v of a lane's part of a block of y (ld elements between rows) at (row, col).
template <int OUT, bool COLUMNS>
__device__ __forceinline__ void store_block(void *y, size_t ld, int m, int n, int row, int col, int lane, const float (&v)[16])
{
    using T = OutElement<OUT>;
    T *dst = (T *)y;
    if constexpr (COLUMNS) {
        const int c = col + (lane & 31), r0 = row + 4 * (lane >> 5);
        dst += (size_t)r0 * ld + c;
        if (c < n) {
#pragma unroll
            for (int t = 0; t < 16; ++t) {
                const int dr = 8 * (t / 4) + t % 4;
                if (r0 + dr < m)
                    dst[(size_t)dr * ld] = (T)v[t];
            }
        }
    } else {
        const v4i out[2] = {gather_row<OUT>(v), gather_row<OUT>(v + 8)};
        const int r = row + (lane & 31), c = col + 8 * (lane >> 5);
        dst += (size_t)r * ld + c;
        if (r < m) {  // (n is a multiple of 8)
            if (c < n)
                *(v4i *)dst = out[0];
            if (c + 16 < n)
                *(v4i *)(dst + 16) = out[1];
        }
    }
}

// y = sums + bias, rounded once to OUT.
template <int OUT, bool COLUMNS>
struct PlainEpilogue {
    static constexpr bool kPair = false, kColumns = COLUMNS;
    void *y;
    const float *bias;
    size_t ld;
    int m, n;

    template <int FM, int FN>
    __device__ __forceinline__ void operator()(v16f (&acc)[FM][FN], int row, int col, int lane) const
    {
#pragma unroll
        for (int i = 0; i < FN; ++i) {
            const int c = col + kFrag * i;
            float add[16];
#pragma unroll
            for (int t = 0; t < 16; ++t)
                add[t] = 0.0f;
            if (bias) {
                if constexpr (COLUMNS) {
                    const float b = bias[min(c + (lane & 31), n - 1)];
#pragma unroll
                    for (int t = 0; t < 16; ++t)
                        add[t] = b;
                } else {
#pragma unroll
                    for (int t = 0; t < 16; ++t)
                        add[t] = bias[min(c + 8 * (t / 4) + 4 * (lane >> 5) + t % 4, n - 1)];
                }
            }
#pragma unroll
            for (int j = 0; j < FM; ++j) {
                float v[16];
#pragma unroll
                for (int t = 0; t < 16; ++t)
                    v[t] = acc[j][i][t] + add[t];
                store_block<OUT, COLUMNS>(y, ld, m, n, row + kFrag * j, c, lane, v);
            }
        }
    }
};

// h = act(g) * u, rounded once to OUT.
template <int OUT, bool COLUMNS>
struct GatedEpilogue {
    static constexpr bool kPair = true, kColumns = COLUMNS;
    void *h;
    size_t ld;
    int m, n, act;

    template <int FM, int FN>
    __device__ __forceinline__ void operator()(v16f (&acc)[FM][FN], int row, int col, int lane) const
    {
#pragma unroll
        for (int j = 0; j < FM; ++j)
#pragma unroll
            for (int i = 0; i < FN; i += 2) {
                float v[16];
#pragma unroll
                for (int t = 0; t < 16; ++t)
                    v[t] = activate(act, acc[j][i][t]) * acc[j][i + 1][t];
                store_block<OUT, COLUMNS>(h, ld, m, n, row + kFrag * j, col + kFrag * (i / 2), lane, v);
            }
    }
};

// The same in MXFP4: a block of 32 columns of a row sits in lanes l and l + 32.
struct GatedMxEpilogue {
    static constexpr bool kPair = true, kColumns = false;
    uint8_t *codes, *scales;
    size_t code_stride, scale_stride;
    int m, n, act;

    template <int FM, int FN>
    __device__ __forceinline__ void operator()(v16f (&acc)[FM][FN], int row, int col, int lane) const
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
                const auto both = __builtin_amdgcn_permlane32_swap(big, big, false, false);
                big = max(both[0], both[1]);
                unsigned code, bits[2];
                bits[0] = encode_block_part({v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]}, big, code);
                bits[1] = encode_block_part({v[8], v[9], v[10], v[11], v[12], v[13], v[14], v[15]}, big, code);
                // bits[h]: 16 bits for columns 16 h + 4 (lane / 32) .., 16 for those 8 further on.  The lane pair's four words
                // make dwords 2 h and 2 h + 1 of the block; the lower lane takes h = 0, the upper h = 1.
                const auto x = __builtin_amdgcn_permlane32_swap(bits[0], bits[1], false, false);
                const unsigned lo = (x[0] & 0xFFFFu) | (x[1] << 16), hi = (x[0] >> 16) | (x[1] & 0xFFFF0000u);
                if (r < m && (size_t)c0 < code_stride * 2) {
                    *(unsigned long long *)(codes + (size_t)r * code_stride + c0 / 2 + 8 * (lane >> 5)) =
                        lo | ((unsigned long long)hi << 32);
                    if (lane < 32)
                        store_block_scale(scales + (size_t)r * scale_stride, c0, code_stride, code);
                }
            }
        }
    }
};

// dg = dh * u * act'(g), du = dh * act(g), rounded to bfloat16: they are the operands of two more products
// on matrix cores that take 16 bits; the roundings of the terms (2^-8 at most, of random sign) add up to as much as
// the rounding of the result itself.
struct GradientEpilogue {
    static constexpr bool kPair = true, kColumns = false;
    const __bf16 *dh;
    __bf16 *d, *dt;
    size_t ld_n, ld_m;
    int m, n, act;
    bool vec;  // dh's rows are multiples of 8 bytes

    template <int FM, int FN>
    __device__ __forceinline__ void operator()(v16f (&acc)[FM][FN], int row, int col, int lane) const
    {
        // (All loads first, where there are registers for them: behind one another they cost a way to memory each.)
        constexpr bool kAhead = FM * FN > 4;
        v4bf in[FM][FN / 2][4];
        auto fetch = [&](int j, int i, int q) {
            const int r = row + kFrag * j + (lane & 31), c = col + kFrag * i + 8 * q + 4 * (lane >> 5);
            in[j][i][q] = (v4bf){};
            if (r < m) {
                const __bf16 *src = dh + (size_t)r * n + c;
                if (vec) {
                    if (c < n)
                        in[j][i][q] = *(const v4bf *)src;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (c + e < n)
                            in[j][i][q][e] = src[e];
                }
            }
        };
        if constexpr (kAhead) {
#pragma unroll
            for (int j = 0; j < FM; ++j)
#pragma unroll
                for (int i = 0; i < FN / 2; ++i)
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        fetch(j, i, q);
        }
#pragma unroll
        for (int j = 0; j < FM; ++j) {
            const int r = row + kFrag * j + (lane & 31);
#pragma unroll
            for (int i = 0; i < FN; i += 2) {
                const int c0 = col + kFrag * (i / 2);
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    float dg[8], du[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int t = 8 * half + e;
                        if (!kAhead && t % 4 == 0)
                            fetch(j, i / 2, t / 4);
                        float value, slope;
                        activate_with_slope(act, acc[j][i][t], value, slope);
                        // padding: exact zeros, whatever the clamped rows gave
                        const bool there = r < m && c0 + 8 * (t / 4) + 4 * (lane >> 5) + t % 4 < n;
                        const float g = (float)in[j][i / 2][t / 4][t % 4];
                        dg[e] = there ? g * acc[j][i + 1][t] * slope : 0.0f;
                        du[e] = there ? g * value : 0.0f;
                    }
                    const v4i g8 = gather_row<kOutBF16>(dg), u8 = gather_row<kOutBF16>(du);
                    const int c = c0 + 16 * half + 8 * (lane >> 5);
                    if (r < m && (size_t)c < ld_n) {
                        __bf16 *to = d + (size_t)r * 2 * ld_n + c;
                        *(v4i *)to = g8;
                        *(v4i *)(to + ld_n) = u8;
                    }
                    if ((size_t)r < ld_m) {
                        store_transposed(dt, r, c0 + 16 * half, lane, dg);
                        store_transposed(dt + (size_t)n * ld_m, r, c0 + 16 * half, lane, du);
                    }
                }
            }
        }
    }

    // The transposes.  A quad's 4 rows x 4 columns change places, twice: between neighbours, then between pairs.  A lane then has four rows of
    // column lane % 4 of each four: 8 bytes a store.  (With stores of 2 bytes, and dh fetched block by block, 4096 x 14336 x 4096 takes
    // 466 us, so 400; the product alone with h as its result 275.)
    __device__ __forceinline__ void store_transposed(__bf16 *to, int r, int c0, int lane, const float (&v)[8]) const
    {
        const unsigned halves = lane & 1 ? 0x03020706u : 0x05040100u;
        const bool upper = lane & 2;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            unsigned two[2];  // rows r & ~1, r | 1 of column 2 i + lane % 2 of the four
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const unsigned own = __builtin_bit_cast(unsigned, (v2bf){(__bf16)v[4 * q + 2 * i], (__bf16)v[4 * q + 2 * i + 1]});
                two[i] = __builtin_amdgcn_perm((unsigned)__builtin_amdgcn_mov_dpp((int)own, 0xB1, 0xF, 0xF, true), own, halves);
            }
            const unsigned kept = upper ? two[1] : two[0];
            const unsigned got = (unsigned)__builtin_amdgcn_mov_dpp((int)(upper ? two[0] : two[1]), 0x4E, 0xF, 0xF, true);
            const int c = c0 + 8 * q + 4 * (lane >> 5) + (lane & 3);
            if (c < n)
                *(v2u *)(to + (size_t)c * ld_m + (r & ~3)) = upper ? (v2u){got, kept} : (v2u){kept, got};
        }
    }
};

// ---- the kernel -------------------------------------------------------------------------------

constexpr int kChunkRows = 8;    // rows of a 1-KiB load
constexpr int kScaleStages = 2;  // stages whose scales are 16 bytes of a row
constexpr int kSteps = 4;        // steps of a stage

// WAVES_M x WAVES_N wavefronts multiply, each FM x FN blocks of 32 x 32; LOADERS more load for them (0: each of the
// others loads its share); STAGES stages in LDS; operands are read AHEAD steps ahead; OCC waves per SIMD.
template <int WAVES_M_, int WAVES_N_, int FM_, int FN_, int LOADERS_, int STAGES_, int AHEAD_, int OCC_>
struct LineTile {
    static constexpr int AHEAD = AHEAD_, SETS = AHEAD == 1 ? 2 : 4;  // register sets of a step's operands
    static constexpr int WAVES_M = WAVES_M_, WAVES_N = WAVES_N_, FM = FM_, FN = FN_, LOADERS = LOADERS_, STAGES = STAGES_, OCC = OCC_;
    static constexpr int NWAVES = WAVES_M * WAVES_N, THREADS = (NWAVES + LOADERS) * 64;
    static constexpr int LOADING = LOADERS ? LOADERS : NWAVES;    // waves that load
    static constexpr int BM = WAVES_M * FM * kFrag, BN = WAVES_N * FN * kFrag;
    static constexpr int STAGE = (BM + BN) * kLineBytes;
    static constexpr int SCALES = (BM + BN) * 16;                 // scales of two stages
    template <bool FP4>
    static constexpr int LDS = STAGES * (STAGE + (FP4 ? SCALES : 0));
    static constexpr int A_CH = BM / kChunkRows / LOADING, B_CH = BN / kChunkRows / LOADING;  // loads per wave and stage
    static constexpr int SLOTS = FM * FN;                         // matrix instructions per step
    static_assert(BM % (kChunkRows * LOADING) == 0 && BN % (kChunkRows * LOADING) == 0 && LOADING % 2 == 0 && BM % 64 == 0 && BN % 64 == 0);
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

// Marks a value as used at this point of the program without generating code.
__device__ __forceinline__ void pin(const v16f &v) { asm volatile("" ::"v"(v)); }

// Sums without a single term: y = bias.
template <int OUT>
__global__ __launch_bounds__(256) void fill_rows_kernel(void *y, const float *bias, size_t count, size_t n)
{
    for (size_t at = (size_t)blockIdx.x * 256 + threadIdx.x; at < count; at += (size_t)gridDim.x * 256) {
        ((OutElement<OUT> *)y)[at] = (OutElement<OUT>)(bias ? bias[at % n] : 0.0f);
    }
}

template <int OUT>
hipError_t fill_rows(void *y, const float *bias, size_t m, size_t n, hipStream_t stream)
{
    const size_t groups = (m * n + 255) / 256;
    fill_rows_kernel<OUT><<<(unsigned)(groups < 4096 ? groups : 4096), 256, 0, stream>>>(y, bias, m * n, n);
    return hipGetLastError();
}

// Persistent: a workgroup walks tiles first, first + by, ... and its loads run ahead of the
// arithmetic across the ends of tiles.  With the smaller tiles four waves of their own do the loading: a load holds up the
// wave that issues it, and these tiles have fewer matrix instructions to hide that behind (64 x 128 tiles, four loaders
// against none: 512 x 4096 x 11008 23.6 us and 26.2; 64 x 4096 x 4096 8.6 and 10.5).  The 256 x 256 tile has no registers left
// for more waves.  STAGES stages ring in LDS.  A stage is four steps of FM x FN matrix
// instructions; while a step's instructions run, those of the step AHEAD further on are read from LDS into another register
// set.  Before a stage's AHEAD last steps every read of the stage has been made: there the waves meet, the next stage must
// have landed (younger ones stay in flight), and the stage's buffer is given to the loads of the stage STAGES further on.
template <bool FP4, class C, class Ep>
__device__ __forceinline__ void line_gemm(const LineOperands &o, int tiles_m, int tiles_n, const Ep &ep, int first, int by)
{
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / C::WAVES_N, wn = wave % C::WAVES_N;
    const int total = tiles_m * tiles_n;
    const int my_tiles = (total - first + by - 1) / by;
    const uint8_t *a_data = o.a;
    const int stages = o.stages;
    constexpr int kTileN = Ep::kPair ? C::BN / 2 : C::BN;  // columns of y

    v16f acc[C::FM][C::FN];
    auto clear = [&] {
#pragma unroll
        for (int j = 0; j < C::FM; ++j)
#pragma unroll
            for (int i = 0; i < C::FN; ++i)
                acc[j][i] = (v16f)0.0f;
    };
    auto finish = [&](int it) {
        int tm, tn;
        tile_coords(first + it * by, total, tiles_m, tiles_n, tm, tn);
        ep(acc, tm * C::BM + wm * C::FM * kFrag, tn * kTileN + wn * C::FN * kFrag / (Ep::kPair ? 2 : 1), lane);
        clear();
    };
    clear();

    // ---- loads.  Load c of loading wave l fills LDS rows 8 (c * LOADING + l) .. + 7 of its operand's part of a
    // stage, each lane the 16 bytes at place lane % 8 of row lane / 8.  The chunk that lies at place p of row r is
    // p ^ (r / 2 % 8): the 16 lanes that an LDS read serves together then touch every bank once.
    const unsigned lds_base = (unsigned)(size_t)I4L_LDS(lds);
    const int loader = C::LOADERS ? wave - C::NWAVES : wave;
    const int ld_row = loader * kChunkRows + (lane >> 3);
    const unsigned ld_chunk = (unsigned)(((lane & 7) ^ ((ld_row >> 1) & 7)) * 16);
    const uint8_t *a_base = nullptr, *b_base[2] = {};  // this tile's rows, this stage's line
    unsigned a_off[C::A_CH], b_off[C::B_CH];
    // FP4: loads of scales, 64 rows each; a wave's are rows 64 (c * LOADING + l) .. of the stage
    constexpr int kScaleLoads = (C::BM + C::BN) / 64, kMyScales = (kScaleLoads + C::LOADING - 1) / C::LOADING;
    const uint8_t *scale_at[kMyScales] = {};
    int ld_it = 0, ld_s = 0;
    unsigned ld_buffer = 0, ld_slot = 0;

    // Matrix and row (of the tile) of LDS row r of b's part.
    auto b_row = [](int r) { return Ep::kPair ? r / (2 * kFrag) * kFrag + r % kFrag : r; };
    auto b_second = [](int r) { return Ep::kPair && (r / kFrag) % 2 != 0; };

    auto ld_tile = [&](int it) {
        int tm, tn;
        tile_coords(first + it * by, total, tiles_m, tiles_n, tm, tn);
        const int m0 = tm * C::BM, n0 = tn * kTileN;
        a_base = uniform(a_data + (size_t)m0 * o.stride);
        // rows behind the matrix: the last one again
        const int last_a = o.a_rows - 1 - m0, last_b = o.b_rows - 1 - n0;
#pragma unroll
        for (int c = 0; c < C::A_CH; ++c)
            a_off[c] = (unsigned)min(c * C::LOADING * kChunkRows + ld_row, last_a) * o.stride + ld_chunk;
        // (last_b is negative where h's padding alone is in the tile: then the matrix's last row)
        const int nb = min(n0, o.b_rows - 1);
        b_base[0] = uniform(o.b0 + (size_t)nb * o.stride);
        b_base[1] = uniform(o.b1 + (size_t)nb * o.stride);
#pragma unroll
        for (int c = 0; c < C::B_CH; ++c)
            b_off[c] = (unsigned)max(min(b_row(c * C::LOADING * kChunkRows + ld_row), last_b), 0) * o.stride + ld_chunk;
        if constexpr (FP4) {
#pragma unroll
            for (int c = 0; c < kMyScales; ++c) {
                const int r = (c * C::LOADING + loader) * 64 + lane;
                if (r < C::BM) {
                    scale_at[c] = o.a_scales + (size_t)(m0 + min(r, last_a)) * o.scale_stride;
                } else {
                    const int br = r - C::BM;
                    scale_at[c] = (b_second(br) ? o.b1_scales : o.b0_scales) + (size_t)(nb + max(min(b_row(br), last_b), 0)) * o.scale_stride;
                }
            }
        }
    };
    constexpr int kLoads = C::A_CH + C::B_CH;
    auto load = [&](int c) {
        const unsigned to = lds_base + ld_buffer + (unsigned)loader * 1024u;
        if (c < C::A_CH)
            dma16(a_base, a_off[c], to + (unsigned)(c * C::LOADING) * 1024u);
        else
            dma16(b_base[b_second(((c - C::A_CH) * C::LOADING + loader) * kChunkRows)], b_off[c - C::A_CH],
                  to + (unsigned)(C::BM * kLineBytes) + (unsigned)((c - C::A_CH) * C::LOADING) * 1024u);
    };
    auto next_in_ring = [](unsigned at, unsigned step) { return at == (C::STAGES - 1) * step ? 0u : at + step; };
    // After a stage's loads: its scales, if they are not there already, and on to the next stage.  Behind the
    // last stage the cursor stays: it is loaded again, into buffers that nobody reads.
    auto load_rest = [&] {
        if constexpr (FP4) {
            if (ld_s % kScaleStages == 0) {
#pragma unroll
                for (int c = 0; c < kMyScales; ++c)
                    if (kScaleLoads % C::LOADING == 0 || c * C::LOADING + loader < kScaleLoads)
                        dma16(scale_at[c], lds_base + C::STAGES * C::STAGE + ld_slot + (unsigned)(c * C::LOADING + loader) * 1024u);
            }
        }
        ld_buffer = next_in_ring(ld_buffer, C::STAGE);
        if (ld_s + 1 < stages) {
            ++ld_s;
            a_base += kLineBytes;
            b_base[0] += kLineBytes;
            b_base[1] += kLineBytes;
            if (FP4 && ld_s % kScaleStages == 0) {
#pragma unroll
                for (int c = 0; c < kMyScales; ++c)
                    scale_at[c] += 16;
                ld_slot = next_in_ring(ld_slot, C::SCALES);
            }
        } else if (ld_it + 1 < my_tiles) {
            ld_s = 0;
            ld_slot = next_in_ring(ld_slot, C::SCALES);
            ld_tile(++ld_it);
        }
    };
    // All but the youngest IN_FLIGHT stages have landed, this wave's reads are done, and every wave is here.  (Loads
    // complete in order; scales and stores in between only make the wait a little longer.)
    auto meet = [&](auto in_flight) {
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" : : "n"(decltype(in_flight)::value * kLoads) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    auto meet_without_loads = [&] {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    static_assert((C::STAGES - 1) * kLoads <= 63);

    if (C::LOADERS == 0 || wave >= C::NWAVES) {
        ld_tile(0);
#pragma unroll
        for (int st = 0; st < C::STAGES; ++st) {
#pragma unroll
            for (int c = 0; c < kLoads; ++c)
                load(c);
            load_rest();
        }
        meet(std::integral_constant<int, C::STAGES - 1>{});
        if constexpr (C::LOADERS != 0) {
            for (int left = my_tiles * stages; left > 0; --left) {
                meet(std::integral_constant<int, C::STAGES - 2>{});
#pragma unroll
                for (int c = 0; c < kLoads; ++c)
                    load(c);
                load_rest();
            }
            // (loads into buffers that nobody reads may be in flight: they end before the LDS is given away)
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            return;
        }
    } else {
        meet_without_loads();
    }

    // ---- arithmetic
    const int fr = lane & 31, fg = lane >> 5;
    unsigned chunk_at[kSteps];
#pragma unroll
    for (int J = 0; J < kSteps; ++J)
        chunk_at[J] = (unsigned)(((kSteps * fg + J) ^ ((fr >> 1) & 7)) * 16 + fr * kLineBytes);
    const unsigned a_rd = (unsigned)(wm * C::FM * kFrag * kLineBytes);
    const unsigned b_rd = (unsigned)((C::BM + wn * C::FN * kFrag) * kLineBytes);
    const unsigned as_rd = (unsigned)(C::STAGES * C::STAGE + (wm * C::FM * kFrag + fr) * 16 + 4 * fg);
    const unsigned bs_rd = (unsigned)(C::STAGES * C::STAGE + (C::BM + wn * C::FN * kFrag + fr) * 16 + 4 * fg);
    v4i fa[C::SETS][C::FM], fb[C::SETS][C::FN];
    int sa[2][C::FM] = {}, sb[2][C::FN] = {};

    // Operand r of step J of the stage in `buffer`, into register set p.
    constexpr int kReads = C::FM + C::FN;
    auto read = [&](unsigned buffer, int J, int p, int r) {
        const uint8_t *at = lds + (buffer + chunk_at[J]);
        if (r < C::FM)
            fa[p][r] = *(const v4i *)(at + a_rd + r * kFrag * kLineBytes);
        else
            fb[p][r - C::FM] = *(const v4i *)(at + b_rd + (r - C::FM) * kFrag * kLineBytes);
    };
    auto read_scales = [&](unsigned slot, int s, int p) {
        if constexpr (FP4) {
            const uint8_t *at = lds + (slot + 8 * (s % kScaleStages));
#pragma unroll
            for (int j = 0; j < C::FM; ++j)
                sa[p][j] = *(const int *)(at + as_rd + j * kFrag * 16);
#pragma unroll
            for (int i = 0; i < C::FN; ++i)
                sb[p][i] = *(const int *)(at + bs_rd + i * kFrag * 16);
        }
    };
    // The matrix instructions of step J, `behind` called after each with its number.
    auto step = [&](auto j_tag, auto &&behind) {
        constexpr int J = decltype(j_tag)::value, p = J % C::SETS;
        [&]<int... SLOT>(std::integer_sequence<int, SLOT...>) {
            ([&] {
                constexpr int j = SLOT / C::FN, i = SLOT % C::FN;
                if constexpr (FP4) {
                    const v8i wide_a = {fa[p][j][0], fa[p][j][1], fa[p][j][2], fa[p][j][3], 0, 0, 0, 0};
                    const v8i wide_b = {fb[p][i][0], fb[p][i][1], fb[p][i][2], fb[p][i][3], 0, 0, 0, 0};
                    if constexpr (Ep::kColumns)
                        acc[j][i] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wide_a, wide_b, acc[j][i], 4, 4, J, sa[0][j], J, sb[0][i]);
                    else
                        acc[j][i] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wide_b, wide_a, acc[j][i], 4, 4, J, sb[0][i], J, sa[0][j]);
                } else {
                    const v8bf wide_a = __builtin_bit_cast(v8bf, fa[p][j]), wide_b = __builtin_bit_cast(v8bf, fb[p][i]);
                    if constexpr (Ep::kColumns)
                        acc[j][i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wide_a, wide_b, acc[j][i], 0, 0, 0);
                    else
                        acc[j][i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wide_b, wide_a, acc[j][i], 0, 0, 0);
                }
                pin(acc[j][i]);
                __builtin_amdgcn_sched_barrier(0);
                behind(std::integral_constant<int, SLOT>{});
                __builtin_amdgcn_sched_barrier(0);
            }(), ...);
        }(std::make_integer_sequence<int, C::SLOTS>{});
    };
    constexpr int kReadsPerSlot = (kReads + C::SLOTS - 1) / C::SLOTS;
    constexpr int kLoadsPerSlot = (kLoads + C::SLOTS - 1) / C::SLOTS;

#pragma unroll
    for (int J = 0; J < C::AHEAD; ++J)
#pragma unroll
        for (int r = 0; r < kReads; ++r)
            read(0, J, J, r);
    read_scales(0, 0, 1);

    unsigned buffer = 0, slot = 0;
    int it = 0, s = 0;
    while (true) {
        if constexpr (FP4) {
#pragma unroll
            for (int j = 0; j < C::FM; ++j)
                sa[0][j] = sa[1][j];
#pragma unroll
            for (int i = 0; i < C::FN; ++i)
                sb[0][i] = sb[1][i];
        }
        const bool last = s + 1 == stages;
        const int next_s = last ? 0 : s + 1;
        const unsigned next_buffer = next_in_ring(buffer, C::STAGE);
        [&]<int... J>(std::integer_sequence<int, J...>) {
            ([&] {
                if constexpr (J == kSteps - C::AHEAD) {
                    if constexpr (C::LOADERS == 0)
                        meet(std::integral_constant<int, C::STAGES - 2>{});
                    else
                        meet_without_loads();
                    if (FP4 && next_s % kScaleStages == 0)
                        slot = next_in_ring(slot, C::SCALES);
                    read_scales(slot, next_s, 1);
                }
                step(std::integral_constant<int, J>{}, [&](auto slot_tag) {
                    constexpr int at = decltype(slot_tag)::value * kReadsPerSlot, then = J + C::AHEAD;
#pragma unroll
                    for (int r = at; r < at + kReadsPerSlot && r < kReads; ++r)
                        read(then < kSteps ? buffer : next_buffer, then % kSteps, then % C::SETS, r);
                    if constexpr (C::LOADERS == 0 && J == kSteps - 1) {
                        constexpr int load_at = decltype(slot_tag)::value * kLoadsPerSlot;
#pragma unroll
                        for (int c = load_at; c < load_at + kLoadsPerSlot && c < kLoads; ++c)
                            load(c);
                    }
                });
            }(), ...);
        }(std::make_integer_sequence<int, kSteps>{});
        if constexpr (C::LOADERS == 0)
            load_rest();
        buffer = next_buffer;
        s = next_s;
        if (last) {
            finish(it);
            if (++it == my_tiles)
                break;
        }
    }
    // (loads into buffers that nobody reads may be in flight: they end before the workgroup's LDS is given away)
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

template <bool FP4, class C, class Ep>
__global__ __launch_bounds__(C::THREADS, C::OCC) void line_gemm_kernel(LineOperands o, int tiles_m, int tiles_n, Ep ep)
{
    line_gemm<FP4, C>(o, tiles_m, tiles_n, ep, blockIdx.x, gridDim.x);
}

// Up to three products in one launch, by blockIdx.z: those of a small layer's backward pass, each of which would leave
// most CUs idle.  A workgroup makes one slice of one tile of 64 x 64: slice blockIdx.x % slices of stages
// slice * stages / slices on.  The last product is dx; the others, the weights', share a type.
struct LineGroup {
    LineOperands o[3];
    int tiles_m[3], tiles_n[3], slices[3];
    void *y[3];
    int first[3];  // number of a product's first tile-slice and, times waves, of its first counter
    int count;
    float *partial;      // sums of a tile-slice: 64 x 64 floats
    unsigned *arrivals;  // counters, zero before the launch
    // Column sums to be completed on the way (sums null: none): of `parts` rows of partial sums.
    float *sums;
    const float *sum_parts;
    int parts, columns;
};

// An epilogue behind sums that are one of `slices` shares: every wave leaves its share, waits until that has been acknowledged
// and counts itself in.  The last of a tile's waves of one number to arrive adds all shares up in the order of their
// slices, whoever came when, and goes on to the epilogue; nobody waits for anybody.  (Relaxed atomic operations at device scope go
// through to the level that all XCDs share.)
template <class Ep>
struct SliceEpilogue {
    static constexpr bool kPair = Ep::kPair, kColumns = Ep::kColumns;
    Ep ep;
    float *partial;     // of this tile's slice 0, wave 0
    unsigned *arrived;  // of this tile's wave 0
    int slice, slices;

    __device__ __forceinline__ void operator()(v16f (&acc)[1][1], int row, int col, int lane) const
    {
        typedef unsigned long long u64;
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        if (slices > 1) {
            constexpr int kSlice = 64 * 64 / 2, kWords = 8;  // words of two floats, of a slice and of a lane
            u64 *mine = (u64 *)partial + (size_t)wave * kWords * 64 + lane;
            float v[16];
#pragma unroll
            for (int t = 0; t < 16; ++t)
                v[t] = acc[0][0][t];
#pragma unroll
            for (int i = 0; i < kWords; ++i)
                __hip_atomic_store(mine + (size_t)slice * kSlice + i * 64, __builtin_bit_cast(u64, (v2f){v[2 * i], v[2 * i + 1]}),
                                   __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            int before = 0;
            if (lane == 0)
                before = (int)__hip_atomic_fetch_add(arrived + wave, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            if (__builtin_amdgcn_readfirstlane(before) != slices - 1)
                return;
            asm volatile("" ::: "memory");
#pragma unroll
            for (int t = 0; t < 16; ++t)
                v[t] = 0.0f;
            for (int from = 0; from < slices; ++from) {
                u64 got[kWords];
#pragma unroll
                for (int i = 0; i < kWords; ++i)
                    got[i] = __hip_atomic_load(mine + (size_t)from * kSlice + i * 64, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
                for (int i = 0; i < kWords; ++i) {
                    const v2f pair = __builtin_bit_cast(v2f, got[i]);
                    v[2 * i] += pair[0];
                    v[2 * i + 1] += pair[1];
                }
            }
#pragma unroll
            for (int t = 0; t < 16; ++t)
                acc[0][0][t] = v[t];
        }
        ep(acc, row, col, lane);
    }
};

__device__ __forceinline__ void complete_sums(float *sums, const float *partial, int parts, int columns, int first, int by)
{
    for (int c = first; c < columns; c += by) {
        float sum[4] = {};  // in the order of column_sums_kernel
        for (int i = 0; i < parts; i += 4)
#pragma unroll
            for (int w = 0; w < 4; ++w)
                if (i + w < parts)
                    sum[w] += partial[(size_t)(i + w) * columns + c];
        sums[c] = ((sum[0] + sum[1]) + sum[2]) + sum[3];
    }
}

template <class C, class EpW, class EpX>
__global__ __launch_bounds__(C::THREADS, C::OCC) void line_group_kernel(LineGroup g, EpW ep_w, EpX ep_x)
{
    const int z = blockIdx.z;
    if (g.sums && z == 0)
        complete_sums(g.sums, g.sum_parts, g.parts, g.columns, blockIdx.x * C::THREADS + threadIdx.x, gridDim.x * C::THREADS);
    const int tiles = g.tiles_m[z] * g.tiles_n[z], slices = g.slices[z];
    const int tile = (int)blockIdx.x / slices, slice = (int)blockIdx.x % slices;
    if (tile >= tiles)
        return;
    LineOperands o = g.o[z];
    const int from = (int)((long)slice * o.stages / slices), to = (int)((long)(slice + 1) * o.stages / slices);
    o.a += (size_t)from * kLineBytes;
    o.b0 += (size_t)from * kLineBytes;
    o.b1 = o.b0;
    o.stages = to - from;
    auto run = [&](auto ep) {
        ep.y = g.y[z];
        ep.m = o.a_rows;
        const SliceEpilogue<decltype(ep)> shared{ep, g.partial + (size_t)(g.first[z] + tile * slices) * 64 * 64,
                                                 g.arrivals + (g.first[z] + tile * slices) * C::NWAVES, slice, slices};
        line_gemm<false, C>(o, g.tiles_m[z], g.tiles_n[z], shared, tile, tiles);
    };
    if (z == g.count - 1)
        run(ep_x);
    else
        run(ep_w);
}

using Tile256 = LineTile<4, 2, 2, 4, 0, 2, 1, 2>;
using Tile128 = LineTile<2, 2, 2, 2, 4, 2, 1, 4>;
using Tile64x128 = LineTile<2, 2, 1, 2, 4, 3, 2, 4>;
using Tile64 = LineTile<2, 2, 1, 1, 4, 4, 2, 4>;  // (too narrow for pairs of blocks)

// Workgroups of a tile that a CU's LDS holds.
template <class C, bool FP4>
constexpr int per_cu = 160 * 1024 / C::template LDS<FP4>;

template <bool FP4, class C, class Ep>
hipError_t launch_tile(const LineOperands &o, int n, const Ep &ep, const DeviceInfo &dev, hipStream_t stream)
{
    const int bn = Ep::kPair ? C::BN / 2 : C::BN;
    const int tiles_m = (o.a_rows + C::BM - 1) / C::BM, tiles_n = (n + bn - 1) / bn;
    const int groups = min(tiles_m * tiles_n, max(1, dev.cu_count * per_cu<C, FP4>));
    line_gemm_kernel<FP4, C, Ep><<<groups, C::THREADS, C::template LDS<FP4>, stream>>>(o, tiles_m, tiles_n, ep);
    return hipGetLastError();
}

template <class C>
constexpr bool described_by(const LineTileCost &t)
{
    return t.m == C::BM && t.n == C::BN && t.lds[0] == C::template LDS<false> && t.lds[1] == C::template LDS<true>;
}
static_assert(described_by<Tile256>(kLineTiles[0]) && described_by<Tile128>(kLineTiles[1]) && described_by<Tile64x128>(kLineTiles[2]) &&
              described_by<Tile64>(kLineTiles[3]));

// n: columns of the product that have to be covered.
template <bool FP4, class Ep>
hipError_t launch(const LineOperands &o, int n, const Ep &ep, const DeviceInfo &dev, hipStream_t stream)
{
    switch (quickest_tile(FP4, o.a_rows, (long)n * (Ep::kPair ? 2 : 1), o.stages, Ep::kPair, dev.cu_count)) {
    case 0:
        return launch_tile<FP4, Tile256>(o, n, ep, dev, stream);
    case 1:
        return launch_tile<FP4, Tile128>(o, n, ep, dev, stream);
    case 2:
        return launch_tile<FP4, Tile64x128>(o, n, ep, dev, stream);
    default:
        if constexpr (Ep::kPair)
            return hipErrorInvalidValue;
        else
            return launch_tile<FP4, Tile64>(o, n, ep, dev, stream);
    }
}

LineOperands operands(const MxMatrix &x, const MxMatrix &w0, const MxMatrix &w1, int k)
{
    return {x.codes, w0.codes, w1.codes, x.scales, w0.scales, w1.scales, (unsigned)mx_code_stride(k), (unsigned)mx_scale_stride(k),
            x.rows, w0.rows, (k + kLineFp4 - 1) / kLineFp4};
}

// Up to here the weight-streaming kernel.  us streaming and on tiles, weights from HBM (from the caches streaming takes up to a fifth
// less, tiles up to a third):
//   rows of x            4           16          17          32          48
//   4096 x 4096          4.7, 7.7    5.3, 8.1    5.8, 8.1    6.6, 8.7    8.8, 9.2
//   4096 x 14336         7.9, 18.8   10.9, 20.5  12.0, 20.6  14.6, 22.2  23.1, 23.8
//   8192 x 8192          10.2, 13.4  10.6, 13.5  11.4, 13.6  13.1, 14.7  21.6, 15.4
//   14336 x 4096         8.7, 8.8    9.7, 9.2    10.6, 9.3   12.6, 9.9   19.0, 10.4
//   14336 x 4096, gated  14.0, 15.3  15.7, 15.6  16.7, 15.7  18.9, 16.1  29.9, 16.6
// Weights that give the device few tiles are streamed faster up to 48 rows, those that fill it up to 16: one line for both costs the
// second up to a quarter at 32 rows.
constexpr int kSkinnyRows = 32;

// f(type, columns) with the output type of a call and the epilogue's form for rows of n elements.
template <class F>
hipError_t by_type(int out, int n, F &&f)
{
    if (out == kOutF32)
        return f(std::integral_constant<int, kOutF32>{}, std::true_type{});
    if (out == kOutF16)
        return n % 8 ? f(std::integral_constant<int, kOutF16>{}, std::true_type{}) : f(std::integral_constant<int, kOutF16>{}, std::false_type{});
    return n % 8 ? f(std::integral_constant<int, kOutBF16>{}, std::true_type{}) : f(std::integral_constant<int, kOutBF16>{}, std::false_type{});
}

}  // namespace

// Lets the kernels of an epilogue have their LDS.
template <bool FP4, class Ep>
static hipError_t allow_lds()
{
    hipError_t e = hipSuccess;
    auto allow = [&](auto tile) {
        using C = decltype(tile);
        if (e == hipSuccess)
            e = hipFuncSetAttribute((const void *)line_gemm_kernel<FP4, C, Ep>, hipFuncAttributeMaxDynamicSharedMemorySize, C::template LDS<FP4>);
    };
    allow(Tile256{});
    allow(Tile128{});
    allow(Tile64x128{});
    if constexpr (!Ep::kPair)
        allow(Tile64{});
    return e;
}

template <class EpW, class EpX>
static hipError_t allow_group_lds()
{
    return hipFuncSetAttribute((const void *)line_group_kernel<Tile64, EpW, EpX>, hipFuncAttributeMaxDynamicSharedMemorySize,
                               Tile64::LDS<false>);
}

hipError_t line_gemm_init(const DeviceInfo &)
{
    hipError_t e = hipSuccess;
    using Columns32 = PlainEpilogue<kOutF32, true>;
    using Columns16 = PlainEpilogue<kOutBF16, true>;
    using Rows16 = PlainEpilogue<kOutBF16, false>;
    for (auto allow : {allow_group_lds<Columns32, Columns16>, allow_group_lds<Columns32, Rows16>, allow_group_lds<Columns16, Columns16>,
                       allow_group_lds<Rows16, Rows16>})
        if (e == hipSuccess)
            e = allow();
    for (auto allow : {allow_lds<true, PlainEpilogue<kOutF32, true>>, allow_lds<true, PlainEpilogue<kOutF16, true>>,
                       allow_lds<true, PlainEpilogue<kOutF16, false>>, allow_lds<true, PlainEpilogue<kOutBF16, true>>,
                       allow_lds<true, PlainEpilogue<kOutBF16, false>>, allow_lds<true, GatedEpilogue<kOutF32, true>>,
                       allow_lds<true, GatedEpilogue<kOutF16, true>>, allow_lds<true, GatedEpilogue<kOutF16, false>>,
                       allow_lds<true, GatedEpilogue<kOutBF16, true>>, allow_lds<true, GatedEpilogue<kOutBF16, false>>,
                       allow_lds<true, GatedMxEpilogue>, allow_lds<true, GradientEpilogue>,
                       allow_lds<false, PlainEpilogue<kOutF32, true>>, allow_lds<false, PlainEpilogue<kOutBF16, true>>,
                       allow_lds<false, PlainEpilogue<kOutBF16, false>>})
        if (e == hipSuccess)
            e = allow();
    return e;
}

hipError_t launch_mx_linear(const MxMatrix &x, const MxMatrix &w, const float *bias, void *y, int out, int k, const DeviceInfo &dev,
                            hipStream_t stream)
{
    if (k > 0 && x.rows <= kSkinnyRows)
        return launch_mx_linear_skinny(x, w, bias, y, out, k, stream);
    return by_type(out, w.rows, [&](auto type, auto columns) {
        constexpr int OUT = decltype(type)::value;
        if (k == 0)
            return fill_rows<OUT>(y, bias, (size_t)x.rows, (size_t)w.rows, stream);
        const PlainEpilogue<OUT, decltype(columns)::value> ep{y, bias, (size_t)w.rows, x.rows, w.rows};
        return launch<true>(operands(x, w, w, k), w.rows, ep, dev, stream);
    });
}

hipError_t launch_mx_gated(const MxMatrix &x, const MxMatrix &wg, const MxMatrix &wu, Activation act, void *h, int out, int k,
                           const DeviceInfo &dev, hipStream_t stream)
{
    if (k > 0 && x.rows <= kSkinnyRows)
        return launch_mx_gated_skinny(x, wg, wu, act, h, out, k, stream);
    return by_type(out, wg.rows, [&](auto type, auto columns) {
        constexpr int OUT = decltype(type)::value;
        if (k == 0)
            return fill_rows<OUT>(h, nullptr, (size_t)x.rows, (size_t)wg.rows, stream);
        const GatedEpilogue<OUT, decltype(columns)::value> ep{h, (size_t)wg.rows, x.rows, wg.rows, act};
        return launch<true>(operands(x, wg, wu, k), wg.rows, ep, dev, stream);
    });
}

hipError_t launch_mx_gated_quantized(const MxMatrix &x, const MxMatrix &wg, const MxMatrix &wu, Activation act, uint8_t *codes,
                                     uint8_t *scales, int k, const DeviceInfo &dev, hipStream_t stream)
{
    const int n = wg.rows;
    if (k == 0) {
        hipError_t e = fill_rows<kOutF32>(codes, nullptr, (size_t)x.rows, mx_code_stride(n) / 4, stream);
        return e == hipSuccess ? fill_rows<kOutF32>(scales, nullptr, (size_t)x.rows, mx_scale_stride(n) / 4, stream) : e;
    }
    if (x.rows <= kSkinnyRows)
        return launch_mx_gated_quantized_skinny(x, wg, wu, act, codes, scales, k, stream);
    const GatedMxEpilogue ep{codes, scales, mx_code_stride(n), mx_scale_stride(n), x.rows, n, act};
    // (the grid covers the padding at the end of h's rows)
    return launch<true>(operands(x, wg, wu, k), (int)(mx_code_stride(n) * 2), ep, dev, stream);
}

hipError_t launch_mx_gated_gradients(const MxMatrix &x, const MxMatrix &wg, const MxMatrix &wu, Activation act, const uint16_t *dh,
                                     uint16_t *d, size_t ld_n, uint16_t *dt, size_t ld_m, int k, const DeviceInfo &dev,
                                     hipStream_t stream)
{
    const GradientEpilogue ep{(const __bf16 *)dh, (__bf16 *)d, (__bf16 *)dt, ld_n, ld_m, x.rows, wg.rows, act, wg.rows % 4 == 0};
    return launch<true>(operands(x, wg, wu, k), wg.rows, ep, dev, stream);
}

static LineOperands operands(const Bf16Product &p)
{
    return {(const uint8_t *)p.a, (const uint8_t *)p.b, (const uint8_t *)p.b, nullptr, nullptr, nullptr, (unsigned)(p.ld * 2), 0, p.m, p.n,
            (p.k + kLineBf16 - 1) / kLineBf16};
}

template <int OUT, bool COLUMNS>
static PlainEpilogue<OUT, COLUMNS> epilogue(const Bf16Product &p)
{
    return {p.y, nullptr, (size_t)p.n, p.m, p.n};
}

// One product by itself.
static hipError_t launch_bf16(const Bf16Product &p, const DeviceInfo &dev, hipStream_t stream)
{
    if (p.k == 0)
        return p.out == kOutF32 ? fill_rows<kOutF32>(p.y, nullptr, (size_t)p.m, (size_t)p.n, stream)
                                : fill_rows<kOutBF16>(p.y, nullptr, (size_t)p.m, (size_t)p.n, stream);
    if (p.out == kOutF32)
        return launch<false>(operands(p), p.n, epilogue<kOutF32, true>(p), dev, stream);
    return p.n % 8 ? launch<false>(operands(p), p.n, epilogue<kOutBF16, true>(p), dev, stream)
                   : launch<false>(operands(p), p.n, epilogue<kOutBF16, false>(p), dev, stream);
}

template <class EpW, class EpX>
static hipError_t launch_group(const LineGroup &g, const EpW &ep_w, const EpX &ep_x, hipStream_t stream)
{
    int most = 1;
    for (int i = 0; i < g.count; ++i)
        most = max(most, g.tiles_m[i] * g.tiles_n[i] * g.slices[i]);
    line_group_kernel<Tile64, EpW, EpX><<<dim3((unsigned)most, 1, (unsigned)g.count), Tile64::THREADS, Tile64::LDS<false>, stream>>>(g, ep_w, ep_x);
    return hipGetLastError();
}

constexpr int kMostTogether = 1536;

// How long a slice of k is at least, in stages: meeting costs as much as about six.
constexpr int kLeastSlice = 6;

hipError_t launch_bf16_products(const Bf16Product *p, int count, const ColumnSums &sums, const SliceSpace &space, const DeviceInfo &dev,
                                hipStream_t stream)
{
    // Together up to three rounds of tiles of 64 x 64 (us apart and together: 257 x 1400 x 1000, gated, 784 tiles 39, 32.6; 700 x 2000 x 1000, gated,
    // 1200 tiles 53.2, 52.5; 1600 x 2048 x 1536, linear, 1368 tiles 50.4, 46.1; 1000 x 2000 x 2000, linear, 1536 tiles 42.7, 43.7; 2048^3, 2048 tiles
    // 60, 66): beyond that each fills the device alone, on larger tiles.  Long k is cut into slices as far as they go.  (Backward pass of a gated layer, 257 x 1400 x 1000, and of a linear one,
    // 130 x 1001 x 515: a launch for each product and operand 39 and 27 us, grouped 33 and 14, with slices 29 and 14: the
    // gated products 21 us, with dx in four slices 17.)
    long tiles = 0;
    bool together = count > 0 && p[count - 1].out == kOutBF16;
    for (int i = 0; i < count; ++i) {
        tiles += ((p[i].m + 63l) / 64) * ((p[i].n + 63l) / 64);
        together = together && p[i].k > 0 && p[i].n == p[0].n && (i == count - 1 || p[i].out == p[0].out);
    }
    if (!together || tiles > kMostTogether) {
        hipError_t e = hipSuccess;
        for (int i = 0; i < count && e == hipSuccess; ++i)
            if (p[i].y)
                e = launch_bf16(p[i], dev, stream);
        return e == hipSuccess && sums.sums ? launch_column_sums(sums, stream) : e;
    }
    LineGroup g{};
    g.count = count;
    for (int i = 0; i < count; ++i) {
        g.o[i] = operands(p[i]);
        g.y[i] = p[i].y;
        g.tiles_m[i] = (p[i].m + 63) / 64;
        g.tiles_n[i] = (p[i].n + 63) / 64;
    }
    int total = 0;
    for (int least = kLeastSlice;; least += least / 4) {
        total = 0;
        for (int i = 0; i < count; ++i) {
            g.slices[i] = min(max(g.o[i].stages / least, 1), 16);
            g.first[i] = total;
            total += g.tiles_m[i] * g.tiles_n[i] * g.slices[i];
        }
        if (total <= kMostSlices || total == tiles)
            break;
    }
    bool any = false;
    for (int i = 0; i < count; ++i) {
        any = any || p[i].y;
        if (!p[i].y)
            g.tiles_m[i] = 0;  // not wanted; the others' slices are the same with it and without
    }
    if (!any)
        return sums.sums ? launch_column_sums(sums, stream) : hipSuccess;
    g.partial = space.partial;
    g.arrivals = space.arrivals;
    g.sums = sums.sums;
    g.sum_parts = sums.partial;
    g.parts = sums.parts;
    g.columns = sums.columns;
    const Bf16Product &w = p[0], &x = p[count - 1];
    if (w.out == kOutF32)
        return x.n % 8 ? launch_group(g, epilogue<kOutF32, true>(w), epilogue<kOutBF16, true>(x), stream)
                       : launch_group(g, epilogue<kOutF32, true>(w), epilogue<kOutBF16, false>(x), stream);
    return x.n % 8 ? launch_group(g, epilogue<kOutBF16, true>(w), epilogue<kOutBF16, true>(x), stream)
                   : launch_group(g, epilogue<kOutBF16, false>(w), epilogue<kOutBF16, false>(x), stream);
}

}  // namespace int4linear
