// Which tile a product of kernels_line_gemm.hip runs on: a rule on sizes and element type, plain C++.
#pragma once

namespace int4linear {

// A tile's rows and columns, the LDS of a workgroup with bfloat16 operands and with 4-bit ones (whose scales come on top), and
// what it costs in units of 10 ns: a stage, where every CU is busy with such tiles (`full`) and where there are few (`few`: nothing
// hides the way to memory), and what a launch spends before its first stage and after its last.  Read off the products below,
// products that fill the device (8192^3: 283, 342, 461 us, 64 x 64 about 600) and short ones (1024^3: 11.7, 5.9, 5.2, 4.8 us).
struct LineTileCost {
    int m, n, lds[2], full, few, fixed;
};
constexpr LineTileCost kLineTiles[] = {{256, 256, {131072, 147456}, 175, 175, 1100},
                                       {128, 128, {65536, 73728}, 62, 70, 600},
                                       {64, 128, {73728, 82944}, 46, 45, 380},
                                       {64, 64, {65536, 73728}, 29, 29, 330}};

// Workgroups of a tile that a CU's LDS holds: with bfloat16 operands 64 x 128 fits twice, with 4-bit ones once.
constexpr int line_tiles_per_cu(const LineTileCost &t, bool fp4) { return 160 * 1024 / t.lds[fp4]; }

// The tile that makes a product of m x n (columns of b) in `stages` stages quickest by these costs; the last is too narrow for a pair of
// matrices b.  Measured, us by tile, bfloat16 results, operands in the caches; 4-bit operands:
//   512 x 4096 x 11008   64, 32.9, 23.6, 29.8        333 x 11008 x 4999   36, 21.2, 27.8, 27.1
//   2048 x 4096 x 4096   33, 25.6, 34.5, 44.7        128 x 14336 x 4096   26, 14.4, 10.3, 12.3
//   64 x 4096 x 4096     23, 10.1, 8.6, 7.5          200 x 4096 x 14336   -, 37.7, 24.1, 20.4
// and bfloat16 ones:
//   1030 x 1990 x 2000   57, 29.3, 23.0, 22.8        1280 x 2048 x 4096   84, 40.9, 36.6, 37.1
//   2048 x 2816 x 4096   92, 51.0, 58.9, 79.8        4096^3               116, 124, 160, 202
inline int quickest_tile(bool fp4, long m, long n, int stages, bool pair, int cu_count)
{
    const long cus = cu_count > 0 ? cu_count : 256;
    int best = 0;
    double least = 0;
    for (int i = 0; i < 3 + !pair; ++i) {
        const LineTileCost &t = kLineTiles[i];
        const int per_cu = line_tiles_per_cu(t, fp4);
        const long tiles = ((m + t.m - 1) / t.m) * ((n + t.n - 1) / t.n);
        const long places = cus * per_cu, rounds = tiles / places, rest = tiles % places;
        double stage = (double)rounds * per_cu * t.full;
        if (rest) {
            const double shared = (double)rest / cus * t.full;
            stage += shared > t.few ? shared : t.few;
        }
        const double cost = stage * stages + t.fixed;
        if (i == 0 || cost < least) {
            best = i;
            least = cost;
        }
    }
    return best;
}

}  // namespace int4linear
