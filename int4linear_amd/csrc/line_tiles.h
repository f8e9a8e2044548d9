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
inline double line_tile_cost(const LineTileCost &t, int per_cu, long tiles, int stages, long cus)
{
    const long places = cus * per_cu, rounds = tiles / places, rest = tiles % places;
    double stage = (double)rounds * per_cu * t.full;
    if (rest) {
        const double shared = (double)rest / cus * t.full;
        stage += shared > t.few ? shared : t.few;
    }
    return stage * stages + t.fixed;
}

inline int quickest_tile(bool fp4, long m, long n, int stages, bool pair, int cu_count, double *its_cost = nullptr)
{
    const long cus = cu_count > 0 ? cu_count : 256;
    int best = 0;
    double least = 0;
    for (int i = 0; i < 3 + !pair; ++i) {
        const LineTileCost &t = kLineTiles[i];
        const long tiles = ((m + t.m - 1) / t.m) * ((n + t.n - 1) / t.n);
        const double cost = line_tile_cost(t, line_tiles_per_cu(t, fp4), tiles, stages, cus);
        if (i == 0 || cost < least) {
            best = i;
            least = cost;
        }
    }
    if (its_cost)
        *its_cost = least;
    return best;
}

// Operands without scales also go in tiles that have a CU to themselves and more bytes on their way, where there are no more of
// them than CUs: numbers kDeepTiles and up.  us without them and with them, weights from HBM, 8-bit operands:
//   128 x 128   256 x 11008 x 4999 42.8, 32.3; 1024 x 4096 x 4096 25.6, 19.6; 130 x 16384 x 2048 16.0, 12.1; 2048^3 15.3, 12.2
//   192 x 128   333 x 11008 x 4999 41.4, 35.1; 384 x 11008 x 4096 34.3, 27.7; 333 x 14336 x 2048 21.8, 15.8
//   128 x 192   512 x 11008 x 4096 43.0, 30.9; 1024 x 5120 x 5120 39.5, 31.7
//   192 x 192   3000 x 2900 x 4000 48.6, 39.8; 2048 x 4096 x 4096 39.0, 36.0; 2700^3 29.1, 29.5
// and the gradients, with bfloat16 ones, of 2048^3 59.7, 49.3; 3000^3 152, 122.  Where there are few of them, smaller tiles bring more CUs'
// loads: 512 x 4096 x 11008 42.7 on 64 x 128, 53.2 on 128 x 128 of this kind; 200 x 4096 x 14336 31.3 on 64 x 64, 57.4.
constexpr int kDeepTiles = 4;
constexpr LineTileCost kDeepTileCosts[] = {{128, 128, {131072, 0}, 46, 46, 740},
                                           {192, 128, {122880, 0}, 58, 58, 950},
                                           {128, 192, {122880, 0}, 58, 58, 950},
                                           {192, 192, {147456, 0}, 85, 85, 1050}};
inline int quickest_tile_without_scales(long m, long n, int stages, int cu_count, double *its_cost = nullptr)
{
    const long cus = cu_count > 0 ? cu_count : 256;
    double cost;
    int best = quickest_tile(false, m, n, stages, false, cu_count, &cost);
    for (int i = 0; i < 4; ++i) {
        const LineTileCost &t = kDeepTileCosts[i];
        const long tiles = ((m + t.m - 1) / t.m) * ((n + t.n - 1) / t.n);
        const double deep = line_tile_cost(t, 1, tiles, stages, cus);
        if (tiles <= cus && deep < cost) {
            best = kDeepTiles + i;
            cost = deep;
        }
    }
    if (its_cost)
        *its_cost = cost;
    return best;
}

// Slices of k that make a product of bfloat16 operands on 64 x 64 tiles quicker than the quickest tile does unsliced, by the same
// costs; 1: none do.  At most `room` tile-slices; a slice is `least` stages long at least, and meeting costs as much as that.
inline int quicker_slices(long m, long n, int stages, long room, int least, int cu_count)
{
    const long cus = cu_count > 0 ? cu_count : 256, tiles = ((m + 63) / 64) * ((n + 63) / 64);
    const LineTileCost &t = kLineTiles[3];
    double cost;
    quickest_tile_without_scales(m, n, stages, cu_count, &cost);
    int best = 1;
    for (int slices = 2; slices <= 16 && slices * tiles <= room && slices * least <= stages; ++slices) {
        const double sliced = line_tile_cost(t, line_tiles_per_cu(t, false), tiles * slices, (stages + slices - 1) / slices + least, cus);
        if (sliced < cost) {
            cost = sliced;
            best = slices;
        }
    }
    return best;
}

// Slices of the products of one launch on 64 x 64 tiles, as short as `room` tile-slices allow but of `least` stages at least, and the
// number of each product's first tile-slice.  If that leaves all of them whole, with `long_alone` those are sliced whose sums are
// twice as long and more as what the device's `places` have on average. (us: 8192 x 512 x 512 73, so 61; with slices for ever longer sums, 1000 x 2000 x 2000 45, 50.)
inline void group_slices(int count, const int *tiles, const int *stages, int least, int room, bool long_alone, long places, int *slices,
                         int *first)
{
    long work = 0;
    for (int i = 0; i < count; ++i)
        work += (long)tiles[i] * stages[i];
    bool only = false;
    for (int shortest = least;;) {
        int total = 0;
        bool any = false;
        for (int i = 0; i < count; ++i) {
            const int most = only && stages[i] * places < 2 * work ? 1 : stages[i] / shortest;
            slices[i] = most < 1 ? 1 : most > 16 ? 16 : most;
            first[i] = total;
            any = any || slices[i] > 1;
            if (slices[i] > 1 || !only)  // (one slice has no one to meet)
                total += tiles[i] * slices[i];
        }
        if (any ? total <= room : only || !long_alone)
            return;
        if (!any) {
            only = true;
            shortest = least;
        } else {
            shortest += shortest / 4;
        }
    }
}

}  // namespace int4linear
