// How a call's matrices are laid out and cut into tiles for the Newton-Schulz products.  Free of HIP calls, so that the host
// can check it without a GPU.
//
// A matrix is held as two float16 halves (split_gemm.h) in slabs of 32 columns, or for many steps as float32 (muon_f32.h).  Rows and
// columns are padded with zeros to multiples of 32, or 64; zeros stay zeros through all products.
#pragma once

#include <stdint.h>

#if defined(__HIPCC__)
#define MUON_HD __host__ __device__ __forceinline__
#else
#define MUON_HD inline
#endif

namespace aeth {

constexpr int kMuonMax = 32;                             // matrices of a call
constexpr int kMuonLongest = 1 << 21;                    // rows or columns: a sum of more float32 products in line would be worth little
constexpr int kMuonParts = 1024;                          // partial sums of a matrix's norm

MUON_HD int64_t muon_pad(int64_t n) { return (n + 31) / 32 * 32; }

// Whether two float16 halves carry a matrix of n columns (the longer side) through so many steps.  The halves end 2^-40 below |u|:
// a row, a column or a block of the matrix that is much weaker than the rest is held with that error, which every step multiplies
// by up to 3.4445 until the part has grown to full size.  An element's share of that is worth sqrt(n) in a row, so the result is off
// by 2^-40 3.4445^steps sqrt(n) of its norm in the worst case (a part that reaches full size with the last step).  The limit is 2^-20,
// what float32 products cost on the same matrices (64 x 96, 8 steps: 1.1e-6 against 2.3e-6; 64 x 2048: 2.2e-6 and 3.7e-6; above the
// limit, 12 steps: 1.2e-5 and 7e-6; 8.8e-5 and 6.8e-6).  It allows 9 steps up to 236 columns, 8 up to 2800, 7 up to 33222, 5 up to 2^21.
static inline bool muon_in_halves(int64_t n, int steps) {
    double off = 1.0 / ((int64_t)1 << 40);               // squared: the square root is not needed
    off = off * off * (double)n;
    const double limit = 1.0 / ((int64_t)1 << 40);
    for (int s = 0; s < steps && off <= limit; ++s) off *= 3.4445 * 3.4445;
    return off <= limit;
}

// The buffers of a matrix held as float32 (byte offsets): X and the next X [mp][np], A and B [mp][mp].
struct MuonFloatLayout {
    int64_t mp, np;
    int64_t x[2], a, b, end;
};
MUON_HD MuonFloatLayout muon_float_layout(int64_t m, int64_t n, int64_t begin) {
    MuonFloatLayout l;
    l.mp = (m + 63) / 64 * 64;
    l.np = (n + 63) / 64 * 64;
    l.x[0] = begin;
    l.x[1] = l.x[0] + 4 * l.mp * l.np;
    l.a = l.x[1] + 4 * l.mp * l.np;
    l.b = l.a + 4 * l.mp * l.mp;
    l.end = l.b + 4 * l.mp * l.mp;
    return l;
}

// Byte offsets of one matrix's buffers in the workspace (m x n with m <= n; X is [m][n], Xt its transpose).
struct MuonLayout {
    int64_t mp, np;                                      // padded sides
    int64_t x, xt0, xt1, a, b, end;
};

static inline MuonLayout muon_layout(int64_t m, int64_t n, int64_t begin) {
    MuonLayout l;
    l.mp = muon_pad(m);
    l.np = muon_pad(n);
    l.x = begin;
    l.xt0 = l.x + 4 * l.mp * l.np;
    l.xt1 = l.xt0 + 4 * l.mp * l.np;
    l.a = l.xt1 + 4 * l.mp * l.np;
    l.b = l.a + 4 * l.mp * l.mp;
    l.end = l.b + 4 * l.mp * l.mp;
    return l;
}

// The tiles of a product whose result is symmetric: those on and above the diagonal, column by column.
// t -> (i, j), 0 <= i <= j, t = j (j + 1) / 2 + i.
MUON_HD void muon_triangle(int t, int* i, int* j) {
    int c = (int)((__builtin_sqrtf(8.0f * (float)t + 1.0f) - 1.0f) * 0.5f);
    while ((int64_t)c * (c + 1) / 2 > t) --c;            // (the square root is rounded)
    while ((int64_t)(c + 1) * (c + 2) / 2 <= t) ++c;
    *i = t - (int)((int64_t)c * (c + 1) / 2);
    *j = c;
}

static inline int64_t muon_tiles(int64_t rows, int64_t cols, int bm, int bn, bool symmetric) {
    const int64_t tm = (rows + bm - 1) / bm, tn = (cols + bn - 1) / bn;
    return symmetric ? tm * (tm + 1) / 2 : tm * tn;
}

// The tile shapes a product can be cut into, with what a tile costs: `start` us a launch, `again` us for every further tile of a
// CU (its first loads and its epilogue, as far as no other tile hides them), then us a slab of 32 columns on a CU whose neighbours
// are idle (`alone`) and with a tile on every CU (`full`: the tiles then share the L2 caches' bandwidth and the power that the
// matrix units may draw).  CUs with one tile more than others hold the launch up by `slack` of that tile (several small tiles are
// on a CU at once).  Fitted to square and wide products of 64 to 4096 rows; the tile with the least cost is taken: 3000 x 3000
// gram 94 us in tiles of 160 x 160 (120 in 96, 121 in 192, 132 in 64), step 136 in 192 x 192 (169 in 96); 4096 x 4096 gram 180 in
// 192 x 192 (240 in 160), step 330 in 256 x 128 (373 in 192 x 192).  (Products alone, repeated; within an update, after one another,
// the large ones take 2-3 % more.)
struct MuonTile {
    int bm, bn;
    bool symmetric, general, runs;     // offered for symmetric results, for others, for gram products in runs
    float start, again, slack, alone, full;
};
enum { kTile32, kTile64, kTile96, kTile128, kTile160, kTile192, kTile256x128, kMuonTiles };
static const MuonTile kMuonTileTable[kMuonTiles] = {
    {32, 32, true, true, true, 3.3f, 4.0f, 0.2f, 0.11f, 0.12f},
    {64, 64, true, true, true, 4.5f, 0.5f, 0.5f, 0.21f, 0.25f},
    {96, 96, true, true, false, 6.0f, 1.0f, 0.6f, 0.33f, 0.48f},
    {128, 128, true, true, true, 6.0f, 5.0f, 1.0f, 0.50f, 0.74f},
    {160, 160, true, true, false, 10.0f, 5.0f, 1.0f, 0.75f, 0.96f},
    {192, 192, true, true, false, 10.0f, 5.0f, 1.0f, 1.00f, 1.34f},
    {256, 128, false, true, false, 5.0f, 5.0f, 1.0f, 0.95f, 1.26f},
};
constexpr int kMuonCus = 256;

struct MuonShape {
    int64_t rows, cols, k;       // padded
};

// Tiles that the busiest CU is held up by.
static inline float muon_turns(const MuonTile& t, int64_t tiles) {
    const float even = (float)tiles / kMuonCus, most = (float)((tiles + kMuonCus - 1) / kMuonCus);
    return even <= 1.f ? 1.f : even + (most - even) * t.slack;
}
static inline float muon_slab(const MuonTile& t, int64_t tiles) {
    return t.alone + (t.full - t.alone) * (tiles < kMuonCus ? (float)tiles / kMuonCus : 1.f);
}

// What a launch of these products costs with one tile shape, in us: all tiles in turn, of average length, or one product's alone.
static inline float muon_cost(const MuonTile& t, const MuonShape* p, int count, bool symmetric) {
    int64_t tiles = 0, slabs = 0;
    float longest = 0.f;
    for (int i = 0; i < count; ++i) {
        const int64_t n = muon_tiles(p[i].rows, p[i].cols, t.bm, t.bn, symmetric);
        tiles += n;
        slabs += n * (p[i].k / 32);
        const float mine = muon_turns(t, n) * (float)(p[i].k / 32);
        if (mine > longest) longest = mine;
    }
    const float turns = muon_turns(t, tiles), all = turns * (float)slabs / (float)tiles;
    return t.start + t.again * (turns - 1.f) + (longest > all ? longest : all) * muon_slab(t, tiles);
}

static inline int muon_choose(const MuonShape* p, int count, bool symmetric) {
    int best = -1;
    float least = 0.f;
    for (int i = 0; i < kMuonTiles; ++i) {
        if (!(symmetric ? kMuonTileTable[i].symmetric : kMuonTileTable[i].general)) continue;
        const float c = muon_cost(kMuonTileTable[i], p, count, symmetric);
        if (best < 0 || c < least) {
            best = i;
            least = c;
        }
    }
    return best;
}

// Gram products of few rows and many columns: every tile's columns in `runs` runs, so that all CUs have work, and the runs' sums
// added by a second launch.  Per product: runs and slabs a run.
struct MuonRuns {
    int tile;                    // of kMuonTileTable
    int64_t runs[kMuonMax], run;
    int64_t bytes;               // of partial sums, all products
};
// The second launch: us at least, us for every 32 runs (8 waves add four at a time), bytes a us of partial sums written and read.
constexpr float kMuonJoin = 2.6f, kMuonJoinRuns = 1.0f, kMuonJoinRate = 3.5e6f;

// False where one launch without runs is the faster way.
static inline bool muon_choose_runs(const MuonShape* p, int count, MuonRuns* out) {
    bool found = false;
    *out = MuonRuns{};
    float least = muon_cost(kMuonTileTable[muon_choose(p, count, true)], p, count, true);
    for (int k = 0; k < kMuonTiles; ++k) {
        const MuonTile& t = kMuonTileTable[k];
        if (!t.runs) continue;
        MuonRuns r = {};
        r.tile = k;
        int64_t units = 0, longest = 0;
        for (int i = 0; i < count; ++i) {
            units += muon_tiles(p[i].rows, p[i].cols, t.bm, t.bn, true) * (p[i].k / 32);
            if (p[i].k / 32 > longest) longest = p[i].k / 32;
        }
        // (from four runs a CU, where one alone would be too uneven, to one)
        for (r.run = (units + 4 * kMuonCus - 1) / (4 * kMuonCus); r.run < longest; r.run += (r.run + 3) / 4) {
            int64_t tiles = 0, most = 0;
            r.bytes = 0;
            for (int i = 0; i < count; ++i) {
                const int64_t side = p[i].rows / 32;
                r.runs[i] = (p[i].k / 32 + r.run - 1) / r.run;
                if (r.runs[i] > most) most = r.runs[i];
                tiles += r.runs[i] * muon_tiles(p[i].rows, p[i].cols, t.bm, t.bn, true);
                r.bytes += r.runs[i] * (side * (side + 1) / 2) * 4096;
            }
            const float turns = muon_turns(t, tiles);
            const float c = t.start + t.again * (turns - 1.f) + turns * (float)r.run * muon_slab(t, tiles) + kMuonJoin +
                            kMuonJoinRuns * (float)((most + 31) / 32) + (float)r.bytes / kMuonJoinRate;
            if (c < least) {
                least = c;
                *out = r;
                found = true;
            }
        }
    }
    return found;
}

}  // namespace aeth
