// How a call's matrices are laid out and cut into tiles for the Newton-Schulz products.  Free of HIP calls, so that the host
// can check it without a GPU.
//
// A matrix is held as two float16 halves (split_gemm.h) in rows of slabs: 32 columns are 64 bytes of high halves and 64 bytes
// of low ones.  Rows and columns are padded to multiples of 32 with zeros; zeros stay zeros through all products.
#pragma once

#include <stdint.h>

#if defined(__HIPCC__)
#define MUON_HD __host__ __device__ __forceinline__
#else
#define MUON_HD inline
#endif

namespace aeth {

constexpr int kMuonMax = 32;                             // matrices of a call
constexpr int kMuonLongest = 1 << 21;                    // rows or columns: a 256-row tile's bytes stay below 2^31
constexpr int kMuonParts = 256;                          // partial sums of a matrix's norm

MUON_HD int64_t muon_pad(int64_t n) { return (n + 31) / 32 * 32; }

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

}  // namespace aeth
