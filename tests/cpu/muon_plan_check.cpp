// Host checks of aether-ml_amd/csrc/muon_plan.h: the triangle's tiles are numbered one to one, the chosen tiles and runs cover every
// product, the buffers of a matrix do not overlap and hold what the kernels write.
#include "muon_plan.h"

#include <stdio.h>
#include <stdlib.h>
#include <vector>

using namespace aeth;

#define CHECK(c)                                                              \
    do {                                                                      \
        if (!(c)) {                                                           \
            printf("FAILED line %d: %s\n", __LINE__, #c);                     \
            return 1;                                                         \
        }                                                                     \
    } while (0)

static int triangles() {
    for (int T = 1; T <= 150; ++T) {
        const int n = T * (T + 1) / 2;
        std::vector<int> seen(T * T);
        for (int t = 0; t < n; ++t) {
            int i, j;
            muon_triangle(t, &i, &j);
            CHECK(0 <= i && i <= j && j < T && !seen[i * T + j]++);
            CHECK(j * (j + 1) / 2 + i == t);
        }
    }
    // large numbers, where a float32 square root is off by several
    for (int T : {5000, 20000, 60000}) {
        const int64_t n = (int64_t)T * (T + 1) / 2;
        for (int64_t t = 0; t < n; t += 1 + n / 100003) {
            int i, j;
            muon_triangle((int)t, &i, &j);
            CHECK(0 <= i && i <= j && j < T && (int64_t)j * (j + 1) / 2 + i == t);
        }
    }
    printf("ok triangles\n");
    return 0;
}

static int choices() {
    unsigned seed = 1;
    const auto next = [&] { return (int)((seed = seed * 1664525u + 1013904223u) >> 8); };
    for (int trial = 0; trial < 20000; ++trial) {
        const int count = trial % 3 == 0 ? 1 + next() % kMuonMax : 1;
        MuonShape g[kMuonMax], s[kMuonMax];
        for (int i = 0; i < count; ++i) {
            const int64_t m = muon_pad(1 + next() % (trial % 2 ? 5000 : 300)), n = m + muon_pad(next() % (trial % 5 ? 3000 : 200000));
            g[i] = MuonShape{m, m, n};
            s[i] = MuonShape{m, n, m};
        }
        const int a = muon_choose(g, count, true), b = muon_choose(s, count, false);
        CHECK(a >= 0 && kMuonTileTable[a].symmetric && kMuonTileTable[a].bm == kMuonTileTable[a].bn);
        CHECK(b >= 0 && kMuonTileTable[b].general);
        MuonRuns r;
        if (muon_choose_runs(g, count, &r)) {
            // the tiles that kSplitPart is built for; runs that cover all slabs, none empty
            CHECK(r.tile >= 0 && r.tile < kMuonTiles && kMuonTileTable[r.tile].runs && r.run >= 1);
            int64_t bytes = 0;
            for (int i = 0; i < count; ++i) {
                const int64_t slabs = g[i].k / 32, side = g[i].rows / 32;
                CHECK(r.runs[i] >= 1 && r.runs[i] * r.run >= slabs && (r.runs[i] - 1) * r.run < slabs);
                bytes += r.runs[i] * side * (side + 1) / 2 * 4096;
            }
            CHECK(bytes == r.bytes);
        }
    }
    printf("ok choices\n");
    return 0;
}

static int layouts() {
    for (int64_t m : {1, 31, 32, 33, 64, 1000, 4096})
        for (int64_t n : {1, 32, 65, 1000, 5000, 2000000}) {
            if (n < m) continue;
            const MuonLayout l = muon_layout(m, n, 8192);
            CHECK(l.mp >= m && l.np >= n && l.mp % 32 == 0 && l.np % 32 == 0 && l.mp - m < 32 && l.np - n < 32);
            const int64_t x = l.np / 32 * l.mp * 128, xt = l.mp / 32 * l.np * 128, a = l.mp / 32 * l.mp * 128;
            CHECK(l.x == 8192 && l.xt0 >= l.x + x && l.xt1 >= l.xt0 + xt && l.a >= l.xt1 + xt && l.b >= l.a + a && l.end >= l.b + a);
            CHECK(l.xt0 % 128 == 0 && l.xt1 % 128 == 0 && l.a % 128 == 0 && l.b % 128 == 0 && l.end % 128 == 0);
        }
    printf("ok layouts\n");
    return 0;
}

int main() { return triangles() || choices() || layouts(); }
