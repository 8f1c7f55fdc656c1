// Host checks of the limit up to which two float16 halves carry a matrix through the steps, and of the float32 buffers
// (aether-ml_amd/csrc/muon_plan.h).
#include "muon_plan.h"

#include <initializer_list>
#include <math.h>
#include <stdio.h>

using namespace aeth;

#define CHECK(c)                                                              \
    do {                                                                      \
        if (!(c)) {                                                           \
            printf("FAILED line %d: %s\n", __LINE__, #c);                     \
            return 1;                                                         \
        }                                                                     \
    } while (0)

int main() {
    for (int64_t n = 1; n <= kMuonLongest; n += 1 + n / 50) {
        bool last = true;
        for (int steps = 1; steps <= 100; ++steps) {
            const bool in = muon_in_halves(n, steps);
            const double off = pow(3.4445, steps) * sqrt((double)n) * pow(2.0, -20);
            if (off < 0.999) CHECK(in);
            if (off > 1.001) CHECK(!in);
            CHECK(last || !in);                          // (never again with more steps)
            last = in;
        }
        CHECK(muon_in_halves(n, 5) && !muon_in_halves(n, 12));
    }
    CHECK(muon_in_halves(236, 9) && !muon_in_halves(237, 9) && muon_in_halves(2800, 8) && !muon_in_halves(2801, 8));
    CHECK(muon_in_halves(33222, 7) && !muon_in_halves(33223, 7));
    for (int64_t m : {1, 31, 64, 65, 1000, 4096})
        for (int64_t n : {1, 64, 65, 1000, 5000, 2000000}) {
            if (n < m) continue;
            const MuonFloatLayout l = muon_float_layout(m, n, 8192);
            CHECK(l.mp >= m && l.np >= n && l.mp % 64 == 0 && l.np % 64 == 0 && l.mp - m < 64 && l.np - n < 64);
            const int64_t x = l.mp * l.np * 4, a = l.mp * l.mp * 4;
            CHECK(l.x[0] == 8192 && l.x[1] == l.x[0] + x && l.a == l.x[1] + x && l.b == l.a + a && l.end == l.b + a);
        }
    printf("ok halves\n");
    return 0;
}
