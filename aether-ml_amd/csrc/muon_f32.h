// Newton-Schulz products of float32 matrices, for more steps than two float16 halves carry (muon_in_halves).
//
//   A = X X^T,  B = b A + c A A,  X <- a X + B X
//
// Every matrix is stored times 2^60.  X's norm is 1 at first, so what is weak in it, down to 2^-186 of the norm, stays a normal number
// until a hundred steps (a factor of up to 3.4445 each, 2^178 together) have brought it to full size, in X as in the products of it with
// what is strong; and no sum passes 2^123 (the elements of A are at most 1.47, of B 3.45, of X 1.21, and a sum's terms are bounded by
// the norms of a row and a column).  A weak row of A or B is a sum of products with that row, so it is as exact, for its size, as a strong one.
#pragma once

#include "conv_common.h"
#include "muon_plan.h"

namespace aeth {

constexpr float kFloatScale = 0x1p60f;

// D = alpha R + beta P Q^T (`rows`: Q is [N][K]) or alpha R + beta P Q (Q is [K][N]); P [M][K], R and D [M][N]; all sides multiples of 64.
struct FloatProduct {
    const float *P, *Q, *R;
    float* D;
    float *theta, *out;  // the last step writes here instead of D: theta <- keep theta - step D, or out = D, both [rows][cols]
    int M, N, K;
    int rows, cols;
    int first;           // this product's first tile
    float gain;
};
struct FloatTable {
    int count;
    FloatProduct p[kMuonMax];
};
static_assert(sizeof(FloatTable) + 64 <= 4096, "a launch's arguments");

// 64 x 64 of the result a workgroup, 32 x 32 a wave; slabs of 16 columns through two LDS buffers, the next slab's loads on their way while
// this one is multiplied.  A float32 sum of 2^20 terms in line would be worth little, so every 1024 columns go into a total of their own.
// Bound: the float32 matrix instructions on large matrices (4096 x 4096: 10 steps 33 ms, 124 TFLOP/s of 132 that a library's float32
// product of that size reaches; without the symmetry of A and B, and five times what halves take), few tiles on small ones (64 x 576: 307
// us for 10 steps, 77 on halves).  A call takes this way only where halves would be wrong, so it was left simple.
template <bool kRows, bool kApply>
__global__ __launch_bounds__(256) void float_product(const FloatTable tb, float alpha, float beta, float lr,
                                                     const double* __restrict__ state, float wd) {
    constexpr int S = 68;                                // floats of an LDS row
    __shared__ float p[2][16][S], q[2][16][S];
    typedef const FloatTable __attribute__((address_space(4)))* table_ptr;
    const table_ptr args = (table_ptr)__builtin_amdgcn_kernarg_segment_ptr();
    int k = 0;
    while (k + 1 < tb.count && (int)blockIdx.x >= args->p[k + 1].first) ++k;
    FloatProduct pr = tb.p[0];
    __builtin_memcpy(&pr, (const void*)(args->p + k), sizeof(pr));
    const int tile = blockIdx.x - pr.first, tn = pr.N / 64, i0 = tile / tn * 64, j0 = tile % tn * 64;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, l32 = lane & 31, lh = lane >> 5, wm = wave / 2 * 32, wn = wave % 2 * 32;
    // a thread's four floats of a slab: of one row, or of one row of Q as it is
    const int line = t >> 2, part = 4 * (t & 3), qline = t >> 4, qpart = 4 * (t & 15);
    const float* sp = pr.P + (size_t)(i0 + line) * pr.K + part;
    const float* sq = kRows ? pr.Q + (size_t)(j0 + line) * pr.K + part : pr.Q + (size_t)qline * pr.N + j0 + qpart;
    const size_t step = kRows ? 16 : (size_t)16 * pr.N;
    f4 np, nq;
    const auto load = [&] {
        np = *reinterpret_cast<const f4*>(sp);
        nq = *reinterpret_cast<const f4*>(sq);
        sp += 16;
        sq += step;
    };
    const auto put = [&](int buf) {
#pragma unroll
        for (int e = 0; e < 4; ++e) p[buf][part + e][line] = np[e];
        if (kRows) {
#pragma unroll
            for (int e = 0; e < 4; ++e) q[buf][part + e][line] = nq[e];
        } else {
            *reinterpret_cast<f4*>(&q[buf][qline][qpart]) = nq;
        }
    };
    f16v total, acc;
#pragma unroll
    for (int v = 0; v < 16; ++v) total[v] = acc[v] = 0.f;
    const int slabs = pr.K / 16;
    load();
    put(0);
    __syncthreads();
    for (int s = 0; s < slabs; ++s) {
        const int buf = s & 1;
        if (s + 1 < slabs) load();
#pragma unroll
        for (int c = 0; c < 16; c += 2)
            acc = __builtin_amdgcn_mfma_f32_32x32x2f32(p[buf][c + lh][wm + l32], q[buf][c + lh][wn + l32], acc, 0, 0, 0);
        if ((s & 63) == 63) {
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                total[v] += acc[v];
                acc[v] = 0.f;
            }
        }
        if (s + 1 < slabs) put(buf ^ 1);                 // (read by nobody since the barrier before)
        __syncthreads();
    }
    float keep = 0.f, move = 0.f;
    if (kApply) {
        if (state != nullptr) lr = (float)state[3];
        keep = 1.0f - lr * wd;
        move = lr * pr.gain;
    }
    const bool tall = pr.rows > pr.cols;
#pragma unroll
    for (int v = 0; v < 16; ++v) {
        const int i = i0 + wm + 8 * (v >> 2) + 4 * lh + (v & 3), j = j0 + wn + l32;
        const size_t at = (size_t)i * pr.N + j;
        const float d = (pr.R != nullptr ? alpha * pr.R[at] : 0.f) + beta * (total[v] + acc[v]);
        if (!kApply) {
            pr.D[at] = d;
            continue;
        }
        const int y = tall ? j : i, x = tall ? i : j;
        if (y >= pr.rows || x >= pr.cols) continue;
        const size_t w = (size_t)y * pr.cols + x;
        const float o = d * (1.f / kFloatScale);
        if (pr.theta != nullptr) pr.theta[w] = keep * pr.theta[w] - move * o;
        else pr.out[w] = o;
    }
}

}  // namespace aeth
