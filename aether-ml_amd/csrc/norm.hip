// Layer norm over the last axis of a row-major [rows, C] tensor, forward and backward.
//
//   mean_r = sum_c x / C,  var_r = sum_c (x - mean_r)^2 / C,  invstd_r = 1 / sqrt(var_r + eps)
//   y = (x - mean_r) invstd_r gamma_c + beta_c
//
//   xhat = (x - mean_r) invstd_r,  g = dy gamma_c
//   dx = invstd_r (g - sum_c g / C - xhat sum_c g xhat / C)
//   dgamma_c = sum_r dy xhat,  dbeta_c = sum_r dy
//
// All sums are in a fixed order: results do not depend on timing.  They are float32 where no lane adds more than a few dozen numbers in
// line (a row in registers), and a few hundred over the rows (kLnRun); a row of any length is summed in 64 bits.
#include "common.h"

#include <algorithm>

namespace aeth {

constexpr int kLnLong = 1024;                            // threads of the kernels for rows of any length

// Rows that a lane adds in line to its columns' sums, at most: a float32 sum of n like terms in line is off by up to n 2^-24 of itself
// (0.1 added 65536 times: 6e-4 of the sum).
constexpr int kLnRun = 256;

// Outputs of this size and more are stored with the non-temporal hint: the next kernel will not find them in a cache anyway.
constexpr int64_t kLnStreamBytes = 64 << 20;

// float32 -> bfloat16 bits, round to nearest even; NaN stays NaN
__device__ __forceinline__ unsigned ln_bf16(float f) {
    const unsigned u = __float_as_uint(f);
    if ((u & 0x7fffffffu) > 0x7f800000u) return (u >> 16) | 0x40u;
    return (u + 0x7fffu + ((u >> 16) & 1u)) >> 16;
}

// A row is handled in units of four consecutive floats: unit k is columns 4k .. 4k + 3, and lane s of the row's L lanes holds units
// s, s + L, ..., V of them.  Where C is no multiple of four, units start at any float, which 16-byte loads and stores of the
// vector unit take, and the row's last unit is read from its last four columns; places behind the row's end read there too.  So
// no load waits for a branch (units that went through the rest float by float: 1000000 x 20 backward 124 us instead of 64,
// 400000 x 100 203 instead of 103).  V is the least that covers the row: only a lane's last unit can be such a one.
typedef float ln_f4 __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned ln_u2 __attribute__((ext_vector_type(2), aligned(2)));

// kTiny: rows of one to three floats, which no 16-byte load fits (V = 1; only own columns are read).
template <int V, bool kTiny = false>
struct LnLane {
    int c0, step;                                        // first column of unit 0, columns from unit to unit
    int last, skip;                                      // first column read for the last unit; so many of its four are not its own
    __device__ __forceinline__ LnLane(int s, int L, int C) {
        c0 = 4 * s;
        step = 4 * L;
        const int c = c0 + step * (V - 1);
        last = c + 4 <= C ? c : C - 4;
        skip = c + 4 <= C ? 0 : c < C ? c - last : 4;
    }
    __device__ __forceinline__ int at(int j) const { return j == V - 1 ? last : c0 + step * j; }
    __device__ __forceinline__ bool own(int j, int e) const { return j < V - 1 || e >= skip; }
    __device__ __forceinline__ void load(const float* __restrict__ row, int j, float* v) const {
        if (kTiny) {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = own(j, e) ? row[at(j) + e] : 0.f;
        } else {
            const ln_f4 t = *reinterpret_cast<const ln_f4*>(row + at(j));
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = t[e];
        }
    }
    __device__ __forceinline__ void store(float* __restrict__ row, int j, const float* v, bool stream) const {
        if (j < V - 1 || skip == 0) {
            const ln_f4 t = {v[0], v[1], v[2], v[3]};
            if (stream) __builtin_nontemporal_store(t, reinterpret_cast<ln_f4*>(row + at(j)));
            else *reinterpret_cast<ln_f4*>(row + at(j)) = t;
        } else if (skip < 4) {
#pragma unroll
            for (int e = 1; e < 4; ++e)
                if (own(j, e)) row[at(j) + e] = v[e];
        }
    }
    __device__ __forceinline__ void store16(uint16_t* __restrict__ row, int j, const float* v) const {
        if (j < V - 1 || skip == 0) {
            *reinterpret_cast<ln_u2*>(row + at(j)) =
                ln_u2{ln_bf16(v[0]) | (ln_bf16(v[1]) << 16), ln_bf16(v[2]) | (ln_bf16(v[3]) << 16)};
        } else if (skip < 4) {
#pragma unroll
            for (int e = 1; e < 4; ++e)
                if (own(j, e)) row[at(j) + e] = (uint16_t)ln_bf16(v[e]);
        }
    }
};

// Sum over aligned groups of L lanes, the same value in every lane of the group: within 16 lanes by the cross-lane paths of
// the vector unit, beyond through the LDS crossbar.
template <int kCtrl>
__device__ __forceinline__ float ln_dpp(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), kCtrl, 0xf, 0xf, true));
}
template <int L>
__device__ __forceinline__ float ln_group_sum(float v) {
    if (L >= 2) v += ln_dpp<0xb1>(v);                    // quad_perm 1,0,3,2
    if (L >= 4) v += ln_dpp<0x4e>(v);                    // quad_perm 2,3,0,1
    if (L >= 8) v += ln_dpp<0x141>(v);                   // row_half_mirror
    if (L >= 16) v += ln_dpp<0x140>(v);                  // row_mirror
    if (L >= 32) v += __shfl_xor(v, 16, 64);
    if (L >= 64) v += __shfl_xor(v, 32, 64);
    return v;
}

// Sums over the workgroup (up to 16 waves), the same values in every thread.  Two slots, used in turn, need one barrier a sum: a
// wave can be at most one barrier ahead of the slowest.
struct LnTeam {
    float (*red)[2][16];                                 // [slot][which sum][wave]
    int turn = 0;
    __device__ __forceinline__ explicit LnTeam(float (*r)[2][16]) : red(r) {}
    template <int N>
    __device__ __forceinline__ void sum(float* v) {
        const int waves = blockDim.x >> 6;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            v[i] = ln_group_sum<64>(v[i]);
            if ((threadIdx.x & 63) == 0) red[turn][i][threadIdx.x >> 6] = v[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            v[i] = red[turn][i][0];
            for (int w = 1; w < waves; ++w) v[i] += red[turn][i][w];
        }
        turn ^= 1;
    }
};

// A thread's columns of a row of any length, every kLnLong'th: f(column, terms) of four columns by pairs in float32, the rest in 64 bits.
template <int N, typename F>
__device__ __forceinline__ void ln_long_sum(int C, double* s, F f) {
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = 0.0;
    int64_t c = threadIdx.x;
    for (; c + 3 * kLnLong < C; c += 4 * kLnLong) {
        float v[4][N];
#pragma unroll
        for (int k = 0; k < 4; ++k) f(c + k * kLnLong, v[k]);
#pragma unroll
        for (int i = 0; i < N; ++i) s[i] += (double)((v[0][i] + v[1][i]) + (v[2][i] + v[3][i]));
    }
    for (; c < C; c += kLnLong) {
        float v[N];
        f(c, v);
#pragma unroll
        for (int i = 0; i < N; ++i) s[i] += (double)v[i];
    }
}

// Sums over the workgroup in 64 bits, one at a time; red: one slot, so there is a barrier in front of it.
__device__ __forceinline__ double ln_block_sum(double v, double* red) {
    const int waves = blockDim.x >> 6;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    __syncthreads();                                     // (the last sum has been read)
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
    for (int w = 1; w < waves; ++w) v += red[w];
    return v;
}

// ---- forward -----------------------------------------------------------------------------------------------------------
// Bound: HBM, 8 bytes an element (10 with the bfloat16 copy): 16384 x 8192 201 us = 5.3 TB/s, the rate of a copy; rows that no
// power of two divides 4.2-5.2 TB/s.  A row is read once and stays in registers: the mean, then the sum of
// squares of what is left, then the output, so that no cancellation of two large sums enters the variance.
struct LnFwdArgs {
    const float *x, *gamma, *beta;
    float *mean, *invstd, *y;
    uint16_t* y16;
    int rows, C;
    float inv_c, eps;
    bool stream;
};

// The row's values in v become its output.  Columns that the last unit reads but does not own count 0 times.  `sum(float)`: over
// the row's lanes; `affine(j, g, b)`: gamma and beta of unit j.
template <int V, bool kTiny, typename Sum, typename Affine>
__device__ __forceinline__ void ln_fwd_row(const LnFwdArgs& p, int64_t r, const LnLane<V, kTiny>& u, float (*v)[4], bool first,
                                           Sum sum, Affine affine) {
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) s += u.own(j, e) ? v[j][e] : 0.f;
    const float mean = sum(s) * p.inv_c;
    float q = 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[j][e] -= mean;
            q += u.own(j, e) ? v[j][e] * v[j][e] : 0.f;
        }
    const float invstd = 1.0f / sqrtf(sum(q) * p.inv_c + p.eps);
    if (first && p.mean != nullptr) {
        p.mean[r] = mean;
        p.invstd[r] = invstd;
    }
    const size_t at = (size_t)r * p.C;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        float g[4], b[4];
        affine(j, g, b);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[j][e] = v[j][e] * invstd * g[e] + b[e];
        u.store(p.y + at, j, v[j], p.stream);
        if (p.y16 != nullptr) u.store16(p.y16 + at, j, v[j]);
    }
}

// Rows of at most L V units, 256 / L of them at a time; gamma and beta of up to four units stay in registers over the rows.
template <int L, int V, bool kTiny = false>
__global__ __launch_bounds__(256) void ln_fwd_wave(const LnFwdArgs p) {
    constexpr int K = V <= 4 ? V : 1;
    const int s = threadIdx.x % L, C = p.C;
    const LnLane<V, kTiny> u(s, L, C);
    float gk[K][4], bk[K][4];
    if (V <= 4) {
#pragma unroll
        for (int j = 0; j < K; ++j) {
            u.load(p.gamma, j, gk[j]);
            u.load(p.beta, j, bk[j]);
        }
    }
    const int step = gridDim.x * (256 / L);
    for (int64_t r = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L; r < p.rows; r += step) {
        float v[V][4];
#pragma unroll
        for (int j = 0; j < V; ++j) u.load(p.x + (size_t)r * C, j, v[j]);
        ln_fwd_row(p, r, u, v, s == 0, [](float a) { return ln_group_sum<L>(a); },
                   [&](int j, float* g, float* b) {
                       if (V <= 4) {
#pragma unroll
                           for (int e = 0; e < 4; ++e) {
                               g[e] = gk[V <= 4 ? j : 0][e];
                               b[e] = bk[V <= 4 ? j : 0][e];
                           }
                       } else {
                           u.load(p.gamma, j, g);
                           u.load(p.beta, j, b);
                       }
                   });
    }
}

// Longer rows, up to blockDim V units: a row per workgroup.
template <int T, int V>
__global__ __launch_bounds__(T) void ln_fwd_block(const LnFwdArgs p) {
    __shared__ float red[2][2][16];
    LnTeam team(red);
    const int C = p.C;
    const LnLane<V> u(threadIdx.x, blockDim.x, C);
    for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        float v[V][4];
#pragma unroll
        for (int j = 0; j < V; ++j) u.load(p.x + (size_t)r * C, j, v[j]);
        ln_fwd_row(p, r, u, v, threadIdx.x == 0, [&](float a) { team.sum<1>(&a); return a; },
                   [&](int j, float* g, float* b) {
                       u.load(p.gamma, j, g);
                       u.load(p.beta, j, b);
                   });
    }
}

// Rows of any length: three passes over the row.  The sums are 64-bit (float32, a thread adding its columns in line, gave a row of 2^20
// times 1000.3 the mean 1000.3087).  Bound: 4-byte loads of one workgroup a row: 128 x 200704 116 us (159 on tensors that no cache holds;
// 39 at the rate of a copy), 1 x 200704 55.
__global__ __launch_bounds__(kLnLong) void ln_fwd_rows(const LnFwdArgs p) {
    __shared__ double red[kLnLong / 64];
    const int C = p.C;
    for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const float* xr = p.x + (size_t)r * C;
        double s[1], q[1];
        ln_long_sum<1>(C, s, [&](int64_t c, float* v) { v[0] = xr[c]; });
        const float mean = (float)(ln_block_sum(s[0], red) / C);
        ln_long_sum<1>(C, q, [&](int64_t c, float* v) { v[0] = (xr[c] - mean) * (xr[c] - mean); });
        const float invstd = 1.0f / sqrtf((float)(ln_block_sum(q[0], red) / C) + p.eps);
        if (threadIdx.x == 0 && p.mean != nullptr) {
            p.mean[r] = mean;
            p.invstd[r] = invstd;
        }
        for (int64_t c = threadIdx.x; c < C; c += kLnLong) {
            const float v = (xr[c] - mean) * invstd * p.gamma[c] + p.beta[c];
            p.y[(size_t)r * C + c] = v;
            if (p.y16 != nullptr) p.y16[(size_t)r * C + c] = (uint16_t)ln_bf16(v);
        }
    }
}

// ---- backward ----------------------------------------------------------------------------------------------------------
// Bound: HBM, 12 bytes an element (14 with the bfloat16 copy): 65536 x 1024 152 us = 5.3 TB/s, 802816 x 64 115 us = 5.4 TB/s, ragged
// rows 4.6-5.2 TB/s; a short call (5003 x 1537, 92 MB, 22 us) pays for two launches.  x and dy are read once: the same lanes hold the row
// while its two sums are taken, and the lane that owns a column adds its dy xhat and dy over all rows it sees.  A workgroup walks many
// rows and leaves a partial row of dgamma and one of dbeta for every kLnRun rows of a lane, part[piece][block][2][C]; ln_bwd_finish adds
// those in order.
// Few rows: one launch (part == NULL), in which workgroups of their own read the columns a second time and write dgamma and dbeta.
struct LnBwdArgs {
    const float *x, *dy, *gamma, *mean, *invstd;
    float* dx;
    uint16_t* dx16;
    int rows, C;
    float inv_c;
    float* part;
    bool stream;
    int groups;                                          // workgroups of rows; those behind them have 32 columns each
    int pieces;                                          // partial rows a workgroup leaves, one for every kLnRun rows a lane
    float *dgamma, *dbeta;
};

// What a lane holds of a row: x and dy as loaded.
template <int V>
struct LnBwdRow {
    float x[V][4], dy[V][4], mean, invstd;
    template <bool kTiny>
    __device__ __forceinline__ void load(const LnBwdArgs& p, int64_t r, const LnLane<V, kTiny>& u) {
        const size_t at = (size_t)r * p.C;
        mean = p.mean[r];
        invstd = p.invstd[r];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            u.load(p.x + at, j, x[j]);
            u.load(p.dy + at, j, dy[j]);
        }
    }
};

// gamma of a lane's units, 0 in the places that a unit does not own: used here, it has arrived before the rows' loop (a wait for it
// inside the loop is one for the next row's loads too: 2^27 rows of one float 3.7 ms instead of 2.6).
template <int V, bool kTiny>
__device__ __forceinline__ void ln_gains(const LnBwdArgs& p, const LnLane<V, kTiny>& u, float (*gm)[4]) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
        u.load(p.gamma, j, gm[j]);
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (!u.own(j, e)) gm[j][e] = 0.f;
    }
}

// One row: its part of the column sums, and its dx.  Places that a unit does not own count 0 times in the row's sums, whatever they hold
// (an infinity times a gain of 0 would be NaN); their dx is not written, their column sums are dropped.  `sum(float*)`: two sums over the
// row's lanes.
template <int V, bool kTiny, typename Sum>
__device__ __forceinline__ void ln_bwd_row(const LnBwdArgs& p, int64_t r, const LnLane<V, kTiny>& u, LnBwdRow<V>& w,
                                           const float (*gm)[4], float (*dg)[4], float (*db)[4], Sum sum) {
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const bool own = kTiny || u.own(j, e);       // (of a tiny row other places hold 0)
            const float d = w.dy[j][e], xh = own ? (w.x[j][e] - w.mean) * w.invstd : 0.f, g = own ? d * gm[j][e] : 0.f;
            dg[j][e] = fmaf(d, xh, dg[j][e]);
            db[j][e] += d;
            s[0] += g;
            s[1] = fmaf(g, xh, s[1]);
            w.x[j][e] = xh;
            w.dy[j][e] = g;
        }
    sum(s);
    const float c1 = s[0] * p.inv_c, c2 = s[1] * p.inv_c;
    const size_t at = (size_t)r * p.C;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = w.invstd * (w.dy[j][e] - c1 - w.x[j][e] * c2);
        u.store(p.dx + at, j, v, p.stream);
        if (p.dx16 != nullptr) u.store16(p.dx16 + at, j, v);
    }
}

// dgamma and dbeta of 32 columns, every `lanes`th row a lane, the lanes in order.
__device__ __forceinline__ void ln_bwd_own_columns(const LnBwdArgs& p, int group, int lanes, float (*red)[32][33]) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, c = group * 32 + lane, cc = min(c, p.C - 1);
    float a = 0.f, b = 0.f;
#pragma unroll 8
    for (int r = w; r < p.rows; r += lanes) {
        const float g = p.dy[(size_t)r * p.C + cc];
        a = fmaf(g, (p.x[(size_t)r * p.C + cc] - p.mean[r]) * p.invstd[r], a);
        b += g;
    }
    red[0][w][lane] = a;
    red[1][w][lane] = b;
    __syncthreads();
    if (w < 2 && c < p.C) {
        float v = red[w][0][lane];
        for (int i = 1; i < lanes; ++i) v += red[w][i][lane];
        (w == 0 ? p.dgamma : p.dbeta)[c] = v;
    }
}

// Rows of at most L V units, T / L of them at a time.  Up to V = 6 the next row's loads are on their way while this row's sums are
// taken (beyond there are no registers for it; after the last row that row is read once more rather than have a branch around
// the loads).
template <int T, int L, int V, bool kTiny = false>
__global__ __launch_bounds__(T) void ln_bwd_wave(const LnBwdArgs p) {
    constexpr bool kAhead = V <= 6;
    __shared__ float red[T / 64][L * V * 4], columns[2][32][33];
    if ((int)blockIdx.x >= p.groups) return ln_bwd_own_columns(p, blockIdx.x - p.groups, T / 32, columns);
    const int s = threadIdx.x % L, C = p.C;
    const LnLane<V, kTiny> u(s, L, C);
    float gm[V][4], dg[V][4], db[V][4];
    ln_gains(p, u, gm);
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) dg[j][e] = db[j][e] = 0.f;
    const int step = p.groups * (T / L);
    int64_t r = (int64_t)blockIdx.x * (T / L) + threadIdx.x / L;
    LnBwdRow<V> next;
    if (kAhead && r < p.rows) next.load(p, r, u);
    for (int piece = 0; piece < p.pieces; ++piece) {
        const int64_t end = min((int64_t)p.rows, (int64_t)(piece + 1) * kLnRun * step);
        while (r < end) {
            LnBwdRow<V> w;
            if (kAhead) w = next;
            else w.load(p, r, u);
            const int64_t now = r;
            r += step;
            if (kAhead) next.load(p, r < p.rows ? r : now, u);
            ln_bwd_row(p, now, u, w, gm, dg, db, [](float* a) {
                a[0] = ln_group_sum<L>(a[0]);
                a[1] = ln_group_sum<L>(a[1]);
            });
        }
        if (p.part == nullptr) return;
        // the rows of a wave, then the waves in order
        float* out = p.part + ((size_t)piece * p.groups + blockIdx.x) * 2 * C;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
#pragma unroll
            for (int j = 0; j < V; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float& sum = k == 0 ? dg[j][e] : db[j][e];
                    float v = sum;
                    sum = 0.f;
#pragma unroll
                    for (int o = L; o < 64; o <<= 1) v += __shfl_xor(v, o, 64);
                    if ((threadIdx.x & 63) < L && u.own(j, e)) red[threadIdx.x >> 6][u.at(j) + e] = v;
                }
            __syncthreads();
            for (int c = threadIdx.x; c < C; c += T) {
                float v = red[0][c];
#pragma unroll
                for (int w = 1; w < T / 64; ++w) v += red[w][c];
                out[(size_t)k * C + c] = v;
            }
            __syncthreads();
        }
    }
}

// Longer rows, up to blockDim V units: a row per workgroup.  Up to V = 4 with the next row on its way and gamma in registers.
template <int T, int V>
__global__ __launch_bounds__(T) void ln_bwd_block(const LnBwdArgs p) {
    constexpr bool kAhead = V <= 4;
    __shared__ float red[2][2][16], columns[2][32][33];
    if ((int)blockIdx.x >= p.groups) return ln_bwd_own_columns(p, blockIdx.x - p.groups, blockDim.x >> 5, columns);
    LnTeam team(red);
    const int C = p.C;
    const LnLane<V> u(threadIdx.x, blockDim.x, C);
    float gm[V][4], dg[V][4], db[V][4];
    if (kAhead) ln_gains(p, u, gm);
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) dg[j][e] = db[j][e] = 0.f;
    int64_t r = blockIdx.x;
    LnBwdRow<V> next;
    if (kAhead && r < p.rows) next.load(p, r, u);
    for (int piece = 0; piece < p.pieces; ++piece) {
        const int64_t end = min((int64_t)p.rows, (int64_t)(piece + 1) * kLnRun * p.groups);
        while (r < end) {
            LnBwdRow<V> w;
            if (kAhead) {
                w = next;
            } else {
                w.load(p, r, u);
                ln_gains(p, u, gm);
            }
            const int64_t now = r;
            r += p.groups;
            if (kAhead) next.load(p, r < p.rows ? r : now, u);
            ln_bwd_row(p, now, u, w, gm, dg, db, [&](float* a) { team.sum<2>(a); });
        }
        if (p.part == nullptr) return;
        float* out = p.part + ((size_t)piece * p.groups + blockIdx.x) * 2 * C;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            u.store(out, j, dg[j], false);
            u.store(out + C, j, db[j], false);
#pragma unroll
            for (int e = 0; e < 4; ++e) dg[j][e] = db[j][e] = 0.f;
        }
    }
}

// Rows of any length: the gradient of the rows in two passes over each (sums in 64 bits), the column sums in a kernel of their own, a
// third pass.  Bound: as forward; 128 x 200704 155 us (182 + 32 on tensors that no cache holds; 58 at the rate of a copy).
__global__ __launch_bounds__(kLnLong) void ln_bwd_rows(const LnBwdArgs p) {
    __shared__ double red[kLnLong / 64];
    const int C = p.C;
    for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const size_t at = (size_t)r * C;
        const float m = p.mean[r], is = p.invstd[r];
        double s[2];
        ln_long_sum<2>(C, s, [&](int64_t c, float* v) {
            v[0] = p.dy[at + c] * p.gamma[c];
            v[1] = v[0] * ((p.x[at + c] - m) * is);
        });
        const float c1 = (float)(ln_block_sum(s[0], red) / C), c2 = (float)(ln_block_sum(s[1], red) / C);
        for (int64_t c = threadIdx.x; c < C; c += kLnLong) {
            const float v = is * (p.dy[at + c] * p.gamma[c] - c1 - (p.x[at + c] - m) * is * c2);
            p.dx[at + c] = v;
            if (p.dx16 != nullptr) p.dx16[at + c] = (uint16_t)ln_bf16(v);
        }
    }
}

// Sums of dy xhat and dy over a run of rows: 64 columns x 4 row lanes per workgroup, to part[run][2][C], or to dgamma and dbeta where one
// run has all rows (part == NULL).
__global__ __launch_bounds__(256) void ln_bwd_columns(const LnBwdArgs p, int run) {
    __shared__ float red[2][4][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, C = p.C;
    const int beg = blockIdx.y * run, end = min(p.rows, beg + run);
    for (int64_t at = (int64_t)blockIdx.x * 64; at < C; at += (int64_t)gridDim.x * 64) {
        const int64_t c = at + lane;
        float a = 0.f, b = 0.f;
        if (c < C)
            for (int r = beg + w; r < end; r += 4) {
                const float g = p.dy[(size_t)r * C + c];
                a += g * ((p.x[(size_t)r * C + c] - p.mean[r]) * p.invstd[r]);
                b += g;
            }
        __syncthreads();                                 // (the last group's sums have been read)
        red[0][w][lane] = a;
        red[1][w][lane] = b;
        __syncthreads();
        if (w < 2 && c < C) {
            float* out = p.part != nullptr ? p.part + ((size_t)blockIdx.y * 2 + w) * C : w == 0 ? p.dgamma : p.dbeta;
            out[c] = (red[w][0][lane] + red[w][1][lane]) + (red[w][2][lane] + red[w][3][lane]);
        }
    }
}

// dgamma | dbeta = the partial rows part[block][2C] added up: 32 columns (128 bytes of a row) a workgroup, 128 lanes of blocks
// each, so that all of a lane's few loads are in flight at once; then the lanes by a tree.  Fixed order.
__global__ __launch_bounds__(1024) void ln_bwd_finish(const float* __restrict__ part, int blocks, int C,
                                                      float* __restrict__ dgamma, float* __restrict__ dbeta) {
    __shared__ float red[128][33];
    const int unit = threadIdx.x & 7, w = threadIdx.x >> 3;
    const int64_t C2 = 2 * (int64_t)C;
    for (int64_t at = (int64_t)blockIdx.x * 32; at < C2; at += (int64_t)gridDim.x * 32) {
        const int64_t c = at + unit * 4;
        float a[4] = {0.f, 0.f, 0.f, 0.f};
        if (c + 4 <= C2) {
            for (int i0 = w; i0 < blocks; i0 += 512) {
                ln_f4 v[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int i = i0 + 128 * k;
                    v[k] = i < blocks ? *reinterpret_cast<const ln_f4*>(part + i * C2 + c) : ln_f4{0.f, 0.f, 0.f, 0.f};
                }
#pragma unroll
                for (int k = 0; k < 4; ++k)
#pragma unroll
                    for (int e = 0; e < 4; ++e) a[e] += v[k][e];
            }
        } else {                                         // (the last two columns of an odd C)
            for (int i = w; i < blocks; i += 128)
#pragma unroll
                for (int e = 0; e < 4; ++e) a[e] += c + e < C2 ? part[i * C2 + c + e] : 0.f;
        }
        __syncthreads();                                 // (the last group's sums have been read)
#pragma unroll
        for (int e = 0; e < 4; ++e) red[w][unit * 4 + e] = a[e];
        __syncthreads();
        const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int col = wave * 2 + h;
            const int64_t k = at + col;
            const float v = ln_group_sum<64>(red[lane][col] + red[lane + 64][col]);
            if (lane == 0 && k < C2) {
                if (k < C) dgamma[k] = v;
                else dbeta[k - C] = v;
            }
        }
    }
}

// A launch's threads along one axis stay below 2^32.
constexpr int kLnMostGroups = 1 << 20;

// Tensors of a call; no output may overlap another output or an input.
struct LnSpan {
    const void* p;
    int64_t bytes;
};
template <int W, int R>
static bool ln_apart(const LnSpan (&written)[W], const LnSpan (&read)[R]) {
    const auto apart = [](const LnSpan& a, const LnSpan& b) {
        const char *p = (const char*)a.p, *q = (const char*)b.p;
        return p == nullptr || q == nullptr || a.bytes == 0 || b.bytes == 0 || p + a.bytes <= q || q + b.bytes <= p;
    };
    for (int i = 0; i < W; ++i) {
        for (int j = 0; j < i; ++j)
            if (!apart(written[i], written[j])) return false;
        for (int j = 0; j < R; ++j)
            if (!apart(written[i], read[j])) return false;
    }
    return true;
}

// How a row is laid over lanes: the way with the fewest idle places, and of those the one with the most lanes (802816 x 64 backward:
// 16 lanes of one unit 114 us, 4 of four 123).  Up to 512 units (2048 columns) a row has L lanes of a wave, beyond a workgroup of
// whole waves, as long as `most` units a lane allow; there, of equals, the fewest waves.
// Idle places cost what used ones do: 65536 x 1028 forward took 200 us on 256 lanes of two units, half of them idle, where
// 65536 x 1024 took 97.
struct LnShape {
    int lanes;                                           // of a wave; 0: a workgroup a row; -1: rows of any length
    int v, threads;
    bool tiny;
};
static LnShape ln_shape(int C, int most_threads, int most) {
    const int units = cdiv(C, 4);
    if (C < 4) return LnShape{4, 1, 0, true};
    LnShape best{-1, 0, kLnLong, false};
    if (units <= 512) {
        for (int lanes = 64; lanes >= 4; lanes >>= 1) {
            const int v = cdiv(units, lanes);
            if (v <= (lanes == 64 ? 8 : 4) && (best.lanes < 0 || lanes * v < best.lanes * best.v)) best = LnShape{lanes, v, 0, false};
        }
        return best;
    }
    for (int v = 1; v <= most; ++v) {
        const int threads = cdiv(cdiv(units, v), 64) * 64;
        if (threads <= most_threads && (best.lanes < 0 || threads * v <= best.threads * best.v)) best = LnShape{0, v, threads, false};
    }
    return best;
}

typedef void (*LnFwd)(const LnFwdArgs);
typedef void (*LnBwd)(const LnBwdArgs);

// Of fewer than 64 lanes ln_shape takes one unit or three (two and four are one and two of twice the lanes).
template <int L>
static LnFwd ln_fwd_wave_of(int v) {
    return v == 1 ? ln_fwd_wave<L, 1> : ln_fwd_wave<L, 3>;
}
static LnFwd ln_fwd_kernel(const LnShape& s) {
    static const LnFwd wave[8] = {ln_fwd_wave<64, 1>, ln_fwd_wave<64, 2>, ln_fwd_wave<64, 3>, ln_fwd_wave<64, 4>,
                                  ln_fwd_wave<64, 5>, ln_fwd_wave<64, 6>, ln_fwd_wave<64, 7>, ln_fwd_wave<64, 8>};
    static const LnFwd block[4] = {ln_fwd_block<512, 5>, ln_fwd_block<512, 6>, ln_fwd_block<512, 7>, ln_fwd_block<512, 8>};
    static const LnFwd large[4] = {ln_fwd_block<1024, 5>, ln_fwd_block<1024, 6>, ln_fwd_block<1024, 7>, ln_fwd_block<1024, 8>};
    if (s.tiny) return ln_fwd_wave<4, 1, true>;
    switch (s.lanes) {
        case 4: return ln_fwd_wave_of<4>(s.v);
        case 8: return ln_fwd_wave_of<8>(s.v);
        case 16: return ln_fwd_wave_of<16>(s.v);
        case 32: return ln_fwd_wave_of<32>(s.v);
        case 64: return wave[s.v - 1];
        case 0: return s.v == 3 ? ln_fwd_block<512, 3> : s.threads <= 512 ? block[s.v - 5] : large[s.v - 5];
    }
    return ln_fwd_rows;
}

constexpr int kLnBwdWaveThreads = 512;
template <int L>
static LnBwd ln_bwd_wave_of(int v) {
    return v == 1 ? ln_bwd_wave<kLnBwdWaveThreads, L, 1> : ln_bwd_wave<kLnBwdWaveThreads, L, 3>;
}
static LnBwd ln_bwd_kernel(const LnShape& s) {
    constexpr int T = kLnBwdWaveThreads;
    static const LnBwd wave[8] = {ln_bwd_wave<T, 64, 1>, ln_bwd_wave<T, 64, 2>, ln_bwd_wave<T, 64, 3>, ln_bwd_wave<T, 64, 4>,
                                  ln_bwd_wave<T, 64, 5>, ln_bwd_wave<T, 64, 6>, ln_bwd_wave<T, 64, 7>, ln_bwd_wave<T, 64, 8>};
    static const LnBwd ahead[3] = {ln_bwd_block<512, 2>, ln_bwd_block<512, 3>, ln_bwd_block<512, 4>};
    static const LnBwd block[3] = {ln_bwd_block<512, 6>, ln_bwd_block<512, 7>, ln_bwd_block<512, 8>};
    if (s.tiny) return ln_bwd_wave<T, 4, 1, true>;
    switch (s.lanes) {
        case 4: return ln_bwd_wave_of<4>(s.v);
        case 8: return ln_bwd_wave_of<8>(s.v);
        case 16: return ln_bwd_wave_of<16>(s.v);
        case 32: return ln_bwd_wave_of<32>(s.v);
        case 64: return wave[s.v - 1];
        case 0:
            if (s.threads > 512) return s.v == 6 ? ln_bwd_block<768, 6> : ln_bwd_block<768, 7>;
            return s.v <= 4 ? ahead[s.v - 2] : block[s.v - 6];
    }
    return nullptr;                                      // (rows of any length: ln_bwd_rows and ln_bwd_columns)
}

// Backward: with the next row on its way where that fits 512 threads, else without; then 768 threads, whose 168 registers take up to
// seven units.
static LnShape ln_bwd_shape(int C) {
    LnShape s = ln_shape(C, 512, 4);
    if (s.lanes < 0) s = ln_shape(C, 512, 8);
    if (s.lanes < 0) s = ln_shape(C, 768, 7);
    return s;
}
static LnShape ln_fwd_shape(int C) {
    LnShape s = ln_shape(C, 512, 8);
    if (s.lanes < 0) s = ln_shape(C, 1024, 8);
    return s;
}

// The arguments are checked before the context: a bad call is refused alike with and without a GPU.
static int ln_fwd_impl(const float* x, const float* gamma, const float* beta, float* save_mean, float* save_invstd, float* y,
                       uint16_t* y16, int rows, int C, float eps) {
    AETH_CHECK_ARG(rows >= 0 && C > 0 && (int64_t)rows * C < ((int64_t)1 << 31));
    AETH_CHECK_ARG(eps >= 0.f);
    AETH_CHECK_ARG((save_mean == nullptr) == (save_invstd == nullptr));
    AETH_CHECK_ARG(rows == 0 || (x && gamma && beta && y));
    const int64_t n = (int64_t)rows * C;
    const int64_t r4 = 4 * (int64_t)rows, c4 = rows ? 4 * (int64_t)C : 0;
    const LnSpan written[] = {{y, 4 * n}, {y16, 2 * n}, {save_mean, r4}, {save_invstd, r4}};
    const LnSpan read[] = {{x, 4 * n}, {gamma, c4}, {beta, c4}};
    AETH_CHECK_ARG(ln_apart(written, read));
    AETH_REQUIRE_INIT();
    if (rows == 0) return AETH_OK;
    const LnShape s = ln_fwd_shape(C);
    const int threads = s.lanes > 0 ? 256 : s.threads, turns = s.lanes > 0 ? cdiv(rows, 256 / s.lanes) : rows;
    // workgroups that walk the rows, 1024 threads a CU: 16384 x 8192 took 204 us with 1024 workgroups of 256 threads, 207 with
    // 4096, 218 with one a row; pixels x64 with twin 95.7, 98.6, 98.9
    const int cap = 256 * 1024 / threads;
    const LnFwdArgs p{x, gamma, beta, save_mean, save_invstd, y, y16, rows, C, 1.0f / (float)C, eps, 4 * n >= kLnStreamBytes};
    hipLaunchKernelGGL(ln_fwd_kernel(s), dim3(turns < cap ? turns : cap), dim3(threads), 0, ctx().stream, p);
    AETH_LAUNCH_CHECK();
    return AETH_OK;
}

static int ln_bwd_impl(const float* x, const float* dy, const float* gamma, const float* mean, const float* invstd, float* dx,
                       uint16_t* dx16, float* dgamma, float* dbeta, int rows, int C) {
    AETH_CHECK_ARG(rows >= 0 && C > 0 && (int64_t)rows * C < ((int64_t)1 << 31));
    AETH_CHECK_ARG(dgamma && dbeta && (rows == 0 || (x && dy && gamma && mean && invstd && dx)));
    const int64_t n = (int64_t)rows * C;
    const int64_t r4 = 4 * (int64_t)rows, c4 = 4 * (int64_t)C;
    const LnSpan written[] = {{dx, 4 * n}, {dx16, 2 * n}, {dgamma, c4}, {dbeta, c4}};
    const LnSpan read[] = {{x, 4 * n}, {dy, 4 * n}, {gamma, rows ? c4 : 0}, {mean, r4}, {invstd, r4}};
    AETH_CHECK_ARG(ln_apart(written, read));
    AETH_REQUIRE_INIT();
    hipStream_t st = ctx().stream;
    int blocks = 0;
    void* ws = nullptr;
    if (rows > 0) {
        const LnShape s = ln_bwd_shape(C);
        int threads = s.threads, turns = rows, cap = 0;
        if (s.lanes > 0) {
            threads = kLnBwdWaveThreads;
            turns = cdiv(rows, threads / s.lanes);
            cap = 256;                                   // (pixels x64 with twin: 512 workgroups 143 us, 256 129)
        } else if (s.lanes == 0) {
            // whole workgroups a CU, 512 threads of them (16384 x 5000: 182 us with 512 threads a CU, 193 with 640 and 768, 197 with
            // 1024; 4096 x 16384: 171, 171, 170, 183); more leave more partial rows, a part of one leaves CUs idle
            cap = 256 * (threads < 512 ? 512 / threads : 1);
        }
        // One launch for few rows: 128 x 256 3.1 us instead of 5.6, 512 x 256 4.1 and 5.6, 512 x 2048 5.4 and 9.3, 128 x 8192 6.0 and 12.4,
        // 256 x 20000 27 and 36; but a column's rows are one workgroup's: 1024 x 256 6.3 and 5.8, 512 x 8192 18 and 17 (repeated on the
        // same tensors; on rotating ones 128 x 256 3.6 instead of 7.5)
        if (s.lanes >= 0 && rows <= (s.lanes > 0 ? 512 : 256)) {
            const LnBwdArgs p{x, dy, gamma, mean, invstd, dx, dx16, rows, C, 1.0f / (float)C, nullptr, 4 * n >= kLnStreamBytes, turns, 1, dgamma,
                              dbeta};
            hipLaunchKernelGGL(ln_bwd_kernel(s), dim3(turns + cdiv(C, 32)), dim3(threads), 0, st, p);
            AETH_LAUNCH_CHECK();
            return AETH_OK;
        }
        if (s.lanes < 0) {
            // runs for eight workgroups a CU, as far as the columns leave too few, of 16 rows at least (a partial row each: an eighth of
            // the tensor's bytes at most) and 512 at most (128 a lane)
            const int columns = cdiv(C, 64), run = std::min(std::max(cdiv(rows, cdiv(2048, columns)), 16), 512);
            blocks = cdiv(rows, run);
            if (blocks > 1) {
                const int rc = workspace((int64_t)2 * blocks * C * sizeof(float), &ws);
                if (rc) return rc;
            }
            const LnBwdArgs p{x, dy, gamma, mean, invstd, dx, dx16, rows, C, 1.0f / (float)C, (float*)ws, false, 0, 0, dgamma, dbeta};
            hipLaunchKernelGGL(ln_bwd_rows, dim3(rows < 4096 ? rows : 4096), dim3(threads), 0, st, p);
            AETH_LAUNCH_CHECK();
            hipLaunchKernelGGL(ln_bwd_columns, dim3(columns < kLnMostGroups ? columns : kLnMostGroups, blocks), dim3(256), 0, st, p, run);
            AETH_LAUNCH_CHECK();
            if (blocks == 1) return AETH_OK;
        } else {
            // as many workgroups as are needed for each to take no more rows than with `cap` of them
            const int run = cdiv(turns, cap), groups = cdiv(turns, run), pieces = cdiv(run, kLnRun);
            blocks = groups * pieces;
            const int rc = workspace((int64_t)2 * blocks * C * sizeof(float), &ws);
            if (rc) return rc;
            const LnBwdArgs p{x, dy, gamma, mean, invstd, dx, dx16, rows, C, 1.0f / (float)C, (float*)ws, 4 * n >= kLnStreamBytes, groups,
                              pieces, nullptr, nullptr};
            hipLaunchKernelGGL(ln_bwd_kernel(s), dim3(groups), dim3(threads), 0, st, p);
            AETH_LAUNCH_CHECK();
        }
    }
    const int groups = cdiv(2 * (int64_t)C, 32);
    hipLaunchKernelGGL(ln_bwd_finish, dim3(groups < kLnMostGroups ? groups : kLnMostGroups), dim3(1024), 0, st, (const float*)ws, blocks,
                       C, dgamma, dbeta);
    AETH_LAUNCH_CHECK();
    return AETH_OK;
}

}  // namespace aeth

using namespace aeth;

extern "C" {

int aeth_ln_fwd_f32(const float* x, const float* gamma, const float* beta, float* save_mean, float* save_invstd, float* y,
                    int rows, int C, float eps) {
    return ln_fwd_impl(x, gamma, beta, save_mean, save_invstd, y, nullptr, rows, C, eps);
}

int aeth_ln_fwd_twin_f32(const float* x, const float* gamma, const float* beta, float* save_mean, float* save_invstd,
                         float* y, uint16_t* y_bf16, int rows, int C, float eps) {
    AETH_CHECK_ARG(y_bf16 != nullptr || rows == 0);
    return ln_fwd_impl(x, gamma, beta, save_mean, save_invstd, y, y_bf16, rows, C, eps);
}

int aeth_ln_bwd_f32(const float* x, const float* dy, const float* gamma, const float* save_mean, const float* save_invstd,
                    float* dx, float* dgamma, float* dbeta, int rows, int C) {
    return ln_bwd_impl(x, dy, gamma, save_mean, save_invstd, dx, nullptr, dgamma, dbeta, rows, C);
}

int aeth_ln_bwd_twin_f32(const float* x, const float* dy, const float* gamma, const float* save_mean,
                         const float* save_invstd, float* dx, uint16_t* dx_bf16, float* dgamma, float* dbeta, int rows,
                         int C) {
    AETH_CHECK_ARG(dx_bf16 != nullptr || rows == 0);
    return ln_bwd_impl(x, dy, gamma, save_mean, save_invstd, dx, dx_bf16, dgamma, dbeta, rows, C);
}

}  // extern "C"
