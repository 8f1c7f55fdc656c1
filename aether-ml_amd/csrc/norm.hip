// Layer norm over the last axis of a row-major [rows, C] tensor, forward and backward.
//
//   mean_r = sum_c x / C,  var_r = sum_c (x - mean_r)^2 / C,  invstd_r = 1 / sqrt(var_r + eps)
//   y = (x - mean_r) invstd_r gamma_c + beta_c
//
//   xhat = (x - mean_r) invstd_r,  g = dy gamma_c
//   dx = invstd_r (g - sum_c g / C - xhat sum_c g xhat / C)
//   dgamma_c = sum_r dy xhat,  dbeta_c = sum_r dy
//
// All sums are float32 in a fixed order: results do not depend on timing.
#include "common.h"

#include <initializer_list>

namespace aeth {

constexpr int kLnThreads = 256;
constexpr int kLnGrid = 8192;

// float32 -> bfloat16 bits, round to nearest even; NaN stays NaN
__device__ __forceinline__ unsigned ln_bf16(float f) {
    const unsigned u = __float_as_uint(f);
    if ((u & 0x7fffffffu) > 0x7f800000u) return (u >> 16) | 0x40u;
    return (u + 0x7fffu + ((u >> 16) & 1u)) >> 16;
}

typedef float ln_f4 __attribute__((ext_vector_type(4)));

// W consecutive floats (16-byte aligned for W = 4)
template <int W>
__device__ __forceinline__ void ln_load(const float* __restrict__ p, float* v) {
    if (W == 4) {
        const ln_f4 t = *reinterpret_cast<const ln_f4*>(p);
#pragma unroll
        for (int e = 0; e < W; ++e) v[e] = t[e];
    } else {
        v[0] = *p;
    }
}

template <int W>
__device__ __forceinline__ void ln_store(float* __restrict__ p, const float* v) {
    if (W == 4) *reinterpret_cast<ln_f4*>(p) = ln_f4{v[0], v[1], v[2], v[3]};
    else *p = v[0];
}

template <int W>
__device__ __forceinline__ void ln_store16(uint16_t* __restrict__ p, const float* v) {
    if (W == 4) {
        const unsigned lo = ln_bf16(v[0]) | (ln_bf16(v[1]) << 16), hi = ln_bf16(v[2]) | (ln_bf16(v[3]) << 16);
        *reinterpret_cast<uint2*>(p) = uint2{lo, hi};
    } else {
        *p = (uint16_t)ln_bf16(v[0]);
    }
}

// Sum over aligned groups of L lanes, the same value in every lane of the group: within 16 lanes by the cross-lane paths of
// the vector unit, beyond by swapping halves.
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

// Sum over the workgroup's T threads, the same value in every thread.  Two slots of `red`, used in turn, need one barrier a
// sum: a wave can be at most one barrier ahead of the slowest.
template <int T>
__device__ __forceinline__ float ln_block_sum(float v, float (*red)[T / 64], int& turn) {
    v = ln_group_sum<64>(v);
    if ((threadIdx.x & 63) == 0) red[turn][threadIdx.x >> 6] = v;
    __syncthreads();
    float s = red[turn][0];
#pragma unroll
    for (int w = 1; w < T / 64; ++w) s += red[turn][w];
    turn ^= 1;
    return s;
}

// ---- forward -----------------------------------------------------------------------------------------------------------
// Bound: HBM, 8 bytes an element (10 with the bfloat16 copy).  A row is read once and stays in registers: lane s of the row's
// L lanes (or of the workgroup's T threads) holds the W-float units s, s + L, ... (V of them); the mean, then the sum of
// squares of what is left, then the output, so that no cancellation of two large sums enters the variance.
// Units are 16 bytes where C and every pointer allow it, 4 bytes otherwise.

// Rows of at most 64 V units: a row per L lanes, 256 / L rows a workgroup; gamma and beta stay in registers over the rows.
template <int L, int V, int W>
__global__ __launch_bounds__(256) void ln_fwd_wave(const float* __restrict__ x, const float* __restrict__ gamma,
                                                   const float* __restrict__ beta, float* __restrict__ save_mean,
                                                   float* __restrict__ save_invstd, float* __restrict__ y,
                                                   uint16_t* __restrict__ y16, int rows, int C, float eps) {
    const int s = threadIdx.x % L;
    float g[V][W], b[V][W];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int c = (s + L * j) * W;
        if (c < C) {
            ln_load<W>(gamma + c, g[j]);
            ln_load<W>(beta + c, b[j]);
        }
    }
    const int step = gridDim.x * (256 / L);
    for (int64_t r = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L; r < rows; r += step) {
        const size_t at = (size_t)r * C;
        float v[V][W], sum = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int c = (s + L * j) * W;
            if (c < C) ln_load<W>(x + at + c, v[j]);
#pragma unroll
            for (int e = 0; e < W; ++e) {
                if (c >= C) v[j][e] = 0.f;
                sum += v[j][e];
            }
        }
        const float mean = ln_group_sum<L>(sum) / (float)C;
        float q = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const bool in = (s + L * j) * W < C;
#pragma unroll
            for (int e = 0; e < W; ++e) {
                v[j][e] -= mean;
                q += in ? v[j][e] * v[j][e] : 0.f;
            }
        }
        const float invstd = 1.0f / sqrtf(ln_group_sum<L>(q) / (float)C + eps);
        if (save_mean != nullptr && s == 0) {
            save_mean[r] = mean;
            save_invstd[r] = invstd;
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int c = (s + L * j) * W;
            if (c < C) {
#pragma unroll
                for (int e = 0; e < W; ++e) v[j][e] = v[j][e] * invstd * g[j][e] + b[j][e];
                ln_store<W>(y + at + c, v[j]);
                if (y16 != nullptr) ln_store16<W>(y16 + at + c, v[j]);
            }
        }
    }
}

// Longer rows, up to T V units: a row per workgroup.
template <int T, int V, int W>
__global__ __launch_bounds__(T) void ln_fwd_block(const float* __restrict__ x, const float* __restrict__ gamma,
                                                  const float* __restrict__ beta, float* __restrict__ save_mean,
                                                  float* __restrict__ save_invstd, float* __restrict__ y,
                                                  uint16_t* __restrict__ y16, int rows, int C, float eps) {
    __shared__ float red[2][T / 64];
    int turn = 0;
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const size_t at = (size_t)r * C;
        float v[V][W], sum = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int c = (threadIdx.x + T * j) * W;
            if (c < C) ln_load<W>(x + at + c, v[j]);
#pragma unroll
            for (int e = 0; e < W; ++e) {
                if (c >= C) v[j][e] = 0.f;
                sum += v[j][e];
            }
        }
        const float mean = ln_block_sum<T>(sum, red, turn) / (float)C;
        float q = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const bool in = (int)(threadIdx.x + T * j) * W < C;
#pragma unroll
            for (int e = 0; e < W; ++e) {
                v[j][e] -= mean;
                q += in ? v[j][e] * v[j][e] : 0.f;
            }
        }
        const float invstd = 1.0f / sqrtf(ln_block_sum<T>(q, red, turn) / (float)C + eps);
        if (save_mean != nullptr && threadIdx.x == 0) {
            save_mean[r] = mean;
            save_invstd[r] = invstd;
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int c = (threadIdx.x + T * j) * W;
            if (c < C) {
                float g[W], b[W];
                ln_load<W>(gamma + c, g);
                ln_load<W>(beta + c, b);
#pragma unroll
                for (int e = 0; e < W; ++e) v[j][e] = v[j][e] * invstd * g[e] + b[e];
                ln_store<W>(y + at + c, v[j]);
                if (y16 != nullptr) ln_store16<W>(y16 + at + c, v[j]);
            }
        }
    }
}

// Rows of any length: three passes over the row.
__global__ __launch_bounds__(kLnThreads) void ln_fwd_rows(const float* __restrict__ x, const float* __restrict__ gamma,
                                                          const float* __restrict__ beta, float* __restrict__ save_mean,
                                                          float* __restrict__ save_invstd, float* __restrict__ y,
                                                          uint16_t* __restrict__ y16, int rows, int C, float eps) {
    __shared__ float red[2][kLnThreads / 64];
    int turn = 0;
    for (int r = blockIdx.x; r < rows; r += gridDim.x) {
        const float* xr = x + (size_t)r * C;
        float s = 0.f;
        for (int c = threadIdx.x; c < C; c += kLnThreads) s += xr[c];
        const float mean = ln_block_sum<kLnThreads>(s, red, turn) / (float)C;
        float q = 0.f;
        for (int c = threadIdx.x; c < C; c += kLnThreads) {
            const float d = xr[c] - mean;
            q += d * d;
        }
        const float invstd = 1.0f / sqrtf(ln_block_sum<kLnThreads>(q, red, turn) / (float)C + eps);
        if (threadIdx.x == 0 && save_mean != nullptr) {
            save_mean[r] = mean;
            save_invstd[r] = invstd;
        }
        for (int c = threadIdx.x; c < C; c += kLnThreads) {
            const float v = (xr[c] - mean) * invstd * gamma[c] + beta[c];
            y[(size_t)r * C + c] = v;
            if (y16 != nullptr) y16[(size_t)r * C + c] = (uint16_t)ln_bf16(v);
        }
    }
}

// ---- backward ----------------------------------------------------------------------------------------------------------
// Bound: HBM, 12 bytes an element (14 with the bfloat16 copy).  x and dy are read once: the same lanes hold the row while its
// two sums are taken, and the lane that owns a column adds its dy xhat and dy over all rows it sees.  A workgroup walks many
// rows and leaves one partial row of dgamma and one of dbeta, part[block][2][C]; ln_bwd_finish adds those in block order.

// Rows of at most 64 V units, as ln_fwd_wave; T / L rows at a time.
template <int T, int L, int V, int W>
__global__ __launch_bounds__(T) void ln_bwd_wave(const float* __restrict__ x, const float* __restrict__ dy,
                                                 const float* __restrict__ gamma, const float* __restrict__ mean,
                                                 const float* __restrict__ invstd, float* __restrict__ dx,
                                                 uint16_t* __restrict__ dx16, int rows, int C, float* __restrict__ part) {
    __shared__ float red[T / 64][L * V * W];
    const int s = threadIdx.x % L;
    float gm[V][W], dg[V][W], db[V][W];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int c = (s + L * j) * W;
#pragma unroll
        for (int e = 0; e < W; ++e) dg[j][e] = db[j][e] = gm[j][e] = 0.f;
        if (c < C) ln_load<W>(gamma + c, gm[j]);
    }
    const int step = gridDim.x * (T / L);
    for (int64_t r = (int64_t)blockIdx.x * (T / L) + threadIdx.x / L; r < rows; r += step) {
        const size_t at = (size_t)r * C;
        const float m = mean[r], is = invstd[r];
        float xh[V][W], g[V][W], s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int c = (s + L * j) * W;
            if (c < C) {
                ln_load<W>(x + at + c, xh[j]);
                ln_load<W>(dy + at + c, g[j]);
            }
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const bool in = (s + L * j) * W < C;
#pragma unroll
            for (int e = 0; e < W; ++e) {
                xh[j][e] = in ? (xh[j][e] - m) * is : 0.f;
                const float d = in ? g[j][e] : 0.f;
                dg[j][e] += d * xh[j][e];
                db[j][e] += d;
                g[j][e] = d * gm[j][e];
                s1 += g[j][e];
                s2 += g[j][e] * xh[j][e];
            }
        }
        const float c1 = ln_group_sum<L>(s1) / (float)C, c2 = ln_group_sum<L>(s2) / (float)C;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int c = (s + L * j) * W;
            if (c < C) {
                float v[W];
#pragma unroll
                for (int e = 0; e < W; ++e) v[e] = is * (g[j][e] - c1 - xh[j][e] * c2);
                ln_store<W>(dx + at + c, v);
                if (dx16 != nullptr) ln_store16<W>(dx16 + at + c, v);
            }
        }
    }
    // the rows of a wave, then the waves in order
    float* out = part + (size_t)blockIdx.x * 2 * C;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
        for (int j = 0; j < V; ++j)
#pragma unroll
            for (int e = 0; e < W; ++e) {
                float v = k == 0 ? dg[j][e] : db[j][e];
#pragma unroll
                for (int o = L; o < 64; o <<= 1) v += __shfl_xor(v, o, 64);
                if ((threadIdx.x & 63) < L) red[threadIdx.x >> 6][(s + L * j) * W + e] = v;
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

// Longer rows, up to T V units: a row per workgroup.
template <int T, int V, int W>
__global__ __launch_bounds__(T) void ln_bwd_block(const float* __restrict__ x, const float* __restrict__ dy,
                                                  const float* __restrict__ gamma, const float* __restrict__ mean,
                                                  const float* __restrict__ invstd, float* __restrict__ dx,
                                                  uint16_t* __restrict__ dx16, int rows, int C, float* __restrict__ part) {
    __shared__ float red1[2][T / 64], red2[2][T / 64];
    int turn = 0;
    float dg[V][W], db[V][W];
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
        for (int e = 0; e < W; ++e) dg[j][e] = db[j][e] = 0.f;
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const size_t at = (size_t)r * C;
        const float m = mean[r], is = invstd[r];
        float xh[V][W], g[V][W], s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int c = (threadIdx.x + T * j) * W;
            if (c < C) {
                ln_load<W>(x + at + c, xh[j]);
                ln_load<W>(dy + at + c, g[j]);
            }
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int c = (threadIdx.x + T * j) * W;
            float gm[W];
            if (c < C) ln_load<W>(gamma + c, gm);
#pragma unroll
            for (int e = 0; e < W; ++e) {
                xh[j][e] = c < C ? (xh[j][e] - m) * is : 0.f;
                const float d = c < C ? g[j][e] : 0.f;
                dg[j][e] += d * xh[j][e];
                db[j][e] += d;
                g[j][e] = c < C ? d * gm[e] : 0.f;
                s1 += g[j][e];
                s2 += g[j][e] * xh[j][e];
            }
        }
        // (both sums behind one barrier; the slots are used in turn as in ln_block_sum)
        s1 = ln_group_sum<64>(s1);
        s2 = ln_group_sum<64>(s2);
        if ((threadIdx.x & 63) == 0) {
            red1[turn][threadIdx.x >> 6] = s1;
            red2[turn][threadIdx.x >> 6] = s2;
        }
        __syncthreads();
        s1 = red1[turn][0];
        s2 = red2[turn][0];
#pragma unroll
        for (int w = 1; w < T / 64; ++w) {
            s1 += red1[turn][w];
            s2 += red2[turn][w];
        }
        turn ^= 1;
        const float c1 = s1 / (float)C, c2 = s2 / (float)C;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int c = (threadIdx.x + T * j) * W;
            if (c < C) {
                float v[W];
#pragma unroll
                for (int e = 0; e < W; ++e) v[e] = is * (g[j][e] - c1 - xh[j][e] * c2);
                ln_store<W>(dx + at + c, v);
                if (dx16 != nullptr) ln_store16<W>(dx16 + at + c, v);
            }
        }
    }
    float* out = part + (size_t)blockIdx.x * 2 * C;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int c = (threadIdx.x + T * j) * W;
        if (c < C) {
            if (W == 4 && (reinterpret_cast<uintptr_t>(out) & 15) == 0) {
                ln_store<W>(out + c, dg[j]);
                ln_store<W>(out + C + c, db[j]);
            } else {
#pragma unroll
                for (int e = 0; e < W; ++e) {
                    out[c + e] = dg[j][e];
                    out[C + c + e] = db[j][e];
                }
            }
        }
    }
}

// Rows of any length: the gradient of the rows in two passes, the column sums in a kernel of their own.
__global__ __launch_bounds__(kLnThreads) void ln_bwd_rows(const float* __restrict__ x, const float* __restrict__ dy,
                                                          const float* __restrict__ gamma, const float* __restrict__ mean,
                                                          const float* __restrict__ invstd, float* __restrict__ dx,
                                                          uint16_t* __restrict__ dx16, int rows, int C) {
    __shared__ float red[2][kLnThreads / 64];
    int turn = 0;
    for (int r = blockIdx.x; r < rows; r += gridDim.x) {
        const size_t at = (size_t)r * C;
        const float m = mean[r], is = invstd[r];
        float s1 = 0.f, s2 = 0.f;
        for (int c = threadIdx.x; c < C; c += kLnThreads) {
            const float g = dy[at + c] * gamma[c];
            s1 += g;
            s2 += g * ((x[at + c] - m) * is);
        }
        const float c1 = ln_block_sum<kLnThreads>(s1, red, turn) / (float)C;
        const float c2 = ln_block_sum<kLnThreads>(s2, red, turn) / (float)C;
        for (int c = threadIdx.x; c < C; c += kLnThreads) {
            const float v = is * (dy[at + c] * gamma[c] - c1 - (x[at + c] - m) * is * c2);
            dx[at + c] = v;
            if (dx16 != nullptr) dx16[at + c] = (uint16_t)ln_bf16(v);
        }
    }
}

// Partial sums of dy xhat and dy over a run of rows: 64 columns x 4 row lanes per workgroup, part[run][2][C].
__global__ __launch_bounds__(kLnThreads) void ln_bwd_columns(const float* __restrict__ x, const float* __restrict__ dy,
                                                             const float* __restrict__ mean,
                                                             const float* __restrict__ invstd, int rows, int C, int run,
                                                             float* __restrict__ part) {
    __shared__ float red[2][4][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int c = blockIdx.x * 64 + lane;
    const int beg = blockIdx.y * run, end = min(rows, beg + run);
    float a = 0.f, b = 0.f;
    if (c < C)
        for (int r = beg + w; r < end; r += 4) {
            const float g = dy[(size_t)r * C + c];
            a += g * ((x[(size_t)r * C + c] - mean[r]) * invstd[r]);
            b += g;
        }
    red[0][w][lane] = a;
    red[1][w][lane] = b;
    __syncthreads();
    if (w < 2 && c < C)
        part[((size_t)blockIdx.y * 2 + w) * C + c] =
            (red[w][0][lane] + red[w][1][lane]) + (red[w][2][lane] + red[w][3][lane]);
}

// dgamma | dbeta = the partial rows part[block][2C], added in block order: 64 columns a workgroup, 16 lanes of blocks each.
__global__ __launch_bounds__(1024) void ln_bwd_finish(const float* __restrict__ part, int blocks, int C,
                                                      float* __restrict__ dgamma, float* __restrict__ dbeta) {
    __shared__ float red[16][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int64_t c = (int64_t)blockIdx.x * 64 + lane, C2 = 2 * (int64_t)C;
    float a[4] = {0.f, 0.f, 0.f, 0.f};
    if (c < C2) {
        int i = w;
        for (; i + 48 < blocks; i += 64) {
#pragma unroll
            for (int u = 0; u < 4; ++u) a[u] += part[(i + 16 * u) * C2 + c];
        }
        for (; i < blocks; i += 16) a[0] += part[i * C2 + c];
    }
    red[w][lane] = (a[0] + a[1]) + (a[2] + a[3]);
    __syncthreads();
    if (w == 0 && c < C2) {
        float v = red[0][lane];
#pragma unroll
        for (int k = 1; k < 16; ++k) v += red[k][lane];
        if (c < C) dgamma[c] = v;
        else dbeta[c - C] = v;
    }
}

static bool ln_apart(const void* a, const void* b, int64_t na, int64_t nb) {
    const char *p = (const char*)a, *q = (const char*)b;
    return p == nullptr || q == nullptr || p + na <= q || q + nb <= p;
}

static bool ln_vec4(int C, std::initializer_list<const void*> pointers) {
    if (C % 4 != 0) return false;
    for (const void* p : pointers)
        if ((reinterpret_cast<uintptr_t>(p) & 15) != 0) return false;
    return true;
}

typedef void (*LnFwd)(const float*, const float*, const float*, float*, float*, float*, uint16_t*, int, int, float);

// The kernel for rows of `units` W-float units, its threads and the rows it takes at a time.
template <int W>
static LnFwd ln_fwd_kernel(int units, int* threads, int* rows_per_block) {
    constexpr int F = 4 / W;                             // 4-byte units: four times as many of them for the same registers
    *threads = 256;
    const auto wave = [&](LnFwd k, int lanes) { *rows_per_block = 256 / lanes; return k; };
    if (units <= 4) return wave(ln_fwd_wave<4, 1, W>, 4);
    if (units <= 8) return wave(ln_fwd_wave<8, 1, W>, 8);
    if (units <= 16) return wave(ln_fwd_wave<16, 1, W>, 16);
    if (units <= 32) return wave(ln_fwd_wave<32, 1, W>, 32);
    if (units <= 64) return wave(ln_fwd_wave<64, 1, W>, 64);
    if (units <= 128) return wave(ln_fwd_wave<64, 2, W>, 64);
    if (units <= 256) return wave(ln_fwd_wave<64, 4, W>, 64);
    *rows_per_block = 1;
    if (units <= 512 * F) return ln_fwd_block<256, 2 * F, W>;
    if (units <= 1024 * F) return ln_fwd_block<256, 4 * F, W>;
    if (units <= 2048 * F) return ln_fwd_block<256, 8 * F, W>;
    *threads = 1024;
    if (units <= 4096 * F) return ln_fwd_block<1024, 4 * F, W>;
    if (units <= 8192 * F) return ln_fwd_block<1024, 8 * F, W>;
    *threads = 256;
    return ln_fwd_rows;
}

typedef void (*LnBwd)(const float*, const float*, const float*, const float*, const float*, float*, uint16_t*, int, int,
                      float*);

// As ln_fwd_kernel; `cap`: the most workgroups to launch.  NULL: rows too long for the registers of a workgroup.
template <int W>
static LnBwd ln_bwd_kernel(int units, int* threads, int* rows_per_block, int* cap) {
    constexpr int F = 4 / W;
    constexpr int T = 512;
    *threads = T;
    *cap = 512;
    const auto wave = [&](LnBwd k, int lanes) { *rows_per_block = T / lanes; return k; };
    if (units <= 4) return wave(ln_bwd_wave<T, 4, 1, W>, 4);
    if (units <= 8) return wave(ln_bwd_wave<T, 8, 1, W>, 8);
    if (units <= 16) return wave(ln_bwd_wave<T, 16, 1, W>, 16);
    if (units <= 32) return wave(ln_bwd_wave<T, 32, 1, W>, 32);
    if (units <= 64) return wave(ln_bwd_wave<T, 64, 1, W>, 64);
    if (units <= 128) return wave(ln_bwd_wave<T, 64, 2, W>, 64);
    if (units <= 256) return wave(ln_bwd_wave<T, 64, 4, W>, 64);
    *rows_per_block = 1;
    *threads = 256;
    *cap = 768;
    if (units <= 512 * F) return ln_bwd_block<256, 2 * F, W>;
    if (units <= 1024 * F) return ln_bwd_block<256, 4 * F, W>;
    *threads = 512;
    *cap = 512;
    if (units <= 2048 * F) return ln_bwd_block<512, 4 * F, W>;
    *threads = 1024;
    *cap = 256;
    if (units <= 4096 * F) return ln_bwd_block<1024, 4 * F, W>;
    *rows_per_block = 256;
    return nullptr;
}

// The arguments are checked before the context: a bad call is refused alike with and without a GPU.
static int ln_fwd_impl(const float* x, const float* gamma, const float* beta, float* save_mean, float* save_invstd, float* y,
                       uint16_t* y16, int rows, int C, float eps) {
    AETH_CHECK_ARG(rows >= 0 && C > 0 && (int64_t)rows * C < ((int64_t)1 << 31));
    AETH_CHECK_ARG(eps >= 0.f);
    AETH_CHECK_ARG((save_mean == nullptr) == (save_invstd == nullptr));
    AETH_CHECK_ARG(rows == 0 || (x && gamma && beta && y));
    const int64_t n = (int64_t)rows * C;
    AETH_CHECK_ARG(ln_apart(x, y, 4 * n, 4 * n) && ln_apart(x, y16, 4 * n, 2 * n) && ln_apart(y, y16, 4 * n, 2 * n));
    AETH_REQUIRE_INIT();
    if (rows == 0) return AETH_OK;
    int threads, per;
    const LnFwd kernel = ln_vec4(C, {x, gamma, beta, y, y16}) ? ln_fwd_kernel<4>(C / 4, &threads, &per)
                                                              : ln_fwd_kernel<1>(C, &threads, &per);
    const int want = cdiv(rows, per);
    hipLaunchKernelGGL(kernel, dim3(want < kLnGrid ? want : kLnGrid), dim3(threads), 0, ctx().stream, x, gamma, beta, save_mean,
                       save_invstd, y, y16, rows, C, eps);
    AETH_LAUNCH_CHECK();
    return AETH_OK;
}

static int ln_bwd_impl(const float* x, const float* dy, const float* gamma, const float* mean, const float* invstd, float* dx,
                       uint16_t* dx16, float* dgamma, float* dbeta, int rows, int C) {
    AETH_CHECK_ARG(rows >= 0 && C > 0 && (int64_t)rows * C < ((int64_t)1 << 31));
    AETH_CHECK_ARG(dgamma && dbeta && (rows == 0 || (x && dy && gamma && mean && invstd && dx)));
    const int64_t n = (int64_t)rows * C;
    AETH_CHECK_ARG(ln_apart(x, dx, 4 * n, 4 * n) && ln_apart(dy, dx, 4 * n, 4 * n));
    AETH_CHECK_ARG(ln_apart(x, dx16, 4 * n, 2 * n) && ln_apart(dy, dx16, 4 * n, 2 * n) && ln_apart(dx, dx16, 4 * n, 2 * n));
    AETH_REQUIRE_INIT();
    hipStream_t st = ctx().stream;
    int threads, per, cap, blocks = 0;
    void* ws = nullptr;
    if (rows > 0) {
        const LnBwd kernel = ln_vec4(C, {x, dy, gamma, dx, dx16}) ? ln_bwd_kernel<4>(C / 4, &threads, &per, &cap)
                                                                  : ln_bwd_kernel<1>(C, &threads, &per, &cap);
        blocks = cdiv(rows, per) < cap ? cdiv(rows, per) : cap;
        const int run = cdiv(rows, blocks);
        if (kernel == nullptr) blocks = cdiv(rows, run);
        const int rc = workspace((int64_t)2 * blocks * C * sizeof(float), &ws);
        if (rc) return rc;
        if (kernel != nullptr) {
            hipLaunchKernelGGL(kernel, dim3(blocks), dim3(threads), 0, st, x, dy, gamma, mean, invstd, dx, dx16, rows, C,
                               (float*)ws);
        } else {
            hipLaunchKernelGGL(ln_bwd_rows, dim3(rows < kLnGrid ? rows : kLnGrid), dim3(kLnThreads), 0, st, x, dy, gamma, mean,
                               invstd, dx, dx16, rows, C);
            AETH_LAUNCH_CHECK();
            hipLaunchKernelGGL(ln_bwd_columns, dim3(cdiv(C, 64), blocks), dim3(kLnThreads), 0, st, x, dy, mean, invstd, rows, C,
                               run, (float*)ws);
        }
        AETH_LAUNCH_CHECK();
    }
    hipLaunchKernelGGL(ln_bwd_finish, dim3(cdiv(2 * (int64_t)C, 64)), dim3(1024), 0, st, (const float*)ws, blocks, C, dgamma, dbeta);
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
