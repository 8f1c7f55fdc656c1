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

namespace aeth {

constexpr int kLnThreads = 256;

// float32 -> bfloat16 bits, round to nearest even; NaN stays NaN
__device__ __forceinline__ unsigned ln_bf16(float f) {
    const unsigned u = __float_as_uint(f);
    if ((u & 0x7fffffffu) > 0x7f800000u) return (u >> 16) | 0x40u;
    return (u + 0x7fffu + ((u >> 16) & 1u)) >> 16;
}

// sum over the workgroup, the same value in every thread
__device__ __forceinline__ float ln_block_sum(float v, float* red) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    __syncthreads();                                     // the last use of `red` is over
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
}

// One workgroup per row, three passes over it.
__global__ __launch_bounds__(kLnThreads) void ln_fwd_rows(const float* __restrict__ x, const float* __restrict__ gamma,
                                                          const float* __restrict__ beta, float* __restrict__ save_mean,
                                                          float* __restrict__ save_invstd, float* __restrict__ y,
                                                          uint16_t* __restrict__ y16, int rows, int C, float eps) {
    __shared__ float red[4];
    for (int r = blockIdx.x; r < rows; r += gridDim.x) {
        const float* xr = x + (size_t)r * C;
        float s = 0.f;
        for (int c = threadIdx.x; c < C; c += kLnThreads) s += xr[c];
        const float mean = ln_block_sum(s, red) / (float)C;
        float q = 0.f;
        for (int c = threadIdx.x; c < C; c += kLnThreads) {
            const float d = xr[c] - mean;
            q += d * d;
        }
        const float invstd = 1.0f / sqrtf(ln_block_sum(q, red) / (float)C + eps);
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

__global__ __launch_bounds__(kLnThreads) void ln_bwd_rows(const float* __restrict__ x, const float* __restrict__ dy,
                                                          const float* __restrict__ gamma, const float* __restrict__ mean,
                                                          const float* __restrict__ invstd, float* __restrict__ dx,
                                                          uint16_t* __restrict__ dx16, int rows, int C) {
    __shared__ float red[4];
    for (int r = blockIdx.x; r < rows; r += gridDim.x) {
        const size_t at = (size_t)r * C;
        const float m = mean[r], is = invstd[r];
        float s1 = 0.f, s2 = 0.f;
        for (int c = threadIdx.x; c < C; c += kLnThreads) {
            const float g = dy[at + c] * gamma[c];
            s1 += g;
            s2 += g * ((x[at + c] - m) * is);
        }
        const float c1 = ln_block_sum(s1, red) / (float)C;
        const float c2 = ln_block_sum(s2, red) / (float)C;
        for (int c = threadIdx.x; c < C; c += kLnThreads) {
            const float v = is * (dy[at + c] * gamma[c] - c1 - (x[at + c] - m) * is * c2);
            dx[at + c] = v;
            if (dx16 != nullptr) dx16[at + c] = (uint16_t)ln_bf16(v);
        }
    }
}

// Partial sums of dy xhat and dy over a run of rows: 64 columns x 4 row lanes per workgroup, part[2][runs][C].
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
        part[((size_t)w * gridDim.y + blockIdx.y) * C + c] =
            (red[w][0][lane] + red[w][1][lane]) + (red[w][2][lane] + red[w][3][lane]);
}

__global__ __launch_bounds__(kLnThreads) void ln_bwd_finish(const float* __restrict__ part, int runs, int C,
                                                            float* __restrict__ dgamma, float* __restrict__ dbeta) {
    const int c = blockIdx.x * kLnThreads + threadIdx.x;
    if (c >= C) return;
    float a = 0.f, b = 0.f;
    for (int i = 0; i < runs; ++i) {
        a += part[(size_t)i * C + c];
        b += part[((size_t)runs + i) * C + c];
    }
    dgamma[c] = a;
    dbeta[c] = b;
}

static bool ln_apart(const void* a, const void* b, int64_t na, int64_t nb) {
    const char *p = (const char*)a, *q = (const char*)b;
    return p == nullptr || q == nullptr || p + na <= q || q + nb <= p;
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
    hipLaunchKernelGGL(ln_fwd_rows, dim3(rows < 65536 ? rows : 65536), dim3(kLnThreads), 0, ctx().stream, x, gamma, beta,
                       save_mean, save_invstd, y, y16, rows, C, eps);
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
    int runs = cdiv(rows, 256);
    if (runs > 256) runs = 256;
    const int run = runs > 0 ? cdiv(rows, runs) : 0;
    if (runs > 0) runs = cdiv(rows, run);
    void* ws = nullptr;
    if (runs > 0) {
        const int rc = workspace((int64_t)2 * runs * C * sizeof(float), &ws);
        if (rc) return rc;
        hipLaunchKernelGGL(ln_bwd_rows, dim3(rows < 65536 ? rows : 65536), dim3(kLnThreads), 0, st, x, dy, gamma, mean, invstd,
                           dx, dx16, rows, C);
        AETH_LAUNCH_CHECK();
        hipLaunchKernelGGL(ln_bwd_columns, dim3(cdiv(C, 64), runs), dim3(kLnThreads), 0, st, x, dy, mean, invstd, rows, C, run,
                           (float*)ws);
        AETH_LAUNCH_CHECK();
    }
    hipLaunchKernelGGL(ln_bwd_finish, dim3(cdiv(C, kLnThreads)), dim3(kLnThreads), 0, st, (const float*)ws, runs, C, dgamma,
                       dbeta);
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
