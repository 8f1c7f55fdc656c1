// The Muon update of weight matrices: momentum, orthogonalisation of the update by Newton-Schulz products, step.
//
//   m <- mu m + g,   u = g + mu m (Nesterov) or m
//   X = u / |u| (Frobenius norm; a zero u stays zero), taken with rows <= cols (transposed otherwise)
//   `steps` times:  A = X X^T,  X <- a X + (b A + c A^2) X        (a, b, c) = (3.4445, -4.7750, 2.0315)
//   theta <- theta (1 - lr wd) - lr sqrt(max(1, cols / rows)) X
//
// Every singular value s of X goes to p(s) = a s + b s^3 + c s^5; from s <= 1 (the norm bounds them) all stay below 1.21 and
// those that are not tiny end in about [0.7, 1.2]: u's singular vectors with singular values near one.
#include "common.h"

#include <math.h>

namespace aeth {

constexpr float kNsA = 3.4445f, kNsB = -4.7750f, kNsC = 2.0315f;
constexpr int kMuonMax = 32;
constexpr int kNormBlocks = 256;

// One matrix of a call.  g is the update itself where m is NULL (orthogonalisation alone).
struct MuonMatrix {
    float* theta;       // the weights; NULL: write X to out
    const float* grad;
    float* mom;
    float* out;
    int rows, cols;
    int m, n;           // the shorter and the longer side
};

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

__device__ __forceinline__ double block_sum(double v, double* red) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
}

// m <- mu m + g and the partial sums of u^2.  They are 64-bit: no gradient overflows or vanishes in the square.
__global__ __launch_bounds__(256) void muon_momentum(MuonMatrix t, float mu, int nesterov, double* __restrict__ part) {
    __shared__ double red[4];
    const int64_t n = (int64_t)t.rows * t.cols;
    double s = 0.0;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        float u = t.grad[i];
        if (t.mom != nullptr) {
            const float g = u;
            const float v = mu * t.mom[i] + g;
            t.mom[i] = v;
            u = nesterov ? g + mu * v : v;
        }
        s += (double)u * (double)u;
    }
    s = block_sum(s, red);
    if (threadIdx.x == 0) part[blockIdx.x] = s;
}

// X = u / |u|, transposed to [m][n] where the matrix is tall
__global__ __launch_bounds__(256) void muon_normalise(MuonMatrix t, float mu, int nesterov, const double* __restrict__ part,
                                                      int parts, float* __restrict__ X) {
    __shared__ double red[4];
    const double sum = block_sum((int)threadIdx.x < parts ? part[threadIdx.x] : 0.0, red);
    const double inv = sum != 0.0 ? 1.0 / sqrt(sum) : 0.0;
    const int64_t n = (int64_t)t.rows * t.cols;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        float u = t.grad[i];
        if (t.mom != nullptr) u = nesterov ? u + mu * t.mom[i] : t.mom[i];
        const int64_t r = i / t.cols, c = i % t.cols;
        X[t.rows <= t.cols ? i : c * t.rows + r] = (float)((double)u * inv);
    }
}

// out = alpha R + beta P Q (R may be NULL), or P Q^T: 64 x 64 per workgroup, 4 x 4 per thread, slabs of 16 through LDS
template <bool kTransposed>
__global__ __launch_bounds__(256) void muon_product(const float* __restrict__ P, const float* __restrict__ Q,
                                                    const float* __restrict__ R, float* __restrict__ out, int M, int N,
                                                    int K, float alpha, float beta) {
    __shared__ float p[16][65], q[16][65];
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int i0 = blockIdx.y * 64, j0 = blockIdx.x * 64;
    float acc[4][4] = {};
    for (int k0 = 0; k0 < K; k0 += 16) {
        for (int e = threadIdx.x; e < 1024; e += 256) {
            const int k = e & 15, r = e >> 4;
            p[k][r] = i0 + r < M && k0 + k < K ? P[(size_t)(i0 + r) * K + k0 + k] : 0.f;
            if (kTransposed) {
                q[k][r] = j0 + r < N && k0 + k < K ? Q[(size_t)(j0 + r) * K + k0 + k] : 0.f;
            } else {
                const int kk = e >> 6, c = e & 63;
                q[kk][c] = j0 + c < N && k0 + kk < K ? Q[(size_t)(k0 + kk) * N + j0 + c] : 0.f;
            }
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 16; ++k)
#pragma unroll
            for (int a = 0; a < 4; ++a)
#pragma unroll
                for (int b = 0; b < 4; ++b) acc[a][b] += p[k][ty + 16 * a] * q[k][tx + 16 * b];
        __syncthreads();
    }
    for (int a = 0; a < 4; ++a)
        for (int b = 0; b < 4; ++b) {
            const int i = i0 + ty + 16 * a, j = j0 + tx + 16 * b;
            if (i >= M || j >= N) continue;
            const size_t at = (size_t)i * N + j;
            out[at] = (R != nullptr ? alpha * R[at] : 0.f) + beta * acc[a][b];
        }
}

// theta <- theta (1 - lr wd) - lr gain X, or out = X
__global__ __launch_bounds__(256) void muon_apply(MuonMatrix t, const float* __restrict__ X, float lr,
                                                  const double* __restrict__ state, float wd, float gain) {
    if (state != nullptr) lr = (float)state[3];
    const float keep = 1.0f - lr * wd, step = lr * gain;
    const int64_t n = (int64_t)t.rows * t.cols;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / t.cols, c = i % t.cols;
        const float o = X[t.rows <= t.cols ? i : c * t.rows + r];
        if (t.theta != nullptr) t.theta[i] = keep * t.theta[i] - step * o;
        else t.out[i] = o;
    }
}

static int muon_matrix(const MuonMatrix& t, float lr, const double* state, float mu, int nesterov, float wd, int steps) {
    const int64_t m = t.m, n = t.n;
    void* ws;
    const int rc = workspace((2 * m * n + 2 * m * m) * (int64_t)sizeof(float) + kNormBlocks * (int64_t)sizeof(double), &ws);
    if (rc) return rc;
    double* part = (double*)ws;
    float* X = (float*)(part + kNormBlocks);
    float* Y = X + m * n;
    float* A = Y + m * n;
    float* B = A + m * m;
    hipStream_t st = ctx().stream;
    const int64_t size = m * n;
    const int blocks = size > 4096 * kNormBlocks ? kNormBlocks : cdiv(size, 4096);
    hipLaunchKernelGGL(muon_momentum, dim3(blocks), dim3(256), 0, st, t, mu, nesterov, part);
    AETH_LAUNCH_CHECK();
    hipLaunchKernelGGL(muon_normalise, dim3(cdiv(size, 1024) < 4096 ? cdiv(size, 1024) : 4096), dim3(256), 0, st, t, mu,
                       nesterov, part, blocks, X);
    AETH_LAUNCH_CHECK();
    const dim3 small(cdiv(m, 64), cdiv(m, 64)), wide(cdiv(n, 64), cdiv(m, 64));
    for (int s = 0; s < steps; ++s) {
        hipLaunchKernelGGL((muon_product<true>), small, dim3(256), 0, st, X, X, nullptr, A, t.m, t.m, t.n, 0.f, 1.f);
        AETH_LAUNCH_CHECK();
        hipLaunchKernelGGL((muon_product<false>), small, dim3(256), 0, st, A, A, A, B, t.m, t.m, t.m, kNsB, kNsC);
        AETH_LAUNCH_CHECK();
        hipLaunchKernelGGL((muon_product<false>), wide, dim3(256), 0, st, B, X, X, Y, t.m, t.n, t.m, kNsA, 1.f);
        AETH_LAUNCH_CHECK();
        float* swap = X;
        X = Y;
        Y = swap;
    }
    const float gain = t.cols > t.rows ? sqrtf((float)t.cols / (float)t.rows) : 1.f;
    hipLaunchKernelGGL(muon_apply, dim3(cdiv(size, 1024) < 4096 ? cdiv(size, 1024) : 4096), dim3(256), 0, st, t, X, lr, state,
                       wd, gain);
    AETH_LAUNCH_CHECK();
    return AETH_OK;
}

static bool muon_apart(const void* a, int64_t na, const void* b, int64_t nb) {
    const char *p = (const char*)a, *q = (const char*)b;
    return p + na <= q || q + nb <= p;
}

// The arguments are checked before the context: a bad call is refused alike with and without a GPU.
static int muon_multi_impl(const char* fn, int count, float* const* theta, const float* const* grad, float* const* mom,
                           const int* rows, const int* cols, float lr, const double* state, float mu, int nesterov, float wd,
                           int steps) {
    if (count < 1 || count > kMuonMax) return fail(AETH_E_INVALID, "%s: count %d, expected 1 to %d", fn, count, kMuonMax);
    if (!theta || !grad || !mom || !rows || !cols) return fail(AETH_E_INVALID, "%s: a host array is NULL", fn);
    if (!(mu >= 0.f && mu < 1.f)) return fail(AETH_E_INVALID, "%s: momentum %g, expected 0 <= momentum < 1", fn, (double)mu);
    if (!(wd >= 0.f) || !isfinite(wd) || !isfinite(lr))
        return fail(AETH_E_INVALID, "%s: learning rate %g, weight decay %g", fn, (double)lr, (double)wd);
    if (steps < 1 || steps > 100) return fail(AETH_E_INVALID, "%s: %d Newton-Schulz steps, expected 1 to 100", fn, steps);
    MuonMatrix t[kMuonMax];
    int k = 0;
    for (int i = 0; i < count; ++i) {
        const int r = rows[i], c = cols[i];
        if (r < 0 || c < 0 || (int64_t)r * c >= ((int64_t)1 << 31))
            return fail(AETH_E_INVALID, "%s: matrix %d is %d x %d", fn, i, r, c);
        if (r == 0 || c == 0) continue;
        if (!theta[i] || !grad[i] || !mom[i]) return fail(AETH_E_INVALID, "%s: matrix %d has a NULL tensor", fn, i);
        t[k++] = MuonMatrix{theta[i], grad[i], mom[i], nullptr, r, c, r < c ? r : c, r < c ? c : r};
    }
    // what is written (weights, momentum) may overlap nothing else of the call
    for (int i = 0; i < k; ++i) {
        const int64_t ni = (int64_t)t[i].rows * t[i].cols * 4;
        for (int j = 0; j < k; ++j) {
            const int64_t nj = (int64_t)t[j].rows * t[j].cols * 4;
            if (!muon_apart(t[i].theta, ni, t[j].grad, nj) || !muon_apart(t[i].mom, ni, t[j].grad, nj) ||
                !muon_apart(t[i].theta, ni, t[j].mom, nj) ||
                (i != j && (!muon_apart(t[i].theta, ni, t[j].theta, nj) || !muon_apart(t[i].mom, ni, t[j].mom, nj))))
                return fail(AETH_E_INVALID, "%s: tensors of the matrices overlap (the same matrix twice?)", fn);
        }
    }
    if (!ctx().ready) return fail(AETH_E_STATE, "%s: aeth_init has not been called", fn);
    for (int i = 0; i < k; ++i) {
        const int rc = muon_matrix(t[i], lr, state, mu, nesterov, wd, steps);
        if (rc) return rc;
    }
    return AETH_OK;
}

}  // namespace aeth

using namespace aeth;

extern "C" {

int aeth_newton_schulz_f32(const float* g, float* o, int rows, int cols, int steps) {
    AETH_CHECK_ARG(rows >= 0 && cols >= 0 && (int64_t)rows * cols < ((int64_t)1 << 31));
    AETH_CHECK_ARG(steps >= 1 && steps <= 100);
    const int64_t bytes = (int64_t)rows * cols * 4;
    AETH_CHECK_ARG(bytes == 0 || (g && o && muon_apart(g, bytes, o, bytes)));
    AETH_REQUIRE_INIT();
    if (bytes == 0) return AETH_OK;
    const MuonMatrix t{nullptr, g, nullptr, o, rows, cols, rows < cols ? rows : cols, rows < cols ? cols : rows};
    return muon_matrix(t, 0.f, nullptr, 0.f, 0, 0.f, steps);
}

int aeth_muon_multi_f32(int count, float* const* host_theta, const float* const* host_grad, float* const* host_m,
                        const int* host_rows, const int* host_cols, float lr, float momentum, int nesterov,
                        float weight_decay, int steps) {
    return muon_multi_impl(__func__, count, host_theta, host_grad, host_m, host_rows, host_cols, lr, nullptr, momentum,
                           nesterov, weight_decay, steps);
}

int aeth_muon_multi_dev_f32(int count, float* const* host_theta, const float* const* host_grad, float* const* host_m,
                            const int* host_rows, const int* host_cols, float momentum, int nesterov, float weight_decay,
                            int steps, const double* state) {
    AETH_CHECK_ARG(state != nullptr);
    return muon_multi_impl(__func__, count, host_theta, host_grad, host_m, host_rows, host_cols, 0.f, state, momentum,
                           nesterov, weight_decay, steps);
}

}  // extern "C"
