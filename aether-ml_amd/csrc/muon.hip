// The Muon update of weight matrices: momentum, orthogonalisation of the update by Newton-Schulz products, step.
//
//   m <- mu m + g,   u = g + mu m (Nesterov) or m
//   X = u / |u| (Frobenius norm; a zero u stays zero), taken with rows <= cols (transposed otherwise)
//   `steps` times:  A = X X^T,  X <- a X + (b A + c A^2) X        (a, b, c) = (3.4445, -4.7750, 2.0315)
//   theta <- theta (1 - lr wd) - lr sqrt(max(1, cols / rows)) X
//
// Every singular value s of X goes to p(s) = a s + b s^3 + c s^5; from s <= 1 (the norm bounds them) all stay below 1.21 and
// those that are not tiny end in about [0.7, 1.2]: u's singular vectors with singular values near one.
#include "muon_f32.h"
#include "split_gemm.h"

#include <math.h>

#include <algorithm>

namespace aeth {

// One matrix of a call.  mom == NULL: grad is the update itself (orthogonalisation alone, written to out).
struct MuonMatrix {
    float* theta;
    const float* grad;
    float* mom;
    float* out;
    int rows, cols;
    float gain;
};

struct MuonTable {
    int count;
    MuonMatrix t[kMuonMax];
    int parts[kMuonMax];                                 // workgroups of muon_momentum
    int first[kMuonMax];                                 // first workgroup of muon_split
    char *same[kMuonMax], *turned[kMuonMax];             // X in the matrix's own orientation and transposed
    double* sums;                                        // [count][kMuonParts]
};
typedef const MuonTable __attribute__((address_space(4)))* muon_table_ptr;

// Workgroups of muon_momentum for a matrix
static int muon_parts(const MuonMatrix& t) {
    const int64_t size = (int64_t)t.rows * t.cols;
    return size > 4096 * (int64_t)kMuonParts ? kMuonParts : cdiv(size, 4096);
}

__device__ __forceinline__ double muon_block_sum(double v, double* red) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
}

// The update u from a gradient and the new momentum.
__device__ __forceinline__ float muon_update(float g, float m, float mu, int nesterov) { return nesterov ? fmaf(mu, m, g) : m; }

// m <- mu m + g and the partial sums of u^2, blockIdx.y = matrix.  They are 64-bit: no gradient overflows or vanishes in the square.
// Bound: HBM, 12 bytes an element.
__global__ __launch_bounds__(256) void muon_momentum(const MuonTable tb, float mu, int nesterov) {
    __shared__ double red[4];
    const muon_table_ptr args = (muon_table_ptr)__builtin_amdgcn_kernarg_segment_ptr();
    const int k = blockIdx.y, parts = args->parts[k];
    if ((int)blockIdx.x >= parts) return;
    const float* __restrict__ grad = args->t[k].grad;
    float* __restrict__ mom = args->t[k].mom;
    const int64_t n = (int64_t)args->t[k].rows * args->t[k].cols, n4 = n / 4, step = (int64_t)parts * 256;
    typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
    double s = 0.0;
    const auto one = [&](float g, float m) {
        const float u = mom != nullptr ? muon_update(g, m, mu, nesterov) : g;
        s += (double)u * (double)u;
    };
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n4; i += step) {
        const f4u g = *reinterpret_cast<const f4u*>(grad + 4 * i);
        f4u m = {0.f, 0.f, 0.f, 0.f};
        if (mom != nullptr) {
            m = *reinterpret_cast<const f4u*>(mom + 4 * i);
#pragma unroll
            for (int e = 0; e < 4; ++e) m[e] = fmaf(mu, m[e], g[e]);
            *reinterpret_cast<f4u*>(mom + 4 * i) = m;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) one(g[e], m[e]);
    }
    if (blockIdx.x == 0 && threadIdx.x < n - 4 * n4) {
        const int64_t i = 4 * n4 + threadIdx.x;
        float m = 0.f;
        if (mom != nullptr) mom[i] = m = fmaf(mu, mom[i], grad[i]);
        one(grad[i], m);
    }
    s = muon_block_sum(s, red);
    if (threadIdx.x == 0) args->sums[k * kMuonParts + blockIdx.x] = s;
}

// X = u / |u| and its transpose as float16 halves, a 32 x 32 block a wave; padding becomes 0.
// Bound: HBM, 8 bytes read and 8 written an element; for small matrices the chain partial sums - norm - loads - stores, so the loads
// go out first, all at once (behind a branch each they came back one by one: 576 x 64 10 us).
__global__ __launch_bounds__(256) void muon_split(const MuonTable tb, float mu, int nesterov) {
    __shared__ double red[4];
    __shared__ unsigned blocks[4][32][33];
    const muon_table_ptr args = (muon_table_ptr)__builtin_amdgcn_kernarg_segment_ptr();
    int k = 0;
    while (k + 1 < tb.count && (int)blockIdx.x >= args->first[k + 1]) ++k;
    const float* __restrict__ grad = args->t[k].grad;
    const float* __restrict__ mom = args->t[k].mom;
    const int rows = args->t[k].rows, cols = args->t[k].cols;
    const int64_t rp = muon_pad(rows), cp = muon_pad(cols), across = cp / 32;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, l32 = lane & 31, lh = lane >> 5;
    const int64_t b = ((int64_t)blockIdx.x - args->first[k]) * 4 + wave;
    const bool mine = b < rp / 32 * across;
    const int64_t r = mine ? b / across * 32 : 0, c = mine ? b % across * 32 : 0;
    const int64_t x = c + l32, xc = x < cols ? x : cols - 1;
    float u[16], m[16];
#pragma unroll
    for (int v = 0; v < 16; ++v) {
        const int64_t y = r + 2 * v + lh, at = (y < rows ? y : rows - 1) * cols + xc;
        u[v] = grad[at];
        m[v] = mom != nullptr ? mom[at] : 0.f;
    }
    double part = 0.0;
#pragma unroll
    for (int i = 0; i < kMuonParts; i += 256)
        if ((int)threadIdx.x + i < args->parts[k]) part += args->sums[k * kMuonParts + threadIdx.x + i];
    const double sum = muon_block_sum(part, red);
    // 1 / |u| as a power of two and a factor near one: u times the power is exact, whatever its size
    int power = 0;
    const float factor = sum != 0.0 ? (float)frexp((double)kScaleX / sqrt(sum), &power) : 0.f;
    if (!mine) return;
    unsigned(*blk)[33] = blocks[wave];
#pragma unroll
    for (int v = 0; v < 16; ++v) {
        const float w = mom != nullptr ? muon_update(u[v], m[v], mu, nesterov) : u[v];
        const bool in = r + 2 * v + lh < rows && x < cols;
        blk[2 * v + lh][l32] = split_pack(in ? ldexpf(w, power) * factor : 0.f);
    }
    __builtin_amdgcn_wave_barrier();
    // four lanes a row: a store covers whole pieces of 64 bytes
    const int row = lane >> 2, col = 8 * (lane & 3);
    char* same = args->same[k] + ((size_t)(c / 32) * rp + r + row) * 128 + 2 * col;
    char* turned = args->turned[k] + ((size_t)(r / 32) * cp + c + row) * 128 + 2 * col;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        unsigned s[8], t[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            s[e] = blk[16 * h + row][col + e];
            t[e] = blk[col + e][16 * h + row];
        }
        u32x4 hi, lo;
        split_halves(s, hi, lo);
        *reinterpret_cast<u32x4*>(same + 2048 * h) = hi;
        *reinterpret_cast<u32x4*>(same + 2048 * h + 64) = lo;
        split_halves(t, hi, lo);
        *reinterpret_cast<u32x4*>(turned + 2048 * h) = hi;
        *reinterpret_cast<u32x4*>(turned + 2048 * h + 64) = lo;
    }
}

// ---- small matrices: the whole update in one workgroup -------------------------------------------------------------------
// For matrices of at most 64 rows (the shorter side) and few columns, whose chain of seventeen launches of 4 us each is all that
// the update costs.  X stays in the registers of 8 waves as packed halves: wave w has the 32-column blocks w, w + 8, ..., a lane
// one column j of a block and of each 32-row block the 16 rows i that an MFMA's result has in a lane.  So the result of a step,
// B X with a column a lane, is the next step's operand as it is, with B's columns stored in the order in which a lane has its
// rows (muon_slot); X X^T needs a row a lane, which a wave turns round through LDS of its own.  The waves' parts of A are added
// in their order, A^2 is 1 or 3 blocks, and the weights take the last step's result from the accumulators.
// Bound: latency, 3 us a step on 64 x 64 and 7 on 64 x 576 (its MFMAs 2.5), and what one CU loads and stores.
constexpr int kWholeWaves = 8, kWholePitch = 72;         // halves of a row of A and B: 16-byte reads of 8 rows in different banks

// Where column k of B stands in its row: a lane's 8 values of a 16-column step are rows 4 h + e and 8 + 4 h + e.
__device__ __forceinline__ int muon_slot(int k) { return (k & ~15) | (k & 4) << 1 | (k & 8) >> 1 | (k & 3); }

__device__ __forceinline__ void whole_split(const float* v, half4& hi, half4& lo) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const _Float16 h = (_Float16)v[e];
        hi[e] = h;
        lo[e] = (_Float16)(v[e] - (float)h);
    }
}

__device__ __forceinline__ void whole_halves(const unsigned* w, half8& hi, half8& lo) {
    typedef unsigned u4 __attribute__((ext_vector_type(4)));
    u4 h, l;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        h[e] = __builtin_amdgcn_perm(w[2 * e + 1], w[2 * e], 0x05040100u);
        l[e] = __builtin_amdgcn_perm(w[2 * e + 1], w[2 * e], 0x07060302u);
    }
    hi = __builtin_bit_cast(half8, h);
    lo = __builtin_bit_cast(half8, l);
}

__device__ __forceinline__ f16v whole_mfma(const half8& ah, const half8& al, const half8& bh, const half8& bl, f16v acc) {
    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah, bl, acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(al, bh, acc, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(ah, bh, acc, 0, 0, 0);
}

// MB 32-row blocks, CB column blocks a wave; kUpdate: a step of weights with momentum, else the orthogonalisation alone.
template <int MB, int CB, bool kUpdate>
__global__ __launch_bounds__(64 * kWholeWaves) void muon_whole(const MuonTable tb, float mu, int nesterov, float lr,
                                                              const double* __restrict__ state, float wd, int steps) {
    constexpr int NP = MB * (MB + 1) / 2;                // blocks of A on and above the diagonal
    constexpr int REGION = (NP > 2 ? NP * 4096 : 9216);  // a wave's: X turned round (32 MB rows of 36 words), or its part of A
    static_assert(REGION >= 32 * MB * 36 * 4 && REGION >= NP * 4096, "both fit");
    __shared__ __attribute__((aligned(16))) char regions[kWholeWaves][REGION];
    __shared__ __attribute__((aligned(16))) _Float16 a_hi[32 * MB][kWholePitch], a_lo[32 * MB][kWholePitch];
    __shared__ __attribute__((aligned(16))) _Float16 b_hi[32 * MB][kWholePitch], b_lo[32 * MB][kWholePitch];
    __shared__ double red[kWholeWaves];
    const muon_table_ptr args = (muon_table_ptr)__builtin_amdgcn_kernarg_segment_ptr();
    const int k = blockIdx.x;
    const float* __restrict__ grad = args->t[k].grad;
    float* mom = args->t[k].mom;
    float* theta = args->t[k].theta;
    float* out = args->t[k].out;
    const int rows = args->t[k].rows, cols = args->t[k].cols;
    const bool tall = rows > cols;
    const int m = tall ? cols : rows, n = tall ? rows : cols, blocks = (n + 31) / 32, busy = min(blocks, kWholeWaves);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, l32 = lane & 31, lh = lane >> 5;
    char* region = regions[wave];

    // Element (i, j) of X is at si i + sj j of the matrix's memory: a part of the lane's own and a part that is the same for all.
    // Places behind the matrix's end are cut off by the descriptors, other places that are no element are masked.
    const int bytes = rows * cols * 4;
    const auto rsrc = [&](const float* q) { return __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(q), 0, bytes, 0x00020000); };
    const auto row = [&](int ib, int v) { return 32 * ib + 8 * (v >> 2) + 4 * lh + (v & 3); };
    const auto column = [&](int cb) { return 32 * (wave + kWholeWaves * cb) + l32; };
    const auto inside = [&](int cb, int ib, int v) { return row(ib, v) < m && column(cb) < n; };
    // byte offset of a block's element; the strides pass through the asm so that the compiler works offsets out where they are used
    // rather than keep one for every element from phase to phase
    const auto offsets = [&](int cb, int ib, auto use) {
        int si = tall ? 4 : 4 * cols, sj = tall ? 4 * cols : 4;
        asm volatile("" : "+s"(si), "+s"(sj));
        const int at = si * (32 * ib + 4 * lh) + sj * column(cb);
        use([&](int v) { return at + si * (8 * (v >> 2) + (v & 3)); });
    };
    typedef unsigned u4 __attribute__((ext_vector_type(4)));
    // a lane's 16 elements of a block; of a tall matrix four neighbours at a time
    const auto load = [&](const __amdgpu_buffer_rsrc_t& q, int cb, int ib, unsigned* d) {
        offsets(cb, ib, [&](auto at) {
            if (tall) {
#pragma unroll
                for (int v = 0; v < 16; v += 4) {
                    const u4 t = __builtin_bit_cast(u4, __builtin_amdgcn_raw_buffer_load_b128(q, at(v), 0, 0));
#pragma unroll
                    for (int e = 0; e < 4; ++e) d[v + e] = t[e];
                }
            } else {
#pragma unroll
                for (int v = 0; v < 16; ++v) d[v] = __builtin_amdgcn_raw_buffer_load_b32(q, at(v), 0, 0);
            }
        });
    };
    const auto store = [&](const __amdgpu_buffer_rsrc_t& q, int cb, int ib, const unsigned* d) {
        offsets(cb, ib, [&](auto at) {
            if (tall && m % 4 == 0) {                    // (groups of four rows are in or out as one)
#pragma unroll
                for (int v = 0; v < 16; v += 4)
                    __builtin_amdgcn_raw_buffer_store_b128(u4{d[v], d[v + 1], d[v + 2], d[v + 3]}, q, inside(cb, ib, v) ? at(v) : -1, 0, 0);
            } else {
#pragma unroll
                for (int v = 0; v < 16; ++v) __builtin_amdgcn_raw_buffer_store_b32(d[v], q, inside(cb, ib, v) ? at(v) : -1, 0, 0);
            }
        });
    };

    unsigned w[CB][MB][16];                              // X: first u, float32, then packed halves
    const __amdgpu_buffer_rsrc_t gr = rsrc(grad), mr = rsrc(mom);
#pragma unroll
    for (int cb = 0; cb < CB; ++cb)
#pragma unroll
        for (int ib = 0; ib < MB; ++ib) load(gr, cb, ib, w[cb][ib]);
    unsigned old[2][16];                                 // the momentum, a block ahead
    if (kUpdate) load(mr, 0, 0, old[0]);
    double sum = 0.0;
#pragma unroll
    for (int b = 0; b < CB * MB; ++b) {
        const int cb = b / MB, ib = b % MB;
        if (kUpdate && b + 1 < CB * MB) load(mr, (b + 1) / MB, (b + 1) % MB, old[(b + 1) & 1]);
        unsigned now[16];
#pragma unroll
        for (int v = 0; v < 16; ++v) {
            float u = __uint_as_float(w[cb][ib][v]);
            if (kUpdate) {
                const float x = fmaf(mu, __uint_as_float(old[b & 1][v]), u);
                now[v] = __float_as_uint(x);
                u = muon_update(u, x, mu, nesterov);
            }
            u = inside(cb, ib, v) ? u : 0.f;
            sum += (double)u * (double)u;
            w[cb][ib][v] = __float_as_uint(u);
        }
        if (kUpdate) store(mr, cb, ib, now);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
    if (lane == 0) red[wave] = sum;
    __syncthreads();
    sum = 0.0;
#pragma unroll
    for (int i = 0; i < kWholeWaves; ++i) sum += red[i];
    int power = 0;
    const float factor = sum != 0.0 ? (float)frexp((double)kScaleX / sqrt(sum), &power) : 0.f;
#pragma unroll
    for (int cb = 0; cb < CB; ++cb)
#pragma unroll
        for (int ib = 0; ib < MB; ++ib)
#pragma unroll
            for (int v = 0; v < 16; ++v) w[cb][ib][v] = split_pack(ldexpf(__uint_as_float(w[cb][ib][v]), power) * factor);

    if (state != nullptr) lr = (float)state[3];
    const float keep = 1.0f - lr * wd, step = lr * args->t[k].gain;
    for (int s = 0; s < steps; ++s) {
        {   // A = X X^T: this wave's columns
            f16v acc[NP];
#pragma unroll
            for (int p = 0; p < NP; ++p)
#pragma unroll
                for (int v = 0; v < 16; ++v) acc[p][v] = 0.f;
            unsigned(*turned)[36] = reinterpret_cast<unsigned(*)[36]>(region);
#pragma unroll
            for (int cb = 0; cb < CB; ++cb) {
                if (wave + kWholeWaves * cb >= blocks) continue;
#pragma unroll
                for (int ib = 0; ib < MB; ++ib)
#pragma unroll
                    for (int v = 0; v < 16; ++v) turned[row(ib, v)][l32] = w[cb][ib][v];
                __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    half8 h[MB], l[MB];
#pragma unroll
                    for (int ib = 0; ib < MB; ++ib) {
                        const u4* q = reinterpret_cast<const u4*>(&turned[32 * ib + l32][16 * t + 8 * lh]);
                        const u4 x = q[0], y = q[1];
                        const unsigned z[8] = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
                        whole_halves(z, h[ib], l[ib]);
                    }
                    acc[0] = whole_mfma(h[0], l[0], h[0], l[0], acc[0]);
                    if constexpr (MB == 2) {
                        acc[1] = whole_mfma(h[0], l[0], h[1], l[1], acc[1]);
                        acc[2] = whole_mfma(h[1], l[1], h[1], l[1], acc[2]);
                    }
                }
                __builtin_amdgcn_wave_barrier();
            }
            f4* part = reinterpret_cast<f4*>(region);
#pragma unroll
            for (int p = 0; p < NP; ++p)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    part[(p * 4 + q) * 64 + lane] = f4{acc[p][4 * q], acc[p][4 * q + 1], acc[p][4 * q + 2], acc[p][4 * q + 3]};
        }
        __syncthreads();
        for (int e = threadIdx.x; e < NP * 256; e += 64 * kWholeWaves) {
            f4 a = reinterpret_cast<const f4*>(regions[0])[e];
            for (int i = 1; i < busy; ++i) a += reinterpret_cast<const f4*>(regions[i])[e];
            const int p = e >> 8, q = (e >> 6) & 3, ln = e & 63;
            const int ib = p == 2 ? 1 : 0, jb = p == 0 ? 0 : 1;         // (0, 0), (0, 1), (1, 1)
            const int r = 32 * ib + 8 * q + 4 * (ln >> 5), c = 32 * jb + (ln & 31);
            half4 hi, lo;
            const float x[4] = {a[0] * split_scale<kSplitGram>(), a[1] * split_scale<kSplitGram>(), a[2] * split_scale<kSplitGram>(),
                                a[3] * split_scale<kSplitGram>()};
            whole_split(x, hi, lo);
            *reinterpret_cast<half4*>(&a_hi[c][r]) = hi;
            *reinterpret_cast<half4*>(&a_lo[c][r]) = lo;
            if (ib != jb)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    a_hi[r + i][c] = hi[i];
                    a_lo[r + i][c] = lo[i];
                }
        }
        __syncthreads();
        if (wave < MB * MB) {                            // B = a I + b A + c A^2, a block a wave
            const int ib = wave / MB, jb = wave % MB;
            f16v acc, low;                               // high.high; the two with a low half
#pragma unroll
            for (int v = 0; v < 16; ++v) acc[v] = low[v] = 0.f;
#pragma unroll
            for (int t = 0; t < 2 * MB; ++t) {
                const int x = 16 * t + 8 * lh;
                const half8 ah = *reinterpret_cast<const half8*>(&a_hi[32 * ib + l32][x]), al = *reinterpret_cast<const half8*>(&a_lo[32 * ib + l32][x]);
                const half8 bh = *reinterpret_cast<const half8*>(&a_hi[32 * jb + l32][x]), bl = *reinterpret_cast<const half8*>(&a_lo[32 * jb + l32][x]);
                low = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah, bl, low, 0, 0, 0);
                acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah, bh, acc, 0, 0, 0);
                low = __builtin_amdgcn_mfma_f32_32x32x16_f16(al, bh, low, 0, 0, 0);
            }
            const int c = 32 * jb + l32;
#pragma unroll
            for (int v = 0; v < 16; v += 4) {
                const int r = row(ib, v);
                const half4 ah = *reinterpret_cast<const half4*>(&a_hi[c][r]), al = *reinterpret_cast<const half4*>(&a_lo[c][r]);
                half4 hi, lo;
                float b[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    b[e] = (acc[v + e] + low[v + e]) * split_scale<kSplitPoly>() + ((float)ah[e] + (float)al[e]) * (kNsB * kScaleB / kScaleA);
                    if (r + e == c) b[e] += kNsA * kScaleB;
                }
                whole_split(b, hi, lo);
                *reinterpret_cast<half4*>(&b_hi[c][muon_slot(r)]) = hi;
                *reinterpret_cast<half4*>(&b_lo[c][muon_slot(r)]) = lo;
            }
        }
        __syncthreads();
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) {                // X = B X
            if (wave + kWholeWaves * cb >= blocks) continue;
            f16v acc[MB];
#pragma unroll
            for (int ib = 0; ib < MB; ++ib)
#pragma unroll
                for (int v = 0; v < 16; ++v) acc[ib][v] = 0.f;
#pragma unroll
            for (int t = 0; t < 2 * MB; ++t) {
                half8 xh, xl;
                whole_halves(&w[cb][t >> 1][8 * (t & 1)], xh, xl);
#pragma unroll
                for (int ib = 0; ib < MB; ++ib) {
                    const half8 bh = *reinterpret_cast<const half8*>(&b_hi[32 * ib + l32][16 * t + 8 * lh]);
                    const half8 bl = *reinterpret_cast<const half8*>(&b_lo[32 * ib + l32][16 * t + 8 * lh]);
                    acc[ib] = whole_mfma(bh, bl, xh, xl, acc[ib]);
                }
            }
            if (s + 1 < steps) {
#pragma unroll
                for (int ib = 0; ib < MB; ++ib)
#pragma unroll
                    for (int v = 0; v < 16; ++v) w[cb][ib][v] = split_pack(acc[ib][v] * split_scale<kSplitStep>());
                continue;
            }
#pragma unroll
            for (int ib = 0; ib < MB; ++ib) {
                const __amdgpu_buffer_rsrc_t d = rsrc(kUpdate ? theta : out);
                unsigned t[16];
                if (kUpdate) load(d, cb, ib, t);
#pragma unroll
                for (int v = 0; v < 16; ++v) {
                    const float o = acc[ib][v] * split_scale<kSplitApply>();
                    t[v] = __float_as_uint(kUpdate ? keep * __uint_as_float(t[v]) - step * o : o);
                }
                store(d, cb, ib, t);
            }
        }
    }
}

// ---- many steps: float32 products ------------------------------------------------------------------------------------
struct MuonScaleTable {
    int count;
    MuonMatrix t[kMuonMax];
    int parts[kMuonMax];                                 // workgroups of muon_momentum
    int first[kMuonMax];                                 // first workgroup of muon_scale
    float* x[kMuonMax];
    double* sums;                                        // [count][kMuonParts]
};
static_assert(sizeof(MuonScaleTable) + 64 <= 4096 && sizeof(MuonTable) + 64 <= 4096, "a launch's arguments");

// X = u / |u| times 2^60, rows <= cols (transposed otherwise), padding 0; a 32 x 32 block of X a workgroup.
__global__ __launch_bounds__(256) void muon_scale(const MuonScaleTable tb, float mu, int nesterov) {
    __shared__ double red[4];
    __shared__ float block[32][33];
    typedef const MuonScaleTable __attribute__((address_space(4)))* table_ptr;
    const table_ptr args = (table_ptr)__builtin_amdgcn_kernarg_segment_ptr();
    int k = 0;
    while (k + 1 < tb.count && (int)blockIdx.x >= args->first[k + 1]) ++k;
    const float* __restrict__ grad = args->t[k].grad;
    const float* __restrict__ mom = args->t[k].mom;
    const int rows = args->t[k].rows, cols = args->t[k].cols;
    const bool tall = rows > cols;
    const MuonFloatLayout at = muon_float_layout(tall ? cols : rows, tall ? rows : cols, 0);
    const int b = blockIdx.x - args->first[k], across = (int)(at.np / 32);
    const int64_t i0 = (int64_t)(b / across) * 32, j0 = (int64_t)(b % across) * 32;         // of X
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
    double part = 0.0;
    for (int i = threadIdx.x; i < args->parts[k]; i += 256) part += args->sums[k * kMuonParts + i];
    const double sum = muon_block_sum(part, red);
    int power = 0;
    const float factor = sum != 0.0 ? (float)frexp((double)kFloatScale / sqrt(sum), &power) : 0.f;
    const int64_t r0 = tall ? j0 : i0, c0 = tall ? i0 : j0;                                  // of the matrix
#pragma unroll
    for (int v = y; v < 32; v += 8) {
        float w = 0.f;
        if (r0 + v < rows && c0 + x < cols) {
            const int64_t e = (r0 + v) * cols + c0 + x;
            w = mom != nullptr ? muon_update(grad[e], mom[e], mu, nesterov) : grad[e];
            w = ldexpf(w, power) * factor;
        }
        block[v][x] = w;
    }
    __syncthreads();
#pragma unroll
    for (int v = y; v < 32; v += 8) args->x[k][(i0 + v) * at.np + j0 + x] = tall ? block[x][v] : block[v][x];
}

// One launch for one product of every matrix.
template <bool kRows, bool kApply>
static int muon_float_product(FloatTable tb, float alpha, float beta, float lr, const double* state, float wd) {
    int64_t tiles = 0;
    for (int i = 0; i < tb.count; ++i) {
        tb.p[i].first = (int)tiles;
        tiles += (int64_t)(tb.p[i].M / 64) * (tb.p[i].N / 64);
    }
    hipLaunchKernelGGL((float_product<kRows, kApply>), dim3((unsigned)tiles), dim3(256), 0, ctx().stream, tb, alpha, beta, lr, state, wd);
    AETH_LAUNCH_CHECK();
    return AETH_OK;
}

static int muon_float_group(const MuonMatrix* t, int count, float lr, const double* state, float mu, int nesterov, float wd, int steps,
                            int64_t* need) {
    MuonTable norm = {};
    MuonScaleTable scale = {};
    FloatTable gram = {}, poly = {}, step[2] = {};
    MuonFloatLayout at[kMuonMax];
    int64_t bytes = (int64_t)count * kMuonParts * sizeof(double), blocks = 0;
    int parts = 1;
    norm.count = scale.count = gram.count = poly.count = step[0].count = step[1].count = count;
    for (int i = 0; i < count; ++i) {
        const int m = t[i].rows < t[i].cols ? t[i].rows : t[i].cols, n = t[i].rows < t[i].cols ? t[i].cols : t[i].rows;
        at[i] = muon_float_layout(m, n, bytes);
        bytes = at[i].end;
        norm.t[i] = scale.t[i] = t[i];
        norm.parts[i] = scale.parts[i] = muon_parts(t[i]);
        if (norm.parts[i] > parts) parts = norm.parts[i];
        scale.first[i] = (int)blocks;
        blocks += at[i].mp / 32 * (at[i].np / 32);
    }
    if (need != nullptr) {
        *need = std::max(*need, bytes);
        return AETH_OK;
    }
    void* ws;
    const int rc = workspace(bytes, &ws);
    if (rc) return rc;
    char* base = static_cast<char*>(ws);
    norm.sums = scale.sums = static_cast<double*>(ws);
    for (int i = 0; i < count; ++i) {
        float *x[2] = {(float*)(base + at[i].x[0]), (float*)(base + at[i].x[1])}, *a = (float*)(base + at[i].a), *b = (float*)(base + at[i].b);
        const int mp = (int)at[i].mp, np = (int)at[i].np;
        scale.x[i] = x[0];
        FloatProduct p = {};
        p.rows = t[i].rows, p.cols = t[i].cols, p.theta = t[i].theta, p.out = t[i].out, p.gain = t[i].gain;
        poly.p[i] = p;
        poly.p[i].P = poly.p[i].Q = poly.p[i].R = a, poly.p[i].D = b, poly.p[i].M = poly.p[i].N = poly.p[i].K = mp;
        for (int s = 0; s < 2; ++s) {
            p.P = b, p.Q = p.R = x[s], p.D = x[1 - s], p.M = p.K = mp, p.N = np;
            step[s].p[i] = p;
        }
    }
    hipStream_t st = ctx().stream;
    hipLaunchKernelGGL(muon_momentum, dim3(parts, count), dim3(256), 0, st, norm, mu, nesterov);
    AETH_LAUNCH_CHECK();
    hipLaunchKernelGGL(muon_scale, dim3((unsigned)blocks), dim3(256), 0, st, scale, mu, nesterov);
    AETH_LAUNCH_CHECK();
    const float unit = 1.f / kFloatScale;
    gram.count = count;
    for (int s = 0; s < steps; ++s) {
        for (int i = 0; i < count; ++i) {
            FloatProduct& p = gram.p[i];
            p.P = p.Q = step[s & 1].p[i].Q, p.D = (float*)(base + at[i].a);
            p.M = p.N = (int)at[i].mp, p.K = (int)at[i].np;
        }
        int e = muon_float_product<true, false>(gram, 0.f, unit, 0.f, nullptr, 0.f);
        if (e == AETH_OK) e = muon_float_product<true, false>(poly, kNsB, kNsC * unit, 0.f, nullptr, 0.f);     // (A is symmetric)
        if (e == AETH_OK)
            e = s + 1 < steps ? muon_float_product<false, false>(step[s & 1], kNsA, unit, 0.f, nullptr, 0.f)
                              : muon_float_product<false, true>(step[s & 1], kNsA, unit, lr, state, wd);
        if (e) return e;
    }
    return AETH_OK;
}

// ---- the products on float16 halves ------------------------------------------------------------------------------------
// One launch for one product of every matrix, in tiles of BM x BN.
template <int BM, int BN, int WM, int WN, int NBUF, int BLOCK, int USE>
static int muon_launch(SplitTable tb, float lr, const double* state, float wd) {
    constexpr bool kSym = USE == kSplitGram || USE == kSplitPoly || USE == kSplitPart;
    int64_t tiles = 0;
    for (int i = 0; i < tb.count; ++i) {
        tb.p[i].first = (int)tiles;
        tb.p[i].tm = cdiv(tb.p[i].M, BM);
        tb.p[i].tn = cdiv(tb.p[i].N, BN);
        tb.p[i].tiles = (int)muon_tiles(tb.p[i].M, tb.p[i].N, BM, BN, kSym) * (USE == kSplitPart ? tb.p[i].runs : 1);
        tiles += tb.p[i].tiles;
    }
    if constexpr (BM == 32)
        hipLaunchKernelGGL((split_block<USE>), dim3((unsigned)tiles), dim3(256), 0, ctx().stream, tb, lr, state, wd);
    else
        hipLaunchKernelGGL((split_product<BM, BN, WM, WN, NBUF, BLOCK, USE>), dim3((unsigned)tiles), dim3(64 * (BM / WM) * (BN / WN)), 0,
                           ctx().stream, tb, lr, state, wd);
    AETH_LAUNCH_CHECK();
    return AETH_OK;
}

template <int USE>
static int muon_launch_tile(int tile, const SplitTable& tb, float lr, const double* state, float wd) {
    if (tile == kTile32) return muon_launch<32, 32, 32, 32, 3, 32, USE>(tb, lr, state, wd);
    if (tile == kTile64) return muon_launch<64, 64, 32, 32, 4, 32, USE>(tb, lr, state, wd);
    if constexpr (USE != kSplitPart) {
        if (tile == kTile96) return muon_launch<96, 96, 48, 48, 3, 16, USE>(tb, lr, state, wd);
        if (tile == kTile160) return muon_launch<160, 160, 80, 80, 3, 16, USE>(tb, lr, state, wd);
        if (tile == kTile192) return muon_launch<192, 192, 96, 96, 3, 16, USE>(tb, lr, state, wd);
        if constexpr (USE == kSplitStep || USE == kSplitApply) {
            if (tile == kTile256x128) return muon_launch<256, 128, 64, 64, 3, 32, USE>(tb, lr, state, wd);
        }
    }
    return muon_launch<128, 128, 64, 64, 4, 32, USE>(tb, lr, state, wd);
}

template <int USE>
static int muon_product(const SplitTable& tb, float lr, const double* state, float wd) {
    MuonShape shapes[kMuonMax];
    for (int i = 0; i < tb.count; ++i) shapes[i] = MuonShape{tb.p[i].M, tb.p[i].N, tb.p[i].K};
    return muon_launch_tile<USE>(muon_choose(shapes, tb.count, USE == kSplitGram || USE == kSplitPoly), tb, lr, state, wd);
}

// A = X X^T in runs of its columns.
static int muon_gram_runs(SplitTable tb, int tile) {
    const int rc = muon_launch_tile<kSplitPart>(tile, tb, 0.f, nullptr, 0.f);
    if (rc) return rc;
    int64_t groups = 0;
    for (int i = 0; i < tb.count; ++i) {
        tb.p[i].first = (int)groups;
        const int64_t side = tb.p[i].M / 32;
        tb.p[i].tiles = (int)(side * (side + 1) / 2);
        groups += tb.p[i].tiles;
    }
    hipLaunchKernelGGL(split_join, dim3((unsigned)groups), dim3(512), 0, ctx().stream, tb);
    AETH_LAUNCH_CHECK();
    return AETH_OK;
}

// The whole update of at most kMuonMax matrices that share the workspace.  With `need`: only the bytes of it, if they are more.
static int muon_group(const MuonMatrix* t, int count, float lr, const double* state, float mu, int nesterov, float wd, int steps,
                      int64_t* need) {
    MuonTable tb = {};
    SplitTable gram = {}, poly = {}, step[2] = {}, apply = {};
    MuonLayout at[kMuonMax];
    int64_t bytes = (int64_t)count * kMuonParts * sizeof(double), blocks = 0;
    int parts = 1;
    tb.count = gram.count = poly.count = step[0].count = step[1].count = apply.count = count;
    for (int i = 0; i < count; ++i) {
        const int m = t[i].rows < t[i].cols ? t[i].rows : t[i].cols, n = t[i].rows < t[i].cols ? t[i].cols : t[i].rows;
        at[i] = muon_layout(m, n, bytes);
        bytes = at[i].end;
        tb.t[i] = t[i];
        tb.parts[i] = muon_parts(t[i]);
        if (tb.parts[i] > parts) parts = tb.parts[i];
        tb.first[i] = (int)blocks;
        blocks += cdiv(at[i].mp / 32 * (at[i].np / 32), 4);
    }
    MuonShape shapes[kMuonMax];
    MuonRuns runs = {};
    for (int i = 0; i < count; ++i) shapes[i] = MuonShape{at[i].mp, at[i].mp, at[i].np};
    const bool in_runs = muon_choose_runs(shapes, count, &runs);
    const int64_t partial = bytes;                       // (after the matrices: a multiple of 4096 bytes from their begin)
    if (in_runs) bytes += runs.bytes;
    if (need != nullptr) {
        *need = std::max(*need, bytes);
        return AETH_OK;
    }
    void* ws;
    const int rc = workspace(bytes, &ws);
    if (rc) return rc;
    char* base = static_cast<char*>(ws);
    int64_t part_at = partial;
    tb.sums = static_cast<double*>(ws);
    for (int i = 0; i < count; ++i) {
        char *x = base + at[i].x, *xt[2] = {base + at[i].xt0, base + at[i].xt1}, *a = base + at[i].a, *b = base + at[i].b;
        const bool tall = t[i].rows > t[i].cols;
        const int mp = (int)at[i].mp, np = (int)at[i].np;
        tb.same[i] = tall ? xt[0] : x;
        tb.turned[i] = tall ? x : xt[0];
        SplitProduct p = {};
        p.rows = t[i].rows;
        p.cols = t[i].cols;
        p.theta = t[i].theta;
        p.out = t[i].out;
        p.gain = t[i].gain;
        p.P = p.Q = x, p.D1 = a, p.M = p.N = mp, p.K = np;
        if (in_runs) {
            p.runs = (int)runs.runs[i], p.run = (int)runs.run;
            p.part = reinterpret_cast<float*>(base + part_at);
            part_at += (int64_t)p.runs * (mp / 32) * (mp / 32 + 1) / 2 * 4096;
        }
        gram.p[i] = p;
        p.P = p.Q = p.A = a, p.D1 = b, p.K = mp;
        poly.p[i] = p;
        for (int s = 0; s < 2; ++s) {
            p.P = b, p.Q = xt[s], p.D1 = x, p.D2 = xt[1 - s], p.M = mp, p.N = np;
            step[s].p[i] = p;
        }
        // the last product comes out in the weights' own orientation: X = B X, or its transpose Xt B (B is symmetric)
        const char* last = xt[(steps - 1) & 1];
        p.P = tall ? last : b, p.Q = tall ? b : last, p.M = tall ? np : mp, p.N = tall ? mp : np;
        apply.p[i] = p;
    }
    hipStream_t st = ctx().stream;
    hipLaunchKernelGGL(muon_momentum, dim3(parts, count), dim3(256), 0, st, tb, mu, nesterov);
    AETH_LAUNCH_CHECK();
    hipLaunchKernelGGL(muon_split, dim3((unsigned)blocks), dim3(256), 0, st, tb, mu, nesterov);
    AETH_LAUNCH_CHECK();
    for (int s = 0; s < steps; ++s) {
        int e = in_runs ? muon_gram_runs(gram, runs.tile) : muon_product<kSplitGram>(gram, lr, state, wd);
        if (e == AETH_OK) e = muon_product<kSplitPoly>(poly, lr, state, wd);
        if (e == AETH_OK)
            e = s + 1 < steps ? muon_product<kSplitStep>(step[s & 1], lr, state, wd) : muon_product<kSplitApply>(apply, lr, state, wd);
        if (e) return e;
    }
    return AETH_OK;
}

// The column blocks a wave of muon_whole would have, 0 where a matrix is too large for it.  Its registers hold six blocks of 32 x 32 a
// wave, and that is also where the launches of all CUs catch up: an update of 64 rows takes 22 us at 64 columns, 29 at 256, 50 at
// 576 (58 on the transpose) and 59 at 768 in one workgroup, 55 to 65 in seventeen launches as fast as the host can queue them.
static int muon_whole_blocks(const MuonMatrix* t, int count, int* row_blocks) {
    int m = 0, n = 0;
    for (int i = 0; i < count; ++i) {
        const int lo = t[i].rows < t[i].cols ? t[i].rows : t[i].cols, hi = t[i].rows < t[i].cols ? t[i].cols : t[i].rows;
        if (lo > m) m = lo;
        if (hi > n) n = hi;
    }
    *row_blocks = cdiv(m, 32);
    const int blocks = cdiv(cdiv(n, 32), kWholeWaves);
    return *row_blocks <= 2 && blocks * *row_blocks <= 6 ? blocks : 0;
}

static int muon_small(const MuonMatrix* t, int count, int row_blocks, int blocks, float lr, const double* state, float mu,
                      int nesterov, float wd, int steps) {
    typedef void (*Whole)(const MuonTable, float, int, float, const double*, float, int);
    static const Whole one[2][4] = {{muon_whole<1, 1, false>, muon_whole<1, 2, false>, muon_whole<1, 4, false>, muon_whole<1, 6, false>},
                                    {muon_whole<1, 1, true>, muon_whole<1, 2, true>, muon_whole<1, 4, true>, muon_whole<1, 6, true>}};
    static const Whole two[2][3] = {{muon_whole<2, 1, false>, muon_whole<2, 2, false>, muon_whole<2, 3, false>},
                                    {muon_whole<2, 1, true>, muon_whole<2, 2, true>, muon_whole<2, 3, true>}};
    MuonTable tb = {};
    tb.count = count;
    for (int i = 0; i < count; ++i) tb.t[i] = t[i];
    const int c = blocks <= 1 ? 0 : blocks <= 2 ? 1 : blocks <= 4 ? 2 : 3;
    const int update = t[0].mom != nullptr;
    hipLaunchKernelGGL(row_blocks == 1 ? one[update][c] : two[update][c], dim3(count), dim3(64 * kWholeWaves), 0, ctx().stream, tb, mu,
                       nesterov, lr, state, wd, steps);
    AETH_LAUNCH_CHECK();
    return AETH_OK;
}

// Matrices whose buffers together pass this go out in several groups, one after the other.
constexpr int64_t kMuonWorkspace = (int64_t)4 << 30;

// group(first, how many) for every group; bytes(matrix): of its buffers.
template <typename Bytes, typename Group>
static int muon_in_groups(const MuonMatrix* t, int count, Bytes bytes, Group group) {
    for (int i = 0; i < count;) {
        int64_t sum = bytes(t[i]);
        int k = 1;
        while (i + k < count && sum + bytes(t[i + k]) <= kMuonWorkspace) sum += bytes(t[i + k++]);
        const int rc = group(t + i, k);
        if (rc) return rc;
        i += k;
    }
    return AETH_OK;
}

static int muon_run(MuonMatrix* t, int count, float lr, const double* state, float mu, int nesterov, float wd, int steps) {
    // those that two halves do not carry through the steps come last
    MuonMatrix* const rest = std::stable_partition(
        t, t + count, [&](const MuonMatrix& x) { return muon_in_halves(std::max(x.rows, x.cols), steps); });
    const int halves = (int)(rest - t), floats = count - halves;
    int row_blocks = 0;
    const int blocks = halves > 0 ? muon_whole_blocks(t, halves, &row_blocks) : 0;
    // the longest tiles first: what is left at a launch's end is short
    std::stable_sort(t, rest, [](const MuonMatrix& a, const MuonMatrix& b) {
        const int n = std::max(a.rows, a.cols), p = std::max(b.rows, b.cols);
        return n != p ? n > p : std::min(a.rows, a.cols) > std::min(b.rows, b.cols);
    });
    const auto all = [&](auto on_floats, auto on_halves) {
        const int rc = muon_in_groups(
            rest, floats, [](const MuonMatrix& x) { return muon_float_layout(std::min(x.rows, x.cols), std::max(x.rows, x.cols), 0).end; }, on_floats);
        if (rc || blocks > 0) return rc;
        return muon_in_groups(
            t, halves, [](const MuonMatrix& x) { return muon_layout(std::min(x.rows, x.cols), std::max(x.rows, x.cols), 0).end; }, on_halves);
    };
    const auto update = [&](int64_t* need) {
        return all([&](const MuonMatrix* g, int k) { return muon_float_group(g, k, lr, state, mu, nesterov, wd, steps, need); },
                   [&](const MuonMatrix* g, int k) { return muon_group(g, k, lr, state, mu, nesterov, wd, steps, need); });
    };
    int groups = 0;
    const auto one = [&](const MuonMatrix*, int) {
        ++groups;
        return AETH_OK;
    };
    all(one, one);
    if (groups > 1) {
        // the scratch of all groups before the first one's launches: a call that cannot have it changes nothing
        int64_t need = 0;
        void* ws;
        update(&need);
        const int rc = workspace(need, &ws);
        if (rc) return rc;
    }
    const int rc = update(nullptr);
    if (rc || blocks == 0) return rc;
    return muon_small(t, halves, row_blocks, blocks, lr, state, mu, nesterov, wd, steps);
}

static bool muon_size(int rows, int cols) {
    return rows >= 0 && cols >= 0 && rows <= kMuonLongest && cols <= kMuonLongest && (int64_t)rows * cols < ((int64_t)1 << 31);
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
        if (!muon_size(r, c))
            return fail(AETH_E_INVALID, "%s: matrix %d is %d x %d (sides of at most %d, below 2^31 elements)", fn, i, r, c, kMuonLongest);
        if (r == 0 || c == 0) continue;
        if (!theta[i] || !grad[i] || !mom[i]) return fail(AETH_E_INVALID, "%s: matrix %d has a NULL tensor", fn, i);
        t[k++] = MuonMatrix{theta[i], grad[i], mom[i], nullptr, r, c, c > r ? sqrtf((float)c / (float)r) : 1.f};
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
    return muon_run(t, k, lr, state, mu, nesterov, wd, steps);
}

}  // namespace aeth

using namespace aeth;

extern "C" {

int aeth_newton_schulz_f32(const float* g, float* o, int rows, int cols, int steps) {
    AETH_CHECK_ARG(muon_size(rows, cols));
    AETH_CHECK_ARG(steps >= 1 && steps <= 100);
    const int64_t bytes = (int64_t)rows * cols * 4;
    AETH_CHECK_ARG(bytes == 0 || (g && o && muon_apart(g, bytes, o, bytes)));
    AETH_REQUIRE_INIT();
    if (bytes == 0) return AETH_OK;
    MuonMatrix t{nullptr, g, nullptr, o, rows, cols, 1.f};
    return muon_run(&t, 1, 0.f, nullptr, 0.f, 0, 0.f, steps);
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
