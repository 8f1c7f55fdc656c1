// Products of matrices whose elements are held as two float16 halves.
//
// x = hi + lo with hi = float16(x) and lo = float16(x - hi): 22 bits of x where neither half leaves float16's normal range.  Every
// matrix is scaled by one power of two (kScale*); the low half is subnormal below 2^-18 of what the scale stands for (1, and |u| = 1
// for X), where x is held to 2^-40 (B, at half the scale, 2^-39).  hi.hi + hi.lo + lo.hi is x y up to 2^-22 of |x y| (the product of the low halves is left out),
// each of the three a float16 MFMA with float32 accumulation.  Three float16 products take 0.19 of the time of one float32 MFMA
// product of the same size at their peaks (2.5 PFLOP/s and 157 TFLOP/s).  muon_in_halves says how many steps of the update that
// bears: five steps on evenly scaled matrices are off by 2e-6 of the result, with float32 products by 3-4e-6.
#pragma once

#include "conv_common.h"
#include "muon_plan.h"

#include <type_traits>

namespace aeth {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));

// What a product's result becomes.
enum SplitUse {
    kSplitGram,          // D1 = P Q^T, symmetric
    kSplitPoly,          // D1 = a I + b A + c P Q^T, symmetric (P = Q = A)
    kSplitStep,          // D1 = P Q^T and D2 its transpose
    kSplitPart,          // part = P Q^T over a run of the columns, symmetric; split_join adds the runs
    kSplitApply,         // theta <- keep theta - step P Q^T, or out = P Q^T; float32, [rows][cols]
};

struct SplitProduct {
    const char *P, *Q, *A;
    char *D1, *D2;
    float *theta, *out;
    int M, N, K;         // padded: rows of P, rows of Q, their columns
    int rows, cols;      // of theta
    int first, tiles;    // this product's first tile; how many it has
    int tm, tn;          // tiles down and across
    int runs, run;       // kSplitPart: runs of so many slabs
    float* part;         // [run][32 x 32 block on or above the diagonal][1024]
    float gain;
};

struct SplitTable {
    int count;
    SplitProduct p[kMuonMax];
};
static_assert(sizeof(SplitTable) + 64 <= 4096, "a launch's arguments");

// Scales of the stored halves: X's elements are at most 1.21 (the step's polynomial maps [0, 1.21] into itself), A = X X^T's at most
// 1.47, the polynomial's a I + b A + c A^2 at most 3.45: all below 65504 times their scale's inverse.
constexpr float kScaleX = 32768.f, kScaleA = 32768.f, kScaleB = 16384.f;
constexpr float kNsA = 3.4445f, kNsB = -4.7750f, kNsC = 2.0315f;

// x's halves in one word: the high one below
__device__ __forceinline__ unsigned split_pack(float v) {
    const _Float16 hi = (_Float16)v, lo = (_Float16)(v - (float)hi);
    return (unsigned)__builtin_bit_cast(unsigned short, hi) | (unsigned)__builtin_bit_cast(unsigned short, lo) << 16;
}

// Eight neighbouring elements of a row: their high halves, their low halves
__device__ __forceinline__ void split_halves(const unsigned* w, u32x4& hi, u32x4& lo) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        hi[e] = __builtin_amdgcn_perm(w[2 * e + 1], w[2 * e], 0x05040100u);
        lo[e] = __builtin_amdgcn_perm(w[2 * e + 1], w[2 * e], 0x07060302u);
    }
}

// A buffer store's cache policy: through the L2 cache (device scope)
constexpr int kThrough = 16;

// What a product's accumulators are times the stored result's scale.
template <int USE>
__device__ constexpr float split_scale() {
    return USE == kSplitGram || USE == kSplitPart ? kScaleA / (kScaleX * kScaleX)
           : USE == kSplitPoly                    ? kNsC * kScaleB / (kScaleA * kScaleA)
           : USE == kSplitStep                    ? 1.f / kScaleB
                                                  : 1.f / (kScaleB * kScaleX);
}

// Half of a 32 x 32 block of a result (16 of its rows, or with `turned` of its columns) to its place in the result, or in the
// transposed one: four lanes a row, eight elements each, so that a store covers whole pieces of 64 bytes.  r, c, turned, h are
// uniform.  t: the block in LDS, [row][S], as halves (split_pack) or, for the polynomial, as float32 sums to which b A + a I is
// added here.  A and the result are symmetric: either way round the same bits are added.
template <int USE>
struct SplitRows {
    size_t block;                                        // of the block's 4096 bytes
    unsigned at;                                         // in them: the lane's eight high halves
    half8 high, low;                                     // of A
    __device__ __forceinline__ SplitRows(const SplitProduct& pr, int r, int c, bool turned, int h) {
        const int lane = threadIdx.x & 63;
        block = (turned ? (size_t)(r / 32) * pr.N + c : (size_t)(c / 32) * pr.M + r) * 128;
        at = (16 * h + (lane >> 2)) * 128 + 16 * (lane & 3);
        if (USE == kSplitPoly) {
            high = *reinterpret_cast<const half8*>(pr.A + block + at);
            low = *reinterpret_cast<const half8*>(pr.A + block + at + 64);
        }
    }
    template <int S>
    __device__ __forceinline__ void store(const SplitProduct& pr, const unsigned* t, int r, int c, bool turned, int h) const {
        const int lane = threadIdx.x & 63, row = 16 * h + (lane >> 2), col = 8 * (lane & 3);
        unsigned w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = turned ? t[(col + e) * S + row] : t[row * S + col + e];
        if (USE == kSplitPoly)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                float o = __builtin_bit_cast(float, w[e]) + ((float)high[e] + (float)low[e]) * (kNsB * kScaleB / kScaleA);
                if (r == c && row == col + e) o += kNsA * kScaleB;
                w[e] = split_pack(o);
            }
        u32x4 hi, lo;
        split_halves(w, hi, lo);
        // Written through to memory at once (kThrough), where the next launch's other dies read it: what stays in an L2 cache is
        // written back between the launches (five steps on 1000 x 1537 226.5 us, so 220.5; on 4096 x 4096 no difference).
        const __amdgpu_buffer_rsrc_t d =
            __builtin_amdgcn_make_buffer_rsrc((turned && USE == kSplitStep ? pr.D2 : pr.D1) + block, 0, 4096, 0x00020000);
        __builtin_amdgcn_raw_buffer_store_b128(hi, d, (int)at, 0, kThrough);
        __builtin_amdgcn_raw_buffer_store_b128(lo, d, (int)at + 64, 0, kThrough);
    }
};

// What lies in LDS of a sum.
template <int USE>
__device__ __forceinline__ unsigned split_word(float sum) {
    const float o = sum * split_scale<USE>();
    return USE == kSplitPoly ? __builtin_bit_cast(unsigned, o) : split_pack(o);
}

// The parameters of the workgroup's product and the number of its tile in it, by scalar loads from the kernel's arguments, of which the
// table is the first (an index into the struct itself would copy it to memory).  Neighbouring tiles are on one die, where they share
// operands in its L2 cache, but product by product, so that every die has its share of the long ones: two products of 128 slabs and
// four of 32 (272 and 544 tiles of 64 x 64) took 100 us with the launch's tiles dealt out as one row, and take 64; eight equal products
// are 5 % slower for it.
__device__ __forceinline__ SplitProduct split_find(const SplitTable& tb, int& tile) {
    typedef const SplitTable __attribute__((address_space(4)))* table_ptr;
    const table_ptr args = (table_ptr)__builtin_amdgcn_kernarg_segment_ptr();
    const int group = blockIdx.x;
    int at = 0;
    while (at + 1 < tb.count && group >= args->p[at + 1].first) ++at;
    SplitProduct pr = tb.p[0];
    __builtin_memcpy(&pr, (const void*)(args->p + at), sizeof(pr));
    tile = xcd_contiguous_id(group - pr.first, pr.tiles);
    return pr;
}

template <int N>
__device__ __forceinline__ void wait_loads() {           // at most N of this wave's loads are still on their way; its LDS reads are done
    static_assert(N < 64, "vmcnt has six bits");
    asm volatile("" ::: "memory");                       // (the compiler keeps its reads of the LDS on their side)
    __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | (0 << 8) | ((N >> 4) << 14));
    asm volatile("" ::: "memory");
}

// The tile of the result that number `t` of a product's tiles is, and the slabs it adds up.
struct SplitTile {
    int i, j, begin, slabs;
};
template <int USE>
__device__ __forceinline__ SplitTile split_tile(const SplitProduct& pr, int t) {
    SplitTile at{0, 0, 0, pr.K / 32};
    if (USE == kSplitPart) {
        // run by run: neighbours in time read the same columns
        const int triangle = pr.tn * (pr.tn + 1) / 2, run = t / triangle;
        muon_triangle(t - run * triangle, &at.i, &at.j);
        at.begin = run * pr.run;
        at.slabs = min(at.slabs - at.begin, pr.run);
    } else if (USE == kSplitGram || USE == kSplitPoly) {
        muon_triangle(t, &at.i, &at.j);
    } else {
        // bands of four tile rows, walked column by column: neighbours in time share operands in their XCD's L2
        const int band = t / (4 * pr.tn), in = t - band * 4 * pr.tn;
        const int height = min(4, pr.tm - band * 4);
        at.j = in / height;
        at.i = band * 4 + in - at.j * height;
    }
    // (the divisions are done in vector registers; what follows from them are the loads' scalar descriptors)
    at.i = __builtin_amdgcn_readfirstlane(at.i);
    at.j = __builtin_amdgcn_readfirstlane(at.j);
    return at;
}

template <int BLOCK>
struct SplitAcc;
template <>
struct SplitAcc<32> {
    typedef f16v type;
};
template <>
struct SplitAcc<16> {
    typedef f4 type;
};

// theta <- keep theta - step D (or out = D) for one block of a product's accumulators: acc[v] is row r + 8 (v / 4) + 4 (lane / 32) +
// v % 4 and column c + lane % 32 of a 32 x 32 block, row r + 4 (lane / 16) + v and column c + lane % 16 of a 16 x 16 one.
// All the loads go out at once, from places clamped into the matrix: behind a branch each they came back one by one.
template <int BLOCK>
__device__ __forceinline__ void split_apply(const SplitProduct& pr, const typename SplitAcc<BLOCK>::type& acc, int r, int c, float keep,
                                            float step) {
    constexpr int N = BLOCK * BLOCK / 64;
    const int lane = threadIdx.x & 63, x = c + (lane & (BLOCK - 1)), cc = min(x, pr.cols - 1), y0 = r + lane / BLOCK * 4;
    float t[N];
    if (pr.theta != nullptr) {
#pragma unroll
        for (int v = 0; v < N; ++v) t[v] = pr.theta[(size_t)min(y0 + 8 * (v >> 2) + (v & 3), pr.rows - 1) * pr.cols + cc];
    }
#pragma unroll
    for (int v = 0; v < N; ++v) {
        const int y = y0 + 8 * (v >> 2) + (v & 3);
        if (y < pr.rows && x < pr.cols) {
            const float o = acc[v] * split_scale<kSplitApply>();
            if (pr.theta != nullptr) pr.theta[(size_t)y * pr.cols + x] = keep * t[v] - step * o;
            else pr.out[(size_t)y * pr.cols + x] = o;
        }
    }
}

// The partial sums of a 32 x 32 block, as the matrix instruction leaves them: quarter q of them (lane's sums 4 q .. 4 q + 3).
__device__ __forceinline__ void split_part(const SplitProduct& pr, const f4& sums, int q, int r, int c, const SplitTile& at) {
    const size_t side = pr.M / 32, x = c / 32, block = x * (x + 1) / 2 + r / 32;
    float* d = pr.part + ((size_t)(at.begin / pr.run) * (side * (side + 1) / 2) + block) * 1024;
    const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(d, 0, 4096, 0x00020000);
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, sums), rsrc, 1024 * q + 16 * (int)(threadIdx.x & 63), 0, kThrough);
}

__device__ __forceinline__ f16v split_mfma(const half8& a, const half8& b, const f16v& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f4 split_mfma(const half8& a, const half8& b, const f4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// A matrix lies slab by slab: slab s holds columns 32 s .. 32 s + 31 of all R rows, row r's 128 bytes (64 of high halves, 64 of low)
// at (s R + r) * 128, so that what a tile reads at a time is one contiguous piece and no offset grows with the matrix.
// One workgroup: BM x BN of the result, waves of WM x WN, slabs through a ring of NBUF LDS buffers, loaded straight into LDS
// NBUF - 1 slabs ahead.  16-byte chunk c of row r lies at c ^ ((r >> 1) & 7): the 16 rows that a fragment read takes at a time
// then lie in different banks.
// BLOCK: the MFMA's result, 32 x 32 (16 columns a step) or 16 x 16 (32 columns, a whole slab).  The small one is for waves of 48 or 80
// rows and columns, and for 96 x 96: there it keeps one step's operands fewer (2048 x 2048 in 96 x 96 tiles: 42 us with four waves
// of 48 x 48, 44 with three of 96 x 32; 4096 x 4096 in 192 x 192: 190 us, with 32 x 32 blocks 198; before the results went through
// LDS).
// Bound: with a tile on every CU, the power the matrix units draw (4096 x 4096: 1.15-1.25 PFLOP/s of float16, what a library's
// float16 product of that size reaches); below that, with one wave a SIMD, a slab's barrier, LDS reads and MFMAs one after the other
// and a tile's first loads and epilogue (more slabs in flight change nothing).
template <int BM, int BN, int WM, int WN, int NBUF, int BLOCK, int USE>
__global__ __launch_bounds__(64 * (BM / WM) * (BN / WN)) void split_product(const SplitTable tb, float lr,
                                                                           const double* __restrict__ state, float wd) {
    constexpr int WAVES = (BM / WM) * (BN / WN), TM = WM / BLOCK, TN = WN / BLOCK, STEPS = BLOCK / 16;
    constexpr int AL = BM / 8 / WAVES, BL = BN / 8 / WAVES;
    static_assert(AL * 8 * WAVES == BM && BL * 8 * WAVES == BN, "whole loads a wave");
    constexpr int BUF = (BM + BN) * 128;
    constexpr bool kSym = USE == kSplitGram || USE == kSplitPoly || USE == kSplitPart;
    constexpr bool kStaged = USE != kSplitPart && USE != kSplitApply;
    constexpr int S = BN + 1, STAGE = kStaged ? BM * S * 4 : 0;
    __shared__ __attribute__((aligned(1024))) char lds[NBUF * BUF > STAGE ? NBUF * BUF : STAGE];

    int tile;
    const SplitProduct pr = split_find(tb, tile);
    const SplitTile at = split_tile<USE>(pr, tile);
    const int slabs = at.slabs;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int r0 = at.i * BM, c0 = at.j * BN;
    // the next slab's rows
    const char *sp = pr.P + ((size_t)at.begin * pr.M + r0) * 128, *sq = pr.Q + ((size_t)at.begin * pr.N + c0) * 128;
    const unsigned np = (unsigned)min(pr.M - r0, BM) * 128u, nq = (unsigned)min(pr.N - c0, BN) * 128u;
    const size_t dp = (size_t)pr.M * 128, dq = (size_t)pr.N * 128;
    unsigned vp[AL], vq[BL];                             // (rows behind the matrix are behind the descriptor's end: they read as zeros)
#pragma unroll
    for (int i = 0; i < AL; ++i) {
        const unsigned r = (unsigned)(wave * AL + i) * 8 + (lane >> 3);
        vp[i] = r * 128u + (((unsigned)lane & 7u) ^ ((r >> 1) & 7u)) * 16u;
    }
#pragma unroll
    for (int i = 0; i < BL; ++i) {
        const unsigned r = (unsigned)(wave * BL + i) * 8 + (lane >> 3);
        vq[i] = r * 128u + (((unsigned)lane & 7u) ^ ((r >> 1) & 7u)) * 16u;
    }
    const unsigned lds0 = lds_address(lds);
    constexpr int LOADS = AL + BL;
    const auto load = [&](int i, int buf) {              // one of a wave's loads of the next slab
        const unsigned base = lds0 + (unsigned)buf * BUF;
        if (i < AL) lds_direct_load16(raw_rsrc(sp, np), base + (unsigned)(wave * AL + i) * 1024u, vp[i]);
        else lds_direct_load16(raw_rsrc(sq, nq), base + BM * 128u + (unsigned)(wave * BL + i - AL) * 1024u, vq[i - AL]);
    };
    const auto advance = [&] {
        sp += dp;
        sq += dq;
    };

    typename SplitAcc<BLOCK>::type acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int v = 0; v < BLOCK * BLOCK / 64; ++v) acc[i][j][v] = 0.f;

    const int wm = (wave / (BN / WN)) * WM, wn = (wave % (BN / WN)) * WN;
    // a lane's operand row and its chunk of the row's columns, in the first block
    const unsigned row = (unsigned)lane & (BLOCK - 1), sw = (((unsigned)lane / BLOCK) ^ ((row >> 1) & 7u)) * 16u;
    const unsigned fa = (wm + row) * 128u + sw, fb = (BM + wn + row) * 128u + sw;
    // One slab: two steps of 16 columns (one of 32), three products each.  The next slab's loads go out one by one between the
    // MFMAs: a wave that issues them all at once waits for the load unit's queue with its MFMAs behind it (4096 x 4096, tiles of
    // 192 x 192: 195 us a product, all at once 215).
    const auto multiply = [&](int buf, int into, auto loads) {
        const char* b = lds + buf * BUF;
        half8 f[STEPS][2 * TM + 2 * TN];                 // high and low halves of both operands' rows, for every step
        const auto read = [&](int t) {
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                f[t][i] = *reinterpret_cast<const half8*>(b + ((fa ^ (t * 32u)) + i * (BLOCK * 128u)));
                f[t][TM + i] = *reinterpret_cast<const half8*>(b + ((fa ^ (t * 32u + 64u)) + i * (BLOCK * 128u)));
            }
#pragma unroll
            for (int j = 0; j < TN; ++j) {
                f[t][2 * TM + j] = *reinterpret_cast<const half8*>(b + ((fb ^ (t * 32u)) + j * (BLOCK * 128u)));
                f[t][2 * TM + TN + j] = *reinterpret_cast<const half8*>(b + ((fb ^ (t * 32u + 64u)) + j * (BLOCK * 128u)));
            }
        };
        read(0);
#pragma unroll
        for (int t = 0; t < STEPS; ++t) {
#pragma unroll
            for (int g = 0; g < 3; ++g) {                // high.low, low.high, high.high
                if (STEPS == 2 && t == 0 && g == 1) read(1);
#pragma unroll
                for (int i = 0; i < TM; ++i) {
                    const half8 x = f[t][(g == 1 ? TM : 0) + i];
#pragma unroll
                    for (int j = 0; j < TN; ++j)
                        acc[i][j] = split_mfma(x, f[t][2 * TM + (g == 0 ? TN : 0) + j], acc[i][j]);
                    constexpr int GROUPS = 3 * STEPS * TM;
                    const int u = (t * 3 + g) * TM + i;
                    if (decltype(loads)::value) {
#pragma unroll
                        for (int k = u * LOADS / GROUPS; k < (u + 1) * LOADS / GROUPS; ++k) {
                            __builtin_amdgcn_sched_barrier(0);
                            load(k, into);
                            __builtin_amdgcn_sched_barrier(0);
                        }
                    }
                }
            }
        }
        if (decltype(loads)::value) advance();
    };
#pragma unroll
    for (int d = 0; d < NBUF - 1; ++d)
        if (d < slabs) {
#pragma unroll
            for (int i = 0; i < LOADS; ++i) load(i, d);
            advance();
        }
    int buf = 0, next = NBUF - 1;
    const auto turn = [&] {
        buf = buf + 1 == NBUF ? 0 : buf + 1;
        next = next + 1 == NBUF ? 0 : next + 1;
    };
    int s = 0;
    for (; s + NBUF - 1 < slabs; ++s) {
        wait_loads<LOADS * (NBUF - 2)>();                // slab s has landed (NBUF - 2 later ones are on their way)
        asm volatile("s_barrier" ::: "memory");          // for every wave; and every wave is done with slab s - 1, whose buffer is next
        multiply(buf, next, std::true_type{});
        turn();
    }
    for (; s < slabs; ++s) {
        wait_loads<0>();
        asm volatile("s_barrier" ::: "memory");
        multiply(buf, next, std::false_type{});
        turn();
    }
    wait_loads<0>();
    asm volatile("s_barrier" ::: "memory");              // the epilogue uses the buffers as well

    if constexpr (!kStaged) {
        if (state != nullptr) lr = (float)state[3];
        const float keep = 1.0f - lr * wd, step = lr * pr.gain;
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) {
                const int r = r0 + wm + BLOCK * i, c = c0 + wn + BLOCK * j;
                if (r >= pr.M || c >= pr.N || (kSym && r > c)) continue;
                if constexpr (USE == kSplitApply) {
                    split_apply<BLOCK>(pr, acc[i][j], r, c, keep, step);
                } else {
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        split_part(pr, f4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]}, q, r, c, at);
                }
            }
        return;
    }
    // The tile goes through LDS, where every wave reads whole blocks of 32 x 32 either way round (from the accumulators, in pieces of
    // 8 or 16 bytes a row: 4096 x 4096 step 345 us instead of 330, 1024 x 4096 33 instead of 30; but the weights, whose rows the
    // accumulators hold in pieces of 64 or 128 bytes, took 38 us that way instead of 32).
    unsigned* t = reinterpret_cast<unsigned*>(lds);
    unsigned* mine = t + (wm + lane / BLOCK * 4) * S + wn + (lane & (BLOCK - 1));
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int v = 0; v < BLOCK * BLOCK / 64; ++v)
                mine[(BLOCK * i + 8 * (v >> 2) + (v & 3)) * S + BLOCK * j] = split_word<USE>(acc[i][j][v]);
    __syncthreads();
    for (int b = wave; b < (BM / 32) * (BN / 32); b += WAVES) {
        const int i = b / (BN / 32), j = b % (BN / 32), r = r0 + 32 * i, c = c0 + 32 * j;
        if (r >= pr.M || c >= pr.N) continue;        // (whole blocks: both are multiples of 32)
        if (kSym && r > c) continue;                 // (below the diagonal of a diagonal tile: written from above it)
        const unsigned* block = t + 32 * i * S + 32 * j;
        const SplitRows<USE> top(pr, r, c, false, 0), bottom(pr, r, c, false, 1), left(pr, r, c, true, 0), right(pr, r, c, true, 1);
        top.template store<S>(pr, block, r, c, false, 0);
        bottom.template store<S>(pr, block, r, c, false, 1);
        if (kSym && r == c) continue;                // (a diagonal block: each place is written once)
        left.template store<S>(pr, block, r, c, true, 0);
        right.template store<S>(pr, block, r, c, true, 1);
    }
}

// The same for products so small that a launch's time is what its loads and its epilogue take one after the other: a 32 x 32
// block a workgroup, every fourth slab a wave, which loads and reads its own ring without a barrier; the waves' sums are added in
// their order.  256 x 256 x 256: 4.5 us where 64 x 64 tiles take 7.1.
template <int USE>
__global__ __launch_bounds__(256) void split_block(const SplitTable tb, float lr, const double* __restrict__ state, float wd) {
    constexpr int NBUF = 3, BUF = 64 * 128;
    __shared__ __attribute__((aligned(1024))) char lds[4 * NBUF * BUF];
    int tile;
    const SplitProduct pr = split_find(tb, tile);
    const SplitTile at = split_tile<USE>(pr, tile);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int l32 = lane & 31, lh = lane >> 5, r0 = at.i * 32, c0 = at.j * 32;
    const char *sp = pr.P + ((size_t)(at.begin + wave) * pr.M + r0) * 128, *sq = pr.Q + ((size_t)(at.begin + wave) * pr.N + c0) * 128;
    const size_t dp = (size_t)pr.M * 512, dq = (size_t)pr.N * 512;
    const int slabs = (at.slabs - wave + 3) / 4;         // this wave's (none for a wave behind the last slab)
    unsigned off[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const unsigned r = (unsigned)i * 8 + (lane >> 3);
        off[i] = r * 128u + (((unsigned)lane & 7u) ^ ((r >> 1) & 7u)) * 16u;
    }
    char* ring = lds + wave * (NBUF * BUF);
    const unsigned ring0 = lds_address(ring);
    const auto fetch = [&](int buf) {
        const u32x4 rp = raw_rsrc(sp, 32 * 128), rq = raw_rsrc(sq, 32 * 128);
#pragma unroll
        for (int i = 0; i < 4; ++i) lds_direct_load16(rp, ring0 + (unsigned)buf * BUF + i * 1024u, off[i]);
#pragma unroll
        for (int i = 0; i < 4; ++i) lds_direct_load16(rq, ring0 + (unsigned)buf * BUF + 4096u + i * 1024u, off[i]);
        sp += dp;
        sq += dq;
    };
    f16v acc;
#pragma unroll
    for (int v = 0; v < 16; ++v) acc[v] = 0.f;
    const unsigned f0 = (unsigned)l32 * 128u + (unsigned)(lh ^ ((l32 >> 1) & 7)) * 16u;
    const auto multiply = [&](int buf) {
        const char* b = ring + buf * BUF;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const half8 ah = *reinterpret_cast<const half8*>(b + (f0 ^ (t * 32u))), al = *reinterpret_cast<const half8*>(b + (f0 ^ (t * 32u + 64u)));
            const half8 bh = *reinterpret_cast<const half8*>(b + 4096 + (f0 ^ (t * 32u))), bl = *reinterpret_cast<const half8*>(b + 4096 + (f0 ^ (t * 32u + 64u)));
            acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah, bl, acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(al, bh, acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah, bh, acc, 0, 0, 0);
        }
    };
#pragma unroll
    for (int d = 0; d < NBUF - 1; ++d)
        if (d < slabs) fetch(d);
    int buf = 0, next = NBUF - 1;
    for (int s = 0; s < slabs; ++s) {
        // slab s has landed, and what was read of the slab before is in registers: its buffer takes the slab after next
        if (s + 1 < slabs) wait_loads<8 * (NBUF - 2)>();
        else wait_loads<0>();
        if (s + NBUF - 1 < slabs) fetch(next);
        multiply(buf);
        buf = buf + 1 == NBUF ? 0 : buf + 1;
        next = next + 1 == NBUF ? 0 : next + 1;
    }
    // (every wave's loads have landed and its reads are done where it writes its sums: over its own ring)
    wait_loads<0>();
    f4* sums = reinterpret_cast<f4*>(ring);
#pragma unroll
    for (int q = 0; q < 4; ++q) sums[64 * q + lane] = f4{acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]};
    // a quarter of the rows is added up by each wave: its sums e are row 8 wave + 4 lh + e, column l32
    const auto add = [&] {
        __syncthreads();
        f4 sum = reinterpret_cast<const f4*>(lds)[64 * wave + lane];
#pragma unroll
        for (int w = 1; w < 4; ++w) sum += reinterpret_cast<const f4*>(lds + w * (NBUF * BUF))[64 * wave + lane];
        return sum;
    };
    if constexpr (USE == kSplitPart) {
        split_part(pr, add(), wave, r0, c0, at);
    } else if constexpr (USE == kSplitApply) {
        if (state != nullptr) lr = (float)state[3];
        const float keep = 1.0f - lr * wd, step = lr * pr.gain;
        const int x = c0 + l32, y = r0 + 8 * wave + 4 * lh;
        float* const theta = pr.theta;
        float* d = pr.out;
        if (theta != nullptr) d = theta;
        d += x;
        float w[4] = {0.f, 0.f, 0.f, 0.f};
        if (theta != nullptr && x < pr.cols)
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = d[(size_t)min(y + e, pr.rows - 1) * pr.cols];
        const f4 sum = add();
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float o = sum[e] * split_scale<USE>();
            if (x < pr.cols && y + e < pr.rows) d[(size_t)(y + e) * pr.cols] = theta != nullptr ? keep * w[e] - step * o : o;
        }
    } else {
        // each stores half of the block one way round
        const bool turned = wave >= 2;
        const SplitRows<USE> rows(pr, r0, c0, turned, wave & 1);
        const f4 sum = add();
        unsigned* t = reinterpret_cast<unsigned*>(lds + 4096);                       // (behind the first wave's sums)
#pragma unroll
        for (int e = 0; e < 4; ++e) t[(8 * wave + 4 * lh + e) * 33 + l32] = split_word<USE>(sum[e]);
        __syncthreads();
        if (USE != kSplitStep && r0 == c0 && turned) return;
        rows.template store<33>(pr, t, r0, c0, turned, wave & 1);
    }
}

// D1 = the sum of kSplitPart's runs: a 32 x 32 block a workgroup, every eighth run a wave, the waves' sums added in their order.
__global__ __launch_bounds__(512) void split_join(const SplitTable tb) {
    __shared__ f4 sums[8][4][64];
    __shared__ unsigned block[32 * 33];
    int t;
    const SplitProduct pr = split_find(tb, t);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int side = pr.M / 32, count = side * (side + 1) / 2;
    const float* p = pr.part + (size_t)t * 1024 + lane * 4;
    f4 sum[4] = {};
    const int runs = pr.runs;
#pragma unroll 4
    for (int k = wave; k < runs; k += 8)
#pragma unroll
        for (int q = 0; q < 4; ++q) sum[q] += *reinterpret_cast<const f4*>(p + (size_t)k * count * 1024 + 256 * q);
#pragma unroll
    for (int q = 0; q < 4; ++q) sums[wave][q][lane] = sum[q];
    __syncthreads();
    if (wave < 4) {
        f4 v = sums[0][wave][lane];
#pragma unroll
        for (int w = 1; w < 8; ++w) v += sums[w][wave][lane];
#pragma unroll
        for (int e = 0; e < 4; ++e) block[(8 * wave + 4 * (lane >> 5) + e) * 33 + (lane & 31)] = split_word<kSplitGram>(v[e]);
    }
    __syncthreads();
    int i, j;
    muon_triangle(t, &i, &j);
    i = __builtin_amdgcn_readfirstlane(i);
    j = __builtin_amdgcn_readfirstlane(j);
    const bool turned = wave >= 2;
    if (wave >= 4 || (turned && i == j)) return;
    SplitRows<kSplitGram>(pr, 32 * i, 32 * j, turned, wave & 1).store<33>(pr, block, 32 * i, 32 * j, turned, wave & 1);
}

}  // namespace aeth
