// muon.cu — matrices orthogonalised by Newton-Schulz products, and the momentum step with them.
//
//   X <- u / (|u| + eps), then `steps` times  A = X X^T,  P = b A + c A^2,  X <- a X + P X
//
// with X (m x n, m <= n) the matrix or its transpose: every singular value s goes through
// a s + b s^3 + c s^5, which pushes it towards 1 (and never above 1.203, from 1 or less).
//
// The products run on the tensor cores (tcgen05, f16 operands, f32 sums in tensor memory). X, A and P are
// bounded in that iteration (entries of at most 1.203, 1.447 and 2.807), so f16 at a fixed scale holds
// 11 bits of every entry down to 2^-29 of the largest: more than bf16 at the same rate. Types of 11 bits
// and more, and small matrices, take operands of 22 bits, as the sum of two f16 numbers, and three products (the
// fourth is below the sums' own rounding). Large bf16 matrices take products of 11 bits, but X keeps 22, for a X: what
// its rounding leaves where u has no singular values grows up to 485 times in five steps. (With X in 11 bits, bf16
// matrices of rank 1 to 64 came out 9.7e-2 to 1.7e-2 off, now 1.7e-3 to 2.4e-3, their own rounding 1.65e-3; full ones
// 1.87e-3, now 1.78e-3. The low parts cost 9 % of 4 matrices' time, 5 % of 8 large ones'.) An update far below
// epsilon makes a small X: see start_of.
//
// The diagonals of A and P, by far their largest entries, stay in f32 beside the operands, which hold zeros
// there: with A = D + O, A^2 = O^2 + D O + O D + D^2, and the last terms, like diag(P) X, are formed where
// sums are taken out. With the diagonals rounded to 11 bits too, results of bf16 matrices were 1.3e-3 to 5.8e-3
// off before their own rounding (a model of the roundings). Where all entries of A are alike, the rounding of
// 11-bit products has one direction and shows: 1024 equal rows 4.0e-3 off, matrices of one number up to 6.3e-3 (the
// model).
//
// Layout in the scratch: X, A and P in blocks of 128 rows x 64 columns, 16 KB each, row by row with their
// 16-byte pieces permuted as the tensor cores want them in shared memory. So every copy is one run of 8 or
// 16 KB that needs no tensor map, matrices of any size and address share a launch, and one block of X
// serves both as a piece of X's rows (A = X X^T) and of its columns (P X).
//
// A and P are symmetric: only tiles on and above the diagonal are computed, and their mirror images stored.
//
//   k_update_squares, k_spread   the momentum, the update's norm, X in blocks (HBM: 6.7 and 5.0 TB/s)
//   k_product                    one of the three products of a step, for a whole list
//   k_small                      small matrices, and rows and columns, from the update to the result
//
// Measured on a B200 (cuBLAS bf16 1637 TFLOP/s in bursts, 1370 sustained): products of 4096 x 4096 and 8192 x 2048
// bf16 matrices 1300, 1240 and 1170 TFLOP/s as issued, launches timed one by one (the last phase moves X's low parts
// beside them; 1370 without); the three products of a 4096 x 4096 f32 matrix 164 + 166 + 290 us; a step over 8 bf16
// matrices of 16M elements 8.3 ms, over 24 f32 ones of 1 to 4M 3.35 ms, over 5 of up to 80 x 64 33 us. In that first
// step the products run at some 1.01 PFLOP/s as issued, at 1365 MHz under the power limit (cuBLAS: 1.40 at 1335 MHz): a
// phase waits for its longest unit, and what else it waits for is not known. Middle sizes lose 20 us and more of a
// phase so (4 matrices of up to 4M in 0.76 ms at some 1800 MHz), small ones are bound by 15 rounds' latency.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <sstream>
#include <string>
#include <tuple>
#include <type_traits>

#include "elements.cuh"
#include "launch.h"
#include "muon.h"
#include "muon_plan.h"
#include "profile.h"
#include "tensor_core.cuh"

namespace arcqml {
namespace {

// Scales of the stored values: the largest powers of two that keep them in f16.
constexpr float kScaleX = 32768.0f; // of X and A; P has half of it
constexpr int kThreads = 256;
constexpr uint32_t kSumBlocks = 148 * 8; // partial sums of a matrix, at most
constexpr uint32_t kRows = 128, kDepth = 64;         // of a block
constexpr uint32_t kBlock = kRows * kDepth * 2;      // bytes
constexpr uint32_t kSMs = 148;
constexpr uint32_t kTakers = 8; // warps that take sums out: each has a quarter of the rows, half of the columns

// One matrix of a launch. The update u is the matrix `in`, or follows from the momentum and the gradient.
struct Matrix {
    void *out;       // the orthogonalised matrix, or the parameter
    const void *in;  // the matrix, or the gradient
    float *momentum; // null without a step
    uint64_t x[2], a, p; // offsets in the scratch; low parts lie behind their high parts
    uint64_t diagonal;   // of A, and behind it of P: f32, as large as the operands are stored
    uint32_t m, n;       // of X
    uint32_t down_blocks, x_blocks, a_blocks; // blocks of X down, and across X and A
    uint8_t flip, out_type, in_type, nesterov;
    float beta, keep; // of the step: momentum, and 1 - momentum
    float down, rate; // the parameter's factor, and the update's
};

struct Group {
    Matrix matrix[kMatrices];
    uint32_t first[kMatrices + 1]; // of the launch's blocks or tiles, by place
    uint8_t order[kMatrices];      // the matrix at each place
    uint32_t count;
    char *scratch;
    uint32_t *fault;   // set by a wait that ran out
    uint32_t *arrived; // parts of a tile that are done, for each warp of the units that begin one
    float *partial;
    double *inverse; // of each matrix: what X is times, stored as it is at first
    double *sums;
    double eps;
};

// The place of the matrix that has the launch's block or tile c.
__device__ __forceinline__ uint32_t place_with(const Group &g, uint32_t c) {
    uint32_t lo = 0, hi = g.count;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (g.first[mid] <= c) lo = mid;
        else hi = mid;
    }
    return lo;
}

// ------------------------------------------------------------------ elements of any type

template <class T> __device__ __forceinline__ void load8_as(float (&v)[8], const T *p, uint32_t count) {
    constexpr int N = 16 / sizeof(T);
    if (count >= 8 && reinterpret_cast<uintptr_t>(p) % 16 == 0) {
#pragma unroll
        for (int i = 0; i < 8; i += N) {
            const auto w = load_vector<T, N>(p + i);
#pragma unroll
            for (int e = 0; e < N; ++e) v[i + e] = to_wide(w.x[e]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = uint32_t(i) < count ? to_wide(p[i]) : 0.0f;
    }
}
// Up to 8 elements from place i on; zeros behind them.
__device__ __forceinline__ void load8(float (&v)[8], const void *p, uint32_t type, uint64_t i, uint32_t count) {
    if (type == ARCQML_F32) load8_as(v, static_cast<const float *>(p) + i, count);
    else if (type == ARCQML_BF16) load8_as(v, static_cast<const __nv_bfloat16 *>(p) + i, count);
    else load8_as(v, static_cast<const __half *>(p) + i, count);
}
template <class T> __device__ __forceinline__ void store8_as(const float (&v)[8], T *p, uint32_t count) {
    constexpr int N = 16 / sizeof(T);
    if (count >= 8 && reinterpret_cast<uintptr_t>(p) % 16 == 0) {
#pragma unroll
        for (int i = 0; i < 8; i += N) {
            VectorOf<T, N> w;
#pragma unroll
            for (int e = 0; e < N; ++e) w.x[e] = to_element<T>(v[i + e]);
            store_vector<T, N>(p + i, w);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (uint32_t(i) < count) p[i] = to_element<T>(v[i]);
    }
}
__device__ __forceinline__ void store1(void *p, uint32_t type, uint64_t i, float x) {
    if (type == ARCQML_F32) static_cast<float *>(p)[i] = x;
    else if (type == ARCQML_BF16) static_cast<__nv_bfloat16 *>(p)[i] = to_element<__nv_bfloat16>(x);
    else static_cast<__half *>(p)[i] = to_element<__half>(x);
}

// u of 8 elements, from the momentum as it is in memory.
__device__ __forceinline__ void update8(float (&u)[8], const Matrix &a, uint64_t i, uint32_t count) {
    if (!a.momentum) return load8(u, a.in, a.in_type, i, count);
    float m[8];
    load8_as(m, a.momentum + i, count);
    if (!a.nesterov) {
#pragma unroll
        for (int e = 0; e < 8; ++e) u[e] = m[e];
        return;
    }
    load8(u, a.in, a.in_type, i, count);
#pragma unroll
    for (int e = 0; e < 8; ++e) u[e] = a.beta * m[e] + a.keep * u[e];
}

// The momentum's update in memory, and u of 8 elements.
__device__ __forceinline__ void new_update8(float (&u)[8], const Matrix &a, uint64_t i, uint32_t count) {
    load8(u, a.in, a.in_type, i, count);
    if (!a.momentum) return;
    float m[8];
    load8_as(m, a.momentum + i, count);
#pragma unroll
    for (int e = 0; e < 8; ++e) m[e] = a.beta * m[e] + a.keep * u[e];
    store8_as(m, a.momentum + i, count);
#pragma unroll
    for (int e = 0; e < 8; ++e) u[e] = a.nesterov ? a.beta * m[e] + a.keep * u[e] : m[e];
}

// X is stored kScaleX / inverse times as large as it is. At first that is u times a power of two, with a norm of
// kScaleX / 2 to kScaleX: 16-bit numbers and their low parts are exact, and none of their roundings has one direction
// (u / |u| of 4 x 1000 bf16 numbers was rounded downwards throughout where |u| is just above a power of two, and 1e-3 off
// for that). X grows by at most 3.4445 a step, so 1 / inverse falls by 4 until it is 1.
struct Start {
    double factor, inverse; // X as stored is u factor
};
// Zeros stay zeros without an epsilon too, where X is 0 / 0; infinities become NaN.
__device__ __forceinline__ Start start_of(double norm, double whole) {
    if (!(norm > 0.0 && norm < INFINITY)) return {norm * 0.0, 1.0};
    const double factor = ldexp(double(kScaleX) / 2, -ilogb(norm));
    return {factor, double(kScaleX) / factor / whole};
}
__device__ __forceinline__ double inverse_at(double first, uint32_t step) {
    return step == 0 ? first : fmin(1.0, first * double(uint64_t(1) << 2 * step));
}
// What a phase's sums, and what they are added to, are times; and the result, as stored, of the last phase. Of P's
// diagonal d of A and the sum of products s make a + (b d + c (s + d^2)): it is formed in f64, since a is nearly lost
// in it (a 2 x 2 matrix of f32 was 1.8e-6 off with the f32 operations of the entries beside it).
struct Scales {
    float sum, old, result;
    double b, c;
    __device__ __forceinline__ float diagonal(float d, float s) const {
        return float(3.4445 + (b * double(d) + c * (double(s) + double(d) * double(d))));
    }
};
template <int PHASE> __device__ __forceinline__ Scales scales_of(double inverse) {
    const double square = inverse * inverse, next = fmin(1.0, 4.0 * inverse);
    const float ratio = float(next < 1.0 ? 0.25 : inverse); // of inverse and next
    if constexpr (PHASE == 0) return {1.0f / kScaleX, 0.0f, 0.0f, 0.0, 0.0};
    else if constexpr (PHASE == 1) {
        const double b = -4.7750 * square, c = 2.0315 * square * square / kScaleX;
        return {float(0.5 * c), float(0.5 * b), 0.0f, b / kScaleX, c / kScaleX};
    } else return {2.0f / kScaleX * ratio, ratio, float(next / kScaleX), 0.0, 0.0};
}

// ------------------------------------------------------------------ the update and its norm

// The sum over a block of kThreads, the same in every thread.
__device__ __forceinline__ double block_sum(double v) {
    __shared__ double part[kThreads / 32];
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.0;
    for (int w = 0; w < kThreads / 32; ++w) v += part[w];
    return v;
}

// The momentum's update, and the squares of u: an f64 sum for each block (201 us for 134M elements with bf16
// gradients, 1.3 GB).
__global__ void __launch_bounds__(kThreads) k_update_squares(const __grid_constant__ Group g) {
    cudaTriggerProgrammaticLaunchCompletion();
    if (blockIdx.x == 0) {
        if (threadIdx.x == 0) *g.fault = 0;
        for (uint32_t i = threadIdx.x; i < kSMs * kTakers * 2; i += kThreads) g.arrived[i] = 0;
    }
    const uint32_t k = place_with(g, blockIdx.x), blocks = g.first[k + 1] - g.first[k];
    const Matrix &a = g.matrix[k];
    const uint64_t n = uint64_t(a.m) * a.n;
    double sum = 0.0;
    for (uint64_t i = (uint64_t(blockIdx.x - g.first[k]) * kThreads + threadIdx.x) * 8; i < n;
         i += uint64_t(blocks) * kThreads * 8) {
        const uint32_t count = uint32_t(min(uint64_t(8), n - i));
        float u[8];
        new_update8(u, a, i, count);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = fma(double(u[e]), double(u[e]), sum);
    }
    sum = block_sum(sum);
    if (threadIdx.x == 0) g.sums[blockIdx.x] = sum;
}

// Where 8 neighbouring values of a row start in an array of blocks.
__device__ __forceinline__ uint64_t place_of(uint32_t row, uint32_t column, uint32_t blocks) {
    return (uint64_t(row / kRows) * blocks + column / kDepth) * kBlock + (row % kRows) * 128 +
           ((column % kDepth / 8) ^ (row % 8)) * 16;
}
__host__ __device__ inline uint64_t bytes_of(uint32_t down, uint32_t across) { return uint64_t(down) * across * kBlock; }

// How far behind 8 of X's high parts their low ones lie. Where products take them, both buffers have their own, laid
// out alike; else one set lies behind both buffers (who writes an entry's new low part is who has read the old one), in
// runs of 512 bytes for 32 rows, as warps take sums out: laid out alike they would cost as much again as the high parts
// (4 matrices 810 us instead of 755).
template <bool SPLIT>
__device__ __forceinline__ uint64_t low_of_x(uint64_t bytes, uint32_t buffer, uint32_t row, uint32_t column) {
    if constexpr (SPLIT) return bytes;
    const uint32_t piece = column % kDepth / 8;
    return bytes * (2 - buffer) + ((row % kRows / 32 * 8 + piece) * 512 + row % 32 * 16) -
           (row % kRows * 128 + (piece ^ row % 8) * 16);
}

// 8 values as f16, and with SPLIT what that leaves behind them.
template <bool SPLIT> __device__ __forceinline__ void store_operand(char *at, uint64_t low, const float (&v)[8]) {
    uint32_t h[4], l[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2 x = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
        h[i] = *reinterpret_cast<const uint32_t *>(&x);
        if constexpr (SPLIT) {
            const float2 y = __half22float2(x);
            const __half2 z = __floats2half2_rn(v[2 * i] - y.x, v[2 * i + 1] - y.y);
            l[i] = *reinterpret_cast<const uint32_t *>(&z);
        }
    }
    *reinterpret_cast<uint4 *>(at) = make_uint4(h[0], h[1], h[2], h[3]);
    if constexpr (SPLIT) *reinterpret_cast<uint4 *>(at + low) = make_uint4(l[0], l[1], l[2], l[3]);
}
template <bool SPLIT> struct OperandWords {
    uint4 high, low;
    __device__ __forceinline__ void load(const char *at, uint64_t apart) {
        high = *reinterpret_cast<const uint4 *>(at);
        if constexpr (SPLIT) low = *reinterpret_cast<const uint4 *>(at + apart);
    }
    __device__ __forceinline__ void unpack(float (&v)[8]) const {
        const uint32_t w[4] = {high.x, high.y, high.z, high.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 y = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
            v[2 * i] = y.x;
            v[2 * i + 1] = y.y;
        }
        if constexpr (SPLIT) {
            const uint32_t z[4] = {low.x, low.y, low.z, low.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 y = __half22float2(*reinterpret_cast<const __half2 *>(&z[i]));
                v[2 * i] += y.x;
                v[2 * i + 1] += y.y;
            }
        }
    }
};
template <bool SPLIT> __device__ __forceinline__ void load_operand(float (&v)[8], const char *at, uint64_t low) {
    OperandWords<SPLIT> w;
    w.load(at, low);
    w.unpack(v);
}

// X = u / (|u| + eps) in blocks, one for each thread block; zeros behind the matrix's edges. u is formed again
// from the momentum and the gradient: storing it between would move more (213 us for 134M elements, 1.1 GB).
template <bool SPLIT> __global__ void __launch_bounds__(kThreads) k_spread(const __grid_constant__ Group g,
                                                                           const __grid_constant__ Group sums) {
    __shared__ float turned[kDepth][kRows + 1];
    cudaTriggerProgrammaticLaunchCompletion();
    const uint32_t k = place_with(g, blockIdx.x), block = blockIdx.x - g.first[k];
    const Matrix &a = g.matrix[k];
    cudaGridDependencySynchronize();
    double sum = 0.0;
    for (uint32_t b = sums.first[k] + threadIdx.x; b < sums.first[k + 1]; b += kThreads) sum += g.sums[b];
    const double norm = sqrt(block_sum(sum)), whole = norm + g.eps;
    const Start start = start_of(norm, whole);
    if (block == 0 && threadIdx.x == 0) g.inverse[k] = start.inverse;
    const uint32_t row0 = block / a.x_blocks * kRows, column0 = block % a.x_blocks * kDepth;
    const uint64_t bytes = bytes_of(a.down_blocks, a.x_blocks);
    char *to = g.scratch + a.x[0];
    if (a.flip) { // X's rows are the matrix's columns
        for (uint32_t t = threadIdx.x; t < kDepth * (kRows / 8); t += kThreads) {
            const uint32_t c = t / (kRows / 8), r = t % (kRows / 8) * 8;
            float u[8];
            if (column0 + c < a.n && row0 + r < a.m)
                update8(u, a, uint64_t(column0 + c) * a.m + row0 + r, min(8u, a.m - row0 - r));
            else
#pragma unroll
                for (int e = 0; e < 8; ++e) u[e] = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) turned[c][r + e] = u[e];
        }
        __syncthreads();
    }
    for (uint32_t t = threadIdx.x; t < kRows * (kDepth / 8); t += kThreads) {
        const uint32_t r = t / (kDepth / 8), c = t % (kDepth / 8) * 8;
        float u[8];
        if (a.flip) {
#pragma unroll
            for (int e = 0; e < 8; ++e) u[e] = turned[c + e][r];
        } else if (row0 + r < a.m && column0 + c < a.n) {
            update8(u, a, uint64_t(row0 + r) * a.n + column0 + c, min(8u, a.n - column0 - c));
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) u[e] = 0.0f;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) // 0 behind the edges also where the factor is not finite
            u[e] = row0 + r < a.m && column0 + c + e < a.n ? float(double(u[e]) * start.factor) : 0.0f;
        store_operand<true>(to + place_of(row0 + r, column0 + c, a.x_blocks), low_of_x<SPLIT>(bytes, 0, r, c), u);
    }
}

// ------------------------------------------------------------------ products

enum Phase { GRAM, POLYNOMIAL, APPLY };
constexpr uint32_t kStageBytes = 32768; // one depth of 64: 128 rows of the left operand, 128 of the right
constexpr uint32_t kProductThreads = 128 + kTakers * 32;

// Stages of a block: 192 KB of operands. Behind them a square of 32 x 32 for each taker.
template <bool SPLIT> constexpr uint32_t kStages = SPLIT ? 3 : 6;
constexpr uint32_t kSquare = 32 * 33 * sizeof(float);
template <bool SPLIT> constexpr uint32_t kProductShared =
    1024 + kStages<SPLIT> * (SPLIT ? 2 : 1) * kStageBytes + 256 + kTakers * kSquare;
// The tensor cores cut what falls behind the last bit of a running sum (they do not round): a chain of k
// steps of 16 loses up to k 2^-24 of it, always towards 0. Operands of 22 bits would show that (a matrix of
// 4096 x 8191 came out 4.4e-5 off), so their sums leave tensor memory and go on in registers: every 128 of
// depth for A, whose diagonal adds up squares (every 512: 130 x 8000 4.9e-6 off instead of 1.0e-6, f32
// operations 1.3e-6; it takes 4 % of the whole), every 512 for sums of both signs. Steps of 64:
template <int PHASE, bool SPLIT> constexpr uint32_t kChain = !SPLIT ? 0xffffffffu : PHASE == 0 ? 2 : 8;

struct ProductState {
    uint64_t full[6], empty[6], peer[6], done[2], taken[2];
    uint32_t tmem, stop;
};
static_assert(sizeof(ProductState) <= 256, "the end of the shared memory");

// Waits for a barrier's phase; false once a wait of this block has run out. CG: 2 if the other block of a pair
// arrives there.
template <int CG> __device__ __forceinline__ bool wait_for(uint64_t *b, uint32_t parity, uint32_t *stop) {
    if (tc::barrier_try<CG>(b, parity)) return true;
    const long long begin = clock64();
    for (uint32_t i = 0; i < (1u << 30); ++i) { // ten seconds at most
        if (tc::barrier_try<CG>(b, parity)) return true;
        if (*reinterpret_cast<volatile uint32_t *>(stop)) return false;
        if (clock64() - begin > 20000000000ll) break;
    }
    *reinterpret_cast<volatile uint32_t *>(stop) = 1;
    return false;
}

// The tile t of a phase.
struct Tile {
    const Matrix *a;
    uint32_t index, i, j; // rows and columns in tiles
};
template <int PHASE, uint32_t SIZE> __device__ __forceinline__ Tile tile_of(const Group &g, uint32_t t) {
    Tile r;
    const uint32_t place = place_with(g, t);
    r.index = g.order[place];
    r.a = &g.matrix[r.index];
    t -= g.first[place];
    if constexpr (PHASE == APPLY) {
        const uint32_t across = (r.a->n + SIZE - 1) / SIZE;
        r.i = t / across;
        r.j = t % across;
    } else { // on and above the diagonal, row by row
        uint32_t side = (r.a->m + SIZE - 1) / SIZE;
        r.i = 0;
        while (t >= side) {
            t -= side;
            --side;
            ++r.i;
        }
        r.j = r.i + t;
    }
    return r;
}

// Up to N elements, `pitch` apart: the result as it is, or the step with it. All are loaded before the first
// is used.
template <class T, int N>
__device__ __forceinline__ void finish(T *at, uint64_t pitch, uint32_t count, const Matrix &a, float rate, const float (&v)[N]) {
    if (!a.momentum) {
#pragma unroll
        for (uint32_t q = 0; q < N; ++q)
            if (q < count) at[q * pitch] = to_element<T>(v[q] * rate);
        return;
    }
    T p[N];
#pragma unroll
    for (uint32_t q = 0; q < N; ++q) p[q] = at[min(q, count - 1) * pitch];
#pragma unroll
    for (uint32_t q = 0; q < N; ++q)
        if (q < count) at[q * pitch] = to_element<T>(fmaf(a.down, to_wide(p[q]), v[q] * rate));
}

// N neighbouring values of X's row for each thread of a warp, `times` what they are stored as, go out. Rows of the
// matrix are turned in shared memory (`square`), so that neighbouring lanes have neighbouring elements; X's rows are the
// columns of a flipped matrix and lie that way already.
template <int N>
__device__ __forceinline__ void give_result(const Matrix &a, float (&v)[N], uint32_t row, uint32_t column, float times,
                                            float *square) {
    constexpr uint32_t ROWS = 32 / N; // of the matrix side by side
    const float rate = a.momentum ? -a.rate * times : times;
    const uint32_t lane = threadIdx.x & 31;
    uint32_t along, mine, step; // v[q] belongs to place (along + q step, mine) of rows of `pitch`
    const uint32_t pitch = a.flip ? a.m : a.n, rows = a.flip ? a.n : a.m;
    if (a.flip) {
        along = column;
        mine = row;
        step = 1;
    } else {
        __syncwarp();
#pragma unroll
        for (uint32_t q = 0; q < N; ++q) square[lane * (N + 1) + q] = v[q];
        __syncwarp();
#pragma unroll
        for (uint32_t q = 0; q < N; ++q) v[q] = square[(q * ROWS + lane / N) * (N + 1) + lane % N];
        along = row - lane + lane / N;
        mine = column + lane % N;
        step = ROWS;
    }
    if (mine < pitch && along < rows) {
        const uint32_t count = (rows - along + step - 1) / step;
        const uint64_t at = uint64_t(along) * pitch + mine, apart = uint64_t(step) * pitch;
        if (a.out_type == ARCQML_F32) finish(static_cast<float *>(a.out) + at, apart, count, a, rate, v);
        else if (a.out_type == ARCQML_BF16) finish(static_cast<__nv_bfloat16 *>(a.out) + at, apart, count, a, rate, v);
        else finish(static_cast<__half *>(a.out) + at, apart, count, a, rate, v);
    }
    __syncwarp();
}

// An entry of P beside the diagonal from that of A (x), the sum of products beside the diagonals, and the diagonal's
// entries of its row and column.
__device__ __forceinline__ float combine(float x, float sum, float row, float column, float of_old, float of_sum) {
    return of_old * x + of_sum * (sum + (row + column) * x);
}

// 32 neighbouring sums of a row, for each thread of a warp, become what the phase stores.
template <int PHASE, bool SPLIT>
__device__ __forceinline__ void take_sums(const Group &g, const Matrix &a, float (&v)[32], uint32_t row, uint32_t column,
                                          bool mirrored, const Scales &scales, uint32_t current, bool last, float *square) {
    // rows and columns up to the end of their block: behind the matrix they are zero
    const uint32_t across = PHASE == APPLY ? a.x_blocks : a.a_blocks;
    if (row >= a.down_blocks * kRows || column >= across * kDepth) return; // the same for the whole warp
    const uint32_t lane = threadIdx.x & 31;
    const float of_sum = scales.sum, of_old = scales.old;
    const uint64_t bytes = bytes_of(a.down_blocks, across);
    const auto low = [&](uint32_t buffer, uint32_t at) {
        return PHASE == APPLY ? low_of_x<SPLIT>(bytes, buffer, row, at) : bytes;
    };
    const char *old = g.scratch + (PHASE == APPLY ? a.x[current] : a.a);
    char *to = g.scratch + (PHASE == APPLY ? a.x[current ^ 1] : PHASE == GRAM ? a.a : a.p);
    float *of_a = reinterpret_cast<float *>(g.scratch + a.diagonal), *of_p = of_a + a.down_blocks * kRows;
    const float mine = PHASE == GRAM ? 0.0f : PHASE == POLYNOMIAL ? of_a[row] : of_old * of_p[row];
    const uint32_t own = row - column; // the diagonal's place among the 32, if below that
    float on_diagonal = 0.0f;
    // what is read is read before the first store, which it might otherwise have to wait for: a round trip to L2
    // for 32 columns, or 16 where registers are short
    constexpr bool BOTH = SPLIT || PHASE == APPLY; // X keeps its low parts
    constexpr uint32_t BATCH = SPLIT ? 16 : 32;
#pragma unroll
    for (uint32_t q0 = 0; q0 < 32; q0 += BATCH) {
        OperandWords<BOTH> was[BATCH / 8];
        float4 other[BATCH / 4];
#pragma unroll
        for (uint32_t q = 0; q < BATCH; q += 8) {
            if constexpr (PHASE != GRAM) was[q / 8].load(old + place_of(row, column + q0 + q, across), low(current, column + q0 + q));
            if constexpr (PHASE == POLYNOMIAL) {
                other[q / 4] = *reinterpret_cast<const float4 *>(of_a + column + q0 + q);
                other[q / 4 + 1] = *reinterpret_cast<const float4 *>(of_a + column + q0 + q + 4);
            }
        }
#pragma unroll
        for (uint32_t i = 0; i < BATCH; i += 8) {
            const uint32_t q = q0 + i;
            float x[8];
            if constexpr (PHASE != GRAM) was[i / 8].unpack(x);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (PHASE == POLYNOMIAL && q + e == own) on_diagonal = v[q + e];
                if constexpr (PHASE == GRAM) v[q + e] *= of_sum;
                else if constexpr (PHASE == APPLY) v[q + e] = mine * x[e] + v[q + e] * of_sum;
                else
                    v[q + e] = combine(x[e], v[q + e], mine, reinterpret_cast<const float *>(other)[i + e], of_old, of_sum);
                if (PHASE != APPLY && q + e == own) {
                    if constexpr (PHASE == GRAM) of_a[row] = v[q + e];
                    v[q + e] = 0.0f;
                }
                x[e] = v[q + e];
            }
            if (PHASE != APPLY || !last) store_operand<BOTH>(to + place_of(row, column + q, across), low(current ^ 1, column + q), x);
        }
    }
    if (PHASE == POLYNOMIAL && own < 32) of_p[row] = scales.diagonal(mine, on_diagonal);
    if (PHASE != APPLY && mirrored) { // lanes in pairs, each with two rows of one column
#pragma unroll
        for (uint32_t q = 0; q < 32; q += 2) {
            const float other = __shfl_xor_sync(0xffffffffu, lane & 1 ? v[q] : v[q + 1], 1);
            const float one = lane & 1 ? other : v[q], two = lane & 1 ? v[q + 1] : other;
            const uint32_t r = column + q + (lane & 1), to_column = row & ~1u;
            const __half2 h = __floats2half2_rn(one, two);
            char *at = to + place_of(r, to_column, across) + to_column % 8 * 2;
            *reinterpret_cast<__half2 *>(at) = h;
            if constexpr (SPLIT) {
                const float2 y = __half22float2(h);
                *reinterpret_cast<__half2 *>(at + bytes) = __floats2half2_rn(one - y.x, two - y.y);
            }
        }
    }
    if (PHASE == APPLY && last) give_result(a, v, row, column, scales.result, square);
}

// One phase for all matrices of a group: D = L R^T in tiles of 128 CG x 128 CG, a pair of blocks a tile with
// CG = 2 (each has half of the tile's rows, and brings half of the right operand's). One thread copies operands
// in, 16 KB of each a stage; one issues the products; eight warps take finished sums out of one half of tensor
// memory while the next tile's go to the other. A step of 64 of the depth moves 32 KB into each block for 512
// (CG = 2) or 256 cycles of products: pairs come near the tensor cores' rate (0.45 us a step), single blocks are
// held by what shared memory takes in (0.32 us).
template <int PHASE, bool SPLIT, int CG>
__global__ void __launch_bounds__(kProductThreads, 1)
    k_product(const __grid_constant__ Group g, const __grid_constant__ TilePlan plan, uint32_t step, uint32_t last) {
    constexpr uint32_t SIZE = kRows * CG, S = kStages<SPLIT>, STAGE = kStageBytes * (SPLIT ? 2 : 1);
    extern __shared__ char raw[];
    char *shared = raw + (1024 - (tc::shared_address(raw) & 1023)) % 1024;
    ProductState &st = *reinterpret_cast<ProductState *>(shared + S * STAGE);
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32, current = step & 1;
    const uint32_t rank = CG == 2 ? tc::block_rank() : 0;
    if (warp == 0 && lane == 0) {
        for (uint32_t s = 0; s < S; ++s) {
            tc::barrier_init(&st.full[s], 1);
            tc::barrier_init(&st.empty[s], 1);
            tc::barrier_init(&st.peer[s], 1);
        }
        for (uint32_t s = 0; s < 2; ++s) {
            tc::barrier_init(&st.done[s], 1);
            tc::barrier_init(&st.taken[s], kTakers * CG);
        }
        st.stop = 0;
        tc::barrier_init_fence();
    }
    if (warp == 1) tc::tmem_alloc<CG>(&st.tmem, 2 * SIZE);
    tc::fence_before();
    __syncthreads();
    if constexpr (CG == 2) tc::cluster_sync();
    tc::fence_after();
    cudaTriggerProgrammaticLaunchCompletion();
    // The first tile is found, and its matrix's entries are read, before the last phase's results are waited
    // for: the launch's parameters come from L2 the first time, some 5000 cycles for all of them.
    const uint32_t tmem = st.tmem;
    const uint32_t units = gridDim.x / CG, unit = blockIdx.x / CG;
    Walk walk(plan, unit, units);
    Part part;
    bool more = walk.next(part);
    if (more) {
        const Matrix &a = *tile_of<PHASE, SIZE>(g, part.tile).a;
        asm volatile("" ::"l"(a.x[current]), "l"(a.x[current ^ 1]), "l"(a.a), "l"(a.p), "l"(a.diagonal), "l"(a.out), "r"(a.m),
                     "r"(a.n), "r"(a.down_blocks), "r"(a.x_blocks), "r"(a.a_blocks), "f"(a.rate), "l"(g.scratch), "l"(g.inverse),
                     "l"(g.fault), "l"(g.partial));
    }
    cudaGridDependencySynchronize();

    // the sums of a tile in registers take more of them than a thread's share: 384 x 168 registers as
    // 128 x 56 and 256 x 216
    if (warp < 4) {
        if constexpr (SPLIT) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        if (warp == 0 && lane == 0) { // copies operands in
            uint32_t at = 0, phase = 0;
            bool on = true;
            for (; on && more; more = walk.next(part)) {
                const Tile tile = tile_of<PHASE, SIZE>(g, part.tile);
                const Matrix &a = *tile.a;
                const uint32_t left = tile.i * CG + rank, right = tile.j * CG + rank;
                const uint32_t left_across = PHASE == GRAM ? a.x_blocks : a.a_blocks;
                const char *from = g.scratch + (PHASE == GRAM ? a.x[current] : PHASE == POLYNOMIAL ? a.a : a.p);
                const char *from_right = PHASE == APPLY ? g.scratch + a.x[current] : from;
                const uint64_t low = bytes_of(a.down_blocks, left_across);
                const uint64_t low_right = PHASE == APPLY ? bytes_of(a.down_blocks, a.x_blocks) : low;
                const uint32_t parts = SPLIT ? 2 : 1;
                // blocks behind the edges are not read: the sums that they would enter are not stored
                const bool has_left = left < a.down_blocks;
                const uint32_t wide = PHASE == APPLY ? min(2u, a.x_blocks - min(a.x_blocks, right * 2)) : 0;
                const bool has_right = right < a.down_blocks;
                const uint32_t bytes = parts * ((has_left ? kBlock : 0) + (PHASE == APPLY ? wide * (kBlock / 2) : has_right ? kBlock : 0));
                for (uint32_t d = part.begin; d < part.end; ++d) {
                    if (!(on = wait_for<CG>(&st.empty[at], phase ^ 1, &st.stop))) break;
                    char *to = shared + at * STAGE;
                    tc::barrier_expect(&st.full[at], bytes);
                    for (uint32_t part = 0; part < parts; ++part, to += kStageBytes) {
                        if (has_left)
                            tc::copy_in(to, from + part * low + (uint64_t(left) * left_across + d) * kBlock, kBlock, &st.full[at]);
                        if constexpr (PHASE == APPLY) {
                            for (uint32_t w = 0; w < wide; ++w)
                                tc::copy_in(to + kBlock + w * (kBlock / 2),
                                            from_right + part * low_right +
                                                (uint64_t(d / 2) * a.x_blocks + right * 2 + w) * kBlock + (d & 1) * (kBlock / 2),
                                            kBlock / 2, &st.full[at]);
                        } else if (has_right) {
                            tc::copy_in(to + kBlock, from_right + part * low_right + (uint64_t(right) * left_across + d) * kBlock,
                                        kBlock, &st.full[at]);
                        }
                    }
                    if (++at == S) at = 0, phase ^= 1;
                }
            }
            // nothing may still be on its way in when the block ends: neither the tensor cores' word that a stage has
            // been read, nor (after a wait that ran out) copies
            uint32_t none = 0;
            for (uint32_t s = 0; s < S; ++s) {
                if (on) wait_for<CG>(&st.empty[s], s < at ? phase : phase ^ 1, &st.stop);
                else wait_for<1>(&st.full[s], s < at ? phase : phase ^ 1, &none);
            }
        } else if (warp == 1 && rank == 0 && lane == 0) { // issues the products
            constexpr uint32_t instr = tc::instruction(SIZE, SIZE, PHASE == APPLY);
            constexpr uint32_t STEP = PHASE == APPLY ? 2048 / 16 : 32 / 16; // of the right operand, 16 of depth
            uint32_t at = 0, phase = 0, n = 0;
            bool on = true;
            for (; on && more; more = walk.next(part)) {
                for (uint32_t d = part.begin; d < part.end && on; ++n) {
                    const uint32_t half = n & 1, end = min(part.end - d, kChain<PHASE, SPLIT>) + d;
                    if (!(on = wait_for<CG>(&st.taken[half], (n >> 1 & 1) ^ 1, &st.stop))) break;
                    tc::fence_after();
                    const uint32_t sums = tmem + half * SIZE;
                    for (bool add = false; d < end; ++d) {
                        if (!(on = wait_for<1>(&st.full[at], phase, &st.stop))) break;
                        if constexpr (CG == 2)
                            if (!(on = wait_for<CG>(&st.peer[at], phase, &st.stop))) break;
                        tc::fence_after();
                        const uint32_t base = tc::shared_address(shared + at * STAGE);
                        const uint64_t left = tc::descriptor(base, 16);
                        const uint64_t right = tc::descriptor(base + kBlock, PHASE == APPLY ? kBlock / 2 : 16);
#pragma unroll
                        for (uint32_t s = 0; s < kDepth / 16; ++s) {
                            tc::mma<CG>(sums, left + s * 2, right + s * STEP, instr, add);
                            add = true;
                            if constexpr (SPLIT) {
                                constexpr uint32_t LOW = kStageBytes / 16;
                                tc::mma<CG>(sums, left + s * 2, right + LOW + s * STEP, instr, true);
                                tc::mma<CG>(sums, left + LOW + s * 2, right + s * STEP, instr, true);
                            }
                        }
                        tc::commit<CG>(&st.empty[at]);
                        if (++at == S) at = 0, phase ^= 1;
                    }
                    if (on) tc::commit<CG>(&st.done[half]);
                }
            }
        } else if (CG == 2 && warp == 2 && rank == 1 && lane == 0) { // tells the first block of its operands
            uint32_t at = 0, phase = 0;
            bool on = true;
            for (; on && more; more = walk.next(part)) {
                for (uint32_t d = part.begin; d < part.end; ++d) {
                    if (!(on = wait_for<1>(&st.full[at], phase, &st.stop))) break;
                    tc::barrier_arrive_at<CG>(tc::in_block(&st.peer[at], 0));
                    if (++at == S) at = 0, phase ^= 1;
                }
            }
        }
    } else {
        if constexpr (SPLIT) asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        // takes the sums out: a thread has a row
        Walk tiles(plan, unit, units);
        constexpr uint32_t COLUMNS = SIZE / 2;
        const uint32_t quarter = warp & 3, first = (warp - 4) / 4 * COLUMNS;
        float *square = reinterpret_cast<float *>(reinterpret_cast<char *>(&st) + 256) + (warp - 4) * (kSquare / 4);
        uint32_t n = 0;
        bool on = true;
        const auto release = [&](uint32_t half) {
            tc::fence_before();
            __syncwarp();
            if (lane == 0)
                tc::barrier_arrive_at<CG>(CG == 2 ? tc::in_block(&st.taken[half], 0) : tc::shared_address(&st.taken[half]));
        };
        const auto wait_done = [&](uint32_t half) {
            on = __all_sync(0xffffffffu, wait_for<CG>(&st.done[half], n >> 1 & 1, &st.stop));
            tc::fence_after();
            return on;
        };
        const uint32_t from = cut(plan, unit), writer = rank * kTakers + warp - 4;
        const auto slice = [&](uint32_t u, uint32_t slot) { // of a unit's parts: 0 of a tile that began earlier
            return reinterpret_cast<float4 *>(g.partial) + ((uint64_t(u) * 2 + slot) * (kTakers * CG) + writer) * (COLUMNS * 8) + lane;
        };
        while (on && tiles.next(part)) {
            const Tile tile = tile_of<PHASE, SIZE>(g, part.tile);
            const Matrix &a = *tile.a;
            const uint32_t row = tile.i * SIZE + rank * kRows + quarter * 32 + lane;
            const uint32_t lanes = quarter * 32 << 16;
            const Scales scales = scales_of<PHASE>(inverse_at(g.inverse[tile.index], step));
            const auto take = [&](float (&v)[32], uint32_t c) {
                take_sums<PHASE, SPLIT>(g, a, v, row, tile.j * SIZE + first + c, tile.i != tile.j, scales, current, last != 0,
                                        square);
            };
            const bool whole = part.whole();
            uint32_t u0 = 0, parts = 1; // the unit with the tile's first step, and how many have parts of it
            if (!whole) sharers(plan, part, u0, parts);
            float4 *mine = whole ? nullptr : slice(unit, slot_of(part, from));
            if constexpr (SPLIT) {
                float sum[COLUMNS];
#pragma unroll
                for (uint32_t c = 0; c < COLUMNS; ++c) sum[c] = 0.0f;
#pragma unroll 1
                for (uint32_t d = part.begin; d < part.end; d += kChain<PHASE, SPLIT>, ++n) {
                    const uint32_t half = n & 1;
                    if (!wait_done(half)) break;
#pragma unroll
                    for (uint32_t c = 0; c < COLUMNS; c += 16) tc::tmem_add(sum + c, tmem + half * SIZE + lanes + first + c);
                    release(half);
                }
                if (!on) break;
                if (whole) {
#pragma unroll
                    for (uint32_t c = 0; c < COLUMNS; c += 32) {
                        float v[32];
#pragma unroll
                        for (uint32_t e = 0; e < 32; ++e) v[e] = sum[c + e];
                        take(v, c);
                    }
                    continue;
                }
#pragma unroll
                for (uint32_t c = 0; c < COLUMNS; c += 4) mine[c * 8] = make_float4(sum[c], sum[c + 1], sum[c + 2], sum[c + 3]);
            } else {
                const uint32_t half = n & 1;
                if (!wait_done(half)) break;
#pragma unroll 1
                for (uint32_t c = 0; c < COLUMNS; c += 32) {
                    float v[32];
                    __syncwarp();
                    tc::tmem_load(v, tmem + half * SIZE + lanes + first + c);
                    if (whole) {
                        take(v, c);
                    } else {
#pragma unroll
                        for (uint32_t e = 0; e < 32; e += 4)
                            mine[(c + e) * 8] = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
                    }
                }
                release(half);
                ++n;
                if (whole) continue;
            }
            // a part: the warp that brings its rows and columns' last one puts them together
            __threadfence();
            __syncwarp();
            uint32_t before = 0;
            if (lane == 0) before = atomicAdd(&g.arrived[u0 * (kTakers * 2) + writer], 1u);
            if (__shfl_sync(0xffffffffu, before, 0) + 1 != parts) continue;
            if (lane == 0) g.arrived[u0 * (kTakers * 2) + writer] = 0;
            __threadfence();
#pragma unroll 1
            for (uint32_t c = 0; c < COLUMNS; c += 32) {
                float v[32];
#pragma unroll
                for (uint32_t e = 0; e < 32; ++e) v[e] = 0.0f;
#pragma unroll 2
                for (uint32_t u = 0; u < parts; ++u) {
                    const float4 *from = slice(u0 + u, u ? 0 : 1) + c * 8;
                    float4 w[8];
#pragma unroll
                    for (uint32_t e = 0; e < 8; ++e) w[e] = __ldcg(from + e * 32);
#pragma unroll
                    for (uint32_t e = 0; e < 8; ++e) {
                        v[4 * e] += w[e].x;
                        v[4 * e + 1] += w[e].y;
                        v[4 * e + 2] += w[e].z;
                        v[4 * e + 3] += w[e].w;
                    }
                }
                take(v, c);
            }
        }
    }
    __syncwarp();
    tc::fence_before();
    __syncthreads();
    if constexpr (CG == 2) tc::cluster_sync();
    tc::fence_after();
    if (threadIdx.x == 0 && st.stop) *g.fault = 1;
    if (warp == 1) tc::tmem_free<CG>(tmem, 2 * SIZE);
}

// A wait that ran out left the products unfinished: everything that the call was to write is NaN.
__global__ void __launch_bounds__(kThreads) k_check_fault(const __grid_constant__ Group g) {
    cudaGridDependencySynchronize();
    if (!*g.fault) return;
    for (uint32_t k = 0; k < g.count; ++k) {
        const Matrix &a = g.matrix[k];
        const uint64_t n = uint64_t(a.m) * a.n;
        for (uint64_t i = uint64_t(blockIdx.x) * kThreads + threadIdx.x; i < n; i += uint64_t(gridDim.x) * kThreads)
            store1(a.out, a.out_type, i, __int_as_float(0x7fffffff));
    }
}

// ------------------------------------------------------------------ small matrices

// A matrix of at most 128 rows of X whose 22-bit operands fit into a block's shared memory is orthogonalised by
// that block from its update to its result: one launch for a list, 15 rounds of some 2900 cycles each.
constexpr uint32_t kSmallThreads = 256;
static_assert(kSmallThreads == 2 * kRows, "a thread for each diagonal entry of A and P");
constexpr uint32_t kSmallBlocks = 4; // of X: 256 columns
constexpr uint32_t kSmallShared =
    1024 + (kSmallBlocks + 2) * 2 * kBlock + 256 + kSmallThreads / 32 * 32 * 17 * sizeof(float) + 2 * kRows * sizeof(float);

struct SmallState {
    uint64_t done;
    uint32_t tmem, stop;
};

__device__ __forceinline__ void shared_writes_to_tensor_cores() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// A row or column: A is one number, s^2, and s becomes s (a + b s^2 + c s^4). So the result is u times one number,
// formed in f64, and as exact as its rounding. (With 22-bit operands rows came out up to 1.5e-6 off, f32 operations
// up to 6e-7.) One block goes through it at 8 elements a thread: 14 us a call up to 8191 elements, 0.36 ms for 2^20
// (as tiles of 128 rows 247 us and 13 ms), bound by what one SM has in flight.
__device__ __forceinline__ void take_row(const Matrix &a, double eps, int steps) {
    const uint32_t all = a.m * a.n;
    double sum = 0.0;
    for (uint32_t i = threadIdx.x * 8; i < all; i += kSmallThreads * 8) {
        float u[8];
        new_update8(u, a, i, min(8u, all - i));
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = fma(double(u[e]), double(u[e]), sum);
    }
    const double norm = sqrt(block_sum(sum)), whole = norm + eps;
    double times = whole == 0.0 ? 0.0 : 1.0 / whole, square = norm * times * (norm * times);
    for (int step = 0; step < steps; ++step) {
        const double f = 3.4445 + square * (-4.7750 + 2.0315 * square);
        times *= f;
        square *= f * f;
    }
    for (uint32_t i = threadIdx.x * 8; i < all; i += kSmallThreads * 8) {
        const uint32_t count = min(8u, all - i);
        float u[8], p[8];
        update8(u, a, i, count);
        if (a.momentum) load8(p, a.out, a.out_type, i, count);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            u[e] = float(double(u[e]) * times);
            if (a.momentum) u[e] = fmaf(a.down, p[e], u[e] * -a.rate);
        }
        if (a.out_type == ARCQML_F32) store8_as(u, static_cast<float *>(a.out) + i, count);
        else if (a.out_type == ARCQML_BF16) store8_as(u, static_cast<__nv_bfloat16 *>(a.out) + i, count);
        else store8_as(u, static_cast<__half *>(a.out) + i, count);
    }
}

__global__ void __launch_bounds__(kSmallThreads, 1) k_small(const __grid_constant__ Group g, int steps) {
    constexpr uint32_t LOW = kSmallBlocks * kBlock; // X's low parts behind its high ones
    extern __shared__ char raw[];
    char *x = raw + (1024 - (tc::shared_address(raw) & 1023)) % 1024;
    char *p = x + LOW * 2; // A, then P; low parts 2 blocks behind
    SmallState &st = *reinterpret_cast<SmallState *>(p + 2 * kBlock * 2);
    const Matrix &a = g.matrix[blockIdx.x];
    if (a.m == 1) return take_row(a, g.eps, steps);
    const uint32_t thread = threadIdx.x, warp = thread / 32, lane = thread % 32;
    float *square = reinterpret_cast<float *>(reinterpret_cast<char *>(&st) + 256) + warp * 32 * 17;
    float *of_a = reinterpret_cast<float *>(reinterpret_cast<char *>(&st) + 256) + kSmallThreads / 32 * 32 * 17, *of_p = of_a + kRows;
    of_a[thread] = 0.0f; // both: rows behind the matrix keep it
    if (thread == 0) {
        tc::barrier_init(&st.done, 1);
        st.stop = 0;
        tc::barrier_init_fence();
    }
    if (warp == 1) tc::tmem_alloc<1>(&st.tmem, 512);
    tc::fence_before();

    // the update, its norm, and X
    const uint32_t all = a.m * a.n;
    double sum = 0.0;
    for (uint32_t i = thread * 8; i < all; i += kSmallThreads * 8) {
        const uint32_t count = min(8u, all - i);
        float u[8];
        new_update8(u, a, i, count);
        if (a.momentum) // the parameter, which the last step will want
            asm volatile("prefetch.global.L2 [%0];" ::"l"(static_cast<const char *>(a.out) + uint64_t(i) * (a.out_type == ARCQML_F32 ? 4 : 2)));
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = fma(double(u[e]), double(u[e]), sum);
    }
    const uint32_t m16 = (a.m + 15) / 16 * 16, n16 = (a.n + 15) / 16 * 16, used = (a.n + kDepth - 1) / kDepth * kBlock;
    for (uint32_t i = thread * 16; i < used; i += kSmallThreads * 16) {
        *reinterpret_cast<uint4 *>(x + i) = make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint4 *>(x + LOW + i) = make_uint4(0, 0, 0, 0);
    }
    const double norm = sqrt(block_sum(sum)), whole = norm + g.eps; // (and a barrier)
    const Start start = start_of(norm, whole);
    const uint32_t pitch = a.flip ? a.m : a.n;
    for (uint32_t i = thread * 8; i < all; i += kSmallThreads * 8) {
        const uint32_t count = min(8u, all - i);
        float u[8];
        update8(u, a, i, count);
        uint32_t r = i / pitch, c = i % pitch;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (uint32_t(e) < count) {
                const uint32_t row = a.flip ? c : r, column = a.flip ? r : c;
                char *at = x + place_of(row, column, kSmallBlocks) + column % 8 * 2;
                const float v = float(double(u[e]) * start.factor);
                const __half h = __float2half_rn(v);
                *reinterpret_cast<__half *>(at) = h;
                *reinterpret_cast<__half *>(at + LOW) = __float2half_rn(v - __half2float(h));
            }
            if (++c == pitch) c = 0, ++r;
        }
    }
    shared_writes_to_tensor_cores();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = st.tmem, mine = tmem + ((warp & 3) * 32 << 16), row = (warp & 3) * 32 + lane;
    const uint32_t x_at = tc::shared_address(x), p_at = tc::shared_address(p);
    uint32_t parity = 0;
    bool broken = false;
    // steps of 16 of the depth; operands by depth, or the right one by width. Products with low parts have sums
    // of their own: a long chain of additions to the high parts' would cost as much again (see kChain)
    constexpr uint32_t CROSS = 256;
    const auto multiply = [&](uint32_t sums, uint32_t left, uint32_t left_low, uint32_t right, uint32_t right_low,
                              uint32_t depth, uint32_t columns, bool by_width) {
        const uint32_t instr = tc::instruction(128, columns, by_width);
        for (uint32_t k = 0; k < depth / 16; ++k) {
            const uint32_t by_depth = k / 4 * kBlock + k % 4 * 32, along = by_width ? k * 2048 : by_depth;
            const uint32_t apart = by_width ? kBlock : 16;
            tc::mma<1>(sums, tc::descriptor(left + by_depth, 16), tc::descriptor(right + along, apart), instr, k != 0);
            tc::mma<1>(sums + CROSS, tc::descriptor(left + by_depth, 16), tc::descriptor(right_low + along, apart), instr, k != 0);
            tc::mma<1>(sums + CROSS, tc::descriptor(left_low + by_depth, 16), tc::descriptor(right + along, apart), instr, true);
        }
    };
    const auto sums_ready = [&] {
        const bool ok = wait_for<1>(&st.done, parity, &st.stop);
        parity ^= 1;
        broken = __syncthreads_or(!ok);
        tc::fence_after();
        return !broken;
    };
    const auto operands_ready = [&] {
        shared_writes_to_tensor_cores();
        tc::fence_before();
        __syncthreads();
        tc::fence_after();
    };
    int step = 0;
    const auto run_phase = [&](auto which) {
        constexpr int PHASE = which;
        const uint32_t columns = PHASE == APPLY ? n16 : m16;
        if (thread == 0) {
            if (PHASE == GRAM) multiply(tmem, x_at, x_at + LOW, x_at, x_at + LOW, n16, m16, false);
            else if (PHASE == POLYNOMIAL) multiply(tmem, p_at, p_at + 2 * kBlock, p_at, p_at + 2 * kBlock, m16, m16, false);
            else multiply(tmem, p_at, p_at + 2 * kBlock, x_at, x_at + LOW, m16, n16, true);
            tc::commit<1>(&st.done);
        }
        const Scales scales = scales_of<PHASE>(inverse_at(start.inverse, step));
        const float of_sum = scales.sum, of_old = scales.old;
        const float diagonal = PHASE == GRAM ? 0.0f : PHASE == POLYNOMIAL ? of_a[row] : of_old * of_p[row];
        char *to = PHASE == APPLY ? x : p;
        constexpr uint64_t low = PHASE == APPLY ? LOW : 2 * kBlock;
        constexpr uint32_t across = PHASE == APPLY ? kSmallBlocks : 2;
        if (!sums_ready()) return;
#pragma unroll 1
        for (uint32_t c = warp / 4 * 16; c < columns; c += 32) {
            float v[16];
            tc::tmem_load2(v, mine + c, mine + CROSS + c);
            const uint32_t own = row - c;
            float on_diagonal = 0.0f;
#pragma unroll
            for (uint32_t q = 0; q < 16; q += 8) {
                char *at = to + place_of(row, c + q, across);
                float y[8];
                if constexpr (PHASE != GRAM) load_operand<true>(y, at, low);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    float &z = v[q + e];
                    if (PHASE == POLYNOMIAL && q + e == own) on_diagonal = z;
                    if constexpr (PHASE == GRAM) z *= of_sum;
                    else if constexpr (PHASE == APPLY) z = diagonal * y[e] + z * of_sum;
                    else z = combine(y[e], z, diagonal, of_a[c + q + e], of_old, of_sum);
                    if (PHASE != APPLY && q + e == own) {
                        if constexpr (PHASE == GRAM) of_a[row] = z;
                        z = 0.0f;
                    }
                    y[e] = z;
                }
                store_operand<true>(at, low, y);
            }
            if (PHASE == POLYNOMIAL && own < 16) of_p[row] = scales.diagonal(diagonal, on_diagonal);
            if (PHASE == APPLY && step + 1 == steps) give_result(a, v, row, c, scales.result, square);
        }
        operands_ready();
    };
    for (; step < steps && !broken; ++step) {
        run_phase(std::integral_constant<int, GRAM>{});
        if (!broken) run_phase(std::integral_constant<int, POLYNOMIAL>{});
        if (!broken) run_phase(std::integral_constant<int, APPLY>{});
    }
    if (broken)
        for (uint32_t i = thread; i < all; i += kSmallThreads) store1(a.out, a.out_type, i, __int_as_float(0x7fffffff));
    __syncthreads();
    if (warp == 1) tc::tmem_free<1>(tmem, 512);
}

// ------------------------------------------------------------------ host

[[noreturn]] void refuse(const char *list, size_t i, const char *why) {
    std::ostringstream m;
    m << list << " matrix " << i << " " << why;
    fail(m.str());
}

bool present(const ArcqmlMatrix &a) { return a.dtype != ARCQML_NO_TENSOR && a.rows && a.columns; }

void check_list(const ArcqmlMatrix *list, size_t count, const char *name) {
    if (count && !list) fail(std::string(name) + " list is null");
    for (size_t i = 0; i < count; ++i) {
        const ArcqmlMatrix &a = list[i];
        if (a.dtype == ARCQML_F64) refuse(name, i, "is f64: matrices are f32, bf16 or f16");
        if (a.dtype > ARCQML_NO_TENSOR) refuse(name, i, "has an unknown type");
        if (a.reserved != 0) refuse(name, i, "has a nonzero reserved field");
        if (!present(a)) continue;
        if (a.rows >> 24 || a.columns >> 24 || (a.rows * a.columns) >> 36 || std::min(a.rows, a.columns) >> 17)
            refuse(name, i, "is too large");
        if (!a.data) refuse(name, i, "is null");
        if (reinterpret_cast<uintptr_t>(a.data) % bytes_of_element(a.dtype)) refuse(name, i, "is not aligned to its elements");
    }
}

void check_scratch(const double *ws, size_t len, size_t need) {
    if (!need) return;
    if (!ws) fail("workspace is null");
    if (reinterpret_cast<uintptr_t>(ws) % 16) fail("workspace is not aligned to 16 bytes");
    if (len < need) {
        std::ostringstream m;
        m << "workspace of " << len << " doubles is too small: the list needs " << need;
        fail(m.str());
    }
}

template <class... P, class... A>
void start(void (*kernel)(P...), uint32_t blocks, uint32_t threads, uint32_t cluster, uint32_t shared, bool follows,
           double bytes, cudaStream_t s, const A &...args) {
    cudaLaunchConfig_t c{};
    cudaLaunchAttribute at[2]{};
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = follows;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = cluster;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    c.gridDim = dim3(blocks);
    c.blockDim = dim3(threads);
    c.dynamicSmemBytes = shared;
    c.stream = s;
    c.attrs = at;
    c.numAttrs = cluster > 1 ? 2 : 1;
    std::tuple<P...> held{P(args)...};
    const ProfToken tok = prof_begin(PROF_OTHER, s);
    const cudaError_t e = std::apply([&](auto &...x) { return cudaLaunchKernelEx(&c, kernel, x...); }, held);
    check_cuda(e, "orthogonalisation kernel launch");
    prof_end(tok, s, bytes);
}

// Types of 11 bits and more take operands of 22 bits; so do bf16 matrices of up to 128 rows (of X), whose few singular
// values do not even out what 11 bits do to one of them (and whose products are short).
bool is_split(const ArcqmlMatrix &a, uint32_t type) { return type != ARCQML_BF16 || std::min(a.rows, a.columns) <= kRows; }

// The scratch: the fault, the scales, the parts that arrived, sums of squares, parts of tiles, then operands.
constexpr size_t kScalesAt = 256, kArrivedAt = kScalesAt + kMatrices * sizeof(double), kSumsAt = kArrivedAt + kSMs * kTakers * 2 * sizeof(uint32_t);
constexpr size_t kPartialAt = (kSumsAt + size_t(kMatrices) * kSumBlocks * sizeof(double) + 1023) / 1024 * 1024;
// two tiles for each pair of blocks (single blocks: half as much)
constexpr size_t kOperandsAt = kPartialAt + size_t(kSMs / 2) * 2 * (2 * kRows) * (2 * kRows) * sizeof(float);

// Matrices that one block takes whole; rows and columns of any length.
bool is_small(const ArcqmlMatrix &a) {
    const uint64_t m = std::min(a.rows, a.columns), n = std::max(a.rows, a.columns);
    return m == 1 || (m <= kRows && n <= kSmallBlocks * kDepth);
}

// Scratch bytes of a matrix's X (twice), A, P and their diagonals.
uint64_t operand_bytes(const ArcqmlMatrix &a, bool split) {
    const uint64_t m = std::min(a.rows, a.columns), n = std::max(a.rows, a.columns);
    const uint32_t down = uint32_t((m + kRows - 1) / kRows), across = 2 * uint32_t((n + kRows - 1) / kRows);
    return bytes_of(down, across) * (split ? 4 : 3) + bytes_of(down, 2 * down) * (split ? 4 : 2) + uint64_t(down) * kRows * 8;
}

// The scratch of a launch's matrices: what one needs, and more of them while that stays below 2 GB.
constexpr uint64_t kGroupBytes = uint64_t(2) << 30;

// The places of a launch's matrices (of a fixed size: the workspace query allocates nothing, so it cannot throw).
struct Members {
    size_t at[kMatrices];
    uint32_t count = 0;
};

template <class F>
void for_groups(const ArcqmlMatrix *list, const ArcqmlMatrix *kinds, size_t count, uint64_t most, F &&f) {
    Members members;
    for (int kind = 0; kind < 3; ++kind) {
        const bool split = kind == 1, small = kind == 2;
        uint64_t bytes = 0;
        const auto flush = [&] {
            if (members.count) f(members, bytes, split, small);
            members.count = 0;
            bytes = 0;
        };
        for (size_t i = 0; i < count; ++i) {
            if (!present(list[i]) || is_small(list[i]) != small || (!small && is_split(list[i], kinds[i].dtype) != split)) continue;
            const uint64_t need = small ? 0 : operand_bytes(list[i], split);
            if (members.count == kMatrices || (bytes && bytes + need > most)) flush();
            members.at[members.count++] = i;
            bytes += need;
        }
        flush();
    }
}

// Lets a kernel have `bytes` of shared memory, once on each device.
template <auto KERNEL> void allow_shared(uint32_t bytes) {
    static std::atomic<uint64_t> set{0};
    int device = 0;
    check_cuda(cudaGetDevice(&device), "cudaGetDevice");
    if (device < 64 && (set.load() >> device & 1)) return;
    check_cuda(cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes)),
               "orthogonalisation kernel attribute");
    if (device < 64) set |= uint64_t(1) << device;
}

template <int PHASE> uint32_t tiles_of(const Matrix &a, uint32_t size) {
    const uint32_t down = (a.m + size - 1) / size, across = (a.n + size - 1) / size;
    return PHASE == APPLY ? down * across : down * (down + 1) / 2;
}
template <int PHASE> uint32_t depth_of(const Matrix &a) { return ((PHASE == GRAM ? a.n : a.m) + kDepth - 1) / kDepth; }

// Who does which tile of 128 CG x 128 CG, and how many steps of 64 of the depth the longest unit has. g's
// matrices are put in order.
template <int PHASE> uint32_t make_plan(Group &g, TilePlan &p, uint32_t cg, bool split) {
    std::stable_sort(g.order, g.order + g.count, [&](uint8_t x, uint8_t y) {
        return depth_of<PHASE>(g.matrix[x]) > depth_of<PHASE>(g.matrix[y]);
    });
    uint32_t tiles = 0;
    for (uint32_t i = 0; i < g.count; ++i) {
        g.first[i] = tiles;
        tiles += tiles_of<PHASE>(g.matrix[g.order[i]], cg * kRows);
    }
    g.first[g.count] = tiles;
    const uint32_t units = kSMs / cg;
    uint32_t whole = 0;
    p.classes = p.left[0] = 0;
    for (uint32_t i = 0, next; i < g.count; i = next) {
        const uint32_t c = p.classes++, depth = depth_of<PHASE>(g.matrix[g.order[i]]);
        for (next = i; next < g.count && depth_of<PHASE>(g.matrix[g.order[next]]) == depth;) ++next;
        const uint32_t has = g.first[next] - g.first[i];
        p.tile[c] = g.first[i];
        p.depth[c] = depth;
        p.rounds[c] = has / units;
        p.left[c + 1] = p.left[c] + has % units * weight(depth);
        whole += p.rounds[c] * weight(depth);
    }
    return whole + share_out(p, units, split);
}

template <int PHASE, bool SPLIT, int CG> void product(const Group &g, const TilePlan &p, uint32_t step, bool last, cudaStream_t s) {
    allow_shared<k_product<PHASE, SPLIT, CG>>(kProductShared<SPLIT>);
    start(k_product<PHASE, SPLIT, CG>, kSMs, kProductThreads, CG, kProductShared<SPLIT>, true, 0.0, s, g, p, step, uint32_t(last));
}

template <int PHASE, bool SPLIT> void phase(Group &g, uint32_t step, bool last, cudaStream_t s) {
    // A pair's step is four times the work of a single block's and takes 1.4 times as long (11-bit operands 0.45
    // and 0.32 us, 22-bit ones 0.85 and 0.62): pairs for many tiles (4096 x 4096: 107 and 179 us for the last
    // phase), single blocks where whole tiles of pairs are too few (the second phase of 2048 x 2048 has 36 for
    // 74 pairs: 25.6 and 20.5 us).
    TilePlan pairs, singles;
    const uint32_t single = make_plan<PHASE>(g, singles, 1, SPLIT), pair = make_plan<PHASE>(g, pairs, 2, SPLIT);
    if (7 * pair <= 5 * single) return product<PHASE, SPLIT, 2>(g, pairs, step, last, s);
    make_plan<PHASE>(g, singles, 1, SPLIT);
    product<PHASE, SPLIT, 1>(g, singles, step, last, s);
}

// The members' `out`, `in` and step are set; shapes and places are filled in here.
template <bool SPLIT> void run_group(Group &g, int steps, cudaStream_t s) {
    uint32_t blocks = 0, spread = 0;
    double elements = 0.0;
    uint64_t at = kOperandsAt;
    static thread_local Group tiles;
    for (uint32_t i = 0; i < g.count; ++i) g.order[i] = tiles.order[i] = uint8_t(i);
    for (uint32_t i = 0; i < g.count; ++i) {
        Matrix &a = g.matrix[i];
        a.down_blocks = (a.m + kRows - 1) / kRows;
        a.x_blocks = 2 * ((a.n + kRows - 1) / kRows);
        a.a_blocks = 2 * a.down_blocks;
        const uint64_t x = bytes_of(a.down_blocks, a.x_blocks);
        const uint64_t square = bytes_of(a.down_blocks, a.a_blocks) * (SPLIT ? 2 : 1);
        a.x[0] = at;
        a.x[1] = at + (SPLIT ? 2 : 1) * x;
        a.a = at + (SPLIT ? 4 : 3) * x;
        a.p = a.a + square;
        a.diagonal = a.p + square;
        at = a.diagonal + uint64_t(a.down_blocks) * kRows * 8;
        const uint64_t all = uint64_t(a.m) * a.n;
        g.first[i] = blocks;
        tiles.first[i] = spread;
        blocks += uint32_t(std::min<uint64_t>(kSumBlocks, (all + kThreads * 8 - 1) / (kThreads * 8)));
        spread += a.down_blocks * a.x_blocks;
        elements += double(all);
    }
    g.first[g.count] = blocks;
    tiles.first[g.count] = spread;
    start(k_update_squares, blocks, kThreads, 1, 0, false, 8.0 * elements, s, g);
    std::copy(g.matrix, g.matrix + g.count, tiles.matrix);
    tiles.count = g.count;
    tiles.scratch = g.scratch;
    tiles.fault = g.fault;
    tiles.inverse = g.inverse;
    tiles.sums = g.sums;
    tiles.eps = g.eps;
    start(k_spread<SPLIT>, spread, kThreads, 1, 0, true, 8.0 * elements, s, tiles, g);
    for (int i = 0; i < steps; ++i) {
        phase<GRAM, SPLIT>(g, i, false, s);
        phase<POLYNOMIAL, SPLIT>(g, i, false, s);
        phase<APPLY, SPLIT>(g, i, i + 1 == steps, s);
    }
    start(k_check_fault, 8, kThreads, 1, 0, true, 0.0, s, g);
}

void run_small(Group &g, int steps, cudaStream_t s) {
    allow_shared<k_small>(kSmallShared);
    start(k_small, g.count, kSmallThreads, 1, kSmallShared, false, 0.0, s, g, steps);
}

// fill(matrix, place) sets what the call does to a place of the list.
template <class F>
void run(const ArcqmlMatrix *list, const ArcqmlMatrix *kinds, size_t count, int steps, double eps, double *ws, size_t ws_len,
         cudaStream_t s, F &&fill) {
    const uint64_t have = ws_len * sizeof(double), head = kOperandsAt;
    for_groups(list, kinds, count, have > head ? have - head : 0, [&](const Members &members, uint64_t, bool split, bool small) {
        static thread_local Group g;
        g.count = members.count;
        g.scratch = reinterpret_cast<char *>(ws);
        g.fault = reinterpret_cast<uint32_t *>(ws);
        g.inverse = reinterpret_cast<double *>(g.scratch + kScalesAt);
        g.arrived = reinterpret_cast<uint32_t *>(g.scratch + kArrivedAt);
        g.sums = reinterpret_cast<double *>(g.scratch + kSumsAt);
        g.partial = reinterpret_cast<float *>(g.scratch + kPartialAt);
        g.eps = eps;
        for (uint32_t i = 0; i < g.count; ++i) {
            const ArcqmlMatrix &a = list[members.at[i]];
            Matrix &m = g.matrix[i];
            m = Matrix{};
            m.flip = a.rows > a.columns;
            m.m = uint32_t(std::min(a.rows, a.columns));
            m.n = uint32_t(std::max(a.rows, a.columns));
            fill(m, members.at[i]);
        }
        if (small) run_small(g, steps, s);
        else if (split) run_group<true>(g, steps, s);
        else run_group<false>(g, steps, s);
    });
}

void check_steps(int steps, double eps) {
    if (steps < 1 || steps > 20) fail("the steps of an orthogonalisation must be 1 to 20");
    if (!std::isfinite(eps) || eps < 0.0) fail("epsilon must be finite and not negative");
}

}  // namespace

size_t orthogonalize_workspace(const ArcqmlMatrix *list, size_t count) {
    if (!list) return 0;
    uint64_t most = 0;
    for_groups(list, list, count, kGroupBytes,
               [&](const Members &, uint64_t bytes, bool, bool) { most = std::max(most, bytes); });
    return most ? size_t((kOperandsAt + most) / sizeof(double)) : 0;
}

void orthogonalize_device(const ArcqmlMatrix *in, const ArcqmlMatrix *out, size_t count, int steps, double eps,
                          double *ws, size_t ws_len, cudaStream_t s) {
    check_steps(steps, eps);
    check_list(in, count, "input");
    check_list(out, count, "output");
    for (size_t i = 0; i < count; ++i)
        if (in[i].dtype != out[i].dtype || in[i].rows != out[i].rows || in[i].columns != out[i].columns)
            refuse("output", i, "differs from its input in type or shape");
    check_scratch(ws, ws_len, orthogonalize_workspace(in, count));
    run(in, in, count, steps, eps, ws, ws_len, s, [&](Matrix &m, size_t i) {
        m.out = out[i].data;
        m.in = in[i].data;
        m.out_type = uint8_t(out[i].dtype);
        m.in_type = uint8_t(in[i].dtype);
    });
}

void muon_step_device(const ArcqmlMatrix *params, const ArcqmlMatrix *grads, const ArcqmlMatrix *momenta, size_t count,
                      const ArcqmlMuonOptions &o, double *ws, size_t ws_len, cudaStream_t s) {
    check_steps(o.steps, o.epsilon);
    if (!std::isfinite(o.learning_rate) || !std::isfinite(o.weight_decay) || !(o.momentum >= 0.0 && o.momentum < 1.0) ||
        (o.nesterov != 0 && o.nesterov != 1))
        fail("invalid Muon hyperparameters (finite lr and weight decay, 0 <= momentum < 1, nesterov 0 or 1)");
    check_list(params, count, "parameter");
    check_list(grads, count, "gradient");
    check_list(momenta, count, "momentum");
    for (size_t i = 0; i < count; ++i) {
        if (params[i].dtype == ARCQML_NO_TENSOR) refuse("parameter", i, "is missing");
        if (grads[i].dtype == ARCQML_NO_TENSOR) continue;
        if (grads[i].rows != params[i].rows || grads[i].columns != params[i].columns)
            refuse("gradient", i, "differs in shape from its parameter");
        if (momenta[i].dtype != ARCQML_F32 || momenta[i].rows != params[i].rows || momenta[i].columns != params[i].columns)
            refuse("momentum", i, "differs in shape from its parameter, or is not f32");
    }
    check_scratch(ws, ws_len, orthogonalize_workspace(params, count));
    run(grads, params, count, o.steps, o.epsilon, ws, ws_len, s, [&](Matrix &m, size_t i) {
        m.out = params[i].data;
        m.in = grads[i].data;
        m.momentum = static_cast<float *>(momenta[i].data);
        m.out_type = uint8_t(params[i].dtype);
        m.in_type = uint8_t(grads[i].dtype);
        m.nesterov = uint8_t(o.nesterov);
        m.beta = float(o.momentum);
        m.keep = float(1.0 - o.momentum);
        m.down = float(1.0 - o.learning_rate * o.weight_decay);
        m.rate = float(o.learning_rate * std::sqrt(std::max(1.0, double(params[i].rows) / double(params[i].columns))));
    });
}

}  // namespace arcqml
