// muon.cu — matrices orthogonalised by Newton-Schulz products, and the momentum step with them.
//
//   X <- u / (|u| + eps), then `steps` times  A = X X^T,  P = b A + c A^2,  X <- a X + P X
//
// with X (m x n, m <= n) the matrix or its transpose: every singular value s goes through
// a s + b s^3 + c s^5, which pushes it towards 1 (and never above 1.203, from 1 or less).
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <sstream>
#include <string>
#include <tuple>

#include "elements.cuh"
#include "launch.h"
#include "muon.h"
#include "profile.h"

namespace arcqml {
namespace {

constexpr float kA = 3.4445f, kB = -4.7750f, kC = 2.0315f;
constexpr int kThreads = 256;
constexpr uint32_t kSumBlocks = 256; // partial sums of a matrix

// One matrix of a call. The update u is the matrix `in`, or follows from the momentum and the gradient.
struct Job {
    void *out;       // the orthogonalised matrix, or the parameter
    const void *in;  // the matrix, or the gradient
    float *momentum; // null without a step
    uint64_t rows, columns;
    uint32_t out_type, in_type;
    float beta, keep; // of the step: momentum, and 1 - momentum
    float down, rate; // the parameter's factor, and the update's
    uint32_t nesterov;
};

__device__ __forceinline__ float load_as(const void *p, uint32_t type, uint64_t i) {
    if (type == ARCQML_F32) return static_cast<const float *>(p)[i];
    if (type == ARCQML_BF16) return to_wide(static_cast<const __nv_bfloat16 *>(p)[i]);
    return to_wide(static_cast<const __half *>(p)[i]);
}
__device__ __forceinline__ void store_as(void *p, uint32_t type, uint64_t i, float x) {
    if (type == ARCQML_F32) static_cast<float *>(p)[i] = x;
    else if (type == ARCQML_BF16) static_cast<__nv_bfloat16 *>(p)[i] = to_element<__nv_bfloat16>(x);
    else static_cast<__half *>(p)[i] = to_element<__half>(x);
}

__device__ __forceinline__ float update_of(const Job &j, uint64_t i) {
    const float g = load_as(j.in, j.in_type, i);
    if (!j.momentum) return g;
    const float m = j.momentum[i];
    return j.nesterov ? j.beta * m + j.keep * g : m;
}

// The momentum's update, and the squares of u: one f64 sum for each block.
__global__ void __launch_bounds__(kThreads) k_update_squares(const __grid_constant__ Job j, double *sums) {
    __shared__ double part[kThreads / 32];
    const uint64_t n = j.rows * j.columns;
    double sum = 0.0;
    for (uint64_t i = uint64_t(blockIdx.x) * kThreads + threadIdx.x; i < n; i += uint64_t(gridDim.x) * kThreads) {
        if (j.momentum) j.momentum[i] = j.beta * j.momentum[i] + j.keep * load_as(j.in, j.in_type, i);
        const double u = update_of(j, i);
        sum = fma(u, u, sum);
    }
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        sum = 0.0;
        for (int w = 0; w < kThreads / 32; ++w) sum += part[w];
        sums[blockIdx.x] = sum;
    }
}

// X = u / (|u| + eps), transposed where the matrix has more rows than columns.
__global__ void __launch_bounds__(kThreads) k_scale_update(const __grid_constant__ Job j, const double *sums,
                                                           uint32_t blocks, double eps, float *x) {
    double sum = 0.0;
    for (uint32_t b = 0; b < blocks; ++b) sum += sums[b];
    const double factor = 1.0 / (sqrt(sum) + eps);
    const bool flip = j.rows > j.columns;
    const uint64_t n = j.rows * j.columns;
    for (uint64_t i = uint64_t(blockIdx.x) * kThreads + threadIdx.x; i < n; i += uint64_t(gridDim.x) * kThreads) {
        const uint64_t r = i / j.columns, c = i % j.columns;
        x[flip ? c * j.rows + r : i] = float(double(update_of(j, i)) * factor);
    }
}

// out (m x n) = f add + h left right, right transposed with `turned`; 16 x 16 tiles.
__global__ void __launch_bounds__(256) k_product(const float *left, const float *right, const float *add, float *out,
                                                 uint64_t m, uint64_t n, uint64_t k, bool turned, float f, float h) {
    __shared__ float l[16][17], r[16][17];
    const uint32_t tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const uint64_t row = uint64_t(blockIdx.y) * 16 + ty, col = uint64_t(blockIdx.x) * 16 + tx;
    float sum = 0.0f;
    for (uint64_t k0 = 0; k0 < k; k0 += 16) {
        l[ty][tx] = row < m && k0 + tx < k ? left[row * k + k0 + tx] : 0.0f;
        const uint64_t c = uint64_t(blockIdx.x) * 16 + (turned ? ty : tx), kk = k0 + (turned ? tx : ty);
        const float v = c < n && kk < k ? right[turned ? c * k + kk : kk * n + c] : 0.0f;
        if (turned) r[tx][ty] = v;
        else r[ty][tx] = v;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 16; ++i) sum = fmaf(l[ty][i], r[i][tx], sum);
        __syncthreads();
    }
    if (row < m && col < n) out[row * n + col] = h * sum + (add ? f * add[row * n + col] : 0.0f);
}

// The result as it is, or the step with it.
__global__ void __launch_bounds__(kThreads) k_finish(const __grid_constant__ Job j, const float *x) {
    const bool flip = j.rows > j.columns;
    const uint64_t n = j.rows * j.columns;
    for (uint64_t i = uint64_t(blockIdx.x) * kThreads + threadIdx.x; i < n; i += uint64_t(gridDim.x) * kThreads) {
        const float v = x[flip ? i % j.columns * j.rows + i / j.columns : i];
        store_as(j.out, j.out_type, i, j.momentum ? j.down * load_as(j.out, j.out_type, i) - j.rate * v : v);
    }
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
        if (a.rows >> 24 || a.columns >> 24 || (a.rows * a.columns) >> 36) refuse(name, i, "is too large");
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
void start(void (*kernel)(P...), dim3 blocks, uint32_t threads, double bytes, cudaStream_t s, const A &...args) {
    cudaLaunchConfig_t c{};
    c.gridDim = blocks;
    c.blockDim = dim3(threads);
    c.stream = s;
    std::tuple<P...> held{P(args)...};
    const ProfToken tok = prof_begin(PROF_OTHER, s);
    const cudaError_t e = std::apply([&](auto &...x) { return cudaLaunchKernelEx(&c, kernel, x...); }, held);
    check_cuda(e, "orthogonalisation kernel launch");
    prof_end(tok, s, bytes);
}

// Scratch of one matrix: sums, X twice, A, P.
size_t scratch_of(const ArcqmlMatrix &a) {
    if (!present(a)) return 0;
    const uint64_t m = std::min(a.rows, a.columns), n = std::max(a.rows, a.columns);
    return kSumBlocks + size_t(m * n + m * m) + 8;
}

void run_job(const Job &j, int steps, double eps, double *ws, cudaStream_t s) {
    const uint64_t m = std::min(j.rows, j.columns), n = std::max(j.rows, j.columns), all = m * n;
    const uint32_t blocks = uint32_t(std::min<uint64_t>(kSumBlocks, (all + kThreads - 1) / kThreads));
    start(k_update_squares, blocks, kThreads, 4.0 * double(all), s, j, ws);
    float *x = reinterpret_cast<float *>(ws + kSumBlocks), *y = x + all, *a = y + all, *p = a + m * m;
    const uint32_t grid = uint32_t(std::min<uint64_t>(148 * 8, (all + kThreads - 1) / kThreads));
    start(k_scale_update, grid, kThreads, 4.0 * double(all), s, j, ws, blocks, eps, x);
    const auto tiles = [](uint64_t v) { return uint32_t((v + 15) / 16); };
    const float *none = nullptr;
    for (int i = 0; i < steps; ++i) {
        start(k_product, dim3(tiles(m), tiles(m)), 256, 0.0, s, x, x, none, a, m, m, n, true, 0.0f, 1.0f);
        start(k_product, dim3(tiles(m), tiles(m)), 256, 0.0, s, a, a, a, p, m, m, m, true, kB, kC);
        start(k_product, dim3(tiles(n), tiles(m)), 256, 0.0, s, p, x, x, y, m, n, m, false, kA, 1.0f);
        std::swap(x, y);
    }
    start(k_finish, grid, kThreads, 4.0 * double(all), s, j, x);
}

void check_steps(int steps, double eps) {
    if (steps < 1 || steps > 20) fail("the steps of an orthogonalisation must be 1 to 20");
    if (!std::isfinite(eps) || eps < 0.0) fail("epsilon must be finite and not negative");
}

}  // namespace

size_t orthogonalize_workspace(const ArcqmlMatrix *list, size_t count) {
    size_t most = 0;
    for (size_t i = 0; list && i < count; ++i) most = std::max(most, scratch_of(list[i]));
    return most;
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
    for (size_t i = 0; i < count; ++i) {
        if (!present(in[i])) continue;
        run_job({out[i].data, in[i].data, nullptr, in[i].rows, in[i].columns, out[i].dtype, in[i].dtype}, steps, eps, ws, s);
    }
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
    for (size_t i = 0; i < count; ++i) {
        if (!present(grads[i])) continue;
        const double ratio = double(params[i].rows) / double(params[i].columns);
        run_job({params[i].data, grads[i].data, static_cast<float *>(momenta[i].data), params[i].rows, params[i].columns,
                 params[i].dtype, grads[i].dtype, float(o.momentum), float(1.0 - o.momentum),
                 float(1.0 - o.learning_rate * o.weight_decay),
                 float(o.learning_rate * std::sqrt(std::max(1.0, ratio))), uint32_t(o.nesterov)},
                o.steps, o.epsilon, ws, s);
    }
}

}  // namespace arcqml
