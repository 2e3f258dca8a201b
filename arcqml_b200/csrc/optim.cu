// optim.cu — training over many device tensors: the global norm of a list of gradients, clipping
// by that norm, and the Adam step with the clip factor folded in.
//
// All of it is bound by HBM at real sizes (2 to 14 operations per element against 2 to 64 bytes)
// and by launches at small ones. One launch covers a whole list of any element types: the tensors'
// pointers and lengths travel as a kernel parameter, every tensor is cut into chunks, and blocks (in
// short lists warps) take chunks. No call reads anything back: the norm, the clip factor and the bias
// corrections pass between the launches in device scratch that the caller gives, so nothing is
// shared between calls. Sums are formed without atomics, in an order that the lengths, the types and the
// tensors' starts within 16 bytes fix (vectors begin at the first boundary).
//
//   k_square_sums      per block the f64 sum of squares of its chunks
//   k_scalars          one block: the sums in order -> norm, clip factor, step, bias corrections
//   k_clip, k_adam     the list scaled, or updated
//   k_short_*          all of it for a short list, in one launch of one cluster
//
// The norm has to be known before the first element is scaled, so a list larger than L2 is read
// twice: the update takes the chunks in reverse, and meets first what the norm left in L2.
//
// Measured on a B200 (copy rate 6535 GB/s), whole calls: norm of a 28-qubit state's gradient (4.3 GB)
// 594 us, 7.2 TB/s; norm of 251M bf16 elements in 300 tensors 91 us, 5.5 TB/s (the conversion to f64
// keeps its unit 75 % busy); clip of a 26-qubit state's gradient 485 us, 6.6 TB/s of its three passes;
// Adam on 400M f32 parameters with clipping 1914 us, 6.7 TB/s with the second read of the gradients;
// f32 parameters with bf16 gradients and copies (150M) 700 us, 6.4 TB/s; 8 f64 parameters' norm 7 us
// (the host's time for one launch).
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <sstream>
#include <string>
#include <type_traits>

#include "launch.h"
#include "optim.h"
#include "profile.h"

namespace cg = cooperative_groups;

namespace arcqml {
namespace {

constexpr int kOT = 256;  // threads per block
// Blocks of k_square_sums: what is resident at once (6 per SM; 8 per SM on the same places left a
// tail, 652 against 597 us for the norm of a 28-qubit state's gradient).
constexpr uint32_t kMaxBlocks = 148 * 6;
// The most 16-byte vectors (k_square_sums, k_clip) or groups (k_adam) of a chunk: one full batch of
// accesses per thread. Half of it costs the bf16 norm of 300 tensors 109 instead of 86 us, twice as
// much gains it 4 us and costs Adam 20 of 718.
constexpr uint32_t kChunk = 2048;
// Tensors of one launch. A launch costs the host 2.3 us more with 28 KB of parameters than with 3 KB,
// and blocks look their tensor up faster in a small table.
constexpr uint32_t kFewTensors = 64, kSomeTensors = 512, kMaxTensors = 1500;
// Short lists: one cluster, a warp per chunk. Against the several launches (whose time is the host's),
// f32 in 20 tensors: norm of 4 MB 10 and 12 us, of 6 MB 12 and 12, of 10 MB 16 and 12; clip of 2 MB 12
// and 15, of 2.8 MB 14 and 15, of 4 MB 16 and 15; Adam with 0.8 MB in each array 17 and 21, with 1.2 MB
// 20 and 21, with 1.6 MB 25 and 21.
constexpr uint32_t kShortTensors = kFewTensors;
constexpr uint64_t kShortNorm = uint64_t(6) << 20, kShortClip = uint64_t(5) << 19,
                   kShortMoments = uint64_t(1) << 20;
constexpr uint32_t kCluster = 16, kShortThreads = 512;
// Chunks of a warp: one batch of accesses per thread.
constexpr uint32_t kShortVectors = 256, kShortGroups = 64;

struct AdamScalars64 {
    double lr, b1, b2, nb1, nb2, eps, wd, down, bc1, bc2, factor;
};
// The clip factor in f32, as a power of two and a rest: a factor below f32's normal range (a norm
// near f32's largest values) keeps its precision.
struct Factor32 {
    float pre, rest;
};
struct AdamScalars32 {
    float b1, b2, nb1, nb2, eps, wd, down, rate;
    Factor32 factor;
};

// What k_scalars leaves for the launches behind it (the head of the scratch).
struct Scalars {
    double factor;
    AdamScalars64 h;
    AdamScalars32 hf;
};
constexpr size_t kScalarDoubles = 32;
static_assert(sizeof(Scalars) <= kScalarDoubles * sizeof(double), "the head of the scratch");

// The tensors of one launch. first[i]: the number of chunks before tensor i; first[count]: of all.
template <uint32_t CAP> struct TensorTable {
    void *data[CAP];
    uint64_t length[CAP];
    uint32_t first[CAP + 1];
    uint8_t dtype[CAP];
    uint32_t count, per; // tensors; vectors of a chunk
};

template <uint32_t CAP> struct AdamTable {
    void *p[CAP], *m[CAP], *v[CAP], *copy[CAP];
    const void *g[CAP];
    uint64_t length[CAP];
    uint32_t first[CAP + 1];
    uint8_t types[CAP];   // of the parameter, the gradient (<< 2) and the copy (<< 4)
    uint8_t aligned[CAP]; // kAligned*: arrays whose groups start on their own size
    uint8_t head[CAP];    // elements before the first group
    uint32_t count, per;  // tensors; groups of a chunk
};
enum { kAlignedG = 1, kAlignedM = 2, kAlignedV = 4, kAlignedCopy = 8, kHasCopy = 16 };
static_assert(sizeof(TensorTable<kMaxTensors>) < 32600 && sizeof(AdamTable<kSomeTensors>) < 32600,
              "kernel parameters hold 32764 bytes");

// The tensor of chunk c: the last i with first[i] <= c (tensors without chunks are not listed).
template <class T>
__device__ __forceinline__ uint32_t tensor_of(const T &t, uint32_t c) {
    uint32_t lo = 0, hi = t.count;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (t.first[mid] <= c) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Element types: their 16-byte vectors, and conversion from and to the type of the arithmetic.
template <uint32_t DTYPE> struct Elem;
template <> struct Elem<ARCQML_F64> {
    using type = double;
    using wide = double;
};
template <> struct Elem<ARCQML_F32> {
    using type = float;
    using wide = float;
};
template <> struct Elem<ARCQML_BF16> {
    using type = __nv_bfloat16;
    using wide = float;
};
template <> struct Elem<ARCQML_F16> {
    using type = __half;
    using wide = float;
};
__device__ __forceinline__ double widen(double x) { return x; }
__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ float widen(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float widen(__half x) { return __half2float(x); }
__device__ __forceinline__ void narrow(double x, double &y) { y = x; }
__device__ __forceinline__ void narrow(float x, float &y) { y = x; }
__device__ __forceinline__ void narrow(float x, __nv_bfloat16 &y) { y = __float2bfloat16_rn(x); }
__device__ __forceinline__ void narrow(float x, __half &y) { y = __float2half_rn(x); }

// N elements as the words that one or two accesses move; elements of 16 bits stay in pairs until
// they are used (one register each would double the registers of a load in flight).
template <uint32_t DTYPE, int N>
struct alignas(sizeof(typename Elem<DTYPE>::type) * N >= 16 ? 16 : 8) Words {
    using T = typename Elem<DTYPE>::type;
    using W = typename Elem<DTYPE>::wide;
    uint32_t w[sizeof(T) * N / 4];
    __device__ __forceinline__ void unpack(W (&x)[N]) const {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            if constexpr (DTYPE == ARCQML_F64) {
                x[j] = __hiloint2double(int(w[2 * j + 1]), int(w[2 * j]));
            } else if constexpr (DTYPE == ARCQML_F32) {
                x[j] = __uint_as_float(w[j]);
            } else if constexpr (DTYPE == ARCQML_BF16) {
                x[j] = __uint_as_float(j & 1 ? w[j / 2] & 0xffff0000u : w[j / 2] << 16);
            } else {
                x[j] = __half2float(__ushort_as_half(uint16_t(w[j / 2] >> (j & 1 ? 16 : 0))));
            }
        }
    }
    __device__ __forceinline__ void pack(const W (&x)[N]) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            if constexpr (DTYPE == ARCQML_F64) {
                w[2 * j] = uint32_t(__double2loint(x[j]));
                w[2 * j + 1] = uint32_t(__double2hiint(x[j]));
            } else if constexpr (DTYPE == ARCQML_F32) {
                w[j] = __float_as_uint(x[j]);
            } else if constexpr (DTYPE == ARCQML_BF16) {
                if (j & 1) {
                    const __nv_bfloat162 y = __floats2bfloat162_rn(x[j - 1], x[j]);
                    w[j / 2] = *reinterpret_cast<const uint32_t *>(&y);
                }
            } else {
                if (j & 1) {
                    const __half2 y = __floats2half2_rn(x[j - 1], x[j]);
                    w[j / 2] = *reinterpret_cast<const uint32_t *>(&y);
                }
            }
        }
    }
};

// The vectors of a tensor: elements before the first 16-byte boundary, whole vectors behind them.
template <class T> __device__ __forceinline__ uint32_t head_of(const T *p, uint64_t length) {
    const uint32_t h = uint32_t(-reinterpret_cast<uintptr_t>(p) & 15) / sizeof(T);
    return h < length ? h : uint32_t(length);
}

// The launches of one call follow each other without a gap: each lets the next one's blocks start as
// its own finish, and those wait before they read what an earlier launch wrote.
__device__ __forceinline__ void let_next_start() { cudaTriggerProgrammaticLaunchCompletion(); }
__device__ __forceinline__ void wait_for_last() { cudaGridDependencySynchronize(); }

// Sum over the block in a fixed order; valid in thread 0.
template <int THREADS> __device__ __forceinline__ double o_block_sum(double v) {
    __shared__ double red[THREADS / 32];
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    double r = 0.0;
    if (threadIdx.x == 0)
        for (int w = 0; w < THREADS / 32; ++w) r += red[w];
    return r;
}

// A chunk is taken by LANES threads, of which this is `lane`, and holds `per` vectors or groups.
//
// Squares of one chunk, added to acc in f64: the squares of f32 values leave the range of f32, and a
// norm that comes back in f64 is wanted to its precision.
template <uint32_t DTYPE, uint32_t LANES>
__device__ __forceinline__ void square_chunk(const void *data, uint64_t length, uint32_t chunk,
                                             uint32_t per, uint32_t lane, double (&acc)[4]) {
    using T = typename Elem<DTYPE>::type;
    using W = typename Elem<DTYPE>::wide;
    constexpr int N = 16 / sizeof(T), U = 8;
    const T *p = static_cast<const T *>(data);
    const uint32_t head = head_of(p, length);
    const uint64_t vectors = (length - head) / N;
    const auto *q = reinterpret_cast<const Words<DTYPE, N> *>(p + head);
    const uint64_t v0 = uint64_t(chunk) * per;
    const uint32_t n = uint32_t(min(uint64_t(per), vectors - min(v0, vectors)));
    const auto add = [&](const Words<DTYPE, N> &raw) {
        W x[N];
        raw.unpack(x);
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const double d = double(x[j]);
            acc[j % 4] = fma(d, d, acc[j % 4]);
        }
    };
    uint32_t v = lane;
    for (; v + (U - 1) * LANES < n; v += U * LANES) {
        Words<DTYPE, N> x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) x[u] = q[v0 + v + u * LANES];
#pragma unroll
        for (int u = 0; u < U; ++u) add(x[u]);
    }
    if (v < n) {  // less than a batch is left
        Words<DTYPE, N> x[U] = {};
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (v + u * LANES < n) x[u] = q[v0 + v + u * LANES];
#pragma unroll
        for (int u = 0; u < U; ++u) add(x[u]);
    }
    // the elements before the first vector (chunk 0) and behind the last one (the last chunk)
    if (chunk == 0 && lane < head) {
        const double d = double(widen(p[lane]));
        acc[0] = fma(d, d, acc[0]);
    }
    const uint64_t done = head + vectors * N;
    if (v0 + per >= vectors && lane < length - done) {
        const double d = double(widen(p[done + lane]));
        acc[1] = fma(d, d, acc[1]);
    }
}

// The squares of one chunk of tensor k of a table.
template <uint32_t LANES, class Table>
__device__ __forceinline__ void square_chunk_of(const Table &t, uint32_t k, uint32_t chunk,
                                                uint32_t lane, double (&acc)[4]) {
    const void *g = t.data[k];
    const uint64_t n = t.length[k];
    switch (t.dtype[k]) {
    case ARCQML_F64: square_chunk<ARCQML_F64, LANES>(g, n, chunk, t.per, lane, acc); break;
    case ARCQML_F32: square_chunk<ARCQML_F32, LANES>(g, n, chunk, t.per, lane, acc); break;
    case ARCQML_BF16: square_chunk<ARCQML_BF16, LANES>(g, n, chunk, t.per, lane, acc); break;
    default: square_chunk<ARCQML_F16, LANES>(g, n, chunk, t.per, lane, acc);
    }
}

// 48 warps of an SM with 8 accesses of 16 bytes each in flight. Measured without gain on the bf16 norm
// (86 us): contiguous ranges of chunks per block (86), the next batch loaded while one is added (115),
// bf16 values put into f64's places by bits instead of the conversion unit (96), 4 blocks and 16
// accesses (100).
template <uint32_t CAP>
__global__ void __launch_bounds__(kOT, 6)
    k_square_sums(const __grid_constant__ TensorTable<CAP> t, double *__restrict__ sums) {
    let_next_start();
    double acc[4] = {0.0, 0.0, 0.0, 0.0};
    for (uint32_t c = blockIdx.x; c < t.first[t.count]; c += gridDim.x) {
        const uint32_t k = tensor_of(t, c);
        square_chunk_of<kOT>(t, k, c - t.first[k], threadIdx.x, acc);
    }
    const double sum = o_block_sum<kOT>((acc[0] + acc[1]) + (acc[2] + acc[3]));
    if (threadIdx.x == 0) sums[blockIdx.x] = sum;
}

// min(1, max_norm / (norm + 1e-6)), 1 without clipping (max_norm < 0). A NaN norm gives NaN.
__device__ __forceinline__ double clip_factor(double norm, double max_norm) {
    if (!(max_norm >= 0.0)) return 1.0;
    const double f = max_norm / (norm + 1e-6);
    return f > 1.0 ? 1.0 : f;
}

__device__ __forceinline__ Factor32 factor32(double f) {
    return f < 0x1p-126 ? Factor32{0x1p-96f, float(f * 0x1p+96)} : Factor32{1.f, float(f)};
}

__device__ __forceinline__ double bias_correction(double beta, int64_t t) {
    return 1.0 - pow(beta, double(t));
}

__device__ __forceinline__ AdamScalars64 scalars64(const ArcqmlAdamOptions &o, double bc1,
                                                   double bc2, double factor) {
    return AdamScalars64{o.learning_rate, o.beta1, o.beta2, 1.0 - o.beta1, 1.0 - o.beta2,
                         o.epsilon, o.weight_decay, 1.0 - o.learning_rate * o.weight_decay, bc1,
                         bc2, factor};
}
// f32: with r = sqrt(1 - beta2^t) the step is lr r / (1 - beta1^t) times m / (sqrt(v) + r epsilon). The
// two factors are formed in f64 and rounded once. An epsilon below f32's range stays its smallest value:
// with 0 in its place a zero gradient's step would be 0 / 0.
__device__ __forceinline__ AdamScalars32 scalars32(const AdamScalars64 &h) {
    const double r = sqrt(h.bc2);
    const float eps = h.eps > 0.0 ? fmaxf(float(r * h.eps), 0x1p-149f) : 0.f;
    return AdamScalars32{float(h.b1), float(h.b2), float(h.nb1), float(h.nb2), eps,
                         float(h.wd), float(h.down), float(h.lr * r / h.bc1),
                         factor32(h.factor)};
}

// One block of a thread per sum. given != null: n = *given; else the root of the count sums.
// step != null: one more step is counted. The step count is no work of the launch before this one:
// what follows from it alone is formed without waiting for that launch. This block fits on an SM once four
// of the six blocks of k_square_sums there have ended (40 registers for each of its 1024 threads): behind a
// full grid that is in its tail, where no gain was measured; behind a smaller one it runs beside it.
constexpr int kScalarThreads = 1024;
__global__ void __launch_bounds__(kScalarThreads)
    k_scalars(const double *sums, uint32_t count, const double *given,
              const __grid_constant__ ArcqmlAdamOptions o, int64_t *step, double *norm,
              Scalars *out) {
    let_next_start();
    if (step && threadIdx.x == kScalarThreads - 32) {
        const int64_t now = *step + 1;
        const AdamScalars64 h =
            scalars64(o, bias_correction(o.beta1, now), bias_correction(o.beta2, now), 1.0);
        out->h = h;
        out->hf = scalars32(h);
    }
    wait_for_last();
    double acc = 0.0;
    for (uint32_t i = threadIdx.x; i < count; i += kScalarThreads) acc += sums[i];
    acc = o_block_sum<kScalarThreads>(acc);  // and the scalars above are written
    if (threadIdx.x != 0) return;
    const double n = given ? *given : sqrt(acc);
    if (norm) *norm = n;
    const double factor = clip_factor(n, o.max_norm);
    out->factor = factor;
    if (step) {
        out->h.factor = factor;
        out->hf.factor = factor32(factor);
        *step += 1;
    }
}

// One chunk times the factor: the product in the type of the arithmetic (f32 for 16-bit types, the
// factor rounded to it), rounded once to the element's type.
template <uint32_t DTYPE, uint32_t LANES>
__device__ __forceinline__ void clip_chunk(void *data, uint64_t length, uint32_t chunk,
                                           uint32_t per, uint32_t lane, double factor) {
    using T = typename Elem<DTYPE>::type;
    using W = typename Elem<DTYPE>::wide;
    constexpr int N = 16 / sizeof(T), U = 4;
    const auto times = [&](W x) {
        if constexpr (DTYPE == ARCQML_F64) {
            return x * factor;
        } else {
            const Factor32 f = factor32(factor);
            return x * f.pre * f.rest;
        }
    };
    T *p = static_cast<T *>(data);
    const uint32_t head = head_of(p, length);
    const uint64_t vectors = (length - head) / N;
    auto *q = reinterpret_cast<Words<DTYPE, N> *>(p + head);
    const uint64_t v0 = uint64_t(chunk) * per;
    const uint32_t n = uint32_t(min(uint64_t(per), vectors - min(v0, vectors)));
    const auto scale = [&](Words<DTYPE, N> &raw) {
        W x[N];
        raw.unpack(x);
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] = times(x[j]);
        raw.pack(x);
    };
    uint32_t v = lane;
    for (; v + (U - 1) * LANES < n; v += U * LANES) {
        Words<DTYPE, N> x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) x[u] = q[v0 + v + u * LANES];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            scale(x[u]);
            q[v0 + v + u * LANES] = x[u];
        }
    }
    if (v < n) {  // less than a batch is left
        Words<DTYPE, N> x[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (v + u * LANES < n) x[u] = q[v0 + v + u * LANES];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (v + u * LANES < n) {
                scale(x[u]);
                q[v0 + v + u * LANES] = x[u];
            }
    }
    if (chunk == 0 && lane < head) narrow(times(widen(p[lane])), p[lane]);
    const uint64_t done = head + vectors * N;
    if (v0 + per >= vectors && lane < length - done)
        narrow(times(widen(p[done + lane])), p[done + lane]);
}

template <uint32_t LANES, class Table>
__device__ __forceinline__ void clip_chunk_of(const Table &t, uint32_t k, uint32_t chunk,
                                              uint32_t lane, double factor) {
    void *g = t.data[k];
    const uint64_t n = t.length[k];
    switch (t.dtype[k]) {
    case ARCQML_F64: clip_chunk<ARCQML_F64, LANES>(g, n, chunk, t.per, lane, factor); break;
    case ARCQML_F32: clip_chunk<ARCQML_F32, LANES>(g, n, chunk, t.per, lane, factor); break;
    case ARCQML_BF16: clip_chunk<ARCQML_BF16, LANES>(g, n, chunk, t.per, lane, factor); break;
    default: clip_chunk<ARCQML_F16, LANES>(g, n, chunk, t.per, lane, factor);
    }
}

template <uint32_t CAP>
__global__ void __launch_bounds__(kOT, 4)
    k_clip(const __grid_constant__ TensorTable<CAP> t, const Scalars *sc) {
    let_next_start();
    wait_for_last();
    const double factor = sc->factor;
    if (factor == 1.0) return;
    // the last chunks first: they are the ones that the norm left in L2
    const uint32_t c = t.first[t.count] - 1 - blockIdx.x, k = tensor_of(t, c);
    clip_chunk_of<kOT>(t, k, c - t.first[k], threadIdx.x, factor);
}

// f64, every operation rounded on its own, in the order of the host's update and of the optimizer
// loop (crates/arcqml-optim/src/adam.rs:190-240), so the three agree to the bias corrections.
__device__ __forceinline__ void adam_update(double &p, double &m, double &v, double g,
                                            const AdamScalars64 &h, bool decoupled) {
    double a = __dmul_rn(g, h.factor);
    if (!decoupled) a = __dadd_rn(a, __dmul_rn(h.wd, p));
    m = __dadd_rn(__dmul_rn(h.b1, m), __dmul_rn(h.nb1, a));
    v = __dadd_rn(__dmul_rn(h.b2, v), __dmul_rn(__dmul_rn(h.nb2, a), a));
    const double mh = __ddiv_rn(m, h.bc1), vh = __ddiv_rn(v, h.bc2);
    if (decoupled) p = __dmul_rn(p, h.down);
    p = __dsub_rn(p, __ddiv_rn(__dmul_rn(h.lr, mh), __dadd_rn(__dsqrt_rn(vh), h.eps)));
}

// f32 for every other type. A 16-bit parameter is rounded to nearest once per step: updates below
// half its step are lost, which is what f32 parameters with 16-bit copies are for. v's own root is taken,
// its bias correction is in the scalars: in the first steps v / (1 - beta2^t) leaves f32's range from
// gradients of 2e19 on, which v itself holds up to 6e20.
__device__ __forceinline__ void adam_update(float &p, float &m, float &v, float g,
                                            const AdamScalars32 &h, bool decoupled) {
    float a = g * h.factor.pre * h.factor.rest;
    if (!decoupled) a = fmaf(h.wd, p, a);
    m = fmaf(h.b1, m, h.nb1 * a);
    v = fmaf(h.b2, v, h.nb2 * a * a);
    const float u = m / (sqrtf(v) + h.eps);
    if (decoupled) p *= h.down;
    p = fmaf(-h.rate, u, p);
}

// The elements of a group of k_adam: one 16-byte access to the f64 or f32 arrays.
template <uint32_t DTYPE> constexpr int kGroup = DTYPE == ARCQML_F64 ? 2 : 4;

// A group (from element e on) of an array: one access, or one per element.
template <uint32_t DTYPE>
__device__ __forceinline__ Words<DTYPE, kGroup<DTYPE>> load_group(const void *p, uint64_t e,
                                                                  bool aligned) {
    constexpr int N = kGroup<DTYPE>;
    using T = typename Elem<DTYPE>::type;
    const T *q = static_cast<const T *>(p) + e;
    if (aligned) return *reinterpret_cast<const Words<DTYPE, N> *>(q);
    typename Elem<DTYPE>::wide x[N];
    for (int j = 0; j < N; ++j) x[j] = widen(q[j]);
    Words<DTYPE, N> raw;
    raw.pack(x);
    return raw;
}
template <uint32_t DTYPE>
__device__ __forceinline__ void store_group(void *p, uint64_t e, bool aligned,
                                            const typename Elem<DTYPE>::wide (&x)[kGroup<DTYPE>]) {
    constexpr int N = kGroup<DTYPE>;
    using T = typename Elem<DTYPE>::type;
    T *q = static_cast<T *>(p) + e;
    if (aligned) {
        Words<DTYPE, N> raw;
        raw.pack(x);
        *reinterpret_cast<Words<DTYPE, N> *>(q) = raw;
    } else {
        for (int j = 0; j < N; ++j) narrow(x[j], q[j]);
    }
}

// One chunk of tensor k: two groups of each array in flight per thread. The groups start where the
// parameter's are aligned; an array that is not aligned there (a gradient in an unpadded bucket) is
// taken element by element, through L1.
template <uint32_t PT, uint32_t GT, uint32_t LANES, class Table, class H>
__device__ __forceinline__ void adam_chunk(const Table &t, uint32_t k, uint32_t chunk,
                                           uint32_t lane, const H &h, bool decoupled) {
    using P = typename Elem<PT>::type;
    using G = typename Elem<GT>::type;
    using W = typename Elem<PT>::wide;
    constexpr uint32_t WT = sizeof(W) == 8 ? ARCQML_F64 : ARCQML_F32;
    constexpr int U = 2, N = kGroup<PT>;
    const uint64_t length = t.length[k];
    const uint32_t per = t.per, head = t.head[k], aligned = t.aligned[k], ct = t.types[k] >> 4;
    void *p = t.p[k], *m = t.m[k], *v = t.v[k], *copy = t.copy[k];
    const void *g = t.g[k];
    const uint64_t groups = (length - head) / N;
    const uint64_t i0 = uint64_t(chunk) * per;
    const uint32_t n = uint32_t(min(uint64_t(per), groups - min(i0, groups)));
    const uint64_t e0 = head + N * i0;
    const auto update = [&](uint64_t e, const Words<PT, N> &rp, const Words<GT, N> &rg,
                            const Words<WT, N> &rm, const Words<WT, N> &rv) {
        W x[N], y[N], mm[N], vv[N];
        rp.unpack(x);
        rg.unpack(y);
        rm.unpack(mm);
        rv.unpack(vv);
#pragma unroll
        for (int j = 0; j < N; ++j) adam_update(x[j], mm[j], vv[j], y[j], h, decoupled);
        store_group<PT>(p, e, true, x);
        store_group<WT>(m, e, aligned & kAlignedM, mm);
        store_group<WT>(v, e, aligned & kAlignedV, vv);
        if constexpr (PT == ARCQML_F32) {
            if (aligned & kHasCopy) {
                if (ct == ARCQML_BF16) store_group<ARCQML_BF16>(copy, e, aligned & kAlignedCopy, x);
                else store_group<ARCQML_F16>(copy, e, aligned & kAlignedCopy, x);
            }
        }
    };
    uint32_t i = lane;
    for (; i + (U - 1) * LANES < n; i += U * LANES) {
        Words<PT, N> xp[U];
        Words<GT, N> xg[U];
        Words<WT, N> xm[U], xv[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint64_t e = e0 + N * (i + u * LANES);
            xp[u] = load_group<PT>(p, e, true);
            xg[u] = load_group<GT>(g, e, aligned & kAlignedG);
            xm[u] = load_group<WT>(m, e, aligned & kAlignedM);
            xv[u] = load_group<WT>(v, e, aligned & kAlignedV);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) update(e0 + N * (i + u * LANES), xp[u], xg[u], xm[u], xv[u]);
    }
    for (; i < n; i += LANES) {
        const uint64_t e = e0 + N * i;
        update(e, load_group<PT>(p, e, true), load_group<GT>(g, e, aligned & kAlignedG),
               load_group<WT>(m, e, aligned & kAlignedM), load_group<WT>(v, e, aligned & kAlignedV));
    }
    // the elements before the first group (chunk 0) and behind the last one (the last chunk)
    const uint64_t done = head + groups * N;
    const uint32_t tail = i0 + per >= groups ? uint32_t(length - done) : 0;
    const uint32_t first = chunk == 0 ? head : 0;
    if (lane < first + tail) {
        const uint64_t e = lane < first ? lane : done + lane - first;
        P &rp = static_cast<P *>(p)[e];
        W x = widen(rp);
        adam_update(x, static_cast<W *>(m)[e], static_cast<W *>(v)[e],
                    widen(static_cast<const G *>(g)[e]), h, decoupled);
        narrow(x, rp);
        if constexpr (PT == ARCQML_F32) {
            if (aligned & kHasCopy) {
                if (ct == ARCQML_BF16) narrow(x, static_cast<__nv_bfloat16 *>(copy)[e]);
                else narrow(x, static_cast<__half *>(copy)[e]);
            }
        }
    }
}

template <uint32_t PT, uint32_t LANES, class Table>
__device__ __forceinline__ void adam_chunk_g(const Table &t, uint32_t k, uint32_t chunk,
                                             uint32_t lane, const AdamScalars32 &h,
                                             bool decoupled) {
    switch (t.types[k] >> 2 & 3) {
    case ARCQML_F32: adam_chunk<PT, ARCQML_F32, LANES>(t, k, chunk, lane, h, decoupled); break;
    case ARCQML_BF16: adam_chunk<PT, ARCQML_BF16, LANES>(t, k, chunk, lane, h, decoupled); break;
    default: adam_chunk<PT, ARCQML_F16, LANES>(t, k, chunk, lane, h, decoupled);
    }
}

template <uint32_t LANES, class Table>
__device__ __forceinline__ void adam_chunk_of(const Table &t, uint32_t k, uint32_t chunk,
                                              uint32_t lane, const AdamScalars32 &h,
                                              bool decoupled) {
    switch (t.types[k] & 3) {
    case ARCQML_F32: adam_chunk_g<ARCQML_F32, LANES>(t, k, chunk, lane, h, decoupled); break;
    case ARCQML_BF16: adam_chunk_g<ARCQML_BF16, LANES>(t, k, chunk, lane, h, decoupled); break;
    default: adam_chunk_g<ARCQML_F16, LANES>(t, k, chunk, lane, h, decoupled);
    }
}

// One block per chunk: the hardware deals them out as others finish (a grid of the resident blocks that
// take chunks in turn: 801 instead of 718 us with bf16 gradients and copies). 4 blocks per SM, 64
// registers; 3 or 5 cost 1 %. One launch for every type: the f64 arithmetic, three divisions and a root
// per element, spills a little there and still runs as fast as in a launch of its own (366 us for a
// 24-qubit state, 2.1 GB).
template <uint32_t CAP>
__global__ void __launch_bounds__(kOT, 4)
    k_adam(const __grid_constant__ AdamTable<CAP> t, bool decoupled, const Scalars *sc) {
    let_next_start();
    wait_for_last();
    // the last chunks first: their gradients are the ones that the norm left in L2
    const uint32_t chunks = t.first[t.count];
    const uint32_t c = chunks - 1 - blockIdx.x, k = tensor_of(t, c), chunk = c - t.first[k];
    // copies of the scalars: for all the compiler knows the stores change what sc points to
    if ((t.types[k] & 3) == ARCQML_F64) {
        const AdamScalars64 h = sc->h;
        adam_chunk<ARCQML_F64, ARCQML_F64, kOT>(t, k, chunk, threadIdx.x, h, decoupled);
    } else {
        const AdamScalars32 h = sc->hf;
        adam_chunk_of<kOT>(t, k, chunk, threadIdx.x, h, decoupled);
    }
}

// ------------------------------------------------------------------ short lists

// The sum of v over the cluster, in rank order, in every thread. The blocks' sums are read from
// their shared memory: no block may end before the cluster has met again.
__device__ __forceinline__ double cluster_sum(double v, cg::cluster_group &cluster) {
    __shared__ double mine;
    const double sum = o_block_sum<kShortThreads>(v);
    if (threadIdx.x == 0) mine = sum;
    cluster.sync();
    double r = 0.0;
    for (uint32_t b = 0; b < cluster.num_blocks(); ++b) r += *cluster.map_shared_rank(&mine, b);
    return r;
}

// Norm (or the given one) and clip of a short list: clips when max_norm >= 0.
__global__ void __launch_bounds__(kShortThreads, 1)
    k_short_clip(const __grid_constant__ TensorTable<kShortTensors> t, const double *given,
                 double max_norm, double *norm) {
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t lane = threadIdx.x & 31, chunks = t.first[t.count];
    const uint32_t warp = cluster.block_rank() * (kShortThreads / 32) + (threadIdx.x >> 5);
    const uint32_t warps = cluster.num_blocks() * (kShortThreads / 32);
    double acc[4] = {0.0, 0.0, 0.0, 0.0};
    double n;
    if (given) {
        n = *given;
    } else {
        for (uint32_t c = warp; c < chunks; c += warps) {
            const uint32_t k = tensor_of(t, c);
            square_chunk_of<32>(t, k, c - t.first[k], lane, acc);
        }
        n = sqrt(cluster_sum((acc[0] + acc[1]) + (acc[2] + acc[3]), cluster));
    }
    if (warp == 0 && lane == 0 && norm) *norm = n;
    const double factor = clip_factor(n, max_norm);
    if (factor != 1.0)
        for (uint32_t c = warp; c < chunks; c += warps) {
            const uint32_t k = tensor_of(t, c);
            clip_chunk_of<32>(t, k, c - t.first[k], lane, factor);
        }
    cluster.sync();
}

// The squares of a chunk's gradients, over the same elements that adam_chunk takes.
template <uint32_t GT, uint32_t LANES, class Table>
__device__ __forceinline__ void square_groups(const Table &t, uint32_t k, uint32_t chunk,
                                              uint32_t lane, double (&acc)[4]) {
    using G = typename Elem<GT>::type;
    constexpr int N = kGroup<GT>;  // f64 gradients belong to f64 parameters
    const uint32_t per = t.per, head = t.head[k];
    const uint64_t length = t.length[k], groups = (length - head) / N, i0 = uint64_t(chunk) * per;
    const uint32_t n = uint32_t(min(uint64_t(per), groups - min(i0, groups)));
    const void *g = t.g[k];
#pragma unroll 2
    for (uint32_t i = lane; i < n; i += LANES) {
        typename Elem<GT>::wide x[N];
        load_group<GT>(g, head + N * (i0 + i), t.aligned[k] & kAlignedG).unpack(x);
#pragma unroll
        for (int j = 0; j < N; ++j) acc[j] = fma(double(x[j]), double(x[j]), acc[j]);
    }
    const uint64_t done = head + groups * N;
    const uint32_t tail = i0 + per >= groups ? uint32_t(length - done) : 0;
    const uint32_t first = chunk == 0 ? head : 0;
    if (lane < first + tail) {
        const double x =
            double(widen(static_cast<const G *>(g)[lane < first ? lane : done + lane - first]));
        acc[0] = fma(x, x, acc[0]);
    }
}

// One Adam step of a short list. Every block reads the step count before the cluster first meets;
// the first block writes the new one after that.
__global__ void __launch_bounds__(kShortThreads, 1)
    k_short_adam(const __grid_constant__ AdamTable<kShortTensors> t,
                 const __grid_constant__ ArcqmlAdamOptions o, int64_t *step, const double *given,
                 double *norm) {
    __shared__ double bc[2];
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t lane = threadIdx.x & 31, chunks = t.first[t.count];
    const uint32_t warp = cluster.block_rank() * (kShortThreads / 32) + (threadIdx.x >> 5);
    const uint32_t warps = cluster.num_blocks() * (kShortThreads / 32);
    const int64_t now = *step + 1;
    // the last warp has the fewest chunks
    if (threadIdx.x == kShortThreads - 1) bc[0] = bias_correction(o.beta1, now);
    if (threadIdx.x == kShortThreads - 2) bc[1] = bias_correction(o.beta2, now);
    double n = 0.0;
    if (o.max_norm >= 0.0 && !given) {
        double acc[4] = {0.0, 0.0, 0.0, 0.0};
        for (uint32_t c = warp; c < chunks; c += warps) {
            const uint32_t k = tensor_of(t, c), chunk = c - t.first[k];
            switch (t.types[k] >> 2 & 3) {
            case ARCQML_F64: square_groups<ARCQML_F64, 32>(t, k, chunk, lane, acc); break;
            case ARCQML_F32: square_groups<ARCQML_F32, 32>(t, k, chunk, lane, acc); break;
            case ARCQML_BF16: square_groups<ARCQML_BF16, 32>(t, k, chunk, lane, acc); break;
            default: square_groups<ARCQML_F16, 32>(t, k, chunk, lane, acc);
            }
        }
        n = sqrt(cluster_sum((acc[0] + acc[1]) + (acc[2] + acc[3]), cluster));
    } else {
        if (given) n = *given;
        cluster.sync();
    }
    if (warp == 0 && lane == 0) {
        if (norm) *norm = n;
        *step = now;
    }
    const bool decoupled = o.decoupled != 0;
    const AdamScalars64 h = scalars64(o, bc[0], bc[1], clip_factor(n, o.max_norm));
    const AdamScalars32 hf = scalars32(h);
    for (uint32_t c = warp; c < chunks; c += warps) {
        const uint32_t k = tensor_of(t, c), chunk = c - t.first[k];
        if ((t.types[k] & 3) == ARCQML_F64)
            adam_chunk<ARCQML_F64, ARCQML_F64, 32>(t, k, chunk, lane, h, decoupled);
        else adam_chunk_of<32>(t, k, chunk, lane, hf, decoupled);
    }
    cluster.sync();
}

// ------------------------------------------------------------------ host side

uint32_t element_size(uint32_t dtype) {
    return dtype == ARCQML_F64 ? 8 : dtype == ARCQML_F32 ? 4 : 2;
}

// Elements of a group of k_adam (kGroup).
uint32_t group_size(const ArcqmlTensor &t) { return t.dtype == ARCQML_F64 ? 2 : 4; }

[[noreturn]] void fail_at(const char *list, size_t i, const char *what) {
    std::ostringstream m;
    m << list << " tensor " << i << " " << what;
    fail(m.str());
}

bool present(const ArcqmlTensor &t) { return t.dtype != ARCQML_NO_TENSOR && t.length != 0; }

// Whether place i of the list holds a tensor with elements; fails for a malformed entry.
bool check_tensor(const ArcqmlTensor &t, const char *list, size_t i) {
    if (t.dtype > ARCQML_NO_TENSOR) fail_at(list, i, "has an unknown type");
    if (t.reserved != 0) fail_at(list, i, "has a nonzero reserved field");
    if (!present(t)) return false;
    if (t.length >> 40) fail_at(list, i, "is too long");
    if (!t.data) fail_at(list, i, "is null");
    if (reinterpret_cast<uintptr_t>(t.data) % element_size(t.dtype))
        fail_at(list, i, "is not aligned to its elements");
    return true;
}

void check_workspace(const double *ws, size_t len, size_t need) {
    if (!ws) fail("workspace is null");
    if (reinterpret_cast<uintptr_t>(ws) % 16) fail("workspace is not aligned to 16 bytes");
    if (len < need) {
        std::ostringstream m;
        m << "workspace of " << len << " doubles is too small: the list needs " << need;
        fail(m.str());
    }
}

// Chunks of `per` vectors of a tensor: at least one, for the elements outside vectors.
uint64_t chunks_of(const ArcqmlTensor &t, uint32_t per) {
    const uint32_t size = element_size(t.dtype);
    const uint64_t head = (-reinterpret_cast<uintptr_t>(t.data) & 15) / size;
    const uint64_t vectors = t.length > head ? (t.length - head) / (16 / size) : 0;
    return std::max<uint64_t>(1, (vectors + per - 1) / per);
}

// The whole list is checked before anything is launched. Chunks are counted in 32 bits.
void check_tensors(const ArcqmlTensor *list, size_t count, const char *name) {
    if (count && !list) fail(std::string(name) + " list is null");
    uint64_t chunks = 0;
    for (size_t i = 0; i < count; ++i)
        if (check_tensor(list[i], name, i)) chunks += list[i].length / kChunk + 1;
    if (chunks >> 31) fail(std::string(name) + " list holds too many elements");
}

// Whether one cluster takes the list in one launch: a list of gradients by its bytes, a list of
// parameters (adam) by its moments'.
bool is_short(const ArcqmlTensor *list, size_t count, uint64_t most, bool adam = false) {
    uint64_t bytes = 0;
    uint32_t tensors = 0;
    for (size_t i = 0; i < count; ++i) {
        if (!present(list[i])) continue;
        const uint32_t size = element_size(list[i].dtype);
        bytes += list[i].length * (adam ? std::max(size, 4u) : size);
        if (++tensors > kShortTensors || bytes > most) return false;
    }
    return true;
}

// Fills tables with a list's (checked) tensors in chunks of `per` vectors and calls
// launch(table, bytes) for each full one and the last.
template <uint32_t CAP, class F>
void for_tensor_tables(const ArcqmlTensor *list, size_t count, uint32_t per, F &&launch) {
    TensorTable<CAP> t;
    t.count = 0;
    t.per = per;
    uint64_t chunks = 0;
    double bytes = 0.0;
    const auto flush = [&] {
        t.first[t.count] = uint32_t(chunks);
        launch(t, bytes);
        t.count = 0;
        chunks = 0;
        bytes = 0.0;
    };
    for (size_t i = 0; i < count; ++i) {
        if (!present(list[i])) continue;
        if (t.count == CAP) flush();
        t.data[t.count] = list[i].data;
        t.length[t.count] = list[i].length;
        t.dtype[t.count] = uint8_t(list[i].dtype);
        t.first[t.count++] = uint32_t(chunks);
        chunks += chunks_of(list[i], per);
        bytes += double(list[i].length) * element_size(list[i].dtype);
    }
    flush();
}

// The same for a (checked) Adam step. Calls launch for no empty table.
struct AdamLists {
    const ArcqmlTensor *params, *grads, *m, *v, *copies;
    size_t count;
};
template <uint32_t CAP, class F>
void for_adam_tables(const AdamLists &l, uint32_t per, F &&launch) {
    AdamTable<CAP> t;
    t.count = 0;
    t.per = per;
    uint64_t chunks = 0;
    double bytes = 0.0;
    const auto flush = [&] {
        t.first[t.count] = uint32_t(chunks);
        launch(t, bytes);
        t.count = 0;
        chunks = 0;
        bytes = 0.0;
    };
    // groups from the first place on where the parameter's start on their size
    const auto apart = [](const ArcqmlTensor &x) {
        return (reinterpret_cast<uintptr_t>(x.data) / element_size(x.dtype)) & (group_size(x) - 1);
    };
    for (size_t i = 0; i < l.count; ++i) {
        const ArcqmlTensor &p = l.params[i], &g = l.grads[i];
        if (!present(p) || g.dtype == ARCQML_NO_TENSOR) continue;
        if (t.count == CAP) flush();
        const bool copy = l.copies && l.copies[i].dtype != ARCQML_NO_TENSOR;
        const uint64_t at = apart(p), head = std::min<uint64_t>(-at & (group_size(p) - 1), p.length);
        const uint32_t k = t.count++;
        t.p[k] = p.data;
        t.g[k] = g.data;
        t.m[k] = l.m[i].data;
        t.v[k] = l.v[i].data;
        t.copy[k] = copy ? l.copies[i].data : nullptr;
        t.length[k] = p.length;
        t.first[k] = uint32_t(chunks);
        t.types[k] = uint8_t(p.dtype | g.dtype << 2 | (copy ? l.copies[i].dtype << 4 : 0));
        t.aligned[k] = uint8_t((apart(g) == at ? kAlignedG : 0) |
                               (apart(l.m[i]) == at ? kAlignedM : 0) |
                               (apart(l.v[i]) == at ? kAlignedV : 0) |
                               (copy && apart(l.copies[i]) == at ? kAlignedCopy : 0) |
                               (copy ? kHasCopy : 0));
        t.head[k] = uint8_t(head);
        chunks += std::max<uint64_t>(1, ((p.length - head) / group_size(p) + per - 1) / per);
        bytes += double(p.length) *
                 (2.0 * element_size(p.dtype) + element_size(g.dtype) +
                  4.0 * element_size(l.m[i].dtype) +
                  (copy ? element_size(l.copies[i].dtype) : 0.0));
    }
    if (t.count) flush();
}

// A launch of one cluster of no more blocks than the list's chunks give warps to work, at most 16: a
// small list takes few SMs (its time is the launch's either way).
template <auto KERNEL, class... Args>
void launch_cluster(uint32_t chunks, double bytes, cudaStream_t s, const char *what,
                    const Args &...args) {
    static_assert(std::is_same_v<decltype(KERNEL), void (*)(Args...)>);
    uint32_t blocks = 1;
    while (blocks < kCluster && blocks * (kShortThreads / 32) < chunks) blocks *= 2;
    if (blocks > 8) {
        // above 8 blocks a cluster's size has to be allowed, once per kernel and device
        static std::atomic<uint64_t> allowed{0};
        int dev = 0;
        check_cuda(cudaGetDevice(&dev), "cudaGetDevice");
        const uint64_t bit = uint64_t(1) << (dev & 63);
        if (dev > 63 || !(allowed.load(std::memory_order_relaxed) & bit)) {
            check_cuda(cudaFuncSetAttribute(reinterpret_cast<const void *>(KERNEL),
                                            cudaFuncAttributeNonPortableClusterSizeAllowed, 1),
                       what);
            allowed.fetch_or(bit, std::memory_order_relaxed);
        }
    }
    cudaLaunchConfig_t c{};
    cudaLaunchAttribute a{};
    a.id = cudaLaunchAttributeClusterDimension;
    a.val.clusterDim.x = blocks;
    a.val.clusterDim.y = a.val.clusterDim.z = 1;
    c.gridDim = dim3(blocks);
    c.blockDim = dim3(kShortThreads);
    c.stream = s;
    c.attrs = &a;
    c.numAttrs = blocks > 1 ? 1 : 0;
    void *params[] = {const_cast<void *>(static_cast<const void *>(&args))...};
    const ProfToken tok = prof_begin(PROF_OTHER, s);
    check_cuda(cudaLaunchKernelExC(&c, reinterpret_cast<const void *>(KERNEL), params), what);
    prof_end(tok, s, bytes);
}

// A launch of `blocks` blocks that, with `follows`, may start while the last one ends. A call's first
// launch never does: all that came before it on the stream is complete when it starts.
template <auto KERNEL, int THREADS = kOT, class... Args>
void launch(uint32_t blocks, bool follows, double bytes, cudaStream_t s, const char *what,
            const Args &...args) {
    cudaLaunchConfig_t c{};
    cudaLaunchAttribute a{};
    a.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    a.val.programmaticStreamSerializationAllowed = 1;
    c.gridDim = dim3(blocks);
    c.blockDim = dim3(THREADS);
    c.stream = s;
    c.attrs = &a;
    c.numAttrs = follows ? 1 : 0;
    static_assert(std::is_same_v<decltype(KERNEL), void (*)(Args...)>);
    void *params[] = {const_cast<void *>(static_cast<const void *>(&args))...};
    const ProfToken tok = prof_begin(PROF_OTHER, s);
    check_cuda(cudaLaunchKernelExC(&c, reinterpret_cast<const void *>(KERNEL), params), what);
    prof_end(tok, s, bytes);
}

// Vectors or groups of a chunk, from all of the list's: two chunks for each place that the launch
// has on the GPU, between 256 (one access per thread) and 2048.
uint32_t chunk_size(uint64_t total, uint32_t places) {
    uint32_t per = kOT;
    while (per < kChunk && uint64_t(per) * places * 2 < total) per *= 2;
    return per;
}

// Calls f(capacity) with the smallest table that holds the list's tensors, or else the largest.
template <class F> void for_table_size(const ArcqmlTensor *list, size_t count, F &&f) {
    size_t tensors = count;
    if (count > kFewTensors)
        tensors = size_t(std::count_if(list, list + count, [](auto &t) { return present(t); }));
    if (tensors <= kFewTensors) f(std::integral_constant<uint32_t, kFewTensors>{});
    else if (tensors <= kSomeTensors) f(std::integral_constant<uint32_t, kSomeTensors>{});
    else f(std::integral_constant<uint32_t, kMaxTensors>{});
}

// The sums of squares of one table's tensors, or of a list's; returns their count.
template <uint32_t CAP>
uint32_t square_sums(const TensorTable<CAP> &t, double bytes, double *sums, cudaStream_t s) {
    if (!t.count) return 0;
    const uint32_t blocks = std::min(t.first[t.count], kMaxBlocks);
    launch<k_square_sums<CAP>>(blocks, false, bytes, s, "gradient norm kernel launch", t, sums);
    return blocks;
}

uint32_t square_sums(const ArcqmlTensor *grads, size_t count, uint32_t per, double *ws,
                     cudaStream_t s) {
    uint32_t sums = 0;
    for_table_size(grads, count, [&](auto capacity) {
        for_tensor_tables<capacity>(grads, count, per, [&](const auto &t, double bytes) {
            sums += square_sums(t, bytes, ws + kScalarDoubles + sums, s);
        });
    });
    return sums;
}

// The chunk size of k_square_sums and k_clip for a list.
uint32_t vectors_per_chunk(const ArcqmlTensor *list, size_t count) {
    uint64_t bytes = 0;
    for (size_t i = 0; i < count; ++i)
        if (present(list[i])) bytes += list[i].length * element_size(list[i].dtype);
    return chunk_size(bytes / 16, kMaxBlocks);
}

const Scalars *scalars(uint32_t sums, const double *given, const ArcqmlAdamOptions &o,
                       int64_t *step, double *norm, double *ws, cudaStream_t s) {
    auto *out = reinterpret_cast<Scalars *>(ws);
    const double *first = ws + kScalarDoubles;
    launch<k_scalars, kScalarThreads>(1, sums != 0, 8.0 * sums, s, "gradient norm kernel launch",
                                      first, sums, given, o, step, norm, out);
    return out;
}

ArcqmlAdamOptions clip_options(double max_norm) {
    ArcqmlAdamOptions o{};
    o.max_norm = max_norm;
    return o;
}

// The norm of a short list, or its clipping (max_norm >= 0).
void short_clip(const ArcqmlTensor *grads, size_t count, const double *given, double max_norm,
                double *norm, cudaStream_t s) {
    for_tensor_tables<kShortTensors>(
        grads, count, kShortVectors, [&](const TensorTable<kShortTensors> &t, double bytes) {
            launch_cluster<k_short_clip>(t.first[t.count], max_norm >= 0.0 ? 2.0 * bytes : bytes, s,
                                         "gradient norm kernel launch", t, given, max_norm, norm);
        });
}

}  // namespace

static size_t workspace_of(size_t count) {
    return kScalarDoubles + (count / kMaxTensors + 1) * size_t(kMaxBlocks);
}

size_t gradient_workspace(const ArcqmlTensor *list, size_t count) {
    return !list || is_short(list, count, kShortClip) ? 0 : workspace_of(count);
}

size_t adam_workspace(const ArcqmlTensor *list, size_t count) {
    return !list || is_short(list, count, kShortMoments, true) ? 0 : workspace_of(count);
}

void gradient_norm_device(const ArcqmlTensor *grads, size_t count, double *norm, double *ws,
                          size_t ws_len, cudaStream_t s) {
    check_tensors(grads, count, "gradient");
    if (is_short(grads, count, kShortNorm)) return short_clip(grads, count, nullptr, -1.0, norm, s);
    check_workspace(ws, ws_len, workspace_of(count));
    const uint32_t sums = square_sums(grads, count, vectors_per_chunk(grads, count), ws, s);
    scalars(sums, nullptr, clip_options(-1.0), nullptr, norm, ws, s);
}

void clip_gradients_device(const ArcqmlTensor *grads, size_t count, double max_norm,
                           const double *given, double *norm, double *ws, size_t ws_len,
                           cudaStream_t s) {
    check_tensors(grads, count, "gradient");
    if (!std::isfinite(max_norm) || max_norm < 0.0)
        fail("the maximum norm must be finite and not negative");
    if (is_short(grads, count, kShortClip)) return short_clip(grads, count, given, max_norm, norm, s);
    check_workspace(ws, ws_len, workspace_of(count));
    const uint32_t per = vectors_per_chunk(grads, count);
    const auto o = clip_options(max_norm);
    for_table_size(grads, count, [&](auto capacity) {
        constexpr uint32_t CAP = capacity;
        const auto clip = [&](const TensorTable<CAP> &t, const Scalars *sc, double bytes) {
            if (t.count)
                launch<k_clip<CAP>>(t.first[t.count], true, 2.0 * bytes, s,
                                    "clip kernel launch", t, sc);
        };
        if (count <= CAP) {  // one table for the norm and the scaling
            for_tensor_tables<CAP>(grads, count, per, [&](const TensorTable<CAP> &t, double bytes) {
                const uint32_t sums =
                    given ? 0 : square_sums(t, bytes, ws + kScalarDoubles, s);
                clip(t, scalars(sums, given, o, nullptr, norm, ws, s), bytes);
            });
            return;
        }
        const uint32_t sums = given ? 0 : square_sums(grads, count, per, ws, s);
        const Scalars *sc = scalars(sums, given, o, nullptr, norm, ws, s);
        for_tensor_tables<CAP>(grads, count, per, [&](const TensorTable<CAP> &t, double bytes) {
            clip(t, sc, bytes);
        });
    });
}

void adam_step_device(const ArcqmlTensor *params, const ArcqmlTensor *grads,
                      const ArcqmlTensor *m, const ArcqmlTensor *v, const ArcqmlTensor *copies,
                      size_t count, int64_t *step, const ArcqmlAdamOptions &o,
                      const double *given, double *norm, double *ws, size_t ws_len,
                      cudaStream_t s) {
    check_tensors(params, count, "parameter");
    check_tensors(grads, count, "gradient");
    check_tensors(m, count, "first moment");
    check_tensors(v, count, "second moment");
    if (copies) check_tensors(copies, count, "copy");
    if (!std::isfinite(o.learning_rate) || !(o.beta1 >= 0.0 && o.beta1 < 1.0) ||
        !(o.beta2 >= 0.0 && o.beta2 < 1.0) || !std::isfinite(o.epsilon) || o.epsilon < 0.0 ||
        !std::isfinite(o.weight_decay))
        fail("invalid Adam hyperparameters (finite lr and weight decay, 0 <= beta < 1, eps >= 0)");
    if (!std::isfinite(o.max_norm)) fail("the maximum norm must be finite");
    if (o.reserved != 0 || (o.decoupled != 0 && o.decoupled != 1)) fail("invalid Adam options");
    const bool one = is_short(params, count, kShortMoments, true);
    if (!one) check_workspace(ws, ws_len, workspace_of(count));
    for (size_t i = 0; i < count; ++i) {
        const uint32_t pt = params[i].dtype, wide = pt == ARCQML_F64 ? ARCQML_F64 : ARCQML_F32;
        const uint64_t n = params[i].length;
        if (pt == ARCQML_NO_TENSOR) fail_at("parameter", i, "is missing");
        if (grads[i].dtype == ARCQML_NO_TENSOR) continue;
        if (grads[i].length != n) fail_at("gradient", i, "differs in length from its parameter");
        if ((pt == ARCQML_F64) != (grads[i].dtype == ARCQML_F64))
            fail_at("gradient", i, "is f64 and its parameter is not, or the other way round");
        if (m[i].length != n || m[i].dtype != wide)
            fail_at("first moment", i, "differs in length or type from what its parameter takes");
        if (v[i].length != n || v[i].dtype != wide)
            fail_at("second moment", i, "differs in length or type from what its parameter takes");
        if (!copies || copies[i].dtype == ARCQML_NO_TENSOR) continue;
        if (pt != ARCQML_F32 || (copies[i].dtype != ARCQML_BF16 && copies[i].dtype != ARCQML_F16))
            fail_at("copy", i, "is not a 16-bit copy of an f32 parameter");
        if (copies[i].length != n) fail_at("copy", i, "differs in length from its parameter");
    }
    const bool clips = o.max_norm >= 0.0;
    if (!clips) given = nullptr;
    if (!clips) norm = nullptr;
    const AdamLists lists{params, grads, m, v, copies, count};
    if (one) {
        bool launched = false;
        const auto run = [&](const AdamTable<kShortTensors> &t, double bytes) {
            launch_cluster<k_short_adam>(t.first[t.count], bytes, s, "Adam kernel launch", t, o, step,
                                         given, norm);
            launched = true;
        };
        for_adam_tables<kShortTensors>(lists, kShortGroups, run);
        if (!launched) {  // nothing to update: the step counts all the same
            AdamTable<kShortTensors> none;
            none.count = none.first[0] = 0;
            run(none, 0.0);
        }
        return;
    }
    const uint32_t sums =
        clips && !given ? square_sums(grads, count, vectors_per_chunk(grads, count), ws, s) : 0;
    const Scalars *sc = scalars(sums, given, o, step, norm, ws, s);
    uint64_t groups = 0;
    for (size_t i = 0; i < count; ++i) groups += params[i].length / group_size(params[i]);
    const uint32_t per = chunk_size(groups, kMaxBlocks);
    for_table_size(params, count, [&](auto capacity) {
        constexpr uint32_t CAP = capacity < kSomeTensors ? uint32_t(capacity) : kSomeTensors;
        for_adam_tables<CAP>(lists, per, [&](const AdamTable<CAP> &t, double bytes) {
            launch<k_adam<CAP>>(t.first[t.count], true, bytes, s, "Adam kernel launch", t,
                                o.decoupled != 0, sc);
        });
    });
}

}  // namespace arcqml
