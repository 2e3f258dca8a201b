// optim.cu — training over many device tensors: the global norm of a list of gradients, clipping
// by that norm, and the Adam step with the clip factor folded in.
//
// All of it is bound by HBM at real sizes (2 to 14 operations per element against 2 to 56 bytes)
// and by launches at small ones. One launch covers a whole list: the tensors' pointers and lengths
// travel as a kernel parameter, every tensor is cut into chunks of elements, and the blocks take the
// chunks of the list in turn. No call reads anything back: the norm, the clip factor and the bias
// corrections pass between the launches in device scratch that the caller gives, so nothing is
// shared between calls and no sum depends on the order in which blocks finish.
//
//   k_square_sums   per block the f64 sum of squares of its chunks
//   k_scalars       one block: the sums in order -> norm, clip factor, step count, bias corrections
//   k_clip, k_adam  the list scaled, or updated
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <sstream>
#include <string>

#include "launch.h"
#include "optim.h"
#include "profile.h"

namespace arcqml {
namespace {

constexpr int kOT = 256;                 // threads per block
constexpr uint32_t kMaxBlocks = 148 * 8; // blocks of one launch
constexpr uint32_t kMaxTensors = 512;    // tensors of one launch
constexpr uint32_t kVectors = 2048;      // 16-byte vectors of one chunk (k_square_sums, k_clip)
constexpr uint32_t kGroups = 2048;       // groups of 4 elements of one chunk (k_adam)

// What k_scalars leaves for the launches behind it (the head of the scratch).
struct Scalars {
    double norm, factor, bc1, bc2;
};
constexpr size_t kScalarDoubles = sizeof(Scalars) / sizeof(double);

// The tensors of one launch. first[i]: the number of chunks before tensor i; first[count]: of all.
struct TensorTable {
    void *data[kMaxTensors];
    uint64_t length[kMaxTensors];
    uint32_t first[kMaxTensors + 1];
    uint8_t dtype[kMaxTensors];
    uint32_t count;
};

struct AdamTable {
    void *p[kMaxTensors], *m[kMaxTensors], *v[kMaxTensors], *copy[kMaxTensors];
    const void *g[kMaxTensors];
    uint64_t length[kMaxTensors];
    uint32_t first[kMaxTensors + 1];
    uint8_t types[kMaxTensors];   // of the parameter, the gradient (<< 2) and the copy (<< 4)
    uint8_t aligned[kMaxTensors]; // kAligned*: arrays whose groups start on their own size
    uint8_t head[kMaxTensors];    // elements before the first group
    uint32_t count;
};
enum { kAlignedG = 1, kAlignedM = 2, kAlignedV = 4, kAlignedCopy = 8, kHasCopy = 16 };
static_assert(sizeof(AdamTable) < 32000, "kernel parameters hold 32764 bytes");

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
template <uint32_t DTYPE, int N> struct alignas(sizeof(typename Elem<DTYPE>::type) * N >= 16 ? 16 : 8) Words {
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

// Sum over the block in a fixed order; valid in thread 0.
__device__ __forceinline__ double o_block_sum(double v) {
    __shared__ double red[kOT / 32];
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    double r = 0.0;
    if (threadIdx.x == 0)
        for (int w = 0; w < kOT / 32; ++w) r += red[w];
    return r;
}

// Squares of one chunk, added to acc in f64: the squares of f32 values leave the range of f32, and a
// norm that comes back in f64 is wanted to its precision.
template <uint32_t DTYPE>
__device__ __forceinline__ void square_chunk(const void *data, uint64_t length, uint32_t chunk,
                                             double (&acc)[4]) {
    using T = typename Elem<DTYPE>::type;
    using W = typename Elem<DTYPE>::wide;
    constexpr int N = 16 / sizeof(T), U = 8;
    const T *p = static_cast<const T *>(data);
    const uint32_t head = head_of(p, length);
    const uint64_t vectors = (length - head) / N;
    const auto *q = reinterpret_cast<const Words<DTYPE, N> *>(p + head);
    const uint64_t v0 = uint64_t(chunk) * kVectors;
    const uint32_t n = uint32_t(min(uint64_t(kVectors), vectors - min(v0, vectors)));
    const auto add = [&](const Words<DTYPE, N> &raw) {
        W x[N];
        raw.unpack(x);
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const double d = double(x[j]);
            acc[j % 4] = fma(d, d, acc[j % 4]);
        }
    };
    uint32_t v = threadIdx.x;
    for (; v + (U - 1) * kOT < n; v += U * kOT) {
        Words<DTYPE, N> x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) x[u] = q[v0 + v + u * kOT];
#pragma unroll
        for (int u = 0; u < U; ++u) add(x[u]);
    }
    for (; v < n; v += kOT) add(q[v0 + v]);
    // the elements before the first vector (chunk 0) and behind the last one (the last chunk)
    if (chunk == 0 && threadIdx.x < head) {
        const double d = double(widen(p[threadIdx.x]));
        acc[0] = fma(d, d, acc[0]);
    }
    const uint64_t done = head + vectors * N;
    if (v0 + kVectors >= vectors && threadIdx.x < length - done) {
        const double d = double(widen(p[done + threadIdx.x]));
        acc[1] = fma(d, d, acc[1]);
    }
}

__global__ void __launch_bounds__(kOT)
    k_square_sums(const __grid_constant__ TensorTable t, double *__restrict__ sums) {
    double acc[4] = {0.0, 0.0, 0.0, 0.0};
    for (uint32_t c = blockIdx.x; c < t.first[t.count]; c += gridDim.x) {
        const uint32_t k = tensor_of(t, c), chunk = c - t.first[k];
        const void *g = t.data[k];
        const uint64_t n = t.length[k];
        switch (t.dtype[k]) {
        case ARCQML_F64: square_chunk<ARCQML_F64>(g, n, chunk, acc); break;
        case ARCQML_F32: square_chunk<ARCQML_F32>(g, n, chunk, acc); break;
        case ARCQML_BF16: square_chunk<ARCQML_BF16>(g, n, chunk, acc); break;
        default: square_chunk<ARCQML_F16>(g, n, chunk, acc);
        }
    }
    const double sum = o_block_sum((acc[0] + acc[1]) + (acc[2] + acc[3]));
    if (threadIdx.x == 0) sums[blockIdx.x] = sum;
}

// One block. given != null: n = *given; else the root of the count sums. factor: 1 without
// clipping (max_norm < 0); a NaN norm stays a NaN factor. step != null: one more step is counted.
__global__ void __launch_bounds__(kOT)
    k_scalars(const double *__restrict__ sums, uint32_t count, const double *given,
              double max_norm, int64_t *step, double beta1, double beta2, double *norm,
              Scalars *out) {
    double acc = 0.0;
    for (uint32_t i = threadIdx.x; i < count; i += kOT) acc += sums[i];
    acc = o_block_sum(acc);
    if (threadIdx.x != 0) return;
    const double n = given ? *given : sqrt(acc);
    if (norm) *norm = n;
    double factor = 1.0;
    if (max_norm >= 0.0) {
        factor = max_norm / (n + 1e-6);
        if (factor > 1.0) factor = 1.0;
    }
    Scalars r{n, factor, 1.0, 1.0};
    if (step) {
        const int64_t now = *step + 1;
        *step = now;
        r.bc1 = 1.0 - pow(beta1, double(now));
        r.bc2 = 1.0 - pow(beta2, double(now));
    }
    *out = r;
}

// One chunk times the factor: the product in the type of the arithmetic (f32 for 16-bit types, the
// factor rounded to it), rounded once to the element's type.
template <uint32_t DTYPE>
__device__ __forceinline__ void clip_chunk(void *data, uint64_t length, uint32_t chunk,
                                           double factor) {
    using T = typename Elem<DTYPE>::type;
    using W = typename Elem<DTYPE>::wide;
    constexpr int N = 16 / sizeof(T), U = 4;
    const W f = W(factor);
    T *p = static_cast<T *>(data);
    const uint32_t head = head_of(p, length);
    const uint64_t vectors = (length - head) / N;
    auto *q = reinterpret_cast<Words<DTYPE, N> *>(p + head);
    const uint64_t v0 = uint64_t(chunk) * kVectors;
    const uint32_t n = uint32_t(min(uint64_t(kVectors), vectors - min(v0, vectors)));
    const auto scale = [&](Words<DTYPE, N> &raw) {
        W x[N];
        raw.unpack(x);
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] *= f;
        raw.pack(x);
    };
    uint32_t v = threadIdx.x;
    for (; v + (U - 1) * kOT < n; v += U * kOT) {
        Words<DTYPE, N> x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) x[u] = q[v0 + v + u * kOT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            scale(x[u]);
            q[v0 + v + u * kOT] = x[u];
        }
    }
    for (; v < n; v += kOT) {
        Words<DTYPE, N> x = q[v0 + v];
        scale(x);
        q[v0 + v] = x;
    }
    if (chunk == 0 && threadIdx.x < head) narrow(widen(p[threadIdx.x]) * f, p[threadIdx.x]);
    const uint64_t done = head + vectors * N;
    if (v0 + kVectors >= vectors && threadIdx.x < length - done)
        narrow(widen(p[done + threadIdx.x]) * f, p[done + threadIdx.x]);
}

__global__ void __launch_bounds__(kOT, 4)
    k_clip(const __grid_constant__ TensorTable t, const Scalars *__restrict__ sc) {
    const double factor = sc->factor;
    if (factor == 1.0) return;
    for (uint32_t c = blockIdx.x; c < t.first[t.count]; c += gridDim.x) {
        const uint32_t k = tensor_of(t, c), chunk = c - t.first[k];
        void *g = t.data[k];
        const uint64_t n = t.length[k];
        switch (t.dtype[k]) {
        case ARCQML_F64: clip_chunk<ARCQML_F64>(g, n, chunk, factor); break;
        case ARCQML_F32: clip_chunk<ARCQML_F32>(g, n, chunk, factor); break;
        case ARCQML_BF16: clip_chunk<ARCQML_BF16>(g, n, chunk, factor); break;
        default: clip_chunk<ARCQML_F16>(g, n, chunk, factor);
        }
    }
}

struct AdamScalars64 {
    double lr, b1, b2, nb1, nb2, eps, wd, down, bc1, bc2, factor;
};

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

struct AdamScalars32 {
    float b1, b2, nb1, nb2, eps, wd, down, rate, root, factor;
};

// f32: rate = lr / (1 - beta1^t) and root = 1 / (1 - beta2^t) are formed in f64 and rounded once.
__device__ __forceinline__ void adam_update(float &p, float &m, float &v, float g,
                                            const AdamScalars32 &h, bool decoupled) {
    float a = g * h.factor;
    if (!decoupled) a = fmaf(h.wd, p, a);
    m = fmaf(h.b1, m, h.nb1 * a);
    v = fmaf(h.b2, v, h.nb2 * a * a);
    const float u = m / (sqrtf(v * h.root) + h.eps);
    if (decoupled) p *= h.down;
    p = fmaf(-h.rate, u, p);
}

// A group (4 elements from element e on) of an array: one access, or one per element.
template <uint32_t DTYPE>
__device__ __forceinline__ Words<DTYPE, 4> load4(const void *p, uint64_t e, bool aligned) {
    using T = typename Elem<DTYPE>::type;
    const T *q = static_cast<const T *>(p) + e;
    if (aligned) return *reinterpret_cast<const Words<DTYPE, 4> *>(q);
    typename Elem<DTYPE>::wide x[4];
    for (int j = 0; j < 4; ++j) x[j] = widen(q[j]);
    Words<DTYPE, 4> raw;
    raw.pack(x);
    return raw;
}
template <uint32_t DTYPE>
__device__ __forceinline__ void store4(void *p, uint64_t e, bool aligned,
                                       const typename Elem<DTYPE>::wide (&x)[4]) {
    using T = typename Elem<DTYPE>::type;
    T *q = static_cast<T *>(p) + e;
    if (aligned) {
        Words<DTYPE, 4> raw;
        raw.pack(x);
        *reinterpret_cast<Words<DTYPE, 4> *>(q) = raw;
    } else {
        for (int j = 0; j < 4; ++j) narrow(x[j], q[j]);
    }
}

template <uint32_t PT, uint32_t GT, class H>
__device__ __forceinline__ void adam_chunk(const AdamTable &t, uint32_t k, uint32_t chunk,
                                           const H &h, bool decoupled) {
    using P = typename Elem<PT>::type;
    using G = typename Elem<GT>::type;
    using W = typename Elem<PT>::wide;
    constexpr uint32_t WT = sizeof(W) == 8 ? ARCQML_F64 : ARCQML_F32;
    constexpr int U = sizeof(W) == 8 ? 1 : 2;
    const uint64_t length = t.length[k];
    const uint32_t head = t.head[k], aligned = t.aligned[k], ct = t.types[k] >> 4;
    void *p = t.p[k], *m = t.m[k], *v = t.v[k], *copy = t.copy[k];
    const void *g = t.g[k];
    const uint64_t groups = (length - head) / 4;
    const uint64_t i0 = uint64_t(chunk) * kGroups;
    const uint32_t n = uint32_t(min(uint64_t(kGroups), groups - min(i0, groups)));
    const uint64_t e0 = head + 4 * i0;
    const auto update = [&](uint64_t e, const Words<PT, 4> &rp, const Words<GT, 4> &rg,
                            const Words<WT, 4> &rm, const Words<WT, 4> &rv) {
        W x[4], y[4], mm[4], vv[4];
        rp.unpack(x);
        rg.unpack(y);
        rm.unpack(mm);
        rv.unpack(vv);
#pragma unroll
        for (int j = 0; j < 4; ++j) adam_update(x[j], mm[j], vv[j], y[j], h, decoupled);
        store4<PT>(p, e, true, x);
        store4<WT>(m, e, aligned & kAlignedM, mm);
        store4<WT>(v, e, aligned & kAlignedV, vv);
        if constexpr (PT == ARCQML_F32) {
            if (aligned & kHasCopy) {
                if (ct == ARCQML_BF16) store4<ARCQML_BF16>(copy, e, aligned & kAlignedCopy, x);
                else store4<ARCQML_F16>(copy, e, aligned & kAlignedCopy, x);
            }
        }
    };
    uint32_t i = threadIdx.x;
    for (; i + (U - 1) * kOT < n; i += U * kOT) {
        Words<PT, 4> xp[U];
        Words<GT, 4> xg[U];
        Words<WT, 4> xm[U], xv[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint64_t e = e0 + 4 * (i + u * kOT);
            xp[u] = load4<PT>(p, e, true);
            xg[u] = load4<GT>(g, e, aligned & kAlignedG);
            xm[u] = load4<WT>(m, e, aligned & kAlignedM);
            xv[u] = load4<WT>(v, e, aligned & kAlignedV);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) update(e0 + 4 * (i + u * kOT), xp[u], xg[u], xm[u], xv[u]);
    }
    if constexpr (U > 1) {
        for (; i < n; i += kOT) {
            const uint64_t e = e0 + 4 * i;
            update(e, load4<PT>(p, e, true), load4<GT>(g, e, aligned & kAlignedG),
                   load4<WT>(m, e, aligned & kAlignedM), load4<WT>(v, e, aligned & kAlignedV));
        }
    }
    // the elements before the first group (chunk 0) and behind the last one (the last chunk)
    const uint64_t done = head + groups * 4;
    const uint32_t tail = i0 + kGroups >= groups ? uint32_t(length - done) : 0;
    const uint32_t first = chunk == 0 ? head : 0;
    if (threadIdx.x < first + tail) {
        const uint64_t e = threadIdx.x < first ? threadIdx.x : done + threadIdx.x - first;
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

template <uint32_t PT>
__device__ __forceinline__ void adam_chunk_of(const AdamTable &t, uint32_t k, uint32_t chunk,
                                              const AdamScalars32 &h, bool decoupled) {
    switch (t.types[k] >> 2 & 3) {
    case ARCQML_F32: adam_chunk<PT, ARCQML_F32>(t, k, chunk, h, decoupled); break;
    case ARCQML_BF16: adam_chunk<PT, ARCQML_BF16>(t, k, chunk, h, decoupled); break;
    default: adam_chunk<PT, ARCQML_F16>(t, k, chunk, h, decoupled);
    }
}

// The f64 tensors of a list and the others go to launches of their own: the f64 arithmetic
// (two or three divisions and a root per element) takes twice the registers.
template <bool F64>
__global__ void __launch_bounds__(kOT, F64 ? 2 : 4)
    k_adam(const __grid_constant__ AdamTable t, const __grid_constant__ ArcqmlAdamOptions o,
           const Scalars *__restrict__ sc) {
    const double factor = sc->factor, bc1 = sc->bc1, bc2 = sc->bc2;
    const bool decoupled = o.decoupled != 0;
    const double lr = o.learning_rate, down = 1.0 - lr * o.weight_decay;
    const AdamScalars64 h{lr, o.beta1, o.beta2, 1.0 - o.beta1, 1.0 - o.beta2, o.epsilon,
                          o.weight_decay, down, bc1, bc2, factor};
    const AdamScalars32 hf{float(h.b1), float(h.b2), float(h.nb1), float(h.nb2), float(h.eps),
                           float(h.wd), float(down), float(lr / bc1), float(1.0 / bc2),
                           float(factor)};
    for (uint32_t c = blockIdx.x; c < t.first[t.count]; c += gridDim.x) {
        const uint32_t k = tensor_of(t, c), chunk = c - t.first[k];
        if constexpr (F64) {
            adam_chunk<ARCQML_F64, ARCQML_F64>(t, k, chunk, h, decoupled);
        } else {
            switch (t.types[k] & 3) {
            case ARCQML_F32: adam_chunk_of<ARCQML_F32>(t, k, chunk, hf, decoupled); break;
            case ARCQML_BF16: adam_chunk_of<ARCQML_BF16>(t, k, chunk, hf, decoupled); break;
            default: adam_chunk_of<ARCQML_F16>(t, k, chunk, hf, decoupled);
            }
        }
    }
}

// ------------------------------------------------------------------ host side

uint32_t element_size(uint32_t dtype) {
    return dtype == ARCQML_F64 ? 8 : dtype == ARCQML_F32 ? 4 : 2;
}

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

void check_workspace(const double *ws, size_t len, size_t count) {
    if (!ws) fail("workspace is null");
    if (reinterpret_cast<uintptr_t>(ws) % 16) fail("workspace is not aligned to 16 bytes");
    if (len < tensor_workspace(count)) {
        std::ostringstream m;
        m << "workspace of " << len << " doubles is too small for " << count << " tensors: needs "
          << tensor_workspace(count);
        fail(m.str());
    }
}

uint32_t blocks_for(uint64_t chunks) {
    return uint32_t(std::max<uint64_t>(1, std::min<uint64_t>(chunks, kMaxBlocks)));
}

// Chunks of a tensor in k_square_sums and k_clip: at least one, for the elements outside vectors.
uint64_t chunks_of(const ArcqmlTensor &t) {
    const uint32_t size = element_size(t.dtype);
    const uint64_t head = (-reinterpret_cast<uintptr_t>(t.data) & 15) / size;
    const uint64_t vectors = t.length > head ? (t.length - head) / (16 / size) : 0;
    return std::max<uint64_t>(1, (vectors + kVectors - 1) / kVectors);
}

// The whole list is checked before anything is launched. Chunks are counted in 32 bits.
void check_tensors(const ArcqmlTensor *list, size_t count, const char *name) {
    if (count && !list) fail(std::string(name) + " list is null");
    uint64_t chunks = 0;
    for (size_t i = 0; i < count; ++i)
        if (check_tensor(list[i], name, i)) chunks += list[i].length / kVectors + 1;
    if (chunks >> 31) fail(std::string(name) + " list holds too many elements");
}

// Calls launch(table, blocks, bytes) for every launch that the (checked) list takes.
template <class F>
void for_tensor_launches(const ArcqmlTensor *list, size_t count, F &&launch) {
    TensorTable t;
    t.count = 0;
    uint64_t chunks = 0;
    double bytes = 0.0;
    auto flush = [&] {
        if (!t.count) return;
        t.first[t.count] = uint32_t(chunks);
        launch(t, blocks_for(chunks), bytes);
        t.count = 0;
        chunks = 0;
        bytes = 0.0;
    };
    for (size_t i = 0; i < count; ++i) {
        if (!present(list[i])) continue;
        const uint64_t n = chunks_of(list[i]);
        if (t.count == kMaxTensors) flush();
        t.data[t.count] = list[i].data;
        t.length[t.count] = list[i].length;
        t.dtype[t.count] = uint8_t(list[i].dtype);
        t.first[t.count++] = uint32_t(chunks);
        chunks += n;
        bytes += double(list[i].length) * element_size(list[i].dtype);
    }
    flush();
}

// Sums of squares of the list into ws; returns their count.
uint32_t square_sums(const ArcqmlTensor *grads, size_t count, double *ws, cudaStream_t s) {
    uint32_t sums = 0;
    for_tensor_launches(grads, count, [&](const TensorTable &t, uint32_t blocks, double bytes) {
        const ProfToken tok = prof_begin(PROF_OTHER, s);
        k_square_sums<<<blocks, kOT, 0, s>>>(t, ws + kScalarDoubles + sums);
        prof_end(tok, s, bytes);
        check_cuda(cudaGetLastError(), "gradient norm kernel launch");
        sums += blocks;
    });
    return sums;
}

Scalars *scalars(uint32_t sums, const double *given, double max_norm, int64_t *step, double beta1,
                 double beta2, double *norm, double *ws, cudaStream_t s) {
    auto *out = reinterpret_cast<Scalars *>(ws);
    const ProfToken tok = prof_begin(PROF_OTHER, s);
    k_scalars<<<1, kOT, 0, s>>>(ws + kScalarDoubles, sums, given, max_norm, step, beta1, beta2,
                                norm, out);
    prof_end(tok, s, 8.0 * sums);
    check_cuda(cudaGetLastError(), "gradient norm kernel launch");
    return out;
}

}  // namespace

size_t tensor_workspace(size_t num_tensors) {
    return kScalarDoubles + (num_tensors / kMaxTensors + 1) * size_t(kMaxBlocks);
}

void gradient_norm_device(const ArcqmlTensor *grads, size_t count, double *norm, double *ws,
                          size_t ws_len, cudaStream_t s) {
    check_tensors(grads, count, "gradient");
    check_workspace(ws, ws_len, count);
    const uint32_t sums = square_sums(grads, count, ws, s);
    scalars(sums, nullptr, -1.0, nullptr, 0.0, 0.0, norm, ws, s);
}

void clip_gradients_device(const ArcqmlTensor *grads, size_t count, double max_norm,
                           const double *given, double *norm, double *ws, size_t ws_len,
                           cudaStream_t s) {
    check_tensors(grads, count, "gradient");
    if (!std::isfinite(max_norm) || max_norm < 0.0)
        fail("the maximum norm must be finite and not negative");
    check_workspace(ws, ws_len, count);
    const uint32_t sums = given ? 0 : square_sums(grads, count, ws, s);
    const Scalars *sc = scalars(sums, given, max_norm, nullptr, 0.0, 0.0, norm, ws, s);
    for_tensor_launches(grads, count, [&](const TensorTable &t, uint32_t blocks, double bytes) {
        const ProfToken tok = prof_begin(PROF_OTHER, s);
        k_clip<<<blocks, kOT, 0, s>>>(t, sc);
        prof_end(tok, s, 2.0 * bytes);
        check_cuda(cudaGetLastError(), "clip kernel launch");
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
    check_workspace(ws, ws_len, count);
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
    const uint32_t sums = clips && !given ? square_sums(grads, count, ws, s) : 0;
    const Scalars *sc = scalars(sums, clips ? given : nullptr, clips ? o.max_norm : -1.0, step,
                                o.beta1, o.beta2, clips ? norm : nullptr, ws, s);
    AdamTable t;
    t.count = 0;
    uint64_t chunks = 0;
    double bytes = 0.0;
    bool f64 = false;
    auto flush = [&] {
        if (!t.count) return;
        t.first[t.count] = uint32_t(chunks);
        const ProfToken tok = prof_begin(PROF_OTHER, s);
        if (f64) k_adam<true><<<blocks_for(chunks), kOT, 0, s>>>(t, o, sc);
        else k_adam<false><<<blocks_for(chunks), kOT, 0, s>>>(t, o, sc);
        prof_end(tok, s, bytes);
        check_cuda(cudaGetLastError(), "Adam kernel launch");
        t.count = 0;
        chunks = 0;
        bytes = 0.0;
    };
    for (size_t j = 0; j < 2 * count; ++j) {  // the others, then the f64 tensors
        const size_t i = j < count ? j : j - count;
        if (j == count) {
            flush();
            f64 = true;
        }
        if (!present(params[i]) || grads[i].dtype == ARCQML_NO_TENSOR ||
            (params[i].dtype == ARCQML_F64) != f64)
            continue;
        if (t.count == kMaxTensors) flush();
        const uint32_t k = t.count++;
        const uint32_t ct = copies ? copies[i].dtype : uint32_t(ARCQML_NO_TENSOR);
        const bool copy = ct != ARCQML_NO_TENSOR;
        const uint64_t length = params[i].length;
        // groups of 4 elements from the first place on where the parameter's start on their size
        const auto apart = [&](const ArcqmlTensor &x) {
            return (reinterpret_cast<uintptr_t>(x.data) / element_size(x.dtype)) & 3;
        };
        const uint64_t at = apart(params[i]), head = std::min<uint64_t>(-at & 3, length);
        t.p[k] = params[i].data;
        t.g[k] = grads[i].data;
        t.m[k] = m[i].data;
        t.v[k] = v[i].data;
        t.copy[k] = copy ? copies[i].data : nullptr;
        t.length[k] = length;
        t.first[k] = uint32_t(chunks);
        t.types[k] = uint8_t(params[i].dtype | grads[i].dtype << 2 | (copy ? ct << 4 : 0));
        t.aligned[k] = uint8_t((apart(grads[i]) == at ? kAlignedG : 0) |
                               (apart(m[i]) == at ? kAlignedM : 0) |
                               (apart(v[i]) == at ? kAlignedV : 0) |
                               (copy && apart(copies[i]) == at ? kAlignedCopy : 0) |
                               (copy ? kHasCopy : 0));
        t.head[k] = uint8_t(head);
        chunks += std::max<uint64_t>(1, ((length - head) / 4 + kGroups - 1) / kGroups);
        bytes += double(params[i].length) *
                 (2.0 * element_size(params[i].dtype) + element_size(grads[i].dtype) +
                  4.0 * element_size(m[i].dtype) +
                  (ct == ARCQML_NO_TENSOR ? 0.0 : element_size(ct)));
    }
    flush();
}

}  // namespace arcqml
