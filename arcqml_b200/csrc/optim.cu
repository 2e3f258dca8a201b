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
constexpr uint32_t kChunk = 8192;        // elements

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
    uint8_t pt[kMaxTensors], gt[kMaxTensors], ct[kMaxTensors];
    uint32_t count;
};
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

__device__ __forceinline__ float load_f32(const void *p, uint64_t i, uint32_t dtype) {
    if (dtype == ARCQML_F32) return static_cast<const float *>(p)[i];
    if (dtype == ARCQML_BF16) return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
    return __half2float(static_cast<const __half *>(p)[i]);
}

__device__ __forceinline__ void store_f32(void *p, uint64_t i, uint32_t dtype, float x) {
    if (dtype == ARCQML_F32) static_cast<float *>(p)[i] = x;
    else if (dtype == ARCQML_BF16) static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(x);
    else static_cast<__half *>(p)[i] = __float2half_rn(x);
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

__global__ void __launch_bounds__(kOT)
    k_square_sums(const __grid_constant__ TensorTable t, double *__restrict__ sums) {
    double acc = 0.0;
    for (uint32_t c = blockIdx.x; c < t.first[t.count]; c += gridDim.x) {
        const uint32_t k = tensor_of(t, c), dtype = t.dtype[k];
        const uint64_t i0 = uint64_t(c - t.first[k]) * kChunk;
        const uint64_t i1 = min(i0 + kChunk, t.length[k]);
        const void *g = t.data[k];
        for (uint64_t i = i0 + threadIdx.x; i < i1; i += kOT) {
            const double x = dtype == ARCQML_F64 ? static_cast<const double *>(g)[i]
                                                 : double(load_f32(g, i, dtype));
            acc = fma(x, x, acc);
        }
    }
    acc = o_block_sum(acc);
    if (threadIdx.x == 0) sums[blockIdx.x] = acc;
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

__global__ void __launch_bounds__(kOT)
    k_clip(const __grid_constant__ TensorTable t, const Scalars *__restrict__ sc) {
    const double factor = sc->factor;
    if (factor == 1.0) return;
    const float f = float(factor);
    for (uint32_t c = blockIdx.x; c < t.first[t.count]; c += gridDim.x) {
        const uint32_t k = tensor_of(t, c), dtype = t.dtype[k];
        const uint64_t i0 = uint64_t(c - t.first[k]) * kChunk;
        const uint64_t i1 = min(i0 + kChunk, t.length[k]);
        void *g = t.data[k];
        for (uint64_t i = i0 + threadIdx.x; i < i1; i += kOT) {
            if (dtype == ARCQML_F64) static_cast<double *>(g)[i] *= factor;
            else store_f32(g, i, dtype, load_f32(g, i, dtype) * f);
        }
    }
}

struct AdamScalars64 {
    double lr, b1, b2, nb1, nb2, eps, wd, down;
};

// f64, every operation rounded on its own, in the order of the host's update and of the optimizer
// loop (crates/arcqml-optim/src/adam.rs:190-240), so the three agree to the bias corrections.
__device__ __forceinline__ void adam64(double &p, double &m, double &v, double g, double factor,
                                       const AdamScalars64 &h, bool decoupled, double bc1,
                                       double bc2) {
    double a = __dmul_rn(g, factor);
    if (!decoupled) a = __dadd_rn(a, __dmul_rn(h.wd, p));
    m = __dadd_rn(__dmul_rn(h.b1, m), __dmul_rn(h.nb1, a));
    v = __dadd_rn(__dmul_rn(h.b2, v), __dmul_rn(__dmul_rn(h.nb2, a), a));
    const double mh = __ddiv_rn(m, bc1), vh = __ddiv_rn(v, bc2);
    if (decoupled) p = __dmul_rn(p, h.down);
    p = __dsub_rn(p, __ddiv_rn(__dmul_rn(h.lr, mh), __dadd_rn(__dsqrt_rn(vh), h.eps)));
}

struct AdamScalars32 {
    float b1, b2, nb1, nb2, eps, wd, down, rate, root, factor;
};

// f32: rate = lr / (1 - beta1^t) and root = 1 / (1 - beta2^t) are formed in f64 and rounded once.
__device__ __forceinline__ void adam32(float &p, float &m, float &v, float g,
                                       const AdamScalars32 &h, bool decoupled) {
    float a = g * h.factor;
    if (!decoupled) a = fmaf(h.wd, p, a);
    m = fmaf(h.b1, m, h.nb1 * a);
    v = fmaf(h.b2, v, h.nb2 * a * a);
    const float u = m / (sqrtf(v * h.root) + h.eps);
    if (decoupled) p *= h.down;
    p = fmaf(-h.rate, u, p);
}

__global__ void __launch_bounds__(kOT)
    k_adam(const __grid_constant__ AdamTable t, const __grid_constant__ ArcqmlAdamOptions o,
           const Scalars *__restrict__ sc) {
    const double factor = sc->factor, bc1 = sc->bc1, bc2 = sc->bc2;
    const bool decoupled = o.decoupled != 0;
    const double lr = o.learning_rate, down = 1.0 - lr * o.weight_decay;
    const AdamScalars64 h{lr, o.beta1, o.beta2, 1.0 - o.beta1, 1.0 - o.beta2, o.epsilon,
                          o.weight_decay, down};
    const AdamScalars32 hf{float(h.b1), float(h.b2), float(h.nb1), float(h.nb2), float(h.eps),
                           float(h.wd), float(down), float(lr / bc1), float(1.0 / bc2),
                           float(factor)};
    for (uint32_t c = blockIdx.x; c < t.first[t.count]; c += gridDim.x) {
        const uint32_t k = tensor_of(t, c), pt = t.pt[k], gt = t.gt[k];
        const uint64_t i0 = uint64_t(c - t.first[k]) * kChunk;
        const uint64_t i1 = min(i0 + kChunk, t.length[k]);
        for (uint64_t i = i0 + threadIdx.x; i < i1; i += kOT) {
            if (pt == ARCQML_F64) {
                double p = static_cast<double *>(t.p[k])[i], m = static_cast<double *>(t.m[k])[i],
                       v = static_cast<double *>(t.v[k])[i];
                adam64(p, m, v, static_cast<const double *>(t.g[k])[i], factor, h, decoupled, bc1,
                       bc2);
                static_cast<double *>(t.p[k])[i] = p;
                static_cast<double *>(t.m[k])[i] = m;
                static_cast<double *>(t.v[k])[i] = v;
            } else {
                float p = load_f32(t.p[k], i, pt), m = static_cast<float *>(t.m[k])[i],
                      v = static_cast<float *>(t.v[k])[i];
                adam32(p, m, v, load_f32(t.g[k], i, gt), hf, decoupled);
                store_f32(t.p[k], i, pt, p);
                static_cast<float *>(t.m[k])[i] = m;
                static_cast<float *>(t.v[k])[i] = v;
                if (t.ct[k] != ARCQML_NO_TENSOR) store_f32(t.copy[k], i, t.ct[k], p);
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

uint64_t chunks_of(uint64_t length) { return (length + kChunk - 1) / kChunk; }

// The whole list is checked before anything is launched. Chunks are counted in 32 bits.
void check_tensors(const ArcqmlTensor *list, size_t count, const char *name) {
    if (count && !list) fail(std::string(name) + " list is null");
    uint64_t chunks = 0;
    for (size_t i = 0; i < count; ++i)
        if (check_tensor(list[i], name, i)) chunks += chunks_of(list[i].length);
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
        const uint64_t n = chunks_of(list[i].length);
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
    auto flush = [&] {
        if (!t.count) return;
        t.first[t.count] = uint32_t(chunks);
        const ProfToken tok = prof_begin(PROF_OTHER, s);
        k_adam<<<blocks_for(chunks), kOT, 0, s>>>(t, o, sc);
        prof_end(tok, s, bytes);
        check_cuda(cudaGetLastError(), "Adam kernel launch");
        t.count = 0;
        chunks = 0;
        bytes = 0.0;
    };
    for (size_t i = 0; i < count; ++i) {
        if (!present(params[i]) || grads[i].dtype == ARCQML_NO_TENSOR) continue;
        const uint64_t n = chunks_of(params[i].length);
        if (t.count == kMaxTensors) flush();
        const uint32_t k = t.count++;
        const uint32_t ct = copies ? copies[i].dtype : uint32_t(ARCQML_NO_TENSOR);
        t.p[k] = params[i].data;
        t.g[k] = grads[i].data;
        t.m[k] = m[i].data;
        t.v[k] = v[i].data;
        t.copy[k] = ct == ARCQML_NO_TENSOR ? nullptr : copies[i].data;
        t.length[k] = params[i].length;
        t.first[k] = uint32_t(chunks);
        t.pt[k] = uint8_t(params[i].dtype);
        t.gt[k] = uint8_t(grads[i].dtype);
        t.ct[k] = uint8_t(ct);
        chunks += n;
        bytes += double(params[i].length) *
                 (2.0 * element_size(params[i].dtype) + element_size(grads[i].dtype) +
                  4.0 * element_size(m[i].dtype) +
                  (ct == ARCQML_NO_TENSOR ? 0.0 : element_size(ct)));
    }
    flush();
}

}  // namespace arcqml
