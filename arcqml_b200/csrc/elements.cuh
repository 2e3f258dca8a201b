// elements.cuh — element types of device tensors: conversion, and vectors of them as one access moves
// them (embedding.cu, muon.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "../../include/arcqml_runtime_v2.h"

namespace arcqml {

// The type in memory, and the type of the arithmetic on it.
template <uint32_t DTYPE> struct ElementOf;
template <> struct ElementOf<ARCQML_F64> {
    using type = double;
    using wide = double;
};
template <> struct ElementOf<ARCQML_F32> {
    using type = float;
    using wide = float;
};
template <> struct ElementOf<ARCQML_BF16> {
    using type = __nv_bfloat16;
    using wide = float;
};
template <> struct ElementOf<ARCQML_F16> {
    using type = __half;
    using wide = float;
};
template <uint32_t DTYPE> using Element = typename ElementOf<DTYPE>::type;
template <uint32_t DTYPE> using WideElement = typename ElementOf<DTYPE>::wide;

inline uint32_t bytes_of_element(uint32_t dtype) {
    return dtype == ARCQML_F64 ? 8 : dtype == ARCQML_F32 ? 4 : 2;
}

__device__ __forceinline__ double to_wide(double x) { return x; }
__device__ __forceinline__ float to_wide(float x) { return x; }
__device__ __forceinline__ float to_wide(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_wide(__half x) { return __half2float(x); }
template <class T> __device__ __forceinline__ T to_element(double x);
template <> __device__ __forceinline__ double to_element<double>(double x) { return x; }
template <> __device__ __forceinline__ float to_element<float>(double x) { return float(x); }
template <class T> __device__ __forceinline__ T to_element(float x);
template <> __device__ __forceinline__ float to_element<float>(float x) { return x; }
template <> __device__ __forceinline__ double to_element<double>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 to_element<__nv_bfloat16>(float x) {
    return __float2bfloat16_rn(x);
}
template <> __device__ __forceinline__ __half to_element<__half>(float x) { return __float2half_rn(x); }

// N elements that are loaded and stored as one access of N * sizeof(T) bytes (2, 4, 8 or 16).
template <class T, int N> struct alignas(sizeof(T) * N) VectorOf {
    T x[N];
};

template <class T, int N> __device__ __forceinline__ VectorOf<T, N> load_vector(const void *p) {
    constexpr int BYTES = sizeof(T) * N;
    VectorOf<T, N> v;
    if constexpr (BYTES == 16) *reinterpret_cast<uint4 *>(&v) = *static_cast<const uint4 *>(p);
    else if constexpr (BYTES == 8) *reinterpret_cast<uint2 *>(&v) = *static_cast<const uint2 *>(p);
    else if constexpr (BYTES == 4) *reinterpret_cast<uint32_t *>(&v) = *static_cast<const uint32_t *>(p);
    else *reinterpret_cast<uint16_t *>(&v) = *static_cast<const uint16_t *>(p);
    return v;
}

template <class T, int N> __device__ __forceinline__ void store_vector(void *p, const VectorOf<T, N> &v) {
    constexpr int BYTES = sizeof(T) * N;
    if constexpr (BYTES == 16) *static_cast<uint4 *>(p) = *reinterpret_cast<const uint4 *>(&v);
    else if constexpr (BYTES == 8) *static_cast<uint2 *>(p) = *reinterpret_cast<const uint2 *>(&v);
    else if constexpr (BYTES == 4) *static_cast<uint32_t *>(p) = *reinterpret_cast<const uint32_t *>(&v);
    else *static_cast<uint16_t *>(p) = *reinterpret_cast<const uint16_t *>(&v);
}

// N elements as the words that one access moves. 16-bit elements stay in pairs until they are used: a register
// each would double those of a load in flight.
template <class T, int N> struct Packed {
    using W = decltype(to_wide(T()));
    static constexpr int BYTES = sizeof(T) * N, WORDS = BYTES < 4 ? 1 : BYTES / 4; // in memory; here 4 at least
    uint32_t w[WORDS];
    __device__ __forceinline__ W wide(int e) const {
        if constexpr (sizeof(T) == 8) return __hiloint2double(int(w[2 * e + 1]), int(w[2 * e]));
        else if constexpr (sizeof(T) == 4) return __uint_as_float(w[e]);
        else if constexpr (sizeof(T) == 2 && __is_same(T, __nv_bfloat16))
            return __uint_as_float(e & 1 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
        else return __half2float(__ushort_as_half(uint16_t(e & 1 ? w[e / 2] >> 16 : w[e / 2] & 0xffffu)));
    }
    // 16-bit elements in pairs: converted one by one and put together, they bound a copy of 2 KB rows
    __device__ __forceinline__ void pack(const W (&x)[N]) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
            if constexpr (sizeof(T) == 8) {
                w[2 * e] = uint32_t(__double2loint(x[e]));
                w[2 * e + 1] = uint32_t(__double2hiint(x[e]));
            } else if constexpr (sizeof(T) == 4) {
                w[e] = __float_as_uint(x[e]);
            } else if constexpr (N == 1) {
                const T y = to_element<T>(x[0]);
                w[0] = *reinterpret_cast<const uint16_t *>(&y);
            } else if constexpr (__is_same(T, __nv_bfloat16)) {
                if (e & 1) {
                    const __nv_bfloat162 y = __floats2bfloat162_rn(x[e - 1], x[e]);
                    w[e / 2] = *reinterpret_cast<const uint32_t *>(&y);
                }
            } else if (e & 1) {
                const __half2 y = __floats2half2_rn(x[e - 1], x[e]);
                w[e / 2] = *reinterpret_cast<const uint32_t *>(&y);
            }
        }
    }
    __device__ __forceinline__ void fill(uint32_t word) {
#pragma unroll
        for (int i = 0; i < WORDS; ++i) w[i] = word;
    }
    __device__ __forceinline__ void load(const void *p) {
        if constexpr (BYTES == 16) {
            const uint4 v = *static_cast<const uint4 *>(p);
            w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
        } else if constexpr (BYTES == 8) {
            const uint2 v = *static_cast<const uint2 *>(p);
            w[0] = v.x, w[1] = v.y;
        } else if constexpr (BYTES == 4) {
            w[0] = *static_cast<const uint32_t *>(p);
        } else {
            w[0] = *static_cast<const uint16_t *>(p);
        }
    }
    __device__ __forceinline__ void store(void *p) const {
        if constexpr (BYTES == 16) *static_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
        else if constexpr (BYTES == 8) *static_cast<uint2 *>(p) = make_uint2(w[0], w[1]);
        else if constexpr (BYTES == 4) *static_cast<uint32_t *>(p) = w[0];
        else *static_cast<uint16_t *>(p) = uint16_t(w[0]);
    }
};

}  // namespace arcqml
