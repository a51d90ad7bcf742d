// fp32 / bf16 / fp16 element access for the kernels that take all three (groupnorm.hip, relbias.hip, xattn.h).
// Arithmetic is always fp32; a value is rounded once (to nearest even) where it is stored.
#pragma once
#include "camli_common.h"

// type codes of the C entry points
#define CAMLI_F32 0
#define CAMLI_BF16 1
#define CAMLI_F16 2

static inline int camli_type_size(int type) { return type == CAMLI_F32 ? 4 : 2; }

template <typename T, int N>
struct alignas(sizeof(T) * N) TypedVec {
    T v[N];
};

template <typename T, int N>
__device__ __forceinline__ void load_f32(const T* p, float (&out)[N]) {
    const TypedVec<T, N> t = *reinterpret_cast<const TypedVec<T, N>*>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = (float)t.v[i];
}

template <typename T, int N>
__device__ __forceinline__ void store_f32(T* p, const float (&in)[N]) {
    TypedVec<T, N> t;
#pragma unroll
    for (int i = 0; i < N; ++i) t.v[i] = (T)in[i];
    *reinterpret_cast<TypedVec<T, N>*>(p) = t;
}

typedef unsigned vec16_t __attribute__((ext_vector_type(4)));

// as load_f32 / store_f32, with a choice of not keeping the line in the caches
template <typename T, int N>
__device__ __forceinline__ void load_f32(const T* p, float (&out)[N], bool stream) {
    if constexpr (sizeof(T) * N == 16) {
        if (stream) {
            union { TypedVec<T, N> t; vec16_t u; } v;
            v.u = __builtin_nontemporal_load(reinterpret_cast<const vec16_t*>(p));
#pragma unroll
            for (int i = 0; i < N; ++i) out[i] = (float)v.t.v[i];
            return;
        }
    }
    load_f32<T, N>(p, out);
}

template <typename T, int N>
__device__ __forceinline__ void store_f32(T* p, const float (&in)[N], bool stream) {
    if constexpr (sizeof(T) * N == 16) {
        if (stream) {
            union { TypedVec<T, N> t; vec16_t u; } v;
#pragma unroll
            for (int i = 0; i < N; ++i) v.t.v[i] = (T)in[i];
            __builtin_nontemporal_store(v.u, reinterpret_cast<vec16_t*>(p));
            return;
        }
    }
    store_f32<T, N>(p, in);
}

// element i of a small parameter vector whose type is a run-time code
__device__ __forceinline__ float load_param(const void* p, int type, int64_t i) {
    if (type == CAMLI_F32) return static_cast<const float*>(p)[i];
    if (type == CAMLI_BF16) return (float)static_cast<const __bf16*>(p)[i];
    return (float)static_cast<const _Float16*>(p)[i];
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor(v, off, CAMLI_WAVE);
    return v;
}
