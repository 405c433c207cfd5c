// Shared pieces of the token operators (qk_norm.hip, dropout.hip, attention_*.hip): element types, vectors of elements,
// launch checks.  All arithmetic is fp32; 16-bit types are rounded to nearest-even once, when a result is stored.
#pragma once
#include "common.h"
#include <type_traits>

typedef __bf16 bf16;
typedef _Float16 f16;

template <typename T> struct Vec16 { static constexpr int N = 16 / (int)sizeof(T); };      // elements of a 16-byte access

// N consecutive elements as floats; `vec`: the address is 16-byte aligned (else element by element)
template <typename T, int N>
__device__ __forceinline__ void load_floats(const T* __restrict__ p, float* v) {
    typedef T V __attribute__((ext_vector_type(Vec16<T>::N)));
    static_assert(N % Vec16<T>::N == 0, "whole 16-byte accesses");
#pragma unroll
    for (int j = 0; j < N; j += Vec16<T>::N) {
        const V u = *reinterpret_cast<const V*>(p + j);
#pragma unroll
        for (int i = 0; i < Vec16<T>::N; ++i) v[j + i] = (float)u[i];
    }
}
template <typename T, int N>
__device__ __forceinline__ void store_floats(T* __restrict__ p, const float* v) {
    typedef T V __attribute__((ext_vector_type(Vec16<T>::N)));
#pragma unroll
    for (int j = 0; j < N; j += Vec16<T>::N) {
        V u;
#pragma unroll
        for (int i = 0; i < Vec16<T>::N; ++i) u[i] = (T)v[j + i];
        *reinterpret_cast<V*>(p + j) = u;
    }
}

// Runs f with a value of the descriptor's element type; an unknown code is refused by the caller beforehand.
template <typename F>
static inline int with_dtype(int dtype, F f) {
    switch (dtype) {
        case SEMPYR_F32: return f(float());
        case SEMPYR_F16: return f(f16());
        default: return f(bf16());
    }
}
static inline bool dtype_ok(int dtype) { return dtype == SEMPYR_F32 || dtype == SEMPYR_F16 || dtype == SEMPYR_BF16; }
static inline int dtype_size(int dtype) { return dtype == SEMPYR_F32 ? 4 : 2; }
// a launch of `blocks` workgroups: the threads of a dimension have to stay below 2^32
static inline bool grid_fits(int64_t blocks, int threads) { return blocks <= 0xFFFFFFFFll / threads; }
static inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
