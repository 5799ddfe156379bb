// gm_rows.h -- what the typed row kernels share (gm_token.hip, gm_norm.hip, gm_logprob.hip): the 32- and 16-bit element
// types, 16-byte vector access and reductions over a wave or a workgroup.
#pragma once
#include "gm_common.h"

namespace gm {

using bf16_t = __bf16;
using f16_t = _Float16;

// all arithmetic is float; a store rounds once, to nearest even (f16 overflows to infinity, as a conversion does)
template <class T> __device__ __forceinline__ float to_f32(T v) { return (float)v; }
template <class T> __device__ __forceinline__ T from_f32(float v) { return (T)v; }

template <class T, int V> struct alignas(sizeof(T) * V) Vec { T v[V]; };
template <class T, int V> __device__ __forceinline__ void load_vec(const T* __restrict__ p, float (&x)[V]) {
    const Vec<T, V> t = *reinterpret_cast<const Vec<T, V>*>(p);
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = to_f32(t.v[i]);
}
template <class T, int V> __device__ __forceinline__ void store_vec(T* __restrict__ p, const float (&x)[V]) {
    Vec<T, V> t;
#pragma unroll
    for (int i = 0; i < V; ++i) t.v[i] = from_f32<T>(x[i]);
    *reinterpret_cast<Vec<T, V>*>(p) = t;
}

// sum over the 64 lanes, the same bits in every lane (a butterfly adds the same pairs on both sides)
template <class T> __device__ __forceinline__ T wave_add(T v) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) v = v + __shfl_xor(v, off);
    return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) v = __builtin_fmaxf(v, __shfl_xor(v, off));
    return v;
}

// orders one wave's LDS accesses among its lanes: nothing moves across it (the hardware keeps a wave's LDS order)
__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// an index that the caller gives as int32 or int64 (tokens, classes, sequence offsets)
struct IndexArray {
    const void* p;
    int is64;
    __device__ __forceinline__ int64_t at(int64_t i) const {
        return is64 ? static_cast<const int64_t*>(p)[i] : (int64_t)static_cast<const int32_t*>(p)[i];
    }
};

static inline bool dtype_ok(int dtype) { return dtype == GM_DTYPE_F32 || dtype == GM_DTYPE_BF16 || dtype == GM_DTYPE_F16; }
static inline int dtype_size(int dtype) { return dtype == GM_DTYPE_F32 ? 4 : 2; }

// run fn.template operator()<T>() for the element type that `dtype` names
template <class Fn> static inline int with_dtype(int dtype, Fn&& fn) {
    if (dtype == GM_DTYPE_F32) return fn(float{});
    if (dtype == GM_DTYPE_BF16) return fn(bf16_t{});
    return fn(f16_t{});
}

}  // namespace gm
