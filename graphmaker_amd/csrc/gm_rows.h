// gm_rows.h -- what the typed row kernels share (gm_token.hip, gm_norm.hip, gm_logprob.hip): the 32- and 16-bit element
// types, 16-byte vector access and reductions over a wave or a workgroup.
#pragma once
#include <type_traits>

#include "gm_common.h"

namespace gm {

using bf16_t = __bf16;
using f16_t = _Float16;

// all arithmetic is float; a store rounds once, to nearest even (f16 overflows to infinity, as a conversion does)
template <class T> __device__ __forceinline__ float to_f32(T v) { return (float)v; }
template <class T> __device__ __forceinline__ T from_f32(float v) { return (T)v; }

// ---- rows of N elements as pieces of V, from any address that an element may have: global accesses of 16 bytes need no
// alignment here, and a row whose start straddles lines costs one line more a wave.  A kernel has up to three forms:
//   V = VEC, TAIL = false   N is a multiple of V
//   V = VEC, TAIL = true    N is at least V: the last piece is loaded where it ends with the row, and shifted
//   V = 1,   TAIL = false   rows of less than 16 bytes
// No load is behind a branch, so that all of a thread's loads are in flight together; lanes behind the row load its last
// piece and see zeros.
template <class T> constexpr int VEC = 16 / (int)sizeof(T);
template <class T, int V> struct __attribute__((packed, aligned(alignof(T)))) Vec { T v[V]; };
// The zeros come from masks: of `in ? loaded : 0` the compiler makes a branch around the load and a wait behind it.
template <class T, int V, bool TAIL> __device__ __forceinline__ Vec<T, V> load_vec(const T* __restrict__ row, int col, int N) {
    const int at = col + V <= N ? col : N - V;
    Vec<T, V> x = *reinterpret_cast<const Vec<T, V>*>(row + at);
    if constexpr (V == 1) {
        using Bits = std::conditional_t<sizeof(T) == 4, uint32_t, uint16_t>;
        x.v[0] = __builtin_bit_cast(T, (Bits)(__builtin_bit_cast(Bits, x.v[0]) & (Bits)(col < N ? ~0u : 0u)));
    } else {
        static_assert(sizeof(x) == 16, "a piece of 16 bytes");
        uint64_t w[2];
        __builtin_memcpy(w, &x, 16);
        if constexpr (!TAIL) {
            const uint64_t in = col < N ? ~0ull : 0ull;
            w[0] &= in;
            w[1] &= in;
        } else {
            const int past = col - at, bits = (past < V ? past : V) * 8 * (int)sizeof(T), low = bits & 63;        // 0 .. 128
            const uint64_t in = bits < 128 ? ~0ull : 0ull, half = bits >= 64 ? ~0ull : 0ull;
            const uint64_t hi = (w[1] >> low) & in, lo = (w[0] >> low) | ((w[1] << 1) << (63 - low));
            w[0] = (lo & ~half & in) | (hi & half);
            w[1] = hi & ~half;
        }
        __builtin_memcpy(&x, w, 16);
    }
    return x;
}
// the piece itself, as a value that has arrived: keeps the loads of the piece behind it from being moved into its place
template <class T, int V> __device__ __forceinline__ Vec<T, V> settled(Vec<T, V> x) {
    typedef uint32_t words __attribute__((ext_vector_type(4)));
    static_assert(sizeof(x) == sizeof(words), "a piece of 16 bytes");
    words w;
    __builtin_memcpy(&w, &x, 16);
    asm volatile("" : "+v"(w));
    __builtin_memcpy(&x, &w, 16);
    return x;
}
template <class T, int V, bool TAIL> __device__ __forceinline__ void store_vec(T* __restrict__ row, int col, int N, const float (&x)[V]) {
    if (!TAIL ? col < N : col + V <= N) {
        Vec<T, V> t;
#pragma unroll
        for (int i = 0; i < V; ++i) t.v[i] = from_f32<T>(x[i]);
        *reinterpret_cast<Vec<T, V>*>(row + col) = t;
    } else if (TAIL) {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (col + i < N) row[col + i] = from_f32<T>(x[i]);
    }
}
// fn(V, TAIL) as integral constants for rows of N elements of T
template <class T, class Fn> static inline void with_row_form(int64_t N, Fn&& fn) {
    if (N < VEC<T>) fn(std::integral_constant<int, 1>{}, std::false_type{});
    else if (N % VEC<T>) fn(std::integral_constant<int, VEC<T>>{}, std::true_type{});
    else fn(std::integral_constant<int, VEC<T>>{}, std::false_type{});
}

// sum over the 64 lanes, the same bits in every lane (a butterfly adds the same pairs on both sides)
template <class T> __device__ __forceinline__ T wave_add(T v) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) v = v + __shfl_xor(v, off);
    return v;
}

// exp(x) within about two units in the last place: 2^(x log2 e), with the product's rounding error (|x| 2^-24 relative, were it
// left) put back as a factor.  exp(-inf) = 0, overflow gives infinity, NaN stays NaN.
__device__ __forceinline__ float exp_any(float x) {
    x = x < -120.0f ? -120.0f : x > 100.0f ? 100.0f : x;       // 2^-173 and 2^144: what lies beyond is 0 or infinite anyway
    const float t = x * 1.44269502f;
    const float lo = __builtin_fmaf(x, 1.92596299e-8f, __builtin_fmaf(x, 1.44269502f, -t));
    return __builtin_amdgcn_exp2f(t) * __builtin_fmaf(lo, 0.693147182f, 1.0f);
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

// workgroups for `want` pieces of work: a launch has less than 2^32 threads, the kernels walk on by the grid's size
static inline unsigned grid_for(int64_t want, int threads) {
    const int64_t most = ((1ll << 32) - 1) / threads;
    return (unsigned)(want < most ? want : most);
}

static inline bool dtype_ok(int dtype) { return dtype == GM_DTYPE_F32 || dtype == GM_DTYPE_BF16 || dtype == GM_DTYPE_F16; }
static inline int dtype_size(int dtype) { return dtype == GM_DTYPE_F32 ? 4 : 2; }

// run fn.template operator()<T>() for the element type that `dtype` names
template <class Fn> static inline int with_dtype(int dtype, Fn&& fn) {
    if (dtype == GM_DTYPE_F32) return fn(float{});
    if (dtype == GM_DTYPE_BF16) return fn(bf16_t{});
    return fn(f16_t{});
}

}  // namespace gm
