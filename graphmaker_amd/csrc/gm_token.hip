// gm_token.hip -- embedding of tokens drawn from a large vocabulary and its gradient.
//
//   forward    y[i] = scale * W[t_i]
//   gradient   dW[c] = scale * sum_{i : t_i = c} G[i]      (0 for a row no token names, and for the padding row)
//
// The gradient groups the tokens by value first: a stable radix sort of (token, position), so that each row of dW is the
// sum of one run of the sorted positions, taken in ascending position.  No atomics on values: the sum's order depends on
// the tokens alone.  A token outside [0, C) reads no memory: its output row is NaN and it adds to no row.
#include "gm_rows.h"

namespace gm {

template <class T>
__global__ void __launch_bounds__(256)
k_token_embedding_fwd(int64_t n, int64_t C, int64_t w, IndexArray tok, const T* __restrict__ W, int64_t ldw, float scale,
                      T* __restrict__ out, int64_t ldo) {
    const int64_t g = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (g >= n * w) return;
    const int64_t i = g / w, col = g - i * w;
    const int64_t c = tok.at(i);
    out[i * ldo + col] = c >= 0 && c < C ? from_f32<T>(to_f32(W[c * ldw + col]) * scale) : from_f32<T>(__builtin_nanf(""));
}

// ---- stable radix sort of n keys in [0, C] (C: tokens that add to no row, sorted behind the others), RADIX_BITS at a time
constexpr int RADIX_BITS = 9, RADIX_BINS = 1 << RADIX_BITS;
constexpr int SORT_KEYS = 2048;                       // keys per workgroup: 4 waves x 8 rounds x 64 lanes
__device__ __forceinline__ uint32_t token_key(const IndexArray& tok, int64_t i, int64_t C, int64_t padding) {
    const int64_t c = tok.at(i);
    return c >= 0 && c < C && c != padding ? (uint32_t)c : (uint32_t)C;
}

// counts[digit][workgroup]
__global__ void __launch_bounds__(256)
k_radix_count(int64_t n, int64_t C, int64_t padding, IndexArray tok, const uint32_t* __restrict__ keys, int shift,
              uint32_t* __restrict__ counts) {
    __shared__ uint32_t hist[RADIX_BINS];
    for (int b = threadIdx.x; b < RADIX_BINS; b += 256) hist[b] = 0;
    __syncthreads();
    const int64_t base = (int64_t)blockIdx.x * SORT_KEYS;
    for (int r = 0; r < SORT_KEYS / 256; ++r) {
        const int64_t i = base + r * 256 + threadIdx.x;
        if (i < n) {
            const uint32_t key = keys ? keys[i] : token_key(tok, i, C, padding);
            atomicAdd(&hist[(key >> shift) & (RADIX_BINS - 1)], 1u);
        }
    }
    __syncthreads();
    for (int b = threadIdx.x; b < RADIX_BINS; b += 256) counts[(int64_t)b * gridDim.x + blockIdx.x] = hist[b];
}

// exclusive prefix sum of m counts by one workgroup
__global__ void __launch_bounds__(1024) k_radix_scan(int64_t m, uint32_t* __restrict__ counts) {
    __shared__ uint32_t tot[16];
    uint32_t carry = 0;
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    for (int64_t b = 0; b < m; b += 1024) {
        const int64_t i = b + threadIdx.x;
        const uint32_t v = i < m ? counts[i] : 0;
        uint32_t s = v;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const uint32_t t = __shfl_up(s, off);
            if (lane >= off) s += t;
        }
        if (lane == 63) tot[wv] = s;
        __syncthreads();
        uint32_t before = 0, all = 0;
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            if (k < wv) before += tot[k];
            all += tot[k];
        }
        if (i < m) counts[i] = carry + before + s - v;
        carry += all;
        __syncthreads();
    }
}

// Each wave owns SORT_KEYS/4 consecutive keys and keeps the next free place of every digit; the rank among the 64 keys of
// a round is the number of lower lanes with the same digit (one ballot per digit bit), so equal digits keep their order.
__global__ void __launch_bounds__(256)
k_radix_scatter(int64_t n, int64_t C, int64_t padding, IndexArray tok, const uint32_t* __restrict__ keys,
                const uint32_t* __restrict__ pos, int shift, const uint32_t* __restrict__ starts, uint32_t* __restrict__ keys_out,
                uint32_t* __restrict__ pos_out) {
    __shared__ uint32_t next[4][RADIX_BINS];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    for (int b = threadIdx.x; b < 4 * RADIX_BINS; b += 256) (&next[0][0])[b] = 0;
    __syncthreads();
    const int64_t base = (int64_t)blockIdx.x * SORT_KEYS + wv * (SORT_KEYS / 4);
    uint32_t key[SORT_KEYS / 256];
#pragma unroll
    for (int r = 0; r < SORT_KEYS / 256; ++r) {
        const int64_t i = base + r * 64 + lane;
        key[r] = 0;
        if (i < n) {
            key[r] = keys ? keys[i] : token_key(tok, i, C, padding);
            atomicAdd(&next[wv][(key[r] >> shift) & (RADIX_BINS - 1)], 1u);
        }
    }
    __syncthreads();
    for (int b = threadIdx.x; b < RADIX_BINS; b += 256) {
        uint32_t at = starts[(int64_t)b * gridDim.x + blockIdx.x];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t c = next[k][b];
            next[k][b] = at;
            at += c;
        }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < SORT_KEYS / 256; ++r) {
        const int64_t i = base + r * 64 + lane;
        const bool in = i < n;
        const uint32_t d = (key[r] >> shift) & (RADIX_BINS - 1);
        uint64_t same = __ballot(in);
#pragma unroll
        for (int bit = 0; bit < RADIX_BITS; ++bit) {
            const uint64_t set = __ballot((d >> bit) & 1u);
            same &= (d >> bit) & 1u ? set : ~set;
        }
        const int rank = __popcll(same & ((1ull << lane) - 1ull));
        uint32_t at = 0;
        if (in) at = next[wv][d] + rank;
        wave_fence();                                   // every lane has read its place before a leader moves it on
        if (in && rank == 0) next[wv][d] = at + (uint32_t)__popcll(same);
        wave_fence();
        if (in) {
            keys_out[at] = key[r];
            pos_out[at] = pos ? pos[i] : (uint32_t)i;
        }
    }
}

// rowptr[c] = number of sorted keys below c, c = 0..C
__global__ void __launch_bounds__(256)
k_token_rowptr(int64_t n, int64_t C, const uint32_t* __restrict__ keys, uint32_t* __restrict__ rowptr) {
    const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (c > C) return;
    int64_t lo = 0, hi = n;
    while (lo < hi) {
        const int64_t mid = (lo + hi) >> 1;
        if (keys[mid] < (uint32_t)c) lo = mid + 1;
        else hi = mid;
    }
    rowptr[c] = (uint32_t)lo;
}

// one wave per row of dW
template <class T>
__global__ void __launch_bounds__(256)
k_token_grad(int64_t C, int64_t w, const uint32_t* __restrict__ rowptr, const uint32_t* __restrict__ pos,
             const T* __restrict__ G, int64_t ldg, float scale, T* __restrict__ dW, int64_t ldw) {
    const int lane = threadIdx.x & 63;
    const int64_t c = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (c >= C) return;
    const uint32_t a = rowptr[c], b = rowptr[c + 1];
    for (int64_t col = lane; col < w; col += 64) {
        float acc = 0.0f;
        for (uint32_t k = a; k < b; ++k) acc = acc + to_f32(G[(int64_t)pos[k] * ldg + col]);
        dW[c * ldw + col] = from_f32<T>(acc * scale);
    }
}

struct TokenLayout {
    int64_t nblk, keys[2], pos[2], counts, rowptr, bytes;
    int passes;
};
static inline TokenLayout token_layout(int64_t n, int64_t C) {
    TokenLayout l;
    int bits = 1;
    while ((C >> bits) != 0) ++bits;                   // keys are 0..C
    l.passes = (bits + RADIX_BITS - 1) / RADIX_BITS;
    l.nblk = (n + SORT_KEYS - 1) / SORT_KEYS;
    int64_t at = 0;
    auto take = [&at](int64_t words) { const int64_t p = at; at += (words * 4 + 255) / 256 * 256; return p; };
    for (int k = 0; k < 2; ++k) { l.keys[k] = take(n); l.pos[k] = take(n); }
    l.counts = take(l.nblk * RADIX_BINS);
    l.rowptr = take(C + 1);
    l.bytes = at;
    return l;
}

}  // namespace gm

using namespace gm;

#define GM_TOKEN_CHECK(ptr_)                                                                                              \
    GM_REQUIRE(n >= 0 && C > 0 && w > 0 && (n == 0 || (tokens && ptr_)), "bad arguments");                                \
    GM_REQUIRE(dtype_ok(dtype), "dtype %d is none of GM_DTYPE_*", dtype);                                                 \
    GM_REQUIRE(C < (1ll << 31) && n < (1ll << 31) && w < (1ll << 31), "n, C or w of 2^31 or more")

extern "C" int gm_token_embedding_fwd(int64_t n, int64_t C, int64_t w, const void* tokens, int tokens_i64, const void* weight,
                                      int64_t ldw, int dtype, float scale, void* out, int64_t ldo, gm_stream_t stream) {
    GM_TOKEN_CHECK(out);
    GM_REQUIRE(weight && ldw >= w && ldo >= w, "weight missing or leading dimension too small");
    if (n == 0) return GM_OK;
    GM_REQUIRE((n * w + 255) / 256 < (1ll << 31), "n * w too large");
    return with_dtype(dtype, [&](auto t) -> int {
        using T = decltype(t);
        hipLaunchKernelGGL((k_token_embedding_fwd<T>), dim3((unsigned)((n * w + 255) / 256)), dim3(256), 0, as_stream(stream), n, C,
                           w, IndexArray{tokens, tokens_i64}, static_cast<const T*>(weight), ldw, scale, static_cast<T*>(out), ldo);
        GM_LAUNCH_CHECK();
        return GM_OK;
    });
}

extern "C" int64_t gm_token_embedding_bwd_workspace_bytes(int64_t n, int64_t C, int64_t w) {
    if (n < 0 || C <= 0 || w <= 0 || n >= (1ll << 31) || C >= (1ll << 31)) return -1;
    return token_layout(n, C).bytes;
}

extern "C" int gm_token_embedding_bwd(int64_t n, int64_t C, int64_t w, const void* tokens, int tokens_i64, int64_t padding_idx,
                                      const void* G, int64_t ldg, int dtype, float scale, void* dW, int64_t ldw,
                                      void* workspace, int64_t workspace_bytes, gm_stream_t stream) {
    GM_TOKEN_CHECK(G);
    GM_REQUIRE(dW && ldg >= w && ldw >= w, "dW missing or leading dimension too small");
    GM_REQUIRE(padding_idx < C, "padding_idx %lld is not below C = %lld", (long long)padding_idx, (long long)C);
    const TokenLayout l = token_layout(n, C);
    GM_REQUIRE(workspace && workspace_bytes >= l.bytes && aligned(workspace, 16),
               "gm_token_embedding_bwd needs %lld workspace bytes (gm_token_embedding_bwd_workspace_bytes)", (long long)l.bytes);
    hipStream_t s = as_stream(stream);
    char* ws = static_cast<char*>(workspace);
    auto u32 = [ws](int64_t at) { return reinterpret_cast<uint32_t*>(ws + at); };
    const IndexArray tok{tokens, tokens_i64};
    uint32_t *counts = u32(l.counts), *rowptr = u32(l.rowptr);
    const uint32_t *keys = nullptr, *pos = nullptr;
    for (int p = 0; p < l.passes && n > 0; ++p) {
        uint32_t *ko = u32(l.keys[p & 1]), *po = u32(l.pos[p & 1]);
        hipLaunchKernelGGL(k_radix_count, dim3((unsigned)l.nblk), dim3(256), 0, s, n, C, padding_idx, tok, keys, p * RADIX_BITS, counts);
        GM_LAUNCH_CHECK();
        hipLaunchKernelGGL(k_radix_scan, dim3(1), dim3(1024), 0, s, l.nblk * RADIX_BINS, counts);
        GM_LAUNCH_CHECK();
        hipLaunchKernelGGL(k_radix_scatter, dim3((unsigned)l.nblk), dim3(256), 0, s, n, C, padding_idx, tok, keys, pos, p * RADIX_BITS,
                           counts, ko, po);
        GM_LAUNCH_CHECK();
        keys = ko;
        pos = po;
    }
    hipLaunchKernelGGL(k_token_rowptr, dim3((unsigned)((C + 1 + 255) / 256)), dim3(256), 0, s, n, C, keys, rowptr);
    GM_LAUNCH_CHECK();
    return with_dtype(dtype, [&](auto t) -> int {
        using T = decltype(t);
        hipLaunchKernelGGL((k_token_grad<T>), dim3((unsigned)((C + 3) / 4)), dim3(256), 0, s, C, w, rowptr, pos,
                           static_cast<const T*>(G), ldg, scale, static_cast<T*>(dW), ldw);
        GM_LAUNCH_CHECK();
        return GM_OK;
    });
}
