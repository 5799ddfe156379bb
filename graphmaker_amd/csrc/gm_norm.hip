// gm_norm.hip -- layer norm of rows of any width in float32, bfloat16 or float16, and its gradients.
//
//   y  = (x - mu) r gamma + beta,   mu = mean(x),   r = 1 / sqrt(mean((x - mu)^2) + eps)      over the N columns of a row
//   dx = r (g gamma - mean(g gamma) - xh mean(g gamma xh)),   xh = (x - mu) r
//   dgamma = sum over rows of g xh,   dbeta = sum over rows of g
//
// The variance is that of the differences from the mean, never mean(x^2) - mu^2.  Statistics and sums are float32 whatever
// the element type; gamma and beta have the element type or are float32 (`weight_dtype`), and may be absent (1 and 0).
#include "gm_rows.h"

namespace gm {

template <class T, class W>
__global__ void __launch_bounds__(256)
k_layer_norm_fwd(int64_t M, int64_t N, const T* __restrict__ X, int64_t ldx, const W* __restrict__ gamma, const W* __restrict__ beta,
                 float eps, T* __restrict__ Y, int64_t ldy, float* __restrict__ mean_out, float* __restrict__ rstd_out) {
    const int lane = threadIdx.x & 63;
    const int64_t m = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (m >= M) return;
    const T* x = X + m * ldx;
    float s = 0.0f, q = 0.0f;
    for (int64_t c = lane; c < N; c += 64) s = s + to_f32(x[c]);
    const float mean = wave_add(s) / (float)N;
    for (int64_t c = lane; c < N; c += 64) {
        const float t = to_f32(x[c]) - mean;
        q = __builtin_fmaf(t, t, q);
    }
    const float rstd = 1.0f / __builtin_sqrtf(wave_add(q) / (float)N + eps);
    for (int64_t c = lane; c < N; c += 64) {
        const float t = (to_f32(x[c]) - mean) * rstd;
        Y[m * ldy + c] = from_f32<T>(__builtin_fmaf(t, gamma ? to_f32(gamma[c]) : 1.0f, beta ? to_f32(beta[c]) : 0.0f));
    }
    if (lane == 0 && mean_out) {
        mean_out[m] = mean;
        rstd_out[m] = rstd;
    }
}

// dx, and the column sums of g xh and g over a workgroup's rows: part[workgroup][0][c], part[workgroup][1][c]
template <class T, class W>
__global__ void __launch_bounds__(256)
k_layer_norm_bwd(int64_t M, int64_t N, const T* __restrict__ G, int64_t ldg, const T* __restrict__ X, int64_t ldx,
                 const float* __restrict__ mean, const float* __restrict__ rstd, const W* __restrict__ gamma, T* __restrict__ dX,
                 int64_t lddx, float* __restrict__ part) {
    __shared__ float red[2][4];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    bool first = true;
    for (int64_t m = blockIdx.x; m < M; m += gridDim.x) {
        const float mu = mean[m], rs = rstd[m];
        const T *x = X + m * ldx, *gr = G + m * ldg;
        float s1 = 0.0f, s2 = 0.0f;
        for (int64_t c = threadIdx.x; c < N; c += 256) {
            const float g = to_f32(gr[c]), xh = (to_f32(x[c]) - mu) * rs;
            if (part) {
                float* p = part + (int64_t)blockIdx.x * 2 * N + c;
                p[0] = (first ? 0.0f : p[0]) + g * xh;
                p[N] = (first ? 0.0f : p[N]) + g;
            }
            const float gg = g * (gamma ? to_f32(gamma[c]) : 1.0f);
            s1 = s1 + gg;
            s2 = __builtin_fmaf(gg, xh, s2);
        }
        first = false;
        s1 = wave_add(s1);
        s2 = wave_add(s2);
        __syncthreads();
        if (lane == 0) { red[0][wv] = s1; red[1][wv] = s2; }
        __syncthreads();
        s1 = (red[0][0] + red[0][1] + red[0][2] + red[0][3]) / (float)N;
        s2 = (red[1][0] + red[1][1] + red[1][2] + red[1][3]) / (float)N;
        if (dX)
            for (int64_t c = threadIdx.x; c < N; c += 256) {
                const float xh = (to_f32(x[c]) - mu) * rs;
                const float gg = to_f32(gr[c]) * (gamma ? to_f32(gamma[c]) : 1.0f);
                dX[m * lddx + c] = from_f32<T>(rs * ((gg - s1) - xh * s2));
            }
    }
}

// dgamma[c], dbeta[c]: the workgroups' sums in ascending order
template <class W>
__global__ void __launch_bounds__(256)
k_layer_norm_cols(int64_t nblk, int64_t N, const float* __restrict__ part, W* __restrict__ dgamma, W* __restrict__ dbeta) {
    const int64_t g = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (g >= 2 * N) return;
    float acc = 0.0f;
    for (int64_t b = 0; b < nblk; ++b) acc = acc + part[b * 2 * N + g];
    W* out = g < N ? dgamma : dbeta;
    if (out) out[g < N ? g : g - N] = from_f32<W>(acc);
}

static inline int64_t norm_blocks(int64_t M) { return M < 512 ? M : 512; }

template <class Fn> static inline int with_weight_dtype(int dtype, int weight_dtype, Fn&& fn) {
    return with_dtype(dtype, [&](auto t) -> int {
        if (weight_dtype == GM_DTYPE_F32) return fn(t, float{});
        return fn(t, t);
    });
}

}  // namespace gm

using namespace gm;

#define GM_NORM_CHECK()                                                                                                   \
    GM_REQUIRE(M >= 0 && N > 0, "bad arguments");                                                                         \
    GM_REQUIRE(dtype_ok(dtype) && (weight_dtype == dtype || weight_dtype == GM_DTYPE_F32),                                \
               "dtype %d with weight_dtype %d: the weights have the rows' type or are float32", dtype, weight_dtype);     \
    GM_REQUIRE(M < (1ll << 31) && N < (1ll << 31), "M or N of 2^31 or more")

extern "C" int gm_layer_norm_fwd(int64_t M, int64_t N, const void* X, int64_t ldx, int dtype, const void* gamma, const void* beta,
                                 int weight_dtype, float eps, void* Y, int64_t ldy, float* mean, float* rstd, gm_stream_t stream) {
    GM_NORM_CHECK();
    if (M == 0) return GM_OK;
    GM_REQUIRE(X && Y && ldx >= N && ldy >= N && !mean == !rstd, "bad arguments");
    return with_weight_dtype(dtype, weight_dtype, [&](auto t, auto u) -> int {
        using T = decltype(t);
        using W = decltype(u);
        hipLaunchKernelGGL((k_layer_norm_fwd<T, W>), dim3((unsigned)((M + 3) / 4)), dim3(256), 0, as_stream(stream), M, N,
                           static_cast<const T*>(X), ldx, static_cast<const W*>(gamma), static_cast<const W*>(beta), eps,
                           static_cast<T*>(Y), ldy, mean, rstd);
        GM_LAUNCH_CHECK();
        return GM_OK;
    });
}

extern "C" int64_t gm_layer_norm_bwd_workspace_bytes(int64_t M, int64_t N) {
    if (M < 0 || N <= 0 || M >= (1ll << 31) || N >= (1ll << 31)) return -1;
    return norm_blocks(M) * 2 * N * 4;
}

extern "C" int gm_layer_norm_bwd(int64_t M, int64_t N, const void* G, int64_t ldg, const void* X, int64_t ldx, int dtype,
                                 const float* mean, const float* rstd, const void* gamma, int weight_dtype, void* dX, int64_t lddx,
                                 void* dgamma, void* dbeta, void* workspace, int64_t workspace_bytes, gm_stream_t stream) {
    GM_NORM_CHECK();
    GM_REQUIRE(M == 0 || (G && X && mean && rstd && ldg >= N && ldx >= N && (!dX || lddx >= N)), "bad arguments");
    const bool cols = dgamma || dbeta;
    const int64_t nblk = norm_blocks(M), need = nblk * 2 * N * 4;
    GM_REQUIRE(!cols || M == 0 || (workspace && workspace_bytes >= need && aligned(workspace, 16)),
               "gm_layer_norm_bwd needs %lld workspace bytes (gm_layer_norm_bwd_workspace_bytes)", (long long)need);
    hipStream_t s = as_stream(stream);
    float* part = cols ? static_cast<float*>(workspace) : nullptr;
    return with_weight_dtype(dtype, weight_dtype, [&](auto t, auto u) -> int {
        using T = decltype(t);
        using W = decltype(u);
        if (M > 0) {
            hipLaunchKernelGGL((k_layer_norm_bwd<T, W>), dim3((unsigned)nblk), dim3(256), 0, s, M, N, static_cast<const T*>(G), ldg,
                               static_cast<const T*>(X), ldx, mean, rstd, static_cast<const W*>(gamma), static_cast<T*>(dX), lddx, part);
            GM_LAUNCH_CHECK();
        }
        if (cols) {
            hipLaunchKernelGGL((k_layer_norm_cols<W>), dim3((unsigned)((2 * N + 255) / 256)), dim3(256), 0, s, nblk, N, part,
                               static_cast<W*>(dgamma), static_cast<W*>(dbeta));
            GM_LAUNCH_CHECK();
        }
        return GM_OK;
    });
}
