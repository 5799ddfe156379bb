// gm_logprob.hip -- log-probability of one class of every row of logits, and its gradient.
//
//   forward    lp[i] = x[i][c_i] - log sum_j exp(x[i][j])
//   gradient   dx[i][j] = g[i] ([j = c_i] - softmax(x[i])[j])
//
// A row whose class is `ignore_index` has log-probability 0 and a zero gradient, and its logits are not read; so is the
// gradient of a row whose g is 0.  Any other class outside [0, V) gives NaN in both.  Sums are float32 whatever the
// logits' type, about the row's largest logit.  stats[i] = (largest logit, log of the sum of exponentials about it).
#include "gm_rows.h"

namespace gm {

// exp(x) for x <= 0 within about one unit in the last place: 2^(x log2 e) with the product's rounding error put back as a
// factor (the product alone would cost |x| 2^-24 relative).  exp(-inf) = 0, NaN stays NaN.
__device__ __forceinline__ float exp_nonpos(float x) {
    x = x < -120.0f ? -120.0f : x;                       // 2^-173: below every float
    const float t = x * 1.44269502f;
    const float lo = __builtin_fmaf(x, 1.92596299e-8f, __builtin_fmaf(x, 1.44269502f, -t));
    const float e = __builtin_amdgcn_exp2f(t);
    return __builtin_fmaf(e * lo, 0.693147182f, e);
}

template <class T>
__global__ void __launch_bounds__(256)
k_class_log_prob_fwd(int64_t M, int64_t V, const T* __restrict__ X, int64_t ldx, IndexArray cls, int64_t ignore,
                     float* __restrict__ lp, float2* __restrict__ stats) {
    const int lane = threadIdx.x & 63;
    const int64_t m = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (m >= M) return;
    const int64_t c = cls.at(m);
    if (c == ignore) {
        if (lane == 0) {
            lp[m] = 0.0f;
            if (stats) stats[m] = make_float2(0.0f, 0.0f);
        }
        return;
    }
    const T* x = X + m * ldx;
    float mx = -INFINITY, s = 0.0f;
    for (int64_t j = lane; j < V; j += 64) mx = __builtin_fmaxf(mx, to_f32(x[j]));
    mx = wave_max(mx);
    for (int64_t j = lane; j < V; j += 64) s = s + exp_nonpos(to_f32(x[j]) - mx);
    s = wave_add(s);
    if (lane == 0) {
        const float ls = logf(s);
        lp[m] = c >= 0 && c < V ? (to_f32(x[c]) - mx) - ls : __builtin_nanf("");
        if (stats) stats[m] = make_float2(mx, ls);
    }
}

template <class T>
__global__ void __launch_bounds__(256)
k_class_log_prob_bwd(int64_t M, int64_t V, const float* __restrict__ g, const T* __restrict__ X, int64_t ldx, IndexArray cls,
                     int64_t ignore, const float2* __restrict__ stats, T* __restrict__ dX, int64_t lddx) {
    const int lane = threadIdx.x & 63;
    const int64_t m = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (m >= M) return;
    const int64_t c = cls.at(m);
    const float gm_ = c == ignore ? 0.0f : g[m];
    const bool valid = c >= 0 && c < V;
    const T* x = X + m * ldx;
    T* d = dX + m * lddx;
    const float2 st = stats[m];
    for (int64_t j = lane; j < V; j += 64) {
        float v = 0.0f;
        if (gm_ != 0.0f) {
            const float p = exp_nonpos((to_f32(x[j]) - st.x) - st.y);
            v = valid ? gm_ * ((j == c ? 1.0f : 0.0f) - p) : __builtin_nanf("");
        }
        d[j] = from_f32<T>(v);
    }
}

}  // namespace gm

using namespace gm;

#define GM_LOGPROB_CHECK()                                                                                                \
    GM_REQUIRE(M >= 0 && V > 0, "bad arguments");                                                                         \
    GM_REQUIRE(dtype_ok(dtype), "dtype %d is none of GM_DTYPE_*", dtype);                                                 \
    GM_REQUIRE(M < (1ll << 31) && V < (1ll << 31), "M or V of 2^31 or more")

extern "C" int gm_class_log_prob_fwd(int64_t M, int64_t V, const void* logits, int64_t ldx, int dtype, const void* classes,
                                     int classes_i64, int64_t ignore_index, float* log_prob, float* stats, void* workspace,
                                     int64_t workspace_bytes, gm_stream_t stream) {
    GM_LOGPROB_CHECK();
    if (M == 0) return GM_OK;
    GM_REQUIRE(logits && classes && log_prob && ldx >= V && aligned(stats, 8), "bad arguments");
    return with_dtype(dtype, [&](auto t) -> int {
        using T = decltype(t);
        hipLaunchKernelGGL((k_class_log_prob_fwd<T>), dim3((unsigned)((M + 3) / 4)), dim3(256), 0, as_stream(stream), M, V,
                           static_cast<const T*>(logits), ldx, IndexArray{classes, classes_i64}, ignore_index, log_prob,
                           reinterpret_cast<float2*>(stats));
        GM_LAUNCH_CHECK();
        return GM_OK;
    });
}

extern "C" int64_t gm_class_log_prob_workspace_bytes(int64_t M, int64_t V) {
    if (M < 0 || V <= 0 || M >= (1ll << 31) || V >= (1ll << 31)) return -1;
    return 0;
}

extern "C" int gm_class_log_prob_bwd(int64_t M, int64_t V, const float* g, const void* logits, int64_t ldx, int dtype,
                                     const void* classes, int classes_i64, int64_t ignore_index, const float* stats, void* dlogits,
                                     int64_t lddx, gm_stream_t stream) {
    GM_LOGPROB_CHECK();
    if (M == 0) return GM_OK;
    GM_REQUIRE(g && logits && classes && stats && dlogits && ldx >= V && lddx >= V && aligned(stats, 8), "bad arguments");
    return with_dtype(dtype, [&](auto t) -> int {
        using T = decltype(t);
        hipLaunchKernelGGL((k_class_log_prob_bwd<T>), dim3((unsigned)((M + 3) / 4)), dim3(256), 0, as_stream(stream), M, V, g,
                           static_cast<const T*>(logits), ldx, IndexArray{classes, classes_i64}, ignore_index,
                           reinterpret_cast<const float2*>(stats), static_cast<T*>(dlogits), lddx);
        GM_LAUNCH_CHECK();
        return GM_OK;
    });
}
