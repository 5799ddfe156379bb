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

// gamma and beta as the caller has them
struct Weights {
    const void *gamma, *beta;
    int f32;
    template <class T, int V, bool TAIL> __device__ __forceinline__ void load(const void* p, int col, int N, float absent, float (&x)[V]) const {
        if (!p) {
#pragma unroll
            for (int i = 0; i < V; ++i) x[i] = absent;
        } else if (f32 && sizeof(T) != 4) {
            constexpr int F = V < 4 ? V : 4;
#pragma unroll
            for (int i = 0; i < V; i += F) {
                const Vec<float, F> t = load_vec<float, F, TAIL>(static_cast<const float*>(p), col + i, N);
#pragma unroll
                for (int j = 0; j < F; ++j) x[i + j] = t.v[j];
            }
        } else {
            const Vec<T, V> t = load_vec<T, V, TAIL>(static_cast<const T*>(p), col, N);
#pragma unroll
            for (int i = 0; i < V; ++i) x[i] = to_f32(t.v[i]);
        }
    }
    template <class T> __device__ __forceinline__ float at(const void* p, int64_t col, float absent) const {
        return !p ? absent : f32 ? static_cast<const float*>(p)[col] : to_f32(static_cast<const T*>(p)[col]);
    }
};

// sum of v over the TPR threads of a row, in each of them.  `red` holds one float a wave and is a fresh one at every call
// between two barriers of the workgroup.
template <int TPR> __device__ __forceinline__ float lanes_add(float v) {
#pragma unroll
    for (int off = (TPR < 64 ? TPR : 64) / 2; off >= 1; off >>= 1) v = v + __shfl_xor(v, off);
    return v;
}
template <int TPR> __device__ __forceinline__ float row_add(float v, float* red) {
    v = lanes_add<TPR>(v);
    if (TPR > 64) {
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = red[0];
#pragma unroll
        for (int k = 1; k < TPR / 64; ++k) v = v + red[k];
    }
    return v;
}

// the same of two values behind one barrier
template <int TPR> __device__ __forceinline__ void row_add(float& a, float& b, float (*red)[16]) {
    a = lanes_add<TPR>(a);
    b = lanes_add<TPR>(b);
    if (TPR > 64) {
        if ((threadIdx.x & 63) == 0) { red[0][threadIdx.x >> 6] = a; red[1][threadIdx.x >> 6] = b; }
        __syncthreads();
        a = red[0][0];
        b = red[1][0];
#pragma unroll
        for (int k = 1; k < TPR / 64; ++k) { a = a + red[0][k]; b = b + red[1][k]; }
    }
}

// A row stays in registers: TPR threads hold K x 16 bytes each, so HBM sees every element once.  A workgroup walks several
// rows with gamma and beta in registers too, and loads the next row before it reduces the one it has: what a row waits for
// is HBM alone (8191 x 8192 bf16: 55 us, the card's copy rate; reading gamma and beta and waiting for the row took 92).  Rows of
// 1024 threads are LEAN, without either: half the registers, so that a second workgroup fits a CU.
template <class T, int V, bool TAIL, int K, int TPR>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR)
k_layer_norm_fwd(int64_t M, int N, const T* __restrict__ X, int64_t ldx, Weights w, float eps, T* __restrict__ Y, int64_t ldy,
                 float* __restrict__ mean_out, float* __restrict__ rstd_out) {
    constexpr int ROWS = TPR < 256 ? 256 / TPR : 1;
    constexpr bool LEAN = TPR == 1024;
    constexpr int HELD = LEAN ? 1 : K;
    __shared__ float red[2][16];
    const int t = threadIdx.x & (TPR - 1);
    const int64_t step = (int64_t)gridDim.x * ROWS;
    int64_t m = (int64_t)blockIdx.x * ROWS + threadIdx.x / TPR;
    if (m >= M) return;
    Vec<T, V> r[K], next[HELD];
    float ga[HELD][V], be[HELD][V];
    if constexpr (!LEAN) {
#pragma unroll
        for (int k = 0; k < K; ++k) next[k] = load_vec<T, V, TAIL>(X + m * ldx, (k * TPR + t) * V, N);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            w.load<T, V, TAIL>(w.gamma, (k * TPR + t) * V, N, 1.0f, ga[k]);
            w.load<T, V, TAIL>(w.beta, (k * TPR + t) * V, N, 0.0f, be[k]);
        }
    }
    for (; m < M; m += step) {
        if constexpr (LEAN) {
#pragma unroll
            for (int k = 0; k < K; ++k) r[k] = load_vec<T, V, TAIL>(X + m * ldx, (k * TPR + t) * V, N);
        } else {
            const int64_t ahead = m + step < M ? m + step : m;
#pragma unroll
            for (int k = 0; k < K; ++k) r[k] = next[k];
#pragma unroll
            for (int k = 0; k < K; ++k) next[k] = load_vec<T, V, TAIL>(X + ahead * ldx, (k * TPR + t) * V, N);
        }
        float s = 0.0f, q = 0.0f;
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) s = s + to_f32(r[k].v[i]);
        const float mean = row_add<TPR>(s, red[0]) / (float)N;
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float d = to_f32(r[k].v[i]) - mean;
                if ((k * TPR + t) * V + i < N) q = __builtin_fmaf(d, d, q);
            }
        const float rstd = 1.0f / __builtin_sqrtf(row_add<TPR>(q, red[1]) / (float)N + eps);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float y[V];
            const int h = LEAN ? 0 : k;
            if constexpr (LEAN) {
                w.load<T, V, TAIL>(w.gamma, (k * TPR + t) * V, N, 1.0f, ga[0]);
                w.load<T, V, TAIL>(w.beta, (k * TPR + t) * V, N, 0.0f, be[0]);
            }
#pragma unroll
            for (int i = 0; i < V; ++i) y[i] = __builtin_fmaf((to_f32(r[k].v[i]) - mean) * rstd, ga[h][i], be[h][i]);
            store_vec<T, V, TAIL>(Y + m * ldy, (k * TPR + t) * V, N, y);
        }
        if (t == 0 && mean_out) {
            mean_out[m] = mean;
            rstd_out[m] = rstd;
        }
    }
}

// dx of a workgroup's rows, and the column sums of g xh and g over them, held in registers until the last row:
// part[workgroup][0][c], part[workgroup][1][c].  HBM-bound: 8191 x 8192 bf16 100 us, 4.0 TB/s and the 32 MB of column sums besides.
template <class T, int V, bool TAIL, int K, int TPR>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR)
k_layer_norm_bwd(int64_t M, int N, const T* __restrict__ G, int64_t ldg, const T* __restrict__ X, int64_t ldx,
                 const float* __restrict__ mean, const float* __restrict__ rstd, Weights w, T* __restrict__ dX, int64_t lddx,
                 float* __restrict__ part) {
    constexpr int ROWS = TPR < 256 ? 256 / TPR : 1;
    constexpr bool LEAN = TPR == 1024;
    constexpr int HELD = LEAN ? 1 : K;
    __shared__ float red[2][2][16];
    const int t = threadIdx.x & (TPR - 1);
    const int64_t step = (int64_t)gridDim.x * ROWS;
    int64_t m = (int64_t)blockIdx.x * ROWS + threadIdx.x / TPR;
    float ga[HELD][V], dga[K][V], dbe[K][V];
    Vec<T, V> xr[K], gr[K], xn[HELD], gn[HELD];
    float mu_n = 0.0f, rs_n = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) dga[k][i] = dbe[k][i] = 0.0f;
    if (!LEAN && m < M) {
#pragma unroll
        for (int k = 0; k < HELD; ++k) {
            xn[k] = load_vec<T, V, TAIL>(X + m * ldx, (k * TPR + t) * V, N);
            gn[k] = load_vec<T, V, TAIL>(G + m * ldg, (k * TPR + t) * V, N);
        }
        mu_n = mean[m];
        rs_n = rstd[m];
#pragma unroll
        for (int k = 0; k < HELD; ++k) w.load<T, V, TAIL>(w.gamma, (k * TPR + t) * V, N, 1.0f, ga[k]);
    }
    for (int turn = 0; m < M; m += step, turn ^= 1) {
        float mu = mu_n, rs = rs_n;
        if constexpr (LEAN) {
#pragma unroll
            for (int k = 0; k < K; ++k) {
                xr[k] = load_vec<T, V, TAIL>(X + m * ldx, (k * TPR + t) * V, N);
                gr[k] = load_vec<T, V, TAIL>(G + m * ldg, (k * TPR + t) * V, N);           // 0 behind the row: adds to no sum
            }
            mu = mean[m];
            rs = rstd[m];
        } else {
            const int64_t ahead = m + step < M ? m + step : m;
#pragma unroll
            for (int k = 0; k < K; ++k) { xr[k] = xn[k]; gr[k] = gn[k]; }
#pragma unroll
            for (int k = 0; k < K; ++k) {
                xn[k] = load_vec<T, V, TAIL>(X + ahead * ldx, (k * TPR + t) * V, N);
                gn[k] = load_vec<T, V, TAIL>(G + ahead * ldg, (k * TPR + t) * V, N);
            }
            mu_n = mean[ahead];
            rs_n = rstd[ahead];
        }
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int h = LEAN ? 0 : k;
            if constexpr (LEAN) w.load<T, V, TAIL>(w.gamma, (k * TPR + t) * V, N, 1.0f, ga[0]);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float g = to_f32(gr[k].v[i]), xh = (to_f32(xr[k].v[i]) - mu) * rs, gg = g * ga[h][i];
                if ((k * TPR + t) * V + i < N) {                    // x is 0 there, xh is not, and may be infinite
                    dga[k][i] = __builtin_fmaf(g, xh, dga[k][i]);
                    s2 = __builtin_fmaf(gg, xh, s2);
                    s1 = s1 + gg;
                }
                dbe[k][i] = dbe[k][i] + g;
            }
        }
        row_add<TPR>(s1, s2, red[turn]);
        s1 = s1 / (float)N;
        s2 = s2 / (float)N;
        if (dX)
#pragma unroll
            for (int k = 0; k < K; ++k) {
                float y[V];
                const int h = LEAN ? 0 : k;
                if constexpr (LEAN) w.load<T, V, TAIL>(w.gamma, (k * TPR + t) * V, N, 1.0f, ga[0]);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float xh = (to_f32(xr[k].v[i]) - mu) * rs;
                    y[i] = rs * ((to_f32(gr[k].v[i]) * ga[h][i] - s1) - xh * s2);
                }
                store_vec<T, V, TAIL>(dX + m * lddx, (k * TPR + t) * V, N, y);
            }
    }
    if (!part) return;
    float* out = part + (int64_t)blockIdx.x * 2 * N;
    if (ROWS == 1) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int col = (k * TPR + t) * V;
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (col + i < N) {
                    out[col + i] = dga[k][i];
                    out[N + col + i] = dbe[k][i];
                }
        }
    } else {                                                        // the waves' sums, in order
        __shared__ float sums[ROWS][TPR * V];
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int which = 0; which < 2; ++which) {
                __syncthreads();
#pragma unroll
                for (int i = 0; i < V; ++i) sums[threadIdx.x / TPR][i * TPR + t] = which ? dbe[k][i] : dga[k][i];
                __syncthreads();
                for (int c = threadIdx.x; c < TPR * V; c += 256) {
                    const int col = k * TPR * V + c;
                    const int at = (c % V) * TPR + c / V;
                    float v = sums[0][at];
#pragma unroll
                    for (int r = 1; r < ROWS; ++r) v = v + sums[r][at];
                    if (col < N) out[which * N + col] = v;
                }
            }
    }
}

// rows too wide for registers: the same, reading the row again for every sum
template <class T>
__global__ void __launch_bounds__(1024)
k_layer_norm_fwd_long(int64_t M, int64_t N, const T* __restrict__ X, int64_t ldx, Weights w, float eps, T* __restrict__ Y, int64_t ldy,
                      float* __restrict__ mean_out, float* __restrict__ rstd_out) {
    __shared__ float red[2][16];
    for (int64_t m = blockIdx.x; m < M; m += gridDim.x) {
        const T* x = X + m * ldx;
        float s = 0.0f, q = 0.0f;
        for (int64_t c = threadIdx.x; c < N; c += 1024) s = s + to_f32(x[c]);
        const float mean = row_add<1024>(s, red[0]) / (float)N;
        for (int64_t c = threadIdx.x; c < N; c += 1024) {
            const float d = to_f32(x[c]) - mean;
            q = __builtin_fmaf(d, d, q);
        }
        const float rstd = 1.0f / __builtin_sqrtf(row_add<1024>(q, red[1]) / (float)N + eps);
        for (int64_t c = threadIdx.x; c < N; c += 1024)
            Y[m * ldy + c] = from_f32<T>(__builtin_fmaf((to_f32(x[c]) - mean) * rstd, w.at<T>(w.gamma, c, 1.0f), w.at<T>(w.beta, c, 0.0f)));
        if (threadIdx.x == 0 && mean_out) {
            mean_out[m] = mean;
            rstd_out[m] = rstd;
        }
    }
}
// column sums go through the workgroup's own `part`, which each thread reads and writes at its own columns, row after row: three
// times the traffic of the held form, 1.5 TB/s (1023 x 32768 float32)
template <class T>
__global__ void __launch_bounds__(1024)
k_layer_norm_bwd_long(int64_t M, int64_t N, const T* __restrict__ G, int64_t ldg, const T* __restrict__ X, int64_t ldx,
                      const float* __restrict__ mean, const float* __restrict__ rstd, Weights w, T* __restrict__ dX, int64_t lddx,
                      float* __restrict__ part) {
    __shared__ float red[2][2][16];
    bool first = true;
    int turn = 0;
    for (int64_t m = blockIdx.x; m < M; m += gridDim.x, turn ^= 1) {
        const float mu = mean[m], rs = rstd[m];
        const T *x = X + m * ldx, *gr = G + m * ldg;
        float s1 = 0.0f, s2 = 0.0f;
        for (int64_t c = threadIdx.x; c < N; c += 1024) {
            const float g = to_f32(gr[c]), xh = (to_f32(x[c]) - mu) * rs, gg = g * w.at<T>(w.gamma, c, 1.0f);
            if (part) {
                float* p = part + (int64_t)blockIdx.x * 2 * N + c;
                p[0] = __builtin_fmaf(g, xh, first ? 0.0f : p[0]);
                p[N] = (first ? 0.0f : p[N]) + g;
            }
            s1 = s1 + gg;
            s2 = __builtin_fmaf(gg, xh, s2);
        }
        first = false;
        row_add<1024>(s1, s2, red[turn]);
        s1 = s1 / (float)N;
        s2 = s2 / (float)N;
        if (dX)
            for (int64_t c = threadIdx.x; c < N; c += 1024) {
                const float xh = (to_f32(x[c]) - mu) * rs;
                dX[m * lddx + c] = from_f32<T>(rs * ((to_f32(gr[c]) * w.at<T>(w.gamma, c, 1.0f) - s1) - xh * s2));
            }
    }
}

// dgamma[c], dbeta[c]: 16 lanes of rows each add every 16th workgroup's sums, then the lanes are added in order (512 x 2 x 8192
// sums, 6 us)
template <class W>
__global__ void __launch_bounds__(1024)
k_layer_norm_cols(int64_t nblk, int64_t N, const float* __restrict__ part, W* __restrict__ dgamma, W* __restrict__ dbeta) {
    __shared__ float red[16][64];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const int64_t g = (int64_t)blockIdx.x * 64 + lane;
    float acc = 0.0f;
    if (g < 2 * N)
#pragma unroll 8
        for (int64_t b = wv; b < nblk; b += 16) acc = acc + part[b * 2 * N + g];
    red[wv][lane] = acc;
    __syncthreads();
    if (wv != 0 || g >= 2 * N) return;
#pragma unroll
    for (int k = 1; k < 16; ++k) acc = acc + red[k][lane];
    W* out = g < N ? dgamma : dbeta;
    if (out) out[g < N ? g : g - N] = from_f32<W>(acc);
}

// Threads a row and 16-byte pieces a thread, from the width alone, so that a row's bits do not depend on how many others come
// with it: as few threads as hold the row in four pieces, 8 to a wave (no barrier, several rows a workgroup; 2.8 million rows of
// 24 bf16 took 746 us with a wave each and 96 us with 8 lanes), then 256, 512 and 1024.  tpr = 0: too wide.
struct RowShape { int tpr, K; };
static inline RowShape row_shape(int64_t N, int vec, int most) {
    const int64_t v = (N + vec - 1) / vec;
    if (v <= 8) return {8, 1};
    if (v <= 16) return {16, 1};
    if (v <= 32) return {32, 1};
    for (const int tpr : {64, 256, 512, 1024})
        if (v <= 4 * tpr) return {tpr, (int)((v + tpr - 1) / tpr)};
    return v <= 8 * 1024 && most >= 8 ? RowShape{1024, 8} : RowShape{0, 0};
}
// workgroups of the forward: what the CUs hold at once
static inline int64_t norm_blocks_fwd(int64_t M, int rows, int threads) {
    const int64_t want = (M + rows - 1) / rows, most = 256 * (1024 / threads);
    return want < most ? want : most;
}
// Workgroups of the backward, each with as many rows as it takes: two on every CU, or one of 512 and 1024 threads that hold their
// row, whose registers leave no room for a second (a second round of them writes the column sums twice: 4095 x 16384 bf16 121
// instead of 99 us).  Rows that are not held (tpr = 0) keep two (1023 x 32768 float32: 270 us, with one 334).
static inline int64_t norm_blocks(int64_t M, int rows, int tpr) {
    const int64_t most = tpr >= 512 ? 256 : 512;
    return M < most * rows ? (M + rows - 1) / rows : most;
}

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
    GM_REQUIRE(M < (1ll << 31) && N < (1ll << 26), "M of 2^31 or more, or N of 2^26 or more")

extern "C" int gm_layer_norm_fwd(int64_t M, int64_t N, const void* X, int64_t ldx, int dtype, const void* gamma, const void* beta,
                                 int weight_dtype, float eps, void* Y, int64_t ldy, float* mean, float* rstd, gm_stream_t stream) {
    GM_NORM_CHECK();
    if (M == 0) return GM_OK;
    GM_REQUIRE(X && Y && ldx >= N && ldy >= N && !mean == !rstd, "bad arguments");
    const Weights w{gamma, beta, weight_dtype == GM_DTYPE_F32};
    return with_dtype(dtype, [&](auto t) -> int {
        using T = decltype(t);
        const RowShape r = row_shape(N, VEC<T>, 8);
#define GM_LAUNCH_NORM(KERNEL, ROWS, THREADS)                                                                             \
    hipLaunchKernelGGL(KERNEL, dim3((unsigned)norm_blocks_fwd(M, ROWS, THREADS)), dim3(THREADS), 0, as_stream(stream), M, N, \
                       static_cast<const T*>(X), ldx, w, eps, static_cast<T*>(Y), ldy, mean, rstd)
        with_row_form<T>(N, [&](auto v, auto tail) {
            constexpr int V = decltype(v)::value;
            constexpr bool TAIL = decltype(tail)::value;
            if constexpr (V == 1) {
                GM_LAUNCH_NORM((k_layer_norm_fwd<T, 1, false, 1, 8>), 32, 256);
            } else {
                switch (r.tpr * 16 + r.K) {
                    case 8 * 16 + 1: GM_LAUNCH_NORM((k_layer_norm_fwd<T, V, TAIL, 1, 8>), 32, 256); break;
                    case 16 * 16 + 1: GM_LAUNCH_NORM((k_layer_norm_fwd<T, V, TAIL, 1, 16>), 16, 256); break;
                    case 32 * 16 + 1: GM_LAUNCH_NORM((k_layer_norm_fwd<T, V, TAIL, 1, 32>), 8, 256); break;
                    case 64 * 16 + 1: GM_LAUNCH_NORM((k_layer_norm_fwd<T, V, TAIL, 1, 64>), 4, 256); break;
                    case 64 * 16 + 2: GM_LAUNCH_NORM((k_layer_norm_fwd<T, V, TAIL, 2, 64>), 4, 256); break;
                    case 64 * 16 + 3: GM_LAUNCH_NORM((k_layer_norm_fwd<T, V, TAIL, 3, 64>), 4, 256); break;
                    case 64 * 16 + 4: GM_LAUNCH_NORM((k_layer_norm_fwd<T, V, TAIL, 4, 64>), 4, 256); break;
                    case 256 * 16 + 2: GM_LAUNCH_NORM((k_layer_norm_fwd<T, V, TAIL, 2, 256>), 1, 256); break;
                    case 256 * 16 + 3: GM_LAUNCH_NORM((k_layer_norm_fwd<T, V, TAIL, 3, 256>), 1, 256); break;
                    case 256 * 16 + 4: GM_LAUNCH_NORM((k_layer_norm_fwd<T, V, TAIL, 4, 256>), 1, 256); break;
                    case 512 * 16 + 3: GM_LAUNCH_NORM((k_layer_norm_fwd<T, V, TAIL, 3, 512>), 1, 512); break;
                    case 512 * 16 + 4: GM_LAUNCH_NORM((k_layer_norm_fwd<T, V, TAIL, 4, 512>), 1, 512); break;
                    case 1024 * 16 + 3: GM_LAUNCH_NORM((k_layer_norm_fwd<T, V, TAIL, 3, 1024>), 1, 1024); break;
                    case 1024 * 16 + 4: GM_LAUNCH_NORM((k_layer_norm_fwd<T, V, TAIL, 4, 1024>), 1, 1024); break;
                    case 1024 * 16 + 8: GM_LAUNCH_NORM((k_layer_norm_fwd<T, V, TAIL, 8, 1024>), 1, 1024); break;
                    default: GM_LAUNCH_NORM((k_layer_norm_fwd_long<T>), 1, 1024); break;
                }
            }
        });
#undef GM_LAUNCH_NORM
        GM_LAUNCH_CHECK();
        return GM_OK;
    });
}

extern "C" int64_t gm_layer_norm_bwd_workspace_bytes(int64_t M, int64_t N) {
    if (M < 0 || N <= 0 || M >= (1ll << 31) || N >= (1ll << 26)) return -1;
    return norm_blocks(M, 1, 0) * 2 * N * 4;                 // whatever the row type
}

extern "C" int gm_layer_norm_bwd(int64_t M, int64_t N, const void* G, int64_t ldg, const void* X, int64_t ldx, int dtype,
                                 const float* mean, const float* rstd, const void* gamma, int weight_dtype, void* dX, int64_t lddx,
                                 void* dgamma, void* dbeta, void* workspace, int64_t workspace_bytes, gm_stream_t stream) {
    GM_NORM_CHECK();
    GM_REQUIRE(M == 0 || (G && X && mean && rstd && ldg >= N && ldx >= N && (!dX || lddx >= N)), "bad arguments");
    const bool cols = dgamma || dbeta;
    int64_t nblk = norm_blocks(M, 1, 0);
    const int64_t need = nblk * 2 * N * 4;
    GM_REQUIRE(!cols || M == 0 || (workspace && workspace_bytes >= need && aligned(workspace, 16)),
               "gm_layer_norm_bwd needs %lld workspace bytes (gm_layer_norm_bwd_workspace_bytes)", (long long)need);
    hipStream_t s = as_stream(stream);
    float* part = cols ? static_cast<float*>(workspace) : nullptr;
    return with_weight_dtype(dtype, weight_dtype, [&](auto t, auto u) -> int {
        using T = decltype(t);
        using W = decltype(u);
        if (M > 0) {
            const Weights w{gamma, nullptr, weight_dtype == GM_DTYPE_F32};
            const RowShape r = row_shape(N, VEC<T>, 4);
#define GM_LAUNCH_NORM(KERNEL, ROWS, THREADS)                                                                             \
    do {                                                                                                                  \
        nblk = norm_blocks(M, ROWS, r.tpr);                                                                                        \
        hipLaunchKernelGGL(KERNEL, dim3((unsigned)nblk), dim3(THREADS), 0, s, M, N, static_cast<const T*>(G), ldg,        \
                           static_cast<const T*>(X), ldx, mean, rstd, w, static_cast<T*>(dX), lddx, part);                \
    } while (0)
            with_row_form<T>(N, [&](auto v, auto tail) {
                constexpr int V = decltype(v)::value;
                constexpr bool TAIL = decltype(tail)::value;
                if constexpr (V == 1) {
                    GM_LAUNCH_NORM((k_layer_norm_bwd<T, 1, false, 1, 8>), 32, 256);
                } else {
                    switch (r.tpr * 16 + r.K) {
                        case 8 * 16 + 1: GM_LAUNCH_NORM((k_layer_norm_bwd<T, V, TAIL, 1, 8>), 32, 256); break;
                        case 16 * 16 + 1: GM_LAUNCH_NORM((k_layer_norm_bwd<T, V, TAIL, 1, 16>), 16, 256); break;
                        case 32 * 16 + 1: GM_LAUNCH_NORM((k_layer_norm_bwd<T, V, TAIL, 1, 32>), 8, 256); break;
                        case 64 * 16 + 1: GM_LAUNCH_NORM((k_layer_norm_bwd<T, V, TAIL, 1, 64>), 4, 256); break;
                        case 64 * 16 + 2: GM_LAUNCH_NORM((k_layer_norm_bwd<T, V, TAIL, 2, 64>), 4, 256); break;
                        case 64 * 16 + 3: GM_LAUNCH_NORM((k_layer_norm_bwd<T, V, TAIL, 3, 64>), 4, 256); break;
                        case 64 * 16 + 4: GM_LAUNCH_NORM((k_layer_norm_bwd<T, V, TAIL, 4, 64>), 4, 256); break;
                        case 256 * 16 + 2: GM_LAUNCH_NORM((k_layer_norm_bwd<T, V, TAIL, 2, 256>), 1, 256); break;
                        case 256 * 16 + 3: GM_LAUNCH_NORM((k_layer_norm_bwd<T, V, TAIL, 3, 256>), 1, 256); break;
                        case 256 * 16 + 4: GM_LAUNCH_NORM((k_layer_norm_bwd<T, V, TAIL, 4, 256>), 1, 256); break;
                        case 512 * 16 + 3: GM_LAUNCH_NORM((k_layer_norm_bwd<T, V, TAIL, 3, 512>), 1, 512); break;
                        case 512 * 16 + 4: GM_LAUNCH_NORM((k_layer_norm_bwd<T, V, TAIL, 4, 512>), 1, 512); break;
                        case 1024 * 16 + 3: GM_LAUNCH_NORM((k_layer_norm_bwd<T, V, TAIL, 3, 1024>), 1, 1024); break;
                        case 1024 * 16 + 4: GM_LAUNCH_NORM((k_layer_norm_bwd<T, V, TAIL, 4, 1024>), 1, 1024); break;
                        default: GM_LAUNCH_NORM((k_layer_norm_bwd_long<T>), 1, 1024); break;
                    }
                }
            });
#undef GM_LAUNCH_NORM
            GM_LAUNCH_CHECK();
        }
        if (cols) {
            hipLaunchKernelGGL((k_layer_norm_cols<W>), dim3((unsigned)((2 * N + 63) / 64)), dim3(1024), 0, s, nblk, N, part,
                               static_cast<W*>(dgamma), static_cast<W*>(dbeta));
            GM_LAUNCH_CHECK();
        }
        return GM_OK;
    });
}
