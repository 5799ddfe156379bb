// gm_logprob.hip -- log-probability of one class of every row of logits, and its gradient.
//
//   forward    lp[i] = x[i][c_i] - log sum_j exp(x[i][j])
//   gradient   dx[i][j] = g[i] ([j = c_i] - softmax(x[i])[j])
//
// A row whose class is `ignore_index` has log-probability 0 and a zero gradient, whatever its logits; the gradient of a row
// whose g is 0 is 0 too.  Any other class outside [0, V) gives NaN in both.  Sums are float32 whatever the logits' type, of
// exponentials about the row's largest logit.  stats[i] = (largest logit, that sum).
//
// HBM-bound: the forward reads the logits once, the backward reads them and writes as much.  Three forms by the row's size:
//   narrow   under 16 bytes: one thread a row, which forms the softmax again in the backward instead of keeping stats
//   held     up to 5 pieces of 16 bytes a lane: 1 to 64 lanes a row, the row in registers
//   long     a workgroup a row, or several where rows are few, with one running (maximum, sum) a thread
#include "gm_rows.h"

namespace gm {

// exp(x), x <= 0, without exp_any's correction, off by 1.2 |x| 2^-24 relative: for the sums of long rows, where |x| weighted by exp(x) is
// small against the number of additions, and for gradients of 16 bits, beside whose rounding it is nothing (2^-17 at x = -88)
__device__ __forceinline__ float exp_quick(float x) { return __builtin_amdgcn_exp2f(x * 1.44269502f); }

// x inside the row, -inf outside (by masks, as in load_vec)
__device__ __forceinline__ float or_neg_inf(float x, bool in) {
    const uint32_t m = in ? ~0u : 0u;
    return __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, x) & m) | (0xFF800000u & ~m));
}

// ---- narrow: these are draws of few classes, one of them often nearly certain.  Its log-probability -log(1 + rest) and its own
// gradient g (1 - p) are formed from the rest, which cancels nothing, and keep their own places, not those of 1.
// 2,097,152 x 2 float32 with int64 classes 10 us forward, 10.5 us gradient (4.2 and 5.6 TB/s)
constexpr int NARROW_ROWS = 4;                           // rows a thread has in flight
template <class T, int E, bool GRAD>
__global__ void __launch_bounds__(256)
k_log_prob_narrow(int64_t M, const float* __restrict__ g, const T* __restrict__ X, int64_t ldx, IndexArray cls, int64_t ignore,
                  float* __restrict__ lp, T* __restrict__ dX, int64_t lddx) {
    const int64_t step = (int64_t)gridDim.x * 256;
    for (int64_t i0 = (int64_t)blockIdx.x * 256 + threadIdx.x; i0 < M; i0 += step * NARROW_ROWS) {
        Vec<T, E> r[NARROW_ROWS];
        int64_t c[NARROW_ROWS];
        float up[NARROW_ROWS];
#pragma unroll
        for (int u = 0; u < NARROW_ROWS; ++u) {
            const int64_t i = i0 + u * step < M ? i0 + u * step : i0;
            r[u] = *reinterpret_cast<const Vec<T, E>*>(X + i * ldx);
            c[u] = cls.at(i);
            if constexpr (GRAD) up[u] = g[i];
        }
#pragma unroll
        for (int u = 0; u < NARROW_ROWS; ++u) {
            const int64_t i = i0 + u * step;
            if (i >= M) continue;
            float x[E], mx = to_f32(r[u].v[0]), xc = __builtin_nanf("");
            int top = 0;
#pragma unroll
            for (int j = 0; j < E; ++j) {
                x[j] = to_f32(r[u].v[j]);
                top = x[j] > mx ? j : top;
                mx = x[j] > mx ? x[j] : mx;
                if (j == c[u]) xc = x[j];
            }
            float e[E], rest = 0.0f, others = 0.0f;      // sums without the largest one, which is 1, and without the class
#pragma unroll
            for (int j = 0; j < E; ++j) {
                e[j] = exp_any(x[j] - mx);
                rest = rest + (j == top ? e[j] - 1.0f : e[j]);               // 0, or NaN
                others = others + (j == c[u] ? 0.0f : e[j]);
            }
            const float s = 1.0f + rest;
            if constexpr (!GRAD) {
                const float ls = logf(s) + (rest - (s - 1.0f)) / s;          // with what the sum's rounding left out
                lp[i] = c[u] == ignore ? 0.0f : (xc - mx) - ls;
            } else {
                const float gu = c[u] == ignore ? 0.0f : up[u];
                const float bad = gu == 0.0f || (c[u] >= 0 && c[u] < E) ? 0.0f : __builtin_nanf("");
                const float over = gu / s;
                Vec<T, E> d;
#pragma unroll
                for (int j = 0; j < E; ++j)
                    d.v[j] = from_f32<T>(gu == 0.0f ? 0.0f : (j == c[u] ? others : -e[j]) * over + bad);
                *reinterpret_cast<Vec<T, E>*>(dX + i * lddx) = d;
            }
        }
    }
}

// ---- held: LANES lanes a row, K pieces of V elements a lane.  Rows of 64 lanes add enough terms for exp_quick; with exp_any
// the forward of rows of 256 to 2000 bf16 logits is bound by its arithmetic (3.7 to 4.2 TB/s).
template <int LANES> __device__ __forceinline__ float exp_row(float x) { return LANES == 64 ? exp_quick(x) : exp_any(x); }
// an element of the gradient stands for itself: of float32 it has all its places.  It is exp(x - largest) over the row's sum, not
// exp(x - largest - log of the sum), whose argument is rounded twice.
template <class T> __device__ __forceinline__ float exp_grad(float x) { return sizeof(T) == 4 ? exp_any(x) : exp_quick(x); }
template <class T, int V, bool TAIL, int K, int LANES>
__global__ void __launch_bounds__(256)
k_log_prob_held(int64_t M, int N, const T* __restrict__ X, int64_t ldx, IndexArray cls, int64_t ignore, float* __restrict__ lp,
                float2* __restrict__ stats) {
    const int t = threadIdx.x & (LANES - 1);
    const int64_t step = (int64_t)gridDim.x * (256 / LANES);
    for (int64_t m = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES; m < M; m += step) {
        const int64_t c = cls.at(m);
        const bool valid = c >= 0 && c < N;
        const T* row = X + m * ldx;
        const float xc = to_f32(row[valid ? c : 0]);
        Vec<T, V> r[K];
#pragma unroll
        for (int k = 0; k < K; ++k) r[k] = load_vec<T, V, TAIL>(row, (k * LANES + t) * V, N);
        float mx = -INFINITY, s = 0.0f;
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) mx = __builtin_fmaxf(mx, or_neg_inf(to_f32(r[k].v[i]), (k * LANES + t) * V + i < N));
#pragma unroll
        for (int off = LANES / 2; off >= 1; off >>= 1) mx = __builtin_fmaxf(mx, __shfl_xor(mx, off));
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) s = s + exp_row<LANES>(or_neg_inf(to_f32(r[k].v[i]), (k * LANES + t) * V + i < N) - mx);
#pragma unroll
        for (int off = LANES / 2; off >= 1; off >>= 1) s = s + __shfl_xor(s, off);
        if (t == 0) {
            const float ls = logf(s);
            lp[m] = c == ignore ? 0.0f : valid ? (xc - mx) - ls : __builtin_nanf("");
            if (stats) stats[m] = make_float2(mx, s);
        }
    }
}
template <class T, int V, bool TAIL, int K, int LANES>
__global__ void __launch_bounds__(256)
k_log_prob_held_bwd(int64_t M, int N, const float* __restrict__ g, const T* __restrict__ X, int64_t ldx, IndexArray cls, int64_t ignore,
                    const float2* __restrict__ stats, T* __restrict__ dX, int64_t lddx) {
    const int t = threadIdx.x & (LANES - 1);
    const int64_t step = (int64_t)gridDim.x * (256 / LANES);
    for (int64_t m = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES; m < M; m += step) {
        const int64_t c = cls.at(m);
        const float2 st = stats[m];
        const float gu = c == ignore ? 0.0f : g[m];
        const float bad = gu == 0.0f || (c >= 0 && c < N) ? 0.0f : __builtin_nanf(""), over = gu / st.y;
        Vec<T, V> r[K];
#pragma unroll
        for (int k = 0; k < K; ++k) r[k] = load_vec<T, V, TAIL>(X + m * ldx, (k * LANES + t) * V, N);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int col = (k * LANES + t) * V;
            float y[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float v = -over * exp_grad<T>(to_f32(r[k].v[i]) - st.x);
                y[i] = gu == 0.0f ? 0.0f : (col + i == c ? gu + v : v) + bad;
            }
            store_vec<T, V, TAIL>(dX + m * lddx, col, N, y);
        }
    }
}

// ---- long
constexpr int READ_PIECES = 2;                           // pieces of 16 bytes a thread works on while it loads as many
constexpr int LONG_PIECES = 4;                           // pieces of the gradient a thread has in flight
// Elements of a row in front of its first 16-byte boundary.  The gradient of a long row is written from there: 4095 odd rows
// of 50,021 bf16 took 184 us in pieces that straddle boundaries and take 150 us so.  The forward's pieces count from the
// row's start instead: which elements a thread adds, and so the bits of the sum, must not depend on where a row lies.
template <class T> __device__ __forceinline__ int head_of(const T* row) {
    return (int)((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / (int)sizeof(T);
}
constexpr float LOWEST = -3.40282347e+38f;

// running maximum and sum of exp(x - maximum)
struct Running {
    float m = LOWEST, s = 0.0f;                          // a finite start: -inf adds exp(-inf) = 0, never -inf - -inf
    template <int C> __device__ __forceinline__ void add(const float (&x)[C]) {
        float m2 = m;
#pragma unroll
        for (int i = 0; i < C; ++i) m2 = __builtin_fmaxf(m2, x[i]);
        s = s * exp_quick(m - m2);
        m = m2;
#pragma unroll
        for (int i = 0; i < C; ++i) s = s + exp_quick(x[i] - m2);
    }
    __device__ __forceinline__ void add(float om, float os) {
        const float m2 = __builtin_fmaxf(m, om);
        s = s * exp_quick(m - m2) + os * exp_quick(om - m2);
        m = m2;
    }
};

// part[row][blockIdx.y] of columns [blockIdx.y * span, + span); with one part a row (gridDim.y = 1) lp and stats at once.
// 4095 x 50,021 bf16: 98 us, 4.2 TB/s (odd rows straddle lines: 4096 x 50,016 take 84 us)
template <class T>
__global__ void __launch_bounds__(256)
k_log_prob_long(int64_t M, int N, int span, const T* __restrict__ X, int64_t ldx, IndexArray cls, int64_t ignore, float* __restrict__ lp,
                float2* __restrict__ stats, float2* __restrict__ part) {
    constexpr int V = VEC<T>, STEP = 256 * V;
    __shared__ float2 red[4];
    for (int64_t m = blockIdx.x; m < M; m += gridDim.x) {
        const int64_t c = cls.at(m);
        if (c == ignore) {                               // uniform over the workgroup
            if (threadIdx.x == 0 && blockIdx.y == 0) {
                lp[m] = 0.0f;
                if (stats) stats[m] = make_float2(0.0f, 0.0f);
            }
            continue;
        }
        const T* row = X + m * ldx;
        int j = blockIdx.y * span;
        const int end = N - j < span ? N : j + span;
        Running run;
        if (j + READ_PIECES * STEP <= end) {
            Vec<T, V> next[READ_PIECES];
#pragma unroll
            for (int u = 0; u < READ_PIECES; ++u) next[u] = *reinterpret_cast<const Vec<T, V>*>(row + j + u * STEP + threadIdx.x * V);
            for (; j + READ_PIECES * STEP <= end; j += READ_PIECES * STEP) {
                Vec<T, V> now[READ_PIECES];
#pragma unroll
                for (int u = 0; u < READ_PIECES; ++u) now[u] = settled(next[u]);
                const int ahead = j + 2 * READ_PIECES * STEP <= end ? j + READ_PIECES * STEP : j;
#pragma unroll
                for (int u = 0; u < READ_PIECES; ++u) next[u] = *reinterpret_cast<const Vec<T, V>*>(row + ahead + u * STEP + threadIdx.x * V);
                __builtin_amdgcn_sched_barrier(0);
                float x[READ_PIECES * V];
#pragma unroll
                for (int u = 0; u < READ_PIECES; ++u)
#pragma unroll
                    for (int i = 0; i < V; ++i) x[u * V + i] = to_f32(now[u].v[i]);
                run.add(x);
            }
        }
        for (; j < end; j += STEP) {                     // the rest: fewer steps than READ_PIECES, and one that ends inside
            const Vec<T, V> r = load_vec<T, V, true>(row, j + threadIdx.x * V, end);
            float x[V];
#pragma unroll
            for (int i = 0; i < V; ++i) x[i] = or_neg_inf(to_f32(r.v[i]), j + (int)threadIdx.x * V + i < end);
            run.add(x);
        }
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) {
            const float om = __shfl_xor(run.m, off), os = __shfl_xor(run.s, off);
            run.add(om, os);
        }
        __syncthreads();
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = make_float2(run.m, run.s);
        __syncthreads();
        if (threadIdx.x == 0) {
#pragma unroll
            for (int k = 1; k < 4; ++k) run.add(red[k].x, red[k].y);
            if (gridDim.y > 1) {
                part[m * gridDim.y + blockIdx.y] = make_float2(run.m, run.s);
            } else {
                const float ls = logf(run.s);
                lp[m] = c >= 0 && c < N ? (to_f32(row[c]) - run.m) - ls : __builtin_nanf("");
                if (stats) stats[m] = make_float2(run.m, run.s);
            }
        }
    }
}
// joins the parts of a row, one wave a row
template <class T>
__global__ void __launch_bounds__(64)
k_log_prob_join(int N, int parts, const float2* __restrict__ part, const T* __restrict__ X, int64_t ldx, IndexArray cls, int64_t ignore,
                float* __restrict__ lp, float2* __restrict__ stats) {
    const int64_t m = blockIdx.x, c = cls.at(m);
    if (c == ignore) return;
    Running run;
    for (int k = threadIdx.x; k < parts; k += 64) run.add(part[m * parts + k].x, part[m * parts + k].y);
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) {
        const float om = __shfl_xor(run.m, off), os = __shfl_xor(run.s, off);
        run.add(om, os);
    }
    if (threadIdx.x == 0) {
        const float ls = logf(run.s);
        lp[m] = c >= 0 && c < N ? (to_f32(X[m * ldx + c]) - run.m) - ls : __builtin_nanf("");
        if (stats) stats[m] = make_float2(run.m, run.s);
    }
}

// A gradient whose pass moves more than the 256 MB of the last cache goes past it, and so do the logits, which are read for the
// last time (PAST): kept there, they push out what is still to be read, and are themselves gone before a reader comes.
// Forward and gradient of 4095 x 50,021 bf16 one behind the other: 287 -> 247 us.
constexpr int64_t LAST_CACHE = 256ll << 20;
typedef uint32_t Words __attribute__((ext_vector_type(4)));
typedef Words WordsAnywhere __attribute__((aligned(2)));
template <bool PAST, class T, int V> __device__ __forceinline__ void put_vec(T* __restrict__ at, const Vec<T, V>& t) {
    if constexpr (PAST) {
        Words w;
        static_assert(sizeof(t) == sizeof(w), "a piece of 16 bytes");
        __builtin_memcpy(&w, &t, sizeof(w));
        __builtin_nontemporal_store(w, reinterpret_cast<WordsAnywhere*>(at));
    } else {
        *reinterpret_cast<Vec<T, V>*>(at) = t;
    }
}
template <bool PAST, class T, int V> __device__ __forceinline__ Vec<T, V> get_vec(const T* __restrict__ at) {
    if constexpr (PAST) {
        const Words w = __builtin_nontemporal_load(reinterpret_cast<const WordsAnywhere*>(at));
        Vec<T, V> t;
        __builtin_memcpy(&t, &w, sizeof(w));
        return t;
    } else {
        return *reinterpret_cast<const Vec<T, V>*>(at);
    }
}

// columns head + [blockIdx.y * span, + span) of a row, span = LONG_PIECES steps, the head with the first (4095 x 50,021 bf16:
// 140 us, 5.9 TB/s)
template <class T, bool PAST>
__global__ void __launch_bounds__(256)
k_log_prob_long_bwd(int64_t M, int N, const float* __restrict__ g, const T* __restrict__ X, int64_t ldx, IndexArray cls, int64_t ignore,
                    const float2* __restrict__ stats, T* __restrict__ dX, int64_t lddx) {
    constexpr int V = VEC<T>, STEP = 256 * V;
    for (int64_t m = blockIdx.x; m < M; m += gridDim.x) {
        const int64_t c = cls.at(m);
        const float2 st = stats[m];
        const float gu = c == ignore ? 0.0f : g[m];
        const float scale = c >= 0 && c < N ? -gu / st.y : __builtin_nanf("");
        const T* row = X + m * ldx;
        T* out = dX + m * lddx;
        const int head = head_of(out), j = head + blockIdx.y * (LONG_PIECES * STEP) + threadIdx.x * V;
        const bool first = blockIdx.y == 0 && (int)threadIdx.x < head;
        if (gu == 0.0f) {                                // uniform: the row is written without being read
            const float zero[V] = {};
#pragma unroll
            for (int u = 0; u < LONG_PIECES; ++u) store_vec<T, V, true>(out, j + u * STEP, N, zero);
            if (first) out[threadIdx.x] = from_f32<T>(0.0f);
            continue;
        }
        Vec<T, V> r[LONG_PIECES];
        const bool whole = head + (int)(blockIdx.y + 1) * (LONG_PIECES * STEP) <= N;          // uniform
        if (whole) {
#pragma unroll
            for (int u = 0; u < LONG_PIECES; ++u) r[u] = get_vec<PAST, T, V>(row + j + u * STEP);
        } else {
#pragma unroll
            for (int u = 0; u < LONG_PIECES; ++u) r[u] = load_vec<T, V, true>(row, j + u * STEP, N);
        }
        if (first) {
            const float p = scale * exp_grad<T>(to_f32(row[threadIdx.x]) - st.x);
            out[threadIdx.x] = from_f32<T>((int)threadIdx.x == c ? p + gu : p);
        }
#pragma unroll
        for (int u = 0; u < LONG_PIECES; ++u) {
            const int col = j + u * STEP;
            float y[V];
#pragma unroll
            for (int i = 0; i < V; ++i) y[i] = scale * exp_grad<T>(to_f32(r[u].v[i]) - st.x);
            if (c >= col && c < col + V)
#pragma unroll
                for (int i = 0; i < V; ++i) y[i] = col + i == c ? y[i] + gu : y[i];
            if (whole) {
                Vec<T, V> d;
#pragma unroll
                for (int i = 0; i < V; ++i) d.v[i] = from_f32<T>(y[i]);
                put_vec<PAST, T, V>(out + col, d);
            } else {
                store_vec<T, V, true>(out, col, N, y);
            }
        }
    }
}

// Pieces a row, and lanes and pieces a lane of the held form; lanes = 0: long.  Up to five pieces: 20,000 x 1280 float32 are held
// in 17 us forward, 20,000 x 1284 take 34 by a workgroup each.
struct LogProbShape { int lanes, K; };
static inline LogProbShape log_prob_shape(int64_t N, int vec) {
    const int64_t v = (N + vec - 1) / vec;
    int lanes = 1, K = 1;
    while (lanes < 64 && lanes < v) lanes *= 2;
    while ((int64_t)lanes * K < v) ++K;
    return K > 5 ? LogProbShape{0, 0} : LogProbShape{lanes, K};
}
static inline int64_t held_blocks(int64_t M, int lanes) {
    const int64_t want = (M + 256 / lanes - 1) / (256 / lanes);
    return want < 256 * 32 ? want : 256 * 32;
}
// parts of a long row: rows fewer than two workgroups a CU are split, down to 4 steps a part
static inline int64_t long_parts(int64_t M, int64_t N, int vec) {
    const int64_t most = (N + 4 * 256 * vec - 1) / (4 * 256 * vec), want = M < 512 ? 512 / (M ? M : 1) : 1;
    return want < most ? want : most;
}

template <class T, class Fn> static inline void with_held(int64_t N, Fn&& fn) {
    with_row_form<T>(N, [&](auto v, auto tail) {
        if constexpr (decltype(v)::value > 1) {
            const LogProbShape r = log_prob_shape(N, VEC<T>);
            auto with = [&](auto lanes, auto k) { fn(v, tail, k, lanes); };
            using std::integral_constant;
            switch (r.lanes * 16 + r.K) {
                case 1 * 16 + 1: with(integral_constant<int, 1>{}, integral_constant<int, 1>{}); break;
                case 2 * 16 + 1: with(integral_constant<int, 2>{}, integral_constant<int, 1>{}); break;
                case 4 * 16 + 1: with(integral_constant<int, 4>{}, integral_constant<int, 1>{}); break;
                case 8 * 16 + 1: with(integral_constant<int, 8>{}, integral_constant<int, 1>{}); break;
                case 16 * 16 + 1: with(integral_constant<int, 16>{}, integral_constant<int, 1>{}); break;
                case 32 * 16 + 1: with(integral_constant<int, 32>{}, integral_constant<int, 1>{}); break;
                case 64 * 16 + 1: with(integral_constant<int, 64>{}, integral_constant<int, 1>{}); break;
                case 64 * 16 + 2: with(integral_constant<int, 64>{}, integral_constant<int, 2>{}); break;
                case 64 * 16 + 3: with(integral_constant<int, 64>{}, integral_constant<int, 3>{}); break;
                case 64 * 16 + 4: with(integral_constant<int, 64>{}, integral_constant<int, 4>{}); break;
                default: with(integral_constant<int, 64>{}, integral_constant<int, 5>{}); break;
            }
        }
    });
}
template <class T, class Fn> static inline void with_narrow(int64_t N, Fn&& fn) {
    using std::integral_constant;
    switch (N) {
        case 1: fn(integral_constant<int, 1>{}); break;
        case 2: fn(integral_constant<int, 2>{}); break;
        case 3: fn(integral_constant<int, 3>{}); break;
        default:
            if constexpr (VEC<T> > 4) {
                switch (N) {
                    case 4: fn(integral_constant<int, 4>{}); break;
                    case 5: fn(integral_constant<int, 5>{}); break;
                    case 6: fn(integral_constant<int, 6>{}); break;
                    default: fn(integral_constant<int, 7>{}); break;
                }
            }
    }
}
static inline unsigned narrow_blocks(int64_t M) {
    const int64_t want = (M + 256 * NARROW_ROWS - 1) / (256 * NARROW_ROWS);
    return (unsigned)(want < 256 * 16 ? want : 256 * 16);
}

}  // namespace gm

using namespace gm;

#define GM_LOGPROB_CHECK()                                                                                                \
    GM_REQUIRE(M >= 0 && V > 0, "bad arguments");                                                                         \
    GM_REQUIRE(dtype_ok(dtype), "dtype %d is none of GM_DTYPE_*", dtype);                                                 \
    GM_REQUIRE(M < (1ll << 31) && V < (1ll << 27), "M of 2^31 or more, or V of 2^27 or more")

extern "C" int64_t gm_class_log_prob_stats_floats(int64_t M, int64_t V, int dtype) {
    if (M < 0 || V <= 0 || M >= (1ll << 31) || V >= (1ll << 27) || !dtype_ok(dtype)) return -1;
    return V < 16 / dtype_size(dtype) ? 0 : 2 * M;
}

extern "C" int64_t gm_class_log_prob_workspace_bytes(int64_t M, int64_t V, int dtype) {
    if (M < 0 || V <= 0 || M >= (1ll << 31) || V >= (1ll << 27) || !dtype_ok(dtype)) return -1;
    const int vec = 16 / dtype_size(dtype);
    if (V < vec || log_prob_shape(V, vec).lanes) return 0;
    const int64_t parts = long_parts(M, V, vec);
    return parts > 1 ? M * parts * (int64_t)sizeof(float2) : 0;
}

extern "C" int gm_class_log_prob_fwd(int64_t M, int64_t V, const void* logits, int64_t ldx, int dtype, const void* classes,
                                     int classes_i64, int64_t ignore_index, float* log_prob, float* stats, void* workspace,
                                     int64_t workspace_bytes, gm_stream_t stream) {
    GM_LOGPROB_CHECK();
    if (M == 0) return GM_OK;
    GM_REQUIRE(logits && classes && log_prob && ldx >= V && aligned(stats, 8), "bad arguments");
    const int64_t need = gm_class_log_prob_workspace_bytes(M, V, dtype);
    GM_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && aligned(workspace, 8)),
               "gm_class_log_prob_fwd needs %lld workspace bytes (gm_class_log_prob_workspace_bytes)", (long long)need);
    hipStream_t s = as_stream(stream);
    const IndexArray cls{classes, classes_i64};
    float2* st = reinterpret_cast<float2*>(stats);
    return with_dtype(dtype, [&](auto t) -> int {
        using T = decltype(t);
        const T* X = static_cast<const T*>(logits);
        if (V < VEC<T>) {
            with_narrow<T>(V, [&](auto e) {
                hipLaunchKernelGGL((k_log_prob_narrow<T, decltype(e)::value, false>), dim3(narrow_blocks(M)), dim3(256), 0, s, M, nullptr, X,
                                   ldx, cls, ignore_index, log_prob, static_cast<T*>(nullptr), (int64_t)0);
            });
        } else if (const LogProbShape r = log_prob_shape(V, VEC<T>); r.lanes) {
            with_held<T>(V, [&](auto v, auto tail, auto k, auto lanes) {
                hipLaunchKernelGGL((k_log_prob_held<T, decltype(v)::value, decltype(tail)::value, decltype(k)::value, decltype(lanes)::value>),
                                   dim3((unsigned)held_blocks(M, r.lanes)), dim3(256), 0, s, M, (int)V, X, ldx, cls, ignore_index, log_prob, st);
            });
        } else {
            const int64_t parts = long_parts(M, V, VEC<T>), step = 256 * VEC<T>;
            const int64_t span = ((V + parts - 1) / parts + step - 1) / step * step;
            float2* part = static_cast<float2*>(workspace);
            hipLaunchKernelGGL((k_log_prob_long<T>), dim3(grid_for(M, 256), (unsigned)parts), dim3(256), 0, s, M, (int)V, (int)span, X, ldx, cls,
                               ignore_index, log_prob, st, part);
            if (parts > 1) {
                GM_LAUNCH_CHECK();
                hipLaunchKernelGGL((k_log_prob_join<T>), dim3((unsigned)M), dim3(64), 0, s, (int)V, (int)parts, part, X, ldx, cls, ignore_index,
                                   log_prob, st);
            }
        }
        GM_LAUNCH_CHECK();
        return GM_OK;
    });
}

extern "C" int gm_class_log_prob_bwd(int64_t M, int64_t V, const float* g, const void* logits, int64_t ldx, int dtype,
                                     const void* classes, int classes_i64, int64_t ignore_index, const float* stats, void* dlogits,
                                     int64_t lddx, gm_stream_t stream) {
    GM_LOGPROB_CHECK();
    if (M == 0) return GM_OK;
    GM_REQUIRE(g && logits && classes && dlogits && ldx >= V && lddx >= V && aligned(stats, 8), "bad arguments");
    GM_REQUIRE(stats || V < 16 / dtype_size(dtype), "stats missing (gm_class_log_prob_stats_floats)");
    hipStream_t s = as_stream(stream);
    const IndexArray cls{classes, classes_i64};
    const float2* st = reinterpret_cast<const float2*>(stats);
    return with_dtype(dtype, [&](auto t) -> int {
        using T = decltype(t);
        const T* X = static_cast<const T*>(logits);
        T* dX = static_cast<T*>(dlogits);
        if (V < VEC<T>) {
            with_narrow<T>(V, [&](auto e) {
                hipLaunchKernelGGL((k_log_prob_narrow<T, decltype(e)::value, true>), dim3(narrow_blocks(M)), dim3(256), 0, s, M, g, X, ldx, cls,
                                   ignore_index, static_cast<float*>(nullptr), dX, lddx);
            });
        } else if (const LogProbShape r = log_prob_shape(V, VEC<T>); r.lanes) {
            with_held<T>(V, [&](auto v, auto tail, auto k, auto lanes) {
                hipLaunchKernelGGL((k_log_prob_held_bwd<T, decltype(v)::value, decltype(tail)::value, decltype(k)::value, decltype(lanes)::value>),
                                   dim3((unsigned)held_blocks(M, r.lanes)), dim3(256), 0, s, M, (int)V, g, X, ldx, cls, ignore_index, st, dX, lddx);
            });
        } else {
            const int64_t span = LONG_PIECES * 256 * VEC<T>, parts = (V + span - 1) / span;
            const int64_t most = ((1ll << 32) - 1) / 256 / parts;              // a launch has less than 2^32 threads in all
            auto launch = [&](auto past) {
                hipLaunchKernelGGL((k_log_prob_long_bwd<T, decltype(past)::value>), dim3((unsigned)(M < most ? M : most), (unsigned)parts),
                                   dim3(256), 0, s, M, (int)V, g, X, ldx, cls, ignore_index, st, dX, lddx);
            };
            if (2 * M * V * (int64_t)sizeof(T) > LAST_CACHE) launch(std::true_type{});
            else launch(std::false_type{});
        }
        GM_LAUNCH_CHECK();
        return GM_OK;
    });
}
