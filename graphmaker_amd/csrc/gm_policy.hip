// gm_policy.hip -- losses over the log-probabilities of a batch of ragged sequences (answers, or the draws of generated
// graphs, each under the distribution it was drawn from): the clipped policy loss with a KL term, and the preference loss of
// pairs.  Item i has log-probability l under the trained model, `old` under the one that drew it and `ref` under a fixed
// reference; a sequence is a run of items [offsets[s], offsets[s+1]).  An item is live if it is inside a sequence and its mask
// byte is set; the values of the others are never used.
//
//   policy       r = exp(l - old),  t = -min(r A, clip(r, 1 - low, 1 + high) A) + k (exp(q) - q - 1),  q = ref - l
//                loss = mean of t over the live items, or mean over sequences of each one's mean
//                dt/dl = (0 where the clipped product is the smaller one, else -r A) + k (1 - exp(q))
//   preference   h_s = sum (or mean) over the live items of l - ref,  z = beta (h_2p - h_2p+1)
//                loss = mean over pairs of -(1 - e) log sig(z) - e log sig(-z),  dloss/dz = (sig(z) - (1 - e)) / P
//
// Both make one pass over the items and reduce per sequence: a workgroup takes `chunk` consecutive items, whatever the
// sequences' lengths, and sums each sequence's piece in float64 (the losses are small differences of long sums).  A
// sequence inside one chunk has its sum at once; one that crosses chunks has a piece per chunk, added in ascending order.
// The order of every sum depends on (M, offsets) alone.  Offsets that decrease or leave [0, M] read and write no memory
// out of range; the results are then unspecified.
#include "gm_rows.h"

namespace gm {

constexpr int SEQ_FUSED = 64;        // sequences up to which one workgroup both gathers the pieces and forms the loss
// Sequences up to which one workgroup forms the loss and the weights (8000: 9 us, in two launches 12), and the most workgroups that
// do beyond.
constexpr int SEQ_ONE = 8192, FINISH_BLOCKS = 256;
static inline unsigned finish_blocks(int64_t S) {
    const int64_t want = S <= SEQ_ONE ? 1 : (S + 4095) / 4096;
    return (unsigned)(want < FINISH_BLOCKS ? want : FINISH_BLOCKS);
}

struct Sequences {
    IndexArray offsets;              // p == NULL: all items are one sequence
    int64_t S, M;
    __device__ __forceinline__ int64_t lo(int64_t s) const {
        if (!offsets.p) return 0;
        const int64_t v = offsets.at(s);
        return v < 0 ? 0 : v > M ? M : v;
    }
    __device__ __forceinline__ int64_t hi(int64_t s) const {
        if (!offsets.p) return M;
        const int64_t v = offsets.at(s + 1);
        return v < 0 ? 0 : v > M ? M : v;
    }
    // the last sequence of [first, last] that starts at or before item i (first if none does)
    __device__ __forceinline__ int64_t of(int64_t i, int64_t first, int64_t last) const {
        if (!offsets.p) return 0;
        while (first < last) {
            const int64_t mid = (first + last + 1) >> 1;
            if (offsets.at(mid) <= i) first = mid;
            else last = mid - 1;
        }
        return first;
    }
    // the same for a whole wave and one i: 64 starts are tried at once, so that the search waits once per factor of 64
    __device__ __forceinline__ int64_t of_wave(int64_t i, int64_t first, int64_t last) const {
        if (!offsets.p) return 0;
        while (first < last) {
            const int64_t step = (last - first + 63) / 64;           // tries first + step, first + 2 step, ... up to last
            const int64_t at = first + step * ((threadIdx.x & 63) + 1);
            const int n = __popcll(__ballot(at <= last && offsets.at(at <= last ? at : last) <= i));
            const int64_t next = first + step * (n + 1) - 1;
            first += step * n;
            last = next < last ? next : last;
        }
        return first;
    }
};

// items a workgroup sums: as few as make 2048 chunks (one round of the chip, and the most pieces that one sequence can have)
static inline int64_t chunk_items(int64_t M) { return M <= 2048 * 256 ? 256 : ((M + 2047) / 2048 + 255) / 256 * 256; }
// items a workgroup of the gradient writes: it joins nothing, so its chunks stay short (10.5 million items: 30 us in chunks
// of 6144, whose workgroups all look for their sequence at once and then all write, 18 us in chunks of 2048)
static inline int64_t spread_items(int64_t M) { return M <= 1024 * 512 ? 512 : 2048; }

template <int Q> struct alignas(8) Sums { double v[Q]; };

// A batch's items are formed times `unit`, 2^-20 / M rounded down to a power of two: e^89 leaves float32, its share of the mean and
// the KL coefficient's share of that do not.  What it takes from the small side, values below 2^-72, is nothing beside any other
// item.  The sums take the unit back at the end, the weights of the gradient carry it the other way round.
struct Unit { float u; int shift; };                     // u = 2^-shift
static inline Unit item_unit(int64_t M) {
    const int shift = 20 + (M > 0 ? 63 - __builtin_clzll((unsigned long long)M) : 0);
    return {1.0f / (float)(1ull << shift), shift};
}
// exp(x) 2^-shift within about two units in the last place: exp_any with its power of two put on at the end
__device__ __forceinline__ float exp_shifted(float x, int shift) {
    x = x < -2000.0f ? -2000.0f : x > 2000.0f ? 2000.0f : x;   // 0 and infinity either way
    const float t = x * 1.44269502f, n = __builtin_rintf(t);
    const float lo = __builtin_fmaf(x, 1.92596299e-8f, __builtin_fmaf(x, 1.44269502f, -t));
    return __builtin_ldexpf(__builtin_amdgcn_exp2f(t - n) * __builtin_fmaf(lo, 0.693147182f, 1.0f), (int)n - shift);
}
// (exp(x) - 1 - x) / x^2 for |x| < 1 (the first term left out is below 1.2 x 2^-24 of the sum)
__device__ __forceinline__ float exp_series(float x) {
    float p = 2.75573192e-7f;                           // 1/10!
    p = __builtin_fmaf(p, x, 2.75573192e-6f);
    p = __builtin_fmaf(p, x, 2.48015873e-5f);
    p = __builtin_fmaf(p, x, 1.98412698e-4f);
    p = __builtin_fmaf(p, x, 1.38888889e-3f);
    p = __builtin_fmaf(p, x, 8.33333333e-3f);
    p = __builtin_fmaf(p, x, 4.16666667e-2f);
    p = __builtin_fmaf(p, x, 1.66666667e-1f);
    return __builtin_fmaf(p, x, 0.5f);
}

// What an item adds to its sequence's sums: `add` takes W consecutive items of one sequence, loads first.  An item's exponentials
// are float32, and carry |x| 2^-24 from the rounded difference x of two float32 log-probabilities, which carry as much themselves.
// Below |x| = 1, where a model and its near past lie, they are 1 and a small part from the series, off by a few 2^-24 of the part:
// nothing cancels, and the gain, formed of both in float64 as the clip borders are, keeps its places where advantages cancel.
// Beyond they are exp_shifted, behind a branch.  (10,547,784 items take 42 us, and 5 more where every wave has items beyond;
// two float32 exponentials without the branch take 43.6, float64 made of them 47, float64 exponentials 54.)
template <bool MASK, bool REF, bool ITEM_ADV> struct PolicyTerm {
    static constexpr int Q = 4;                          // sums: surrogate, KL, clipped items, live items
    struct Acc { double surrogate = 0.0, kl = 0.0; int cut = 0, live = 0; };
    const float *lp, *old, *adv, *ref;
    const uint8_t* mask;
    Unit unit;
    double low, high;                                    // 1 - clip_low and 1 + clip_high, times the unit
    float low_f, high_f, kl;                             // the same, KL coefficient
    float* slope;
    __device__ __forceinline__ float of_sequence(int64_t s) const { return ITEM_ADV ? 0.0f : adv[s]; }
    template <int W> __device__ __forceinline__ void add(int64_t i, float of_seq, Acc& a) const {
        using F = Vec<float, W>;
        const F l = *reinterpret_cast<const F*>(lp + i), o = *reinterpret_cast<const F*>(old + i);
        F A, q, d;
        Vec<uint8_t, W> on;
        if constexpr (ITEM_ADV) A = *reinterpret_cast<const F*>(adv + i);
        if constexpr (REF) q = *reinterpret_cast<const F*>(ref + i);
        if constexpr (MASK) on = *reinterpret_cast<const Vec<uint8_t, W>*>(mask + i);
#pragma unroll
        for (int k = 0; k < W; ++k) {
            const bool live = !MASK || on.v[k] != 0;
            const float adv_k = ITEM_ADV ? A.v[k] : of_seq, d_k = l.v[k] - o.v[k];
            // the ratio is base + part, the KL argument's exponential less 1 and less a line are `one` and `line`; all times the unit
            const float u = unit.u, x = REF ? q.v[k] - l.v[k] : 0.0f, du = d_k * u, xu = x * u;
            float base = u, part = __builtin_fmaf(exp_series(d_k) * d_k, du, du);
            float line = REF ? exp_series(x) * x * xu : 0.0f, one = xu + line;
            if (__builtin_expect(!(__builtin_fabsf(d_k) < 1.0f && __builtin_fabsf(x) < 1.0f), 0)) {
                if (!(__builtin_fabsf(d_k) < 1.0f)) {    // no advantage: 0 for any finite ratio, also one past float32; NaN for an infinite one
                    base = 0.0f;
                    part = adv_k == 0.0f && d_k < INFINITY ? 0.0f : exp_shifted(d_k, unit.shift);
                }
                if (!(__builtin_fabsf(x) < 1.0f)) {
                    one = exp_shifted(x, unit.shift) - u;
                    line = one - xu;
                }
            }
            const float r = base + part;
            const bool cut = (adv_k > 0.0f && r > high_f) || (adv_k < 0.0f && r < low_f);
            const double gain = (cut ? (adv_k > 0.0f ? high : low) : (double)base + (double)part) * (double)adv_k;
            float slope_k = cut ? 0.0f : -(r * adv_k);
            if constexpr (REF) {
                if (kl != 0.0f) slope_k = slope_k - kl * one;
                a.kl += live ? (double)line : 0.0;
            }
            a.surrogate -= live ? gain : 0.0;
            a.cut += live && cut ? 1 : 0;
            a.live += live ? 1 : 0;
            d.v[k] = live ? slope_k : 0.0f;
        }
        if (slope) *reinterpret_cast<F*>(slope + i) = d;
    }
    __device__ __forceinline__ static Sums<4> sums(const Acc& a) { return {{a.surrogate, a.kl, (double)a.cut, (double)a.live}}; }
};

template <bool MASK> struct PreferenceTerm {
    static constexpr int Q = 2;                          // sums: log ratio, live items
    struct Acc { double ratio = 0.0; int live = 0; };
    const float *lp, *ref;
    const uint8_t* mask;
    __device__ __forceinline__ float of_sequence(int64_t) const { return 0.0f; }
    template <int W> __device__ __forceinline__ void add(int64_t i, float, Acc& a) const {
        using F = Vec<float, W>;
        const F l = *reinterpret_cast<const F*>(lp + i), o = *reinterpret_cast<const F*>(ref + i);
        Vec<uint8_t, W> on;
        if constexpr (MASK) on = *reinterpret_cast<const Vec<uint8_t, W>*>(mask + i);
#pragma unroll
        for (int k = 0; k < W; ++k) {
            const bool live = !MASK || on.v[k] != 0;
            a.ratio += live ? (double)l.v[k] - (double)o.v[k] : 0.0;
            a.live += live ? 1 : 0;
        }
    }
    __device__ __forceinline__ static Sums<2> sums(const Acc& a) { return {{a.ratio, (double)a.live}}; }
};

// pieces of the sequences: `whole`[s] of one inside this chunk; `piece`[2k] of one that began before chunk k,
// `piece`[2k+1] of one that begins in it and goes on.  HBM-bound: 10,547,784 items with KL and slopes 42 us, 4.0 TB/s
template <class F>
__global__ void __launch_bounds__(256)
k_sequence_pieces(Sequences q, int64_t chunk, F f, Sums<F::Q>* __restrict__ whole, Sums<F::Q>* __restrict__ piece) {
    constexpr int Q = F::Q;
    __shared__ Sums<Q> red[4];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const int64_t a = (int64_t)blockIdx.x * chunk, b = a + chunk < q.M ? a + chunk : q.M;
    const int64_t s0 = q.of_wave(a, 0, q.S - 1), s1 = q.of_wave(b - 1, s0, q.S - 1);
    if (s1 - s0 >= 64) {                                 // many: a lane each, and a wave together for those of over 32 items
        for (int64_t base = s0 + wv * 64; base <= s1; base += 256) {
            const int64_t s = base + lane;
            const int64_t lo = s <= s1 ? q.lo(s) : 0, hi = s <= s1 ? q.hi(s) : 0;
            const int64_t i0 = lo > a ? lo : a, i1 = hi < b ? hi : b;
            Sums<Q>* to = lo >= a && hi <= b ? whole + s : piece + 2 * (int64_t)blockIdx.x + (lo < a ? 0 : 1);
            if (i0 < i1 && i1 - i0 <= 32) {
                const float of_seq = f.of_sequence(s);
                typename F::Acc acc;
                for (int64_t i = i0; i < i1; ++i) f.template add<1>(i, of_seq, acc);
                *to = F::sums(acc);
            }
            for (uint64_t left = __ballot(i1 - i0 > 32); left; left &= left - 1) {
                const int from = __ffsll((unsigned long long)left) - 1;
                const int64_t j0 = __shfl(i0, from), j1 = __shfl(i1, from);
                const float of_seq = f.of_sequence(base + from);
                typename F::Acc acc;
                for (int64_t i = j0 + lane; i < j1; i += 64) f.template add<1>(i, of_seq, acc);
                Sums<Q> sum = F::sums(acc);
#pragma unroll
                for (int c = 0; c < Q; ++c) sum.v[c] = wave_add(sum.v[c]);
                if (lane == from) *to = sum;
            }
        }
        return;
    }
    const bool alone = s0 == s1;                         // one sequence: all four waves sum it together, else one wave each
    const int t = alone ? (int)threadIdx.x : lane, threads = alone ? 256 : 64;
    for (int64_t s = s0 + (alone ? 0 : wv); s <= s1; s += 4) {
        const int64_t lo = q.lo(s), hi = q.hi(s);
        const int64_t i0 = lo > a ? lo : a, i1 = hi < b ? hi : b;
        if (i0 >= i1) continue;                          // uniform over the workgroup if `alone`, over the wave if not
        const float of_seq = f.of_sequence(s);
        typename F::Acc acc;
        for (int64_t i = i0 + 8 * t; i + 8 <= i1; i += 8 * threads) f.template add<8>(i, of_seq, acc);
        const int64_t rest = i0 + (i1 - i0) / 8 * 8 + t;
        if (rest < i1) f.template add<1>(rest, of_seq, acc);
        Sums<Q> sum = F::sums(acc);
#pragma unroll
        for (int c = 0; c < Q; ++c) sum.v[c] = wave_add(sum.v[c]);
        if (alone) {
            if (lane == 0) red[wv] = sum;
            __syncthreads();
#pragma unroll
            for (int c = 0; c < Q; ++c) sum.v[c] = ((red[0].v[c] + red[1].v[c]) + red[2].v[c]) + red[3].v[c];
        }
        if (lane == 0 && (wv == 0 || !alone)) {
            Sums<Q>* to = lo >= a && hi <= b ? whole + s : piece + 2 * (int64_t)blockIdx.x + (lo < a ? 0 : 1);
            *to = sum;
        }
    }
}

// sums of sequence s by LANES lanes, the first of which gets them
template <int Q, int LANES>
__device__ __forceinline__ Sums<Q> gather_sequence(const Sequences& q, int64_t chunk, int64_t s, int lane, const Sums<Q>* __restrict__ whole,
                                                   const Sums<Q>* __restrict__ piece) {
    const int64_t lo = q.lo(s), hi = q.hi(s);
    Sums<Q> acc = {};
    if (lo < hi) {
        const int64_t k0 = lo / chunk, k1 = (hi - 1) / chunk;
        if (k0 == k1) return whole[s];
#pragma unroll 4
        for (int64_t k = k0 + lane; k <= k1; k += LANES)
#pragma unroll
            for (int c = 0; c < Q; ++c) acc.v[c] += piece[2 * k + (k == k0 ? 1 : 0)].v[c];
#pragma unroll
        for (int c = 0; c < Q; ++c)
#pragma unroll
            for (int off = LANES / 2; off >= 1; off >>= 1) acc.v[c] = acc.v[c] + __shfl_xor(acc.v[c], off);
    }
    return acc;
}
template <int Q>
__global__ void __launch_bounds__(256)
k_sequence_gather(Sequences q, int64_t chunk, int per, Sums<Q>* __restrict__ whole, const Sums<Q>* __restrict__ piece) {
    // a lane looks at each of a wave's `per` sequences, the wave sums those that cross chunks: all of a few thousand may, of
    // more only as many as there are chunks (whole loss with one and with 64 a wave: 8000 sequences 29 and 50 us, 16,384 32 and
    // 30, a million 200 and 58)
    const int lane = threadIdx.x & 63;
    const int64_t step = (int64_t)gridDim.x * 4 * per;
    for (int64_t base = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * per; base < q.S; base += step) {
        const int64_t s = base + lane;
        const bool mine = lane < per && s < q.S;
        const int64_t lo = mine ? q.lo(s) : 0, hi = mine ? q.hi(s) : 0;
        if (mine && lo >= hi) whole[s] = Sums<Q>{};
        for (uint64_t left = __ballot(lo < hi && lo / chunk != (hi - 1) / chunk); left; left &= left - 1) {
            const int64_t t = base + __ffsll((unsigned long long)left) - 1;
            const Sums<Q> sum = gather_sequence<Q, 64>(q, chunk, t, lane, whole, piece);
            if (lane == 0) whole[t] = sum;
        }
    }
}
// the same into LDS by a workgroup of 1024 threads, for up to SEQ_FUSED sequences: all of them at once
template <int Q, int LANES>
__device__ __forceinline__ void gather_all(const Sequences& q, int64_t chunk, const Sums<Q>* __restrict__ whole,
                                           const Sums<Q>* __restrict__ piece, Sums<Q>* held) {
    const int64_t s = threadIdx.x / LANES;
    const int lane = threadIdx.x & (LANES - 1);
    if (s < q.S) {
        const Sums<Q> sum = gather_sequence<Q, LANES>(q, chunk, s, lane, whole, piece);
        if (lane == 0) held[s] = sum;
    }
    __syncthreads();
}
template <int Q>
__device__ __forceinline__ void gather_all(const Sequences& q, int64_t chunk, const Sums<Q>* __restrict__ whole,
                                           const Sums<Q>* __restrict__ piece, Sums<Q>* held) {
    if (q.S <= 16) gather_all<Q, 64>(q, chunk, whole, piece, held);
    else gather_all<Q, 1024 / SEQ_FUSED>(q, chunk, whole, piece, held);
}

// sums over a workgroup of 1024 threads, in every thread
template <int N> __device__ __forceinline__ void block_add(double (&v)[N], double (*red)[N]) {
#pragma unroll
    for (int c = 0; c < N; ++c) v[c] = wave_add(v[c]);
    if ((threadIdx.x & 63) == 0)
#pragma unroll
        for (int c = 0; c < N; ++c) red[threadIdx.x >> 6][c] = v[c];
    __syncthreads();
#pragma unroll
    for (int c = 0; c < N; ++c) {
        v[c] = 0.0;
#pragma unroll
        for (int k = 0; k < 16; ++k) v[c] = v[c] + red[k][c];
    }
}

// what sequence s adds to a batch's totals: the sums, live items, sequences that have one
__device__ __forceinline__ void add_sequence(const Sums<4>& w, int by_sequence, double (&tot)[5]) {
    const double unit = w.v[3] > 0.0 && by_sequence ? 1.0 / w.v[3] : 1.0;
    tot[4] += w.v[3] > 0.0 ? 1.0 : 0.0;
#pragma unroll
    for (int c = 0; c < 3; ++c) tot[c] += w.v[c] * unit;
    tot[3] += w.v[3];
}
// totals of a workgroup's share of many sequences
__global__ void __launch_bounds__(1024)
k_policy_totals(int64_t S, int by_sequence, const Sums<4>* __restrict__ whole, Sums<5>* __restrict__ totals) {
    __shared__ double red[16][5];
    double tot[5] = {0.0, 0.0, 0.0, 0.0, 0.0};
#pragma unroll 4
    for (int64_t s = (int64_t)blockIdx.x * 1024 + threadIdx.x; s < S; s += (int64_t)gridDim.x * 1024) add_sequence(whole[s], by_sequence, tot);
    block_add(tot, red);
    if (threadIdx.x == 0)
#pragma unroll
        for (int c = 0; c < 5; ++c) totals[blockIdx.x].v[c] = tot[c];
}
// The losses and the sequences' weights.  One workgroup up to SEQ_ONE sequences: 8 us, latency of the pieces, the sums and the
// weights one behind the other.  Beyond, every workgroup adds all workgroups' totals in order and writes its share of the weights
// (100,000 sequences 14 us with k_policy_totals, by one workgroup 160; 4 million 48 us, by one 3900).
__global__ void __launch_bounds__(1024)
k_policy_finish(Sequences q, int64_t chunk, int gather, int by_sequence, float kl, float unit, const Sums<4>* __restrict__ whole,
                const Sums<4>* __restrict__ piece, const Sums<5>* __restrict__ totals, float* __restrict__ loss, float* __restrict__ stats,
                float* __restrict__ weight) {
    __shared__ double red[16][5];
    __shared__ Sums<4> held[SEQ_FUSED];
    if (gather) gather_all<4>(q, chunk, whole, piece, held);
    double tot[5] = {0.0, 0.0, 0.0, 0.0, 0.0};
    if (gridDim.x > 1) {
        if (threadIdx.x < gridDim.x)
#pragma unroll
            for (int c = 0; c < 5; ++c) tot[c] = totals[threadIdx.x].v[c];
    } else {
#pragma unroll 4
        for (int64_t s = threadIdx.x; s < q.S; s += 1024) add_sequence(gather ? held[s] : whole[s], by_sequence, tot);
    }
    block_add(tot, red);
    const double over = by_sequence ? tot[4] : tot[3];
    const double norm = over > 0.0 ? 1.0 / over : 0.0;    // no live item: the loss and every gradient are 0
#pragma unroll 4
    for (int64_t s = (int64_t)blockIdx.x * 1024 + threadIdx.x; s < q.S; s += (int64_t)gridDim.x * 1024) {
        const double n = gather ? held[s].v[3] : whole[s].v[3];
        if (weight) weight[s] = n > 0.0 ? (float)((by_sequence ? norm / n : norm) / (double)unit) : 0.0f;
    }
    if (threadIdx.x == 0 && blockIdx.x == 0) {
        const double surrogate = tot[0] * norm / (double)unit, apart = tot[1] * norm / (double)unit;
        loss[0] = (float)(kl != 0.0f ? surrogate + (double)kl * apart : surrogate);
        stats[0] = (float)surrogate;
        stats[1] = (float)apart;
        stats[2] = (float)(tot[2] * norm);
        stats[3] = (float)tot[3];
    }
}

__global__ void __launch_bounds__(1024)
k_preference_finish(Sequences q, int64_t chunk, int gather, double beta, double smoothing, int average, const Sums<2>* __restrict__ whole,
                    const Sums<2>* __restrict__ piece, double* __restrict__ totals, float* __restrict__ loss, float* __restrict__ rewards,
                    float* __restrict__ weight) {
    __shared__ double red[16][1];
    __shared__ Sums<2> held[SEQ_FUSED];
    if (gather) gather_all<2>(q, chunk, whole, piece, held);
    const int64_t P = q.S / 2;
    double tot[1] = {0.0};
#pragma unroll 2
    for (int64_t p = (int64_t)blockIdx.x * 1024 + threadIdx.x; p < P; p += (int64_t)gridDim.x * 1024) {
        double h[2], unit[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const Sums<2> w = gather ? held[2 * p + k] : whole[2 * p + k];
            unit[k] = average && w.v[1] > 1.0 ? 1.0 / w.v[1] : 1.0;
            h[k] = w.v[0] * unit[k];
            rewards[2 * p + k] = (float)(beta * h[k]);
        }
        const double z = beta * (h[0] - h[1]), e = exp(-fabs(z));
        const double up = (z < 0.0 ? -z : 0.0) + log1p(e), down = (z > 0.0 ? z : 0.0) + log1p(e);    // -log sig(z), -log sig(-z); z NaN: e is
        tot[0] += smoothing != 0.0 ? (1.0 - smoothing) * up + smoothing * down : up;
        const double dz = (smoothing - (z >= 0.0 ? e : 1.0) / (1.0 + e)) / (double)P;    // sig(z) - 1 = -sig(-z)
        if (weight) {
            weight[2 * p] = (float)(beta * dz * unit[0]);
            weight[2 * p + 1] = (float)(-beta * dz * unit[1]);
        }
    }
    block_add(tot, red);
    if (threadIdx.x == 0) {
        if (gridDim.x > 1) totals[blockIdx.x] = tot[0];
        else loss[0] = (float)(tot[0] / (double)P);
    }
}
// the loss from the workgroups' totals
__global__ void __launch_bounds__(1024) k_preference_total(int parts, int64_t P, const double* __restrict__ totals, float* __restrict__ loss) {
    __shared__ double red[16][1];
    double tot[1] = {(int)threadIdx.x < parts ? totals[threadIdx.x] : 0.0};
    block_add(tot, red);
    if (threadIdx.x == 0) loss[0] = (float)(tot[0] / (double)P);
}

// dl[i] = g weight[s] slope[i] for the live items of sequence s, 0 for every other item (10,547,784 items 17 us, 4.9 TB/s).  Slope
// and weight are float32, as the gradient is: the first halves what a pass reads, and the three roundings are half a step each.
template <bool SLOPE, bool MASK>
__global__ void __launch_bounds__(256)
k_sequence_spread(Sequences q, int64_t chunk, const float* __restrict__ slope, const uint8_t* __restrict__ mask,
                  const float* __restrict__ weight, const float* __restrict__ g, float* __restrict__ dl) {
    const int64_t a = (int64_t)blockIdx.x * chunk, b = a + chunk < q.M ? a + chunk : q.M;
    const int64_t s0 = q.of_wave(a, 0, q.S - 1), s1 = q.of_wave(b - 1, s0, q.S - 1);
    const float up = g[0];
    auto put = [&](int64_t i, auto width, float w0, int64_t lo, int64_t hi) {       // width items of one sequence [lo, hi)
        constexpr int W = decltype(width)::value;
        Vec<float, W> x, y;
        Vec<uint8_t, W> on;
        if constexpr (SLOPE) x = *reinterpret_cast<const Vec<float, W>*>(slope + i);
        if constexpr (MASK) on = *reinterpret_cast<const Vec<uint8_t, W>*>(mask + i);
#pragma unroll
        for (int k = 0; k < W; ++k) {
            const bool live = i + k >= lo && i + k < hi && (!MASK || on.v[k]);
            y.v[k] = live ? (SLOPE ? w0 * x.v[k] : w0) : 0.0f;
        }
        *reinterpret_cast<Vec<float, W>*>(dl + i) = y;
    };
    if (s0 == s1) {
        const float w0 = weight[s0] * up;
        const int64_t lo = q.lo(s0), hi = q.hi(s0);
        for (int64_t i = a + 8 * (int)threadIdx.x; i < b; i += 2048) {
            if (i + 8 <= b) put(i, std::integral_constant<int, 8>{}, w0, lo, hi);
            else for (int64_t k = i; k < b; ++k) put(k, std::integral_constant<int, 1>{}, w0, lo, hi);
        }
    } else {
        for (int64_t i = a + 8 * (int)threadIdx.x; i < b; i += 2048) {
            int64_t s = q.of(i, s0, s1), lo = q.lo(s), hi = q.hi(s);
            if (i >= lo && i + 8 <= hi && i + 8 <= b) {
                put(i, std::integral_constant<int, 8>{}, weight[s] * up, lo, hi);
                continue;
            }
            for (int64_t k = i; k < i + 8 && k < b; ++k) {
                if (k >= hi && s < s1) {                  // on to the sequence that holds item k
                    s = q.of(k, s, s1);
                    lo = q.lo(s);
                    hi = q.hi(s);
                }
                put(k, std::integral_constant<int, 1>{}, weight[s] * up, lo, hi);
            }
        }
    }
}

static inline unsigned gather_blocks(int64_t S, int per) {
    const int64_t want = (S + 4 * per - 1) / (4 * per);
    return (unsigned)(want < 4096 ? want : 4096);
}

struct SequenceLayout { int64_t nchunk, whole, piece, totals, bytes; };
static inline SequenceLayout sequence_layout(int64_t M, int64_t S) {
    SequenceLayout l;
    const int64_t chunk = chunk_items(M);
    l.nchunk = (M + chunk - 1) / chunk;
    l.whole = 0;
    l.piece = S * (int64_t)sizeof(Sums<4>);
    l.totals = l.piece + 2 * l.nchunk * (int64_t)sizeof(Sums<4>);
    l.bytes = l.totals + (finish_blocks(S) > 1 ? FINISH_BLOCKS * (int64_t)sizeof(Sums<5>) : 0);
    return l;
}

template <class F, class Finish>
static int launch_sequence_loss(const Sequences& q, const F& f, void* workspace, int64_t workspace_bytes, hipStream_t s,
                                Finish&& finish) {
    constexpr int Q = F::Q;
    const SequenceLayout l = sequence_layout(q.M, q.S);
    GM_REQUIRE(workspace && workspace_bytes >= l.bytes && aligned(workspace, 16),
               "needs %lld workspace bytes (gm_sequence_loss_workspace_bytes)", (long long)l.bytes);
    Sums<Q>* whole = reinterpret_cast<Sums<Q>*>(static_cast<char*>(workspace) + l.whole);
    Sums<Q>* piece = reinterpret_cast<Sums<Q>*>(static_cast<char*>(workspace) + l.piece);
    const int64_t chunk = chunk_items(q.M);
    if (l.nchunk > 0) {
        hipLaunchKernelGGL((k_sequence_pieces<F>), dim3((unsigned)l.nchunk), dim3(256), 0, s, q, chunk, f, whole, piece);
        GM_LAUNCH_CHECK();
    }
    const int fused = q.S <= SEQ_FUSED;
    if (!fused) {
        const int per = q.S <= 16384 ? 1 : 64;
        hipLaunchKernelGGL((k_sequence_gather<Q>), dim3(gather_blocks(q.S, per)), dim3(256), 0, s, q, chunk, per, whole, piece);
        GM_LAUNCH_CHECK();
    }
    return finish(chunk, fused, whole, piece, static_cast<void*>(static_cast<char*>(workspace) + l.totals));
}

// fn(b0, b1, ...) with each flag as an integral constant
template <class Fn> static inline int with_flags(bool a, Fn&& fn) { return a ? fn(std::true_type{}) : fn(std::false_type{}); }
template <class Fn> static inline int with_flags(bool a, bool b, Fn&& fn) {
    return with_flags(b, [&](auto y) { return a ? fn(std::true_type{}, y) : fn(std::false_type{}, y); });
}
template <class Fn> static inline int with_flags(bool a, bool b, bool c, Fn&& fn) {
    return with_flags(b, c, [&](auto y, auto z) { return a ? fn(std::true_type{}, y, z) : fn(std::false_type{}, y, z); });
}

}  // namespace gm

using namespace gm;

#define GM_SEQUENCE_CHECK()                                                                                               \
    GM_REQUIRE(M >= 0 && S > 0 && (M == 0 || log_prob), "bad arguments");                                                 \
    GM_REQUIRE(M < (1ll << 34) && S < (1ll << 31), "2^34 items or 2^31 sequences or more")

extern "C" int64_t gm_sequence_loss_workspace_bytes(int64_t M, int64_t S) {
    if (M < 0 || S <= 0 || M >= (1ll << 34) || S >= (1ll << 31)) return -1;
    return sequence_layout(M, S).bytes;
}

extern "C" int gm_policy_loss_fwd(int64_t M, int64_t S, const float* log_prob, const float* old_log_prob, const float* advantage,
                                  const float* ref_log_prob, const uint8_t* mask, const void* offsets, int offsets_i64,
                                  float clip_low, float clip_high, float kl_coef, int by_sequence, float* loss, float* stats,
                                  float* slope, float* weight, void* workspace, int64_t workspace_bytes, gm_stream_t stream) {
    GM_SEQUENCE_CHECK();
    GM_REQUIRE(loss && stats && (M == 0 || (advantage && old_log_prob)) && (offsets || S == 1), "bad arguments");
    GM_REQUIRE(clip_low >= 0.0f && clip_low <= 1.0f && clip_high >= 0.0f && clip_high < INFINITY, "clip range: 0 <= clip_low <= 1, 0 <= clip_high");
    GM_REQUIRE(kl_coef == 0.0f || ref_log_prob, "kl_coef without ref_log_prob");
    GM_REQUIRE(kl_coef - kl_coef == 0.0f, "kl_coef is not finite");
    hipStream_t s = as_stream(stream);
    const Sequences q{IndexArray{offsets, offsets_i64}, S, M};
    const Unit unit = item_unit(M);
    return with_flags(mask != nullptr, ref_log_prob != nullptr, offsets == nullptr, [&](auto m, auto r, auto item) {
        const PolicyTerm<decltype(m)::value, decltype(r)::value, decltype(item)::value> f{
            log_prob, old_log_prob, advantage, ref_log_prob, mask, unit, (1.0 - (double)clip_low) * (double)unit.u,
            (1.0 + (double)clip_high) * (double)unit.u, (1.0f - clip_low) * unit.u, (1.0f + clip_high) * unit.u, kl_coef, slope};
        return launch_sequence_loss(q, f, workspace, workspace_bytes, s, [&](int64_t chunk, int fused, Sums<4>* whole, Sums<4>* piece, void* rest) {
            const unsigned blocks = finish_blocks(S);
            Sums<5>* totals = static_cast<Sums<5>*>(rest);
            if (blocks > 1) {
                hipLaunchKernelGGL(k_policy_totals, dim3(blocks), dim3(1024), 0, s, S, by_sequence, whole, totals);
                GM_LAUNCH_CHECK();
            }
            hipLaunchKernelGGL(k_policy_finish, dim3(blocks), dim3(1024), 0, s, q, chunk, fused, by_sequence, kl_coef, unit.u, whole, piece, totals, loss,
                               stats, weight);
            GM_LAUNCH_CHECK();
            return GM_OK;
        });
    });
}

extern "C" int gm_preference_loss_fwd(int64_t M, int64_t P, const float* log_prob, const float* ref_log_prob, const uint8_t* mask,
                                      const void* offsets, int offsets_i64, float beta, float label_smoothing, int average,
                                      float* loss, float* rewards, float* weight, void* workspace, int64_t workspace_bytes,
                                      gm_stream_t stream) {
    GM_REQUIRE(P > 0 && P < (1ll << 30), "no pair, or too many");
    const int64_t S = 2 * P;
    GM_SEQUENCE_CHECK();
    GM_REQUIRE(loss && rewards && offsets && (M == 0 || ref_log_prob), "bad arguments");
    GM_REQUIRE(beta > 0.0f && beta < INFINITY && label_smoothing >= 0.0f && label_smoothing <= 0.5f,
               "0 < beta and 0 <= label_smoothing <= 0.5");
    hipStream_t s = as_stream(stream);
    const Sequences q{IndexArray{offsets, offsets_i64}, S, M};
    return with_flags(mask != nullptr, [&](auto m) {
        const PreferenceTerm<decltype(m)::value> f{log_prob, ref_log_prob, mask};
        return launch_sequence_loss(q, f, workspace, workspace_bytes, s, [&](int64_t chunk, int fused, Sums<2>* whole, Sums<2>* piece, void* rest) {
            const unsigned blocks = finish_blocks(S);
            double* totals = static_cast<double*>(rest);
            hipLaunchKernelGGL(k_preference_finish, dim3(blocks), dim3(1024), 0, s, q, chunk, fused, (double)beta, (double)label_smoothing,
                               average, whole, piece, totals, loss, rewards, weight);
            GM_LAUNCH_CHECK();
            if (blocks > 1) {
                hipLaunchKernelGGL(k_preference_total, dim3(1), dim3(1024), 0, s, (int)blocks, P, totals, loss);
                GM_LAUNCH_CHECK();
            }
            return GM_OK;
        });
    });
}

extern "C" int gm_sequence_loss_bwd(int64_t M, int64_t S, const float* slope, const uint8_t* mask, const void* offsets, int offsets_i64,
                                    const float* weight, const float* g, float* dlog_prob, gm_stream_t stream) {
    GM_REQUIRE(M >= 0 && S > 0 && M < (1ll << 34) && S < (1ll << 31) && (offsets || S == 1), "bad arguments");
    if (M == 0) return GM_OK;
    GM_REQUIRE(weight && g && dlog_prob, "bad arguments");
    const Sequences q{IndexArray{offsets, offsets_i64}, S, M};
    const int64_t chunk = spread_items(M);
    return with_flags(slope != nullptr, mask != nullptr, [&](auto sl, auto m) -> int {
        hipLaunchKernelGGL((k_sequence_spread<decltype(sl)::value, decltype(m)::value>), dim3((unsigned)((M + chunk - 1) / chunk)), dim3(256), 0,
                           as_stream(stream), q, chunk, slope, mask, weight, g, dlog_prob);
        GM_LAUNCH_CHECK();
        return GM_OK;
    });
}
