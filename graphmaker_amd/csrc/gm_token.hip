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

// A row is `tpr` threads wide (a power of two up to the workgroup), V elements a thread and step; a workgroup takes
// FWD_ROWS rows per thread so that their loads are in flight together (the address of each waits for its token).  HBM-bound: 130,941
// rows of 1024 bf16 71 us, 4.4 TB/s of the rows written and the 22,000 different ones read.
constexpr int FWD_ROWS = 4;
template <class T, int V, bool TAIL>
__global__ void __launch_bounds__(256)
k_token_embedding_fwd(int64_t n, int64_t C, int w, int shift, IndexArray tok, const T* __restrict__ W, int64_t ldw, float scale,
                      T* __restrict__ out, int64_t ldo) {
    const int tpr = 1 << shift, rows = 256 >> shift;
    const int t = threadIdx.x & (tpr - 1);
    const int64_t step = (int64_t)gridDim.x * rows * FWD_ROWS;
    for (int64_t i0 = (int64_t)blockIdx.x * rows * FWD_ROWS + (threadIdx.x >> shift); i0 < n; i0 += step) {
        int64_t c[FWD_ROWS];
#pragma unroll
        for (int u = 0; u < FWD_ROWS; ++u) {
            const int64_t i = i0 + u * rows;
            c[u] = i < n ? tok.at(i) : -1;
        }
        for (int col = t * V; col < w; col += tpr * V) {
            Vec<T, V> x[FWD_ROWS];
#pragma unroll
            for (int u = 0; u < FWD_ROWS; ++u)
                x[u] = load_vec<T, V, TAIL>(W + (c[u] >= 0 && c[u] < C ? c[u] : 0) * ldw, col, w);
#pragma unroll
            for (int u = 0; u < FWD_ROWS; ++u) {
                const int64_t i = i0 + u * rows;
                if (i >= n) continue;
                float y[V];
#pragma unroll
                for (int v = 0; v < V; ++v) y[v] = c[u] >= 0 && c[u] < C ? to_f32(x[u].v[v]) * scale : __builtin_nanf("");
                store_vec<T, V, TAIL>(out + i * ldo, col, w, y);
            }
        }
    }
}

// ---- stable radix sort of n keys in [0, C] (C: tokens that add to no row, sorted behind the others), RADIX_BITS at a time
constexpr int RADIX_BITS = 9, RADIX_BINS = 1 << RADIX_BITS;         // at most; the digits of a sort are as even as can be
constexpr int SORT_STEP = 1024;                       // a workgroup's keys in steps of 4 waves x 4 rounds x 64 lanes
// keys of a workgroup: one step where that makes up to 256 workgroups, which all read each other's counts (512 KB at most).  A
// digit takes 12 to 14 us up to 131,001 keys, 22 us of 524,001 (26 us in 128 workgroups) and 32 us of 1,048,001 (46 us).
static inline int64_t sort_keys(int64_t n) {
    int64_t keys = SORT_STEP;
    while (keys * 256 < n) keys *= 2;
    return keys;
}
__device__ __forceinline__ uint32_t token_key(const IndexArray& tok, int64_t i, int64_t C, int64_t padding) {
    const int64_t c = tok.at(i);
    return c >= 0 && c < C && c != padding ? (uint32_t)c : (uint32_t)C;
}

// The place of a lane's key with digit d: the wave's next free place of the digit and the number of lower lanes with the same
// one (found by a ballot per digit bit), so that equal digits keep their order.  Moves the digit's next free place on.
template <int BITS>
__device__ __forceinline__ uint32_t take_place(uint32_t* next, uint32_t d, bool in, int lane) {
    uint64_t same = __ballot(in);
#pragma unroll
    for (int bit = 0; bit < BITS; ++bit) {
        const uint64_t set = __ballot((d >> bit) & 1u);
        same &= (d >> bit) & 1u ? set : ~set;
    }
    const int rank = __popcll(same & ((1ull << lane) - 1ull));
    uint32_t at = 0;
    if (in) at = next[d] + rank;
    wave_fence();                                       // every lane has read its place before a leader moves it on
    if (in && rank == 0) next[d] = at + (uint32_t)__popcll(same);
    wave_fence();
    return at;
}

// counts[workgroup][digit]
__global__ void __launch_bounds__(256)
k_radix_count(int64_t n, int64_t C, int64_t padding, IndexArray tok, const uint32_t* __restrict__ keys, int64_t each, int shift, int bits,
              uint32_t* __restrict__ counts) {
    __shared__ uint32_t hist[RADIX_BINS];
    const int bins = 1 << bits;
    for (int b = threadIdx.x; b < bins; b += 256) hist[b] = 0;
    __syncthreads();
    const int64_t base = (int64_t)blockIdx.x * each;
#pragma unroll 8
    for (int64_t r = 0; r < each; r += 256) {
        const int64_t i = base + r + threadIdx.x;
        if (i < n) {
            const uint32_t key = keys ? keys[i] : token_key(tok, i, C, padding);
            atomicAdd(&hist[(key >> shift) & (bins - 1)], 1u);
        }
    }
    __syncthreads();
    for (int b = threadIdx.x; b < bins; b += 256) counts[(int64_t)blockIdx.x * bins + b] = hist[b];
}

// Each wave owns a quarter of the workgroup's `each` keys, consecutive ones, and keeps the next free place of every digit.
// Where a digit's keys begin, every workgroup sums from all workgroups' counts; a scan by one workgroup between the two
// launches took 5 to 30 us of its own and saved 1 to 3.
template <int BITS>
__global__ void __launch_bounds__(256)
k_radix_scatter(int64_t n, int64_t C, int64_t padding, IndexArray tok, const uint32_t* __restrict__ keys,
                const uint32_t* __restrict__ pos, int64_t each, int shift, const uint32_t* __restrict__ counts, uint32_t* __restrict__ keys_out,
                uint32_t* __restrict__ pos_out) {
    __shared__ uint32_t next[4][RADIX_BINS];
    __shared__ uint32_t tot[4];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    constexpr int bins = 1 << BITS, OWN = bins > 256 ? bins / 256 : 1;       // digits of a thread, consecutive ones
    for (int b = threadIdx.x; b < 4 * RADIX_BINS; b += 256) (&next[0][0])[b] = 0;
    __syncthreads();
    constexpr int ROUNDS = SORT_STEP / 256;
    const int64_t base = (int64_t)blockIdx.x * each + wv * (each / 4);
    uint32_t key[ROUNDS];
    auto fetch = [&](int64_t from) {
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r) {
            const int64_t i = from + r * 64 + lane;
            key[r] = i >= n ? 0 : keys ? keys[i] : token_key(tok, i, C, padding);
        }
    };
    for (int64_t off = 0; off < each / 4; off += ROUNDS * 64) {
        fetch(base + off);
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r)
            if (base + off + r * 64 + lane < n) atomicAdd(&next[wv][(key[r] >> shift) & (bins - 1)], 1u);
    }
    uint32_t at[OWN] = {}, all[OWN] = {}, sum = 0;       // keys of the digit in the workgroups before this one, and in all
    const bool owner = (int)threadIdx.x * OWN < bins;
    if (owner)
#pragma unroll 16
        for (unsigned k = 0; k < gridDim.x; ++k)
#pragma unroll
            for (int j = 0; j < OWN; ++j) {
                const uint32_t c = counts[k * bins + threadIdx.x * OWN + j];
                all[j] += c;
                at[j] += k < blockIdx.x ? c : 0;
            }
#pragma unroll
    for (int j = 0; j < OWN; ++j) sum += all[j];
    uint32_t s = sum;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const uint32_t x = __shfl_up(s, off);
        if (lane >= off) s += x;
    }
    if (lane == 63) tot[wv] = s;
    __syncthreads();
    s -= sum;
    for (int k = 0; k < wv; ++k) s += tot[k];
#pragma unroll
    for (int j = 0; j < OWN; ++j) {
        at[j] += s;
        s += all[j];
    }
    if (owner)
#pragma unroll
        for (int j = 0; j < OWN; ++j)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t c = next[k][threadIdx.x * OWN + j];
                next[k][threadIdx.x * OWN + j] = at[j];
                at[j] += c;
            }
    __syncthreads();
    for (int64_t off = 0; off < each / 4; off += ROUNDS * 64) {
        if (each > SORT_STEP) fetch(base + off);         // a single step still has its keys
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r) {
            const int64_t i = base + off + r * 64 + lane;
            const bool in = i < n;
            const uint32_t place = take_place<BITS>(next[wv], (key[r] >> shift) & (bins - 1), in, lane);
            if (in) {
                keys_out[place] = key[r];
                pos_out[place] = pos ? pos[i] : (uint32_t)i;
            }
        }
    }
}

// The same sort of up to SMALL_KEYS keys by one workgroup, all digits in one launch (2048 tokens 10 us, latency; the whole
// gradient of 8192 tokens, 1000 x 256 bf16, takes 25 us and of 8193, sorted by several, 30).  Each
// wave holds `rounds` x 64 keys that are consecutive in the current order in registers; the keys change places through LDS.
constexpr int SMALL_WAVES = 16, SMALL_ROUNDS = 8, SMALL_KEYS = SMALL_WAVES * SMALL_ROUNDS * 64, SMALL_BITS = 8;
template <int BITS>
__global__ void __launch_bounds__(SMALL_WAVES * 64)
k_token_sort_small(int n, int64_t C, int64_t padding, IndexArray tok, int passes, uint32_t* __restrict__ keys_out,
                   uint32_t* __restrict__ pos_out) {
    static_assert(BITS <= SMALL_BITS, "a thread a digit in the first four waves, and the counts' place in LDS");
    constexpr int bins = 1 << BITS;
    __shared__ uint32_t next[SMALL_WAVES][bins];
    __shared__ uint32_t buf[SMALL_KEYS];
    __shared__ uint32_t tot[4];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const int rounds = (n + SMALL_WAVES * 64 - 1) / (SMALL_WAVES * 64);
    uint32_t key[SMALL_ROUNDS], pos[SMALL_ROUNDS];
#pragma unroll
    for (int r = 0; r < SMALL_ROUNDS; ++r) {
        const int i = (wv * rounds + r) * 64 + lane;
        pos[r] = (uint32_t)i;
        key[r] = r < rounds && i < n ? token_key(tok, i, C, padding) : 0;
    }
    for (int p = 0; p < passes; ++p) {
        const int shift = p * BITS;
        for (int b = threadIdx.x; b < SMALL_WAVES * bins; b += SMALL_WAVES * 64) (&next[0][0])[b] = 0;
        __syncthreads();
#pragma unroll
        for (int r = 0; r < SMALL_ROUNDS; ++r)
            if (r < rounds && (wv * rounds + r) * 64 + lane < n) atomicAdd(&next[wv][(key[r] >> shift) & (bins - 1)], 1u);
        __syncthreads();
        // thread b owns digit b: the digits' starts by a scan, then the start of each wave's share
        uint32_t sum = 0, s = 0;
        if (threadIdx.x < 256) {
            if (threadIdx.x < bins)
#pragma unroll
                for (int k = 0; k < SMALL_WAVES; ++k) sum += next[k][threadIdx.x];
            s = sum;
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) {
                const uint32_t t = __shfl_up(s, off);
                if (lane >= off) s += t;
            }
            if (lane == 63) tot[wv] = s;
        }
        __syncthreads();
        if (threadIdx.x < bins) {
            uint32_t at = s - sum;
            for (int k = 0; k < wv; ++k) at += tot[k];
#pragma unroll
            for (int k = 0; k < SMALL_WAVES; ++k) {
                const uint32_t c = next[k][threadIdx.x];
                next[k][threadIdx.x] = at;
                at += c;
            }
        }
        __syncthreads();
        uint32_t place[SMALL_ROUNDS];
#pragma unroll
        for (int r = 0; r < SMALL_ROUNDS; ++r)
            if (r < rounds) place[r] = take_place<BITS>(next[wv], (key[r] >> shift) & (bins - 1), (wv * rounds + r) * 64 + lane < n, lane);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            uint32_t(&x)[SMALL_ROUNDS] = half ? pos : key;
#pragma unroll
            for (int r = 0; r < SMALL_ROUNDS; ++r)
                if (r < rounds && (wv * rounds + r) * 64 + lane < n) buf[place[r]] = x[r];
            __syncthreads();
#pragma unroll
            for (int r = 0; r < SMALL_ROUNDS; ++r) {
                const int i = (wv * rounds + r) * 64 + lane;
                if (r < rounds && i < n) x[r] = buf[i];
            }
            __syncthreads();
        }
    }
#pragma unroll
    for (int r = 0; r < SMALL_ROUNDS; ++r) {
        const int i = (wv * rounds + r) * 64 + lane;
        if (r < rounds && i < n) {
            keys_out[i] = key[r];
            pos_out[i] = pos[r];
        }
    }
}

// rowptr[c] = number of sorted keys below c, c = 0..C: a binary search each (50,021 rows of 130,941 keys 6 us, latency)
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

// ---- sums of gradient rows.  A wave covers 64 x V columns, or a narrow row with `lanes` lanes (a power of two) and
// per = 64 / lanes rows side by side, joined at the end.  The lanes fetch 64 positions at once; the rows of up to 8 rounds
// are then in flight together (walked one by one, each row waits for its position and then for itself).
template <class T, int V, bool TAIL>
struct RowSum {
    float acc[V];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int v = 0; v < V; ++v) acc[v] = 0.0f;
    }
    // R rounds from round r; an entry behind the last one loads from the last one's row and sees zeros
    template <int R>
    __device__ __forceinline__ void rounds(int r, int count, int sub, int per, uint32_t p, const T* __restrict__ G, int64_t ldg, int w, int col) {
        Vec<T, V> x[R];
#pragma unroll
        for (int u = 0; u < R; ++u) {
            const int e = (r + u) * per + sub;
            x[u] = load_vec<T, V, TAIL>(G + (int64_t)__shfl(p, e & 63) * ldg, e < count ? col : w, w);
        }
#pragma unroll
        for (int u = 0; u < R; ++u)
#pragma unroll
            for (int v = 0; v < V; ++v) acc[v] = acc[v] + to_f32(x[u].v[v]);
    }
    // rows at the sorted positions [a, b)
    __device__ __forceinline__ void add(const uint32_t* __restrict__ pos, uint32_t a, uint32_t b, const T* __restrict__ G, int64_t ldg, int w,
                                        int col0, int lanes) {
        const int lane = threadIdx.x & 63, sub = lane / lanes, per = 64 / lanes;
        const int col = col0 + (lane & (lanes - 1)) * V;
        for (uint32_t i = a; i < b; i += 64) {
            const int count = b - i < 64 ? (int)(b - i) : 64, all = (count + per - 1) / per;
            const uint32_t p = pos[i + (lane < count ? lane : count - 1)];
            for (int r = 0; r < all; r += 8) {
                if (all - r > 4) rounds<8>(r, count, sub, per, p, G, ldg, w, col);
                else if (all - r > 1) rounds<4>(r, count, sub, per, p, G, ldg, w, col);
                else rounds<1>(r, count, sub, per, p, G, ldg, w, col);
            }
        }
    }
    __device__ __forceinline__ void join(int lanes) {
        for (int off = 32; off >= lanes; off >>= 1)
#pragma unroll
            for (int v = 0; v < V; ++v) acc[v] = acc[v] + __shfl_xor(acc[v], off);
    }
};

// A row of more than `cut` tokens is summed in pieces, one for each chunk of `cut` sorted positions that it meets:
// part[2k] of the row that chunk k begins with, part[2k+1] of the row that it ends with and did not begin with.  Such a row
// meets at least two chunks, so a chunk holds pieces of at most two of them.
template <class T, int V, bool TAIL>
__device__ __forceinline__ void token_piece(int64_t n, int64_t C, int w, int lanes, uint32_t cut, uint32_t chunk, int col0, const uint32_t* __restrict__ keys,
                                            const uint32_t* __restrict__ rowptr, const uint32_t* __restrict__ pos, const T* __restrict__ G,
                                            int64_t ldg, float* __restrict__ part, int64_t ldp) {
    const int lane = threadIdx.x & 63;
    const uint32_t a = chunk * cut, b = (int64_t)a + cut < n ? a + cut : (uint32_t)n;
    const uint32_t first = keys[a], last = keys[b - 1];
#pragma unroll 1
    for (int end = 0; end < 2; ++end) {
        const uint32_t c = end ? last : first;
        if (c >= C || (end && last == first)) continue;
        const uint32_t r0 = rowptr[c], r1 = rowptr[c + 1];
        if (r1 - r0 <= cut) continue;
        RowSum<T, V, TAIL> sum;
        sum.clear();
        sum.add(pos, r0 > a ? r0 : a, r1 < b ? r1 : b, G, ldg, w, col0, lanes);
        sum.join(lanes);
        float* to = part + (2 * (int64_t)chunk + end) * ldp;
        const int col = col0 + lane * V;
        if (lane < lanes)
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (col + v < w) to[col + v] = sum.acc[v];
    }
}

// The row that begins in chunk blockIdx.x and goes on behind it, if it is one of more than `cut` tokens.  `wide` threads (a
// power of two) take four columns each, 1024 / wide lanes of them every so-manieth piece; the lanes are added as a tree.  The
// hottest row's 115 pieces (130,941 tokens of 50,021) bound the launch: 16 us, not less with more columns or loads a launch.
template <class T>
__global__ void __launch_bounds__(1024)
k_token_join(int64_t n, int64_t C, int w, int64_t ldp, int wide, uint32_t cut, const uint32_t* __restrict__ keys,
             const uint32_t* __restrict__ rowptr, const float* __restrict__ part, float scale, T* __restrict__ dW, int64_t ldw) {
    __shared__ float4 red[1024];
    const uint32_t a = blockIdx.x * cut, b = (int64_t)a + cut < n ? a + cut : (uint32_t)n;
    const uint32_t c = keys[b - 1];
    if (c >= C) return;
    const uint32_t r0 = rowptr[c], r1 = rowptr[c + 1];
    if (r1 - r0 <= cut || r0 < a) return;
    const uint32_t k1 = (r1 - 1) / cut;
    const int lanes = 1024 / wide, lane = threadIdx.x / wide, t = threadIdx.x & (wide - 1);
    for (int col0 = 0; col0 < w; col0 += 4 * wide) {
        const int col = col0 + 4 * t;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        if (col < w)
#pragma unroll 4
            for (uint32_t q = blockIdx.x + lane; q <= k1; q += lanes) {
                const int64_t at = (2 * (int64_t)q + (q == blockIdx.x && r0 != a ? 1 : 0)) * ldp + col;
                const float4 x = *reinterpret_cast<const float4*>(part + at);
                acc.x += x.x; acc.y += x.y; acc.z += x.z; acc.w += x.w;
            }
        __syncthreads();
        red[threadIdx.x] = acc;
        for (int half = lanes / 2; half >= 1; half /= 2) {
            __syncthreads();
            if (lane < half) {
                const float4 x = red[threadIdx.x + half * wide];
                acc.x += x.x; acc.y += x.y; acc.z += x.z; acc.w += x.w;
                red[threadIdx.x] = acc;
            }
        }
        if (lane == 0) {
            const float y[4] = {acc.x, acc.y, acc.z, acc.w};
#pragma unroll
            for (int v = 0; v < 4; ++v)
                if (col + v < w) dW[c * ldw + col + v] = from_f32<T>(y[v] * scale);
        }
    }
}

// One wave per chunk of a long row (the first `pieces` workgroups) or per other row of dW, and 64 V columns.  One launch for
// both: the pieces are few waves with much to wait for, the rows many with little (99 us together, 46 + 63 us one behind the other).
template <class T, int V, bool TAIL>
__global__ void __launch_bounds__(256)
k_token_grad(int64_t n, int64_t C, int w, int lanes, uint32_t cut, unsigned pieces, const uint32_t* __restrict__ keys,
             const uint32_t* __restrict__ rowptr, const uint32_t* __restrict__ pos, const T* __restrict__ G, int64_t ldg,
             float* __restrict__ part, int64_t ldp, float scale, T* __restrict__ dW, int64_t ldw) {
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    if (blockIdx.x < pieces) {
        const uint32_t chunk = blockIdx.x * 4 + wv;
        if ((int64_t)chunk * cut < n)
            for (int col0 = blockIdx.y * 64 * V; col0 < w; col0 += gridDim.y * 64 * V)
                token_piece<T, V, TAIL>(n, C, w, lanes, cut, chunk, col0, keys, rowptr, pos, G, ldg, part, ldp);
        return;
    }
    for (int64_t c = (int64_t)(blockIdx.x - pieces) * 4 + wv; c < C; c += (int64_t)(gridDim.x - pieces) * 4) {
        const uint32_t a = rowptr[c], b = rowptr[c + 1];
        if (b - a > cut) continue;
        for (int col0 = blockIdx.y * 64 * V; col0 < w; col0 += gridDim.y * 64 * V) {
            RowSum<T, V, TAIL> sum;
            sum.clear();
            if (a < b) {
                sum.add(pos, a, b, G, ldg, w, col0, lanes);
                sum.join(lanes);
            }
            if (lane < lanes) {
                float y[V];
#pragma unroll
                for (int v = 0; v < V; ++v) y[v] = sum.acc[v] * scale;
                store_vec<T, V, TAIL>(dW + c * ldw, col0 + lane * V, w, y);
            }
        }
    }
}

// ---- up to DIRECT tokens: no sort.  The wave of a row holds all tokens, one a lane, and lists the positions of its own in
// ascending order.  One launch where sort, borders and sums take three (82 x 559 bf16, forward and gradient: 44 us of 64 tokens,
// 54 us of 65).
constexpr int DIRECT = 64;
template <class T, int V, bool TAIL>
__global__ void __launch_bounds__(256)
k_token_direct(int n, int64_t C, int w, int lanes, int64_t padding, IndexArray tok, const T* __restrict__ G, int64_t ldg, float scale,
               T* __restrict__ dW, int64_t ldw) {
    __shared__ uint32_t list[4][DIRECT];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const uint32_t key = token_key(tok, lane < n ? lane : n - 1, C, padding);
    for (int64_t c = (int64_t)blockIdx.x * 4 + wv; c < C; c += (int64_t)gridDim.x * 4) {
        const bool mine = lane < n && key == (uint32_t)c;
        const uint64_t all = __ballot(mine);
        wave_fence();                                    // the row before has read its list
        if (mine) list[wv][__popcll(all & ((1ull << lane) - 1ull))] = lane;
        wave_fence();
        for (int col0 = blockIdx.y * 64 * V; col0 < w; col0 += gridDim.y * 64 * V) {
            RowSum<T, V, TAIL> sum;
            sum.clear();
            if (all) {
                sum.add(list[wv], 0, (uint32_t)__popcll(all), G, ldg, w, col0, lanes);
                sum.join(lanes);
            }
            if (lane < lanes) {
                float y[V];
#pragma unroll
                for (int v = 0; v < V; ++v) y[v] = sum.acc[v] * scale;
                store_vec<T, V, TAIL>(dW + c * ldw, col0 + lane * V, w, y);
            }
        }
    }
}

// ---- tables of at most FEW rows (class labels): no sort.  A wave walks `per_wave` tokens and keeps a sum of every row for its
// 64 columns in LDS; its token is the same in all lanes, so each lane adds to its own word.  The four waves' sums are added
// in order and go to part[workgroup][row][column], which k_token_few_join adds in order.  Its time grows with the rows, which
// every wave adds up at its end; us against the sorted form's at 10, 32 and 48 rows:
//   13,752 x 64 float32     10 : 24    19 : 24    26 : 24         1,000 x 64 float32      9 : 16    18 : 13    25 : 13
//   130,000 x 512 float32   71 : 85    65 : 81    80 : 80         130,000 x 512 bf16     62 : 57    58 : 52    75 : 51
//   1,000,000 x 64 float32  76 : 97    64 : 98    81 : 99         1,000,000 x 64 bf16    63 : 66    59 : 67    75 : 68
constexpr int FEW = 32;
template <class T>
__global__ void __launch_bounds__(256)
k_token_few(int64_t n, int C, int w, int64_t padding, IndexArray tok, int64_t per_wave, const T* __restrict__ G, int64_t ldg,
            float* __restrict__ part) {
    __shared__ float sums[4][FEW][64];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, col = blockIdx.y * 64 + lane, at = col < w ? col : w - 1;
    for (int c = 0; c < C; ++c) sums[wv][c][lane] = 0.0f;
    const int64_t i0 = ((int64_t)blockIdx.x * 4 + wv) * per_wave, i1 = i0 + per_wave < n ? i0 + per_wave : n;
    for (int64_t i = i0; i < i1; i += 64) {
        const int count = i1 - i < 64 ? (int)(i1 - i) : 64;
        const uint32_t key = token_key(tok, i + (lane < count ? lane : count - 1), C, padding);
        for (int u0 = 0; u0 < count; u0 += 8) {
            float g[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) g[u] = to_f32(G[(i + (u0 + u < count ? u0 + u : count - 1)) * ldg + at]);
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const uint32_t c = __builtin_amdgcn_readlane(key, (u0 + u) & 63);
                if (u0 + u < count && c < (uint32_t)C) sums[wv][c][lane] = sums[wv][c][lane] + g[u];
            }
        }
    }
    __syncthreads();
    if (col < w)
        for (int c = wv; c < C; c += 4)
            part[((int64_t)blockIdx.x * C + c) * w + col] = ((sums[0][c][lane] + sums[1][c][lane]) + sums[2][c][lane]) + sums[3][c][lane];
}
// dW from the workgroups' sums: 16 lanes of workgroups each add every 16th, then the lanes are added in order
template <class T>
__global__ void __launch_bounds__(1024)
k_token_few_join(int64_t nblk, int C, int w, const float* __restrict__ part, float scale, T* __restrict__ dW, int64_t ldw) {
    __shared__ float red[16][64];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const int64_t size = (int64_t)C * w;
    for (int64_t g0 = (int64_t)blockIdx.x * 64; g0 < size; g0 += (int64_t)gridDim.x * 64) {
        const int64_t g = g0 + lane;
        float acc = 0.0f;
        if (g < size)
#pragma unroll 8
            for (int64_t b = wv; b < nblk; b += 16) acc = acc + part[b * size + g];
        __syncthreads();
        red[wv][lane] = acc;
        __syncthreads();
        if (wv == 0 && g < size) {
#pragma unroll
            for (int k = 1; k < 16; ++k) acc = acc + red[k][lane];
            dW[g / w * ldw + g % w] = from_f32<T>(acc * scale);
        }
    }
}
// tokens a wave walks: 16 C a workgroup at least, which keeps its sums an eighth of what it reads, and at most 4096 workgroups
static inline int64_t few_per_wave(int64_t n, int64_t C) {
    int64_t per = 4 * C < 32 ? 32 : 4 * C;
    while (per * 4 * 4096 < n) per *= 2;
    return per;
}
static inline bool few_rows(int64_t C, int64_t w) { return C <= FEW && (w + 63) / 64 < 65536; }

// fn(BITS) for the digit width of a sort, 5 to 9
template <class Fn> static inline int with_digit(int bits, Fn&& fn) {
    switch (bits) {
        case 5: return fn(std::integral_constant<int, 5>{});
        case 6: return fn(std::integral_constant<int, 6>{});
        case 7: return fn(std::integral_constant<int, 7>{});
        case 8: return fn(std::integral_constant<int, 8>{});
        default: return fn(std::integral_constant<int, 9>{});
    }
}

static inline bool direct_rows(int64_t n) { return n > 0 && n <= DIRECT; }

struct TokenLayout {
    int64_t nblk, keys[2], pos[2], counts, rowptr, part, bytes;
    uint32_t cut;
    int passes, digit;
};
static inline TokenLayout token_layout(int64_t n, int64_t C, int64_t w) {
    TokenLayout l{};
    if (direct_rows(n)) {
        l.bytes = 256;                                   // none is used; never 0, so that every call has a workspace
        return l;
    }
    if (few_rows(C, w)) {
        const int64_t per = 4 * few_per_wave(n, C);
        l.nblk = (n + per - 1) / per;
        l.bytes = (l.nblk * C * w * 4 + 256) / 256 * 256;
        return l;
    }
    int bits = 1;
    while ((C >> bits) != 0) ++bits;                   // keys are 0..C
    const int most = n > SMALL_KEYS ? RADIX_BITS : SMALL_BITS;
    l.passes = (bits + most - 1) / most;
    l.digit = (bits + l.passes - 1) / l.passes;
    if (l.digit < 5) l.digit = 5;                      // with_digit
    l.nblk = (n + sort_keys(n) - 1) / sort_keys(n);
    // Tokens from which a row is summed in pieces.  32, 64, 128 and 256 take 157, 143, 135 and 142 us of 130,941 tokens of 50,021 x
    // 1024 bf16 (few rows with thousands each), and 89, 95, 111 and 142 us of 16,000 such of float32: longer pieces are fewer to
    // join, and each is one wave that the others wait for.
    l.cut = 64;
    while ((int64_t)l.cut * 4096 < n) l.cut *= 2;      // at most 4096 pieces of one row
    int64_t at = 0;
    auto take = [&at](int64_t words) { const int64_t p = at; at += (words * 4 + 255) / 256 * 256; return p; };
    for (int k = 0; k < 2; ++k) { l.keys[k] = take(n); l.pos[k] = take(n); }
    l.counts = take(n > SMALL_KEYS ? l.nblk << l.digit : 0);
    l.rowptr = take(C + 1);
    l.part = take(n > l.cut ? 2 * ((n + l.cut - 1) / l.cut) * ((w + 3) / 4 * 4) : 0);
    l.bytes = at;
    return l;
}

}  // namespace gm

using namespace gm;

#define GM_TOKEN_CHECK(ptr_)                                                                                              \
    GM_REQUIRE(n >= 0 && C > 0 && w > 0 && (n == 0 || (tokens && ptr_)), "bad arguments");                                \
    GM_REQUIRE(dtype_ok(dtype), "dtype %d is none of GM_DTYPE_*", dtype);                                                 \
    GM_REQUIRE(C < (1ll << 31) && n < (1ll << 31) && w < (1ll << 30), "n or C of 2^31 or more, or w of 2^30 or more")

extern "C" int gm_token_embedding_fwd(int64_t n, int64_t C, int64_t w, const void* tokens, int tokens_i64, const void* weight,
                                      int64_t ldw, int dtype, float scale, void* out, int64_t ldo, gm_stream_t stream) {
    GM_TOKEN_CHECK(out);
    GM_REQUIRE(weight && ldw >= w && ldo >= w, "weight missing or leading dimension too small");
    if (n == 0) return GM_OK;
    const int vec = w < 16 / dtype_size(dtype) ? 1 : 16 / dtype_size(dtype);        // with_row_form
    int shift = 0;
    while (shift < 8 && ((int64_t)vec << shift) < w) ++shift;
    const int64_t rows = (int64_t)(256 >> shift) * FWD_ROWS;
    return with_dtype(dtype, [&](auto t) -> int {
        using T = decltype(t);
        with_row_form<T>(w, [&](auto v, auto tail) {
            hipLaunchKernelGGL((k_token_embedding_fwd<T, decltype(v)::value, decltype(tail)::value>), dim3(grid_for((n + rows - 1) / rows, 256)),
                               dim3(256), 0, as_stream(stream), n, C, (int)w, shift, IndexArray{tokens, tokens_i64},
                               static_cast<const T*>(weight), ldw, scale, static_cast<T*>(out), ldo);
        });
        GM_LAUNCH_CHECK();
        return GM_OK;
    });
}

extern "C" int64_t gm_token_embedding_bwd_workspace_bytes(int64_t n, int64_t C, int64_t w) {
    if (n < 0 || C <= 0 || w <= 0 || n >= (1ll << 31) || C >= (1ll << 31) || w >= (1ll << 30)) return -1;
    return token_layout(n, C, w).bytes;
}

extern "C" int gm_token_embedding_bwd(int64_t n, int64_t C, int64_t w, const void* tokens, int tokens_i64, int64_t padding_idx,
                                      const void* G, int64_t ldg, int dtype, float scale, void* dW, int64_t ldw,
                                      void* workspace, int64_t workspace_bytes, gm_stream_t stream) {
    GM_TOKEN_CHECK(G);
    GM_REQUIRE(dW && ldg >= w && ldw >= w, "dW missing or leading dimension too small");
    GM_REQUIRE(padding_idx < C, "padding_idx %lld is not below C = %lld", (long long)padding_idx, (long long)C);
    const TokenLayout l = token_layout(n, C, w);
    GM_REQUIRE(workspace && workspace_bytes >= l.bytes && aligned(workspace, 16),
               "gm_token_embedding_bwd needs %lld workspace bytes (gm_token_embedding_bwd_workspace_bytes)", (long long)l.bytes);
    hipStream_t s = as_stream(stream);
    char* ws = static_cast<char*>(workspace);
    const int vec = w < 16 / dtype_size(dtype) ? 1 : 16 / dtype_size(dtype);        // with_row_form
    const int64_t vecs = (w + vec - 1) / vec;
    int lanes = 64;
    while (lanes > 1 && lanes / 2 >= vecs) lanes /= 2;
    // a wave walks the tiles of its row where the rows alone fill the chip eight times over
    int64_t tiles = (vecs + 63) / 64;
    if (tiles > 1 && C >= 65536 / tiles) tiles = C >= 65536 ? 1 : (65536 + C - 1) / C;
    if (tiles > 65535) tiles = 65535;                   // a launch's second dimension; its workgroups walk on
    const unsigned rows = grid_for((C + 3) / 4, 512);
    if (direct_rows(n))
        return with_dtype(dtype, [&](auto t) -> int {
            using T = decltype(t);
            with_row_form<T>(w, [&](auto v, auto tail) {
                hipLaunchKernelGGL((k_token_direct<T, decltype(v)::value, decltype(tail)::value>), dim3(rows, (unsigned)tiles), dim3(256), 0, s,
                                   (int)n, C, (int)w, lanes, padding_idx, IndexArray{tokens, tokens_i64}, static_cast<const T*>(G), ldg, scale,
                                   static_cast<T*>(dW), ldw);
            });
            GM_LAUNCH_CHECK();
            return GM_OK;
        });
    if (few_rows(C, w)) {
        float* few = static_cast<float*>(workspace);
        return with_dtype(dtype, [&](auto t) -> int {
            using T = decltype(t);
            if (l.nblk > 0) {
                hipLaunchKernelGGL((k_token_few<T>), dim3((unsigned)l.nblk, (unsigned)((w + 63) / 64)), dim3(256), 0, s, n, (int)C, (int)w,
                                   padding_idx, IndexArray{tokens, tokens_i64}, few_per_wave(n, C), static_cast<const T*>(G), ldg, few);
                GM_LAUNCH_CHECK();
            }
            hipLaunchKernelGGL((k_token_few_join<T>), dim3(grid_for((C * w + 63) / 64, 1024)), dim3(1024), 0, s, l.nblk, (int)C, (int)w, few,
                               scale, static_cast<T*>(dW), ldw);
            GM_LAUNCH_CHECK();
            return GM_OK;
        });
    }
    auto u32 = [ws](int64_t at) { return reinterpret_cast<uint32_t*>(ws + at); };
    const IndexArray tok{tokens, tokens_i64};
    uint32_t *counts = u32(l.counts), *rowptr = u32(l.rowptr);
    const uint32_t *keys = u32(l.keys[0]), *pos = u32(l.pos[0]);
    float* part = reinterpret_cast<float*>(ws + l.part);
    const int rc = with_digit(l.digit, [&](auto digit) -> int {
        constexpr int BITS = decltype(digit)::value;
        if constexpr (BITS <= SMALL_BITS) {
            if (n > 0 && n <= SMALL_KEYS) {
                hipLaunchKernelGGL((k_token_sort_small<BITS>), dim3(1), dim3(SMALL_WAVES * 64), 0, s, (int)n, C, padding_idx, tok, l.passes,
                                   u32(l.keys[0]), u32(l.pos[0]));
                GM_LAUNCH_CHECK();
            }
        }
        for (int p = 0; p < l.passes && n > SMALL_KEYS; ++p) {
            uint32_t *ko = u32(l.keys[p & 1]), *po = u32(l.pos[p & 1]);
            hipLaunchKernelGGL(k_radix_count, dim3((unsigned)l.nblk), dim3(256), 0, s, n, C, padding_idx, tok, p ? keys : nullptr, sort_keys(n),
                               p * BITS, BITS, counts);
            GM_LAUNCH_CHECK();
            hipLaunchKernelGGL((k_radix_scatter<BITS>), dim3((unsigned)l.nblk), dim3(256), 0, s, n, C, padding_idx, tok, p ? keys : nullptr,
                               p ? pos : nullptr, sort_keys(n), p * BITS, counts, ko, po);
            GM_LAUNCH_CHECK();
            keys = ko;
            pos = po;
        }
        return GM_OK;
    });
    if (rc != GM_OK) return rc;
    hipLaunchKernelGGL(k_token_rowptr, dim3((unsigned)((C + 1 + 255) / 256)), dim3(256), 0, s, n, C, keys, rowptr);
    GM_LAUNCH_CHECK();
    const unsigned chunks = (unsigned)((n + l.cut - 1) / l.cut);
    const int64_t ldp = (w + 3) / 4 * 4;
    int wide = 1;
    while (wide < 256 && wide * 4 < w) wide *= 2;
    return with_dtype(dtype, [&](auto t) -> int {
        using T = decltype(t);
        int status = GM_OK;
        with_row_form<T>(w, [&](auto v, auto tail) {
            constexpr int V = decltype(v)::value;
            constexpr bool TAIL = decltype(tail)::value;
            status = [&]() -> int {
                const unsigned pieces = n > l.cut ? (chunks + 3) / 4 : 0;
                hipLaunchKernelGGL((k_token_grad<T, V, TAIL>), dim3(pieces + rows, (unsigned)tiles), dim3(256), 0, s, n, C, (int)w,
                                   lanes, l.cut, pieces, keys, rowptr, pos, static_cast<const T*>(G), ldg, part, ldp, scale,
                                   static_cast<T*>(dW), ldw);
                GM_LAUNCH_CHECK();
                if (pieces) {
                    hipLaunchKernelGGL((k_token_join<T>), dim3(chunks), dim3(1024), 0, s, n, C, (int)w, ldp, wide, l.cut, keys, rowptr, part, scale,
                                       static_cast<T*>(dW), ldw);
                    GM_LAUNCH_CHECK();
                }
                return GM_OK;
            }();
        });
        return status;
    });
}
