// Losses that keep a router's experts evenly used, their gradients, and the counts behind them.
//
// Rows t < T of logits l over E experts, K routes a row, S sequences [o_s, o_{s+1}).  A row counts if it lies in a
// sequence and its mask byte (if there is a mask) is set:
//   p = softmax(l), or sigma(l) / sum sigma(l);   n_s = counted rows, c_{s,e} = their routes to expert e
//   f_{s,e} = E c_{s,e} / max(1, sum_j c_{s,j}),   P_{s,e} = 1/n_s sum_t p_{t,e}
//   balance = 1/S' sum_s sum_e f_{s,e} P_{s,e}     (S' = sequences with a counted row)
//   z       = 1/n  sum_t lse(l_t)^2                (n = counted rows)
// and, with a_e = f_{s,e} / n_s of the row's sequence,
//   d balance / dl = p (a - sum p a) / S'  [(1 - sigma) times that for sigmoid scores],   dz / dl = 2/n lse softmax(l).
// A row whose logits are all -inf has p = 0 and adds nothing to z; a row that does not count is not read for the losses.
//
// Forward: balance_rows_kernel gives every block a run of rows; for each sequence that the run meets, the block sums p
// and the routes over its rows and stores them in a slot of their own, block + sequence (along the staircase of
// (block, sequence) pairs that meet, that sum never repeats).  balance_join_kernel adds the slots of a sequence in block
// order.  No floating-point atomics: two runs give the same bytes.
#include <algorithm>

#include "common.cuh"
#include "profile.cuh"

namespace mok {
namespace {

constexpr int kWarps = 8;
constexpr int kRowThreads = kWarps * 32;
constexpr int kMaxRowBlocks = 592;             // not read from the device: the order of the sums is the same on every GPU
constexpr int kJoinThreads = 256;
constexpr int kJoinCols = 32;
constexpr unsigned kAll = 0xffffffffu;

struct SlotHead { float z; int rows, routes, pad; };

// scratch of a forward call, in this order: slot heads, sums of p [slots, E], route counts [slots, E], the join blocks'
// parts of the loss [S * tiles], z and rows of a sequence [S] each, and the counter of finished join blocks
struct Scratch {
    SlotHead* head;
    float* p;
    int* routes;
    float* part;
    float* seq_z;
    int* seq_rows;
    unsigned* ticket;
    size_t bytes;
    Scratch(void* base, int slots, int E, int S) {
        const int tiles = (E + kJoinCols - 1) / kJoinCols;
        char* at = static_cast<char*>(base);
        auto take = [&at](size_t n) { char* p = at; at += n; return p; };
        head = reinterpret_cast<SlotHead*>(take(sizeof(SlotHead) * static_cast<size_t>(slots)));
        p = reinterpret_cast<float*>(take(4 * static_cast<size_t>(slots) * E));
        routes = reinterpret_cast<int*>(take(4 * static_cast<size_t>(slots) * E));
        part = reinterpret_cast<float*>(take(4 * static_cast<size_t>(S) * tiles));
        seq_z = reinterpret_cast<float*>(take(4 * static_cast<size_t>(S)));
        seq_rows = reinterpret_cast<int*>(take(4 * static_cast<size_t>(S)));
        ticket = reinterpret_cast<unsigned*>(take(4));
        bytes = static_cast<size_t>(at - static_cast<char*>(base));
    }
};

int row_blocks(int T) { return std::min(kMaxRowBlocks, (T + kWarps - 1) / kWarps); }

struct BalanceParams {
    const void* logits;
    const long long* top_in;       // finished routes, or null: this launch chooses them
    long long* top_out;
    float* weights;
    const uint8_t* mask;           // null: every row
    const int* offsets;            // [S + 1], null: one sequence of all rows
    const int* load;               // [S, E] counts that stand for the local ones in f, null: the local ones
    float* losses;                 // [2]
    int* counts;                   // [S, E]
    float* coef;                   // [S * E] f / n_s, then 1 / S', 2 / n
    int T, E, K, S;
    int rows_per_block, blocks;
    int sigmoid;
    SlotHead* head;
    float* slot_p;
    int* slot_routes;
    float* part;
    float* seq_z;
    int* seq_rows;
    unsigned* ticket;
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(kAll, v, off);
    return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor_sync(kAll, v, off));
    return v;
}
__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_float(float v, float& out) { out = v; }
__device__ __forceinline__ void from_float(float v, __nv_bfloat16& out) { out = __float2bfloat16_rn(v); }

// Sequence bounds as the kernels use them: inside [0, T] whatever the caller's array holds.
__device__ __forceinline__ int seq_bound(const int* offsets, int s, int T) {
    if (offsets == nullptr) return s ? T : 0;
    return min(max(offsets[s], 0), T);
}
// first sequence that ends behind row `row` (S if none)
__device__ __forceinline__ int first_sequence(const int* offsets, int S, int row, int T) {
    int lo = 0, hi = S;
    while (lo < hi) { const int mid = (lo + hi) >> 1; if (seq_bound(offsets, mid + 1, T) > row) hi = mid; else lo = mid + 1; }
    return lo;
}

// sigma(l) times a factor common to the row, exp(-min(m, 0)) with m the row's maximum: the sum over the row cannot
// underflow, and the factor cancels in every quotient
__device__ __forceinline__ float sigmoid_scaled(float l, float shift) {
    return l >= 0.0f ? 1.0f / (1.0f + expf(-l)) : expf(l - shift) / (1.0f + expf(l));
}
__device__ __forceinline__ float sigmoid_shift(float m) { return m == -INFINITY ? 0.0f : fminf(m, 0.0f); }

// Softmax statistics, probabilities and softmax of one row.  v[j] is the logit of expert lane + 32 j.  q[j] = softmax,
// p[j] = what the balance loss averages (the same for softmax scores); returns lse, 0 for a row without a finite logit.
template <int kPerLane>
__device__ __forceinline__ float row_probs(const float (&v)[kPerLane], int lane, int E, int sigmoid, float (&p)[kPerLane],
                                           float (&q)[kPerLane]) {
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < kPerLane; ++j) m = fmaxf(m, v[j]);
    m = warp_max(m);
    const float base = m == -INFINITY ? 0.0f : m;
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < kPerLane; ++j) { q[j] = expf(v[j] - base); sum += q[j]; }      // lanes past E hold -inf: 0
    sum = warp_sum(sum);
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int j = 0; j < kPerLane; ++j) q[j] *= inv;
    if (sigmoid) {
        const float shift = sigmoid_shift(m);
        float total = 0.0f;
#pragma unroll
        for (int j = 0; j < kPerLane; ++j) { p[j] = sigmoid_scaled(v[j], shift); total += p[j]; }
        total = warp_sum(total);
        const float inv_p = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
        for (int j = 0; j < kPerLane; ++j) p[j] *= inv_p;
    } else {
#pragma unroll
        for (int j = 0; j < kPerLane; ++j) p[j] = q[j];
    }
    return sum == 0.0f ? 0.0f : base + logf(sum);
}

// The K largest logits of a row, descending, the lower expert first among equals; a NaN ranks with -inf.  Lane k keeps
// the k-th (value, expert).
template <int kPerLane>
__device__ __forceinline__ void row_select(const float (&v)[kPerLane], int lane, int E, int K, float& my_val, int& my_idx) {
    unsigned taken = 0;
    my_val = -INFINITY;
    my_idx = 0;
    for (int k = 0; k < K; ++k) {
        float best = -INFINITY;
        int best_e = 0x7fffffff;
#pragma unroll
        for (int j = 0; j < kPerLane; ++j) {
            const int e = lane + 32 * j;
            const float lv = v[j] == v[j] ? v[j] : -INFINITY;
            if (e < E && !((taken >> j) & 1u) && (lv > best || best_e == 0x7fffffff)) { best = lv; best_e = e; }
        }
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) {
            const float ov = __shfl_xor_sync(kAll, best, off);
            const int oe = __shfl_xor_sync(kAll, best_e, off);
            if (oe != 0x7fffffff && (best_e == 0x7fffffff || ov > best || (ov == best && oe < best_e))) { best = ov; best_e = oe; }
        }
        if ((best_e & 31) == lane) taken |= 1u << (best_e >> 5);
        if (lane == k) { my_val = best; my_idx = best_e; }
    }
}

template <typename T, int kPerLane>
__device__ __forceinline__ void load_row(const void* logits, size_t row, int lane, int E, float (&v)[kPerLane]) {
    const T* at = static_cast<const T*>(logits) + row * E;
#pragma unroll
    for (int j = 0; j < kPerLane; ++j) { const int e = lane + 32 * j; v[j] = e < E ? to_float(at[e]) : -INFINITY; }
}

// HBM- or latency-bound: reads T E logits once, writes K routes a row and (p, routes) per slot.
template <typename T, int kPerLane>
__global__ void __launch_bounds__(kRowThreads) balance_rows_kernel(const BalanceParams g) {
    extern __shared__ float smem[];                        // p [kWarps][E], routes [E]
    __shared__ float s_z[kWarps];
    __shared__ int s_rows[kWarps], s_routes;
    int* const hist = reinterpret_cast<int*>(smem + static_cast<size_t>(kWarps) * g.E);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_wait();
    if (blockIdx.x == 0 && threadIdx.x == 0) *g.ticket = 0;
    const bool select = g.top_in == nullptr;
    const long long first = static_cast<long long>(blockIdx.x) * g.rows_per_block;
    int pos = static_cast<int>(min(first, static_cast<long long>(g.T)));
    const int hi = static_cast<int>(min(first + g.rows_per_block, static_cast<long long>(g.T)));
    int s = first_sequence(g.offsets, g.S, pos, g.T);
    while (pos < hi) {
        // the next run of rows: a sequence's, or rows between and behind the sequences
        const int begin = s < g.S ? max(seq_bound(g.offsets, s, g.T), pos) : hi;
        const bool counted = begin <= pos;
        const int end = counted ? min(seq_bound(g.offsets, s + 1, g.T), hi) : min(begin, hi);
        if (counted && end <= pos) { ++s; continue; }
        if (counted) {
            for (int e = threadIdx.x; e < g.E; e += kRowThreads) hist[e] = 0;
            if (threadIdx.x == 0) s_routes = 0;
            __syncthreads();
        }
        float acc[kPerLane], z = 0.0f;
        int rows = 0, routes = 0;
#pragma unroll
        for (int j = 0; j < kPerLane; ++j) acc[j] = 0.0f;
        for (int t = pos + warp; t < end && (counted || select); t += kWarps) {
            float v[kPerLane];
            load_row<T>(g.logits, t, lane, g.E, v);
            const bool live = counted && (g.mask == nullptr || g.mask[t]);
            if (live) {
                float p[kPerLane], q[kPerLane];
                const float lse = row_probs(v, lane, g.E, g.sigmoid, p, q);
#pragma unroll
                for (int j = 0; j < kPerLane; ++j) acc[j] += p[j];
                z += lse * lse;
                ++rows;
            }
            const size_t o = static_cast<size_t>(t) * g.K;
            if (select) {
                float val; int idx;
                row_select(v, lane, g.E, g.K, val, idx);
                const float top = __shfl_sync(kAll, val, 0);
                float w = 0.0f;
                if (lane < g.K && top != -INFINITY) w = g.sigmoid ? sigmoid_scaled(val, sigmoid_shift(top)) : expf(val - top);
                const float sum = warp_sum(w);
                if (lane < g.K) {
                    g.top_out[o + lane] = idx;
                    g.weights[o + lane] = sum == 0.0f ? 0.0f : w / sum;
                    if (live) { atomicAdd(&hist[idx], 1); ++routes; }
                }
            } else if (live) {
                for (int k = lane; k < g.K; k += 32) {
                    const long long e = g.top_in[o + k];
                    if (e >= 0 && e < g.E) { atomicAdd(&hist[e], 1); ++routes; }
                }
            }
        }
        if (counted) {
            float* const mine = smem + static_cast<size_t>(warp) * g.E;
#pragma unroll
            for (int j = 0; j < kPerLane; ++j) { const int e = lane + 32 * j; if (e < g.E) mine[e] = acc[j]; }
            if (routes) atomicAdd(&s_routes, routes);
            if (lane == 0) { s_z[warp] = z; s_rows[warp] = rows; }
            __syncthreads();
            const size_t slot = static_cast<size_t>(blockIdx.x) + s;
            for (int e = threadIdx.x; e < g.E; e += kRowThreads) {
                float sum = 0.0f;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) sum += smem[static_cast<size_t>(w) * g.E + e];
                g.slot_p[slot * g.E + e] = sum;
                g.slot_routes[slot * g.E + e] = hist[e];
            }
            if (threadIdx.x == 0) {
                SlotHead h{0.0f, 0, s_routes, 0};
                for (int w = 0; w < kWarps; ++w) { h.z += s_z[w]; h.rows += s_rows[w]; }
                g.head[slot] = h;
            }
            __syncthreads();
            ++s;
        }
        pos = end;
    }
}

template <typename V>
__device__ __forceinline__ V block_sum(V v, V* tmp) {      // the same order on every run
    tmp[threadIdx.x] = v;
    __syncthreads();
    for (int n = kJoinThreads / 2; n > 0; n >>= 1) {
        if (threadIdx.x < n) tmp[threadIdx.x] += tmp[threadIdx.x + n];
        __syncthreads();
    }
    const V sum = tmp[0];
    __syncthreads();
    return sum;
}

// One block per 32 experts of a sequence: adds the sequence's slots in block order; the block that finishes last adds up
// the losses.
__global__ void __launch_bounds__(kJoinThreads) balance_join_kernel(const BalanceParams g) {
    __shared__ float tmp[kJoinThreads];
    __shared__ int itmp[kJoinThreads];
    __shared__ bool last;
    pdl_wait();
    const int tiles = (g.E + kJoinCols - 1) / kJoinCols;
    const int s = blockIdx.x / tiles, tile = blockIdx.x - s * tiles;
    const int begin = seq_bound(g.offsets, s, g.T), end = seq_bound(g.offsets, s + 1, g.T);
    const int b0 = begin / g.rows_per_block, b1 = end > begin ? (end - 1) / g.rows_per_block + 1 : b0;
    const int tid = threadIdx.x;
    float z = 0.0f;
    int rows = 0, routes = 0;
    for (int b = b0 + tid; b < b1; b += kJoinThreads) {
        const SlotHead h = g.head[b + s];
        z += h.z; rows += h.rows; routes += h.routes;
    }
    rows = block_sum(rows, itmp);
    if (g.load != nullptr) {
        routes = 0;
        for (int e = tid; e < g.E; e += kJoinThreads) routes += g.load[static_cast<size_t>(s) * g.E + e];
    }
    routes = block_sum(routes, itmp);
    z = block_sum(z, tmp);
    const int col = tid % kJoinCols, r = tid / kJoinCols, e = tile * kJoinCols + col;
    float p = 0.0f;
    int c = 0;
    if (e < g.E)
        for (int b = b0 + r; b < b1; b += kJoinThreads / kJoinCols) {
            const size_t at = static_cast<size_t>(b + s) * g.E + e;
            p += g.slot_p[at];
            c += g.slot_routes[at];
        }
    tmp[tid] = p;
    itmp[tid] = c;
    __syncthreads();
    float part = 0.0f;
    if (r == 0 && e < g.E) {
        for (int i = 1; i < kJoinThreads / kJoinCols; ++i) { p += tmp[i * kJoinCols + col]; c += itmp[i * kJoinCols + col]; }
        const size_t at = static_cast<size_t>(s) * g.E + e;
        g.counts[at] = c;
        const int used = g.load != nullptr ? g.load[at] : c;
        const float f = static_cast<float>(g.E) * static_cast<float>(used) / static_cast<float>(max(routes, 1));
        const float a = rows > 0 ? f / static_cast<float>(rows) : 0.0f;
        g.coef[at] = a;
        part = a * p;
    }
    if (r == 0) {
        part = warp_sum(part);
        if (col == 0) {
            g.part[blockIdx.x] = part;
            if (tile == 0) { g.seq_z[s] = z; g.seq_rows[s] = rows; }
        }
    }
    __threadfence();
    __syncthreads();
    if (tid == 0) last = atomicAdd(g.ticket, 1u) == gridDim.x - 1;
    __syncthreads();
    if (!last) return;
    __threadfence();
    float balance = 0.0f;
    z = 0.0f;
    int live = 0;
    rows = 0;
    for (int i = tid; i < static_cast<int>(gridDim.x); i += kJoinThreads) balance += __ldcg(&g.part[i]);
    for (int i = tid; i < g.S; i += kJoinThreads) { const int n = __ldcg(&g.seq_rows[i]); z += __ldcg(&g.seq_z[i]); rows += n; live += n > 0; }
    balance = block_sum(balance, tmp);
    z = block_sum(z, tmp);
    rows = block_sum(rows, itmp);
    live = block_sum(live, itmp);
    if (tid == 0) {
        const float n = static_cast<float>(max(rows, 1)), sequences = static_cast<float>(max(live, 1));
        g.losses[0] = balance / sequences;
        g.losses[1] = z / n;
        g.coef[static_cast<size_t>(g.S) * g.E] = 1.0f / sequences;
        g.coef[static_cast<size_t>(g.S) * g.E + 1] = 2.0f / n;
    }
}

struct BalanceBwdParams {
    const float* d_losses;         // [2]
    const void* logits;
    const float* coef;
    const uint8_t* mask;
    const int* offsets;
    const long long* top;          // with weights and d_weights: add the gradient of the router weights
    const float* weights;
    const float* d_weights;
    void* d_logits;
    int T, E, K, S, sigmoid;
};

// One warp per row; reads and writes T E values.
template <typename T, int kPerLane>
__global__ void __launch_bounds__(kRowThreads) balance_bwd_kernel(const BalanceBwdParams g) {
    const int lane = threadIdx.x & 31;
    pdl_wait();
    const size_t scalars = static_cast<size_t>(g.S) * g.E;
    const float gb = g.d_losses[0] * g.coef[scalars], gz = g.d_losses[1] * g.coef[scalars + 1];
    for (long long t = static_cast<long long>(blockIdx.x) * kWarps + (threadIdx.x >> 5); t < g.T;
         t += static_cast<long long>(gridDim.x) * kWarps) {
        float d[kPerLane];
#pragma unroll
        for (int j = 0; j < kPerLane; ++j) d[j] = 0.0f;
        const int s = first_sequence(g.offsets, g.S, static_cast<int>(t), g.T);
        // without an upstream gradient of the losses the row is not read for them (nothing times NaN stays nothing)
        const bool live = (gb != 0.0f || gz != 0.0f) && s < g.S && seq_bound(g.offsets, s, g.T) <= t && (g.mask == nullptr || g.mask[t]);
        if (live) {
            float v[kPerLane], p[kPerLane], q[kPerLane];
            load_row<T>(g.logits, t, lane, g.E, v);
            const float lse = row_probs(v, lane, g.E, g.sigmoid, p, q);
            const float* a = g.coef + static_cast<size_t>(s) * g.E;
            float av[kPerLane], dot = 0.0f;
#pragma unroll
            for (int j = 0; j < kPerLane; ++j) { const int e = lane + 32 * j; av[j] = e < g.E ? a[e] : 0.0f; dot += p[j] * av[j]; }
            dot = warp_sum(dot);
#pragma unroll
            for (int j = 0; j < kPerLane; ++j) {
                float slope = p[j] * (av[j] - dot);
                if (g.sigmoid) slope /= 1.0f + expf(v[j]);
                d[j] = gb * slope + gz * lse * q[j];
            }
        }
        if (g.top != nullptr) {
            const size_t o = static_cast<size_t>(t) * g.K + lane;
            const float w = lane < g.K ? g.weights[o] : 0.0f, dw = lane < g.K ? g.d_weights[o] : 0.0f;
            const long long top = lane < g.K ? g.top[o] : -1;
            const int idx = top >= 0 && top < g.E ? static_cast<int>(top) : -1;
            const float dot = warp_sum(w * dw);
            float add = w * (dw - dot);
            if (g.sigmoid && idx >= 0) add /= 1.0f + expf(to_float(static_cast<const T*>(g.logits)[static_cast<size_t>(t) * g.E + idx]));
            if (w == 0.0f) add = 0.0f;
            for (int k = 0; k < g.K; ++k) {
                const int e = __shfl_sync(kAll, idx, k);
                const float x = __shfl_sync(kAll, add, k);
#pragma unroll
                for (int j = 0; j < kPerLane; ++j) if (e == lane + 32 * j) d[j] += x;
            }
        }
        T* out = static_cast<T*>(g.d_logits) + static_cast<size_t>(t) * g.E;
#pragma unroll
        for (int j = 0; j < kPerLane; ++j) { const int e = lane + 32 * j; if (e < g.E) from_float(d[j], out[e]); }
    }
}

struct CountParams {
    const void* top;
    int ids_i32;
    const uint8_t* mask;
    const int* offsets;
    int* counts;                   // [S, E], zeroed
    int T, E, K, S, rows_per_block;
};

// Each block counts a run of rows in shared memory, sequence by sequence, and adds what it found: integer sums do not
// depend on their order.  Reads T K ids.
__global__ void __launch_bounds__(kRowThreads) expert_counts_kernel(const CountParams g) {
    extern __shared__ int bins[];
    pdl_wait();
    const long long first = static_cast<long long>(blockIdx.x) * g.rows_per_block;
    int pos = static_cast<int>(min(first, static_cast<long long>(g.T)));
    const int hi = static_cast<int>(min(first + g.rows_per_block, static_cast<long long>(g.T)));
    for (int s = first_sequence(g.offsets, g.S, pos, g.T); s < g.S && pos < hi; ++s) {
        const int begin = max(seq_bound(g.offsets, s, g.T), pos), end = min(seq_bound(g.offsets, s + 1, g.T), hi);
        if (begin >= hi) break;
        if (end <= begin) continue;
        for (int e = threadIdx.x; e < g.E; e += kRowThreads) bins[e] = 0;
        __syncthreads();
        const long long stop = static_cast<long long>(end) * g.K;
        for (long long i = static_cast<long long>(begin) * g.K + threadIdx.x; i < stop; i += kRowThreads) {
            if (g.mask != nullptr && !g.mask[i / g.K]) continue;
            const long long e = g.ids_i32 ? static_cast<const int*>(g.top)[i] : static_cast<const long long*>(g.top)[i];
            if (e >= 0 && e < g.E) atomicAdd(&bins[e], 1);
        }
        __syncthreads();
        for (int e = threadIdx.x; e < g.E; e += kRowThreads)
            if (bins[e]) atomicAdd(&g.counts[static_cast<size_t>(s) * g.E + e], bins[e]);
        __syncthreads();
        pos = end;
    }
}

template <typename T, int kPerLane>
int launch_rows(const BalanceParams& p, cudaStream_t s) {
    const size_t smem = static_cast<size_t>(kWarps + 1) * p.E * 4;
    return launch_kernel(balance_rows_kernel<T, kPerLane>, p.blocks, kRowThreads, smem, s, false, false, p);
}

template <typename T, int kPerLane>
int launch_bwd(const BalanceBwdParams& p, cudaStream_t s) {
    const int blocks = std::min((p.T + kWarps - 1) / kWarps, device_sm_count() * 8);
    return launch_kernel(balance_bwd_kernel<T, kPerLane>, blocks, kRowThreads, 0, s, false, false, p);
}

#define MOK_PER_LANE(call)                                                                       \
    [&] {                                                                                        \
        const int per_lane = (p.E + 31) / 32;                                                    \
        if (per_lane <= 1) return call(1);                                                       \
        if (per_lane <= 2) return call(2);                                                       \
        if (per_lane <= 4) return call(4);                                                       \
        if (per_lane <= 8) return call(8);                                                       \
        if (per_lane <= 16) return call(16);                                                     \
        return call(32);                                                                         \
    }()

bool bad_sizes(int T, int E, int K, int S) { return T <= 0 || E <= 0 || K <= 0 || K > 255 || S <= 0; }
bool too_many_routes(int T, int K) { return static_cast<long long>(T) * K > 0x7fffffffll; }      // counts are 32-bit

}  // namespace
}  // namespace mok

using namespace mok;

extern "C" size_t mok_router_balance_scratch_bytes(int num_tokens, int num_experts, int num_sequences) {
    if (bad_sizes(num_tokens, num_experts, 1, num_sequences)) return 0;
    return Scratch(nullptr, row_blocks(num_tokens) + num_sequences, num_experts, num_sequences).bytes;
}

extern "C" int mok_router_balance(const void* logits, int logits_bf16, int num_tokens, int num_experts, int topk, int num_sequences,
                                  int sigmoid, const int64_t* top_experts_in, int64_t* top_experts_out, float* router_weights,
                                  const uint8_t* token_mask, const int32_t* sequence_offsets, const int32_t* load, float* losses,
                                  int32_t* counts, float* coef, void* scratch, size_t scratch_bytes, void* stream) {
    if (!logits || !losses || !counts || !coef || !scratch || bad_sizes(num_tokens, num_experts, topk, num_sequences)) return MOK_ERR_INVALID;
    if ((top_experts_in == nullptr) != (top_experts_out != nullptr && router_weights != nullptr)) return MOK_ERR_INVALID;
    if (!top_experts_in && (topk > 32 || topk > num_experts)) return MOK_ERR_INVALID;
    if (!sequence_offsets && num_sequences != 1) return MOK_ERR_INVALID;
    if (num_experts > 1024) return MOK_ERR_UNSUPPORTED;
    const int tiles = (num_experts + kJoinCols - 1) / kJoinCols;
    if (too_many_routes(num_tokens, topk) || static_cast<long long>(num_sequences) * tiles > 0x3fffffff) return MOK_ERR_TOO_LARGE;
    BalanceParams p{};
    p.blocks = row_blocks(num_tokens);
    const Scratch at(scratch, p.blocks + num_sequences, num_experts, num_sequences);
    if (scratch_bytes < at.bytes || reinterpret_cast<uintptr_t>(scratch) % 16) return MOK_ERR_INVALID;
    p.logits = logits;
    p.top_in = reinterpret_cast<const long long*>(top_experts_in);
    p.top_out = reinterpret_cast<long long*>(top_experts_out);
    p.weights = router_weights;
    p.mask = token_mask;
    p.offsets = sequence_offsets;
    p.load = load;
    p.losses = losses;
    p.counts = counts;
    p.coef = coef;
    p.T = num_tokens; p.E = num_experts; p.K = topk; p.S = num_sequences;
    p.rows_per_block = (num_tokens + p.blocks - 1) / p.blocks;
    p.sigmoid = sigmoid;
    p.head = at.head; p.slot_p = at.p; p.slot_routes = at.routes; p.part = at.part; p.seq_z = at.seq_z; p.seq_rows = at.seq_rows;
    p.ticket = at.ticket;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    ProfScope prof(kSlotOther, s, 2);
    int rc;
    if (logits_bf16) {
#define MOK_CALL(n) launch_rows<__nv_bfloat16, n>(p, s)
        rc = MOK_PER_LANE(MOK_CALL);
#undef MOK_CALL
    } else {
#define MOK_CALL(n) launch_rows<float, n>(p, s)
        rc = MOK_PER_LANE(MOK_CALL);
#undef MOK_CALL
    }
    if (rc != MOK_OK) return rc;
    return launch_kernel(balance_join_kernel, num_sequences * tiles, kJoinThreads, 0, s, false, false, p);
}

extern "C" int mok_router_balance_bwd(const float* d_losses, const void* logits, int logits_bf16, const float* coef,
                                      const uint8_t* token_mask, const int32_t* sequence_offsets, const int64_t* top_experts,
                                      const float* router_weights, const float* d_router_weights, void* d_logits, int num_tokens,
                                      int num_experts, int topk, int num_sequences, int sigmoid, void* stream) {
    if (!d_losses || !logits || !coef || !d_logits || bad_sizes(num_tokens, num_experts, topk, num_sequences)) return MOK_ERR_INVALID;
    const int with = (top_experts != nullptr) + (router_weights != nullptr) + (d_router_weights != nullptr);
    if (with != 0 && (with != 3 || topk > 32)) return MOK_ERR_INVALID;
    if (!sequence_offsets && num_sequences != 1) return MOK_ERR_INVALID;
    if (num_experts > 1024) return MOK_ERR_UNSUPPORTED;
    BalanceBwdParams p{d_losses, logits, coef, token_mask, sequence_offsets, reinterpret_cast<const long long*>(top_experts),
                       router_weights, d_router_weights, d_logits, num_tokens, num_experts, topk, num_sequences, sigmoid};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    ProfScope prof(kSlotOther, s);
    if (logits_bf16) {
#define MOK_CALL(n) launch_bwd<__nv_bfloat16, n>(p, s)
        return MOK_PER_LANE(MOK_CALL);
#undef MOK_CALL
    }
#define MOK_CALL(n) launch_bwd<float, n>(p, s)
    return MOK_PER_LANE(MOK_CALL);
#undef MOK_CALL
}

extern "C" int mok_expert_counts(const void* top_experts, int ids_i32, int num_tokens, int topk, int num_experts, int num_sequences,
                                 const uint8_t* token_mask, const int32_t* sequence_offsets, int32_t* counts, void* stream) {
    if (!top_experts || !counts || bad_sizes(num_tokens, num_experts, topk, num_sequences)) return MOK_ERR_INVALID;
    if (!sequence_offsets && num_sequences != 1) return MOK_ERR_INVALID;
    if (num_experts > 1024) return MOK_ERR_UNSUPPORTED;
    if (too_many_routes(num_tokens, topk)) return MOK_ERR_TOO_LARGE;
    const int blocks = std::min((num_tokens + 63) / 64, device_sm_count() * 4);
    CountParams p{top_experts, ids_i32, token_mask, sequence_offsets, counts, num_tokens, num_experts, topk, num_sequences,
                  (num_tokens + blocks - 1) / blocks};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    ProfScope prof(kSlotOther, s);
    MOK_CUDA_CHECK(cudaMemsetAsync(counts, 0, static_cast<size_t>(num_sequences) * num_experts * 4, s));
    return launch_kernel(expert_counts_kernel, blocks, kRowThreads, static_cast<size_t>(num_experts) * 4, s, false, false, p);
}
