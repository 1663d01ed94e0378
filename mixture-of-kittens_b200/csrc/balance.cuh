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
// (block, sequence) pairs that meet, that sum never repeats).  balance_join_kernel adds the slots of a sequence in an
// order that depends on the sizes alone.  A small batch of one sequence is one launch of one cluster, whose blocks read one
// another's sums from shared memory.  No floating-point atomics: two runs give the same bytes.
//
// Here: what the kernels share.  balance_rows.cuh holds the two that work on rows, compiled for f32 and bf16 logits in files of
// their own; balance.cu the join, the counts and the C entries.
#pragma once

#include "common.cuh"

namespace mok {
namespace balance {

constexpr int kWarps = 16;
constexpr int kRowThreads = kWarps * 32;
constexpr int kBwdThreads = 256;
// Blocks of the backward pass that an SM has to be able to hold, which bounds their registers; the grid is twice as many.
// One B200, us, losses alone and with the router weights' gradient:
//   131072 x 256 f32                     three 52 and 68   four 47 and 58   five 45 and 54   six 47 and 54
//   the same with sigmoid scores                83              76               77               83  (with the weights)
//   65536 x 500 bf16, 61 sequences       two 49            three 42         four 39          five 51  (losses alone)
//   30000 x 500 f32, sigmoid scores      two 34 and 41     three 36 and 43  four 45 and 51
//   the same in bf16                         34 and 44           34 and 42       40 and 48
//   30000 x 1024 f32                     one 50 and 58     two 43 and 46    three 59 and 65
//   the same with sigmoid scores             69 and 83         71 and 81         148 and 158
//   the same in bf16                         80 and 101        71 and 81         125 and 137
// One block fewer spills nothing.  Those chosen store 12 spilled bytes at 512 experts, with sigmoid scores up to 52 at 256 and fewer, 136
// at 512, 436 (f32) and 476 at 1024; one block more 172 to 412, with sigmoid scores 240 to 948, above 256 experts.
constexpr int bwd_blocks_per_sm(int V, bool sigmoid) { return V <= 8 ? 5 : V == 16 ? 4 - sigmoid : 2; }
constexpr int kSumRows = kWarps / 2;           // rows of E sums in shared memory that a block's warps share, two to a row
// Blocks of the forward pass, all resident at once on 148 SMs: two an SM up to 512 experts, one above (their rows take twice
// the registers).  Not read from the device: the order of the sums is the same on every GPU.
constexpr int row_blocks_per_sm(int E) { return E <= 512 ? 2 : 1; }
constexpr int kCluster = 8;                    // blocks of a forward pass in one launch
constexpr unsigned kAll = 0xffffffffu;
enum : int { kNone = 0, kRounds = 1, kRank = 2, kMany = 3 };      // how a launch chooses its routes (kNone: they are finished)

struct SlotHead { float z; int rows, routes, pad; };

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
    int one_launch;                // the blocks are one cluster and do the join themselves
    int sigmoid;
    int chunk;                     // see chunk_of
    SlotHead* head;
    float* slot_p;
    int* slot_routes;
    float* part;
    float* seq_z;
    int* seq_rows;
    unsigned* ticket;
};

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
    int T, E, K, S, sigmoid, rows_per_block;
    int chunk, coef_chunk;         // see chunk_of: for the logits and their gradient, and for coef
};

// launches for logits of one type (balance_f32.cu, balance_bf16.cu)
int rows_f32(const BalanceParams& p, cudaStream_t s);
int rows_bf16(const BalanceParams& p, cudaStream_t s);
int backward_f32(const BalanceBwdParams& p, cudaStream_t s);
int backward_bf16(const BalanceBwdParams& p, cudaStream_t s);

// Reductions over groups of kLanes neighbouring lanes; every lane of the warp takes part.
template <int kLanes>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
    for (int off = kLanes / 2; off > 0; off >>= 1) v += __shfl_xor_sync(kAll, v, off);
    return v;
}
template <int kLanes>
__device__ __forceinline__ float group_max(float v) {       // a NaN loses against any number
    if constexpr (kLanes == 32) {
        float m;
        asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
        return m;
    }
#pragma unroll
    for (int off = kLanes / 2; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor_sync(kAll, v, off));
    return v;
}

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_float(float v, float& out) { out = v; }
__device__ __forceinline__ void from_float(float v, __nv_bfloat16& out) { out = __float2bfloat16_rn(v); }

// n (4 or 8) values from / to memory on a boundary of n values
template <int n> __device__ __forceinline__ void load_chunk(const float* p, float* v) {
    if constexpr (n == 8) {
        uint32_t r[8];
        ld_global_256(p, r);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r[i]);
    } else {
        const float4 r = *reinterpret_cast<const float4*>(p);
        v[0] = r.x; v[1] = r.y; v[2] = r.z; v[3] = r.w;
    }
}
template <int n> __device__ __forceinline__ void load_chunk(const __nv_bfloat16* p, float* v) {
    uint32_t w[n / 2];
    if constexpr (n == 8) {
        const uint4 r = *reinterpret_cast<const uint4*>(p);
        w[0] = r.x; w[1] = r.y; w[2] = r.z; w[3] = r.w;
    } else {
        const uint2 r = *reinterpret_cast<const uint2*>(p);
        w[0] = r.x; w[1] = r.y;
    }
#pragma unroll
    for (int i = 0; i < n / 2; ++i) { const float2 t = unpack_bf16(w[i]); v[2 * i] = t.x; v[2 * i + 1] = t.y; }
}
template <int n> __device__ __forceinline__ void store_chunk(float* p, const float* v) {
    if constexpr (n == 8)
        st_global_256(p, __float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]), __float_as_uint(v[4]),
                      __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7]));
    else *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}
template <int n> __device__ __forceinline__ void store_chunk(__nv_bfloat16* p, const float* v) {
    if constexpr (n == 8) *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
    else *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]));
}

// How a group of kLanes lanes holds a row of E values, V a lane: eight (four, where V is four) neighbours a lane at a time, so
// that the group's accesses are contiguous.  A lane's values are in the order of the experts.
template <int kLanes, int V> struct Held {
    static constexpr int kUnit = V < 8 ? V : 8;
    static __device__ __forceinline__ int expert(int l, int j) { return (j / kUnit) * (kLanes * kUnit) + l * kUnit + j % kUnit; }
    static __device__ __forceinline__ int count(int l, int E) {          // values of lane l that are there
        int n = 0;
#pragma unroll
        for (int j = 0; j < V; j += kUnit) n += min(max(E - expert(l, j), 0), kUnit);
        return n;
    }
};

// Values past E read as `fill`.
template <int kLanes, int V, typename T>
__device__ __forceinline__ void load_row(const T* row, int l, int E, int chunk, float fill, float (&v)[V]) {
    using At = Held<kLanes, V>;
    if constexpr (V >= 8) {
        if (chunk == 8) {
#pragma unroll
            for (int j = 0; j < V; j += 8) {
                if (At::expert(l, j) < E) load_chunk<8>(row + At::expert(l, j), v + j);
                else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[j + i] = fill;
                }
            }
            return;
        }
    }
    if (chunk >= 4) {
#pragma unroll
        for (int j = 0; j < V; j += 4) {
            if (At::expert(l, j) < E) load_chunk<4>(row + At::expert(l, j), v + j);
            else { v[j] = fill; v[j + 1] = fill; v[j + 2] = fill; v[j + 3] = fill; }
        }
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = At::expert(l, j) < E ? to_float(row[At::expert(l, j)]) : fill;
    }
}
template <int kLanes, int V, typename T>
__device__ __forceinline__ void store_row(T* row, int l, int E, int chunk, const float (&v)[V]) {
    using At = Held<kLanes, V>;
    if constexpr (V >= 8) {
        if (chunk == 8) {
#pragma unroll
            for (int j = 0; j < V; j += 8) if (At::expert(l, j) < E) store_chunk<8>(row + At::expert(l, j), v + j);
            return;
        }
    }
    if (chunk >= 4) {
#pragma unroll
        for (int j = 0; j < V; j += 4) if (At::expert(l, j) < E) store_chunk<4>(row + At::expert(l, j), v + j);
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) if (At::expert(l, j) < E) from_float(v[j], row[At::expert(l, j)]);
    }
}

// another block's copy of a shared-memory object of this cluster
__device__ __forceinline__ uint32_t remote_shared(const void* p, int block) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(block));
    return at;
}
__device__ __forceinline__ float remote_load(const float* p, int block) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(remote_shared(p, block)) : "memory");
    return v;
}
__device__ __forceinline__ int remote_load(const int* p, int block) {
    int v;
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(remote_shared(p, block)) : "memory");
    return v;
}
__device__ __forceinline__ void remote_store(float* p, int block, float v) {
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(remote_shared(p, block)), "f"(v) : "memory");
}

// A row of values in shared memory, where every lane of a group stores and loads its own V of them four at a time: chunk-major
// and padded by one chunk, so that neither the lanes' accesses nor those of threads that take neighbouring experts conflict.
template <int kLanes, int V> struct SharedRow {
    static constexpr int kFloats = V * (kLanes + 1);
    static __device__ __forceinline__ int chunk(int lane, int j) { return ((j >> 2) * (kLanes + 1) + lane) << 2; }
    static __device__ __forceinline__ int at(int e) {
        constexpr int kUnit = Held<kLanes, V>::kUnit;
        return chunk(e / kUnit % kLanes, e / (kLanes * kUnit) * kUnit + e % kUnit) + (e & 3);
    }
};

// Sequence bounds as the kernels use them: inside [0, T] whatever the caller's array holds.
__device__ __forceinline__ int seq_bound(const int* offsets, int s, int T) {
    if (offsets == nullptr) return s ? T : 0;
    return min(max(offsets[s], 0), T);
}
// First sequence that ends behind row `row` (S if none); a whole warp searches, 32 sequences at a time.
__device__ __forceinline__ int first_sequence(const int* offsets, int S, int row, int T) {
    if (offsets == nullptr) return 0;
    const int lane = threadIdx.x & 31;
    int lo = 0, n = S;
    while (n > 0) {
        const int step = (n + 31) / 32, probe = lo + lane * step;
        const bool before = probe < lo + n && seq_bound(offsets, probe + 1, T) <= row;
        const int passed = __popc(__ballot_sync(kAll, before));
        const int hi = min(lo + passed * step, lo + n);            // ends behind the row, or the end of the range
        if (passed > 0) lo += (passed - 1) * step + 1;
        n = passed > 0 ? hi - lo : 0;
    }
    return lo;
}

// Exponentials, logarithms and quotients go through the hardware's approximate base-2 ones, results below 2^-126 flushed to
// zero: 2^-22 relative and the rounding of the argument, below what the sums over a row round away.  The row's maximum is taken
// off before the multiplication by log2(e): a row of the type's lowest value would overflow in one fused multiply-add.
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
__device__ __forceinline__ float exp2_fast(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ float rcp_fast(float x) { float y; asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ float log_fast(float x) { float y; asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y * kLn2; }

// sigma(l) times a factor common to the row whose maximum is m: exp(-m) where m is negative, so that the sum over the row
// cannot underflow; the factor cancels in every quotient
__device__ __forceinline__ float sigmoid_scaled(float l, float m) {
    if (m >= 0.0f) return rcp_fast(1.0f + exp2_fast(-l * kLog2e));
    return exp2_fast((l - (m > -INFINITY ? m : 0.0f)) * kLog2e) * rcp_fast(1.0f + exp2_fast(l * kLog2e));
}
__device__ __forceinline__ float sigmoid_rest(float l) { return rcp_fast(1.0f + exp2_fast(l * kLog2e)); }      // 1 - sigma(l)

// Of one row held by a group of kLanes lanes: ex = exponentials and inv the reciprocal of their sum (softmax = ex inv), for
// sigmoid scores also sg = scaled sigmoids and inv_sg.  inv is 0 for a row without a logit above -inf, and lse then 0.
struct RowStats { float inv, inv_sg, lse; };
template <int kLanes, int V>
__device__ __forceinline__ float row_max(const float (&v)[V]) {              // NaN where there is nothing else
    float m = v[0];
#pragma unroll
    for (int j = 1; j < V; ++j) m = fmaxf(m, v[j]);
    return group_max<kLanes>(m);
}
template <int kLanes, int V, bool kSigmoid>
__device__ __forceinline__ RowStats row_stats(const float (&v)[V], float m, float (&ex)[V], float (&sg)[V]) {      // m: row_max, or -inf for NaN
    const float base = m > -INFINITY ? m : 0.0f;
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < V; ++j) { ex[j] = exp2_fast((v[j] - base) * kLog2e); sum += ex[j]; }     // lanes past E hold -inf: 0
    sum = group_sum<kLanes>(sum);
    RowStats r;
    r.inv = sum == 0.0f ? 0.0f : rcp_fast(sum);
    r.lse = sum == 0.0f ? 0.0f : base + log_fast(sum);
    r.inv_sg = 0.0f;
    if constexpr (kSigmoid) {
        float total = 0.0f;
#pragma unroll
        for (int j = 0; j < V; ++j) { sg[j] = sigmoid_scaled(v[j], m); total += sg[j]; }
        total = group_sum<kLanes>(total);
        r.inv_sg = total == 0.0f ? 0.0f : rcp_fast(total);
    }
    return r;
}

__device__ __forceinline__ int warp_sum(int v) { return __reduce_add_sync(kAll, v); }

__device__ __forceinline__ float expert_share(int E, int routes, int of) {
    return static_cast<float>(E) * static_cast<float>(routes) / static_cast<float>(max(of, 1));
}
__device__ __forceinline__ void write_losses(const BalanceParams& g, float balance, float z, int rows, int live) {
    const float n = static_cast<float>(max(rows, 1)), sequences = static_cast<float>(max(live, 1));
    g.losses[0] = balance / sequences;
    g.losses[1] = z / n;
    g.coef[static_cast<size_t>(g.S) * g.E] = 1.0f / sequences;
    g.coef[static_cast<size_t>(g.S) * g.E + 1] = 2.0f / n;
}

}  // namespace balance
}  // namespace mok
