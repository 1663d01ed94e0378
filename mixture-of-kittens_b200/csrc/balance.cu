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

constexpr int kWarps = 16;
constexpr int kRowThreads = kWarps * 32;
constexpr int kBwdThreads = 256;
// Blocks of the backward pass that an SM has to be able to hold, which bounds their registers; the grid is twice as many.
// One B200, us: 131072 x 256 f32 with five 53, four 58, six 55; 65536 x 500 bf16 with four 56, two 70, sigmoid scores 30000 x 500
// with three 36, four (spills) 44; 30000 x 1024 f32 with two 63, three (spills) 88 to 92.
constexpr int bwd_blocks_per_sm(int V, bool sigmoid) { return V <= 8 ? 5 : V == 16 ? 4 - sigmoid : 2; }
constexpr int kSumRows = kWarps / 2;           // rows of E sums in shared memory that a block's warps share, two to a row
// Blocks of the forward pass, all resident at once on 148 SMs: two an SM up to 512 experts, one above (their rows take twice
// the registers).  Not read from the device: the order of the sums is the same on every GPU.
constexpr int row_blocks_per_sm(int E) { return E <= 512 ? 2 : 1; }
constexpr int kCluster = 8;                    // blocks of a forward pass in one launch
constexpr int kMinCols = 8;                    // fewest experts of a join tile
constexpr unsigned kAll = 0xffffffffu;
enum : int { kNone = 0, kFew = 1, kMany = 2 };      // routes that a launch chooses: finished ones, up to 16, more

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
        const int tiles = (E + kMinCols - 1) / kMinCols;
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

// rows that a block works on at once
int rows_at_once(int E) { return kWarps * (E <= 16 ? 8 : E <= 32 ? 4 : E <= 64 ? 2 : 1); }
// One launch of one cluster that joins its blocks' sums through shared memory and needs no scratch, or one launch of many
// blocks and one that joins their slots.  Up to two rows a group of lanes the cluster saves the caller a launch and an
// allocation, 4 us of its time; the device takes 6.5 us for one row a group and 7.1 to 9.8 for two, against 7 to 9.5 with two launches.
bool in_one_launch(int T, int E, int S) { return S == 1 && T <= 2 * kCluster * rows_at_once(E); }
int rows_per_block(int T, int E, int S) {
    const int most = in_one_launch(T, E, S) ? kCluster : 148 * row_blocks_per_sm(E), at_once = rows_at_once(E);
    const int rows = (T + most - 1) / most;
    return (rows + at_once - 1) / at_once * at_once;
}
int row_blocks(int T, int E, int S) {
    if (in_one_launch(T, E, S)) return kCluster;
    const int rows = rows_per_block(T, E, S);
    return (T + rows - 1) / rows;
}

// how rows of E values of `bytes` bytes at `base` can be read: chunks of eight (16 or 32 bytes), of four, or one by one
int chunk_of(const void* base, int E, int bytes) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(base);
    if (E % 8 == 0 && at % (8 * bytes) == 0) return 8;
    return E % 4 == 0 && at % (4 * bytes) == 0 ? 4 : 1;
}

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
template <int kLanes>
__device__ __forceinline__ int group_min(int v) {
    if constexpr (kLanes == 32) return __reduce_min_sync(kAll, v);
#pragma unroll
    for (int off = kLanes / 2; off > 0; off >>= 1) v = min(v, __shfl_xor_sync(kAll, v, off));
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

// The two largest values a lane has left, the lower index first among equals; slot V: none above -inf (a NaN is never above
// anything, so it ranks with -inf).
template <int V>
__device__ __forceinline__ void two_largest(const float (&v)[V], unsigned taken, float& b1, int& j1, float& b2, int& j2) {
    b1 = b2 = -INFINITY;
    j1 = j2 = V;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const float x = (taken >> j) & 1u ? -INFINITY : v[j];
        const bool first = x > b1, second = x > b2;
        b2 = first ? b1 : second ? x : b2;
        j2 = first ? j1 : second ? j : j2;
        b1 = first ? x : b1;
        j1 = first ? j : j1;
    }
}

// The K largest values of a row, descending, the lower expert first among equals, into chosen[0..K) (shared memory of the
// group) as (value, expert).
//
// In rounds: every lane keeps the two largest values it has left; a round is one maximum over the group, the winner moves its
// second up, and a lane that has used up both looks through its values again (with K = 8 of 256 over 32 lanes in half of
// the rows; one kept value would mean a search in every round).
template <int kLanes, int V>
__device__ __forceinline__ void select_in_rounds(const float (&v)[V], int E, int K, float2* chosen) {
    const int lane = threadIdx.x & 31, l = lane % kLanes;
    const unsigned group = kLanes == 32 ? kAll : ((1u << kLanes) - 1u) << (lane - l);
    const unsigned below = (1u << lane) - 1u;
    using At = Held<kLanes, V>;
    const int mine = At::count(l, E);
    unsigned taken = 0;
    float b1, b2;
    int j1, j2;
    two_largest(v, 0u, b1, j1, b2, j2);
    for (int k = 0; k < K; ++k) {
        const float best = group_max<kLanes>(b1);
        const bool equal = j1 < V && b1 == best;
        const unsigned at = __ballot_sync(kAll, equal) & group;
        bool win = equal && (at & below) == 0;
        if (V > At::kUnit && __any_sync(kAll, (at & (at - 1)) != 0)) {          // equals in several lanes, whose experts interleave
            const int e = equal ? At::expert(l, j1) : 0x7fffffff;
            win = e == group_min<kLanes>(e) && equal;
        }
        if (win) chosen[k] = make_float2(best, __int_as_float(At::expert(l, j1)));
        taken |= win ? 1u << (j1 & 31) : 0u;
        const bool dry = win && j2 == V;
        b1 = win ? b2 : b1;
        j1 = win ? j2 : j1;
        b2 = win ? -INFINITY : b2;
        j2 = win ? V : j2;
        if (__any_sync(kAll, at == 0)) {                           // nothing above -inf left: the lowest experts not taken yet
            const unsigned left = ~taken & (V == 32 && mine == 32 ? kAll : (1u << mine) - 1u);
            const int e = left ? At::expert(l, __ffs(left) - 1) : 0x7fffffff;
            const int lowest = group_min<kLanes>(e);
            if (at == 0 && e == lowest && left) { chosen[k] = make_float2(-INFINITY, __int_as_float(e)); taken |= left & (0u - left); }
        }
        if (__any_sync(kAll, dry)) { if (dry) two_largest(v, taken, b1, j1, b2, j2); }
    }
    __syncwarp();
}

__device__ __forceinline__ float warp_min(float v) {
    float m;
    asm volatile("redux.sync.min.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
    return m;
}

// Values >= t into gathered[0..min(n, 32)), one slot each in no order that matters; returns how many there are.  Written out so
// that the store is predicated: as a branch a value it costs three instructions more.
template <int V>
__device__ __forceinline__ int gather_above(const float (&v)[V], float t, uint2* gathered) {
    const int lane = threadIdx.x & 31;
    const uint32_t below = (1u << lane) - 1u, base = smem_u32(gathered);
    uint32_t n = 0;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        asm volatile(
            "{\n\t.reg .pred p;\n\t.reg .b32 at, to;\n\t"
            "setp.ge.f32 p, %1, %2;\n\t"
            "vote.sync.ballot.b32 at, p, 0xffffffff;\n\t"
            "and.b32 to, at, %3;\n\t"
            "popc.b32 to, to;\n\t"
            "add.u32 to, to, %0;\n\t"
            "and.b32 to, to, 31;\n\t"
            "mad.lo.u32 to, to, 8, %4;\n\t"
            "@p st.shared.v2.b32 [to], {%5, %6};\n\t"
            "popc.b32 at, at;\n\t"
            "add.u32 %0, %0, at;\n\t}"
            : "+r"(n)
            : "f"(v[j]), "f"(t), "r"(below), "r"(base), "r"(Held<32, V>::expert(lane, j)), "r"(__float_as_uint(v[j]))
            : "memory");
    }
    return static_cast<int>(n);
}

// The largest sets of lanes of which there are K (one of which half the lanes have values counts); 0: there are none.
template <int V>
__device__ __forceinline__ int set_of(int E, int K) {
    const int lanes = min(32, (E + Held<32, V>::kUnit - 1) / Held<32, V>::kUnit);
    int set = 32;
    while (set > 0 && (lanes + set / 2) / set < K) set >>= 1;
    return set;
}

// One row a warp.  Let the lanes form K sets of `set` neighbours, as large as they can be, and t be the least of the sets'
// maxima: at least K values are >= t, and few more.  They are gathered, one a lane, and every lane counts those that come before
// its own.  With t the second, third or fourth least for more routes there are fewer to gather and still nearly always K (8 of 256,
// second least: 13 on average, fewer than 8 in 2 rows of 100; least: 21, more than 32 in 9 of 100).  In the rows where that fails t
// is the K-th largest of the lanes' maxima, and where that does not do either (many equal values, few above -inf, no such sets:
// set = 0) the row goes in rounds.
template <int V>
__device__ __forceinline__ void select_by_rank(const float (&v)[V], int E, int K, int set, uint2* gathered, float2* chosen) {
    const int lane = threadIdx.x & 31;
    float b = v[0];
#pragma unroll
    for (int j = 1; j < V; ++j) b = fmaxf(b, v[j]);
    b = b > -INFINITY ? b : -INFINITY;                             // all NaN
    float t = b;
    for (int off = 1; off < set; off <<= 1) t = fmaxf(t, __shfl_xor_sync(kAll, t, off));
    float least = lane < K * set ? t : INFINITY;
    t = warp_min(least);
    for (int i = K < 5 ? 0 : K < 11 ? 1 : K < 15 ? 2 : 3; i > 0; --i) {
        least = least == t ? INFINITY : least;
        t = warp_min(least);
    }
    int n = 33;
    if (set > 0 && t > -INFINITY) n = gather_above(v, t, gathered);
    if (n > 32 || n < K) {
        int found = 0;
        do {
            t = group_max<32>(b);
            const bool equal = b == t;
            found += __popc(__ballot_sync(kAll, equal));
            b = equal ? -INFINITY : b;
        } while (found < K && t > -INFINITY);
        __syncwarp();
        n = t > -INFINITY ? gather_above(v, t, gathered) : 33;
        if (n > 32) { select_in_rounds<32, V>(v, E, K, chosen); return; }
    }
    __syncwarp();
    // (value, expert) as one 64-bit number that grows with the value (-0 as 0) and falls with the expert
    const uint2 own = gathered[lane];                              // past n: left over, not used
    const float value = __uint_as_float(own.y) + 0.0f;
    const unsigned bits = __float_as_uint(value);
    const unsigned order = bits ^ (static_cast<int>(bits) < 0 ? 0xffffffffu : 0x80000000u);
    unsigned long long* const keys = reinterpret_cast<unsigned long long*>(gathered);
    const unsigned long long key = lane < n ? static_cast<unsigned long long>(order) << 32 | (0xffffffffu - own.x) : 0ull;
    keys[lane] = key;
    __syncwarp();
    int before = 0;
#pragma unroll 2
    for (int i = 0; i < n; i += 4) {                               // past n: 0, before nothing
        const ulonglong2 a = *reinterpret_cast<const ulonglong2*>(keys + i), c = *reinterpret_cast<const ulonglong2*>(keys + i + 2);
        before += (a.x > key) + (a.y > key) + (c.x > key) + (c.y > key);
    }
    if (lane < n && before < K) chosen[before] = make_float2(__uint_as_float(own.y), __int_as_float(static_cast<int>(own.x)));
    __syncwarp();
}

// More than 16 of a row would rarely leave 32 or fewer values >= t: 16 are chosen at a time and taken out of v (131072 x 256, 32 of
// them: 444 us in rounds, 179 so; in kernels of their own, because the code beside it costs the choice of fewer 14 % and more).
template <int V>
__device__ __forceinline__ void select_many(float (&v)[V], int E, int K, uint2* gathered, float2* chosen) {
    const int lane = threadIdx.x & 31;
    int above = 0;                                                 // values above -inf; with fewer than K the choice goes beyond them
#pragma unroll
    for (int j = 0; j < V; ++j) above += __popc(__ballot_sync(kAll, v[j] > -INFINITY));
    if (above < K) { select_in_rounds<32, V>(v, E, K, chosen); return; }
    for (int from = 0; from < K; from += 16) {
        const int some = min(K - from, 16);
        select_by_rank<V>(v, E, some, set_of<V>(E, some), gathered, chosen + from);
        const float2 last = chosen[from + some - 1];
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (v[j] > last.x || (v[j] == last.x && Held<32, V>::expert(lane, j) <= __float_as_int(last.y))) v[j] = -INFINITY;
    }
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

template <int kJoinWarps> struct JoinShared {
    float p[kJoinWarps][32], z[kJoinWarps];
    int c[kJoinWarps][32], rows[kJoinWarps], routes[kJoinWarps];
};

// Adds the slots of a sequence for a tile of kCols experts, in an order that only depends on the sizes, and writes the tile's
// counts, coefficients and part of the loss.  A block of kJoinWarps warps; a warp takes 32 / kCols slots at a time.
template <int kCols, int kJoinWarps>
__device__ __forceinline__ void join_tile(const BalanceParams& g, int index, JoinShared<kJoinWarps>& sh) {
    constexpr int kSub = 32 / kCols;
    const int tiles = (g.E + kCols - 1) / kCols;
    const int s = index / tiles, tile = index - s * tiles;
    const int begin = seq_bound(g.offsets, s, g.T), end = seq_bound(g.offsets, s + 1, g.T);
    const int b0 = begin / g.rows_per_block, b1 = end > begin ? (end - 1) / g.rows_per_block + 1 : b0;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, col = lane % kCols, e = tile * kCols + col;
    float p = 0.0f, z = 0.0f;
    int c = 0, rows = 0, routes = 0;
#pragma unroll 4
    for (int b = b0 + warp * kSub + lane / kCols; b < b1; b += kJoinWarps * kSub) {
        const int4 h = __ldcg(reinterpret_cast<const int4*>(g.head + b + s));          // SlotHead
        z += __int_as_float(h.x); rows += h.y; routes += h.z;
        if (e < g.E) {
            const size_t at = static_cast<size_t>(b + s) * g.E + e;
            p += __ldcg(g.slot_p + at);
            c += __ldcg(g.slot_routes + at);
        }
    }
#pragma unroll
    for (int off = kCols; off < 32; off <<= 1) {
        p += __shfl_xor_sync(kAll, p, off);
        z += __shfl_xor_sync(kAll, z, off);
        c += __shfl_xor_sync(kAll, c, off);
        rows += __shfl_xor_sync(kAll, rows, off);
        routes += __shfl_xor_sync(kAll, routes, off);
    }
    sh.p[warp][lane] = p;
    sh.c[warp][lane] = c;
    if (lane == 0) { sh.z[warp] = z; sh.rows[warp] = rows; sh.routes[warp] = routes; }
    __syncthreads();
    if (warp == 0) {
        const bool one = lane < kJoinWarps;
        z = group_sum<32>(one ? sh.z[lane] : 0.0f);
        rows = warp_sum(one ? sh.rows[lane] : 0);
        routes = one ? sh.routes[lane] : 0;
        if (g.load != nullptr) {
            routes = 0;
            for (int i = lane; i < g.E; i += 32) routes += g.load[static_cast<size_t>(s) * g.E + i];
        }
        routes = warp_sum(routes);
        p = 0.0f;
        c = 0;
#pragma unroll
        for (int w = lane / kCols; w < kJoinWarps; w += kSub) { p += sh.p[w][col]; c += sh.c[w][col]; }
#pragma unroll
        for (int off = kCols; off < 32; off <<= 1) { p += __shfl_xor_sync(kAll, p, off); c += __shfl_xor_sync(kAll, c, off); }
        float part = 0.0f;
        if (lane < kCols && e < g.E) {
            const size_t at = static_cast<size_t>(s) * g.E + e;
            g.counts[at] = c;
            const int used = g.load != nullptr ? g.load[at] : c;
            const float a = rows > 0 ? expert_share(g.E, used, routes) / static_cast<float>(rows) : 0.0f;
            g.coef[at] = a;
            part = a * p;
        }
        part = group_sum<32>(part);
        if (lane == 0) {
            g.part[index] = part;
            if (tile == 0) { g.seq_z[s] = z; g.seq_rows[s] = rows; }
        }
    }
}

// The losses and what backward needs beside the coefficients, from the tiles' parts; one block.
template <int kJoinWarps>
__device__ __forceinline__ void finish(const BalanceParams& g, int parts, JoinShared<kJoinWarps>& sh) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float balance = 0.0f, z = 0.0f;
    int live = 0, rows = 0;
    for (int i = threadIdx.x; i < parts; i += kJoinWarps * 32) balance += __ldcg(g.part + i);
    for (int i = threadIdx.x; i < g.S; i += kJoinWarps * 32) {
        const int n = __ldcg(g.seq_rows + i);
        z += __ldcg(g.seq_z + i);
        rows += n;
        live += n > 0;
    }
    balance = group_sum<32>(balance);
    z = group_sum<32>(z);
    rows = warp_sum(rows);
    live = warp_sum(live);
    __syncthreads();                           // the tile before may still be read
    if (lane == 0) { sh.p[warp][0] = balance; sh.z[warp] = z; sh.rows[warp] = rows; sh.routes[warp] = live; }
    __syncthreads();
    if (warp == 0) {
        const bool one = lane < kJoinWarps;
        balance = group_sum<32>(one ? sh.p[lane][0] : 0.0f);
        z = group_sum<32>(one ? sh.z[lane] : 0.0f);
        rows = warp_sum(one ? sh.rows[lane] : 0);
        live = warp_sum(one ? sh.routes[lane] : 0);
        if (lane == 0) write_losses(g, balance, z, rows, live);
    }
}

// A block a tile; the block that finishes last does finish().  Latency-bound: a few hundred slots at most.
template <int kCols, int kJoinWarps>
__global__ void __launch_bounds__(kJoinWarps * 32) balance_join_kernel(const BalanceParams g) {
    __shared__ JoinShared<kJoinWarps> sh;
    __shared__ bool last;
    pdl_wait();
    join_tile<kCols>(g, blockIdx.x, sh);
    if (threadIdx.x == 0) {
        __threadfence();
        last = atomicAdd(g.ticket, 1u) == gridDim.x - 1;
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
    finish(g, gridDim.x, sh);
}

// Bound by instructions and, without the choice, by the latency of its loads.  Reads T E logits once, writes K routes a row and (p,
// routes) per slot.  One B200 with the join, us (floor: bytes at 6456 GB/s): 131072 x 256 f32, K = 8: 74 (21), finished routes
// 36; 65536 x 500 bf16, K = 6, 61 sequences: 69 (10) and 32; 16384 x 128: 16 (1.3) and 10.  A row of 256 takes 470 instructions
// with the choice, 130 without; in rounds of one maximum each the choice alone took 540.  Loading the next row ahead: 53 -> 44
// without the choice at 256 experts; above, the registers it takes cost more (36 -> 46 at 500).  Finished routes are counted for a
// run's rows at once; with their row, each row waited for its ids (44 -> 36).  Rows staged in shared memory two to four ahead by
// asynchronous copies were slower throughout (44 -> 55, backward 54 -> 73 to 77).
template <typename T, int kLanes, int V, bool kSigmoid, int kChoose>
__global__ void __launch_bounds__(kRowThreads, row_blocks_per_sm(kLanes * V)) balance_rows_kernel(const BalanceParams g) {
    using Row = SharedRow<kLanes, V>;
    constexpr bool kSelect = kChoose != kNone;
    constexpr bool kAhead = V <= 8;            // the next row is loaded while this one is worked on
    constexpr int kGroups = kRowThreads / kLanes;              // rows that a block works on at once
    constexpr int kPer = (kLanes * V < 32 ? kLanes * V : 32) / kLanes;          // chosen experts a lane, at most (K <= 32 and <= E)
    extern __shared__ __align__(16) float smem[];               // sums of p [kSumRows], routes [E], then the chosen (value, expert) [kGroups][K]
    __shared__ alignas(16) uint2 s_gathered[kSelect && kLanes == 32 ? kWarps : 1][32];
    __shared__ float s_z[kWarps], s_part[kWarps], s_parts[kCluster];
    __shared__ int s_rows[kWarps], s_routes;
    int* const hist = reinterpret_cast<int*>(smem + kSumRows * Row::kFloats);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, l = lane % kLanes, group = threadIdx.x / kLanes;
    float2* const chosen = reinterpret_cast<float2*>(hist + ((g.E + 1) & ~1)) + static_cast<size_t>(group) * g.K;
    pdl_wait();
    if (blockIdx.x == 0 && threadIdx.x == 0 && !g.one_launch) *g.ticket = 0;
    const int set = kLanes == 32 && kChoose == kFew ? set_of<V>(g.E, g.K) : 0;
    const long long first = static_cast<long long>(blockIdx.x) * g.rows_per_block;
    int pos = static_cast<int>(min(first, static_cast<long long>(g.T)));
    const int hi = static_cast<int>(min(first + g.rows_per_block, static_cast<long long>(g.T)));
    int s = first_sequence(g.offsets, g.S, pos, g.T);
    bool summed = false;
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
        float acc[V], z = 0.0f;
        int rows = 0, routes = 0;
#pragma unroll
        for (int j = 0; j < V; ++j) acc[j] = 0.0f;
        if (!kSelect && counted) {             // finished routes, of all the run's rows at once
            const size_t at = static_cast<size_t>(pos) * g.K;
            const unsigned n = static_cast<unsigned>(end - pos) * static_cast<unsigned>(g.K);        // a call has fewer than 2^31 routes
#pragma unroll 4
            for (unsigned i = threadIdx.x; i < n; i += kRowThreads) {
                const long long e = g.top_in[at + i];
                if (e >= 0 && e < g.E && (g.mask == nullptr || g.mask[pos + i / static_cast<unsigned>(g.K)])) { atomicAdd(&hist[e], 1); ++routes; }
            }
        }
        // all lanes of a warp stay in step; groups past the run work on nothing
        auto load = [&](int t0, float (&v)[V]) {
            load_row<kLanes, V>(static_cast<const T*>(g.logits) + static_cast<size_t>(min(t0 + lane / kLanes, end - 1)) * g.E, l, g.E, g.chunk, -INFINITY, v);
        };
        float next[V];
        const int t_first = pos + warp * (32 / kLanes);
        if (kAhead && t_first < end && (counted || kSelect)) load(t_first, next);
        for (int t0 = t_first; t0 < end && (counted || kSelect); t0 += kGroups) {
            const int t = t0 + lane / kLanes;
            const bool there = t < end;
            float v[V];
            if constexpr (kAhead) {
#pragma unroll
                for (int j = 0; j < V; ++j) v[j] = next[j];
                if (t0 + kGroups < end) load(t0 + kGroups, next);
            } else {
                load(t0, v);
            }
            const bool live = there && counted && (g.mask == nullptr || g.mask[t]);
            float max_known;
            if constexpr (kSelect) {
                const unsigned o = static_cast<unsigned>(t) * static_cast<unsigned>(g.K);        // a call has fewer than 2^31 routes
                if constexpr (kLanes != 32) {
                    select_in_rounds<kLanes, V>(v, g.E, g.K, chosen);
                } else if constexpr (kChoose == kFew) {
                    select_by_rank<V>(v, g.E, g.K, set, s_gathered[warp], chosen);
                } else {
                    select_many<V>(v, g.E, g.K, s_gathered[warp], chosen);
                    load(t0, v);                                   // as it was
                }
                const float top = chosen[0].x;
                max_known = top;
                auto weight = [&](float x) {
                    return top == -INFINITY ? 0.0f : kSigmoid ? sigmoid_scaled(x, top) : exp2_fast((x - top) * kLog2e);
                };
                float w[kPer], sum = 0.0f;
                int e[kPer];
#pragma unroll
                for (int i = 0; i < kPer; ++i) {
                    const bool mine = l + i * kLanes < g.K;
                    const float2 c = mine ? chosen[l + i * kLanes] : make_float2(0.0f, 0.0f);
                    e[i] = __float_as_int(c.y);
                    w[i] = mine ? weight(c.x) : 0.0f;
                    sum += w[i];
                }
                sum = group_sum<kLanes>(sum);
                const float inv = sum == 0.0f ? 0.0f : rcp_fast(sum);
#pragma unroll
                for (int i = 0; i < kPer; ++i) {
                    if (there && l + i * kLanes < g.K) {
                        g.top_out[o + l + i * kLanes] = e[i];
                        g.weights[o + l + i * kLanes] = w[i] * inv;
                        if (live) { atomicAdd(&hist[e[i]], 1); ++routes; }
                    }
                }
                __syncwarp();
            } else {
                max_known = row_max<kLanes, V>(v);
            }
            if (counted) {
                float ex[V], sg[V];
                const RowStats r = row_stats<kLanes, V, kSigmoid>(v, max_known, ex, sg);
                if (live) {
#pragma unroll
                    for (int j = 0; j < V; ++j) acc[j] = kSigmoid ? fmaf(sg[j], r.inv_sg, acc[j]) : fmaf(ex[j], r.inv, acc[j]);
                    z = fmaf(r.lse, r.lse, z);
                    ++rows;
                }
            }
        }
        if (counted) {
            float* const mine = smem + (warp % kSumRows) * Row::kFloats;
#pragma unroll
            for (int j = 0; j < V; j += 4) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int off = kLanes; off < 32; off <<= 1) acc[j + i] += __shfl_xor_sync(kAll, acc[j + i], off);
                if (warp >= kSumRows && lane < kLanes)
                    *reinterpret_cast<float4*>(mine + Row::chunk(l, j)) = make_float4(acc[j], acc[j + 1], acc[j + 2], acc[j + 3]);
            }
            __syncthreads();
#pragma unroll
            for (int j = 0; j < V; j += 4) {
                if (warp < kSumRows && lane < kLanes) {
                    float4& x = *reinterpret_cast<float4*>(mine + Row::chunk(l, j));
                    x = make_float4(x.x + acc[j], x.y + acc[j + 1], x.z + acc[j + 2], x.w + acc[j + 3]);
                }
            }
#pragma unroll
            for (int off = kLanes; off < 32; off <<= 1) { z += __shfl_xor_sync(kAll, z, off); rows += __shfl_xor_sync(kAll, rows, off); }
            if (routes) atomicAdd(&s_routes, routes);
            if (lane == 0) { s_z[warp] = z; s_rows[warp] = rows; }
            __syncthreads();
            const size_t slot = static_cast<size_t>(blockIdx.x) + s;
            for (int e = threadIdx.x * 4; e < g.E; e += kRowThreads * 4) {
                float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int w = 0; w < kSumRows; ++w) {
                    const float4 x = *reinterpret_cast<const float4*>(smem + w * Row::kFloats + Row::at(e));
                    sum[0] += x.x; sum[1] += x.y; sum[2] += x.z; sum[3] += x.w;
                }
                if (g.one_launch) {                                // stays here: only this thread reads these places of the rows
                    *reinterpret_cast<float4*>(smem + Row::at(e)) = make_float4(sum[0], sum[1], sum[2], sum[3]);
                    continue;
                }
                float* const to_p = g.slot_p + slot * g.E + e;
                int* const to_routes = g.slot_routes + slot * g.E + e;
                if (g.E % 4 == 0) {
                    *reinterpret_cast<float4*>(to_p) = make_float4(sum[0], sum[1], sum[2], sum[3]);
                    *reinterpret_cast<int4*>(to_routes) = make_int4(hist[e], hist[e + 1], hist[e + 2], hist[e + 3]);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) if (e + i < g.E) { to_p[i] = sum[i]; to_routes[i] = hist[e + i]; }
                }
            }
            if (threadIdx.x == 0) {
                SlotHead h{0.0f, 0, s_routes, 0};
                for (int w = 0; w < kWarps; ++w) { h.z += s_z[w]; h.rows += s_rows[w]; }
                if (g.one_launch) { s_z[0] = h.z; s_rows[0] = h.rows; } else g.head[slot] = h;
            }
            __syncthreads();
            summed = true;
            ++s;
        }
        pos = end;
    }
    if (!g.one_launch) return;
    // The blocks are one cluster and there is one sequence: every block joins every eighth expert from the blocks' shared memory.
    if (!summed) {                             // no rows of the sequence here
        for (int e = threadIdx.x * 4; e < g.E; e += kRowThreads * 4) *reinterpret_cast<float4*>(smem + Row::at(e)) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int e = threadIdx.x; e < g.E; e += kRowThreads) hist[e] = 0;
        if (threadIdx.x == 0) { s_z[0] = 0.0f; s_rows[0] = 0; s_routes = 0; }
    }
    __syncthreads();
    cluster_sync_all();
    const bool one = lane < kCluster;
    const float z = group_sum<32>(one ? remote_load(&s_z[0], lane) : 0.0f);
    const int rows = __reduce_add_sync(kAll, one ? remote_load(&s_rows[0], lane) : 0);
    int routes = one ? remote_load(&s_routes, lane) : 0;
    if (g.load != nullptr) {
        routes = 0;
        for (int i = lane; i < g.E; i += 32) routes += g.load[i];
    }
    routes = __reduce_add_sync(kAll, routes);
    float part = 0.0f;
    for (int e = blockIdx.x + threadIdx.x * kCluster; e < g.E; e += kRowThreads * kCluster) {
        float p = 0.0f;
        int c = 0;
#pragma unroll
        for (int b = 0; b < kCluster; ++b) { p += remote_load(smem + Row::at(e), b); c += remote_load(hist + e, b); }
        g.counts[e] = c;
        const int used = g.load != nullptr ? g.load[e] : c;
        const float a = rows > 0 ? expert_share(g.E, used, routes) / static_cast<float>(rows) : 0.0f;
        g.coef[e] = a;
        part += a * p;
    }
    part = group_sum<32>(part);
    __syncthreads();
    if (lane == 0) s_part[warp] = part;
    __syncthreads();
    if (warp == 0) {
        part = group_sum<32>(lane < kWarps ? s_part[lane] : 0.0f);
        if (lane == 0) remote_store(&s_parts[blockIdx.x], 0, part);
    }
    __syncthreads();
    cluster_sync_all();                        // nobody leaves while its shared memory may be read
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        float balance = 0.0f;
        for (int b = 0; b < kCluster; ++b) balance += s_parts[b];
        write_losses(g, balance, z, rows, rows > 0);
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
    int T, E, K, S, sigmoid, rows_per_block;
    int chunk, coef_chunk;         // see chunk_of: for the logits and their gradient, and for coef
};

// Bound by DRAM at large sizes: reads T E logits, writes T E gradients.  With c = gb (a - sum p a) + gz lse the softmax row's
// gradient is p c: two operations a value once the sums are there.  The gradient of the chosen weights is scattered into a row
// of shared memory, K values, and picked up by the lanes that hold their experts.
template <typename T, int kLanes, int V, bool kSigmoid>
__global__ void __launch_bounds__(kBwdThreads, bwd_blocks_per_sm(V, kSigmoid)) balance_bwd_kernel(const BalanceBwdParams g) {
    constexpr int kGroups = kBwdThreads / kLanes;
    constexpr int kPer = (kLanes * V < 32 ? kLanes * V : 32) / kLanes;          // routes a lane, at most (topk <= 32 and <= E)
    using Row = SharedRow<kLanes, V>;
    __shared__ alignas(16) float s_add[kGroups][Row::kFloats];
    const int lane = threadIdx.x & 31, l = lane % kLanes, group = threadIdx.x / kLanes;
    float* const add = s_add[group];
#pragma unroll
    for (int j = 0; j < V; j += 4) *reinterpret_cast<float4*>(add + Row::chunk(l, j)) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    pdl_wait();
    const size_t scalars = static_cast<size_t>(g.S) * g.E;
    const float gb = g.d_losses[0] * g.coef[scalars], gz = g.d_losses[1] * g.coef[scalars + 1];
    const bool losses = gb != 0.0f || gz != 0.0f;      // without an upstream gradient the row is not read for them
    const long long first = static_cast<long long>(blockIdx.x) * g.rows_per_block;
    const int lo = static_cast<int>(min(first, static_cast<long long>(g.T)));
    const int hi = static_cast<int>(min(first + g.rows_per_block, static_cast<long long>(g.T)));
    int s = first_sequence(g.offsets, g.S, lo, g.T), held = -1;
    float a[V];                                        // gb times the sequence's f / n
#pragma unroll
    for (int j = 0; j < V; ++j) a[j] = 0.0f;
    __syncwarp();
    for (int t0 = lo + (threadIdx.x >> 5) * (32 / kLanes); t0 < hi; t0 += kGroups) {
        const int t = t0 + lane / kLanes;
        const bool there = t < hi;
        const T* const row = static_cast<const T*>(g.logits) + static_cast<size_t>(there ? t : t0) * g.E;
        float d[V], v[V];
        if (losses) load_row<kLanes, V>(row, l, g.E, g.chunk, -INFINITY, v);
        int expert[kPer];
        float w[kPer], dw[kPer];
        if (g.top != nullptr) {
            const size_t o = static_cast<size_t>(t) * g.K + l;
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const bool mine = there && l + i * kLanes < g.K;
                const long long e = mine ? g.top[o + i * kLanes] : -1;
                w[i] = mine ? g.weights[o + i * kLanes] : 0.0f;
                dw[i] = mine ? g.d_weights[o + i * kLanes] : 0.0f;
                expert[i] = e >= 0 && e < g.E ? static_cast<int>(e) : -1;
            }
        }
        bool live = there && losses && (g.mask == nullptr || g.mask[t]);
        if (g.offsets != nullptr && there) {
            while (s < g.S && seq_bound(g.offsets, s + 1, g.T) <= t) ++s;
            live = live && s < g.S && seq_bound(g.offsets, s, g.T) <= t;
        }
        if (live && s != held) {
            load_row<kLanes, V>(g.coef + static_cast<size_t>(s) * g.E, l, g.E, g.coef_chunk, 0.0f, a);
#pragma unroll
            for (int j = 0; j < V; ++j) a[j] *= gb;
            held = s;
        }
        if (kLanes == 32 ? live : losses) {            // shorter groups of a warp stay in step
            float ex[V], sg[V];
            const RowStats r = row_stats<kLanes, V, kSigmoid>(v, row_max<kLanes, V>(v), ex, sg);
            float dot = 0.0f;
#pragma unroll
            for (int j = 0; j < V; ++j) dot = fmaf(kSigmoid ? sg[j] : ex[j], a[j], dot);
            dot = group_sum<kLanes>(dot);
            if constexpr (kSigmoid) {
                dot *= r.inv_sg;
                const float zs = gz * r.lse * r.inv;
#pragma unroll
                for (int j = 0; j < V; ++j) d[j] = fmaf(sg[j] * r.inv_sg * sigmoid_rest(v[j]), a[j] - dot, ex[j] * zs);
            } else {
                const float c = (gz * r.lse - dot * r.inv) * r.inv;
#pragma unroll
                for (int j = 0; j < V; ++j) d[j] = ex[j] * fmaf(a[j], r.inv, c);
            }
            if constexpr (kLanes != 32) {
#pragma unroll
                for (int j = 0; j < V; ++j) d[j] = live ? d[j] : 0.0f;
            }
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) d[j] = 0.0f;
        }
        if (g.top != nullptr) {
            float dot = 0.0f;
#pragma unroll
            for (int i = 0; i < kPer; ++i) dot = fmaf(w[i], dw[i], dot);
            dot = group_sum<kLanes>(dot);
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                dw[i] = w[i] == 0.0f ? 0.0f : w[i] * (dw[i] - dot);
                if (kSigmoid && expert[i] >= 0) dw[i] *= sigmoid_rest(to_float(row[expert[i]]));
                if (expert[i] >= 0) {
                    expert[i] = Row::at(expert[i]);                // from here on its place in the shared row
                    add[expert[i]] = __int_as_float(l + i * kLanes);
                }
            }
            // an expert that a row names twice (finished routes may) shows in the tag that was overwritten
            bool twice = false;
            __syncwarp();
#pragma unroll
            for (int i = 0; i < kPer; ++i) twice |= expert[i] >= 0 && __float_as_int(add[expert[i]]) != l + i * kLanes;
            if (__any_sync(kAll, twice)) {
#pragma unroll
                for (int i = 0; i < kPer; ++i) if (expert[i] >= 0) add[expert[i]] = 0.0f;
#pragma unroll
                for (int i = 0; i < kPer; ++i)
                    for (int who = 0; who < kLanes; ++who) {       // one at a time, in order
                        __syncwarp();
                        if (l == who && expert[i] >= 0) add[expert[i]] += dw[i];
                    }
            } else {
                __syncwarp();
#pragma unroll
                for (int i = 0; i < kPer; ++i) if (expert[i] >= 0) add[expert[i]] = dw[i];
            }
            __syncwarp();
#pragma unroll
            for (int j = 0; j < V; j += 4) {
                const float4 x = *reinterpret_cast<const float4*>(add + Row::chunk(l, j));
                d[j] += x.x; d[j + 1] += x.y; d[j + 2] += x.z; d[j + 3] += x.w;
            }
            __syncwarp();
#pragma unroll
            for (int i = 0; i < kPer; ++i) if (expert[i] >= 0) add[expert[i]] = 0.0f;
            __syncwarp();
        }
        if (there) store_row<kLanes, V>(static_cast<T*>(g.d_logits) + static_cast<size_t>(t) * g.E, l, g.E, g.chunk, d);
    }
}

constexpr int kCountThreads = 512, kCountBins = 8192;
struct CountParams {
    const void* top;
    int ids_i32;
    const uint8_t* mask;
    const int* offsets;
    int* counts;                   // [S, E], zeroed before a launch of several blocks
    int T, E, K, S, rows_per_block;
    int bins;                      // in shared memory, E at least
};

// Each block counts a run of rows in shared memory, as many sequences at a time as the bins hold, and adds what it found:
// integer sums do not depend on their order.  One block alone has bins for all and stores them.  Reads T K ids.
__global__ void __launch_bounds__(kCountThreads) expert_counts_kernel(const CountParams g) {
    extern __shared__ int bins[];
    pdl_wait();
    const bool alone = gridDim.x == 1;
    const long long first = static_cast<long long>(blockIdx.x) * g.rows_per_block;
    int pos = static_cast<int>(min(first, static_cast<long long>(g.T)));
    const int hi = static_cast<int>(min(first + g.rows_per_block, static_cast<long long>(g.T)));
    const unsigned topk = g.K;
    int s = alone ? 0 : first_sequence(g.offsets, g.S, pos, g.T);
    const int last = alone ? g.S : min(first_sequence(g.offsets, g.S, hi - 1, g.T) + 1, g.S);       // behind the run's sequences
    auto count = [&](size_t at, int* to) {
        const long long e = g.ids_i32 ? static_cast<const int*>(g.top)[at] : static_cast<const long long*>(g.top)[at];
        if (e >= 0 && e < g.E) atomicAdd(to + e, 1);
    };
    while (s < last) {
        const int stop = min(last, s + g.bins / g.E);
        const int begin = max(seq_bound(g.offsets, s, g.T), pos), end = min(seq_bound(g.offsets, stop, g.T), hi);
        for (int e = threadIdx.x; e < (stop - s) * g.E; e += kCountThreads) bins[e] = 0;
        __syncthreads();
        if (stop - s == 1 && end > begin) {
            const size_t at = static_cast<size_t>(begin) * topk;
            const unsigned n = static_cast<unsigned>(end - begin) * topk;          // a call has fewer than 2^31 routes
#pragma unroll 4
            for (unsigned i = threadIdx.x; i < n; i += kCountThreads)
                if (g.mask == nullptr || g.mask[begin + i / topk]) count(at + i, bins);
        } else {
            for (int t = begin + threadIdx.x; t < end; t += kCountThreads) {
                if (g.mask != nullptr && !g.mask[t]) continue;
                int lo = s, up = stop;                     // the last sequence that starts at or before the row
                while (up - lo > 1) { const int mid = (lo + up) >> 1; if (seq_bound(g.offsets, mid, g.T) <= t) lo = mid; else up = mid; }
                const size_t at = static_cast<size_t>(t) * topk;
#pragma unroll 4
                for (unsigned k = 0; k < topk; ++k) count(at + k, bins + (lo - s) * g.E);
            }
        }
        __syncthreads();
        int* const out = g.counts + static_cast<size_t>(s) * g.E;
        for (int e = threadIdx.x; e < (stop - s) * g.E; e += kCountThreads) {
            if (alone) out[e] = bins[e];
            else if (bins[e]) atomicAdd(out + e, bins[e]);
        }
        __syncthreads();
        pos = max(pos, end);
        s = stop;
    }
}

template <typename T, int kLanes, int V, bool kSigmoid, int kChoose>
int launch_rows(const BalanceParams& p, cudaStream_t s) {
    const size_t chosen = kChoose != kNone ? static_cast<size_t>(2) * (kRowThreads / kLanes) * p.K : 0;
    const size_t smem = (static_cast<size_t>(kSumRows) * SharedRow<kLanes, V>::kFloats + ((p.E + 1) & ~1) + chosen) * 4;
    if (!p.one_launch) return launch_kernel(balance_rows_kernel<T, kLanes, V, kSigmoid, kChoose>, p.blocks, kRowThreads, smem, s, false, true, p);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(kCluster);
    cfg.blockDim = dim3(kRowThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2] = {};
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = kCluster; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    auto* kern = balance_rows_kernel<T, kLanes, V, kSigmoid, kChoose>;
    MOK_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, p));
    return MOK_OK;
}

template <typename T, int kLanes, int V, bool kSigmoid>
int launch_choice(const BalanceParams& p, cudaStream_t s) {
    if (p.top_in != nullptr) return launch_rows<T, kLanes, V, kSigmoid, kNone>(p, s);
    if constexpr (kLanes == 32) if (p.K > 16) return launch_rows<T, kLanes, V, kSigmoid, kMany>(p, s);
    return launch_rows<T, kLanes, V, kSigmoid, kFew>(p, s);
}
template <typename T, int kLanes, int V>
int launch_rows_as(const BalanceParams& p, cudaStream_t s) {
    return p.sigmoid ? launch_choice<T, kLanes, V, true>(p, s) : launch_choice<T, kLanes, V, false>(p, s);
}

template <typename T, int kLanes, int V, bool kSigmoid>
int launch_bwd(BalanceBwdParams p, cudaStream_t s) {
    constexpr int kGroups = kBwdThreads / kLanes;
    const int blocks = std::min((p.T + kGroups - 1) / kGroups, device_sm_count() * bwd_blocks_per_sm(V, kSigmoid) * 2);
    p.rows_per_block = (p.T + blocks - 1) / blocks;
    return launch_kernel(balance_bwd_kernel<T, kLanes, V, kSigmoid>, blocks, kBwdThreads, 0, s, false, true, p);
}

// lanes a row and values a lane: four values where a row fits, so that 32 lanes hold several short rows
#define MOK_ROW_SHAPE(E, call)                                                                   \
    [&] {                                                                                        \
        if ((E) <= 16) return call(4, 4);                                                        \
        if ((E) <= 32) return call(8, 4);                                                        \
        if ((E) <= 64) return call(16, 4);                                                       \
        if ((E) <= 128) return call(32, 4);                                                      \
        if ((E) <= 256) return call(32, 8);                                                      \
        if ((E) <= 512) return call(32, 16);                                                     \
        return call(32, 32);                                                                     \
    }()

bool bad_sizes(int T, int E, int K, int S) { return T <= 0 || E <= 0 || K <= 0 || K > 255 || S <= 0; }
// counts are 32-bit, and a row index and a block's rows have to fit an int together
bool too_many_routes(int T, int K) { return T > 0x7fff0000 || static_cast<long long>(T) * K > 0x7fffffffll; }

}  // namespace
}  // namespace mok

using namespace mok;

extern "C" size_t mok_router_balance_scratch_bytes(int num_tokens, int num_experts, int num_sequences) {
    if (bad_sizes(num_tokens, num_experts, 1, num_sequences)) return 0;
    if (in_one_launch(num_tokens, num_experts, num_sequences)) return 0;
    return Scratch(nullptr, row_blocks(num_tokens, num_experts, num_sequences) + num_sequences, num_experts, num_sequences).bytes;
}

extern "C" int mok_router_balance(const mok_router_balance_args* args, void* stream) {
    if (!args) return MOK_ERR_INVALID;
    const mok_router_balance_args& a = *args;
    const int T = a.num_tokens, E = a.num_experts, K = a.topk, S = a.num_sequences;
    if (!a.logits || !a.losses || !a.counts || !a.coef || bad_sizes(T, E, K, S)) return MOK_ERR_INVALID;
    if (a.top_experts_in ? (a.top_experts_out || a.router_weights) : (!a.top_experts_out || !a.router_weights)) return MOK_ERR_INVALID;
    if (!a.top_experts_in && (K > 32 || K > E)) return MOK_ERR_INVALID;
    if (!a.sequence_offsets && S != 1) return MOK_ERR_INVALID;
    if (E > 1024) return MOK_ERR_UNSUPPORTED;
    if (too_many_routes(T, K) || static_cast<long long>(S) * E > 0x7fffffff) return MOK_ERR_TOO_LARGE;
    BalanceParams p{};
    p.blocks = row_blocks(T, E, S);
    p.one_launch = in_one_launch(T, E, S);
    const Scratch at(a.scratch, p.blocks + S, E, S);
    if (!p.one_launch && (!a.scratch || a.scratch_bytes < at.bytes || reinterpret_cast<uintptr_t>(a.scratch) % 16)) return MOK_ERR_INVALID;
    p.logits = a.logits;
    p.top_in = reinterpret_cast<const long long*>(a.top_experts_in);
    p.top_out = reinterpret_cast<long long*>(a.top_experts_out);
    p.weights = a.router_weights;
    p.mask = a.token_mask;
    p.offsets = a.sequence_offsets;
    p.load = a.load;
    p.losses = a.losses;
    p.counts = a.counts;
    p.coef = a.coef;
    p.T = T; p.E = E; p.K = K; p.S = S;
    p.rows_per_block = rows_per_block(T, E, S);
    p.sigmoid = a.sigmoid;
    p.chunk = chunk_of(a.logits, E, a.logits_bf16 ? 2 : 4);
    p.head = at.head; p.slot_p = at.p; p.slot_routes = at.routes; p.part = at.part; p.seq_z = at.seq_z; p.seq_rows = at.seq_rows;
    p.ticket = at.ticket;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    ProfScope prof(kSlotOther, s, p.one_launch ? 1 : 2);
    int rc;
    if (a.logits_bf16) {
#define MOK_CALL(lanes, v) launch_rows_as<__nv_bfloat16, lanes, v>(p, s)
        rc = MOK_ROW_SHAPE(E, MOK_CALL);
#undef MOK_CALL
    } else {
#define MOK_CALL(lanes, v) launch_rows_as<float, lanes, v>(p, s)
        rc = MOK_ROW_SHAPE(E, MOK_CALL);
#undef MOK_CALL
    }
    if (rc != MOK_OK || p.one_launch) return rc;
    // few sequences: narrow tiles and many warps, each sequence has many slots; many: wide tiles, few slots each
    if (S <= 4) return launch_kernel(balance_join_kernel<8, 32>, S * ((E + 7) / 8), 1024, 0, s, false, true, p);
    return launch_kernel(balance_join_kernel<32, 8>, S * ((E + 31) / 32), 256, 0, s, false, true, p);
}

extern "C" int mok_router_balance_bwd(const mok_router_balance_bwd_args* args, void* stream) {
    if (!args) return MOK_ERR_INVALID;
    const mok_router_balance_bwd_args& a = *args;
    const int T = a.num_tokens, E = a.num_experts, K = a.topk, S = a.num_sequences, bytes = a.logits_bf16 ? 2 : 4;
    if (!a.d_losses || !a.logits || !a.coef || !a.d_logits || bad_sizes(T, E, K, S)) return MOK_ERR_INVALID;
    const int with = (a.top_experts != nullptr) + (a.router_weights != nullptr) + (a.d_router_weights != nullptr);
    if (with != 0 && (with != 3 || K > 32 || K > E)) return MOK_ERR_INVALID;
    if (!a.sequence_offsets && S != 1) return MOK_ERR_INVALID;
    if (E > 1024) return MOK_ERR_UNSUPPORTED;
    if (T > 0x7fff0000 || static_cast<long long>(S) * E > 0x7fffffffll) return MOK_ERR_TOO_LARGE;
    BalanceBwdParams p{a.d_losses, a.logits, a.coef, a.token_mask, a.sequence_offsets, reinterpret_cast<const long long*>(a.top_experts),
                       a.router_weights, a.d_router_weights, a.d_logits, T, E, K, S, a.sigmoid, 0,
                       std::min(chunk_of(a.logits, E, bytes), chunk_of(a.d_logits, E, bytes)), chunk_of(a.coef, E, 4)};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    ProfScope prof(kSlotOther, s);
    if (a.logits_bf16) {
#define MOK_CALL(lanes, v) (p.sigmoid ? launch_bwd<__nv_bfloat16, lanes, v, true>(p, s) : launch_bwd<__nv_bfloat16, lanes, v, false>(p, s))
        return MOK_ROW_SHAPE(E, MOK_CALL);
#undef MOK_CALL
    }
#define MOK_CALL(lanes, v) (p.sigmoid ? launch_bwd<float, lanes, v, true>(p, s) : launch_bwd<float, lanes, v, false>(p, s))
    return MOK_ROW_SHAPE(E, MOK_CALL);
#undef MOK_CALL
}

extern "C" int mok_expert_counts(const void* top_experts, int ids_i32, int num_tokens, int topk, int num_experts, int num_sequences,
                                 const uint8_t* token_mask, const int32_t* sequence_offsets, int32_t* counts, void* stream) {
    if (!top_experts || !counts || bad_sizes(num_tokens, num_experts, topk, num_sequences)) return MOK_ERR_INVALID;
    if (!sequence_offsets && num_sequences != 1) return MOK_ERR_INVALID;
    if (num_experts > 1024) return MOK_ERR_UNSUPPORTED;
    if (too_many_routes(num_tokens, topk)) return MOK_ERR_TOO_LARGE;
    const long long routes = static_cast<long long>(num_tokens) * topk;
    // one block, which needs no cleared counts, takes 8192 routes in the time that clearing them takes
    const long long bins = static_cast<long long>(num_sequences) * num_experts;
    const bool alone = routes <= 8192 && bins <= kCountBins;
    const int blocks = alone ? 1 : static_cast<int>(std::min<long long>((routes + 4095) / 4096, device_sm_count() * 4));
    CountParams p{top_experts, ids_i32, token_mask, sequence_offsets, counts, num_tokens, num_experts, topk, num_sequences,
                  (num_tokens + blocks - 1) / blocks, static_cast<int>(std::min<long long>(bins, kCountBins))};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    ProfScope prof(kSlotOther, s);
    if (!alone) MOK_CUDA_CHECK(cudaMemsetAsync(counts, 0, static_cast<size_t>(num_sequences) * num_experts * 4, s));
    return launch_kernel(expert_counts_kernel, blocks, kCountThreads, static_cast<size_t>(p.bins) * 4, s, false, alone, p);
}
