// The routing losses' join, the expert counts and the C entries of both: see balance.cuh for the mathematics.
#include <algorithm>

#include "balance.cuh"
#include "profile.cuh"

namespace mok {
namespace balance {
namespace {

constexpr int kMinCols = 8;                    // fewest experts of a join tile

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
// blocks and one that joins their slots.  The limit is in rows a group of lanes, where the device's times meet; the cluster also saves
// the caller a launch and an allocation, 4 us of its time.  One B200, us, cluster and two launches, choosing K = 2 to 8 / with
// finished routes: 8 experts 1 row 5.4 and 6.7 / 5.0 and 7.4, 3 rows 7.3 and 6.7 / 5.9 and 7.5, 6 rows 10.1 and 7.3 / 7.0 and 7.0; 128 experts
// 3 rows 8.3 and 8.5 / 5.7 and 7.3, 6 rows 11.8 and 8.6 / 6.9 and 7.4; 1000 experts 1 row 10.4 and 11.7 / 7.8 and 8.9, 2 rows 13.9 and 11.8 / 8.7 and 9.1.
bool in_one_launch(int T, int E, int S, bool choose) {
    const int rows = E > 512 ? (choose ? 1 : 2) : (choose ? 3 : 6);
    return S == 1 && T <= rows * kCluster * rows_at_once(E);
}
int rows_per_block(int T, int E, int S, bool choose) {
    const int most = in_one_launch(T, E, S, choose) ? kCluster : 148 * row_blocks_per_sm(E), at_once = rows_at_once(E);
    const int rows = (T + most - 1) / most;
    return (rows + at_once - 1) / at_once * at_once;
}
int row_blocks(int T, int E, int S, bool choose) {
    if (in_one_launch(T, E, S, choose)) return kCluster;
    const int rows = rows_per_block(T, E, S, choose);
    return (T + rows - 1) / rows;
}

// how rows of E values of `bytes` bytes at `base` can be read: chunks of eight (16 or 32 bytes), of four, or one by one
int chunk_of(const void* base, int E, int bytes) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(base);
    if (E % 8 == 0 && at % (8 * bytes) == 0) return 8;
    return E % 4 == 0 && at % (4 * bytes) == 0 ? 4 : 1;
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

bool bad_sizes(int T, int E, int K, int S) { return T <= 0 || E <= 0 || K <= 0 || K > 255 || S <= 0; }
// counts are 32-bit, and a row index and a block's rows have to fit an int together
bool too_many_routes(int T, int K) { return T > 0x7fff0000 || static_cast<long long>(T) * K > 0x7fffffffll; }

}  // namespace
}  // namespace balance
}  // namespace mok

using namespace mok;
using namespace mok::balance;

extern "C" size_t mok_router_balance_scratch_bytes(int num_tokens, int num_experts, int num_sequences, int chooses) {
    if (bad_sizes(num_tokens, num_experts, 1, num_sequences)) return 0;
    if (in_one_launch(num_tokens, num_experts, num_sequences, chooses != 0)) return 0;
    return Scratch(nullptr, row_blocks(num_tokens, num_experts, num_sequences, chooses != 0) + num_sequences, num_experts, num_sequences).bytes;
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
    const bool choose = a.top_experts_in == nullptr;
    p.blocks = row_blocks(T, E, S, choose);
    p.one_launch = in_one_launch(T, E, S, choose);
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
    p.rows_per_block = rows_per_block(T, E, S, choose);
    p.sigmoid = a.sigmoid;
    p.chunk = chunk_of(a.logits, E, a.logits_bf16 ? 2 : 4);
    p.head = at.head; p.slot_p = at.p; p.slot_routes = at.routes; p.part = at.part; p.seq_z = at.seq_z; p.seq_rows = at.seq_rows;
    p.ticket = at.ticket;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    ProfScope prof(kSlotOther, s, p.one_launch ? 1 : 2);
    const int rc = a.logits_bf16 ? rows_bf16(p, s) : rows_f32(p, s);
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
    return a.logits_bf16 ? backward_bf16(p, s) : backward_f32(p, s);
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
