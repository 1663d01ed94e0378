// The kernels of the routing losses that work on rows of logits, and their launches: see balance.cuh.
#pragma once

#include <algorithm>

#include "balance.cuh"

namespace mok {
namespace balance {

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
// In rounds, one row a warp: every lane keeps the two largest values it has left; a round is one maximum over the warp, the winner
// moves its second up, and a lane that has used up both looks through its values again (with K = 8 of 256 in half of the rows; one
// kept value would mean a search in every round).
template <int V>
__device__ __forceinline__ void select_in_rounds(const float (&v)[V], int E, int K, float2* chosen) {
    using At = Held<32, V>;
    const int lane = threadIdx.x & 31;
    const unsigned below = (1u << lane) - 1u;
    const int mine = At::count(lane, E);
    unsigned taken = 0;
    float b1, b2;
    int j1, j2;
    two_largest(v, 0u, b1, j1, b2, j2);
    for (int k = 0; k < K; ++k) {
        const float best = group_max<32>(b1);
        const bool equal = j1 < V && b1 == best;
        const unsigned at = __ballot_sync(kAll, equal);
        bool win = equal && (at & below) == 0;
        if (V > At::kUnit && (at & (at - 1)) != 0) {               // equals in several lanes, whose experts interleave
            const int e = equal ? At::expert(lane, j1) : 0x7fffffff;
            win = e == __reduce_min_sync(kAll, e) && equal;
        }
        if (win) chosen[k] = make_float2(best, __int_as_float(At::expert(lane, j1)));
        taken |= win ? 1u << (j1 & 31) : 0u;
        const bool dry = win && j2 == V;
        b1 = win ? b2 : b1;
        j1 = win ? j2 : j1;
        b2 = win ? -INFINITY : b2;
        j2 = win ? V : j2;
        if (at == 0) {                                             // nothing above -inf left: the lowest expert not taken yet
            const unsigned left = ~taken & (V == 32 && mine == 32 ? kAll : (1u << mine) - 1u);
            const int e = left ? At::expert(lane, __ffs(left) - 1) : 0x7fffffff;
            if (e == __reduce_min_sync(kAll, e) && left) { chosen[k] = make_float2(-INFINITY, __int_as_float(e)); taken |= left & (0u - left); }
        }
        if (__any_sync(kAll, dry)) { if (dry) two_largest(v, taken, b1, j1, b2, j2); }
    }
    __syncwarp();
}

// In rounds with four values a lane: they are sorted once, and the winner moves the rest up.  (131072 rows of 60 experts,
// forward: K = 8 55 us with the two largest kept, 39 so; K = 16 98 and 54.)
template <int kLanes>
__device__ __forceinline__ void select_sorted(const float (&v)[4], int E, int K, float2* chosen) {
    const int lane = threadIdx.x & 31, l = lane % kLanes;
    const unsigned group = kLanes == 32 ? kAll : ((1u << kLanes) - 1u) << (lane - l);
    const unsigned below = (1u << lane) - 1u;
    float b[4];
    unsigned order = 0x03020100u;                                  // a byte each: whose value it is
#pragma unroll
    for (int j = 0; j < 4; ++j) b[j] = fmaxf(v[j], -INFINITY);     // a NaN ranks with -inf
#pragma unroll
    for (int last = 3; last > 0; --last) {
#pragma unroll
        for (int j = 0; j < last; ++j) {                           // neighbours, and only if the right one is larger: equals stay in order
            const bool swap = b[j + 1] > b[j];
            const float larger = swap ? b[j + 1] : b[j];
            b[j + 1] = swap ? b[j] : b[j + 1];
            b[j] = larger;
            order = swap ? __byte_perm(order, 0u, j == 0 ? 0x3201u : j == 1 ? 0x3120u : 0x2310u) : order;
        }
    }
    int left = Held<kLanes, 4>::count(l, E);                       // values past E come last
    for (int k = 0; k < K; ++k) {
        const float best = group_max<kLanes>(b[0]);
        const bool equal = left > 0 && b[0] == best;
        const unsigned at = __ballot_sync(kAll, equal) & group;
        const bool win = equal && (at & below) == 0;               // the lowest lane holds the lowest expert
        if (win) chosen[k] = make_float2(best, __int_as_float(l * 4 + static_cast<int>(order & 3u)));
        b[0] = win ? b[1] : b[0];
        b[1] = win ? b[2] : b[1];
        b[2] = win ? b[3] : b[2];
        b[3] = win ? -INFINITY : b[3];
        order = win ? order >> 8 : order;
        left -= win;
    }
    __syncwarp();
}

template <int kLanes, int V>
__device__ __forceinline__ void rounds(const float (&v)[V], int E, int K, float2* chosen) {
    if constexpr (V == 4) select_sorted<kLanes>(v, E, K, chosen);
    else select_in_rounds<V>(v, E, K, chosen);                     // rows of more than four values a lane have a warp each
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
        if (n > 32) { rounds<32, V>(v, E, K, chosen); return; }
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
    if (above < K) { rounds<32, V>(v, E, K, chosen); return; }
    for (int from = 0; from < K; from += 16) {
        const int some = min(K - from, 16);
        select_by_rank<V>(v, E, some, set_of<V>(E, some), gathered, chosen + from);
        const float2 last = chosen[from + some - 1];
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (v[j] > last.x || (v[j] == last.x && Held<32, V>::expert(lane, j) <= __float_as_int(last.y))) v[j] = -INFINITY;
    }
}

// Bound by instructions and, without the choice, by the latency of its loads.  Reads T E logits once, writes K routes a row and (p,
// routes) per slot.  One B200 with the join, us, inputs not in the cache (floor: bytes at 6456 GB/s): 131072 x 256 f32, K = 8: 71 (23),
// finished routes 35; 65536 x 500 bf16, K = 6, 61 sequences: 69 (11) and 35; 16384 x 128: 15 (1.5) and 12; 30000 x 1024 f32, K = 8: 49 (19) and
// 30.  Sigmoid scores 131072 x 256: 92, 65536 x 500 bf16 without sequences: 85 against 62.  With the choice of 1024 and 512 experts and of
// more than 16 routes the registers do not suffice: 4 to 140 bytes are spilled.  A row of 256 takes 470 instructions
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
    __shared__ alignas(16) uint2 s_gathered[kChoose >= kRank ? kWarps : 1][32];
    __shared__ float s_z[kWarps], s_part[kWarps], s_parts[kCluster];
    __shared__ int s_rows[kWarps], s_routes;
    int* const hist = reinterpret_cast<int*>(smem + kSumRows * Row::kFloats);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, l = lane % kLanes, group = threadIdx.x / kLanes;
    float2* const chosen = reinterpret_cast<float2*>(hist + ((g.E + 1) & ~1)) + static_cast<size_t>(group) * g.K;
    pdl_wait();
    if (blockIdx.x == 0 && threadIdx.x == 0 && !g.one_launch) *g.ticket = 0;
    const int set = kChoose == kRank ? set_of<V>(g.E, g.K) : 0;
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
                if constexpr (kChoose == kRounds) {
                    rounds<kLanes, V>(v, g.E, g.K, chosen);
                } else if constexpr (kChoose == kRank) {
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
                float slope = w[i] * (dw[i] - dot);
                if (kSigmoid && expert[i] >= 0) slope *= sigmoid_rest(to_float(row[expert[i]]));
                dw[i] = w[i] == 0.0f ? 0.0f : slope;       // last: a route of weight 0 takes nothing, its logit may be NaN
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
    // Rows that share a warp cannot choose by rank.  Sorted rounds cost every route the same, ranks little for one more: 131072 x
    // 128, forward, rounds and rank: K = 1 39 and 51 us, 4 48 and 55, 8 59 and 60, 16 80 and 71.
    // Rows of 256 lose from four routes on, with three kept values a lane: K = 1 57 and 64, 2 62 and 64, 4 73 and 67, 8 93 and 73.  What
    // that wins at one and two routes was not thought worth four kernels more.
    if constexpr (kLanes < 32) {
        return launch_rows<T, kLanes, V, kSigmoid, kRounds>(p, s);
    } else {
        if (p.K > 16) return launch_rows<T, kLanes, V, kSigmoid, kMany>(p, s);
        if constexpr (V == 4) if (p.K <= 8) return launch_rows<T, kLanes, V, kSigmoid, kRounds>(p, s);
        return launch_rows<T, kLanes, V, kSigmoid, kRank>(p, s);
    }
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

template <typename T>
int launch_rows_for(const BalanceParams& p, cudaStream_t s) {
#define MOK_CALL(lanes, v) launch_rows_as<T, lanes, v>(p, s)
    return MOK_ROW_SHAPE(p.E, MOK_CALL);
#undef MOK_CALL
}
template <typename T>
int launch_bwd_for(const BalanceBwdParams& p, cudaStream_t s) {
#define MOK_CALL(lanes, v) (p.sigmoid ? launch_bwd<T, lanes, v, true>(p, s) : launch_bwd<T, lanes, v, false>(p, s))
    return MOK_ROW_SHAPE(p.E, MOK_CALL);
#undef MOK_CALL
}

}  // namespace balance
}  // namespace mok
