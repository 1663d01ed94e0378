// Dropout from a counter-based generator, with the residual added in the same pass; no mask is stored.
//
//   out_i = residual_i + (u_i >= threshold ? x_i * 65536 / (65536 - threshold) : 0),   threshold = round(65536 p)
// u_i is a 16-bit number that depends on the seed and on i alone, so the backward pass (the same kernel on d_out without
// a residual) draws it again.  A dropped element is exactly 0, whatever x holds.
//
// Generator: Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011), key =
// the seed's two words, counter = (i >> 3 as two words, 0, 0).  Its four words give eight 16-bit numbers, low half
// first.  The drop probability is therefore p rounded to a multiple of 2^-16, and the factor is that of the rounded
// probability, so the expectation is kept exactly.
#include <algorithm>

#include "common.cuh"
#include "profile.cuh"

namespace mok {
namespace {

constexpr int kDropThreads = 64;

// Groups of eight elements that a thread has in flight, and blocks that an SM has to be able to hold (which bounds the
// registers).  The kernel moves bytes and, in bf16, draws numbers nearly as long as it moves them, so it needs many loads in
// flight and few warps to issue them from; with more resident warps DRAM gets slower again.  One B200, us, groups and blocks
// (floor: bytes at the measured copy rate of 6456 GB/s), without dependent launches, which take 2 us more off:
//   16384 x 7168 bf16 with a residual (109):  6, 10: 106;  5, 10: 108;  6, 12: 112;  256 threads: 112 to 130
//   the same without one (73):                7, 12: 75.5;  8, 12: 77;  6, 12: 80;  5, 10: 89;  256 threads: 83 to 105
//   10000 x 2042 f32 (38.0 and 25.3):         2, 8: 38.7 and 27.4;  3, 12: 39.7 and 27.4;  4, 10: 41.7 and 27.4
// Inputs are read past the cache (they are not needed again), the result is not: whoever reads it next finds part of it there.
// With an elementwise kernel behind it, 16384 x 2048 bf16: 57.6 us with both past the cache, 55 so, 56 with neither.
template <typename T, bool kResidual> struct Shape {
    static constexpr int kUnroll = sizeof(T) == 4 ? 2 : kResidual ? 6 : 7;
    static constexpr int kBlocks = sizeof(T) == 4 ? 8 : kResidual ? 10 : 12;
};

struct DropoutParams {
    const void* x;
    const void* residual;          // may be null
    const long long* seed;
    void* out;
    long long count;
    unsigned threshold;            // 0 .. 65535
    float scale;
};

__device__ __forceinline__ uint4 philox(unsigned long long block, unsigned k0, unsigned k1) {
    uint4 c = make_uint4(static_cast<unsigned>(block), static_cast<unsigned>(block >> 32), 0u, 0u);
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const unsigned long long a = 0xD2511F53ull * c.x, b = 0xCD9E8D57ull * c.z;
        c = make_uint4(static_cast<unsigned>(b >> 32) ^ c.y ^ k0, static_cast<unsigned>(b),
                       static_cast<unsigned>(a >> 32) ^ c.w ^ k1, static_cast<unsigned>(a));
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return c;
}

__device__ __forceinline__ float drop_load(const float* p) { return *p; }
__device__ __forceinline__ float drop_load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void drop_store(float* p, float v) { *p = v; }
__device__ __forceinline__ void drop_store(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// eight elements of 16-byte aligned memory
template <typename T> struct Eight;
template <> struct Eight<__nv_bfloat16> {
    uint4 v;
    __device__ __forceinline__ void load(const __nv_bfloat16* p) { v = __ldcs(reinterpret_cast<const uint4*>(p)); }
    __device__ __forceinline__ void get(float (&f)[8]) const {
        const unsigned w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) { const float2 t = unpack_bf16(w[i]); f[2 * i] = t.x; f[2 * i + 1] = t.y; }
    }
    static __device__ __forceinline__ void store(__nv_bfloat16* p, const float (&f)[8]) {
        *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
    }
};
template <> struct Eight<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const float* p) {
        a = __ldcs(reinterpret_cast<const float4*>(p));
        b = __ldcs(reinterpret_cast<const float4*>(p) + 1);
    }
    __device__ __forceinline__ void get(float (&f)[8]) const {
        f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
    }
    static __device__ __forceinline__ void store(float* p, const float (&f)[8]) {
        *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
    }
};

// Bound by DRAM: reads x (and the residual), writes out, once each.  kAligned: every pointer is on a 16-byte boundary and
// groups of eight go through 128-bit accesses; otherwise, and for the last count % 8 elements, element by element.
template <typename T, bool kResidual, bool kAligned>
__global__ void __launch_bounds__(kDropThreads, Shape<T, kResidual>::kBlocks) dropout_kernel(const DropoutParams g) {
    constexpr int kUnroll = Shape<T, kResidual>::kUnroll;
    pdl_wait();
    const T* const x = static_cast<const T*>(g.x);
    const T* const res = static_cast<const T*>(g.residual);
    T* const out = static_cast<T*>(g.out);
    const unsigned long long seed = static_cast<unsigned long long>(*g.seed);
    // every lane has the same key; as results of a warp-wide reduction the compiler knows it, and keeps the key schedule out
    // of the lanes' arithmetic (16384 x 7168 bf16 without a residual, 256 threads: 84.8 -> 80.7 us)
    const unsigned k0 = __reduce_or_sync(0xffffffffu, static_cast<unsigned>(seed));
    const unsigned k1 = __reduce_or_sync(0xffffffffu, static_cast<unsigned>(seed >> 32));
    const long long groups = (g.count + 7) >> 3, full = g.count >> 3;
    for (long long base = static_cast<long long>(blockIdx.x) * kDropThreads * kUnroll + threadIdx.x; base < groups;
         base += static_cast<long long>(gridDim.x) * kDropThreads * kUnroll) {
        Eight<T> xv[kUnroll], rv[kUnroll];
        if constexpr (kAligned) {
#pragma unroll
            for (int j = 0; j < kUnroll; ++j) {
                const long long b = base + j * kDropThreads;
                if (b < full) { xv[j].load(x + b * 8); if (kResidual) rv[j].load(res + b * 8); }
            }
        }
#pragma unroll
        for (int j = 0; j < kUnroll; ++j) {
            const long long b = base + j * kDropThreads;
            if (b >= groups) break;
            const uint4 r = philox(static_cast<unsigned long long>(b), k0, k1);
            const unsigned words[4] = {r.x, r.y, r.z, r.w};
            if (kAligned && b < full) {
                float f[8], h[8];
                xv[j].get(f);
                if (kResidual) rv[j].get(h);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    bool hi, lo;                   // both halves against the threshold in one instruction (86.8 -> 84.8 us)
                    __vibmax_u16x2(words[i], g.threshold * 0x10001u, &hi, &lo);
                    f[2 * i] = lo ? f[2 * i] * g.scale : 0.0f;
                    f[2 * i + 1] = hi ? f[2 * i + 1] * g.scale : 0.0f;
                    if (kResidual) { f[2 * i] += h[2 * i]; f[2 * i + 1] += h[2 * i + 1]; }
                }
                Eight<T>::store(out + b * 8, f);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const long long at = b * 8 + i;
                    if (at < g.count) {
                        const unsigned u = i & 1 ? words[i >> 1] >> 16 : words[i >> 1] & 0xffffu;
                        const float kept = u >= g.threshold ? drop_load(x + at) * g.scale : 0.0f;
                        drop_store(out + at, kResidual ? kept + drop_load(res + at) : kept);
                    }
                }
            }
        }
    }
}

template <typename T, bool kResidual>
int launch_dropout(const DropoutParams& g, cudaStream_t s) {
    constexpr long long per_block = 8ll * kDropThreads * Shape<T, kResidual>::kUnroll;
    const int grid = static_cast<int>(std::min<long long>((g.count + per_block - 1) / per_block, 0x7fffffff));
    const bool aligned = ((reinterpret_cast<uintptr_t>(g.x) | reinterpret_cast<uintptr_t>(g.residual) | reinterpret_cast<uintptr_t>(g.out)) & 15) == 0;
    ProfScope prof(kSlotOther, s);
    return aligned ? launch_kernel(dropout_kernel<T, kResidual, true>, grid, kDropThreads, 0, s, false, true, g)
                   : launch_kernel(dropout_kernel<T, kResidual, false>, grid, kDropThreads, 0, s, false, true, g);
}

}  // namespace
}  // namespace mok

using namespace mok;

extern "C" int mok_dropout_add(const void* x, const void* residual, const int64_t* seed, void* out, int64_t count, int is_bf16,
                               double p, void* stream) {
    if (!x || !seed || !out || count <= 0 || !(p >= 0.0 && p <= 1.0)) return MOK_ERR_INVALID;
    DropoutParams g{};
    g.x = x; g.residual = residual; g.seed = reinterpret_cast<const long long*>(seed); g.out = out; g.count = count;
    g.threshold = static_cast<unsigned>(p * 65536.0 + 0.5);
    g.scale = g.threshold < 65536u ? 65536.0f / static_cast<float>(65536u - g.threshold) : 0.0f;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (g.threshold >= 65536u) {                // everything is dropped: the kernel's 16-bit comparison has no such threshold
        const size_t bytes = static_cast<size_t>(count) * (is_bf16 ? 2 : 4);
        if (!residual) MOK_CUDA_CHECK(cudaMemsetAsync(out, 0, bytes, s));
        else if (residual != out) MOK_CUDA_CHECK(cudaMemcpyAsync(out, residual, bytes, cudaMemcpyDeviceToDevice, s));
        return MOK_OK;
    }
    if (is_bf16) return residual ? launch_dropout<__nv_bfloat16, true>(g, s) : launch_dropout<__nv_bfloat16, false>(g, s);
    return residual ? launch_dropout<float, true>(g, s) : launch_dropout<float, false>(g, s);
}
