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

constexpr int kDropThreads = 256;

struct DropoutParams {
    const void* x;
    const void* residual;          // may be null
    const long long* seed;
    void* out;
    long long count;
    unsigned threshold;            // 0 .. 65536
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

template <typename T>
__global__ void __launch_bounds__(kDropThreads) dropout_kernel(const DropoutParams g) {
    pdl_wait();
    const unsigned long long seed = static_cast<unsigned long long>(*g.seed);
    const unsigned k0 = static_cast<unsigned>(seed), k1 = static_cast<unsigned>(seed >> 32);
    const long long blocks = (g.count + 7) >> 3;
    for (long long b = static_cast<long long>(blockIdx.x) * kDropThreads + threadIdx.x; b < blocks;
         b += static_cast<long long>(gridDim.x) * kDropThreads) {
        const uint4 r = philox(static_cast<unsigned long long>(b), k0, k1);
        const unsigned words[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const long long i = b * 8 + j;
            if (i < g.count) {
                const unsigned u = (words[j >> 1] >> (16 * (j & 1))) & 0xffffu;
                const float kept = u >= g.threshold ? drop_load(static_cast<const T*>(g.x) + i) * g.scale : 0.0f;
                drop_store(static_cast<T*>(g.out) + i, g.residual ? kept + drop_load(static_cast<const T*>(g.residual) + i) : kept);
            }
        }
    }
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
    const long long blocks = (count + 8 * kDropThreads - 1) / (8 * kDropThreads);
    const int grid = static_cast<int>(std::min<long long>(blocks, device_sm_count() * 8));
    ProfScope prof(kSlotOther, s);
    return is_bf16 ? launch_kernel(dropout_kernel<__nv_bfloat16>, grid, kDropThreads, 0, s, false, false, g)
                   : launch_kernel(dropout_kernel<float>, grid, kDropThreads, 0, s, false, false, g);
}
