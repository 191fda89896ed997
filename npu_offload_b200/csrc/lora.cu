// Low-rank adapters of many requests beside a shared projection:
//
//   out[t] = base[t] + scale_i (x[t] A_i^T) B_i^T,   i = ids[t] (negative: out[t] = base[t])
//
// One launch: a cluster of eight CTAs a token.  Each takes an eighth of the inner dimension of A for all r rows (a warp a
// row, 16-byte loads), the partial sums go to all eight through distributed shared memory and are added there in order,
// and each then takes an eighth of the columns of B, whose first are in registers by then up to r = 32: a row of B is read by as
// many neighbouring lanes as it has 16-byte words (a thread a row: 10.6 instead of 7.5 us at 32 tokens, r = 64, when its columns were held
// early too; 7.9 as it is, below).  All sums are fp32; the result is rounded once.  Bounded by latency for a token (ids, then x and A,
// the exchange, the store), by the adapters' bytes out of L2 for a batch of requests.  4096 x 16 x 2560, one token: 3.6 us (r = 64: 5.3, r = 128: 8.2); 1280 x 32 x 4096, 48 tokens of 32
// adapters: 6.6 us, 1.6 of them for the bytes from HBM.
#include <cooperative_groups.h>

#include <algorithm>

#include "common.cuh"
#include "fp8.cuh"
#include "launch.cuh"
#include "lora.h"
#include "ptx.cuh"

namespace cg = cooperative_groups;

namespace moe {

constexpr int kLoraThreads = 256, kLoraWarps = kLoraThreads / 32;
constexpr int kLoraCluster = 8;

__device__ __forceinline__ float lora_load(const LoraArgs& a, size_t i) {
    return a.out_f32 ? static_cast<const float*>(a.base)[i] : bf2f(static_cast<const uint16_t*>(a.base)[i]);
}
__device__ __forceinline__ void lora_store(const LoraArgs& a, size_t i, float v) {
    if (a.out_f32) static_cast<float*>(a.out)[i] = v;
    else static_cast<uint16_t*>(a.out)[i] = f8_bf16(v);
}

// R: rank rows of A a warp, and 16-byte words of a row of B; r <= 8 R, R a power of two.
template <int R>
__global__ void __cluster_dims__(kLoraCluster, 1, 1) __launch_bounds__(kLoraThreads, R == 16 ? 2 : R == 8 ? 3 : 4) lora_few_kernel(LoraArgs a) {
    __shared__ float part[kLoraCluster][kLoraMaxRank], own[kLoraMaxRank], low[kLoraMaxRank];
    griddep_wait();
    cg::cluster_group cl = cg::this_cluster();
    const int c = (int)cl.block_rank(), t = blockIdx.x / kLoraCluster;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = a.r;
    const int n0 = (int)((int64_t)c * a.N / kLoraCluster), n1 = (int)((int64_t)(c + 1) * a.N / kLoraCluster);
    const int id = a.ids[t];
    const size_t out_row = (size_t)t * a.N;
    if (id < 0 || id >= a.n) {  // the whole cluster alike
        if (id >= a.n && c == 0 && threadIdx.x == 0) atomicOr(a.err, kErrBadIndex);
        if (a.out != a.base)
            for (int n = n0 + threadIdx.x; n < n1; n += kLoraThreads) lora_store(a, out_row + n, lora_load(a, out_row + n));
        return;
    }
    const uint16_t* A = a.a + (size_t)id * r * a.K;
    const uint16_t* B = a.b + (size_t)id * a.N * r;
    const uint16_t* x = a.x + (size_t)t * a.K;
    // Columns of B, 32 a warp: R neighbouring lanes a row of B, 16 bytes each, R rows after one another; the first are on their way early.
    const int chunk = lane % R, g1 = (n1 - n0 + 31) / 32;
    // (Held that early, eight words a lane cost a CTA of each SM: r = 64, 1280 x 4096, 7.5 / 7.8 us with / without at 32 tokens, 13.3 / 8.8 at 48, and
    // 4096 x 2560 8.3 / 8.9 and 14.8 / 9.9; sixteen, r = 128, 20.2 / 13.3 at 24.  Asking L2 for them instead: 7.9, 9.1; 13.9.)
    constexpr bool kEarly = R < 8;
    uint4 bv[R];
    auto ask = [&](int g) {
#pragma unroll
        for (int i = 0; i < R; i++) {
            const int n = n0 + g * 32 + lane / R + 32 / R * i;
            bv[i] = n < n1 && chunk * 8 < r ? ld_cg_u4(B + (size_t)n * r + chunk * 8) : make_uint4(0, 0, 0, 0);
        }
    };
    const int mine = lane / R + 32 / R * chunk;  // the column of 32 whose sum this lane ends up with
    float base = 0.f;
    if (warp < g1) {
        if (kEarly) ask(warp);
        if (n0 + warp * 32 + mine < n1) base = lora_load(a, out_row + n0 + warp * 32 + mine);
    }
    float acc[R];
#pragma unroll
    for (int k = 0; k < R; k++) acc[k] = 0.f;
    const int u1 = (int)((int64_t)(c + 1) * (a.K / 8) / kLoraCluster);
    for (int u = (int)((int64_t)c * (a.K / 8) / kLoraCluster) + lane; u < u1; u += 32) {
        const uint4 xv = ld_cg_u4(x + u * 8);
        uint4 av[R];
#pragma unroll
        for (int k = 0; k < R; k++)
            if (warp + k * kLoraWarps < r) av[k] = ld_cg_u4(A + (size_t)(warp + k * kLoraWarps) * a.K + u * 8);
#pragma unroll
        for (int k = 0; k < R; k++)
            if (warp + k * kLoraWarps < r) acc[k] = dot8_bf16(av[k], xv, acc[k]);
    }
#pragma unroll
    for (int k = 0; k < R; k++) {
        const float v = warp_sum(acc[k]);
        if (lane == 0 && warp + k * kLoraWarps < r) own[warp + k * kLoraWarps] = v;
    }
    cl.sync();  // every CTA has begun (their shared memory may be written to); own is complete
    for (int i = threadIdx.x; i < kLoraCluster * r; i += kLoraThreads) {
        const int to = i / r, k = i - to * r;
        cl.map_shared_rank(&part[c][0], to)[k] = own[k];
    }
    cl.sync();
    if (threadIdx.x < r) {
        float v = 0.f;
#pragma unroll
        for (int i = 0; i < kLoraCluster; i++) v += part[i][threadIdx.x];
        low[threadIdx.x] = v * (a.scale ? a.scale[id] : 1.f);
    }
    __syncthreads();
    float l8[8];
#pragma unroll
    for (int k = 0; k < 8; k++) l8[k] = chunk * 8 < r ? low[chunk * 8 + k] : 0.f;
    for (int g = warp; g < g1; g += kLoraWarps) {
        const int n = n0 + g * 32 + mine;
        if (!kEarly || g != warp) ask(g);
        if (g != warp && n < n1) base = lora_load(a, out_row + n);
        float v[R];
#pragma unroll
        for (int i = 0; i < R; i++) {
            const uint32_t w[4] = {bv[i].x, bv[i].y, bv[i].z, bv[i].w};
            v[i] = 0.f;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                v[i] = fmaf(bf_lo(w[k]), l8[2 * k], v[i]);
                v[i] = fmaf(bf_hi(w[k]), l8[2 * k + 1], v[i]);
            }
        }
        // R sums over R lanes, one left on each: sum i on the lane with chunk i
#pragma unroll
        for (int o = R / 2; o > 0; o /= 2) {
            const bool up = lane & o;
#pragma unroll
            for (int k = 0; k < o; k++) {
                const float give = up ? v[k] : v[k + o];
                v[k] = (up ? v[k + o] : v[k]) + __shfl_xor_sync(0xffffffffu, give, o);
            }
        }
        if (n < n1) lora_store(a, out_row + n, base + v[0]);
    }
}

// Calls of at most so many tokens take a cluster a token, others the kernels of lora_many.cu, us (a cluster a token / the others):
//   r = 16: 64 tokens 5.8 / 11.3, 128: 11.4 / 11.3, 192: 16.1 / 12.0 (4096 x 2560)     r = 32: 64: 7.0 / 13.2, 128: 12.7 / 13.0 (1280 x 4096)
//   r = 64: 48: 8.8 / 14.7, 64: 14.5 / 14.9, 96: 16.0 / 14.9 (1280 x 4096)              r = 128: 32: 13.7 / 20.6, 48: 23.8 / 22.2 (4096 x 2560)
static int lora_few_tokens(int r) { return r <= 32 ? 128 : r <= 64 ? 64 : 32; }

size_t lora_workspace(int T, int n, int r) { return T <= lora_few_tokens(r) ? 0 : lora_many_workspace(T, n, r); }

cudaError_t launch_add_lora(const LoraArgs& a, int sm_count, cudaStream_t st, int* launches) {
    if (a.T <= 0 || a.N <= 0) return cudaSuccess;
    if (a.T > lora_few_tokens(a.r)) return launch_lora_many(a, sm_count, st, launches);
    const Launch l{a.T * kLoraCluster, kLoraThreads, 0, 0, st};
    ++*launches;
    if (a.r <= 8) return l.run(lora_few_kernel<1>, a);
    if (a.r <= 16) return l.run(lora_few_kernel<2>, a);
    if (a.r <= 32) return l.run(lora_few_kernel<4>, a);
    if (a.r <= 64) return l.run(lora_few_kernel<8>, a);
    return l.run(lora_few_kernel<16>, a);
}

}  // namespace moe
