// Low-rank adapters of many requests beside a shared projection:
//
//   out[t] = base[t] + scale_i (x[t] A_i^T) B_i^T,   i = ids[t] (negative: out[t] = base[t])
//
// One launch: a cluster of eight CTAs a token.  Each takes an eighth of the inner dimension of A for all r rows (a warp a
// row, 16-byte loads), the partial sums go to all eight through distributed shared memory and are added there in order,
// and each then takes an eighth of the columns of B, a thread a column, whose first rows are in registers by then.  All
// sums are fp32; the result is rounded once.  Bounded by latency for a token (ids, then x and A, the exchange, the
// store), by the adapters' bytes for a batch of requests with adapters of their own.
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

// R: rank rows of A a warp, and 16-byte words of a row of B; r <= 8 R.
template <int R>
__global__ void __cluster_dims__(kLoraCluster, 1, 1) __launch_bounds__(kLoraThreads) lora_few_kernel(LoraArgs a) {
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
    uint4 first[R];
    float base = 0.f;
    if (n0 + (int)threadIdx.x < n1) {
        base = lora_load(a, out_row + n0 + threadIdx.x);
#pragma unroll
        for (int k = 0; k < R; k++)
            if (k * 8 < r) first[k] = ld_cg_u4(B + (size_t)(n0 + threadIdx.x) * r + k * 8);
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
    for (int n = n0 + threadIdx.x; n < n1; n += kLoraThreads) {
        if (n != n0 + (int)threadIdx.x) {
            base = lora_load(a, out_row + n);
#pragma unroll
            for (int k = 0; k < R; k++)
                if (k * 8 < r) first[k] = ld_cg_u4(B + (size_t)n * r + k * 8);
        }
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < R; k++)
            if (k * 8 < r) {
                const uint32_t w[4] = {first[k].x, first[k].y, first[k].z, first[k].w};
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    v = fmaf(bf_lo(w[j]), low[k * 8 + 2 * j], v);
                    v = fmaf(bf_hi(w[j]), low[k * 8 + 2 * j + 1], v);
                }
            }
        lora_store(a, out_row + n, base + v);
    }
}

// Calls of at most so many tokens take a cluster a token.
#ifndef LORA_FEW
#define LORA_FEW 128
#endif
constexpr int kLoraFewTokens = LORA_FEW;

size_t lora_workspace(int T, int n) { return T <= kLoraFewTokens ? 0 : lora_many_workspace(T, n); }

cudaError_t launch_add_lora(const LoraArgs& a, int sm_count, cudaStream_t st, int* launches) {
    if (a.T <= 0 || a.N <= 0) return cudaSuccess;
    if (a.T > kLoraFewTokens) return launch_lora_many(a, st, launches);
    const Launch l{a.T * kLoraCluster, kLoraThreads, 0, 0, st};
    ++*launches;
    if (a.r <= 8) return l.run(lora_few_kernel<1>, a);
    if (a.r <= 16) return l.run(lora_few_kernel<2>, a);
    if (a.r <= 32) return l.run(lora_few_kernel<4>, a);
    if (a.r <= 64) return l.run(lora_few_kernel<8>, a);
    return l.run(lora_few_kernel<16>, a);
}

}  // namespace moe
