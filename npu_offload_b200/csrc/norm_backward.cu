// Gradients of the root-mean-square norm y = h rstd w of a row h of C values, from the stored sum h and rstd:
//
//   u_c = h_c rstd;  g_c = w_c dy_c;   dh_c = rstd (g_c - u_c mean_j(g_j u_j)) + dsum_c;   dw_c = sum_t dy_tc u_tc
//
// dh is the gradient of both x and the residual.  A row is read once and stays in registers while g . u is summed over the
// CTA, the next row's words already asked for.  A CTA takes every gridDim-th row and keeps its rows' share of dw in
// registers (a column is always the same thread's), writes it once, and a second kernel adds the CTAs' shares in order: no
// sum depends on timing.
//
// Bounded by HBM: 8191 x 4096, bf16 with the stream's gradient, 48 us, 85 % of a copy's rate; 8192 x 5120 71 (72 %), 7168 84 (86 %), fp32 4000 x 4096
// 56 (72 %).  Where one CTA of few threads is all that an SM has, by what is on its way: fp32 4000 x 4099 110 us (36 %; it spills).
#include <algorithm>

#include "launch.cuh"
#include "norm.cuh"
#include "norm.h"

namespace moe {

template <bool S32, bool D32, bool DS, int N, bool V, int THREADS>
__global__ void __launch_bounds__(THREADS, N == 1 && !S32 && !D32 ? 2 : 1) norm_backward_kernel(NormBackwardArgs a, float* shares) {
    __shared__ float part[2][32];
    constexpr bool kAhead = THREADS <= kNormThreads;
    griddep_wait();
    if (shares) griddep_launch_dependents();  // the shares' sum waits for this kernel's end before it does anything
    const int C = a.C, lead = V ? 0 : (int)((int64_t)blockIdx.x * C % 8);
    float w[N][8], dw[N][8];
#pragma unroll
    for (int i = 0; i < N; i++) {
        norm_weight<V>(a.weight, a.weight_f32, norm_col(i, lead), C, w[i]);
#pragma unroll
        for (int k = 0; k < 8; k++) dw[i][k] = 0.f;
    }
    const size_t end = (size_t)a.T * C;
    Raw8<S32> h[N], ds[N];
    Raw8<D32> dy[N];
    float rstd_next = 0.f;
    auto ask = [&](int64_t t) {
        rstd_next = a.rstd[t];
#pragma unroll
        for (int i = 0; i < N; i++) {
            h[i].template load<V>(a.sum, (size_t)t * C, norm_col(i, lead), C, end);
            dy[i].template load<V>(a.dy, (size_t)t * C, norm_col(i, lead), C, end);
            if (DS) ds[i].template load<V>(a.dsum, (size_t)t * C, norm_col(i, lead), C, end);
        }
    };
    int turn = 0;
    if (kAhead && blockIdx.x < a.T) ask(blockIdx.x);
    for (int64_t t = blockIdx.x; t < a.T; t += gridDim.x, turn++) {
        if (!kAhead) ask(t);
        const float rstd = rstd_next;
        float u[N][8], g[N][8], dot = 0.f;
        Raw8<S32> dst[N];
#pragma unroll
        for (int i = 0; i < N; i++) {
            h[i].get(u[i]);
            dy[i].get(g[i]);
            keep_row<V>(u[i], norm_col(i, lead), C);
            keep_row<V>(g[i], norm_col(i, lead), C);
            if (DS) dst[i] = ds[i];
#pragma unroll
            for (int k = 0; k < 8; k++) {
                u[i][k] *= rstd;
                dw[i][k] = fmaf(g[i][k], u[i][k], dw[i][k]);
                g[i][k] *= w[i][k];
                dot = fmaf(g[i][k], u[i][k], dot);
            }
        }
        if (kAhead && t + gridDim.x < a.T) ask(t + gridDim.x);
        const float mean = cta_sum(dot, part, turn) / C;
#pragma unroll
        for (int i = 0; i < N; i++) {
            float o[8];
#pragma unroll
            for (int k = 0; k < 8; k++) o[k] = rstd * fmaf(-u[i][k], mean, g[i][k]);
            if (DS) {
                float d[8];
                dst[i].get(d);
#pragma unroll
                for (int k = 0; k < 8; k++) o[k] += d[k];
            }
            store8<V>(a.dx, S32, (size_t)t * C, norm_col(i, lead), C, o);
        }
    }
    if (shares)
#pragma unroll
        for (int i = 0; i < N; i++) store8<V>(shares, true, (size_t)blockIdx.x * C, norm_col(i, lead), C, dw[i]);
}

// dw = the shares' sum: 32 columns a CTA, 32 warps each every 32nd share, then the warps in order.
__global__ void __launch_bounds__(1024) norm_dweight_kernel(const float* shares, int n, int C, float* dweight) {
    __shared__ float s[32][33];
    griddep_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    float v = 0.f;
    if (c < C)
#pragma unroll 8
        for (int r = warp; r < n; r += 32) v += shares[(size_t)r * C + c];
    s[warp][lane] = v;
    __syncthreads();
    v = warp_sum(s[lane][warp]);  // column `warp`
    const int o = blockIdx.x * 32 + warp;
    if (lane == 0 && o < C) dweight[o] = v;
}

// (64 registers a thread of bf16 rows of one eight a thread, else up to 128; narrow rows have fewer CTAs than fit, for their shares' sake)
static int backward_grid(int64_t T, int C, bool narrow_type, int sm_count) {
    const int threads = norm_threads(C, norm_eights(C)), fit = norm_eights(C) == 1 && narrow_type && threads >= 64 ? 1024 : 512;
    return T > 0 ? norm_grid(T, (int64_t)sm_count * std::max(1, fit / threads), C) : 1;
}
size_t norm_backward_workspace(int64_t T, int C, int sm_count) {
    return (size_t)std::max(backward_grid(T, C, true, sm_count), backward_grid(T, C, false, sm_count)) * C * sizeof(float);
}

template <bool S32, bool D32, bool DS>
static cudaError_t backward_for(const NormBackwardArgs& a, int grid, cudaStream_t st) {
    float* shares = a.dweight ? a.ws : nullptr;
    const int threads = norm_threads(a.C, norm_eights(a.C));
    const Launch l{grid, threads, 0, 0, st};
    if (threads > kNormThreads && a.C % 8)
        return l.run(norm_eights(a.C) == 3 ? norm_backward_kernel<S32, D32, DS, 3, false, 1024> : norm_backward_kernel<S32, D32, DS, 2, false, 1024>, a, shares);
    if (threads > kNormThreads) return l.run(norm_backward_kernel<S32, D32, DS, 2, true, 1024>, a, shares);
    if (a.C % 8) return l.run(norm_eights(a.C) == 1 ? norm_backward_kernel<S32, D32, DS, 1, false, kNormThreads> : norm_backward_kernel<S32, D32, DS, 2, false, kNormThreads>, a, shares);
    return l.run(norm_eights(a.C) == 1 ? norm_backward_kernel<S32, D32, DS, 1, true, kNormThreads> : norm_backward_kernel<S32, D32, DS, 2, true, kNormThreads>, a, shares);
}

cudaError_t launch_add_norm_backward(const NormBackwardArgs& a, int sm_count, cudaStream_t st, int* launches) {
    if (a.C <= 0) return cudaSuccess;
    const int grid = backward_grid(a.T, a.C, !a.stream_f32 && !a.dy_f32, sm_count);
    cudaError_t e = cudaSuccess;
    if (a.T > 0) {
        const int kind = (a.stream_f32 ? 4 : 0) | (a.dy_f32 ? 2 : 0) | (a.dsum ? 1 : 0);
        switch (kind) {
            case 0: e = backward_for<false, false, false>(a, grid, st); break;
            case 1: e = backward_for<false, false, true>(a, grid, st); break;
            case 2: e = backward_for<false, true, false>(a, grid, st); break;
            case 3: e = backward_for<false, true, true>(a, grid, st); break;
            case 4: e = backward_for<true, false, false>(a, grid, st); break;
            case 5: e = backward_for<true, false, true>(a, grid, st); break;
            case 6: e = backward_for<true, true, false>(a, grid, st); break;
            default: e = backward_for<true, true, true>(a, grid, st); break;
        }
        if (e != cudaSuccess) return e;
        ++*launches;
    }
    if (a.dweight) {  // (zeros without a row)
        const Launch l{(a.C + 31) / 32, 1024, 0, 0, st};
        e = l.run(norm_dweight_kernel, (const float*)a.ws, a.T > 0 ? grid : 0, a.C, a.dweight);
        if (e == cudaSuccess) ++*launches;
    }
    return e;
}

}  // namespace moe
