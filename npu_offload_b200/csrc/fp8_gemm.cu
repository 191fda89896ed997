// Products of e4m3 operands with one scale for each 128 values, and the routed-expert FFN built on them.
//
//   out[m, n] = sum_kb xs[m, kb] ws[n / 128, kb] sum_{k in block kb} x[m, k] w[n, k]
//
// The products of two e4m3 values are exact in fp32; all sums are fp32.
#include <algorithm>

#include "common.cuh"
#include "fp8.h"
#include "fp8.cuh"

namespace moe {

// One warp's dot product of an activation row and a weight row; every lane gets the sum.
__device__ __forceinline__ float dot_row(const uint8_t* x, const float* xs, const uint8_t* w, const float* ws, int K) {
    float acc = 0.f;
    for (int k = (threadIdx.x & 31) * 16; k < K; k += 512) {
        float a[16], b[16], d = 0.f;
        f8_unpack16(__ldg(reinterpret_cast<const uint4*>(x + k)), a);
        f8_unpack16(__ldg(reinterpret_cast<const uint4*>(w + k)), b);
#pragma unroll
        for (int i = 0; i < 16; i++) d = fmaf(a[i], b[i], d);
        acc = fmaf(d, xs[k / kF8Block] * ws[k / kF8Block], acc);
    }
    return warp_sum(acc);
}

__device__ __forceinline__ void store_out(void* out, bool f32, size_t i, float v) {
    if (f32) static_cast<float*>(out)[i] = v;
    else static_cast<uint16_t*>(out)[i] = f2bf(v);
}

__global__ void __launch_bounds__(256) matmul_fp8_kernel(const uint8_t* x, const float* xs, const uint8_t* w, const float* ws,
                                                         int64_t M, int64_t N, int K, void* out, bool f32) {
    const int kb = (K + kF8Block - 1) / kF8Block;
    for (int64_t i = blockIdx.x * 8ll + (threadIdx.x >> 5); i < M * N; i += gridDim.x * 8ll) {
        const int64_t m = i / N, n = i - m * N;
        const float v = dot_row(x + m * K, xs + m * kb, w + n * K, ws + n / kF8Block * kb, K);
        if ((threadIdx.x & 31) == 0) store_out(out, f32, i, v);
    }
}

cudaError_t launch_matmul_fp8(const MatmulF8& a, int sm_count, cudaStream_t st) {
    if (a.M <= 0 || a.N <= 0) return cudaSuccess;
    const int64_t ctas = (a.M * a.N + 7) / 8;
    matmul_fp8_kernel<<<(int)std::min<int64_t>(ctas, sm_count * 64ll), 256, 0, st>>>(a.x, a.xs, a.w, a.ws, a.M, a.N, a.K, a.out,
                                                                                    a.out_f32);
    return cudaGetLastError();
}

// ---- routed experts ----

__global__ void __launch_bounds__(256) gate_up_fp8_kernel(ExpertsF8 a, const uint8_t* xq, const float* xs, float* act) {
    const int hb = (a.H + kF8Block - 1) / kF8Block, fb = (a.F + kF8Block - 1) / kF8Block;
    const int64_t n = (int64_t)a.T * a.K * a.F;
    for (int64_t i = blockIdx.x * 8ll + (threadIdx.x >> 5); i < n; i += gridDim.x * 8ll) {
        const int64_t p = i / a.F;
        const int f = (int)(i - p * a.F), e = a.idx[p];
        if (e < 0 || e >= a.E) {
            if (e >= a.E && (threadIdx.x & 31) == 0) atomicOr(a.err, kErrBadIndex);
            continue;
        }
        const int64_t t = p / a.K;
        float v[2];
#pragma unroll
        for (int h = 0; h < 2; h++)
            v[h] = dot_row(xq + t * a.H, xs + t * hb, a.gu + (((int64_t)e * 2 + h) * a.F + f) * a.H,
                           a.gus + (((int64_t)e * 2 + h) * fb + f / kF8Block) * hb, a.H);
        if ((threadIdx.x & 31) == 0) act[i] = v[0] / (1.f + expf(-v[0])) * v[1];
    }
}

__global__ void __launch_bounds__(256) down_fp8_kernel(ExpertsF8 a, const uint8_t* aq, const float* as, float* y) {
    const int hb = (a.H + kF8Block - 1) / kF8Block, fb = (a.F + kF8Block - 1) / kF8Block;
    const int64_t n = (int64_t)a.T * a.K * a.H;
    for (int64_t i = blockIdx.x * 8ll + (threadIdx.x >> 5); i < n; i += gridDim.x * 8ll) {
        const int64_t p = i / a.H;
        const int h = (int)(i - p * a.H), e = a.idx[p];
        if (e < 0 || e >= a.E) continue;
        const float v = dot_row(aq + p * a.F, as + p * fb, a.d + ((int64_t)e * a.H + h) * a.F,
                                a.ds + ((int64_t)e * hb + h / kF8Block) * fb, a.F);
        if ((threadIdx.x & 31) == 0) y[i] = v;
    }
}

__global__ void __launch_bounds__(256) combine_fp8_kernel(ExpertsF8 a, const float* y) {
    const int64_t n = (int64_t)a.T * a.H;
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) {
        const int64_t t = i / a.H, h = i - t * a.H;
        float v = a.accumulate ? static_cast<const float*>(a.out)[i] : 0.f;
        for (int k = 0; k < a.K; k++) {
            const int e = a.idx[t * a.K + k];
            if (e >= 0 && e < a.E) v = fmaf(a.w[t * a.K + k], y[(t * a.K + k) * a.H + h], v);
        }
        store_out(a.out, a.out_f32, i, v);
    }
}

namespace {
struct Ws {
    uint8_t *xq, *aq;
    float *xs, *as, *act, *y;
    size_t bytes;
};
Ws experts_layout(void* ws, int T, int K, int H, int F) {
    Ws w;
    char* p = static_cast<char*>(ws);
    size_t o = 0;
    auto take = [&](size_t n) {
        char* r = p + o;
        o += (n + 255) / 256 * 256;
        return r;
    };
    const size_t P = (size_t)T * K, hb = (H + kF8Block - 1) / kF8Block, fb = (F + kF8Block - 1) / kF8Block;
    w.xq = (uint8_t*)take((size_t)T * H);
    w.xs = (float*)take(4 * (size_t)T * hb);
    w.act = (float*)take(4 * P * F);
    w.aq = (uint8_t*)take(P * F);
    w.as = (float*)take(4 * P * fb);
    w.y = (float*)take(4 * P * H);
    w.bytes = o;
    return w;
}
}  // namespace

size_t experts_fp8_workspace(int T, int K, int H, int F, int E) { return experts_layout(nullptr, T, K, H, F).bytes; }

cudaError_t launch_experts_fp8(const ExpertsF8& a, int sm_count, cudaStream_t st, int* launches) {
    if (a.T <= 0) return cudaSuccess;
    const Ws w = experts_layout(a.ws, a.T, a.K, a.H, a.F);
    cudaError_t e = launch_quantize_fp8(a.x, false, 1, a.T, a.H, 1, w.xq, w.xs, sm_count, st);
    if (e != cudaSuccess) return e;
    const int grid = sm_count * 16;
    gate_up_fp8_kernel<<<grid, 256, 0, st>>>(a, w.xq, w.xs, w.act);
    e = launch_quantize_fp8(w.act, true, 1, (int64_t)a.T * a.K, a.F, 1, w.aq, w.as, sm_count, st);
    if (e != cudaSuccess) return e;
    down_fp8_kernel<<<grid, 256, 0, st>>>(a, w.aq, w.as, w.y);
    combine_fp8_kernel<<<grid, 256, 0, st>>>(a, w.y);
    *launches += 5;
    return cudaGetLastError();
}

}  // namespace moe
