// e4m3 quantiser: values in groups of 128 columns of one row (activations) or of 128 rows (weights).
//
//   s    = the smallest power of two >= 2^-126 with max|x| <= 448 s   (1 for a group of zeros)
//   q[i] = x[i] / s rounded once to e4m3 (ties to even); infinities and NaN become NaN, and take no
//          part in the maximum
//
// A power of two keeps x / s exact, so every value is rounded once and the result does not depend on
// how the quotient is formed; e4m3 being a floating-point type, the precision is that of the scale
// max|x| / 448 except for values near the bottom of its range.  Both kernels read each value once
// into registers, where it stays until the group's maximum is known: 3 (bf16) or 5 (fp32) bytes a
// value, bounded by HBM.
#include <algorithm>

#include "common.cuh"
#include "fp8.h"
#include "fp8.cuh"
#include "launch.cuh"
#include "ptx.cuh"

namespace moe {

// Eight consecutive values as floats, from bf16 or fp32.
template <bool F32>
struct Eight;
template <>
struct Eight<false> {
    uint4 v;
    __device__ __forceinline__ void load(const void* x, size_t i) {
        v = ld_cg_u4(static_cast<const uint16_t*>(x) + i);
    }
    __device__ __forceinline__ void zero() { v = make_uint4(0, 0, 0, 0); }
    __device__ __forceinline__ void get(float (&f)[8]) const {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int k = 0; k < 4; k++) f[2 * k] = bf_lo(w[k]), f[2 * k + 1] = bf_hi(w[k]);
    }
    __device__ __forceinline__ uint32_t top(bool& special) const { return f8_top(v, special); }
};
template <>
struct Eight<true> {
    uint4 a, b;
    __device__ __forceinline__ void load(const void* x, size_t i) {
        a = ld_cg_u4(static_cast<const float*>(x) + i);
        b = ld_cg_u4(static_cast<const float*>(x) + i + 4);
    }
    __device__ __forceinline__ void zero() { a = b = make_uint4(0, 0, 0, 0); }
    __device__ __forceinline__ void get(float (&f)[8]) const {
        const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
        for (int k = 0; k < 8; k++) f[k] = __uint_as_float(w[k]);
    }
    __device__ __forceinline__ uint32_t top(bool& special) const {
        float f[8];
        get(f);
        return f8_top(f, special);
    }
};

// Rows: sixteen lanes hold a group, eight values each, and share its maximum by shuffles; N groups' loads
// in flight for each half warp.
template <bool F32, int N>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const void* x, uint32_t groups, uint32_t per_row,
                                                            uint32_t cols, uint8_t* q, float* s) {
    griddep_wait();
    griddep_launch_dependents();
    const uint32_t sub = threadIdx.x & 15, g0 = blockIdx.x * 16 * N + (threadIdx.x >> 4);
    Eight<F32> v[N];
    size_t at[N];
    bool in[N];
#pragma unroll
    for (int n = 0; n < N; n++) {
        const uint32_t g = g0 + n * 16, row = g / per_row, c = (g - row * per_row) * kF8Block + sub * 8;
        in[n] = g < groups && c < cols;
        at[n] = (size_t)row * cols + c;
        if (in[n]) v[n].load(x, at[n]);
        else v[n].zero();
    }
#pragma unroll
    for (int n = 0; n < N; n++) {
        float f[8];
        bool special;
        v[n].get(f);
        uint32_t top = v[n].top(special);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        const uint32_t se = f8_scale_exp(top);
        const uint2 r = f8_pack8(f, f8_inverse(se), special);
        if (in[n]) *reinterpret_cast<uint2*>(q + at[n]) = r;
        const uint32_t g = g0 + n * 16;
        if (sub == 0 && g < groups) s[g] = __uint_as_float(se << 23);
    }
}

// 128 x 128 blocks: one CTA a block, thread t columns 8 (t % 16) .. of rows t / 16 + 16 i.
template <bool F32>
__global__ void __launch_bounds__(256, F32 ? 2 : 4) quantize_blocks_kernel(const void* x, uint32_t rows, uint32_t cols,
                                                              uint32_t rb, uint32_t cb, uint8_t* q,
                                                              float* s) {
    __shared__ uint32_t top_s[8];
    griddep_wait();
    griddep_launch_dependents();
    const uint32_t b = blockIdx.x / cb, kb = blockIdx.x - b * cb, mat = b / rb, r0 = (b - mat * rb) * kF8Block;
    const uint32_t c = kb * kF8Block + (threadIdx.x & 15) * 8;
    const size_t base = (size_t)mat * rows * cols;
    Eight<F32> v[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const uint32_t r = r0 + (threadIdx.x >> 4) + 16 * i;
        if (r < rows && c < cols) v[i].load(x, base + (size_t)r * cols + c);
        else v[i].zero();
    }
    uint32_t top = 0;
    bool special = false;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        bool s8;
        top = max(top, v[i].top(s8));
        special |= s8;
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if ((threadIdx.x & 31) == 0) top_s[threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; w++) top = max(top, top_s[w]);
    const uint32_t se = f8_scale_exp(top);
    const float inv = f8_inverse(se);
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const uint32_t r = r0 + (threadIdx.x >> 4) + 16 * i;
        float f[8];
        v[i].get(f);
        if (r < rows && c < cols) *reinterpret_cast<uint2*>(q + base + (size_t)r * cols + c) = f8_pack8(f, inv, special);
    }
    if (threadIdx.x == 0) s[blockIdx.x] = __uint_as_float(se << 23);
}

cudaError_t launch_quantize_fp8(const void* x, bool f32, int64_t batch, int64_t rows, int64_t cols, int block_rows,
                                uint8_t* q, float* s, int sm_count, cudaStream_t st) {
    if (batch <= 0 || rows <= 0 || cols <= 0) return cudaSuccess;
    const int64_t cb = (cols + kF8Block - 1) / kF8Block;
    if (block_rows == 1) {
        const int64_t groups = batch * rows * cb;
        if (groups >= (1ll << 31) || cols >= (1ll << 31)) return cudaErrorInvalidValue;
        // few groups: one a half warp, spread over the SMs; else two (fp32) or four (bf16)
        const int n = groups <= 64ll * sm_count ? 1 : f32 ? 2 : 4;
        const int grid = (int)((groups + 16 * n - 1) / (16 * n));
        const uint32_t ng = (uint32_t)groups, per_row = (uint32_t)cb, nc = (uint32_t)cols;
        if (n == 1 && f32) return launch_after(quantize_rows_kernel<true, 1>, grid, 256, 0, 0, st, x, ng, per_row, nc, q, s);
        if (n == 1) return launch_after(quantize_rows_kernel<false, 1>, grid, 256, 0, 0, st, x, ng, per_row, nc, q, s);
        if (f32) return launch_after(quantize_rows_kernel<true, 2>, grid, 256, 0, 0, st, x, ng, per_row, nc, q, s);
        return launch_after(quantize_rows_kernel<false, 4>, grid, 256, 0, 0, st, x, ng, per_row, nc, q, s);
    }
    const int64_t rb = (rows + kF8Block - 1) / kF8Block, blocks = batch * rb * cb;
    if (blocks >= (1ll << 31) || rows >= (1ll << 31) || cols >= (1ll << 31)) return cudaErrorInvalidValue;
    if (f32) return launch_after(quantize_blocks_kernel<true>, (int)blocks, 256, 0, 0, st, x, (uint32_t)rows, (uint32_t)cols, (uint32_t)rb, (uint32_t)cb, q, s);
    return launch_after(quantize_blocks_kernel<false>, (int)blocks, 256, 0, 0, st, x, (uint32_t)rows, (uint32_t)cols, (uint32_t)rb, (uint32_t)cb, q, s);
}

}  // namespace moe
