// Residual addition and root-mean-square norm, to bf16 or fp32 and / or to e4m3 with a scale for each 128 columns.
//
//   h = x + residual, rounded to the residual's type (the stream);  rstd = 1 / sqrt(mean_c h_c^2 + eps)
//   y = h rstd w, rounded once;   s = smallest power of two >= 2^-126 with max|y| <= 448 s;   q = e4m3(y / s)
//
// The norm is of the sum as the stream holds it, so that the gradient can be formed from the stored sum alone.
// A row is read once: it stays in registers, eight values (one 16-byte word of bf16) at a time, while its squares are
// summed over the CTA, and the next row's words are asked for before this one is worked on.
//
// A scale doubles where max|y| passes 448 2^k.  In 32 bits max|y| may be off by 24 steps (of 2^-23, relative: half the
// sum's (at most 32 values a thread and 10 levels of warps and CTA), the root's two and the products' two); where it lies
// within that of such a border, about one group in 10^5, the warp reads the row again and decides in 64 bits: the scales
// are those of the definition.  The same 64-bit sum serves rows whose squares leave fp32's range.
#include <algorithm>

#include "launch.cuh"
#include "norm.cuh"
#include "norm.h"

namespace moe {

// One row's 1 / sqrt(mean h^2 + eps) in 64 bits, by one warp, from memory.
template <bool X32, int R>
__device__ __noinline__ double rstd_64(const void* x, const void* residual, size_t row, int C, float eps) {
    double s = 0;
    for (int c = threadIdx.x & 31; c < C; c += 32) {
        float h = X32 ? static_cast<const float*>(x)[row + c] : bf2f(static_cast<const uint16_t*>(x)[row + c]);
        if (R == 1) h = bf2f(f8_bf16(h + bf2f(static_cast<const uint16_t*>(residual)[row + c])));
        if (R == 2) h += static_cast<const float*>(residual)[row + c];
        s += (double)h * (double)h;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return 1.0 / sqrt(s / C + (double)eps);
}

// R: the residual is none (0), bf16 (1) or fp32 (2).
template <bool X32, int R, int N, bool V, int THREADS>
__global__ void __launch_bounds__(THREADS) add_norm_kernel(NormArgs a, float tiny) {
    __shared__ float part[2][32];
    constexpr bool kAhead = THREADS <= kNormThreads;
    griddep_wait();
    const int step = V ? 1 : blockDim.x, C = a.C, groups = (C + kF8Block - 1) / kF8Block;
    float w[N][8];
#pragma unroll
    for (int i = 0; i < N; i++) {
        if (a.weight_f32) {
            Raw8<true> r;
            r.template load<V>(a.weight, 0, norm_col<V>(i), step, C);
            r.get(w[i]);
        } else {
            Raw8<false> r;
            r.template load<V>(a.weight, 0, norm_col<V>(i), step, C);
            r.get(w[i]);
        }
    }
    Raw8<X32> x[N];
    Raw8<R == 2> res[N];
    auto ask = [&](int64_t t) {
#pragma unroll
        for (int i = 0; i < N; i++) {
            x[i].template load<V>(a.x, (size_t)t * C, norm_col<V>(i), step, C);
            if (R) res[i].template load<V>(a.residual, (size_t)t * C, norm_col<V>(i), step, C);
        }
    };
    int turn = 0;
    if (kAhead && blockIdx.x < a.T) ask(blockIdx.x);
    for (int64_t t = blockIdx.x; t < a.T; t += gridDim.x, turn++) {
        const size_t row = (size_t)t * C;
        if (!kAhead) ask(t);
        float h[N][8], ss = 0.f;
#pragma unroll
        for (int i = 0; i < N; i++) {
            x[i].get(h[i]);
            if (R) {
                float r[8];
                res[i].get(r);
#pragma unroll
                for (int k = 0; k < 8; k++) h[i][k] += r[k];
                if (R == 1)
#pragma unroll
                    for (int k = 0; k < 8; k += 2) {
                        const uint32_t b = f8_bf16x2(h[i][k], h[i][k + 1]);
                        h[i][k] = bf_lo(b), h[i][k + 1] = bf_hi(b);
                    }
            }
#pragma unroll
            for (int k = 0; k < 8; k++) ss = fmaf(h[i][k], h[i][k], ss);
        }
        if (kAhead && t + gridDim.x < a.T) ask(t + gridDim.x);
        if (R)
#pragma unroll
            for (int i = 0; i < N; i++) store8<V>(a.sum, R == 2, row, norm_col<V>(i), step, C, h[i]);
        ss = cta_sum(ss, part, turn);
        const bool wide = !(ss < 1e37f) || ss < tiny;  // squares that leave fp32's range (or are none)
        double rstd64 = 0;
        float rstd;
        if (wide) {
            rstd64 = rstd_64<X32, R>(a.x, a.residual, row, C, a.eps);
            rstd = (float)rstd64;
        } else {
            rstd = rsqrtf(ss / C + a.eps);
        }
        if (threadIdx.x == 0 && a.rstd) a.rstd[t] = rstd;
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int c = norm_col<V>(i);
            float y[8];
#pragma unroll
            for (int k = 0; k < 8; k++) y[k] = h[i][k] * rstd * w[i][k];
            if (wide)
#pragma unroll
                for (int k = 0; k < 8; k++) y[k] = (float)((double)h[i][k] * rstd64 * (double)w[i][k]);
            if (a.y) store8<V>(a.y, a.y_f32, row, c, step, C, y);
            if (V && a.q) {
                bool special;
                uint32_t top = f8_top(y, special);
#pragma unroll
                for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
                uint32_t se = f8_scale_exp(top);
                const bool near = top != 0 && abs((int)(top & 0x7fffffu) - 0x600000) <= 24;
                if (__any_sync(0xffffffffu, near)) {
                    const double r = wide ? rstd64 : rstd_64<X32, R>(a.x, a.residual, row, C, a.eps);
                    double most = 0;
#pragma unroll
                    for (int k = 0; k < 8; k++) {
                        const double v = fabs((double)h[i][k] * r * (double)w[i][k]);
                        if (fabsf(y[k]) < INFINITY) most = fmax(most, v);
                    }
#pragma unroll
                    for (int o = 8; o > 0; o >>= 1) most = fmax(most, __shfl_xor_sync(0xffffffffu, most, o));
                    if (near) {
                        const int e = (int)(top >> 23);  // the border in this octave is 1.75 2^(e - 127)
                        se = max(e - (most > scalbn(1.75, e - 127) ? 7 : 8), 1);
                    }
                }
                if (c < C) *reinterpret_cast<uint2*>(a.q + row + c) = f8_pack8(y, f8_inverse(se), special);
                if (c < C && (threadIdx.x & 15) == 0) a.scale[t * groups + c / kF8Block] = __uint_as_float(se << 23);
            }
        }
    }
}

template <bool X32, int R>
static cudaError_t add_norm_for(const NormArgs& a, int sm_count, cudaStream_t st) {
    // Squares below fp32's range count for nothing beside eps, unless eps is of that kind itself.
    const float tiny = a.eps < 1e-18f ? 1e-24f : 0.f;
    const int threads = norm_threads(a.C);
    const int grid = (int)std::min<int64_t>(a.T, (int64_t)sm_count * std::max(1, 1024 / threads));
    const Launch l{grid, threads, 0, 0, st};
    if (threads > kNormThreads) return l.run(a.C % 8 ? add_norm_kernel<X32, R, 2, false, 1024> : add_norm_kernel<X32, R, 2, true, 1024>, a, tiny);
    if (a.C % 8) return l.run(add_norm_kernel<X32, R, 2, false, kNormThreads>, a, tiny);
    return l.run(norm_eights(a.C) == 1 ? add_norm_kernel<X32, R, 1, true, kNormThreads> : add_norm_kernel<X32, R, 2, true, kNormThreads>, a, tiny);
}

cudaError_t launch_add_norm(const NormArgs& a, int sm_count, cudaStream_t st) {
    if (a.T <= 0 || a.C <= 0) return cudaSuccess;
    const int r = !a.residual ? 0 : a.stream_f32 ? 2 : 1;
    if (a.x_f32) return r == 0 ? add_norm_for<true, 0>(a, sm_count, st) : r == 1 ? add_norm_for<true, 1>(a, sm_count, st) : add_norm_for<true, 2>(a, sm_count, st);
    return r == 0 ? add_norm_for<false, 0>(a, sm_count, st) : r == 1 ? add_norm_for<false, 1>(a, sm_count, st) : add_norm_for<false, 2>(a, sm_count, st);
}

}  // namespace moe
