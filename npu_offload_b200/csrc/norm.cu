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
// are those of the definition.  Rows whose squares leave fp32's range are done in 64 bits.
//
// Bounded by HBM: 16384 x 4096, bf16 with a bf16 residual, 89 us, 92 % of a copy's rate; 2047 x 4096 into e4m3 15 us (61 %: seven rows a
// CTA, one after the other, and the launch).  At other widths by what is on its way, since an SM has 512 / threads CTAs, rounded down, and each
// asks for one row ahead: 8192 x 5120 69 us (75 %), 7168 84 (85 %), 8192 91 (90 %); above 8192 columns for none: 4096 x 12288 105 (59 %).  Rows that
// are no multiples of eight write their ends value by value besides: 4000 x 4099 38 us (52 %), 16384 x 2047 107 (38 %).
#include <algorithm>

#include "launch.cuh"
#include "norm.cuh"
#include "norm.h"

namespace moe {

// ---- Rare paths, from memory and out of line, so that they cost the rows' path no registers.

// Eight values of the sum, from column c on.
template <bool X32, int R, bool V>
__device__ __forceinline__ void sum8(const NormArgs& a, size_t row, int c, float (&h)[8]) {
    Raw8<X32> x;
    const size_t end = (size_t)a.T * a.C;
    x.template load<V>(a.x, row, c, a.C, end);
    x.get(h);
    if (R) {
        Raw8<R == 2> res;
        float r[8];
        res.template load<V>(a.residual, row, c, a.C, end);
        res.get(r);
#pragma unroll
        for (int k = 0; k < 8; k++) h[k] = R == 1 ? bf2f(f8_bf16(h[k] + r[k])) : h[k] + r[k];
    }
    keep_row<V>(h, c, a.C);
}
template <bool V>
__device__ __forceinline__ void weight8(const NormArgs& a, int c, float (&w)[8]) {
    norm_weight<V>(a.weight, a.weight_f32, c, a.C, w);
}
// One row's 1 / sqrt(mean h^2 + eps) in 64 bits, by one warp.
template <bool X32, int R, bool V>
__device__ __forceinline__ double rstd_64(const NormArgs& a, size_t row) {
    double s = 0;
#pragma unroll 2
    for (int c = (int)(threadIdx.x & 31) * 8 - (int)(V ? 0 : row % 8); c < a.C; c += 256) {
        float h[8];
        sum8<X32, R, V>(a, row, c, h);
#pragma unroll
        for (int k = 0; k < 8; k++) s += (double)h[k] * (double)h[k];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return 1.0 / sqrt(s / a.C + (double)a.eps);
}
// Whether the largest |y| of the half warp's 128 columns, this lane's from c on, is over `border`; finite values alone.
template <bool X32, int R>
__device__ __forceinline__ bool over_border(const NormArgs& a, size_t row, int c, double rstd, double border) {
    float h[8], w[8];
    sum8<X32, R, true>(a, row, c, h);
    weight8<true>(a, c, w);
    double most = 0;
#pragma unroll
    for (int k = 0; k < 8; k++) {
        const double v = fabs((double)h[k] * rstd * (double)w[k]);
        if (v < 3e38) most = fmax(most, v);
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) most = fmax(most, __shfl_xor_sync(0xffffffffu, most, o));
    return most > border;
}
// The scale's exponent where the largest |y|, with bits `top`, lies near a border; all lanes of the warp.
template <bool X32, int R>
__device__ __noinline__ uint32_t exact_scale(const NormArgs* a, size_t row, int c, uint32_t top) {
    const int e = (int)(top >> 23);  // the border in this octave is 1.75 2^(e - 127)
    return (uint32_t)max(e - (over_border<X32, R>(*a, row, c, rstd_64<X32, R, true>(*a, row), scalbn(1.75, e - 127)) ? 7 : 8), 1);
}
__device__ __forceinline__ bool near_border(uint32_t top) { return top != 0 && abs((int)(top & 0x7fffffu) - 0x600000) <= 24; }

// A row whose squares leave fp32's range (or are none), by the whole CTA: all of it in 64 bits, but for the sum, which is stored already.
template <bool X32, int R, int N, bool V>
__device__ __noinline__ void wide_row(const NormArgs* p, int64_t t) {
    const NormArgs& a = *p;
    const size_t row = (size_t)t * a.C;
    const int lead = V ? 0 : row % 8;
    const double rstd = rstd_64<X32, R, V>(a, row);
    if (threadIdx.x == 0 && a.rstd) a.rstd[t] = (float)rstd;
#pragma unroll 1
    for (int i = 0; i < N; i++) {
        const int c = norm_col(i, lead);
        float h[8], w[8], y[8];
        sum8<X32, R, V>(a, row, c, h);
        weight8<V>(a, c, w);
#pragma unroll
        for (int k = 0; k < 8; k++) y[k] = (float)((double)h[k] * rstd * (double)w[k]);
        if (a.y) store8<V>(a.y, a.y_f32, row, c, a.C, y);
        if (V && a.q) {
            bool special;
            uint32_t top = f8_top(y, special);
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
            uint32_t se = f8_scale_exp(top);
            const bool near = near_border(top);
            if (__any_sync(0xffffffffu, near)) {
                const int e = (int)(top >> 23);
                const bool over = over_border<X32, R>(a, row, c, rstd, scalbn(1.75, e - 127));
                if (near) se = (uint32_t)max(e - (over ? 7 : 8), 1);
            }
            if (c < a.C) *reinterpret_cast<uint2*>(a.q + row + c) = f8_pack8(y, f8_inverse(se), special);
            if (c < a.C && (threadIdx.x & 15) == 0) a.scale[t * ((a.C + kF8Block - 1) / kF8Block) + c / kF8Block] = __uint_as_float(se << 23);
        }
    }
}

// R: the residual is none (0), bf16 (1) or fp32 (2).
template <bool X32, int R, bool Q, int N, bool V, int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS != 256 ? 1 : N == 1 && !X32 && R != 2 ? 3 : 2) add_norm_kernel(const __grid_constant__ NormArgs a, float tiny) {
    __shared__ float part[2][32];
    constexpr bool kAhead = THREADS <= kNormThreads;
    griddep_wait();
    const int C = a.C, lead = V ? 0 : (int)((int64_t)blockIdx.x * C % 8), groups = (C + kF8Block - 1) / kF8Block;
    float w[N][8];
#pragma unroll
    for (int i = 0; i < N; i++) weight8<V>(a, norm_col(i, lead), w[i]);
    const size_t end = (size_t)a.T * C;
    Raw8<X32> x[N];
    Raw8<R == 2> res[N];
    auto ask = [&](int64_t t) {
#pragma unroll
        for (int i = 0; i < N; i++) {
            x[i].template load<V>(a.x, (size_t)t * C, norm_col(i, lead), C, end);
            if (R) res[i].template load<V>(a.residual, (size_t)t * C, norm_col(i, lead), C, end);
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
            keep_row<V>(h[i], norm_col(i, lead), C);
#pragma unroll
            for (int k = 0; k < 8; k++) ss = fmaf(h[i][k], h[i][k], ss);
        }
        if (kAhead && t + gridDim.x < a.T) ask(t + gridDim.x);
        if (R)
#pragma unroll
            for (int i = 0; i < N; i++) store8<V>(a.sum, R == 2, row, norm_col(i, lead), C, h[i]);
        ss = cta_sum(ss, part, turn);
        if (!(ss < 1e37f) || ss < tiny) {  // the whole CTA
            wide_row<X32, R, N, V>(&a, t);
            continue;
        }
        const float rstd = rsqrtf(ss / C + a.eps);
        if (threadIdx.x == 0 && a.rstd) a.rstd[t] = rstd;
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int c = norm_col(i, lead);
            float y[8];
#pragma unroll
            for (int k = 0; k < 8; k++) y[k] = h[i][k] * rstd * w[i][k];
            if (a.y) store8<V>(a.y, a.y_f32, row, c, C, y);
            if (Q) {
                bool special;
                uint32_t top = f8_top(y, special);
#pragma unroll
                for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
                uint32_t se = f8_scale_exp(top);
                const bool near = near_border(top);
                if (__any_sync(0xffffffffu, near)) {
                    const uint32_t exact = exact_scale<X32, R>(&a, row, c, top);
                    if (near) se = exact;
                }
                if (c < C) *reinterpret_cast<uint2*>(a.q + row + c) = f8_pack8(y, f8_inverse(se), special);
                if (c < C && (threadIdx.x & 15) == 0) a.scale[t * groups + c / kF8Block] = __uint_as_float(se << 23);
            }
        }
    }
}

template <bool X32, int R, bool Q>
static cudaError_t add_norm_for(const NormArgs& a, int sm_count, cudaStream_t st) {
    // Squares below fp32's range count for nothing beside eps, unless eps is of that kind itself.
    const float tiny = a.eps < 1e-18f ? 1e-24f : 0.f;
    // A row on twice the threads where there are no more rows than SMs (4096 columns, one row: 2.4 instead of 2.8 us; 16384 rows: 113
    // instead of 89).  CTAs for as many rows as fit on the SMs at once, the next row's words asked for ahead: a CTA a row without that
    // took 106 us, three CTAs of 80 registers 141 (spills).
    const int eights = a.T <= sm_count && a.C <= 4096 ? 1 : norm_eights(a.C), threads = norm_threads(a.C, eights);
    const int grid = norm_grid(a.T, sm_count * std::max(1, (eights == 1 && threads <= 256 && !X32 && R != 2 ? 768 : 512) / threads), a.C);
    const Launch l{grid, threads, 0, 0, st};
    if constexpr (!Q)
        if (a.C % 8) {
            if (threads > 512) return l.run(eights == 3 ? add_norm_kernel<X32, R, false, 3, false, 1024> : add_norm_kernel<X32, R, false, 2, false, 1024>, a, tiny);
            if (eights == 1) return l.run(threads > 256 ? add_norm_kernel<X32, R, false, 1, false, 512> : add_norm_kernel<X32, R, false, 1, false, 256>, a, tiny);
            return l.run(threads > 256 ? add_norm_kernel<X32, R, false, 2, false, 512> : add_norm_kernel<X32, R, false, 2, false, 256>, a, tiny);
        }
    if (threads > 512) return l.run(add_norm_kernel<X32, R, Q, 2, true, 1024>, a, tiny);
    if (eights == 1) return l.run(threads > 256 ? add_norm_kernel<X32, R, Q, 1, true, 512> : add_norm_kernel<X32, R, Q, 1, true, 256>, a, tiny);
    return l.run(threads > 256 ? add_norm_kernel<X32, R, Q, 2, true, 512> : add_norm_kernel<X32, R, Q, 2, true, 256>, a, tiny);
}
template <bool X32, int R>
static cudaError_t add_norm_of(const NormArgs& a, int sm_count, cudaStream_t st) {
    return a.q ? add_norm_for<X32, R, true>(a, sm_count, st) : add_norm_for<X32, R, false>(a, sm_count, st);
}

cudaError_t launch_add_norm(const NormArgs& a, int sm_count, cudaStream_t st) {
    if (a.T <= 0 || a.C <= 0) return cudaSuccess;
    const int r = !a.residual ? 0 : a.stream_f32 ? 2 : 1;
    if (a.x_f32) return r == 0 ? add_norm_of<true, 0>(a, sm_count, st) : r == 1 ? add_norm_of<true, 1>(a, sm_count, st) : add_norm_of<true, 2>(a, sm_count, st);
    return r == 0 ? add_norm_of<false, 0>(a, sm_count, st) : r == 1 ? add_norm_of<false, 1>(a, sm_count, st) : add_norm_of<false, 2>(a, sm_count, st);
}

}  // namespace moe
