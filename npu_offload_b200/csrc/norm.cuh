// What the norm's forward and backward kernels share: eight values of a row a thread, and sums over a CTA.
#pragma once
#include <cstdint>

#include "common.cuh"
#include "fp8.cuh"
#include "fp8.h"
#include "ptx.cuh"

namespace moe {

// Eight neighbouring values as they come from memory, from column c of the row that begins at value `row` on; row + c is a multiple of
// eight, so that every word of 16 bytes lies at its boundary.  V: rows are multiples of eight values, c is 0 or more.  Else c may be
// negative, and the first and last eight of a row hold values of its neighbours, for keep_row to take out (nothing waits for a word
// before it is used: put together from single values, the next row's words were waited for at once, 64 instead of 38 us at
// 4000 x 4099); the one word that may reach behind the tensor's end comes value by value.  0 where c is behind the row.
template <bool F32>
struct Raw8 {
    uint4 a, b;  // (b: fp32 alone)
    template <bool V>
    __device__ __forceinline__ void load(const void* p, size_t row, int c, int C, size_t end) {
        a = b = make_uint4(0, 0, 0, 0);
        if (c >= C) return;
        if (V || row + c + 8 <= end) {
            if (F32) {
                a = ld_cg_u4(static_cast<const float*>(p) + row + c);
                b = ld_cg_u4(static_cast<const float*>(p) + row + c + 4);
            } else {
                a = ld_cg_u4(static_cast<const uint16_t*>(p) + row + c);
            }
        } else {
            uint32_t w[8];
#pragma unroll
            for (int k = 0; k < 8; k++) {
                w[k] = 0;
                if (c + k >= 0 && c + k < C) w[k] = F32 ? static_cast<const uint32_t*>(p)[row + c + k] : static_cast<const uint16_t*>(p)[row + c + k];
            }
            if (F32) {
                a = make_uint4(w[0], w[1], w[2], w[3]);
                b = make_uint4(w[4], w[5], w[6], w[7]);
            } else {
                a = make_uint4(w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16);
            }
        }
    }
    __device__ __forceinline__ void get(float (&f)[8]) const {
        if (F32) {
            const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
            for (int k = 0; k < 8; k++) f[k] = __uint_as_float(w[k]);
        } else {
            const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
            for (int k = 0; k < 4; k++) f[2 * k] = bf_lo(w[k]), f[2 * k + 1] = bf_hi(w[k]);
        }
    }
};

// Values of other rows become 0.
template <bool V>
__device__ __forceinline__ void keep_row(float (&f)[8], int c, int C) {
    if (V || (c >= 0 && c + 8 <= C)) return;
#pragma unroll
    for (int k = 0; k < 8; k++)
        if (c + k < 0 || c + k >= C) f[k] = 0.f;
}

// Eight floats into a row, as fp32 or rounded to bf16; where they lie as in Raw8::load.
template <bool V>
__device__ __forceinline__ void store8(void* p, bool f32, size_t row, int c, int C, const float (&f)[8]) {
    if (V ? c < C : c >= 0 && c + 8 <= C) {
        if (f32) {
            float4* o = reinterpret_cast<float4*>(static_cast<float*>(p) + row + c);
            o[0] = make_float4(f[0], f[1], f[2], f[3]);
            o[1] = make_float4(f[4], f[5], f[6], f[7]);
        } else {
            *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + row + c) =
                make_uint4(f8_bf16x2(f[0], f[1]), f8_bf16x2(f[2], f[3]), f8_bf16x2(f[4], f[5]), f8_bf16x2(f[6], f[7]));
        }
    } else if (!V && c < C) {
#pragma unroll
        for (int k = 0; k < 8; k++)
            if (c + k >= 0 && c + k < C) {
                if (f32) static_cast<float*>(p)[row + c + k] = f[k];
                else static_cast<uint16_t*>(p)[row + c + k] = f8_bf16(f[k]);
            }
    }
}

// Column of value 0 of a thread's i-th eight, in a row that begins `lead` values behind a multiple of eight.  A CTA's rows
// all have the same lead (norm_grid), so that a thread's columns are the same in all of them.
__device__ __forceinline__ int norm_col(int i, int lead) { return (int)(threadIdx.x + i * blockDim.x) * 8 - lead; }

// Eight weights as floats.
template <bool V>
__device__ __forceinline__ void norm_weight(const void* weight, bool f32, int c, int C, float (&w)[8]) {
    // (row 0 of a tensor at a 16-byte boundary; c is a multiple of eight with V alone)
    if (V) {
        if (f32) {
            Raw8<true> r;
            r.template load<V>(weight, 0, c, C, C);
            r.get(w);
        } else {
            Raw8<false> r;
            r.template load<V>(weight, 0, c, C, C);
            r.get(w);
        }
    } else {
#pragma unroll
        for (int k = 0; k < 8; k++) {
            w[k] = 0.f;
            if (c + k >= 0 && c + k < C) w[k] = f32 ? static_cast<const float*>(weight)[c + k] : bf2f(static_cast<const uint16_t*>(weight)[c + k]);
        }
    }
}

// v summed over the CTA, the same bits on every thread.  part: two sets of 32, used in turn by rows, so that one barrier a
// row is enough: a thread writes a set again two rows later, behind a barrier that every thread reaches after its reads.
__device__ __forceinline__ float cta_sum(float v, float (*part)[32], int turn) {
    v = warp_sum(v);
    const int warps = blockDim.x >> 5;
    if (warps == 1) return v;
    if ((threadIdx.x & 31) == 0) part[turn & 1][threadIdx.x >> 5] = v;
    __syncthreads();
    const int lane = threadIdx.x & 31;
    return warp_sum(lane < warps ? part[turn & 1][lane] : 0.f);
}

// How a row of C <= 16384 columns is spread: eights a thread (1 or 2; 3 where a lead makes it 2049 words), and threads of a CTA.  Rows of more than 8192 columns
// take 1024 threads; with the 64 registers that such a CTA leaves each, the next row's words are not asked for ahead.
inline int norm_words(int C) { return C % 8 ? (C + 14) / 8 : C / 8; }  // (of a row of any lead)
inline int norm_eights(int C) { return C <= 2048 ? 1 : norm_words(C) <= 2048 ? 2 : 3; }
inline int norm_threads(int C, int eights) {
    const int n = (norm_words(C) + eights - 1) / eights;
    return (n + 31) / 32 * 32;
}
constexpr int kNormThreads = 512;
// CTAs for T rows where `most` fit at once: no more than the longest of them needs.  A CTA takes every grid-th row: where it has
// several, and rows are no multiples of eight values, as many CTAs as make them begin alike, and no more than fit all the same (152 where 148
// fit ran four of them behind all others, 16384 x 2047 189 us instead of 107, 8192 x 5121 137 instead of 80).
inline int norm_grid(int64_t T, int64_t most, int C) {
    if (T <= most) return (int)T;
    const int period = C % 8 == 0 ? 1 : C % 4 == 0 ? 2 : C % 2 == 0 ? 4 : 8;
    const int64_t fit = most >= period ? most / period * period : period, rows = (T + fit - 1) / fit, grid = (T + rows - 1) / rows;
    return (int)((grid + period - 1) / period * period);
}

}  // namespace moe
