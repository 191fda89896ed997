// What the norm's forward and backward kernels share: eight values of a row a thread, and sums over a CTA.
#pragma once
#include <cstdint>

#include "common.cuh"
#include "fp8.cuh"
#include "fp8.h"
#include "ptx.cuh"

namespace moe {

// Eight values as they come from memory.  V: neighbours at a 16-byte boundary; else one of every `step`, so that a warp's
// loads are of neighbours where rows are not aligned.
template <bool F32>
struct Raw8 {
    uint4 a, b;  // (b: fp32 alone)
    template <bool V>
    __device__ __forceinline__ void load(const void* p, size_t row, int c, int step, int C) {
        if constexpr (V) {
            if (c < C) {
                if (F32) {
                    a = ld_cg_u4(static_cast<const float*>(p) + row + c);
                    b = ld_cg_u4(static_cast<const float*>(p) + row + c + 4);
                } else {
                    a = ld_cg_u4(static_cast<const uint16_t*>(p) + row + c);
                }
            } else {
                a = b = make_uint4(0, 0, 0, 0);
            }
        } else {
            uint32_t w[8];
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const int i = c + k * step;
                w[k] = 0;
                if (i < C) w[k] = F32 ? static_cast<const uint32_t*>(p)[row + i] : static_cast<const uint16_t*>(p)[row + i];
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

// Eight floats into a row, as fp32 or rounded to bf16; where they lie as in Raw8::load.
template <bool V>
__device__ __forceinline__ void store8(void* p, bool f32, size_t row, int c, int step, int C, const float (&f)[8]) {
    if constexpr (V) {
        if (c >= C) return;
        if (f32) {
            float4* o = reinterpret_cast<float4*>(static_cast<float*>(p) + row + c);
            o[0] = make_float4(f[0], f[1], f[2], f[3]);
            o[1] = make_float4(f[4], f[5], f[6], f[7]);
        } else {
            *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + row + c) =
                make_uint4(f8_bf16x2(f[0], f[1]), f8_bf16x2(f[2], f[3]), f8_bf16x2(f[4], f[5]), f8_bf16x2(f[6], f[7]));
        }
    } else {
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const int i = c + k * step;
            if (i < C) {
                if (f32) static_cast<float*>(p)[row + i] = f[k];
                else static_cast<uint16_t*>(p)[row + i] = f8_bf16(f[k]);
            }
        }
    }
}

// Column of value 0 of a thread's i-th eight, and the step between its values.
template <bool V>
__device__ __forceinline__ int norm_col(int i) {
    return V ? (int)(threadIdx.x + i * blockDim.x) * 8 : (int)(threadIdx.x + i * 8 * blockDim.x);
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

// How a row of C <= 16384 columns is spread: eights a thread (1 or 2), and threads of a CTA.  Rows of more than 8192 columns
// take 1024 threads; with the 64 registers that such a CTA leaves each, the next row's words are not asked for ahead.
inline int norm_eights(int C) { return C <= 2048 ? 1 : 2; }
inline int norm_threads(int C, int eights) {
    const int n = ((C + 7) / 8 + eights - 1) / eights;
    return (n + 31) / 32 * 32;
}
constexpr int kNormThreads = 512;
// CTAs for T rows where `most` fit at once: no more than the longest of them needs.
inline int norm_grid(int64_t T, int64_t most) {
    const int64_t rows = (T + most - 1) / most;
    return (int)((T + rows - 1) / rows);
}

}  // namespace moe
