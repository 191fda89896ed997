// Launch interface of the 8-bit floating-point (e4m3) kernels: quantiser, scaled product, expert FFN.
//
// An e4m3 operand is a row-major byte matrix with an fp32 scale for each 128 columns of a row
// (activations) or each 128 x 128 block (weights); the last block of a row or column may be partial.
#pragma once
#include <cstddef>
#include <cstdint>
#include <cuda_runtime.h>

namespace moe {

constexpr int kF8Block = 128;

// q[i] = e4m3(x[i] / s), s = the smallest power of two (>= 2^-126) with max|x| <= 448 s over the
// group: 128 columns of block_rows rows (1 or 128) of one of `batch` matrices [rows, cols].
// x: bf16 or (f32) fp32.  cols % 16 == 0, x 16-byte and q 8-byte aligned.
cudaError_t launch_quantize_fp8(const void* x, bool f32, int64_t batch, int64_t rows, int64_t cols, int block_rows,
                                uint8_t* q, float* s, int sm_count, cudaStream_t st);

struct MatmulF8 {
    const uint8_t* x;  // [M, K] e4m3, 16-byte aligned
    const float* xs;   // [M, ceil(K / 128)]
    const uint8_t* w;  // [N, K] e4m3, 16-byte aligned
    const float* ws;   // [ceil(N / 128), ceil(K / 128)]
    int64_t M, N;
    int K;             // multiple of 16
    void* out;         // [M, N] bf16, or fp32 (out_f32)
    bool out_f32;
    uint32_t* err;
    uint64_t timeout_ns;
    int inject;        // test hook (MOE_OPT_INJECT_WAIT_TIMEOUT)
};
cudaError_t launch_matmul_fp8(const MatmulF8& a, int sm_count, cudaStream_t st);

// The routed-expert FFN: tokens quantised, gate / up product, SwiGLU, activations quantised, down
// product, weighted sum over each token's experts.
struct ExpertsF8 {
    const uint16_t* x;           // [T, H] bf16
    const uint8_t* gu;           // [E, 2, F, H] e4m3: gate rows, up rows
    const float* gus;            // [E, 2, ceil(F / 128), ceil(H / 128)]
    const uint8_t* d;            // [E, H, F] e4m3
    const float* ds;             // [E, ceil(H / 128), ceil(F / 128)]
    const int32_t* idx;          // [T, K] experts; negative: no expert
    const float* w;              // [T, K]
    int T, H, F, E, K;
    void* out;                   // [T, H] bf16, or fp32 (out_f32)
    bool out_f32, accumulate;    // accumulate: fp32 only
    void* ws;                    // experts_fp8_workspace bytes, 256-byte aligned
    uint32_t* err;
    uint64_t timeout_ns;
    int inject;                  // test hook (MOE_OPT_INJECT_WAIT_TIMEOUT)
};
size_t experts_fp8_workspace(int T, int K, int H, int F, int E);
cudaError_t launch_experts_fp8(const ExpertsF8& a, int sm_count, cudaStream_t st, int* launches);

}  // namespace moe
