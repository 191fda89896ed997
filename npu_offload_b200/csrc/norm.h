// Residual addition with root-mean-square norm, and its gradients: launch interface.
#pragma once
#include <cstddef>
#include <cstdint>
#include <cuda_runtime.h>

namespace moe {

struct NormArgs {
    const void* x;         // [T, C] bf16, or fp32 (x_f32)
    const void* residual;  // [T, C] bf16, or fp32 (stream_f32); null: the sum is x
    const void* weight;    // [C] bf16, or fp32 (weight_f32)
    bool x_f32, stream_f32, weight_f32, y_f32;
    int64_t T;
    int C;
    float eps;
    void* sum;             // [T, C] of the residual's type; null without a residual
    void* y;               // [T, C] bf16, or fp32 (y_f32), or null
    uint8_t* q;            // [T, C] e4m3, or null; C % 16 == 0
    float* scale;          // [T, ceil(C / 128)], with q
    float* rstd;           // [T], or null
};
cudaError_t launch_add_norm(const NormArgs& a, int sm_count, cudaStream_t st);

struct NormBackwardArgs {
    const void* dy;      // [T, C] bf16, or fp32 (dy_f32)
    const void* sum;     // [T, C] bf16, or fp32 (stream_f32)
    const void* dsum;    // [T, C] of sum's type, or null
    const void* weight;  // [C] bf16, or fp32 (weight_f32)
    const float* rstd;   // [T]
    bool dy_f32, stream_f32, weight_f32;
    int64_t T;
    int C;
    void* dx;            // [T, C] of sum's type
    float* dweight;      // [C], or null
    float* ws;           // with dweight: norm_backward_workspace bytes, 256-byte aligned
};
size_t norm_backward_workspace(int64_t T, int C, int sm_count);
cudaError_t launch_add_norm_backward(const NormBackwardArgs& a, int sm_count, cudaStream_t st, int* launches);

}  // namespace moe
