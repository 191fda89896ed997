// Low-rank adapters of many requests beside a shared projection: launch interface.
#pragma once
#include <cstddef>
#include <cstdint>
#include <cuda_runtime.h>

namespace moe {

struct LoraArgs {
    const void* base;       // [T, N] of out's type; may be out itself
    const uint16_t* x;      // [T, K] bf16
    const uint16_t* a;      // [n, r, K] bf16
    const uint16_t* b;      // [n, N, r] bf16
    const int32_t* ids;     // [T] adapter of each token; negative: none
    const float* scale;     // [n] or null: 1
    int T, K, N, r, n;      // K and r multiples of 8, r <= kLoraMaxRank
    void* out;              // [T, N] bf16, or fp32 (out_f32)
    bool out_f32;
    void* ws;               // lora_workspace bytes, 256-byte aligned
    uint32_t* err;
};
size_t lora_workspace(int T, int n, int r);
size_t lora_many_workspace(int T, int n, int r);
cudaError_t launch_lora_many(const LoraArgs& a, int sm_count, cudaStream_t st, int* launches);  // three kernels, any T
cudaError_t launch_add_lora(const LoraArgs& a, int sm_count, cudaStream_t st, int* launches);

}  // namespace moe
