// Router load-balance loss: launch interface.
#pragma once
#include <cstddef>
#include <cstdint>
#include <cuda_runtime.h>

namespace moe {

struct BalanceArgs {
    const float* logits;     // [T, E]
    const int32_t* idx;      // [T, K] chosen experts; negative: no choice
    const int32_t* offsets;  // [B + 1] first token of each sequence, or null: one sequence of all T
    const uint8_t* mask;     // [T] nonzero: the token counts; null: all do
    int T, E, K, B, scoring;
    int32_t* counts;         // [B, E]
    int32_t* tokens;         // [B + 1] tokens that count per sequence; [B] = sequences with any
    float* loss;             // [1]
    const float* grad;       // backward: [1] gradient of the loss, or null: 1
    float* dlogits;          // backward: [T, E]
    void* ws;                // forward: balance_workspace bytes, 256-byte aligned
    uint32_t* err;
};

size_t balance_workspace(int T, int E, int B, int sm_count);
cudaError_t launch_balance_loss(const BalanceArgs& a, int sm_count, cudaStream_t st);      // two kernels
cudaError_t launch_balance_backward(const BalanceArgs& a, int sm_count, cudaStream_t st);  // one kernel

}  // namespace moe
