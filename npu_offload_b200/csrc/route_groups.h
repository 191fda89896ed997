// Routing limited to the best groups of experts, and the gradient of routing weights: launch interface.
#pragma once
#include <cstdint>
#include <cuda_runtime.h>

namespace moe {

constexpr int kRouteMaxGroups = 32;

struct RouteGroupsArgs {
    const float* logits;  // [T, E]
    const float* bias;    // [E] or null (sigmoid scoring)
    int64_t T;
    int E, K, scoring;    // scoring: 0 softmax, 1 sigmoid
    int groups, top;      // groups of E / groups neighbours; the best `top` of them are open
    bool renormalize;
    float scale;
    int32_t* idx;         // [T, K]
    float* w;             // [T, K]
    uint32_t* err;
};
cudaError_t launch_route_groups(const RouteGroupsArgs& a, int sm_count, cudaStream_t st);

struct RouteBackwardArgs {
    const float* logits;  // [T, E]
    const int32_t* idx;   // [T, K]; negative: no choice
    const float* dw;      // [T, K]
    int64_t T;
    int E, K, scoring;
    bool renormalize, accumulate;
    float scale;
    float* dlogits;       // [T, E]
    uint32_t* err;
};
cudaError_t launch_route_backward(const RouteBackwardArgs& a, int sm_count, cudaStream_t st);

}  // namespace moe
