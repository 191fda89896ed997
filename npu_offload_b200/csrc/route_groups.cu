// Routing limited to the best groups of experts, and the gradient of the routing weights.
//
//   key   softmax: the logit;  sigmoid: fp32(s + bias), s = 1 / (1 + exp(-l)), each step rounded as the other router
//         kernels round it (route_core.cuh)
//   group score   softmax: its largest key;  sigmoid: the fp32 sum of its two largest (of the one, where it has one)
//   the best `top` groups (ties to the lower), in them the best K experts by key (ties to the lower), in that order
//   w = scale v, or scale v / sum of the chosen v;  v: the softmax probability, or s
//
// A warp a token.  A group's experts lie on neighbouring lanes, V to a lane, so that a group's score is a matter of a few
// shuffles and a lower lane means a lower index.  The sequence of K maxima runs on 32-bit words: the key's bits in order,
// its last log2 V bits given up for the place within the lane, sorted once in each lane; then a maximum over the warp
// (one instruction) and a shift in the lane that held it, for each choice.  A sigmoid's key is formed with the hardware's 2^x and
// reciprocal for that.
// Such words decide wherever neighbours in the sequence, and the last open and first closed group, lie further apart than
// what was given up; the margins are stated below.  A token with a closer pair is done again with the keys themselves (the exponential in
// double, 64-bit words of key and index): the result is always that of the definition.
#include <algorithm>

#include "common.cuh"
#include "launch.cuh"
#include "ptx.cuh"
#include "route_core.cuh"
#include "route_groups.h"

namespace moe {

constexpr int kRouteWarps = 8;

// How a token's experts lie on a warp: group g on lanes g P .. g P + P - 1, `each` neighbours to a lane.
struct RouteSpread {
    int size;    // experts of a group
    int shift;   // log2 P
    int each;    // ceil(size / P), at most V
};

__device__ __forceinline__ float from_ordered(uint32_t u) { return __uint_as_float((u & 0x80000000u) ? u & 0x7fffffffu : ~u); }
__device__ __forceinline__ float exp2_hw(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp_hw(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// The bits of a key in order: NaN as -inf, -0 as 0.
__device__ __forceinline__ uint32_t key_bits(float k) { return ordered_bits(k != k ? -INFINITY : k + 0.f); }
__device__ __forceinline__ float group_sum(float a, float b) {
    const float s = a + b;
    return s != s ? -INFINITY : s;
}

// Words in falling order (odd-even merge sort).
template <int V>
__device__ __forceinline__ void sort_falling(uint32_t (&u)[V]) {
#pragma unroll
    for (int p = 1; p < V; p *= 2)
#pragma unroll
        for (int k = p; k >= 1; k /= 2)
#pragma unroll
            for (int j = k % p; j + k < V; j += 2 * k)
#pragma unroll
                for (int i = 0; i < k; i++)
                    if (i + j + k < V && (i + j) / (2 * p) == (i + j + k) / (2 * p)) {
                        const uint32_t a = u[i + j], b = u[i + j + k];
                        u[i + j] = max(a, b), u[i + j + k] = min(a, b);
                    }
}

__device__ __forceinline__ unsigned long long warp_max64(unsigned long long v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// The choices of one token by the definition, one warp: expert k on lane k < K.
template <int V, bool SIG>
__device__ __noinline__ int choose_exactly(const float* row, const float* bias, int K, int groups, int top, RouteSpread sp) {
    const int lane = threadIdx.x & 31, P = 1 << sp.shift, g = lane >> sp.shift, m0 = (lane & (P - 1)) * sp.each;
    const int n = g < groups ? min(max(sp.size - m0, 0), sp.each) : 0, e0 = g * sp.size + m0;
    unsigned long long key[V];
    uint32_t a = 0, b = 0;  // the two largest of the group
    for (int j = 0; j < V; j++) {
        key[j] = 0;
        if (j < n) {
            float k = row[e0 + j];
            if (SIG) k = __fdiv_rn(1.0f, 1.0f + router_exp(-k)) + (bias ? bias[e0 + j] : 0.f);
            const uint32_t o = key_bits(k);
            key[j] = (unsigned long long)o << 32 | (uint32_t)~(e0 + j);
            b = max(b, min(a, o)), a = max(a, o);
        }
    }
    for (int o = 1; o < P; o <<= 1) {
        const uint32_t c = __shfl_xor_sync(0xffffffffu, a, o), d = __shfl_xor_sync(0xffffffffu, b, o);
        b = max(min(a, c), max(b, d)), a = max(a, c);
    }
    const uint32_t score = !SIG || b == 0 ? a : ordered_bits(group_sum(from_ordered(a), from_ordered(b)) + 0.f);
    unsigned long long mine = g < groups ? (unsigned long long)score << 32 | (uint32_t)~g : 0;
    bool open = false;
    for (int i = 0; i < top; i++)
        if (warp_max64(mine) == mine && mine) open = true, mine = 0;
    int chosen = 0;
    for (int k = 0; k < K; k++) {
        unsigned long long best = 0;
        for (int j = 0; j < V; j++) best = max(best, open ? key[j] : 0ull);
        best = warp_max64(best);
        if (lane == k) chosen = (int)~(uint32_t)best;
        for (int j = 0; j < V; j++)
            if (key[j] == best) key[j] = 0;
    }
    return chosen;
}

// Margins.  A word's key is short by less than 2^-23 V of it (V <= 16: 2^-19).  The sigmoid's hardware steps: the product l log2 e is off by
// |l| 2^-24 / ln 2 in the exponent, 2^x and the reciprocal by 2^-22 each, the additions by 2^-24, so s by
// s (|l| 2^-24 + 2^-21) at most; with s <= smax, and smax > 2^-20 (else the token is done exactly), s |l| <= 14 smax, so that
// s is off by smax 2^-19.9 < smax 2^-19, and the two keys' difference by that twice plus 2^-23 of each for rounding.
// Neighbours: 2 smax 2^-19 + (2^-19 + 2^-22) (|a| + |b|) < (smax + |a| + |b|) 2^-18.  Groups: two keys a score, so
// 4 smax 2^-19 + 4 k 2^-18.8 + 2 k 2^-22, k the largest |key| of any group's two best, < (smax + 4 k) 2^-17.
template <int V, bool SIG>
__global__ void __launch_bounds__(kRouteWarps * 32) route_groups_kernel(RouteGroupsArgs a, RouteSpread sp, bool vec) {
    griddep_wait();
    constexpr uint32_t kPlace = V - 1;
    const int lane = threadIdx.x & 31, P = 1 << sp.shift, g = lane >> sp.shift, m0 = (lane & (P - 1)) * sp.each;
    const int n = g < a.groups ? min(max(sp.size - m0, 0), sp.each) : 0, e0 = g * sp.size + m0, E = a.E, K = a.K;
    float bias[SIG ? V : 1];
    if (SIG)
#pragma unroll
        for (int j = 0; j < V; j++) bias[j] = a.bias && j < n ? a.bias[e0 + j] : 0.f;
    for (int64_t t = (int64_t)blockIdx.x * kRouteWarps + (threadIdx.x >> 5); t < a.T; t += (int64_t)gridDim.x * kRouteWarps) {
        const float* row = a.logits + t * E;
        float l[V];
        if (V >= 4 && vec) {
#pragma unroll
            for (int j = 0; j < V; j += 4)
                if (j < n) {
                    const float4 q = *reinterpret_cast<const float4*>(row + e0 + j);
                    l[j] = q.x, l[(j + 1) % V] = q.y, l[(j + 2) % V] = q.z, l[(j + 3) % V] = q.w;
                }
        } else {
#pragma unroll
            for (int j = 0; j < V; j++)
                if (j < n) l[j] = row[e0 + j];
        }
        bool bad = false;
        uint32_t u[V], smax = 0;
#pragma unroll
        for (int j = 0; j < V; j++) {
            u[j] = 0;
            if (j < n) {
                float k = l[j];
                if (SIG) {
                    const float s = rcp_hw(1.f + exp2_hw(k * -1.44269504f));
                    smax = max(smax, s == s ? __float_as_uint(s) : 0u);
                    k = s + bias[j];
                }
                bad |= k != k;
                u[j] = (key_bits(k) & ~kPlace) | (kPlace - j);
            }
        }
        sort_falling(u);
        bool near = false;
        if (SIG) {
            smax = __reduce_max_sync(0xffffffffu, smax);
            near = smax <= __float_as_uint(0x1p-20f);
        }
        const float sm = __uint_as_float(smax);
        if (a.top < a.groups) {
            uint32_t score = u[0] & ~kPlace, second = V > 1 ? u[V > 1 ? 1 : 0] & ~kPlace : 0;
            for (int o = 1; o < P; o <<= 1) {
                const uint32_t c = __shfl_xor_sync(0xffffffffu, score, o);
                if (SIG) second = max(min(score, c), max(second, __shfl_xor_sync(0xffffffffu, second, o)));
                score = max(score, c);
            }
            float kmax = 0.f;
            if (SIG && g < a.groups) {
                const float x = from_ordered(score), y = second ? from_ordered(second) : 0.f;
                kmax = fmaxf(fabsf(x), fabsf(y));
                score = ordered_bits(second ? group_sum(x, y) : x);
            }
            if (g >= a.groups) score = 0;
            if (SIG) kmax = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(kmax)));
            bool open = false;
            uint32_t last = 0;
            for (int i = 0; i < a.top; i++) {
                last = __reduce_max_sync(0xffffffffu, score);
                const int owner = __ffs(__ballot_sync(0xffffffffu, score == last)) - 1;
                if (g == owner >> sp.shift) open = true, score = 0;
            }
            const uint32_t next = __reduce_max_sync(0xffffffffu, score);
            if (SIG) near |= !(from_ordered(last) - from_ordered(next) > (sm + 4.f * kmax) * 0x1p-17f);
            else near |= last == next;
            if (!open)
#pragma unroll
                for (int j = 0; j < V; j++) u[j] = 0;
        }
        uint32_t word = 0;
        int e = 0;
        for (int k = 0; k <= K; k++) {
            const uint32_t top = __reduce_max_sync(0xffffffffu, u[0]);
            const int owner = __ffs(__ballot_sync(0xffffffffu, u[0] == top)) - 1;
            if (lane == k) {
                word = top;
                e = (owner >> sp.shift) * sp.size + (owner & (P - 1)) * sp.each + (int)(kPlace - (top & kPlace));
            }
            if (lane == owner) {
#pragma unroll
                for (int j = 0; j + 1 < V; j++) u[j] = u[j + 1];
                u[V - 1] = 0;
            }
        }
        const uint32_t after = __shfl_down_sync(0xffffffffu, word, 1);
        if (lane < K && after) {
            if (SIG) {
                const float x = from_ordered(word & ~kPlace), y = from_ordered(after & ~kPlace);
                near |= !(x - y > (sm + fabsf(x) + fabsf(y)) * 0x1p-18f);
            } else {
                near |= (word & ~kPlace) == (after & ~kPlace);
            }
        }
        if (__any_sync(0xffffffffu, near)) e = choose_exactly<V, SIG>(row, a.bias, K, a.groups, a.top, sp);
        bad = __any_sync(0xffffffffu, bad);
        float v = 0.f;
        if (SIG) {
            if (lane < K) v = __fdiv_rn(1.f, 1.f + expf(-row[e]));
        } else {
            const float mine = lane < K ? row[e] : -INFINITY, most = __shfl_sync(0xffffffffu, mine, 0);
            bad |= !(fabsf(most) < INFINITY);
            v = expf(mine - most);
            if (!a.renormalize) {  // the largest of all is the first chosen
                float z = 0.f;
#pragma unroll
                for (int j = 0; j < V; j++)
                    if (j < n) z += exp2_hw((l[j] - most) * 1.44269504f);
                v = __fdiv_rn(v, warp_sum(z));
            }
        }
        if (a.renormalize) v = __fdiv_rn(v, warp_sum(lane < K ? v : 0.f) + (SIG ? 1e-20f : 0.f));
        if (lane < K) {
            a.idx[t * K + lane] = e;
            a.w[t * K + lane] = bad ? __int_as_float(0x7fffffff) : v * a.scale;
        }
        if (bad && lane == 0) atomicOr(a.err, kErrNonFinite);
    }
}

cudaError_t launch_route_groups(const RouteGroupsArgs& a, int sm_count, cudaStream_t st) {
    if (a.T <= 0) return cudaSuccess;
    RouteSpread sp;
    sp.size = a.E / a.groups;
    for (sp.shift = 5; a.groups << sp.shift > 32; sp.shift--) {}
    sp.each = (sp.size + (1 << sp.shift) - 1) >> sp.shift;
    const bool vec = sp.each % 4 == 0 && sp.size % 4 == 0 && (uintptr_t)a.logits % 16 == 0;  // (a lane has a multiple of four, then)
    const int64_t blocks = (a.T + kRouteWarps - 1) / kRouteWarps;
    const Launch l{(int)std::min<int64_t>(blocks, (int64_t)sm_count * 8), kRouteWarps * 32, 0, 0, st};
    const bool sig = a.scoring != 0;
#define ROUTE_GROUPS(V)                                                                    \
    if (sp.each <= V) return sig ? l.run(route_groups_kernel<V, true>, a, sp, vec) : l.run(route_groups_kernel<V, false>, a, sp, vec)
    ROUTE_GROUPS(1);
    ROUTE_GROUPS(2);
    ROUTE_GROUPS(4);
    ROUTE_GROUPS(8);
    ROUTE_GROUPS(16);
#undef ROUTE_GROUPS
    return cudaErrorInvalidValue;
}

// ---------------------------------------------------------------- gradient
//
// g_k = scale dL/dw_k, v as above, W the sum of the chosen v:
//   dL/dv_k = (g_k - sum_j g_j v_j / W) / W, or g_k where weights are not renormalised
//   softmax: dL/dl_e = v_e (dL/dv_e - sum_j dL/dv_j v_j);   sigmoid: dL/dl_e = dL/dv_e s_e (1 - s_e)
// Where weights are renormalised, or sigmoids, the chosen experts alone have a gradient and only their logits are read:
// p = v / W gives (softmax) p_k (g_k - sum g p), (sigmoid) (1 - s_k) p_k (g_k - sum g p), g_k s_k (1 - s_k) without.
// A warp a token: the choices on lanes 0 to K - 1, their values put in place through a row in shared memory, which is
// then written as it lies.  Bounded by HBM: T E 4 bytes written, and read where the softmax needs its sum.
template <int V, bool DENSE>
__global__ void __launch_bounds__(kRouteWarps * 32) route_backward_kernel(RouteBackwardArgs a, bool vec) {
    __shared__ __align__(16) float rows[kRouteWarps][32 * V];
    griddep_wait();
    const int lane = threadIdx.x & 31, E = a.E, K = a.K;
    float* s_row = rows[threadIdx.x >> 5];
    for (int64_t t = (int64_t)blockIdx.x * kRouteWarps + (threadIdx.x >> 5); t < a.T; t += (int64_t)gridDim.x * kRouteWarps) {
        const float* row = a.logits + t * E;
        float* out = a.dlogits + t * E;
        int i = -1;
        float g = 0.f;
        if (lane < K) {
            i = a.idx[t * K + lane];
            g = a.dw[t * K + lane] * a.scale;
        }
        float l[V];
        if (DENSE) {
#pragma unroll
            for (int j = 0; j < V; j++) l[j] = lane + 32 * j < E ? row[lane + 32 * j] : -INFINITY;
        }
        if (i >= E) {
            atomicOr(a.err, kErrBadIndex);
            i = -1;
        }
        const bool in = i >= 0;
        float d = 0.f;  // what goes to expert i: dL/dl, or (DENSE) dL/dv
        float inv = 0.f, most = 0.f, dot = 0.f;
        if (DENSE) {
            most = l[0];
#pragma unroll
            for (int j = 1; j < V; j++) most = fmaxf(most, l[j]);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
            float z = 0.f;
#pragma unroll
            for (int j = 0; j < V; j++) {
                l[j] = exp2_hw((l[j] - most) * 1.44269504f);
                z += l[j];
            }
            inv = __fdiv_rn(1.f, warp_sum(z));
            d = in ? g : 0.f;
            dot = warp_sum(in ? g * (exp2_hw((row[i] - most) * 1.44269504f) * inv) : 0.f);
        } else if (a.scoring == 0) {
            const float x = in ? row[i] : -INFINITY;
            float m = x;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            const float v = in ? expf(x - m) : 0.f, total = warp_sum(v), p = in ? __fdiv_rn(v, total) : 0.f;
            d = p * (g - warp_sum(in ? g * p : 0.f));
        } else {
            // s and 1 - s from exp(-|l|), so that neither loses bits where the other is near 1
            const float x = in ? row[i] : 0.f, q = expf(-fabsf(x)), big = __fdiv_rn(1.f, 1.f + q), small = q * big;
            const float s = x >= 0.f ? big : small, rest = x >= 0.f ? small : big;
            if (a.renormalize) {
                const float total = warp_sum(in ? s : 0.f) + 1e-20f, p = in ? __fdiv_rn(s, total) : 0.f;
                d = rest * p * (g - warp_sum(in ? g * p : 0.f));
            } else {
                d = g * s * rest;
            }
        }
        if (!in) d = 0.f;
        // the same expert twice: its first lane takes the sum, in the choices' order
        const unsigned same = __match_any_sync(0xffffffffu, in ? i : -1 - lane);
        bool first = in;
        if (__any_sync(0xffffffffu, __popc(same) > 1)) {
            float sum = 0.f;
            for (int k = 0; k < K; k++) {
                const float dk = __shfl_sync(0xffffffffu, d, k);
                if (same >> k & 1) sum += dk;
            }
            if (in) d = sum;
            first = in && __ffs(same) - 1 == lane;
        }
        if (!DENSE && a.accumulate) {
            if (first) out[i] = __fadd_rn(out[i], d);  // (the gradient's own bits, added: not fused with its last product)
            continue;
        }
#pragma unroll
        for (int j = 0; j < V; j++) s_row[lane + 32 * j] = 0.f;
        __syncwarp();
        if (first) s_row[i] = d;
        __syncwarp();
        if (DENSE) {
#pragma unroll
            for (int j = 0; j < V; j++) {
                const int e = lane + 32 * j;
                if (e < E) {
                    const float v = l[j] * inv * (s_row[e] - dot);
                    out[e] = a.accumulate ? __fadd_rn(out[e], v) : v;
                }
            }
        } else if (V >= 4 && vec) {
            for (int e = lane * 4; e < E; e += 128) *reinterpret_cast<float4*>(out + e) = *reinterpret_cast<const float4*>(s_row + e);
        } else {
#pragma unroll
            for (int j = 0; j < V; j++)
                if (lane + 32 * j < E) out[lane + 32 * j] = s_row[lane + 32 * j];
        }
        __syncwarp();
    }
}

cudaError_t launch_route_backward(const RouteBackwardArgs& a, int sm_count, cudaStream_t st) {
    if (a.T <= 0) return cudaSuccess;
    const int64_t blocks = (a.T + kRouteWarps - 1) / kRouteWarps;
    const Launch l{(int)std::min<int64_t>(blocks, (int64_t)sm_count * 8), kRouteWarps * 32, 0, 0, st};
    const bool dense = a.scoring == 0 && !a.renormalize, vec = a.E % 4 == 0 && (uintptr_t)a.dlogits % 16 == 0;
#define ROUTE_BACKWARD(V) \
    if (a.E <= 32 * V) return dense ? l.run(route_backward_kernel<V, true>, a, vec) : l.run(route_backward_kernel<V, false>, a, vec)
    ROUTE_BACKWARD(1);
    ROUTE_BACKWARD(2);
    ROUTE_BACKWARD(4);
    ROUTE_BACKWARD(8);
#undef ROUTE_BACKWARD
    return cudaErrorInvalidValue;
}

}  // namespace moe
