// Load-balance loss of a router and its gradient.
//
// Sequence b holds n_b tokens that count.  With c_be the pairs (token, choice) of the sequence on
// expert e and p_t the token's scores over all experts (softmax, or sigmoid s divided by
// S = sum s + 1e-20):
//   f_be = E c_be / (K n_b)      P_be = (1 / n_b) sum_t p_te      L = 1/B' sum_b sum_e f_be P_be
// over the B' sequences with n_b > 0.  The counts are constants, so
//   softmax:  dL/dl_te = 1/(B' n_b) p_te (f_be - sum_j f_bj p_tj)
//   sigmoid:  dL/dl_te = 1/(B' n_b) s_te (1 - s_te) / S (f_be - sum_j f_bj p_tj)
// Nothing is kept of the scores: the backward pass computes them again from the logits, which costs
// the same read as keeping them would.  Both passes are bounded by HBM: T E 4 bytes read, and T E 4
// bytes written by the backward pass.
//
// Forward: unit u of a sequence is a run of chunk of its tokens, kept or not; a CTA sums p over a unit (a warp a row,
// a lane every 32nd expert or four neighbours of every 128, 32-bit sums over at most chunk / kBalWarps rows, then the
// warps in order) and counts its choices with integer atomics in shared memory, and stores both sums.  The second kernel,
// a cluster of eight CTAs a sequence, adds the units in order (in 64 bits) and forms f . P; the last
// cluster to finish adds the sequences in order.  No sum depends on timing.
#include <cooperative_groups.h>

#include <algorithm>

#include "balance.h"
#include "common.cuh"
#include "launch.cuh"
#include "ptx.cuh"

namespace cg = cooperative_groups;

namespace moe {

constexpr int kBalThreads = 512, kBalWarps = kBalThreads / 32;
constexpr int kSumThreads = 1024, kSumWarps = kSumThreads / 32;
constexpr int kBalCluster = 8;  // second kernel: CTAs a sequence, 32 experts each (E <= 256)

// Tokens a unit: a row a warp, more once there are two units for every SM.
static int balance_chunk(int T, int sm_count) {
    const int per = (T + 2 * sm_count - 1) / (2 * sm_count);
    return std::max(kBalWarps, per);
}
static int balance_units(int T, int B, int chunk) { return T / chunk + B; }

struct BalanceWs {
    float* p;          // [units, E]
    int32_t* c;        // [units, E]
    int32_t* n;        // [units]
    float* loss;       // [B]
    uint32_t* ticket;  // [1]
    size_t bytes;
};
static BalanceWs balance_layout(void* ws, int E, int B, int units) {
    BalanceWs w;
    char* p = static_cast<char*>(ws);
    size_t o = 0;
    auto take = [&](size_t n) {
        char* r = p + o;
        o += (n + 255) / 256 * 256;
        return r;
    };
    w.p = (float*)take(sizeof(float) * units * E);
    w.c = (int32_t*)take(sizeof(int32_t) * units * E);
    w.n = (int32_t*)take(sizeof(int32_t) * units);
    w.loss = (float*)take(sizeof(float) * B);
    w.ticket = (uint32_t*)take(sizeof(uint32_t));
    w.bytes = o;
    return w;
}
size_t balance_workspace(int T, int E, int B, int sm_count) {
    return balance_layout(nullptr, E, B, balance_units(T, B, balance_chunk(T, sm_count))).bytes;
}

// Sequence b's tokens [first, last), clipped to the T there are; an offset that is out of order or
// out of range is an error (and the sequence empty).
__device__ __forceinline__ void sequence(const int32_t* offsets, int b, int T, int& first, int& last) {
    if (!offsets) {
        first = 0, last = T;
        return;
    }
    first = offsets[b], last = offsets[b + 1];
    if (first < 0 || last < first || last > T) first = last = 0;
}
__device__ __forceinline__ bool offsets_bad(const int32_t* offsets, int b, int T) {
    if (!offsets) return false;
    const int first = offsets[b], last = offsets[b + 1];
    return first < 0 || last < first || last > T;
}
// The unit of chunk j of sequence b is offsets[b] / chunk + b + j: it grows with (b, j), and no two
// have the same one, since a sequence has at most offsets[b + 1] / chunk - offsets[b] / chunk + 1.
__device__ __forceinline__ int first_unit(const int32_t* offsets, int b, int chunk) {
    return offsets ? max(offsets[b], 0) / chunk + b : 0;
}

// 2^x of the hardware (2 ulp).
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
constexpr float kLog2e = 1.44269504f;
// The softmax takes exp(d), d = l - m, as 2^(d log2 e), the product rounded: off by 1.25 |d| 2^-24, relative, at most, beside
// the |d| 2^-24 of the rounding of d itself.  Against 64 bits its results are as far off as with exp_nonpositive
// (9.1e-8 and 8.9e-8 at 65536 x 256), which takes 51.0 us there instead of 50.0, and 50.6 instead of 47.9 at
// 65536 x 128.  (The fused l log2 e - m log2 e overflows where d does not.)
//
// The sigmoid's l has lost nothing before: exp(d) of d <= 0, off by five half steps at most.  With t = d log2 e, rounded,
// exp(d) = 2^t exp(d - t ln 2): the hardware's 2^t times 1 + r, where r = d - t ln 2, at most |d| 2^-23, by two fused
// steps with ln 2 in two parts.  d below -104, where 2^t is 0 long since, stays at it, so that -inf gives 0; NaN stays NaN.
__device__ __forceinline__ float exp_nonpositive(float d) {
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(d) : "f"(-104.f));
    const float t = d * kLog2e;
    const float r = fmaf(t, 1.90465421e-9f, fmaf(t, -0.693147182f, d));  // ln 2 = 0.693147182 - 1.90465421e-9
    const float e = exp2_approx(t);
    return fmaf(e, r, e);
}
// 1 / y, y in [1, 2], rounded (to a 2^-20th of a half step): one step of Newton's iteration from the hardware's, which is
// off by 1 ulp.  (1.f / y: 64.5 instead of 53.1 us for loss and gradient at 65536 x 256; both with 2^x alone: 59.0.)
__device__ __forceinline__ float inverse_of_1_to_2(float y) {
    float q;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(q) : "f"(y));
    return fmaf(q, fmaf(-y, q, 1.f), q);
}

// The expert of a lane's value k: every 32nd, or (V: rows of 16-byte words) four neighbours of every 128.
template <bool V>
__device__ __forceinline__ int expert_of(int k) {
    const int lane = threadIdx.x & 31;
    return V ? (k >> 2) * 128 + lane * 4 + (k & 3) : lane + 32 * k;
}

// One token's logits as they come from memory, and whether it counts; a token ahead of the one worked on, so
// that a warp always has a row's loads in flight (without: 4.7 TB/s at best with 32 warps an SM).
template <int NE, bool V, bool FULL>
struct Row {
    float l[NE];
    bool counts;
    __device__ __forceinline__ void load(const BalanceArgs& a, long t) {
        counts = !a.mask || a.mask[t];
        const float* row = a.logits + (size_t)t * a.E;
#pragma unroll
        for (int k = 0; k < NE; k += V ? 4 : 1) {
            const int e = expert_of<V>(k);
            if (V) {
                const float4 v = FULL || e < a.E ? __ldcs(reinterpret_cast<const float4*>(row + e)) : make_float4(0.f, 0.f, 0.f, 0.f);
                l[k] = v.x, l[k + 1 < NE ? k + 1 : k] = v.y, l[k + 2 < NE ? k + 2 : k] = v.z, l[k + 3 < NE ? k + 3 : k] = v.w;
            } else {
                l[k] = FULL || e < a.E ? __ldcs(row + e) : 0.f;
            }
        }
    }
};

// Scores of one token: e[k] = exp(l - max l) or sigmoid(l) of the lane's expert k (0 behind the last),
// and 1 / their sum.  slope (GRAD): e of the softmax, s (1 - s) of the sigmoid as x / (1 + x)^2 with x = exp(-|l|), since
// 1 - s of a rounded s near 1 is off by 17 % at l = 15, and 0 from 17 on.
template <int NE, bool SIG, bool V, bool FULL, bool GRAD>
__device__ __forceinline__ float scores(const float (&l)[NE], int E, float (&e)[NE], float (&slope)[NE]) {
    float sum = 0.f;
    if (SIG) {
#pragma unroll
        for (int k = 0; k < NE; k++) {
            const float x = exp_nonpositive(-fabsf(l[k])), q = inverse_of_1_to_2(1.f + x);
            e[k] = FULL || expert_of<V>(k) < E ? (l[k] < 0.f ? x * q : q) : 0.f;
            if (GRAD) slope[k] = x * q * q;
            sum += e[k];
        }
        return 1.f / (warp_sum(sum) + 1e-20f);
    }
    float m = -__int_as_float(0x7f800000);
#pragma unroll
    for (int k = 0; k < NE; k++)
        if (FULL || expert_of<V>(k) < E) m = fmaxf(m, l[k]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
#pragma unroll
    for (int k = 0; k < NE; k++) {
        e[k] = FULL || expert_of<V>(k) < E ? exp2_approx((l[k] - m) * kLog2e) : 0.f;
        if (GRAD) slope[k] = e[k];
        sum += e[k];
    }
    return 1.f / warp_sum(sum);
}

template <int NE, bool SIG, bool V, bool FULL>
__global__ void __launch_bounds__(kBalThreads) balance_units_kernel(BalanceArgs a, BalanceWs w, int chunk) {
    __shared__ float p_s[kBalWarps][NE * 32];
    __shared__ int32_t c_s[NE * 32];
    __shared__ int32_t n_s[kBalWarps];
    griddep_launch_dependents();
    griddep_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, u = blockIdx.x, E = a.E, K = a.K;
    if (u == 0 && tid == 0) *w.ticket = 0;
    // the last sequence whose first unit is at most u
    int lo = 0, hi = a.B - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (first_unit(a.offsets, mid, chunk) <= u) lo = mid;
        else hi = mid - 1;
    }
    int first, last;
    sequence(a.offsets, lo, a.T, first, last);
    const long t0 = first + (long)(u - first_unit(a.offsets, lo, chunk)) * chunk;
    if (t0 < first || t0 >= last) return;  // no such chunk
    const int t1 = (int)min(t0 + chunk, (long)last);
    for (int e = tid; e < NE * 32; e += kBalThreads) c_s[e] = 0;
    __syncthreads();
    float acc[NE];
#pragma unroll
    for (int k = 0; k < NE; k++) acc[k] = 0.f;
    int n = 0;
    bool bad = false;
    Row<NE, V, FULL> next;
    int next_x = -1;
    int t = (int)t0 + warp;
    auto ahead = [&](int q) {
        if (q >= t1) return;
        next.load(a, q);
        next_x = lane < K ? __ldcs(a.idx + (size_t)q * K + lane) : -1;
    };
    ahead(t);
    for (; t < t1; t += kBalWarps) {
        const Row<NE, V, FULL> row = next;
        const int x = next_x;
        ahead(t + kBalWarps);
        if (!row.counts) continue;
        float e[NE], none[NE];
        if (x >= E) bad = true;
        else if (x >= 0) atomicAdd(&c_s[x], 1);
        const float r = scores<NE, SIG, V, FULL, false>(row.l, E, e, none);
#pragma unroll
        for (int k = 0; k < NE; k++) acc[k] = fmaf(e[k], r, acc[k]);
        n++;
    }
    if (bad) atomicOr(a.err, kErrBadIndex);
#pragma unroll
    for (int k = 0; k < NE; k++) p_s[warp][expert_of<V>(k)] = acc[k];
    if (lane == 0) n_s[warp] = n;
    __syncthreads();
    for (int e = tid; e < E; e += kBalThreads) {
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < kBalWarps; k++) v += p_s[k][e];
        w.p[(size_t)u * E + e] = v;
        w.c[(size_t)u * E + e] = c_s[e];
    }
    if (tid == 0) {
        int v = 0;
#pragma unroll
        for (int k = 0; k < kBalWarps; k++) v += n_s[k];
        w.n[u] = v;
    }
}

// A cluster of eight CTAs a sequence: CTA r adds the units of experts [32 r, 32 r + 32).
__global__ void __cluster_dims__(kBalCluster, 1, 1) __launch_bounds__(kSumThreads)
    balance_sum_kernel(BalanceArgs a, BalanceWs w, int chunk) {
    __shared__ double p_s[kSumWarps][32];
    __shared__ int32_t c_s[kSumWarps][32], n_s[kSumWarps];
    __shared__ double dot_s[kBalCluster];
    __shared__ int last_s;
    cg::cluster_group cl = cg::this_cluster();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, r = (int)cl.block_rank(), E = a.E;
    const int e = r * 32 + lane, clusters = gridDim.x / kBalCluster;
    // A CTA's shared memory may be written once that CTA runs, and the first store to CTA 0's is ahead of the loop's own
    // barriers; met here, behind the kernel before this one, it costs nothing.
    cl.sync();
    griddep_wait();
    griddep_launch_dependents();
    for (int b = blockIdx.x / kBalCluster; b < a.B; b += clusters) {
        int first, last;
        sequence(a.offsets, b, a.T, first, last);
        if (r == 0 && tid == 0 && offsets_bad(a.offsets, b, a.T)) atomicOr(a.err, kErrBadIndex);
        const int u0 = first_unit(a.offsets, b, chunk), nu = (last - first + chunk - 1) / chunk;
        double p = 0.0;
        int32_t c = 0, n = 0;
#pragma unroll 4
        for (int u = warp; u < nu; u += kSumWarps) {
            if (e < E) {
                p += w.p[(size_t)(u0 + u) * E + e];
                c += w.c[(size_t)(u0 + u) * E + e];
            }
            n += w.n[u0 + u];
        }
        p_s[warp][lane] = p;
        c_s[warp][lane] = c;
        if (lane == 0) n_s[warp] = n;
        __syncthreads();
        if (warp == 0) {
            p = 0.0, c = 0, n = 0;
#pragma unroll
            for (int k = 0; k < kSumWarps; k++) p += p_s[k][lane], c += c_s[k][lane], n += n_s[k];
            if (e < E) a.counts[(size_t)b * E + e] = c;
            double v = n > 0 && e < E ? (double)c * p : 0.0;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
            // f . P of these experts, to the cluster's first CTA
            if (lane == 0) *cl.map_shared_rank(&dot_s[r], 0) = n > 0 ? v * E / ((double)a.K * n * n) : 0.0;
            if (r == 0 && lane == 0) a.tokens[b] = n;
        }
        cl.sync();
        if (r == 0 && tid == 0) {
            double v = 0.0;
            for (int k = 0; k < kBalCluster; k++) v += dot_s[k];
            w.loss[b] = (float)v;
        }
        cl.sync();
    }
    if (r != 0) return;
    if (tid == 0) {
        __threadfence();
        last_s = atomicAdd(w.ticket, 1u) == (unsigned)clusters - 1;
        __threadfence();
    }
    __syncthreads();
    if (!last_s) return;
    // the last cluster: the mean over the sequences that have tokens
    double v = 0.0;
    int full = 0;
    for (int b = tid; b < a.B; b += kSumThreads) {
        v += __ldcg(w.loss + b);
        full += __ldcg(a.tokens + b) > 0;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        v += __shfl_xor_sync(0xffffffffu, v, o);
        full += __shfl_xor_sync(0xffffffffu, full, o);
    }
    if (lane == 0) p_s[warp][0] = v, n_s[warp] = full;
    __syncthreads();
    if (tid == 0) {
        v = 0.0, full = 0;
        for (int k = 0; k < kSumWarps; k++) v += p_s[k][0], full += n_s[k];
        *a.loss = full ? (float)(v / full) : 0.f;
        a.tokens[a.B] = full;
    }
}

// A warp a row; rows of a warp are neighbours, so that it keeps its sequence's f in registers.
template <int NE, bool SIG, bool V, bool FULL>
__global__ void __launch_bounds__(kBalThreads) balance_backward_kernel(BalanceArgs a, int per_warp) {
    griddep_wait();
    const int E = a.E;
    const long t0 = ((long)blockIdx.x * kBalWarps + (threadIdx.x >> 5)) * per_warp;
    const long t1 = min(t0 + per_warp, (long)a.T);
    if (t0 >= t1) return;
    Row<NE, V, FULL> next;
    next.load(a, t0);
    const int full = a.tokens[a.B];
    const float grad = a.grad ? *a.grad : 1.f;
    int b = 0;  // the sequence of token t is the last that begins at or before t, -1: none does
    if (a.offsets) {
        int lo = 0, hi = a.B;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (a.offsets[mid] <= t0) lo = mid + 1;
            else hi = mid;
        }
        b = lo - 1;
    }
    float f[NE];
    int have = -1, n = 0;
    for (long t = t0; t < t1; t++) {
        const Row<NE, V, FULL> row = next;
        if (t + 1 < t1) next.load(a, t + 1);
        bool in = true;
        if (a.offsets) {
            while (b + 1 < a.B && a.offsets[b + 1] <= t) b++;
            in = b >= 0 && a.offsets[b + 1] > t;
        }
        if (in && b != have) {
            n = a.tokens[b];
            const float k = n > 0 && full > 0 ? grad * (float)((double)E / ((double)a.K * n * (double)n * full)) : 0.f;
#pragma unroll
            for (int j = 0; j < NE; j++) {
                const int e = expert_of<V>(j);
                f[j] = FULL || e < E ? k * (float)a.counts[(size_t)b * E + e] : 0.f;
            }
            have = b;
        }
        float d[NE];
        if (!in || n <= 0 || !row.counts) {  // a token of no sequence, or one that does not count
#pragma unroll
            for (int j = 0; j < NE; j++) d[j] = 0.f;
        } else {
            float e[NE], slope[NE], inner = 0.f;
            const float r = scores<NE, SIG, V, FULL, true>(row.l, E, e, slope);
#pragma unroll
            for (int j = 0; j < NE; j++) inner = fmaf(f[j], e[j], inner);
            inner = warp_sum(inner) * r;
#pragma unroll
            for (int j = 0; j < NE; j++) d[j] = slope[j] * r * (f[j] - inner);
        }
        float* out = a.dlogits + (size_t)t * E;
#pragma unroll
        for (int j = 0; j < NE; j += V ? 4 : 1) {
            const int e = expert_of<V>(j);
            if (!FULL && e >= E) continue;
            if (V) __stcs(reinterpret_cast<float4*>(out + e), make_float4(d[j], d[j + 1 < NE ? j + 1 : j], d[j + 2 < NE ? j + 2 : j], d[j + 3 < NE ? j + 3 : j]));
            else __stcs(out + e, d[j]);
        }
    }
}

template <int NE, bool V, bool FULL>
static cudaError_t units_launch(const BalanceArgs& a, const BalanceWs& w, int chunk, int units, cudaStream_t st) {
    return launch_after(a.scoring ? balance_units_kernel<NE, true, V, FULL> : balance_units_kernel<NE, false, V, FULL>, units,
                        kBalThreads, 0, 0, st, a, w, chunk);
}
template <int NE, bool V, bool FULL>
static cudaError_t backward_launch(const BalanceArgs& a, int grid, int per_warp, cudaStream_t st) {
    return launch_after(a.scoring ? balance_backward_kernel<NE, true, V, FULL> : balance_backward_kernel<NE, false, V, FULL>, grid,
                        kBalThreads, 0, 0, st, a, per_warp);
}

// Rows of 16-byte words where the sizes and addresses allow them; without bounds in a row of 128 or 256.
cudaError_t launch_balance_loss(const BalanceArgs& a, int sm_count, cudaStream_t st) {
    const int chunk = balance_chunk(a.T, sm_count), units = balance_units(a.T, a.B, chunk);
    const BalanceWs w = balance_layout(a.ws, a.E, a.B, units);
    const bool words = a.E % 4 == 0 && ((uintptr_t)a.logits & 15) == 0;
    cudaError_t e;
    if (words && a.E == 128) e = units_launch<4, true, true>(a, w, chunk, units, st);
    else if (words && a.E == 256) e = units_launch<8, true, true>(a, w, chunk, units, st);
    else if (words && a.E <= 128) e = units_launch<4, true, false>(a, w, chunk, units, st);
    else if (words) e = units_launch<8, true, false>(a, w, chunk, units, st);
    else if (a.E <= 128) e = units_launch<4, false, false>(a, w, chunk, units, st);
    else e = units_launch<8, false, false>(a, w, chunk, units, st);
    if (e != cudaSuccess) return e;
    return launch_after(balance_sum_kernel, kBalCluster * std::min(a.B, sm_count / kBalCluster), kSumThreads, 0, 0, st, a, w, chunk);
}

cudaError_t launch_balance_backward(const BalanceArgs& a, int sm_count, cudaStream_t st) {
    if (a.T <= 0) return cudaSuccess;
    // thirty-two warps an SM at the least before a warp takes a second row
    const int per_warp = std::max(1, std::min(16, a.T / (sm_count * 32)));
    const int grid = (a.T + kBalWarps * per_warp - 1) / (kBalWarps * per_warp);
    const bool words = a.E % 4 == 0 && (((uintptr_t)a.logits | (uintptr_t)a.dlogits) & 15) == 0;
    if (words && a.E == 128) return backward_launch<4, true, true>(a, grid, per_warp, st);
    if (words && a.E == 256) return backward_launch<8, true, true>(a, grid, per_warp, st);
    if (words && a.E <= 128) return backward_launch<4, true, false>(a, grid, per_warp, st);
    if (words) return backward_launch<8, true, false>(a, grid, per_warp, st);
    if (a.E <= 128) return backward_launch<4, false, false>(a, grid, per_warp, st);
    return backward_launch<8, false, false>(a, grid, per_warp, st);
}

}  // namespace moe
