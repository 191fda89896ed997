// Routing limited to the best groups of experts, and the gradient of the routing weights.
//
//   key   softmax: the logit;  sigmoid: fp32(s + bias), s = 1 / (1 + exp(-l)), each step rounded as the other router
//         kernels round it (route_core.cuh)
//   group score   softmax: its largest key;  sigmoid: the fp32 sum of its two largest (of the one, where it has one)
//   the best `top` groups (ties to the lower), in them the best K experts by key (ties to the lower), in that order
//   w = scale v, or scale v / sum of the chosen v;  v: the softmax probability, or s
//
// A warp a token.  A group's experts lie on neighbouring lanes, V to a lane, so that a group's score is a matter of a few
// shuffles and a lower lane means a lower index.  The sequence of K maxima runs on 32-bit words: 22 to 27 bits of the key in
// order, then the place (lane, then place within the lane, the lower the larger, so that no two words are the same and
// ties go to the lower index).  A logit gives the upper bits of its own pattern.  A sigmoid's key is formed with the
// hardware's 2^x and reciprocal and put on a grid of 2^-23 of the range that the biases allow: one fused
// multiplication and addition, biases and range being the warp's for all its tokens.  Each lane sorts its words once and
// keeps the list in shared memory; then each choice is a maximum over the warp (one instruction) and a step in the list of
// the lane that held it.  Groups are opened by words of the same kind.
// Such words decide wherever neighbours in the sequence, and the last open and first closed group, lie further apart than
// the margins stated below.  Where two of the chosen lie closer, the chosen are put in order by the keys themselves (the
// exponential in double); where the last chosen and the next, or two groups, do, the token is done again with 64-bit words
// of key and index: the result is always that of the definition.  That costs 65536 tokens of 256 experts up to 171 us (sigmoid; softmax 124) where
// it comes to every token: all keys the same, sigmoids saturated at 1 without a bias, a bias of -inf, biases 10^4 apart.  Where it comes to those
// whose best eight lie on one lane of route_octet_kernel: 51 to 74 us with experts stored by popularity (logits falling by 4.2 over 256
// experts), 122 with them in strict order.
//
// Bounded by the instructions a token takes and their latency: 258 a token at 65536 x 256, 8 groups, top 8, sigmoid, with four tokens a
// warp (route_octet_kernel; 490 with one), 31 us, of which reading the logits needs 11.
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

// Words u[FROM .. FROM + N) in falling order (odd-even merge sort).
template <int N, int FROM, int V>
__device__ __forceinline__ void sort_falling(uint32_t (&u)[V]) {
#pragma unroll
    for (int p = 1; p < N; p *= 2)
#pragma unroll
        for (int k = p; k >= 1; k /= 2)
#pragma unroll
            for (int j = k % p; j + k < N; j += 2 * k)
#pragma unroll
                for (int i = 0; i < k; i++)
                    if (i + j + k < N && (i + j) / (2 * p) == (i + j + k) / (2 * p)) {
                        const uint32_t a = u[FROM + i + j], b = u[FROM + i + j + k];
                        u[FROM + i + j] = max(a, b), u[FROM + i + j + k] = min(a, b);
                    }
}
// The eight largest of two falling runs of eight, u[A ..] and u[B ..], falling in u[A ..].
template <int A, int B, int V>
__device__ __forceinline__ void merge8(uint32_t (&u)[V]) {
#pragma unroll
    for (int i = 0; i < 8; i++) u[A + i] = max(u[A + i], u[B + 7 - i]);
#pragma unroll
    for (int k = 4; k >= 1; k /= 2)
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (!(i & k)) {
                const uint32_t a = u[A + i], b = u[A + i + k];
                u[A + i] = max(a, b), u[A + i + k] = min(a, b);
            }
}
// The largest min(V, 8), falling, in front.
template <int V>
__device__ __forceinline__ void largest_first(uint32_t (&u)[V]) {
    if constexpr (V <= 8) {
        sort_falling<V, 0>(u);
    } else {
        sort_falling<8, 0>(u), sort_falling<8, 8>(u), merge8<0, 8>(u);
        if constexpr (V == 32) sort_falling<8, 16>(u), sort_falling<8, 24>(u), merge8<16, 24>(u), merge8<0, 16>(u);
    }
}

__device__ __forceinline__ unsigned long long warp_max64(unsigned long long v) {
    const uint32_t high = __reduce_max_sync(0xffffffffu, (uint32_t)(v >> 32));
    const uint32_t low = __reduce_max_sync(0xffffffffu, (uint32_t)(v >> 32) == high ? (uint32_t)v : 0u);
    return (unsigned long long)high << 32 | low;
}
// Key and index of expert e in one word, by the definition.
template <bool SIG>
__device__ __forceinline__ unsigned long long exact_word(const float* row, const float* bias, int e) {
    float k = row[e];
    if (SIG) k = __fdiv_rn(1.0f, 1.0f + router_exp(-k)) + (bias ? bias[e] : 0.f);
    return (unsigned long long)key_bits(k) << 32 | (uint32_t)~e;
}

// The choices of one token by the definition, one warp: expert k on lane k < K.
template <int V, bool SIG>
__device__ __noinline__ int choose_exactly(const float* row, const float* bias, int K, int groups, int top, RouteSpread sp) {
    const int lane = threadIdx.x & 31, P = 1 << sp.shift, g = lane >> sp.shift, m0 = (lane & (P - 1)) * sp.each;
    const int n = g < groups ? min(max(sp.size - m0, 0), sp.each) : 0, e0 = g * sp.size + m0;
    unsigned long long key[V];
    uint32_t a = 0, b = 0;  // the two largest of the group
#pragma unroll
    for (int j = 0; j < V; j++) {
        key[j] = 0;
        if (j < n) {
            key[j] = exact_word<SIG>(row, bias, e0 + j);
            const uint32_t o = (uint32_t)(key[j] >> 32);
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
#pragma unroll
        for (int j = 0; j < V; j++) best = max(best, open ? key[j] : 0ull);
        best = warp_max64(best);
        if (lane == k) chosen = (int)~(uint32_t)best;
#pragma unroll
        for (int j = 0; j < V; j++)
            if (key[j] == best) key[j] = 0;
    }
    return chosen;
}

// The choices e of LANES neighbouring lanes (`in`: this lane has one) in the order of the definition.  slots: LANES ints of them.
template <bool SIG, int LANES>
__device__ __noinline__ int order_exactly(const float* row, const float* bias, int e, bool in, uint32_t* slots) {
    const unsigned long long mine = in ? exact_word<SIG>(row, bias, e) : 0;
    int rank = 0;
#pragma unroll
    for (int o = 1; o < LANES; o++) rank += __shfl_xor_sync(0xffffffffu, mine, o) > mine;
    __syncwarp();
    if (in) slots[rank] = e;
    __syncwarp();
    return in ? (int)slots[threadIdx.x & (LANES - 1)] : 0;
}

// 1 / y to a step, y in [1e-20, inf]: a step of Newton's iteration from the hardware's.
__device__ __forceinline__ float inverse(float y) {
    const float q = rcp_hw(y);
    return y < 1e38f ? fmaf(q, fmaf(-y, q, 1.f), q) : 0.f;
}

// A sigmoid's keys on a grid of 2^23 steps for the range that the biases allow: 2^23 + 1 + (s + bias - least bias) * grid, an
// fp32 number with the steps for its last bits.
struct RouteGrid {
    float grid = 0.f, low = 0.f, apart = 0.f;  // apart: how far two words must be (below)
    bool wild = false;  // a bias is not finite: nothing lies on the grid
    __device__ __forceinline__ void set(const float* bias, int E) {  // by a warp
        float least = bias ? INFINITY : 0.f, most = bias ? -INFINITY : 0.f;
        if (bias)
            for (int e = threadIdx.x & 31; e < E; e += 32) {
                const float b = bias[e];
                least = fminf(least, b), most = fmaxf(most, b);
                wild |= !(fabsf(b) < INFINITY);
            }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            least = fminf(least, __shfl_xor_sync(0xffffffffu, least, o));
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
        }
        const float range = (most - least + 1.f) * 1.00001f;  // (room for rounding, and for no word to be 0)
        wild = __any_sync(0xffffffffu, wild) || !(range < 1e30f);
        grid = wild ? 0.f : 8388608.f / range;
        low = wild ? 0.f : least;
        apart = grid * (0x1p-19f + fmaxf(fabsf(least), fabsf(most) + 1.f) * 0x1p-23f) + 4.f;
    }
    __device__ __forceinline__ float shift(const float* bias, int e) const {  // (what s * grid is added to)
        return wild ? 8388608.f : 8388609.f + ((bias ? bias[e] : 0.f) - low) * grid;
    }
};

// Margins.
// Softmax: the words leave out the last bits of the logit; equal words but for the place are too close.
// Sigmoid, in steps of the grid (2^-23 of the range; `grid` steps make 1): the product l log2 e is off by |l| 2^-24 / ln 2 in the
// exponent, 2^x and the reciprocal by 2^-22 each, the additions by 2^-24, so s by s (1 - s) |l| 2^-24 + s 2^-21 at most, and, since
// s (1 - s) |l| < 0.23, by less than 2^-20.  The bias's place on the grid is off by 1.5 steps, the sum by half a step, and the key
// of the definition by 2^-24 of its size, kmax at most.  Two keys: grid (2^-19 + kmax 2^-23) + 4 = apart.  Two groups of two keys, in
// the same terms: grid 2^-20 and 2 steps for each of the four keys; kmax 2^-24 for the rounding of each, half a unit of kmax 2^-23, two
// units for the four; and 2 kmax 2^-24 for the rounding of each group's fp32 sum, two units for both: grid (2^-18 + 4 kmax 2^-23) + 8,
// which 4 apart covers (with 3 apart biases near 128 that lie within 0.1 have opened a group that was not the definition's).
// (Scores that are all far below 2^-19 are told apart by their biases; without those, exactly.)
// A NaN, like a bias that is not finite, leaves the range of words and is left to the exact choice.
// FULL: every lane has V experts.
template <int V, bool SIG, bool FULL>
__global__ void __launch_bounds__(kRouteWarps * 32, 4) route_groups_kernel(RouteGroupsArgs a, RouteSpread sp, bool vec) {
    __shared__ uint32_t lists[kRouteWarps][(V + 1) * 32];  // word j of lane i at j * 32 + i; zeros behind
    __shared__ uint32_t best[kRouteWarps][kMaxTopK + 1];  // (more than the 16 that order_exactly takes)
    griddep_wait();
    constexpr uint32_t kPlaces = !SIG ? 32 * V : V <= 8 ? 256 : 512;  // the words' last bits
    const int lane = threadIdx.x & 31, P = 1 << sp.shift, g = lane >> sp.shift, m0 = (lane & (P - 1)) * sp.each;
    const int n = FULL ? V : g < a.groups ? min(max(sp.size - m0, 0), sp.each) : 0, e0 = g * sp.size + m0, E = a.E, K = a.K;
    const uint32_t place = (31 - lane) * V + V - 1;
    uint32_t* list = &lists[threadIdx.x >> 5][lane];
    uint32_t* found = best[threadIdx.x >> 5];
    list[V * 32] = 0;
    RouteGrid on;
    if (SIG) on.set(a.bias, E);
    float shift[SIG ? V : 1];
    if (SIG)
#pragma unroll
        for (int j = 0; j < V; j++) shift[j] = j < n ? on.shift(a.bias, e0 + j) : 0.f;
    for (int64_t t = (int64_t)blockIdx.x * kRouteWarps + (threadIdx.x >> 5); t < a.T; t += (int64_t)gridDim.x * kRouteWarps) {
        const float* row = a.logits + t * E;
        float l[V];
        if (V >= 4 && (FULL || vec)) {
#pragma unroll
            for (int j = 0; j < V; j += 4)
                if (FULL || j < n) {
                    const float4 q = *reinterpret_cast<const float4*>(row + e0 + j);
                    l[j] = q.x, l[(j + 1) % V] = q.y, l[(j + 2) % V] = q.z, l[(j + 3) % V] = q.w;
                }
        } else {
#pragma unroll
            for (int j = 0; j < V; j++)
                if (FULL || j < n) l[j] = row[e0 + j];
        }
        bool nan = SIG && on.wild;
        uint32_t u[V];
#pragma unroll
        for (int j = 0; j < V; j++) {
            float k = FULL || j < n ? l[j] : -INFINITY;
            if (SIG) {  // (from 2^23 to 2^24: the exponent's bits leave on the left)
                const float on_grid = fmaf(rcp_hw(1.f + exp2_hw(k * -1.44269504f)), on.grid, shift[j]);
                u[j] = __float_as_uint(on_grid) * kPlaces + (place - j);
                nan |= V > 8 && on_grid != on_grid;
            } else {
                k += 0.f;  // (-0 is 0)
                nan |= k != k;
                u[j] = (ordered_bits(k) & ~(kPlaces - 1)) | (place - j);
            }
            if (!FULL && j >= n) u[j] = 0;
        }
        sort_falling<V, 0>(u);
        if (SIG && V <= 8) nan |= u[0] >= 0x80000000u;  // NaN's pattern alone sets that bit
#pragma unroll
        for (int j = 0; j < V; j++) list[j * 32] = u[j];
        bool again = nan, mixed = false;
        const float apart = on.apart;
        const uint32_t* step = list;
        if (a.top < a.groups) {
            uint32_t score = u[0] / kPlaces, second = V > 1 ? u[V > 1 ? 1 : 0] / kPlaces : 0;
            for (int o = 1; o < P; o <<= 1) {
                const uint32_t c = __shfl_xor_sync(0xffffffffu, score, o);
                if (SIG) second = max(min(score, c), max(second, __shfl_xor_sync(0xffffffffu, second, o)));
                score = max(score, c);
            }
            if (SIG) score += second;
            score = FULL || g < a.groups ? (score + 1) * 32 - 1 - g : 0u;
            bool open = false;
            uint32_t last = 0;
            for (int i = 0; i < a.top; i++) {
                last = __reduce_max_sync(0xffffffffu, score);
                if (score == last) open = true, score = 0;
            }
            const uint32_t next = __reduce_max_sync(0xffffffffu, score);
            if (SIG) again |= !((float)(last / 32 - next / 32) > 4.f * apart);
            else again |= last / 32 == next / 32;
            if (!open) step = list + V * 32;
        }
#pragma unroll 3
        for (int k = 0; k <= K; k++) {
            const uint32_t head = *step, top = __reduce_max_sync(0xffffffffu, head);
            if (head == top) found[k] = top;
            step += head == top && top ? 32 : 0;  // (0: no list has any more)
        }
        __syncwarp();
        const uint32_t word = found[min(lane, K)], after = found[min(lane + 1, K)];
        const uint32_t at = 32 * V - 1 - (word & (kPlaces - 1));
        int e = ((int)(at / V) >> sp.shift) * sp.size + ((int)(at / V) & (P - 1)) * sp.each + (int)(at & (V - 1));
        if (lane < K && after) {
            bool near = word / kPlaces == after / kPlaces;
            if (SIG) near = !((float)(word / kPlaces - after / kPlaces) > apart);
            if (lane == K - 1) again |= near;
            else mixed = near;
        }
        if (__any_sync(0xffffffffu, again || mixed))
            e = __any_sync(0xffffffffu, again) ? choose_exactly<V, SIG>(row, a.bias, K, a.groups, a.top, sp)
                                            : order_exactly<SIG, 16>(row, a.bias, e, lane < K, found);
        float v = 0.f;
        bool bad = false;
        if (SIG) {
            if (nan) {  // (a lane that found nothing but wild biases has nothing to report)
#pragma unroll
                for (int j = 0; j < V; j++)
                    if (j < n) bad |= row[e0 + j] != row[e0 + j] || (a.bias && a.bias[e0 + j] != a.bias[e0 + j]);
            }
            if (lane < K) v = inverse(1.f + expf(-row[e]));
        } else {
            const float mine = lane < K ? row[e] : -INFINITY, most = __shfl_sync(0xffffffffu, mine, 0);
            bad = nan || !(fabsf(most) < INFINITY);
            v = expf(mine - most);
            if (!a.renormalize) {  // the largest of all is the first chosen
                float z = 0.f;
#pragma unroll
                for (int j = 0; j < V; j++)
                    if (FULL || j < n) z += exp2_hw((l[j] - most) * 1.44269504f);
                v *= inverse(warp_sum(z));
            }
        }
        bad = __any_sync(0xffffffffu, bad);
        if (a.renormalize) {
            float total = v;  // of lanes 0 to 15 (zeros from K on)
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
            v *= inverse(total + (SIG ? 1e-20f : 0.f));
        }
        if (lane < K) {
            a.idx[t * K + lane] = e;
            a.w[t * K + lane] = bad ? __int_as_float(0x7fffffff) : v * a.scale;
        }
        if (bad && lane == 0) atomicOr(a.err, kErrNonFinite);
        __syncwarp();  // the words found have been read
    }
}

// Eight lanes a token, four tokens a warp: what a warp does once a token (pops, weights, addresses) is done once for four.
// A lane has E / 8 neighbouring experts, a group one or more whole lanes; K <= 8, E % 32 == 0, groups 1, 2, 4 or 8.  The four rows, one
// run of memory, come through shared memory (cp.async, asked for once the set before has been read), a lane's experts side by side.  A lane keeps its eight largest
// words; where all eight are chosen, or would be next, the token is done exactly (a chance of 2^-7 where two lanes are open and
// experts are in no order, and launch_route_groups takes this kernel for two open lanes or more).  Margins as above.
constexpr int kOctetWarps = 4;
template <int V>
struct OctetSmem {
    static constexpr int kPitch = V + 4;  // floats of a lane's experts: 16-byte loads of eight lanes on different banks
    float rows[kOctetWarps][32 * kPitch];
    float shift[8 * kPitch];
    uint32_t lists[kOctetWarps][(V < 8 ? V + 2 : 10) * 32];  // word j of a lane at j * 32; then what says "no more", then 0
    uint32_t found[kOctetWarps][4][12];
};
constexpr int kOctetCtas = 5;  // of an SM: 96 registers a thread (4: 34.5, 6, with spills: 33.2 instead of 32.3 us at 65536 x 256)
template <int V, bool SIG, bool FULL>
__global__ void __launch_bounds__(kOctetWarps * 32, kOctetCtas) route_octet_kernel(RouteGroupsArgs a, RouteSpread sp) {
    extern __shared__ __align__(16) unsigned char smem[];
    OctetSmem<V>& s = *reinterpret_cast<OctetSmem<V>*>(smem);
    griddep_wait();
    constexpr int kKept = V < 8 ? V : 8, kPitch = OctetSmem<V>::kPitch, W = V <= 4 ? 1 : V / 4;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, tok = lane >> 3, at8 = lane & 7, E = FULL ? 8 * V : a.E, K = a.K, each = E / 8;
    const int spread = 8 / a.groups, g = at8 / spread;
    const int64_t sets = (a.T + 3) / 4, stride = (int64_t)gridDim.x * kOctetWarps;
    // words of 16 bytes of four rows: word lane + 32 i goes to lane `word / (each / 4)`
    int dst[V / 4];
#pragma unroll
    for (int i = 0; i < V / 4; i++) {
        const int w = lane + 32 * i;
        dst[i] = w / (each / 4) * kPitch + w % (each / 4) * 4;
    }
    auto ask = [&](int64_t set) {
        if (set < sets) {
            const int64_t words = min((int64_t)E, (a.T - set * 4) * (E / 4));
            const float* src = a.logits + set * 4 * E;
            const uint32_t to = smem_u32(s.rows[warp]);
#pragma unroll
            for (int i = 0; i < V / 4; i++)
                if (lane + 32 * i < words) cp_async16(to + dst[i] * 4, src + (lane + 32 * i) * 4);
        }
    };
    int64_t set = (int64_t)blockIdx.x * kOctetWarps + warp;
    ask(set);
    RouteGrid on;
    if (SIG) {
        on.set(a.bias, E);
        for (int e = threadIdx.x; e < E; e += kOctetWarps * 32) s.shift[e / each * kPitch + e % each] = on.shift(a.bias, e);
    }
    uint32_t* list = &s.lists[warp][lane];
    list[kKept * 32] = V > 8 ? 0xffffffffu : 0u;
    list[kKept * 32 + 32] = 0;
    __syncthreads();
    for (; set < sets; set += stride) {
        cp_async_wait_all();
        __syncwarp();
        const int64_t t = set * 4 + tok;
        const bool there = t < a.T;
        const float* mine = s.rows[warp] + lane * kPitch;
        const float* shift = s.shift + at8 * kPitch;
        const uint32_t place = (7 - at8) * 32 + 31;
        bool nan = SIG && on.wild;
        uint32_t u[V];
#pragma unroll
        for (int i = 0; i < V; i += 4) {
            float4 l = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY), h = make_float4(0.f, 0.f, 0.f, 0.f);
            if (FULL || i < each) {
                l = *reinterpret_cast<const float4*>(mine + i);
                if (SIG) h = *reinterpret_cast<const float4*>(shift + i);
            }
            const float lk[4] = {l.x, l.y, l.z, l.w}, hk[4] = {h.x, h.y, h.z, h.w};
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int j = i + k;
                if (SIG) {
                    u[j] = __float_as_uint(fmaf(rcp_hw(1.f + exp2_hw(lk[k] * -1.44269504f)), on.grid, hk[k])) * 256 + (place - j);
                } else {
                    const float x = lk[k] + 0.f;
                    nan |= x != x;
                    u[j] = (ordered_bits(x) & ~255u) | (place - j);
                }
                if (!FULL && i >= each) u[j] = 0;
            }
        }
        float z = 0.f, lane_most = -INFINITY;  // (softmax as it is) the lane's largest and its sum
        if (!SIG && !a.renormalize) {
#pragma unroll
            for (int j = 0; j < V; j++)
                if (FULL || j < each) lane_most = fmaxf(lane_most, mine[j]);
#pragma unroll
            for (int j = 0; j < V; j++)
                if ((FULL || j < each) && lane_most > -INFINITY) z += exp2_hw((mine[j] - lane_most) * 1.44269504f);
        }
        bool bad = false;
        if (SIG) {
            uint32_t any = 0;
#pragma unroll
            for (int j = 0; j < V; j++) any |= u[j];
            nan |= any >= 0x80000000u;
            if (nan && there)  // (a lane that found nothing but wild biases has nothing to report)
                for (int j = 0; j < each; j++) bad |= mine[j] != mine[j] || (a.bias && a.bias[at8 * each + j] != a.bias[at8 * each + j]);
        }
        __syncwarp();  // the rows have been read
        ask(set + stride);
        largest_first(u);
#pragma unroll
        for (int j = 0; j < kKept; j++) list[j * 32] = u[j];
        bool again = nan;
        const float apart = on.apart;
        const uint32_t* step = list;
        if (a.top < a.groups) {
            uint32_t score = u[0] >> 8, second = u[1] >> 8;
            for (int o = 1; o < spread; o <<= 1) {
                const uint32_t c = __shfl_xor_sync(0xffffffffu, score, o);
                if (SIG) second = max(min(score, c), max(second, __shfl_xor_sync(0xffffffffu, second, o)));
                score = max(score, c);
            }
            if (SIG) score += second;
            score = score * 32 + 31 - g;
            int before = 0;  // lanes of better groups
#pragma unroll
            for (int o = 1; o < 8; o++) before += __shfl_xor_sync(0xffffffffu, score, o) > score;
            const bool open = before < a.top * spread;
            uint32_t last = open ? score : 0xffffffffu, next = open ? 0u : score;
#pragma unroll
            for (int o = 4; o > 0; o >>= 1) {
                last = min(last, __shfl_xor_sync(0xffffffffu, last, o));
                next = max(next, __shfl_xor_sync(0xffffffffu, next, o));
            }
            if (SIG) again |= !((float)(last / 32 - next / 32) > 4.f * apart);
            else again |= last / 32 == next / 32;
            if (!open) step = list + (kKept + 1) * 32;
        }
        uint32_t* found = s.found[warp][tok];
#pragma unroll 3
        for (int k = 0; k <= K; k++) {
            const uint32_t head = *step;
            uint32_t top = head;
#pragma unroll
            for (int o = 4; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
            if (head == top) found[k] = top;
            step += head == top && top && top != 0xffffffffu ? 32 : 0;
        }
        __syncwarp();
        const uint32_t word = found[min(at8, K)], after = found[min(at8 + 1, K)];
        const int at = 255 - (int)(word & 255);
        int e = (at >> 5) * each + (at & 31);
        bool mixed = false;
        if (at8 < K && after) {
            const bool near = after == 0xffffffffu || (SIG ? !((float)(word / 256 - after / 256) > apart) : word / 256 == after / 256);
            if (at8 == K - 1 || after == 0xffffffffu) again |= near;
            else mixed = near;
        }
        if (__any_sync(0xffffffffu, (again || mixed) && there)) {
            // (other tokens of the warp are put in the order that they have)
            if (__any_sync(0xffffffffu, mixed && there)) e = order_exactly<SIG, 8>(a.logits + t * E, a.bias, e, at8 < K && there, found);
            const unsigned redo = __ballot_sync(0xffffffffu, again && there);
            for (int k = 0; k < 4; k++)
                if (redo >> (8 * k) & 255) {
                    const int chosen = __shfl_sync(0xffffffffu, choose_exactly<W, SIG>(a.logits + (set * 4 + k) * E, a.bias, K, a.groups, a.top, sp), at8);
                    if (tok == k) e = chosen;
                }
        }
        const float l = at8 < K && there ? a.logits[t * E + e] : -INFINITY;
        float v;
        if (SIG) {
            v = at8 < K ? inverse(1.f + expf(-l)) : 0.f;
        } else {
            const float most = __shfl_sync(0xffffffffu, l, lane & 24);
            bad = nan || !(fabsf(most) < INFINITY);
            v = expf(l - most);
            if (!a.renormalize) {  // the largest of all is the first chosen
                z *= exp2_hw((lane_most - most) * 1.44269504f);
#pragma unroll
                for (int o = 4; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
                v *= inverse(z);
            }
        }
        bad = __ballot_sync(0xffffffffu, bad && there) >> (lane & 24) & 255;
        if (a.renormalize) {
            float total = v;
#pragma unroll
            for (int o = 4; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
            v *= inverse(total + (SIG ? 1e-20f : 0.f));
        }
        if (at8 < K && there) {
            a.idx[t * K + at8] = e;
            a.w[t * K + at8] = bad ? __int_as_float(0x7fffffff) : v * a.scale;
        }
        if (bad && at8 == 0) atomicOr(a.err, kErrNonFinite);
        __syncwarp();  // lists and words found have been read
    }
}

template <int V, bool SIG, bool FULL>
static cudaError_t octets_for(const RouteGroupsArgs& a, const RouteSpread& sp, int sm_count, cudaStream_t st) {
    constexpr auto kernel = route_octet_kernel<V, SIG, FULL>;
    const cudaError_t e = allow_smem<kernel>(sizeof(OctetSmem<V>));
    if (e != cudaSuccess) return e;
    const int64_t ctas = ((a.T + 3) / 4 + kOctetWarps - 1) / kOctetWarps;
    const Launch l{(int)std::min<int64_t>(ctas, (int64_t)sm_count * kOctetCtas), kOctetWarps * 32, sizeof(OctetSmem<V>), 0, st};
    return l.run(kernel, a, sp);
}
template <int V>
static cudaError_t octets(const RouteGroupsArgs& a, const RouteSpread& sp, int sm_count, cudaStream_t st) {
    if (a.E == 8 * V) return a.scoring ? octets_for<V, true, true>(a, sp, sm_count, st) : octets_for<V, false, true>(a, sp, sm_count, st);
    return a.scoring ? octets_for<V, true, false>(a, sp, sm_count, st) : octets_for<V, false, false>(a, sp, sm_count, st);
}

cudaError_t launch_route_groups(const RouteGroupsArgs& a, int sm_count, cudaStream_t st) {
    if (a.T <= 0) return cudaSuccess;
    RouteSpread sp;
    sp.size = a.E / a.groups;
    for (sp.shift = 5; a.groups << sp.shift > 32; sp.shift--) {}
    sp.each = (sp.size + (1 << sp.shift) - 1) >> sp.shift;
    const bool vec = sp.each % 4 == 0 && sp.size % 4 == 0 && (uintptr_t)a.logits % 16 == 0;  // (a lane has a multiple of four, then)
    // Four tokens a warp where there are tokens for more than one round of it.  With it and without, us (sigmoid, 8 groups, top 8;
    // E = 64: softmax, 4 groups, top 4):  2400 tokens: 7.3 / 5.9 (E = 256), 5.3 / 4.2 (128), 2.6 / 2.4 (64);  4800: 8.6 / 7.3, 6.0 / 5.8,
    // 2.8 / 3.5;  9600: 11.9 / 11.7, 6.8 / 8.5, 3.5 / 5.3;  19200: 15.9 / 17.7, 10.4 / 14.0, 5.0 / 8.6;  65536: 31 / 44 (256).
    if (a.E % 32 == 0 && a.K <= 8 && 8 % a.groups == 0 && a.top * (8 / a.groups) >= 2 && a.T >= (a.E <= 64 ? 32ll : 64ll) * sm_count && (uintptr_t)a.logits % 16 == 0) {
        if (a.E <= 32) return octets<4>(a, sp, sm_count, st);
        if (a.E <= 64) return octets<8>(a, sp, sm_count, st);
        if (a.E <= 128) return octets<16>(a, sp, sm_count, st);
        return octets<32>(a, sp, sm_count, st);
    }
    const int64_t blocks = (a.T + kRouteWarps - 1) / kRouteWarps;
    const Launch l{(int)std::min<int64_t>(blocks, (int64_t)sm_count * 8), kRouteWarps * 32, 0, 0, st};
    const bool sig = a.scoring != 0;
#define ROUTE_GROUPS(V)                                                                                               \
    if (sp.each <= V) {                                                                                               \
        const bool full = a.groups << sp.shift == 32 && sp.each == V && sp.size == V << sp.shift && (V < 4 || vec);     \
        if (full) return sig ? l.run(route_groups_kernel<V, true, true>, a, sp, vec) : l.run(route_groups_kernel<V, false, true>, a, sp, vec); \
        return sig ? l.run(route_groups_kernel<V, true, false>, a, sp, vec) : l.run(route_groups_kernel<V, false, false>, a, sp, vec);        \
    }
    ROUTE_GROUPS(1)
    ROUTE_GROUPS(2)
    ROUTE_GROUPS(4)
    ROUTE_GROUPS(8)
    ROUTE_GROUPS(16)
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
// Four tokens a warp, whose four rows are one run of memory, 8 lanes a token (K <= 8; else 16, two tokens after two): zeros go out
// while choices and chosen logits are on their way, the values over them (they meet in L2; a run put together in shared memory
// first: 23.6 us at 65536 x 256, so 21.3).  Where the softmax needs the sum over its row (route_dense_kernel), a warp a token.
// Bounded by HBM: T E 4 bytes written, and read where the softmax needs its sum (65536 x 256: 32 us, 66 % of a copy's rate).

// Choices and their gradients: the same expert twice on the lanes of one token: its first lane takes the sum, in the
// choices' order, and `first` is false on the others.  All lanes of the warp; lanes of other tokens never match.
template <int LANES>
__device__ __forceinline__ void merge_repeated(int key, bool in, float& d, bool& first) {
    const unsigned same = __match_any_sync(0xffffffffu, key);
    first = in;
    if (!__any_sync(0xffffffffu, in && __popc(same) > 1)) return;
    const int lane = threadIdx.x & 31, at = lane & ~(LANES - 1);
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < LANES; k++) {
        const float dk = __shfl_sync(0xffffffffu, d, at + k);
        if (same >> (at + k) & 1) sum += dk;
    }
    if (in) d = sum;
    first = in && __ffs(same) - 1 == lane;
}
template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

struct Choice {
    int i;       // the expert; -1: none
    float g, x;  // scale dL/dw, logit
};
// dL/dl of a token's choices, on LANES lanes.
template <int LANES>
__device__ __forceinline__ float choice_gradient(const RouteBackwardArgs& a, const Choice& c) {
    const bool in = c.i >= 0;
    float d;
    if (a.scoring == 0) {
        const float x = in ? c.x : -INFINITY;
        float m = x;
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        const float v = in ? expf(x - m) : 0.f, total = lanes_sum<LANES>(v), p = in ? __fdiv_rn(v, total) : 0.f;
        d = p * (c.g - lanes_sum<LANES>(in ? c.g * p : 0.f));
    } else {
        // s and 1 - s from exp(-|l|), so that neither loses bits where the other is near 1
        const float x = in ? c.x : 0.f, q = expf(-fabsf(x)), big = __fdiv_rn(1.f, 1.f + q), small = q * big;
        const float s = x >= 0.f ? big : small, rest = x >= 0.f ? small : big;
        if (a.renormalize) {
            const float total = lanes_sum<LANES>(in ? s : 0.f) + 1e-20f, p = in ? __fdiv_rn(s, total) : 0.f;
            d = rest * p * (c.g - lanes_sum<LANES>(in ? c.g * p : 0.f));
        } else {
            d = c.g * s * rest;
        }
    }
    return in ? d : 0.f;
}

template <int LANES>
__global__ void __launch_bounds__(kRouteWarps * 32) route_backward_kernel(RouteBackwardArgs a, bool vec) {
    griddep_wait();
    constexpr int kPasses = LANES / 8;  // of 32 / LANES tokens
    const int lane = threadIdx.x & 31, E = a.E, K = a.K, k = lane & (LANES - 1);
    const int64_t set = (int64_t)blockIdx.x * kRouteWarps + (threadIdx.x >> 5);
    if (set * 4 >= a.T) return;  // the whole warp
    auto token = [&](int pass) { return set * 4 + pass * (32 / LANES) + lane / LANES; };
    float* out = a.dlogits + set * 4 * E;
    Choice c[kPasses];
#pragma unroll
    for (int p = 0; p < kPasses; p++) {
        const int64_t t = token(p);
        c[p] = Choice{-1, 0.f, 0.f};
        if (t < a.T && k < K) c[p].i = a.idx[t * K + k], c[p].g = a.dw[t * K + k] * a.scale;
    }
    if (!a.accumulate) {
        const int n = (int)min((int64_t)4, a.T - set * 4) * E;
        if (vec) {
            for (int i = lane * 4; i + 4 <= n; i += 128) *reinterpret_cast<float4*>(out + i) = make_float4(0.f, 0.f, 0.f, 0.f);
            if (lane < (n & 3)) out[(n & ~3) + lane] = 0.f;
        } else {
            for (int i = lane; i < n; i += 32) out[i] = 0.f;
        }
    }
#pragma unroll
    for (int p = 0; p < kPasses; p++) {
        if (c[p].i >= E) {
            atomicOr(a.err, kErrBadIndex);
            c[p].i = -1;
        }
        if (c[p].i >= 0) c[p].x = a.logits[token(p) * E + c[p].i];
    }
    __syncwarp();  // the zeros come before the values
#pragma unroll
    for (int p = 0; p < kPasses; p++) {
        const int row = p * (32 / LANES) + lane / LANES;
        float d = choice_gradient<LANES>(a, c[p]);
        bool first;
        merge_repeated<LANES>(c[p].i >= 0 ? row * E + c[p].i : -1 - lane, c[p].i >= 0, d, first);
        float* at = out + row * E + c[p].i;
        if (first) *at = a.accumulate ? __fadd_rn(*at, d) : d;  // (the gradient's own bits, added: not fused with its last product)
    }
}

// Softmax probabilities as they are: every expert has a gradient.
template <int V>
__global__ void __launch_bounds__(kRouteWarps * 32) route_dense_kernel(RouteBackwardArgs a) {
    __shared__ __align__(16) float rows[kRouteWarps][32 * V];
    griddep_wait();
    const int lane = threadIdx.x & 31, E = a.E, K = a.K;
    float* s_row = rows[threadIdx.x >> 5];
#pragma unroll
    for (int j = 0; j < V; j++) s_row[lane + 32 * j] = 0.f;
    __syncwarp();
    const int64_t stride = (int64_t)gridDim.x * kRouteWarps;
    int64_t t = (int64_t)blockIdx.x * kRouteWarps + (threadIdx.x >> 5);
    float next[V], g_next = 0.f;
    int i_next = -1;
    auto ask = [&](int64_t t) {
        const float* row = a.logits + t * E;
        i_next = -1, g_next = 0.f;
        if (t >= a.T) return;
#pragma unroll
        for (int j = 0; j < V; j++) next[j] = lane + 32 * j < E ? row[lane + 32 * j] : -INFINITY;
        if (lane < K) i_next = a.idx[t * K + lane], g_next = a.dw[t * K + lane];
    };
    ask(t);
    for (; t < a.T; t += stride) {
        float* out = a.dlogits + t * E;
        float l[V];
        int i = i_next;
        float g = g_next * a.scale;
#pragma unroll
        for (int j = 0; j < V; j++) l[j] = next[j];
        ask(t + stride);
        if (i >= E) {
            atomicOr(a.err, kErrBadIndex);
            i = -1;
        }
        const bool in = i >= 0;
        if (!__any_sync(0xffffffffu, in)) {  // no choice, so no gradient, whatever the logits hold (padding, say)
#pragma unroll
            for (int j = 0; j < V; j++)
                if (!a.accumulate && lane + 32 * j < E) out[lane + 32 * j] = 0.f;
            continue;
        }
        if (!in) g = 0.f;
        float most = l[0];
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
        bool first;
        merge_repeated<32>(in ? i : -1 - lane, in, g, first);
        if (first) s_row[i] = g;
        __syncwarp();
        float dot = 0.f;
#pragma unroll
        for (int j = 0; j < V; j++) dot = fmaf(s_row[lane + 32 * j], l[j], dot);
        const float inv = __fdiv_rn(1.f, warp_sum(z));
        dot = warp_sum(dot) * inv;
#pragma unroll
        for (int j = 0; j < V; j++) {
            const int e = lane + 32 * j;
            if (e < E) {
                const float v = l[j] * inv * (s_row[e] - dot);
                out[e] = a.accumulate ? __fadd_rn(out[e], v) : v;
            }
        }
        __syncwarp();
        if (first) s_row[i] = 0.f;
        __syncwarp();
    }
}

cudaError_t launch_route_backward(const RouteBackwardArgs& a, int sm_count, cudaStream_t st) {
    if (a.T <= 0) return cudaSuccess;
    if (a.scoring == 0 && !a.renormalize) {
        const int64_t blocks = (a.T + kRouteWarps - 1) / kRouteWarps;
        const Launch l{(int)std::min<int64_t>(blocks, (int64_t)sm_count * 6), kRouteWarps * 32, 0, 0, st};
        if (a.E <= 32) return l.run(route_dense_kernel<1>, a);
        if (a.E <= 64) return l.run(route_dense_kernel<2>, a);
        if (a.E <= 128) return l.run(route_dense_kernel<4>, a);
        return l.run(route_dense_kernel<8>, a);
    }
    const bool vec = (uintptr_t)a.dlogits % 16 == 0;  // (four rows are a multiple of 16 bytes)
    const int64_t blocks = ((a.T + 3) / 4 + kRouteWarps - 1) / kRouteWarps;
    const Launch l{(int)blocks, kRouteWarps * 32, 0, 0, st};
    return a.K <= 8 ? l.run(route_backward_kernel<8>, a, vec) : l.run(route_backward_kernel<16>, a, vec);
}

}  // namespace moe
