// Scaled products of e4m3 operands and the routed-expert FFN built on them: choice of kernel, tensor maps,
// launches, and the small kernels around the products (token quantiser with the grouping, combine).
#include <cooperative_groups.h>

#include <algorithm>
#include <climits>

#include "common.cuh"
#include "fp8.h"
#include "fp8.cuh"
#include "fp8_tc.cuh"
#include "launch.cuh"

namespace cg = cooperative_groups;

namespace moe {
namespace {

// [mats][rows][cols] bytes, boxes of 128 columns x box_rows rows of one matrix, 128-byte swizzle
bool encode3(EncodeTiledFn enc, CUtensorMap* m, const void* base, int64_t cols, int64_t rows, int64_t mats, int box_rows) {
    const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)mats};
    const cuuint64_t strides[2] = {(cuuint64_t)cols, (cuuint64_t)(cols * rows)};
    const cuuint32_t box[3] = {128, (cuuint32_t)box_rows, 1}, es[3] = {1, 1, 1};
    return enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
bool encode2(EncodeTiledFn enc, CUtensorMap* m, const void* base, int64_t cols, int64_t rows, int box_rows) {
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)cols};
    const cuuint32_t box[2] = {128, (cuuint32_t)box_rows}, es[2] = {1, 1};
    return enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int MODE, int NQ>
struct Few {
    using C = FewCfg<MODE, NQ>;
    // tiles: upper bound of the tiles there may be
    static cudaError_t run(const CUtensorMap& mw, const CUtensorMap& mx, const F8Gemm& g, int64_t tiles, int sm_count,
                           cudaStream_t st) {
        constexpr auto k = f8_few_kernel<MODE, NQ>;
        const cudaError_t e = allow_smem<k>(C::kSmem);
        if (e != cudaSuccess) return e;
        const int slots = sm_count * C::kMinCtas;
        int cs = 1;  // split the inner dimension while all CTAs are still on the GPU at once
        while (cs < 8 && tiles * cs * 2 <= slots && cs * 2 <= g.nkb) cs *= 2;
        const int clusters = (int)std::min<int64_t>(tiles, slots / cs);
        return launch_after(k, clusters * cs, kFewThreads, C::kSmem, cs, st, mw, mx, g);
    }
};

template <int MODE, int NB>
struct Many {
    using C = ManyCfg<MODE, NB>;
    static cudaError_t run(const CUtensorMap& mw, const CUtensorMap& mx, const F8Gemm& g, int64_t tiles, int sm_count,
                           cudaStream_t st) {
        constexpr auto k = f8_many_kernel<MODE, NB>;
        const cudaError_t e = allow_smem<k>(C::kSmem);
        if (e != cudaSuccess) return e;
        return launch_after(k, (int)std::min<int64_t>(tiles, sm_count), kManyThreads, C::kSmem, 0, st, mw, mx, g);
    }
};

}  // namespace

cudaError_t launch_matmul_fp8(const MatmulF8& m, int sm_count, cudaStream_t st) {
    if (m.M <= 0 || m.N <= 0) return cudaSuccess;
    EncodeTiledFn enc = tc_encode_fn();
    if (!enc) return cudaErrorNotSupported;
    F8Gemm g{};
    g.xs = m.xs;
    g.ws = m.ws;
    g.nkb = (m.K + 127) / 128;
    g.nb = (int)((m.N + 127) / 128);
    g.nt = g.nb;
    g.M = (int)m.M;
    g.N = (int)m.N;
    g.out = m.out;
    g.out_f32 = m.out_f32;
    g.err = m.err;
    g.timeout_ns = m.timeout_ns;
    g.inject = m.inject;
    // Few rows: the cluster's exchange of partial sums costs 2 us (16 rows) to 8 us (64), a block of the many-row
    // kernel 0.3 us: it wins where there are few blocks.  us, many / few, at N = 2560: 16 rows, K 1024 5.7 / 6.6, K 2048
    // 8.3 / 6.9; 32 rows, K 2048 8.3 / 8.9, K 4096 13.4 / 9.8; 64 rows, K 4096 13.5 / 14.7, K 8192 23.6 / 17.1.
    const int few = m.M <= 8 ? 0 : m.M <= 16 ? 10 : m.M <= 32 ? 16 : 32;
    const int nq = m.M > 64 || g.nkb <= few ? 128 : m.M <= 16 ? 16 : m.M <= 32 ? 32 : 64;
    CUtensorMap mw, mx;
    if (!encode3(enc, &mw, m.w, m.K, m.N, 1, 128) || !encode2(enc, &mx, m.x, m.K, m.M, nq)) return cudaErrorInvalidValue;
    if (nq == 16) return Few<kF8Dense, 16>::run(mw, mx, g, g.nt, sm_count, st);
    if (nq == 32) return Few<kF8Dense, 32>::run(mw, mx, g, g.nt, sm_count, st);
    if (nq == 64) return Few<kF8Dense, 64>::run(mw, mx, g, g.nt, sm_count, st);
    // Tiles of 128 or of 256 weight rows: a block takes 0.36 or 0.62 us, times the rounds of tiles that the SMs do.
    // 2048 x 2560 x 4096 (320 or 160 tiles): 46 or 53 us; 1024 x 2560 x 4096 (160 or 80): 28 or 24 us.
    const int64_t mt = (m.M + 127) / 128, wide = (m.N + 255) / 256;
    const auto rounds = [&](int64_t tiles) { return (tiles + sm_count - 1) / sm_count; };
    if (4 * rounds(mt * g.nb) < 7 * rounds(mt * wide)) return Many<kF8Dense, 128>::run(mw, mx, g, mt * g.nb, sm_count, st);
    g.nt = (int)wide;
    return Many<kF8Dense, 256>::run(mw, mx, g, mt * wide, sm_count, st);
}

// ---- routed experts ----

constexpr int kPrepThreads = 1024;
constexpr int kPrepPairs = 1024;   // up to here every CTA of the token quantiser groups the pairs itself
constexpr int kPlanCluster = 8;

struct PrepArgs {
    const uint16_t* x;
    const int32_t* idx;
    int T, H, E, K, height;  // height: token rows of a group
    uint8_t* xq;             // [slots, H]: each pair's token, an expert's pairs one after the other
    float* xs;               // [slots, ceil(H / 128)]
    int32_t* pos;            // [T * K] slot of each pair, -1: none
    F8Group* groups;
    int* n_groups;
    uint32_t* err;
};

// off, goff = exclusive sums of the experts' pairs and groups (one warp, eight experts a lane); returns the
// number of groups in lane 31.
__device__ __forceinline__ int prep_scan(const int* cnt, int* off, int* goff, int height) {
    const int lane = threadIdx.x & 31;
    int c = 0, g = 0;
    for (int e = lane * 8; e < lane * 8 + 8; e++) c += cnt[e], g += (cnt[e] + height - 1) / height;
    int ci = c, gi = g;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, ci, o), z = __shfl_up_sync(0xffffffffu, gi, o);
        if (lane >= o) ci += y, gi += z;
    }
    c = ci - c, g = gi - g;
    for (int e = lane * 8; e < lane * 8 + 8; e++) {
        off[e] = c, goff[e] = g;
        c += cnt[e], g += (cnt[e] + height - 1) / height;
    }
    return gi;
}

// Quantises the tokens, sixteen lanes a group of 128 values, and stores each to the slots of its K pairs: the
// products then read an expert's rows as one matrix.  (Gathering the rows in the products, by TMA, took them
// 1.6 us a block of 128 rows where whole tiles take 0.8.)  slots[p - first] = slot of pair p; `v`, `g`: the
// thread's first values and group, already loaded.
struct PrepLoad {
    uint32_t g, stride, groups, per_row;
    uint4 v;
};
__device__ __forceinline__ uint4 prep_load(const PrepArgs& a, const PrepLoad& l, uint32_t g) {
    const uint32_t row = g / l.per_row, c = (g - row * l.per_row) * 128 + (threadIdx.x & 15) * 8;
    return g < l.groups && c < (uint32_t)a.H ? ld_cg_u4(a.x + (size_t)row * a.H + c) : make_uint4(0, 0, 0, 0);
}
__device__ __forceinline__ PrepLoad prep_begin(const PrepArgs& a) {
    PrepLoad l;
    l.per_row = (uint32_t)(a.H + 127) / 128;
    l.groups = (uint32_t)a.T * l.per_row;
    l.stride = gridDim.x * (kPrepThreads / 16);
    l.g = blockIdx.x * (kPrepThreads / 16) + threadIdx.x / 16;
    l.v = prep_load(a, l, l.g);
    return l;
}
__device__ __forceinline__ void prep_rows(const PrepArgs& a, PrepLoad l, const int* slots) {
    const uint32_t sub = threadIdx.x & 15;
    for (uint32_t g = l.g; g - threadIdx.x / 16 < l.groups; g += l.stride) {
        const uint32_t row = g / l.per_row, c = (g - row * l.per_row) * 128 + sub * 8;
        const bool in = g < l.groups && c < (uint32_t)a.H;
        const uint4 w = l.v;
        l.v = prep_load(a, l, g + l.stride);
        const float f[8] = {bf_lo(w.x), bf_hi(w.x), bf_lo(w.y), bf_hi(w.y), bf_lo(w.z), bf_hi(w.z), bf_lo(w.w), bf_hi(w.w)};
        bool special;
        uint32_t top = f8_top(w, special);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        const uint32_t se = f8_scale_exp(top);
        const uint2 q = f8_pack8(f, f8_inverse(se), special);
        if (g < l.groups)
            for (int k = 0; k < a.K; k++) {
                const int s = slots[row * a.K + k];
                if (s < 0) continue;
                if (in) *reinterpret_cast<uint2*>(a.xq + (size_t)s * a.H + c) = q;
                if (sub == 0) a.xs[(size_t)s * l.per_row + (g - row * l.per_row)] = __uint_as_float(se << 23);
            }
    }
}

// Few pairs: every CTA finds all pairs' slots itself, in the pairs' order within each expert (so that all
// agree), and quantises its share of the tokens; CTA 0 stores the slots and groups.
__global__ void __launch_bounds__(kPrepThreads) f8_prep_kernel(PrepArgs a) {
    __shared__ int wc[kPrepPairs / 32][kMaxExperts];  // pairs of each warp on each expert, then their exclusive sums
    __shared__ int cnt[kMaxExperts], off[kMaxExperts], goff[kMaxExperts], slots[kPrepPairs];
    griddep_launch_dependents();
    griddep_wait();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, P = a.T * a.K, warps = (P + 31) / 32;
    const int e = tid < P ? a.idx[tid] : -1;
    const PrepLoad l = prep_begin(a);
    for (int i = tid; i < warps * kMaxExperts; i += kPrepThreads) (&wc[0][0])[i] = 0;
    __syncthreads();
    const bool ok = e >= 0 && e < a.E;
    const uint32_t same = __match_any_sync(0xffffffffu, ok ? e : -1);
    const int before = __popc(same & ((1u << lane) - 1));
    if (ok && before == 0) wc[warp][e] = __popc(same);
    if (e >= a.E && blockIdx.x == 0) atomicOr(a.err, kErrBadIndex);
    __syncthreads();
    if (tid < kMaxExperts) {
        int n = 0;
        for (int w = 0; w < warps; w++) {
            const int t = wc[w][tid];
            wc[w][tid] = n;
            n += t;
        }
        cnt[tid] = n;
    }
    __syncthreads();
    if (tid < 32) {
        const int n = prep_scan(cnt, off, goff, a.height);
        if (tid == 31 && blockIdx.x == 0) *a.n_groups = n;
    }
    __syncthreads();
    const int slot = ok ? off[e] + wc[warp][e] + before : -1;
    if (tid < P) {
        slots[tid] = slot;
        if (blockIdx.x == 0) a.pos[tid] = slot;
    }
    if (blockIdx.x == 0 && tid < a.E)
        for (int g = 0; g * a.height < cnt[tid]; g++)
            a.groups[goff[tid] + g] = F8Group{off[tid] + g * a.height, min(a.height, cnt[tid] - g * a.height), tid, 0};
    __syncthreads();
    prep_rows(a, l, slots);
}

// A few tokens (up to 32 pairs, one a lane): each warp finds the slots by comparing its lanes, with no trip
// through shared memory, and quantises its share (of a lone token, a 4 us chain of barriers otherwise).
constexpr int kTinyThreads = 128;
__global__ void __launch_bounds__(kTinyThreads) f8_prep_tiny_kernel(PrepArgs a) {
    griddep_launch_dependents();
    griddep_wait();
    const int lane = threadIdx.x & 31, P = a.T * a.K;
    int e = lane < P ? a.idx[lane] : -1;
    const uint32_t per_row = (uint32_t)(a.H + 127) / 128, groups = (uint32_t)a.T * per_row, sub = threadIdx.x & 15;
    const uint32_t g = blockIdx.x * (kTinyThreads / 16) + threadIdx.x / 16, row = g / per_row, c = (g - row * per_row) * 128 + sub * 8;
    const bool in = g < groups && c < (uint32_t)a.H;
    const uint4 w = in ? ld_cg_u4(a.x + (size_t)row * a.H + c) : make_uint4(0, 0, 0, 0);
    const bool bad = e >= a.E;
    if (bad || e < 0) e = INT_MAX;
    const uint32_t same = __match_any_sync(0xffffffffu, e);
    const int rank = __popc(same & ((1u << lane) - 1)), of = __popc(same);
    // slots and groups of the experts before this one; a group holds up to `height` of an expert's pairs
    int slot = rank, group = 0;
#pragma unroll
    for (int i = 0; i < 32; i++) {
        const int o = __shfl_sync(0xffffffffu, e, i), r = __shfl_sync(0xffffffffu, rank, i);
        if (o < e) slot++, group += r % a.height == 0;
    }
    const bool ok = e != INT_MAX;
    if (blockIdx.x == 0 && threadIdx.x < 32) {
        if (bad) atomicOr(a.err, kErrBadIndex);
        if (lane < P) a.pos[lane] = ok ? slot : -1;
        const bool head = ok && rank % a.height == 0;
        if (head) a.groups[group + rank / a.height] = F8Group{slot, min(a.height, of - rank), e, 0};
        const int n = __popc(__ballot_sync(0xffffffffu, head));
        if (lane == 0) *a.n_groups = n;
    }
    const float f[8] = {bf_lo(w.x), bf_hi(w.x), bf_lo(w.y), bf_hi(w.y), bf_lo(w.z), bf_hi(w.z), bf_lo(w.w), bf_hi(w.w)};
    bool special;
    uint32_t top = f8_top(w, special);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    const uint32_t se = f8_scale_exp(top);
    const uint2 q = f8_pack8(f, f8_inverse(se), special);
    for (int k = 0; k < a.K; k++) {
        const int p = min((int)(row * a.K) + k, 31);  // rows behind the last token store nothing
        const int s = __shfl_sync(0xffffffffu, ok ? slot : -1, p);
        if (s < 0 || g >= groups) continue;
        if (in) *reinterpret_cast<uint2*>(a.xq + (size_t)s * a.H + c) = q;
        if (sub == 0) a.xs[(size_t)s * per_row + (g - row * per_row)] = __uint_as_float(se << 23);
    }
}

// Many pairs: one cluster finds the slots, an eighth of the pairs a CTA.  A pair's place among its CTA's pairs
// on the expert may differ from run to run: a slot's row is computed from that row alone, so no result does.
__global__ void __cluster_dims__(kPlanCluster, 1, 1) __launch_bounds__(kPrepThreads) f8_plan_kernel(PrepArgs a) {
    __shared__ int mine[kMaxExperts], cnt[kMaxExperts], off[kMaxExperts], goff[kMaxExperts];
    cg::cluster_group cl = cg::this_cluster();
    griddep_wait();
    griddep_launch_dependents();  // after the wait: the scatter kernel reads the tokens ahead of its own
    const int tid = threadIdx.x, rank = (int)cl.block_rank(), E = a.E;
    const int P = a.T * a.K, share = (P + kPlanCluster - 1) / kPlanCluster, first = min(P, rank * share), last = min(P, first + share);
    if (tid < kMaxExperts) mine[tid] = 0;
    __syncthreads();
    constexpr int U = 4;  // index loads in flight
    bool bad = false;
    for (int p0 = first + tid; p0 < last; p0 += U * kPrepThreads) {
        int e[U];
#pragma unroll
        for (int u = 0; u < U; u++) e[u] = p0 + u * kPrepThreads < last ? a.idx[p0 + u * kPrepThreads] : -1;
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int p = p0 + u * kPrepThreads;
            bad |= e[u] >= E;
            if (p < last) a.pos[p] = e[u] >= 0 && e[u] < E ? atomicAdd(&mine[e[u]], 1) : -1;
        }
    }
    if (bad) atomicOr(a.err, kErrBadIndex);
    cl.sync();
    int before = 0;  // pairs on expert tid of the CTAs before this one
    if (tid < kMaxExperts) {
        int n = 0;
#pragma unroll
        for (int r = 0; r < kPlanCluster; r++) {
            const int c = cl.map_shared_rank(mine, r)[tid];
            if (r < rank) before += c;
            n += c;
        }
        cnt[tid] = n;
    }
    __syncthreads();
    if (tid < 32) {
        const int n = prep_scan(cnt, off, goff, a.height);
        if (tid == 31 && rank == 0) *a.n_groups = n;
    }
    cl.sync();  // every CTA has read the others' counts
    if (tid < kMaxExperts) mine[tid] = off[tid] + before;
    __syncthreads();
    for (int p0 = first + tid; p0 < last; p0 += U * kPrepThreads) {
        int e[U], r[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int p = p0 + u * kPrepThreads;
            r[u] = p < last ? a.pos[p] : -1;
            e[u] = p < last ? a.idx[p] : -1;
        }
#pragma unroll
        for (int u = 0; u < U; u++)
            if (r[u] >= 0) a.pos[p0 + u * kPrepThreads] = mine[e[u]] + r[u];
    }
    if (tid < E)
        for (int g = rank; g * a.height < cnt[tid]; g += kPlanCluster)
            a.groups[goff[tid] + g] = F8Group{off[tid] + g * a.height, min(a.height, cnt[tid] - g * a.height), tid, 0};
}
__global__ void __launch_bounds__(kPrepThreads) f8_scatter_kernel(PrepArgs a) {
    griddep_launch_dependents();
    const PrepLoad l = prep_begin(a);  // tokens from before the plan kernel, past L1 (launch.cuh)
    griddep_wait();
    prep_rows(a, l, a.pos);
}

// out[t] = (out[t] +) sum_k w[t, k] y[slot of (t, k)], in order of k; four columns a thread.  Eight slots are
// looked up, and then eight rows read, at a time: two round trips to memory instead of two for each expert.  Three
// CTAs an SM, at 80 registers: with 88, and two, 65 us at 2048 tokens instead of 53.
__global__ void __launch_bounds__(256, 3) f8_combine_kernel(const float* y, const int32_t* pos, const float* w, int T, int K, int H,
                                                            void* out, bool f32, bool accumulate) {
    const int per = H / 4;
    const int64_t n = (int64_t)T * per;
    bool waited = false;  // slots, weights and sums are there when this kernel starts (launch.cuh), the rows after the wait
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) {
        const int64_t t = i / per;
        const int h = (int)(i - t * per) * 4;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (accumulate) v = __ldcg(reinterpret_cast<const float4*>(static_cast<const float*>(out) + t * H + h));
        for (int k0 = 0; k0 < K; k0 += 8) {
            int s[8];
            float c[8];
            float4 a[8];
            if (waited) {  // (through L1, which a CTA's warps share: 52 us at 2048 tokens, 55 past it)
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    s[k] = k0 + k < K ? pos[t * K + k0 + k] : -1;
                    c[k] = k0 + k < K ? w[t * K + k0 + k] : 0.f;
                }
            } else {
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    s[k] = k0 + k < K ? __ldcg(pos + t * K + k0 + k) : -1;
                    c[k] = k0 + k < K ? __ldcg(w + t * K + k0 + k) : 0.f;
                }
                griddep_wait();
                waited = true;
            }
#pragma unroll
            for (int k = 0; k < 8; k++)
                if (s[k] >= 0) a[k] = *reinterpret_cast<const float4*>(y + (size_t)s[k] * H + h);
#pragma unroll
            for (int k = 0; k < 8; k++)
                if (s[k] >= 0)
                    v.x = fmaf(c[k], a[k].x, v.x), v.y = fmaf(c[k], a[k].y, v.y), v.z = fmaf(c[k], a[k].z, v.z), v.w = fmaf(c[k], a[k].w, v.w);
        }
        if (f32) *reinterpret_cast<float4*>(static_cast<float*>(out) + t * H + h) = v;
        else *reinterpret_cast<uint2*>(static_cast<uint16_t*>(out) + t * H + h) = make_uint2(f8_bf16x2(v.x, v.y), f8_bf16x2(v.z, v.w));
    }
    if (!waited) griddep_wait();
}

namespace {

// Token rows of a group, by the pairs an expert gets on average: the few-row kernel on 16 or 32 of them, the many-row
// kernel on 128.  128 experts of 4096 x 1280, 8 a token, evenly (unevenly) routed, us at heights 16 / 32 / 128:
//   64 tokens 306 / 302 / 375 (156 / 161 / 189), 128 tokens 312 / 309 / 390 (213 / 210 / 235),
//   400 tokens 465 / 355 / 421 (430 / 366 / 368), 600 tokens 625 / 523 / 432 (575 / 466 / 435).
int group_height(int64_t pairs, int E) { return pairs <= 6ll * E ? 16 : pairs <= 28ll * E ? 32 : 128; }

struct Ws {
    uint8_t *xq, *aq;
    float *xs, *as, *y;
    int32_t* pos;
    F8Group* groups;
    int* n_groups;
    size_t bytes;
};
Ws experts_layout(void* ws, int T, int K, int H, int F, int E) {
    Ws w;
    char* p = static_cast<char*>(ws);
    size_t o = 0;
    auto take = [&](size_t n) {
        char* r = p + o;
        o += (n + 255) / 256 * 256;
        return r;
    };
    const size_t P = (size_t)T * K, hb = (H + 127) / 128, fb = (F + 127) / 128;
    w.xq = (uint8_t*)take(P * H);
    w.xs = (float*)take(4 * P * hb);
    w.aq = (uint8_t*)take(P * F);
    w.as = (float*)take(4 * P * fb);
    w.y = (float*)take(4 * P * H);
    w.pos = (int32_t*)take(4 * P);
    w.groups = (F8Group*)take(sizeof(F8Group) * (P / 16 + std::min<size_t>(E, P)));
    w.n_groups = (int*)take(4);
    w.bytes = o;
    return w;
}

template <int NQ>
cudaError_t products_few(const CUtensorMap (&m)[4], F8Gemm gu, F8Gemm dn, int64_t groups, int sm_count, cudaStream_t st) {
    const cudaError_t e = Few<kF8GateUp, NQ>::run(m[0], m[1], gu, groups * gu.nt, sm_count, st);
    return e != cudaSuccess ? e : Few<kF8Down, NQ>::run(m[2], m[3], dn, groups * dn.nt, sm_count, st);
}

}  // namespace

size_t experts_fp8_workspace(int T, int K, int H, int F, int E) { return experts_layout(nullptr, T, K, H, F, E).bytes; }

cudaError_t launch_experts_fp8(const ExpertsF8& a, int sm_count, cudaStream_t st, int* launches) {
    if (a.T <= 0) return cudaSuccess;
    EncodeTiledFn enc = tc_encode_fn();
    if (!enc) return cudaErrorNotSupported;
    const Ws w = experts_layout(a.ws, a.T, a.K, a.H, a.F, a.E);
    const int64_t P = (int64_t)a.T * a.K;
    const int height = group_height(P, a.E);
    const int64_t groups = std::min<int64_t>(a.E, P) + P / height;  // at most
    CUtensorMap m[4];
    if (!encode3(enc, &m[0], a.gu, a.H, a.F, 2 * (int64_t)a.E, 128) || !encode2(enc, &m[1], w.xq, a.H, P, height) ||
        !encode3(enc, &m[2], a.d, a.F, a.H, a.E, 128) || !encode2(enc, &m[3], w.aq, a.F, P, height))
        return cudaErrorInvalidValue;
    const PrepArgs pa{a.x, a.idx, a.T, a.H, a.E, a.K, height, w.xq, w.xs, w.pos, w.groups, w.n_groups, a.err};
    const int qctas = (int)std::min<int64_t>(((int64_t)a.T * ((a.H + 127) / 128) + kPrepThreads / 16 - 1) / (kPrepThreads / 16),
                                             2 * sm_count);
    cudaError_t e;
    if (P <= 32) {
        e = launch_after(f8_prep_tiny_kernel, (int)(((int64_t)a.T * ((a.H + 127) / 128) * 16 + kTinyThreads - 1) / kTinyThreads),
                         kTinyThreads, 0, 0, st, pa);
    } else if (P <= kPrepPairs) {
        e = launch_after(f8_prep_kernel, qctas, kPrepThreads, 0, 0, st, pa);
    } else {
        e = launch_after(f8_plan_kernel, kPlanCluster, kPrepThreads, 0, 0, st, pa);
        if (e == cudaSuccess) e = launch_after(f8_scatter_kernel, qctas, kPrepThreads, 0, 0, st, pa);
        ++*launches;
    }
    if (e != cudaSuccess) return e;

    F8Gemm gu{}, dn{};
    gu.xs = w.xs;
    gu.ws = a.gus;
    gu.nkb = (a.H + 127) / 128;
    gu.nb = gu.nt = (a.F + 127) / 128;
    gu.N = a.F;
    gu.groups = w.groups;
    gu.n_groups = w.n_groups;
    gu.aq = w.aq;
    gu.as = w.as;
    gu.err = a.err;
    gu.timeout_ns = a.timeout_ns;
    gu.inject = a.inject;
    dn = gu;
    dn.xs = w.as;
    dn.ws = a.ds;
    dn.nkb = (a.F + 127) / 128;
    dn.nb = dn.nt = (a.H + 127) / 128;
    dn.N = a.H;
    dn.out = w.y;
    dn.out_f32 = 1;
    if (height == 16) e = products_few<16>(m, gu, dn, groups, sm_count, st);
    else if (height == 32) e = products_few<32>(m, gu, dn, groups, sm_count, st);
    else {
        e = Many<kF8GateUp, 256>::run(m[0], m[1], gu, groups * gu.nt, sm_count, st);
        dn.nt = (a.H + 255) / 256;
        if (e == cudaSuccess) e = Many<kF8Down, 256>::run(m[2], m[3], dn, groups * dn.nt, sm_count, st);
    }
    if (e != cudaSuccess) return e;
    *launches += 4;
    return launch_after(f8_combine_kernel, (int)std::min<int64_t>(((int64_t)a.T * a.H / 4 + 255) / 256, sm_count * 8), 256, 0, 0, st,
                        (const float*)w.y, (const int32_t*)w.pos, a.w, a.T, a.K, a.H, a.out, a.out_f32, a.accumulate);
}

}  // namespace moe
