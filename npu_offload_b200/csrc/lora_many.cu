// Low-rank adapters for many tokens: tokens grouped by adapter, tiles of 64 tokens on the tensor cores.
//
//   low[t] = scale_i x[t] A_i^T;   out[t] = base[t] + low[t] B_i^T
//
// What bounds it is x, base and out, each moved once: with r of 8 to 128 there are r to 2 r flops a byte of those, a tenth of what
// a warp's mma.sync takes at the rate of HBM, so the products do not go through tensor memory.
//
// lora_plan_kernel (one CTA) counts the tokens of each adapter, puts tokens of one adapter side by side and lists the tiles.
// Places within an adapter go by integer atomics and may differ from run to run; no result does, since a token's
// sums do not depend on its place.
//
// lora_many_kernel: a cluster a tile.  Each of its CTAs
//   1. multiplies its share of the inner dimension: 128 columns of x's 64 rows (gathered) and of A's r rows a stage, cp.async,
//      a warp 16 tokens and half a stage's columns;
//   2. sends its partial sums to the CTA that owns the tokens, which adds them in order, multiplies by the scale, splits each
//      into bf16 parts (two for a bf16 result: 2^-17 of low; three for an fp32 one: 2^-24) and sends them to all;
//   3. multiplies its share of B's columns: a warp 32 tokens and 16 bytes of four lanes' columns, read and written in whole
//      sectors: the columns of B are dealt to the matrix instruction so that a lane's results are neighbours, as are its inner
//      values, eight bytes of a row of B.
#include <cooperative_groups.h>

#include <algorithm>

#include "common.cuh"
#include "fp8.cuh"
#include "launch.cuh"
#include "lora.h"
#include "ptx.cuh"

namespace cg = cooperative_groups;

namespace moe {

constexpr int kTile = 64;                    // tokens
constexpr int kManyThreads = 256;
constexpr int kManyCluster = 8;
constexpr int kOwned = kTile / kManyCluster; // tokens whose sums a CTA adds
constexpr int kStageCols = 128;
constexpr int kPlanThreads = 1024;

static_assert(kLoraMaxTokens / kTile + kLoraMaxAdapters + 1 < 65536, "tiles are counted in 16 bits");
struct __align__(16) LoraTile {
    int32_t adapter, first, count, pad;  // adapter -1: tokens without one
};
struct LoraWs {
    LoraTile* tiles;   // [max_tiles]
    int32_t* order;    // [T] tokens, an adapter's side by side, those without one last
    int32_t* n_tiles;  // [1]
    size_t bytes;
};
static int lora_max_tiles(int T, int n) { return T / kTile + std::min(n + 1, T); }
static LoraWs lora_layout(void* ws, int T, int n) {
    LoraWs w;
    char* p = static_cast<char*>(ws);
    size_t o = 0;
    auto take = [&](size_t bytes) {
        char* at = p + o;
        o += (bytes + 255) / 256 * 256;
        return at;
    };
    w.tiles = (LoraTile*)take(sizeof(LoraTile) * lora_max_tiles(T, n));
    w.order = (int32_t*)take(sizeof(int32_t) * T);
    w.n_tiles = (int32_t*)take(sizeof(int32_t));
    w.bytes = o;
    return w;
}
size_t lora_many_workspace(int T, int n) { return lora_layout(nullptr, T, n).bytes; }

__global__ void __launch_bounds__(kPlanThreads) lora_plan_kernel(LoraArgs a, LoraWs ws) {
    __shared__ int count[kLoraMaxAdapters + 1], place[kLoraMaxAdapters + 1];
    __shared__ uint16_t tile0[kLoraMaxAdapters + 1];
    __shared__ unsigned long long warp_sum_s[kPlanThreads / 32];
    griddep_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, bins = a.n + 1;
    const bool copies = a.out != a.base;
    for (int i = tid; i < bins; i += kPlanThreads) count[i] = 0;
    __syncthreads();
    const int rounds = (a.T + kPlanThreads - 1) / kPlanThreads;
    auto bin_of = [&](int t) {  // a.n: no adapter
        const int id = a.ids[t];
        if (id >= a.n) atomicOr(a.err, kErrBadIndex);
        return id < 0 || id >= a.n ? a.n : id;
    };
    for (int i = 0; i < rounds; i++) {
        const int t = i * kPlanThreads + tid, bin = t < a.T ? bin_of(t) : -1;
        const unsigned same = __match_any_sync(0xffffffffu, bin);
        if (bin >= 0 && __ffs(same) - 1 == lane) atomicAdd(&count[bin], __popc(same));
    }
    __syncthreads();
    // places and tiles before each bin, bins in order: a few bins a thread, then warps, then the CTA
    const int per = (bins + kPlanThreads - 1) / kPlanThreads, b0 = min(tid * per, bins), b1 = min(b0 + per, bins);
    auto weight = [&](int b) {
        const int tiles = b < a.n || copies ? (count[b] + kTile - 1) / kTile : 0;
        return (unsigned long long)tiles << 32 | (unsigned)count[b];
    };
    unsigned long long sum = 0;
    for (int b = b0; b < b1; b++) sum += weight(b);
    unsigned long long upto = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
    }
    if (lane == 31) warp_sum_s[warp] = upto;
    __syncthreads();
    if (warp == 0) {
        unsigned long long v = warp_sum_s[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned long long u = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += u;
        }
        warp_sum_s[lane] = v;
    }
    __syncthreads();
    unsigned long long at = upto - sum + (warp ? warp_sum_s[warp - 1] : 0);
    for (int b = b0; b < b1; b++) {
        place[b] = (int)(unsigned)at;
        tile0[b] = (uint16_t)(at >> 32);
        at += weight(b);
    }
    const int tiles = (int)(warp_sum_s[kPlanThreads / 32 - 1] >> 32);
    if (tid == 0) *ws.n_tiles = tiles;
    __syncthreads();
    for (int i = tid; i < tiles; i += kPlanThreads) {
        int lo = 0, hi = bins - 1;  // the last bin with tile0 <= i: it has tiles, since those behind begin later
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (tile0[mid] <= i) lo = mid;
            else hi = mid - 1;
        }
        const int j = i - tile0[lo];
        ws.tiles[i] = LoraTile{lo < a.n ? lo : -1, place[lo] + j * kTile, min(kTile, count[lo] - j * kTile), 0};
    }
    __syncthreads();
    for (int i = 0; i < rounds; i++) {
        const int t = i * kPlanThreads + tid, id = t < a.T ? a.ids[t] : 0;
        const int bin = t >= a.T ? -1 : id < 0 || id >= a.n ? a.n : id;
        const unsigned same = __match_any_sync(0xffffffffu, bin);
        const int leader = __ffs(same) - 1;
        int base = 0;
        if (bin >= 0 && leader == lane) base = atomicAdd(&place[bin], __popc(same));
        base = __shfl_sync(0xffffffffu, base, leader);
        if (bin >= 0) ws.order[base + __popc(same & ((1u << lane) - 1))] = t;
    }
}

// 16 bytes to shared memory, zeros where !in.
__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void* src, bool in) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// c [16, 8] += a [16, 16] b [16, 8]
__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// R: r rounded up to 16, 32, 64 or 128.
template <int R>
struct ManySmem {
    static constexpr int kStages = R <= 16 ? 4 : R <= 64 ? 3 : 2;
    static constexpr int kStageBytes = (kTile + R) * kStageCols * 2;
    static constexpr int kSlots = 2 * kManyCluster;           // partial sums of a token: a half stage of each CTA
    static constexpr int kSlotBytes = kOwned * R * 4;
    static constexpr int kPitch = R * 2 + 16;                 // of a row of a part: ldmatrix's eight rows on different banks
    static constexpr int kPartBytes = kTile * kPitch;
    static constexpr int kOffSlots = kStages * kStageBytes;
    static constexpr int kOffParts = kOffSlots + kSlots * kSlotBytes;
    static constexpr int kOffTok = kOffParts + 3 * kPartBytes;
    static constexpr int kBytes = kOffTok + kTile * 4;
};

template <int R, bool F32>
__global__ void __cluster_dims__(kManyCluster, 1, 1) __launch_bounds__(kManyThreads) lora_many_kernel(LoraArgs a, LoraWs ws) {
    using S = ManySmem<R>;
    extern __shared__ __align__(128) unsigned char smem[];
    griddep_wait();
    cg::cluster_group cl = cg::this_cluster();
    const int c = (int)cl.block_rank(), i_tile = blockIdx.x / kManyCluster;
    if (i_tile >= __ldcg(ws.n_tiles)) return;  // the whole cluster alike
    const int4 listed = __ldcg(reinterpret_cast<const int4*>(ws.tiles + i_tile));
    const LoraTile tile{listed.x, listed.y, listed.z, 0};
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, r = a.r, N = a.N;
    int* tok = reinterpret_cast<int*>(smem + S::kOffTok);
    if (tid < kTile) tok[tid] = __ldcg(ws.order + tile.first + min(tid, tile.count - 1));
    __syncthreads();
    constexpr int W = F32 ? 4 : 8;  // neighbours of a lane: 16 bytes
    constexpr int kGroup = 4 * W;   // columns of a warp's task
    const bool vec = N % W == 0;
    const int groups = (N + kGroup - 1) / kGroup;
    const int g0 = (int)((int64_t)c * groups / kManyCluster), g1 = (int)((int64_t)(c + 1) * groups / kManyCluster);
    if (tile.adapter < 0) {
        const int c0 = g0 * kGroup, c1 = min(g1 * kGroup, N), step = vec ? W : 1, each = max(0, c1 - c0) / step;
        for (int i = tid; i < each * tile.count; i += kManyThreads) {
            const size_t at = (size_t)tok[i / each] * N + c0 + (i % each) * step;
            if (vec && F32) *reinterpret_cast<uint4*>(static_cast<float*>(a.out) + at) = ld_cg_u4(static_cast<const float*>(a.base) + at);
            else if (vec) *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + at) = ld_cg_u4(static_cast<const uint16_t*>(a.base) + at);
            else if (F32) static_cast<float*>(a.out)[at] = static_cast<const float*>(a.base)[at];
            else static_cast<uint16_t*>(a.out)[at] = static_cast<const uint16_t*>(a.base)[at];
        }
        return;
    }
    const uint16_t* A = a.a + (size_t)tile.adapter * r * a.K;
    const uint16_t* B = a.b + (size_t)tile.adapter * N * r;

    // ---- 1: this CTA's share of x A^T
    const int U = a.K / 8, u0 = (int)((int64_t)c * U / kManyCluster), u1 = (int)((int64_t)(c + 1) * U / kManyCluster);
    const int stages = (u1 - u0 + 15) / 16;
    const uint32_t s_base = smem_u32(smem);
    auto ask = [&](int s) {  // words of 16 bytes, word w of row q at w ^ (q & 7)
        if (s < stages) {
            const uint32_t buf = s_base + (s % S::kStages) * S::kStageBytes;
            const int w = tid & 15, u = u0 + s * 16 + w;
#pragma unroll
            for (int i = 0; i < (kTile + R) / 16; i++) {
                const int q = (tid >> 4) + i * 16;
                const bool token = q < kTile, in = u < u1 && (token ? q < tile.count : q - kTile < r);
                const uint16_t* src = token ? a.x + (size_t)tok[q & (kTile - 1)] * a.K : A + (size_t)(q - kTile) * a.K;
                cp_async16_or_zero(buf + q * (kStageCols * 2) + (w ^ (q & 7)) * 16, in ? src + (size_t)u * 8 : a.x, in);
            }
        }
        cp_async_commit();
    };
    float acc[R / 8][4];
#pragma unroll
    for (int j = 0; j < R / 8; j++) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
#pragma unroll
    for (int s = 0; s < S::kStages - 1; s++) ask(s);
    const int mt = warp & 3, half = warp >> 2;
    for (int s = 0; s < stages; s++) {
        cp_async_wait<S::kStages - 2>();
        __syncthreads();  // stage s is there; stage s - 1, whose buffer comes next, has been used
        ask(s + S::kStages - 1);
        const uint32_t buf = s_base + (s % S::kStages) * S::kStageBytes;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int w = (half * 4 + k) * 2;
            uint32_t xa[4];
            const int q = mt * 16 + (lane & 15);
            ldmatrix4(xa, buf + q * (kStageCols * 2) + ((w + (lane >> 4)) ^ (q & 7)) * 16);
#pragma unroll
            for (int j = 0; j < R / 8; j += 2) {
                uint32_t ab[4];
                const int p = kTile + j * 8 + (lane & 7) + ((lane >> 4) << 3);
                ldmatrix4(ab, buf + p * (kStageCols * 2) + ((w + ((lane >> 3) & 1)) ^ (p & 7)) * 16);
                mma_bf16(acc[j], xa, ab[0], ab[1]);
                mma_bf16(acc[j + 1], xa, ab[2], ab[3]);
            }
        }
    }

    // ---- 2: sums over the cluster, in order, and their bf16 parts to all
    cl.sync();  // every CTA has begun: its shared memory may be written to
    {
        float* slots = reinterpret_cast<float*>(smem + S::kOffSlots);
        const int slot = c * 2 + half;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int row = mt * 16 + (lane >> 2) + 8 * h;
            float* to = cl.map_shared_rank(slots, row / kOwned) + (size_t)(slot * kOwned + row % kOwned) * R + (lane & 3) * 2;
#pragma unroll
            for (int j = 0; j < R / 8; j++) *reinterpret_cast<float2*>(to + j * 8) = make_float2(acc[j][2 * h], acc[j][2 * h + 1]);
        }
    }
    cl.sync();
    {
        const float* slots = reinterpret_cast<const float*>(smem + S::kOffSlots);
        const float scale = a.scale ? a.scale[tile.adapter] : 1.f;
        for (int i = tid; i < kOwned * R / 2; i += kManyThreads) {
            const int row = i / (R / 2), col = (i % (R / 2)) * 2;
            float v0 = 0.f, v1 = 0.f;
#pragma unroll
            for (int s = 0; s < S::kSlots; s++) {
                const float2 p = *reinterpret_cast<const float2*>(slots + (size_t)(s * kOwned + row) * R + col);
                v0 += p.x, v1 += p.y;
            }
            v0 *= scale, v1 *= scale;
            // of 16 inner values 4 q + {0, 1, 2, 3} take the places 2 q + {0, 1} and 8 + 2 q + {0, 1}, those of one lane
            const int in16 = col & 15, to = (col & ~15) + (in16 & 2) * 4 + (in16 >> 2) * 2;
            unsigned char* dst = smem + S::kOffParts + (c * kOwned + row) * S::kPitch + to * 2;
#pragma unroll
            for (int part = 0; part < (F32 ? 3 : 2); part++) {
                const uint32_t b = f8_bf16x2(v0, v1);
                v0 -= bf_lo(b), v1 -= bf_hi(b);
#pragma unroll
                for (int d = 0; d < kManyCluster; d++) *reinterpret_cast<uint32_t*>(cl.map_shared_rank(dst + part * S::kPartBytes, d)) = b;
            }
        }
    }
    cl.sync();

    // ---- 3: this CTA's columns of low B^T
    const int halves = tile.count > 32 ? 2 : 1;
    const int q = lane & 3, i8 = lane >> 2;
    for (int task = warp; task < (g1 - g0) * halves; task += kManyThreads / 32) {
        const int col0 = (g0 + task / halves) * kGroup, m0 = (task % halves) * 32;
        uint4 base[2][2];
        bool in[2][2];
#pragma unroll
        for (int m = 0; m < 2; m++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int row = m0 + m * 16 + h * 8 + i8;
                in[m][h] = row < tile.count && col0 + W * q < N;
                base[m][h] = make_uint4(0, 0, 0, 0);
                if (in[m][h] && vec) {
                    const size_t at = (size_t)tok[row] * N + col0 + W * q;
                    base[m][h] = F32 ? ld_cg_u4(static_cast<const float*>(a.base) + at) : ld_cg_u4(static_cast<const uint16_t*>(a.base) + at);
                }
            }
        float o[2][W / 2][4];
#pragma unroll
        for (int m = 0; m < 2; m++)
#pragma unroll
            for (int j = 0; j < W / 2; j++) o[m][j][0] = o[m][j][1] = o[m][j][2] = o[m][j][3] = 0.f;
#pragma unroll
        for (int k = 0; k < R / 16; k++) {
            uint2 bv[W / 2];
#pragma unroll
            for (int j = 0; j < W / 2; j++) {
                const int n = col0 + W * (i8 >> 1) + 2 * j + (i8 & 1);
                bv[j] = make_uint2(0, 0);
                if (n < N && k * 16 + 4 * q < r) bv[j] = *reinterpret_cast<const uint2*>(B + (size_t)n * r + k * 16 + 4 * q);
            }
#pragma unroll
            for (int part = 0; part < (F32 ? 3 : 2); part++)
#pragma unroll
                for (int m = 0; m < 2; m++) {
                    uint32_t la[4];
                    ldmatrix4(la, s_base + S::kOffParts + part * S::kPartBytes + (m0 + m * 16 + (lane & 15)) * S::kPitch + k * 32 + (lane >> 4) * 16);
#pragma unroll
                    for (int j = 0; j < W / 2; j++) mma_bf16(o[m][j], la, bv[j].x, bv[j].y);
                }
        }
#pragma unroll
        for (int m = 0; m < 2; m++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                if (!in[m][h]) continue;
                const size_t at = (size_t)tok[m0 + m * 16 + h * 8 + i8] * N + col0 + W * q;
                float v[W];
#pragma unroll
                for (int j = 0; j < W / 2; j++) v[2 * j] = o[m][j][2 * h], v[2 * j + 1] = o[m][j][2 * h + 1];
                if (vec) {
                    const uint32_t b[4] = {base[m][h].x, base[m][h].y, base[m][h].z, base[m][h].w};
                    if constexpr (F32) {
                        *reinterpret_cast<float4*>(static_cast<float*>(a.out) + at) =
                            make_float4(__uint_as_float(b[0]) + v[0], __uint_as_float(b[1]) + v[1], __uint_as_float(b[2]) + v[2], __uint_as_float(b[3]) + v[3]);
                    } else {
                        uint32_t w[4];
#pragma unroll
                        for (int j = 0; j < 4; j++) w[j] = f8_bf16x2(bf_lo(b[j]) + v[2 * j], bf_hi(b[j]) + v[2 * j + 1]);
                        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + at) = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < W; j++)
                        if (col0 + W * q + j < N) {
                            if (F32) static_cast<float*>(a.out)[at + j] = static_cast<const float*>(a.base)[at + j] + v[j];
                            else static_cast<uint16_t*>(a.out)[at + j] = f8_bf16(bf2f(static_cast<const uint16_t*>(a.base)[at + j]) + v[j]);
                        }
                }
            }
    }
}

template <int R, bool F32>
static cudaError_t many_for(const LoraArgs& a, const LoraWs& ws, cudaStream_t st) {
    const cudaError_t e = allow_smem<lora_many_kernel<R, F32>>(ManySmem<R>::kBytes);
    if (e != cudaSuccess) return e;
    const Launch l{lora_max_tiles(a.T, a.n) * kManyCluster, kManyThreads, ManySmem<R>::kBytes, 0, st};
    return l.run(lora_many_kernel<R, F32>, a, ws);
}

cudaError_t launch_lora_many(const LoraArgs& a, cudaStream_t st, int* launches) {
    const LoraWs ws = lora_layout(a.ws, a.T, a.n);
    const Launch l{1, kPlanThreads, 0, 0, st};
    cudaError_t e = l.run(lora_plan_kernel, a, ws);
    if (e != cudaSuccess) return e;
    ++*launches;
    if (a.r <= 16) e = a.out_f32 ? many_for<16, true>(a, ws, st) : many_for<16, false>(a, ws, st);
    else if (a.r <= 32) e = a.out_f32 ? many_for<32, true>(a, ws, st) : many_for<32, false>(a, ws, st);
    else if (a.r <= 64) e = a.out_f32 ? many_for<64, true>(a, ws, st) : many_for<64, false>(a, ws, st);
    else e = a.out_f32 ? many_for<128, true>(a, ws, st) : many_for<128, false>(a, ws, st);
    if (e == cudaSuccess) ++*launches;
    return e;
}

}  // namespace moe
