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
// lora_low_kernel, a cluster of eight or four CTAs a tile: low.  A CTA multiplies its share of the inner dimension, 64 columns of x's 64
// rows (gathered) and of A's r rows a stage, cp.async, a warp 16 tokens; the sums go to the CTA that owns the tokens, which adds them
// in order, multiplies by the scale and splits each into bf16 parts of its own sign (two for a bf16 result, which hold low to 2^-16; three
// for an fp32 one, which hold all of its 24 bits), stored as the fragments that the matrix instruction takes, 16 bytes a lane.  (Three
// for a bf16 result too: 23.8 instead of 23.3 us at 4093 tokens of r = 16, 46.7 / 42.0 at 4096 of r = 64, 58.4 / 50.6 at 2048 of r = 128.)
// lora_out_kernel, a CTA 32 tokens (64 from r = 64 on) and four warps' columns: out.  A warp reads and writes 16 bytes of four lanes a row, whole
// sectors: the columns of B are dealt to the matrix instruction so that a lane's results are neighbours, as are its inner values,
// eight bytes of a row of B.  base and B are asked for ahead of the wait for lora_low_kernel.
//
// 4093 tokens, 4096 x 16 x 2560: 23.4 us, 12 of them the first two kernels; x, base and out alone take 11.8 at a copy's rate.  (One
// kernel for low and out, the cluster going on to its columns: 26 to 29 us, since all CTAs load, exchange and store at the same time.)
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
constexpr int kLowThreads = 128;
constexpr int kOutThreads = 128;
constexpr int kStageCols = 64;
constexpr int kPlanThreads = 1024;

static_assert(kLoraMaxTokens / kTile + kLoraMaxAdapters + 1 < 65536, "tiles are counted in 16 bits");
struct __align__(8) LoraTile {
    int32_t adapter, count;  // adapter -1: tokens without one
};
struct LoraWs {
    LoraTile* tiles;   // [max_tiles]
    int32_t* order;    // [max_tiles][64] a tile's tokens
    int32_t* n_tiles;  // [1]
    uint4* low;        // [max_tiles][4 rows of 16][R / 16][parts][32 lanes]
    size_t bytes;
};
static int lora_max_tiles(int T, int n) { return T / kTile + std::min(n + 1, T); }
static int lora_padded(int r) { return r <= 16 ? 16 : r <= 32 ? 32 : r <= 64 ? 64 : 128; }
static LoraWs lora_layout(void* ws, int T, int n, int r) {
    LoraWs w;
    char* p = static_cast<char*>(ws);
    size_t o = 0;
    auto take = [&](size_t bytes) {
        char* at = p + o;
        o += (bytes + 255) / 256 * 256;
        return at;
    };
    w.tiles = (LoraTile*)take(sizeof(LoraTile) * lora_max_tiles(T, n));
    w.order = (int32_t*)take(sizeof(int32_t) * lora_max_tiles(T, n) * kTile);
    w.n_tiles = (int32_t*)take(sizeof(int32_t));
    w.low = (uint4*)take(sizeof(uint4) * lora_max_tiles(T, n) * 4 * (lora_padded(r) / 16) * 3 * 32);
    w.bytes = o;
    return w;
}
size_t lora_many_workspace(int T, int n, int r) { return lora_layout(nullptr, T, n, r).bytes; }

__global__ void __launch_bounds__(kPlanThreads) lora_plan_kernel(LoraArgs a, LoraWs ws) {
    __shared__ int count[kLoraMaxAdapters + 1], place[kLoraMaxAdapters + 1];
    __shared__ uint16_t tile0[kLoraMaxAdapters + 1];
    __shared__ int warp_sum_s[kPlanThreads / 32];
    griddep_wait();
    griddep_launch_dependents();  // the tiles' kernel waits for this one's end before it does anything
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, bins = a.n + 1;
    const bool copies = a.out != a.base;
    for (int i = tid; i < bins; i += kPlanThreads) count[i] = 0;
    __syncthreads();
    // Four neighbouring tokens a thread, 4096 a round; a.n: no adapter, -1: no token.  A warp of one adapter's tokens counts and places
    // them at once, a thread of one adapter's its four, others one by one.
    const int rounds = (a.T + 4 * kPlanThreads - 1) / (4 * kPlanThreads);
    const bool vec = (uintptr_t)a.ids % 16 == 0;
    bool wrong = false;
    auto bins_of = [&](int t, int (&bin)[4]) {
        int4 id = make_int4(-1, -1, -1, -1);
        if (vec && t + 4 <= a.T) {
            id = *reinterpret_cast<const int4*>(a.ids + t);
        } else {
            if (t < a.T) id.x = a.ids[t];
            if (t + 1 < a.T) id.y = a.ids[t + 1];
            if (t + 2 < a.T) id.z = a.ids[t + 2];
            if (t + 3 < a.T) id.w = a.ids[t + 3];
        }
        const int v[4] = {id.x, id.y, id.z, id.w};
#pragma unroll
        for (int k = 0; k < 4; k++) {
            wrong |= v[k] >= a.n;
            bin[k] = t + k >= a.T ? -1 : v[k] < 0 || v[k] >= a.n ? a.n : v[k];
        }
    };
    auto alike = [&](const int (&bin)[4]) { return bin[0] >= 0 && bin[0] == bin[1] && bin[0] == bin[2] && bin[0] == bin[3]; };
    auto warp_alike = [&](const int (&bin)[4]) {
        const int first = __shfl_sync(0xffffffffu, bin[0], 0);  // (by all lanes, whatever their own four are)
        return __all_sync(0xffffffffu, alike(bin) && bin[0] == first);
    };
#pragma unroll 1
    for (int i = 0; i < rounds; i++) {
        int bin[4];
        bins_of((i * kPlanThreads + tid) * 4, bin);
        if (warp_alike(bin)) {
            if (lane == 0) atomicAdd(&count[bin[0]], 128);
        } else if (alike(bin)) {
            atomicAdd(&count[bin[0]], 4);
        } else {
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (bin[k] >= 0) atomicAdd(&count[bin[k]], 1);
        }
    }
    if (wrong) atomicOr(a.err, kErrBadIndex);
    __syncthreads();
    // tiles before each bin, bins in order: a few bins a thread, then warps, then the CTA
    const int per = (bins + kPlanThreads - 1) / kPlanThreads, b0 = min(tid * per, bins), b1 = min(b0 + per, bins);
    auto weight = [&](int b) { return b < a.n || copies ? (count[b] + kTile - 1) / kTile : 0; };
    int sum = 0;
#pragma unroll 1
    for (int b = b0; b < b1; b++) sum += weight(b);
    int upto = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
    }
    if (lane == 31) warp_sum_s[warp] = upto;
    __syncthreads();
    int before = lane < kPlanThreads / 32 ? warp_sum_s[lane] : 0, tiles = before;  // by every warp for itself
    before = lane < warp ? before : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        before += __shfl_xor_sync(0xffffffffu, before, o);
        tiles += __shfl_xor_sync(0xffffffffu, tiles, o);
    }
    int at = before + upto - sum;
#pragma unroll 1
    for (int b = b0; b < b1; b++) {
        tile0[b] = (uint16_t)at;
        place[b] = at * kTile;
        at += weight(b);
    }
    if (tid == 0) *ws.n_tiles = tiles;
    __syncthreads();
#pragma unroll 1
    for (int i = tid; i < tiles; i += kPlanThreads) {
        int lo = 0, hi = bins - 1;  // the last bin with tile0 <= i: it has tiles, since those behind begin later
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (tile0[mid] <= i) lo = mid;
            else hi = mid - 1;
        }
        const int j = i - tile0[lo];
        ws.tiles[i] = LoraTile{lo < a.n ? lo : -1, min(kTile, count[lo] - j * kTile)};
    }
#pragma unroll 1
    for (int i = 0; i < rounds; i++) {
        const int t = (i * kPlanThreads + tid) * 4;
        int bin[4], at[4];
        bins_of(t, bin);
        if (warp_alike(bin)) {
            if (lane == 0) at[0] = atomicAdd(&place[bin[0]], 128);
            at[0] = __shfl_sync(0xffffffffu, at[0], 0) + lane * 4;
            at[1] = at[0] + 1, at[2] = at[0] + 2, at[3] = at[0] + 3;
        } else if (alike(bin)) {
            at[0] = atomicAdd(&place[bin[0]], 4);
            at[1] = at[0] + 1, at[2] = at[0] + 2, at[3] = at[0] + 3;
        } else {
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (bin[k] >= 0) at[k] = atomicAdd(&place[bin[k]], 1);
        }
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (bin[k] >= 0 && (bin[k] < a.n || copies)) ws.order[at[k]] = t + k;
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

// The first bf16 part of v, in the upper half: v cut to eight bits, or, where nothing would be left, the next smaller.  So the rest has
// v's sign and is 0 with v alone (from 2^-119 on, where all parts are within bf16's range), and an infinity of B times
// the parts is the infinity that it is times v; an infinite v is each part.
__device__ __forceinline__ uint32_t lora_lead(float v) {
    const uint32_t u = __float_as_uint(v);
    return u & 0xffffu || (u << 1) == 0 || !(fabsf(v) < INFINITY) ? u & 0xffff0000u : u - 0x10000u;
}

// R: r rounded up to 16, 32, 64 or 128.  The sums lie where the stages were: nothing is sent before every CTA of the
// cluster is through with those.
template <int R>
struct LowSmem {
    static constexpr int kStages = R <= 32 ? 4 : 3;  // (four CTAs an SM at r = 64: the 576 of 4093 tokens in one round, 34.6 instead of 43.6 us; two: 35.8)
    static constexpr int kStageBytes = (kTile + R) * kStageCols * 2;
    static constexpr int kOffTok = kStages * kStageBytes;
    static constexpr int kBytes = kOffTok + kTile * 4;
    static_assert(kTile * R * 4 <= kOffTok, "the sums fit in the stages");
};

template <int R, int PARTS, int CL>
__global__ void __cluster_dims__(CL, 1, 1) __launch_bounds__(kLowThreads) lora_low_kernel(LoraArgs a, LoraWs ws) {
    using S = LowSmem<R>;
    constexpr int kOwned = kTile / CL;  // tokens whose sums a CTA adds
    extern __shared__ __align__(128) unsigned char smem[];
    griddep_wait();
    griddep_launch_dependents();  // lora_out_kernel waits for this one's end before it reads low
    cg::cluster_group cl = cg::this_cluster();
    const int c = (int)cl.block_rank(), tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, r = a.r;
    const int n_tiles = __ldcg(ws.n_tiles), U = a.K / 8;
    const int u0 = (int)((int64_t)c * U / CL), u1 = (int)((int64_t)(c + 1) * U / CL), stages = (u1 - u0 + 7) / 8;
    int* tok = reinterpret_cast<int*>(smem + S::kOffTok);
    const uint32_t s_base = smem_u32(smem);
    for (int i_tile = blockIdx.x / CL; i_tile < n_tiles; i_tile += gridDim.x / CL) {  // the whole cluster alike
        const int token = tid < kTile ? __ldcg(ws.order + i_tile * kTile + tid) : 0;  // (of no meaning behind the tile's count)
        const int2 tile = __ldcg(reinterpret_cast<const int2*>(ws.tiles + i_tile));   // adapter, count
        if (tile.x < 0) continue;
        if (tid < kTile) tok[tid] = token;
        __syncthreads();
        const uint16_t* A = a.a + (size_t)tile.x * r * a.K;
        auto ask = [&](int s) {  // words of 16 bytes, word w of row q at w ^ (q & 7)
            if (s < stages) {
                const uint32_t buf = s_base + (s % S::kStages) * S::kStageBytes;
                const int w = tid & 7, u = u0 + s * 8 + w;
#pragma unroll
                for (int i = 0; i < (kTile + R) / 16; i++) {
                    const int q = (tid >> 3) + i * 16;
                    const bool token = q < kTile, in = u < u1 && (token ? q < tile.y : q - kTile < r);
                    const uint16_t* src = token ? a.x + (size_t)tok[q & (kTile - 1)] * a.K : A + (size_t)(q - kTile) * a.K;
                    cp_async16_or_zero(buf + q * (kStageCols * 2) + (w ^ (q & 7)) * 16, in ? src + (size_t)u * 8 : a.x, in);
                }
            }
            cp_async_commit();
        };
        float acc[R / 8][4];
#pragma unroll
        for (int j = 0; j < R / 8; j++) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
#pragma unroll 1
        for (int s = 1 - S::kStages; s < stages; s++) {
            if (s >= 0) {
                cp_async_wait<S::kStages - 2>();
                __syncthreads();  // stage s is there; stage s - 1, whose buffer comes next, has been used
            }
            ask(s + S::kStages - 1);
            if (s < 0) continue;
            const uint32_t buf = s_base + (s % S::kStages) * S::kStageBytes;
#pragma unroll
            for (int k = 0; k < kStageCols / 16; k++) {
                uint32_t xa[4];
                const int q = warp * 16 + (lane & 15);
                ldmatrix4(xa, buf + q * (kStageCols * 2) + ((2 * k + (lane >> 4)) ^ (q & 7)) * 16);
#pragma unroll
                for (int j = 0; j < R / 8; j += 2) {
                    uint32_t ab[4];
                    const int p = kTile + j * 8 + (lane & 7) + ((lane >> 4) << 3);
                    ldmatrix4(ab, buf + p * (kStageCols * 2) + ((2 * k + ((lane >> 3) & 1)) ^ (p & 7)) * 16);
                    mma_bf16(acc[j], xa, ab[0], ab[1]);
                    mma_bf16(acc[j + 1], xa, ab[2], ab[3]);
                }
            }
        }
        cl.sync();  // every CTA is through with its stages: their memory may be written to
        float* slots = reinterpret_cast<float*>(smem);
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int row = warp * 16 + (lane >> 2) + 8 * h;
            float* to = cl.map_shared_rank(slots, row / kOwned) + (size_t)(c * kOwned + row % kOwned) * R + (lane & 3) * 2;
#pragma unroll
            for (int j = 0; j < R / 8; j++) *reinterpret_cast<float2*>(to + j * 8) = make_float2(acc[j][2 * h], acc[j][2 * h + 1]);
        }
        cl.sync();
        const float scale = a.scale ? a.scale[tile.x] : 1.f;
        for (int i = tid; i < kOwned * R / 2; i += kLowThreads) {
            const int owned = i / (R / 2), col = (i % (R / 2)) * 2, row = c * kOwned + owned;
            float v0 = 0.f, v1 = 0.f;
#pragma unroll
            for (int s = 0; s < CL; s++) {
                const float2 p = *reinterpret_cast<const float2*>(slots + (size_t)(s * kOwned + owned) * R + col);
                v0 += p.x, v1 += p.y;
            }
            v0 *= scale, v1 *= scale;
            if (col >= r) v0 = v1 = 0.f;  // (an infinity or NaN in x or the scale makes NaN of the zero rows behind A's r)
            // of 16 inner values 4 q + {0, 1, 2, 3} are lane q's: the first two where the instruction has 2 q, the others where it has 2 q + 8
            const int to_lane = (row & 7) * 4 + ((col & 15) >> 2), reg = (col & 2) + (row >> 3 & 1);
            uint32_t* to = reinterpret_cast<uint32_t*>(ws.low + (((size_t)i_tile * 4 + row / 16) * (R / 16) + col / 16) * PARTS * 32 + to_lane) + reg;
#pragma unroll
            for (int part = 0; part < PARTS; part++) {
                const uint32_t b = part + 1 < PARTS ? lora_lead(v0) >> 16 | lora_lead(v1) : f8_bf16x2(v0, v1);
                if (fabsf(v0) < INFINITY) v0 -= bf_lo(b);
                if (fabsf(v1) < INFINITY) v1 -= bf_hi(b);
                to[part * 128] = b;
            }
        }
        __syncthreads();  // the sums have been read
    }
}

// A warp's columns: 16 bytes of four lanes' results.  An item is 32 or 64 tokens and some column blocks of a CTA; the next blocks' base and
// B are on their way into shared memory while one is worked on (in registers, a block ahead: 17 us of 30 at 4093 tokens, since
// 16 warps an SM had too little on its way).
template <int R, bool F32>
struct OutSmem {
    // Halves of a tile.  Both with the same stage of B, four warps each, leave twice the warps an SM where B takes most of shared memory:
    // r = 64: 43.6 us / with one, in three stages, 46.3 (4093 tokens, 4096 x 2560), r = 128: 60.6 / 66.4 (2048 tokens, 4096 x 4096); at r = 16 one is enough: 25.9 / 23.2.
    static constexpr int kHalves = R <= 32 ? 1 : 2;
    static constexpr int kRows = 32 * kHalves, kThreads = kOutThreads * kHalves;
    static constexpr int kStages = R <= 16 ? 4 : R <= 32 ? 3 : 2;
    static constexpr int W = F32 ? 4 : 8, kGroup = 4 * W, kCols = kGroup * kOutThreads / 32;
    static constexpr int kBasePitch = 256 + 16;                    // of a token's 256 bytes of a block
    static constexpr int kBPitch = R * 2 + (R > 16 ? 32 : 0);      // of a column's r values: eight bytes of four rows on different banks
    static constexpr int kStageBytes = kRows * kBasePitch + kCols * kBPitch;
    static constexpr bool kHoldLow = R <= 32;                      // low's fragments in registers, else behind the stages
    static constexpr int kLowBytes = kHoldLow ? 0 : kRows / 16 * (R / 16) * (F32 ? 3 : 2) * 512;
    static constexpr int kBytes = kStages * kStageBytes + kLowBytes;
};
template <int R, bool F32>
__global__ void __launch_bounds__((OutSmem<R, F32>::kThreads)) lora_out_kernel(LoraArgs a, LoraWs ws) {
    using S = OutSmem<R, F32>;
    extern __shared__ __align__(128) unsigned char smem[];
    constexpr int W = S::W, kGroup = S::kGroup, kCols = S::kCols, PARTS = F32 ? 3 : 2, NT = W / 2, kSize = F32 ? 4 : 2;
    constexpr int kRows = S::kRows, kThreads = S::kThreads, kPieces = kTile / kRows;
    constexpr bool kHoldLow = S::kHoldLow;
    const int tid = threadIdx.x, warp = tid >> 5 & 3, m0 = tid >> 7 << 1, lane = tid & 31, q = lane & 3, i8 = lane >> 2, r = a.r, N = a.N;
    const bool vec = N % W == 0;
    const int blocks = (N + kCols - 1) / kCols;
    const uint32_t s_base = smem_u32(smem);
    // Written before lora_low_kernel let this one start: the tiles (its own wait was for them), base and B.  Past L1.
    const int pieces = __ldcg(ws.n_tiles) * kPieces;
    // a piece's (a tile's, or half a tile's) blocks in as many chunks as leave no CTA with two
    const int most = max(1, min(blocks, (int)gridDim.x / max(1, pieces))), per = (blocks + most - 1) / most, chunks = (blocks + per - 1) / per;
    bool waited = false;
#pragma unroll 1
    for (int item = blockIdx.x; item < pieces * chunks; item += gridDim.x) {
        const int piece = item / chunks, i_tile = piece / kPieces, row0 = piece % kPieces * kRows;
        const int* order = ws.order + i_tile * kTile + row0;
        const int2 tile = __ldcg(reinterpret_cast<const int2*>(ws.tiles + i_tile));
        // of this thread: the tokens of its results, and of the rows that it copies
        int token[4], copied[4];
#pragma unroll
        for (int i = 0; i < 4; i++) token[i] = __ldcg(order + m0 * 16 + i * 8 + i8), copied[i] = __ldcg(order + i * 8 * S::kHalves + (tid >> 4));
        const int rows = tile.y - row0;
        if (rows <= 0) continue;
        const uint16_t* B = a.b + (size_t)max(tile.x, 0) * N * r;
        const int block0 = (item - piece * chunks) * per, block1 = min(block0 + per, blocks);
        auto ask = [&](int block) {
            if (block < block1) {
                const uint32_t buf = s_base + (block - block0) % S::kStages * S::kStageBytes;
                const int word = tid & 15, col = block * kCols + word * W;
                if (vec)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int row = i * 8 * S::kHalves + (tid >> 4);
                        const bool in = row < rows && col < N;
                        cp_async16_or_zero(buf + row * S::kBasePitch + word * 16,
                                           static_cast<const char*>(a.base) + (in ? ((size_t)copied[i] * N + col) * kSize : 0), in);
                    }
                if (tile.x >= 0)
#pragma unroll
                    for (int i = 0; i < kCols * (R / 8) / kThreads; i++) {
                        const int at = tid + i * kThreads, n = at / (R / 8), w = at % (R / 8);
                        // column n of a group goes where the instruction's rows i8 of product j are neighbours
                        const int in_group = n % kGroup, pos = n - in_group + in_group % W / 2 * 8 + in_group / W * 2 + (in_group & 1);
                        const bool in = block * kCols + n < N && w * 8 < r;
                        cp_async16_or_zero(buf + kRows * S::kBasePitch + pos * S::kBPitch + w * 16, in ? B + (size_t)(block * kCols + n) * r + w * 8 : a.b, in);
                    }
            }
            cp_async_commit();
        };
        __syncthreads();  // the item before has been read
#pragma unroll 1
        for (int s = 0; s < S::kStages - 1; s++) ask(block0 + s);
        if (!waited) {
            griddep_wait();
            waited = true;
        }
        const uint4* low = ws.low + ((size_t)i_tile * 4 + row0 / 16) * (R / 16) * PARTS * 32;
        const uint4* low_s = reinterpret_cast<const uint4*>(smem + S::kStages * S::kStageBytes) + lane;
        if (!kHoldLow && tile.x >= 0) {
#pragma unroll 1
            for (int i = tid; i < S::kLowBytes / 16; i += kThreads) cp_async16(s_base + S::kStages * S::kStageBytes + i * 16, low + i);
            cp_async_wait_all();  // (the loop's first barrier shows it to all)
        }
        uint4 la[kHoldLow ? 2 : 1][kHoldLow ? R / 16 : 1][kHoldLow ? PARTS : 1];
        if (kHoldLow)
#pragma unroll
            for (int m = 0; m < 2; m++)
#pragma unroll
                for (int k = 0; k < R / 16; k++)
#pragma unroll
                    for (int part = 0; part < PARTS; part++)
                        la[m][k][part] = tile.x >= 0 && (m0 + m) * 16 < rows ? low[(((m0 + m) * (R / 16) + k) * PARTS + part) * 32 + lane] : make_uint4(0, 0, 0, 0);
#pragma unroll 1
        for (int block = block0; block < block1; block++) {
            cp_async_wait<S::kStages - 2>();
            __syncthreads();  // this block is there; the one before, whose buffer comes next, has been used
            ask(block + S::kStages - 1);
            const unsigned char* buf = smem + (block - block0) % S::kStages * S::kStageBytes;
            const unsigned char* b_at = buf + kRows * S::kBasePitch + (warp * kGroup + i8) * S::kBPitch + q * 8;
            const int col = block * kCols + warp * kGroup + W * q;
            if (m0 * 16 >= rows) continue;
            float o[2][NT][4];
#pragma unroll
            for (int m = 0; m < 2; m++)
#pragma unroll
                for (int j = 0; j < NT; j++) o[m][j][0] = o[m][j][1] = o[m][j][2] = o[m][j][3] = tile.x < 0 ? -0.f : 0.f;  // (base + -0 is base)
            if (tile.x >= 0)
#pragma unroll
                for (int k = 0; k < R / 16; k++) {
                    uint2 bv[NT];
#pragma unroll
                    for (int j = 0; j < NT; j++) bv[j] = *reinterpret_cast<const uint2*>(b_at + j * 8 * S::kBPitch + k * 32);
#pragma unroll
                    for (int m = 0; m < 2; m++) {
                        if ((m0 + m) * 16 >= rows) break;
#pragma unroll
                        for (int part = 0; part < PARTS; part++) {
                            const uint4 v = kHoldLow ? la[kHoldLow ? m : 0][kHoldLow ? k : 0][kHoldLow ? part : 0] : low_s[(((m0 + m) * (R / 16) + k) * PARTS + part) * 32];
                            const uint32_t f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                            for (int j = 0; j < NT; j++) mma_bf16(o[m][j], f, bv[j].x, bv[j].y);
                        }
                    }
                }
#pragma unroll
            for (int m = 0; m < 2; m++) {
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const int row = (m0 + m) * 16 + h * 8 + i8;
                    if (row >= rows || col >= N) continue;
                    const size_t to = (size_t)token[m * 2 + h] * N + col;
                    float v[W];
#pragma unroll
                    for (int j = 0; j < NT; j++) v[2 * j] = o[m][j][2 * h], v[2 * j + 1] = o[m][j][2 * h + 1];
                    if (vec) {
                        const uint4 was = *reinterpret_cast<const uint4*>(buf + row * S::kBasePitch + (warp * 4 + q) * 16);
                        const uint32_t b[4] = {was.x, was.y, was.z, was.w};
                        if constexpr (F32) {
                            *reinterpret_cast<float4*>(static_cast<float*>(a.out) + to) =
                                make_float4(__uint_as_float(b[0]) + v[0], __uint_as_float(b[1]) + v[1], __uint_as_float(b[2]) + v[2], __uint_as_float(b[3]) + v[3]);
                        } else {
                            uint32_t w[4];
#pragma unroll
                            for (int j = 0; j < 4; j++) w[j] = f8_bf16x2(bf_lo(b[j]) + v[2 * j], bf_hi(b[j]) + v[2 * j + 1]);
                            *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + to) = make_uint4(w[0], w[1], w[2], w[3]);
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < W; j++)
                            if (col + j < N) {
                                if (F32) static_cast<float*>(a.out)[to + j] = static_cast<const float*>(a.base)[to + j] + v[j];
                                else static_cast<uint16_t*>(a.out)[to + j] = f8_bf16(bf2f(static_cast<const uint16_t*>(a.base)[to + j]) + v[j]);
                            }
                    }
                }
            }
        }
    }
    if (!waited) griddep_wait();
}

template <int R, bool F32, int CL>
static cudaError_t low_for(const LoraArgs& a, const LoraWs& ws, int tiles, int sm_count, cudaStream_t st) {
    constexpr auto low = lora_low_kernel<R, F32 ? 3 : 2, CL>;
    const cudaError_t e = allow_smem<low>(LowSmem<R>::kBytes);
    const Launch l{std::min(tiles, sm_count) * CL, kLowThreads, LowSmem<R>::kBytes, 0, st};
    return e != cudaSuccess ? e : l.run(low, a, ws);
}
template <int R, bool F32>
static cudaError_t many_for(const LoraArgs& a, const LoraWs& ws, int sm_count, cudaStream_t st, int* launches) {
    const int tiles = lora_max_tiles(a.T, a.n);
    cudaError_t e;
    // Clusters of four where eights may not all run at once; up to r = 32 fours are not faster.  Four / eight, us, 4096 x 2560: r = 64,
    // 4096 tokens of 32 adapters 41.8 / 46.9, 300 of 4 (2048 x 2560, fp32) 15.9 / 14.5; r = 16, 4096 of 32: 27.8 / 26.9.
    if (R >= 64 && tiles * 8 > 225 * 1024 / (LowSmem<R>::kBytes + 1024) * sm_count) e = low_for<R, F32, R >= 64 ? 4 : 8>(a, ws, tiles, sm_count, st);
    else e = low_for<R, F32, 8>(a, ws, tiles, sm_count, st);
    if (e != cudaSuccess) return e;
    ++*launches;
    constexpr auto out = lora_out_kernel<R, F32>;
    if ((e = allow_smem<out>(OutSmem<R, F32>::kBytes)) != cudaSuccess) return e;
    const int64_t items = (int64_t)(kTile / OutSmem<R, F32>::kRows) * tiles * ((a.N + OutSmem<R, F32>::kCols - 1) / OutSmem<R, F32>::kCols);
    const int fit = std::max(1, std::min(8, 225 * 1024 / (OutSmem<R, F32>::kBytes + 1024)));  // CTAs that an SM has room for
    const Launch o{(int)std::min<int64_t>(items, (int64_t)fit * sm_count), OutSmem<R, F32>::kThreads, OutSmem<R, F32>::kBytes, 0, st};
    if ((e = o.run(out, a, ws)) == cudaSuccess) ++*launches;
    return e;
}

cudaError_t launch_lora_many(const LoraArgs& a, int sm_count, cudaStream_t st, int* launches) {
    const LoraWs ws = lora_layout(a.ws, a.T, a.n, a.r);
    const Launch l{1, kPlanThreads, 0, 0, st};
    cudaError_t e;
    if ((e = l.run(lora_plan_kernel, a, ws)) != cudaSuccess) return e;
    ++*launches;
    switch (lora_padded(a.r)) {
        case 16: return a.out_f32 ? many_for<16, true>(a, ws, sm_count, st, launches) : many_for<16, false>(a, ws, sm_count, st, launches);
        case 32: return a.out_f32 ? many_for<32, true>(a, ws, sm_count, st, launches) : many_for<32, false>(a, ws, sm_count, st, launches);
        case 64: return a.out_f32 ? many_for<64, true>(a, ws, sm_count, st, launches) : many_for<64, false>(a, ws, sm_count, st, launches);
        default: return a.out_f32 ? many_for<128, true>(a, ws, sm_count, st, launches) : many_for<128, false>(a, ws, sm_count, st, launches);
    }
}

}  // namespace moe
