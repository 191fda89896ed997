// Tensor-core (tcgen05, kind::f8f6f4) kernels of the scaled e4m3 products, sm_100a.
//
//   D[i, j] = sum_kb p[i, kb] q[j, kb] sum_{k in block kb} P[i, k] Q[j, k],   blocks of 128 columns
//
// The tensor core multiplies one 128-column block at a time into one of two fp32 accumulators in tensor
// memory; the epilogue warps read each finished accumulator, scale it and add it to the sums they hold
// in registers while the next block is multiplied into the other accumulator.  Arbitrary fp32 scales are
// applied that way in fp32 (the scaled MMA forms take powers of two only).
//
// Two forms, by the number of token rows:
//   few rows   P = 128 weight rows (lanes), Q = 16, 32 or 64 token rows: each weight byte is loaded once for
//              a group of token rows, by TMA straight to the tensor core's shared memory.  A cluster
//              of CTAs splits the inner dimension and adds its partial sums, in order, through distributed
//              shared memory: enough loads are in flight with few tiles, and no sum depends on timing.
//   many rows  P = 128 token rows, Q = 256 (or 128) weight rows, one persistent CTA an SM.  A block of the 128 x
//              256 tile writes 48 KB and reads 48 KB of shared memory, 768 cycles where its MMAs take 512; the
//              hand-overs between MMAs and epilogue (two accumulators fill tensor memory) make it about 1000.
//
// Roles: one warp issues the TMA loads of a ring of stages (a block of both operands each), one thread
// issues the MMAs, the other warps are the epilogue.  All waits are bounded; after one that gave up, the
// warps run their loops to the end without waiting (so that barriers match) and the call reports it.
#pragma once
#include <type_traits>

#include "fp8.h"
#include "fp8.cuh"
#include "tc.cuh"

namespace moe {

enum F8Mode { kF8Dense, kF8GateUp, kF8Down };

struct F8Group {
    int32_t row0, rows, expert, pad;  // slots [row0, row0 + rows) of one expert
};

struct F8Gemm {
    const float* xs;         // token scales [rows, nkb]
    const float* ws;         // weight scales [.., ceil(N / 128), nkb] (gate / up: [E][2][..])
    int nkb, nt, nb;         // inner blocks; weight tiles a group (nt) and 128-row scale blocks a matrix (nb)
    int M, N;                // tokens; weight rows of a matrix (dense N, gate/up F, down H)
    const F8Group* groups;   // experts: token groups
    const int* n_groups;     //   and their number (device); dense: null
    void* out;               // dense: [M, N]; down: y [slots, N] fp32
    int out_f32;
    uint8_t* aq;             // gate/up: quantised activations [slots, N]
    float* as;               //   and their scales [slots, nb]
    uint32_t* err;
    uint64_t timeout_ns;
    int inject;              // test hook: 1 makes the waits for finished accumulators run out
};

// Bounded wait of all lanes (or of one thread).  The limit is counted in SM cycles (reading the global timer
// takes long beside a wait); 2 cycles a ns are at least the limit's time at any clock below 2 GHz.
__device__ __forceinline__ bool f8_wait(uint64_t* bar, uint32_t parity, int* abort, const F8Gemm& a) {
    if (mbar_try_wait(bar, parity) || mbar_try_wait_sleep(bar, parity, 20000u)) return true;
    const long long t0 = clock64();
    while (!mbar_try_wait_sleep(bar, parity, 20000u)) {
        if (*(volatile int*)abort) return false;
        if ((uint64_t)(clock64() - t0) > 2 * a.timeout_ns) {
            *(volatile int*)abort = 1;
            atomicOr(a.err, kErrTimeout);
            return false;
        }
    }
    return true;
}

__device__ __forceinline__ void umma_f8(uint32_t tmem_d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
        "l"(da), "l"(db), "r"(idesc), "r"(acc));
}

// Instruction descriptor: fp32 accumulator, e4m3 operands, both K-major, M = 128.
__host__ __device__ constexpr uint32_t f8_idesc(int n) { return (1u << 4) | ((uint32_t)(n / 8) << 17) | ((128u / 16) << 24); }

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(taddr));
}

__device__ __forceinline__ void tmem_alloc(uint32_t* dst, int cols) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst)), "r"(cols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
}
__device__ __forceinline__ void tmem_dealloc(uint32_t taddr, int cols) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(cols));
}

// True in one lane of a converged warp.  The MMA warp runs its loop as a whole and one lane issues: descriptors
// stay in uniform registers (issued by one diverged thread, the four MMAs of a block took 800 cycles).
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(p));
    return p != 0;
}

__device__ __forceinline__ void prefetch_map(const CUtensorMap* m) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(m) : "memory");
}

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync_all() {
    asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
// The address of this CTA's shared address in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t cluster_map(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void st_cluster_f32(uint32_t addr, float v) {
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t addr) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
// As f8_wait, acquiring what other CTAs of the cluster wrote before they arrived.
__device__ __forceinline__ bool f8_wait_cluster(uint64_t* bar, uint32_t parity, int* abort, const F8Gemm& a) {
    const long long t0 = clock64();
    while (true) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(smem_u32(bar)), "r"(parity), "r"(20000u)
            : "memory");
        if (ok) return true;
        if (*(volatile int*)abort) return false;
        if ((uint64_t)(clock64() - t0) > 2 * a.timeout_ns) {
            *(volatile int*)abort = 1;
            atomicOr(a.err, kErrTimeout);
            return false;
        }
    }
}

// Scales travel ahead of the epilogue in a ring of their own: a slot holds CHUNK blocks' scales of a
// tile's R token rows and of its (two) weight blocks.  One warp copies them asynchronously.
template <int R, int CHUNK, int SLOTS>
struct F8Scales {
    static constexpr int kChunk = CHUNK, kSlots = SLOTS;
    alignas(16) float tok[SLOTS][CHUNK][R];
    float wt[SLOTS][CHUNK][2];
    uint64_t full[SLOTS], empty[SLOTS];
};
__device__ __forceinline__ void cp_async4(float* dst, const float* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
// Arrives on bar once this thread's copies so far have landed.
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
template <int R, int CH, int SL>
__device__ __forceinline__ void scales_init(F8Scales<R, CH, SL>& sc, int readers) {
    for (int i = 0; i < SL; i++) mbar_init(&sc.full[i], 32), mbar_init(&sc.empty[i], readers);
}
// One item's scales of blocks [kb0, kb1); `chunk` counts on over the items.  All lanes of a warp.
template <int WB, int R, int CH, int SL>
__device__ __forceinline__ bool scales_load(F8Scales<R, CH, SL>& sc, const F8Gemm& a, const F8Group& grp, const float* const (&wsp)[WB], int kb0,
                                            int kb1, uint32_t& chunk, int* abort) {
    constexpr int N = (R + 31) / 32;
    const int lane = threadIdx.x & 31;
    const float* xsp[N];
#pragma unroll
    for (int i = 0; i < N; i++) {
        const int r = lane + 32 * i;
        xsp[i] = nullptr;
        if (r < R && r < grp.rows)
            xsp[i] = a.xs + (size_t)(grp.row0 + r) * a.nkb;
    }
    for (int kb = kb0; kb < kb1; kb += CH, chunk++) {
        const int s = chunk % SL;
        bool ok = true;
        if (chunk >= SL) ok = f8_wait(&sc.empty[s], ((chunk / SL) & 1) ^ 1, abort, a);
        if (!__all_sync(0xffffffffu, ok)) return false;
#pragma unroll
        for (int i = 0; i < N; i++)
            if (xsp[i])
#pragma unroll
                for (int k = 0; k < CH; k++)
                    if (kb + k < kb1) cp_async4(&sc.tok[s][k][lane + 32 * i], xsp[i] + kb + k);
        if (lane < WB * CH) {
            const int h = lane / CH, k = lane % CH;
            if (kb + k < kb1) cp_async4(&sc.wt[s][k][h], wsp[h] + kb + k);
        }
        cp_async_arrive(&sc.full[s]);
    }
    return true;
}

// SwiGLU as the other expert paths form it, in fp32.
__device__ __forceinline__ float swiglu_f32(float g, float u) { return g / (1.f + expf(-g)) * u; }

// A group's token count, experts and rows; dense: rows m0 .. of the one matrix.
template <int MODE>
__device__ __forceinline__ F8Group f8_group(const F8Gemm& a, int g, int height) {
    if (MODE == kF8Dense) return F8Group{g * height, min(height, a.M - g * height), 0, 0};
    return a.groups[g];
}
template <int MODE>
__device__ __forceinline__ int f8_groups(const F8Gemm& a, int height) {
    return MODE == kF8Dense ? (a.M + height - 1) / height : __ldcg(a.n_groups);
}
// The same group for the warp that reads it ahead of the wait: past L1 (launch.cuh).
template <int MODE>
__device__ __forceinline__ F8Group f8_group_early(const F8Gemm& a, int g, int height) {
    if (MODE != kF8Down) return f8_group<MODE>(a, g, height);
    const uint4 v = ld_cg_u4(a.groups + g);
    return F8Group{(int32_t)v.x, (int32_t)v.y, (int32_t)v.z, (int32_t)v.w};
}
// Scales of the 128-row weight block `block` of the matrix a group uses (gate/up: g = 0 gate, 1 up).
template <int MODE>
__device__ __forceinline__ const float* f8_wscale(const F8Gemm& a, int expert, int g, int block) {
    const int mat = MODE == kF8GateUp ? expert * 2 + g : expert;
    return a.ws + ((size_t)mat * a.nb + block) * a.nkb;
}

// ---------------------------------------------------------------- few rows

constexpr int kFewScales = 16;  // floats a token column of the scale ring and the maxima

template <int MODE, int NQ>
struct FewCfg {
    static constexpr int WB = MODE == kF8GateUp ? 2 : 1;  // weight tiles a stage: gate and up, or one
    static constexpr int kStage = WB * 16384 + NQ * 128;
    static constexpr int kMinCtas = 2;  // an SM
    static constexpr int kRed = WB * NQ * 128 * 4;  // the sums on their way to the CTA that finishes them
    static constexpr int kBudget = 112 * 1024 - 2048 - kFewScales * NQ * 4;
    static constexpr int kStages = (kBudget - kRed) / kStage > 8 ? 8 : (kBudget - kRed) / kStage;
    static constexpr int kTmemCols = 2 * WB * NQ < 32 ? 32 : 2 * WB * NQ;
    static constexpr int kSmem = kStages * kStage + kRed + 1024;  // 1 KB: alignment of the ring
    static_assert(kStages >= 2 && kSmem + 1024 + kFewScales * NQ * 4 <= 227 * 1024 / kMinCtas, "stages");
};

constexpr int kFewChunk = 4, kFewSlots = 3;
constexpr int kFewThreads = 224;  // 4 epilogue warps, the TMA, the MMA and the scale warp

template <int NQ>
struct FewCtrl {
    uint64_t full[8], empty[8], dfull[2], dempty[2], red_full, red_free, done;
    uint32_t tmem;
    int abort;
    F8Scales<NQ, kFewChunk, kFewSlots> sc;
    uint32_t top[4][NQ];     // per-warp maxima of the activations
};

template <int MODE, int NQ>
__global__ void __launch_bounds__(kFewThreads, FewCfg<MODE, NQ>::kMinCtas)
    f8_few_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const F8Gemm a) {
    using C = FewCfg<MODE, NQ>;
    constexpr int WB = C::WB, S = C::kStages;
    extern __shared__ __align__(1024) unsigned char f8_smem[];
    __shared__ FewCtrl<NQ> c;
    unsigned char* ring = reinterpret_cast<unsigned char*>(((uintptr_t)f8_smem + 1023) & ~(uintptr_t)1023);
    float* red = reinterpret_cast<float*>(ring + (size_t)S * C::kStage);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int CS = (int)cluster_size(), rank = (int)cluster_rank();
    const int n_clusters = gridDim.x / CS, cid = blockIdx.x / CS;
    const int kb0 = a.nkb * rank / CS, kb1 = a.nkb * (rank + 1) / CS;
    if (warp == 4 && lane == 0) prefetch_map(&map_w), prefetch_map(&map_x);
    if (tid == 0) {
        for (int s = 0; s < S; s++) mbar_init(&c.full[s], 1), mbar_init(&c.empty[s], 1);
        for (int b = 0; b < 2; b++) mbar_init(&c.dfull[b], 1 + a.inject), mbar_init(&c.dempty[b], 4);
        mbar_init(&c.red_full, 4 * CS);
        mbar_init(&c.red_free, 4 * CS);
        mbar_init(&c.done, 1);
        scales_init(c.sc, 4);
        c.abort = 0;
        fence_mbar_init();
    }
    if (warp == 5) tmem_alloc(&c.tmem, C::kTmemCols);
    tc_fence_before();
    __syncthreads();
    if (CS > 1) cluster_sync_all();  // every CTA's barriers are initialised before another arrives on them
    tc_fence_after();
    const uint32_t tmem = c.tmem;
    // The down product's kernel starts when every CTA of the gate / up product has let it, which is after the
    // groups are there: it may read them, and the weights, before it waits for the activations.
    if (MODE == kF8Down) griddep_launch_dependents();
    if (MODE != kF8Down || warp != 4) griddep_wait();
    if (MODE == kF8GateUp) griddep_launch_dependents();
    const int items = f8_groups<MODE>(a, NQ) * a.nt;

    if (warp == 4) {
        uint32_t g = 0;
        bool ok = true;
        const uint64_t pol_w = l2_evict_first(), pol_x = l2_evict_last();
        for (int item = cid; ok && item < items; item += n_clusters) {
            const int n = item % a.nt;
            const F8Group grp = f8_group_early<MODE>(a, item / a.nt, NQ);
            auto load_w = [&](int kb, int s) {
                unsigned char* st = ring + (size_t)s * C::kStage;
                mbar_arrive_expect_tx(&c.full[s], C::kStage);
#pragma unroll
                for (int h = 0; h < WB; h++)
                    tma_load_3d(st + h * 16384, &map_w, kb * 128, n * 128, grp.expert * WB + h, &c.full[s], pol_w);
            };
            auto load_x = [&](int kb, int s) {
                tma_load_2d(ring + (size_t)s * C::kStage + WB * 16384, &map_x, kb * 128, grp.row0, &c.full[s], pol_x);
            };
            int kb = kb0;
            if (MODE == kF8Down && g == 0) {  // the first stages' weights ahead of the wait
                const int ahead = min(S, kb1 - kb0);
                if (lane == 0) {
                    fence_proxy_async_global();  // the weights may have been written by a kernel just before the call
                    for (int k = 0; k < ahead; k++) load_w(kb0 + k, k);
                }
                griddep_wait();
                if (lane == 0)
                    for (int k = 0; k < ahead; k++) load_x(kb0 + k, k);
                __syncwarp();
                kb += ahead;
                g += ahead;
            }
            for (; kb < kb1; kb++, g++) {
                const int s = g % S;
                if (g >= (uint32_t)S) ok = f8_wait(&c.empty[s], ((g / S) & 1) ^ 1, &c.abort, a);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                if (lane == 0) {
                    load_w(kb, s);
                    load_x(kb, s);
                }
            }
        }
        // every issued copy lands before the CTA may exit
        if (lane == 0) {
            const uint64_t t0 = globaltimer_ns();
            for (uint32_t q = g > (uint32_t)S ? g - S : 0; q < g; q++)
                while (!mbar_try_wait(&c.full[q % S], (q / S) & 1))
                    if (globaltimer_ns() - t0 > a.timeout_ns) break;
        }
        __syncwarp();
    } else if (warp == 5) {
        constexpr uint32_t idesc = f8_idesc(NQ);
        const bool leader = elect_one();
        const uint64_t desc0 = sw128_desc(smem_u32(ring));
        {
            uint32_t g = 0;
            bool ok = true;
            for (int item = cid; ok && item < items; item += n_clusters) {
                for (int kb = kb0; kb < kb1; kb++, g++) {
                    const int s = g % S, b = g & 1;
                    if (g >= 2) ok = f8_wait(&c.dempty[b], ((g >> 1) & 1) ^ 1, &c.abort, a);
                    ok = ok && f8_wait(&c.full[s], (g / S) & 1, &c.abort, a);
                    ok = __all_sync(0xffffffffu, ok);  // the warp leaves its loop as a whole
                    if (!ok) break;
                    tc_fence_after();
                    const uint64_t dw = desc0 + (uint64_t)(s * (C::kStage >> 4)), dx = dw + WB * 1024;
                    if (leader) {
#pragma unroll
                        for (int kk = 0; kk < 4; kk++)
#pragma unroll
                            for (int h = 0; h < WB; h++)
                                umma_f8(tmem + (b * WB + h) * NQ, dw + h * 1024 + kk * 2, dx + kk * 2, idesc, kk > 0);
                        umma_commit(&c.empty[s]);
                        umma_commit(&c.dfull[b]);
                    }
                    __syncwarp();
                }
            }
            if (leader && *(volatile int*)&c.abort) {  // MMAs that no warp waited for
                umma_commit(&c.done);
                const uint64_t t0 = globaltimer_ns();
                while (!mbar_try_wait(&c.done, 0))
                    if (globaltimer_ns() - t0 > a.timeout_ns) break;
            }
        }
        __syncwarp();
    } else if (warp == 6) {
        uint32_t chunk = 0;
        bool ok = true;
        for (int item = cid; ok && item < items; item += n_clusters) {
            const F8Group grp = f8_group<MODE>(a, item / a.nt, NQ);
            const float* wsp[WB];
#pragma unroll
            for (int h = 0; h < WB; h++) wsp[h] = f8_wscale<MODE>(a, grp.expert, h, item % a.nt);
            ok = scales_load<WB>(c.sc, a, grp, wsp, kb0, kb1, chunk, &c.abort);
        }
        cp_async_wait_all();
    } else {
        // epilogue: warp w holds weight rows [32 w, 32 w + 32) of the tile, one a lane, all token columns
        const uint32_t taddr = tmem + ((uint32_t)(warp * 32) << 16);
        uint32_t g = 0, it = 0, chunk = 0;
        bool ok = true;
        for (int item = cid; item < items; item += n_clusters, it++) {
            const int n = item % a.nt;
            const F8Group grp = f8_group<MODE>(a, item / a.nt, NQ);
            float acc[WB][NQ];
#pragma unroll
            for (int h = 0; h < WB; h++)
#pragma unroll
                for (int j = 0; j < NQ; j++) acc[h][j] = 0.f;
            for (int kb = kb0; kb < kb1; kb++, g++) {
                const int b = g & 1, s = chunk % kFewSlots, k = (kb - kb0) % kFewChunk;
                if (k == 0) ok = ok && f8_wait(&c.sc.full[s], (chunk / kFewSlots) & 1, &c.abort, a);
                ok = ok && f8_wait(&c.dfull[b], (g >> 1) & 1, &c.abort, a);
                __syncwarp();
                tc_fence_after();
                float sw[WB];
#pragma unroll
                for (int h = 0; h < WB; h++) sw[h] = c.sc.wt[s][k][h];
#pragma unroll
                for (int j0 = 0; j0 < NQ; j0 += 16) {
                    uint32_t v[WB][16];
#pragma unroll
                    for (int h = 0; h < WB; h++) tmem_ld16(taddr + (b * WB + h) * NQ + j0, v[h]);
                    tmem_wait_ld();
#pragma unroll
                    for (int j = 0; j < 16; j += 4) {
                        const float4 q = *reinterpret_cast<const float4*>(&c.sc.tok[s][k][j0 + j]);
                        const float qq[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                        for (int i = 0; i < 4; i++)
#pragma unroll
                            for (int h = 0; h < WB; h++)
                                acc[h][j0 + j + i] = fmaf(__uint_as_float(v[h][j + i]), qq[i] * sw[h], acc[h][j0 + j + i]);
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&c.dempty[b]);
                if (k == kFewChunk - 1 || kb + 1 == kb1) {
                    if (lane == 0) mbar_arrive(&c.sc.empty[s]);
                    chunk++;
                }
            }
            // The sums go through shared memory, a cluster's to the CTA that finishes the column: token column j
            // to CTA j % CS.  What follows runs once an item: short loops, since as unrolled code (registers
            // cannot be indexed) it cost 4 us in instruction fetches alone.
            const int per = NQ / CS;
            const int mine = grp.rows > rank ? (grp.rows - rank + CS - 1) / CS : 0;  // columns of this CTA
            if (CS > 1) {
                if (it > 0) ok = ok && f8_wait_cluster(&c.red_free, (it - 1) & 1, &c.abort, a);
                const uint32_t base = smem_u32(red) + (uint32_t)(rank * per * WB * 128 + tid) * 4;
#pragma unroll
                for (int j = 0; j < NQ; j++)
                    if (j < grp.rows) {
                        const uint32_t to = cluster_map(base + (uint32_t)(j / CS) * WB * 512, j % CS);
#pragma unroll
                        for (int h = 0; h < WB; h++) st_cluster_f32(to + h * 512, acc[h][j]);
                    }
                __syncwarp();
                if (lane < CS) mbar_arrive_cluster(cluster_map(smem_u32(&c.red_full), lane));
                ok = ok && f8_wait_cluster(&c.red_full, it & 1, &c.abort, a);
            } else {  // each thread reads its own alone
#pragma unroll
                for (int j = 0; j < NQ; j++)
                    if (j < grp.rows)
#pragma unroll
                        for (int h = 0; h < WB; h++) red[(j * WB + h) * 128 + tid] = acc[h][j];
            }
            const int i = n * 128 + tid;  // weight row
            constexpr int U = 4;          // columns at a time (one behind the other, 64 of them took 7 us)
            if (MODE == kF8Down || (MODE == kF8Dense && i < a.N)) {
                const size_t at = ((size_t)grp.row0 + rank) * a.N + i, step = (size_t)CS * a.N;
#pragma unroll 1
                for (int j = 0; j < mine; j += U) {
                    float v[U];
#pragma unroll
                    for (int u = 0; u < U; u++) v[u] = red[(j + u) * 128 + tid];
#pragma unroll 1
                    for (int r = 1; r < CS; r++)
#pragma unroll
                        for (int u = 0; u < U; u++) v[u] += j + u < mine ? red[(r * per + j + u) * 128 + tid] : 0.f;
#pragma unroll
                    for (int u = 0; u < U; u++)
                        if (j + u < mine && i < a.N) {
                            if (MODE == kF8Down || a.out_f32) static_cast<float*>(a.out)[at + (j + u) * step] = v[u];
                            else static_cast<uint16_t*>(a.out)[at + (j + u) * step] = f8_bf16(v[u]);
                        }
                }
            }
            if (MODE == kF8GateUp) {
#pragma unroll 1
                for (int j = 0; j < mine; j += U) {
                    float v[U][WB];
#pragma unroll
                    for (int u = 0; u < U; u++)
#pragma unroll
                        for (int h = 0; h < WB; h++) v[u][h] = red[((j + u) * WB + h) * 128 + tid];
#pragma unroll 1
                    for (int r = 1; r < CS; r++)
#pragma unroll
                        for (int u = 0; u < U; u++)
#pragma unroll
                            for (int h = 0; h < WB; h++) v[u][h] += j + u < mine ? red[((r * per + j + u) * WB + h) * 128 + tid] : 0.f;
#pragma unroll
                    for (int u = 0; u < U; u++)
                        if (j + u < mine) {
                            const float act = swiglu_f32(v[u][0], v[u][WB - 1]);
                            red[(j + u) * WB * 128 + tid] = act;
                            uint32_t t = __float_as_uint(act) & 0x7fffffffu;
                            t = __reduce_max_sync(0xffffffffu, t < 0x7f800000u ? t : 0u);
                            if (lane == 0) c.top[warp][j + u] = t;
                        }
                }
                named_bar_sync(1, 128);
#pragma unroll 1
                for (int j = 0; j < mine; j += U) {
#pragma unroll
                    for (int u = 0; u < U; u++)
                        if (j + u < mine) {
                            const int k = j + u;
                            const uint32_t se = f8_scale_exp(max(max(c.top[0][k], c.top[1][k]), max(c.top[2][k], c.top[3][k])));
                            const size_t slot = (size_t)grp.row0 + rank + CS * k;
                            if (i < a.N) a.aq[slot * a.N + i] = (uint8_t)f8_pack1(red[k * WB * 128 + tid], f8_inverse(se));
                            if (tid == 0) a.as[slot * a.nb + n] = __uint_as_float(se << 23);
                        }
                }
                named_bar_sync(1, 128);  // c.top is read before the next item's is written
            }
            if (CS > 1) {
                __syncwarp();
                if (lane < CS) mbar_arrive_cluster(cluster_map(smem_u32(&c.red_free), lane));
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 5) {
        tc_fence_after();
        tmem_dealloc(tmem, C::kTmemCols);
    }
    if (CS > 1) cluster_sync_all();  // no CTA leaves while another may still write to its shared memory
}

// ---------------------------------------------------------------- many rows

constexpr int kManyEpi = 16;                         // epilogue warps: 128 rows x four column quarters
constexpr int kManyThreads = (kManyEpi + 3) * 32;    // and the TMA, the MMA and the scale warp

template <int MODE>
struct ManyCtrl {
    uint64_t full[5], empty[5], dfull[2], dempty[2], done;
    uint32_t tmem;
    int abort;
    F8Scales<128, 2, 2> sc;
    uint32_t top[MODE == kF8GateUp ? 4 : 1][MODE == kF8GateUp ? 128 : 1];  // row maxima of the column quarters
};

template <int MODE, int NB>
struct ManyCfg {
    static constexpr int kStage = 16384 + NB * 128;
    static constexpr int kStages = NB == 256 ? 4 : 5;
    // Blocks the two roles hand over at a time, each with an accumulator of its own: a hand-over costs the epilogue
    // some 400 cycles, as much as adding up a block of 128 columns.
    static constexpr int kPhase = 256 / NB;
    static constexpr int kTurn = MODE == kF8GateUp ? 0 : 2048;  // a warp's 32 rows x 64 bytes on their way to memory
    static constexpr int kSmem = kStages * kStage + kManyEpi * kTurn + (int)sizeof(ManyCtrl<MODE>);
    static_assert(MODE == kF8Dense || NB == 256, "the expert products use 256-row tiles");
    static_assert(kSmem <= 227 * 1024, "shared memory");
};

// Dense tiles in bands of 16 token tiles, weight tiles along the band: the tiles that run at a time share
// both operands in L2.  Experts: a group's weight tiles one after the other.
template <int MODE>
__device__ __forceinline__ void many_tile(const F8Gemm& a, int item, int groups, int& g, int& n) {
    if (MODE == kF8Dense) {
        const int band = item / (16 * a.nt), first = band * 16, in = item - band * 16 * a.nt, h = min(16, groups - first);
        g = first + in % h;
        n = in / h;
    } else {
        g = item / a.nt;
        n = item - g * a.nt;
    }
}

// Stores a warp's 32 rows x 64 bytes (lane l holds row l as four 16-byte words) so that four lanes write a
// row's 64 bytes: through shared memory, word w of row r at place w ^ (r / 2 & 3), conflict-free both ways.
// Rows from `rows` and words from `words` on are left out.  (Each lane writing its own row, a store
// instruction touched 32 rows: the last product of 2048 tokens took 259 us, 209 so.)
__device__ __forceinline__ void turn_rows(unsigned char* turn, const uint4 (&w)[4], char* dst, size_t pitch, int rows, int words) {
    const int lane = threadIdx.x & 31;
    __syncwarp();
#pragma unroll
    for (int k = 0; k < 4; k++) *reinterpret_cast<uint4*>(turn + lane * 64 + ((k ^ (lane >> 1 & 3)) << 4)) = w[k];
    __syncwarp();
    const int k = lane & 3;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int r = i * 8 + (lane >> 2);
        const uint4 v = *reinterpret_cast<const uint4*>(turn + r * 64 + ((k ^ (r >> 1 & 3)) << 4));
        if (r < rows && k < words) *reinterpret_cast<uint4*>(dst + r * pitch + k * 16) = v;
    }
}
// The same where rows are not 16-byte aligned: the values of a row (B bytes each, `left` of them) by as many
// neighbouring lanes.
template <int B>
__device__ __forceinline__ void turn_values(unsigned char* turn, const uint4 (&w)[4], char* dst, size_t pitch, int rows, int left) {
    constexpr int L = 64 / B;  // lanes a row
    const int lane = threadIdx.x & 31, e = lane % L;
    __syncwarp();
#pragma unroll
    for (int k = 0; k < 4; k++) *reinterpret_cast<uint4*>(turn + lane * 64 + ((k ^ (lane >> 1 & 3)) << 4)) = w[k];
    __syncwarp();
#pragma unroll 4
    for (int r = lane / L; r < 32; r += 32 / L) {
        const unsigned char* v = turn + r * 64 + (((e * B >> 4) ^ (r >> 1 & 3)) << 4) + (e * B & 15);
        if (r >= rows || e >= left) continue;
        if (B == 4) *reinterpret_cast<uint32_t*>(dst + r * pitch + e * 4) = *reinterpret_cast<const uint32_t*>(v);
        else *reinterpret_cast<uint16_t*>(dst + r * pitch + e * 2) = *reinterpret_cast<const uint16_t*>(v);
    }
}
// A segment's 32 columns from column n0 on as fp32 or bf16, row0 = the warp's first row.
template <bool F32>
__device__ __forceinline__ void turn_store(unsigned char* turn, const float (&v)[32], void* out, size_t row0, int n0, int N, int rows) {
    constexpr int B = F32 ? 4 : 2, W = 16 / B;  // bytes a value, values a word
    char* dst = static_cast<char*>(out) + (row0 * N + n0) * B;
#pragma unroll
    for (int c = 0; c < 32; c += 4 * W) {
        uint4 w[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const float* q = v + c + k * W;
            if (F32) w[k] = make_uint4(__float_as_uint(q[0]), __float_as_uint(q[1]), __float_as_uint(q[2]), __float_as_uint(q[3]));
            else w[k] = make_uint4(f8_bf16x2(q[0], q[1]), f8_bf16x2(q[2], q[3]), f8_bf16x2(q[W - 4], q[W - 3]), f8_bf16x2(q[W - 2], q[W - 1]));
        }
        if (N % W == 0) turn_rows(turn, w, dst + c * B, (size_t)N * B, rows, (N - n0 - c) / W);
        else turn_values<B>(turn, w, dst + c * B, (size_t)N * B, rows, N - n0 - c);
    }
}

template <int MODE, int NB>
__global__ void __launch_bounds__(kManyThreads, 1)
    f8_many_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const F8Gemm a) {
    using C = ManyCfg<MODE, NB>;
    constexpr int S = C::kStages, SEG = NB / 128, KP = C::kPhase;
    extern __shared__ __align__(1024) unsigned char f8_smem[];
    unsigned char* ring = f8_smem;
    ManyCtrl<MODE>& c = *reinterpret_cast<ManyCtrl<MODE>*>(ring + S * C::kStage + kManyEpi * C::kTurn);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (smem_u32(ring) & 1023) {  // the swizzled operands need it; the array is declared so
        if (tid == 0) atomicOr(a.err, kErrTimeout);
        return;
    }
    if (warp == kManyEpi && lane == 0) prefetch_map(&map_w), prefetch_map(&map_x);
    if (tid == 0) {
        for (int s = 0; s < S; s++) mbar_init(&c.full[s], 1), mbar_init(&c.empty[s], 1);
        for (int b = 0; b < 2; b++) mbar_init(&c.dfull[b], 1 + a.inject), mbar_init(&c.dempty[b], kManyEpi);
        mbar_init(&c.done, 1);
        scales_init(c.sc, kManyEpi);
        c.abort = 0;
        fence_mbar_init();
    }
    if (warp == kManyEpi + 1) tmem_alloc(&c.tmem, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = c.tmem;
    griddep_wait();
    if (MODE != kF8Dense) griddep_launch_dependents();
    const int groups = f8_groups<MODE>(a, 128), items = groups * a.nt, nkb = a.nkb;

    if (warp == kManyEpi) {
        uint32_t g = 0;
        bool ok = true;
        const uint64_t pol_w = MODE == kF8Dense ? l2_evict_last() : l2_evict_first(), pol_x = l2_evict_last();
        for (int item = blockIdx.x; ok && item < items; item += gridDim.x) {
            int gi, n;
            many_tile<MODE>(a, item, groups, gi, n);
            const F8Group grp = f8_group<MODE>(a, gi, 128);
            for (int kb = 0; kb < nkb; kb++, g++) {
                const int s = g % S;
                if (g >= (uint32_t)S) ok = f8_wait(&c.empty[s], ((g / S) & 1) ^ 1, &c.abort, a);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                unsigned char* st = ring + (size_t)s * C::kStage;
                unsigned char* sw = st + 16384;
                if (lane == 0) {
                    mbar_arrive_expect_tx(&c.full[s], C::kStage);
                    tma_load_2d(st, &map_x, kb * 128, grp.row0, &c.full[s], pol_x);
#pragma unroll
                    for (int h = 0; h < SEG; h++) {
                        if (MODE == kF8GateUp) tma_load_3d(sw + h * 16384, &map_w, kb * 128, n * 128, grp.expert * 2 + h, &c.full[s], pol_w);
                        else tma_load_3d(sw + h * 16384, &map_w, kb * 128, n * NB + h * 128, grp.expert, &c.full[s], pol_w);
                    }
                }
            }
        }
        if (lane == 0) {  // every issued copy lands before the CTA may exit
            const uint64_t t0 = globaltimer_ns();
            for (uint32_t q = g > (uint32_t)S ? g - S : 0; q < g; q++)
                while (!mbar_try_wait(&c.full[q % S], (q / S) & 1))
                    if (globaltimer_ns() - t0 > a.timeout_ns) break;
        }
        __syncwarp();
    } else if (warp == kManyEpi + 1) {
        constexpr uint32_t idesc = f8_idesc(NB);
        const bool leader = elect_one();
        const uint64_t desc0 = sw128_desc(smem_u32(ring));
        {
            uint32_t g = 0, ph = 0;  // blocks, phases
            bool ok = true;
            for (int item = blockIdx.x; ok && item < items; item += gridDim.x) {
                for (int kb = 0; kb < nkb; kb++, g++) {
                    const int s = g % S, b = ph & 1, p = kb % KP;
                    ok = f8_wait(&c.full[s], (g / S) & 1, &c.abort, a);
                    if (p == 0 && ph >= 2) ok = ok && f8_wait(&c.dempty[b], ((ph >> 1) & 1) ^ 1, &c.abort, a);
                    ok = __all_sync(0xffffffffu, ok);  // the warp leaves its loop as a whole
                    if (!ok) break;
                    tc_fence_after();
                    const uint64_t dx = desc0 + (uint64_t)(s * (C::kStage >> 4)), dw = dx + 1024;
                    if (leader) {
#pragma unroll
                        for (int kk = 0; kk < 4; kk++) umma_f8(tmem + (b * KP + p) * NB, dx + kk * 2, dw + kk * 2, idesc, kk > 0);
                        umma_commit(&c.empty[s]);
                        if (p == KP - 1 || kb + 1 == nkb) umma_commit(&c.dfull[b]);
                    }
                    if (p == KP - 1 || kb + 1 == nkb) ph++;
                    __syncwarp();
                }
            }
            if (leader && *(volatile int*)&c.abort) {
                umma_commit(&c.done);
                const uint64_t t0 = globaltimer_ns();
                while (!mbar_try_wait(&c.done, 0))
                    if (globaltimer_ns() - t0 > a.timeout_ns) break;
            }
        }
        __syncwarp();
    } else if (warp == kManyEpi + 2) {
        uint32_t chunk = 0;
        bool ok = true;
        for (int item = blockIdx.x; ok && item < items; item += gridDim.x) {
            int gi, n;
            many_tile<MODE>(a, item, groups, gi, n);
            const F8Group grp = f8_group<MODE>(a, gi, 128);
            const float* wsp[SEG];
#pragma unroll
            for (int h = 0; h < SEG; h++)
                wsp[h] = f8_wscale<MODE>(a, grp.expert, h, MODE == kF8GateUp ? n : min(n * SEG + h, a.nb - 1));
            ok = scales_load<SEG>(c.sc, a, grp, wsp, 0, nkb, chunk, &c.abort);
        }
        cp_async_wait_all();
    } else {
        // epilogue: warp w holds token rows [32 (w % 4), ..), one a lane, and a quarter of the columns in segments
        // of 32 (gate/up: one of gate and the same of up).  Sixteen warps, since the scaled sums are bound by
        // latency: eight, with 128 columns each, took 507 cycles a block where these take 320 (the MMAs: 512).
        const int q = warp & 3, quarter = warp >> 2, r = q * 32 + lane;
        unsigned char* turn = ring + S * C::kStage + warp * C::kTurn;
        const uint32_t taddr = tmem + ((uint32_t)(q * 32) << 16) + (MODE == kF8GateUp ? 32 : NB / 4) * quarter;
        constexpr int SEGSTEP = MODE == kF8GateUp ? 128 : 32;  // accumulator columns between a warp's segments
        const int wsel = MODE != kF8GateUp && NB == 256 ? quarter >> 1 : 0;
        uint32_t ph = 0, chunk = 0;
        bool ok = true;
        for (int item = blockIdx.x; item < items; item += gridDim.x) {
            int gi, n;
            many_tile<MODE>(a, item, groups, gi, n);
            const F8Group grp = f8_group<MODE>(a, gi, 128);
            float acc[SEG][32];
#pragma unroll
            for (int i = 0; i < SEG; i++)
#pragma unroll
                for (int j = 0; j < 32; j++) acc[i][j] = 0.f;
            for (int kb = 0; kb < nkb; kb += KP, ph++) {
                const int b = ph & 1, sl = chunk & 1, k = kb & 1;
                if (k == 0) ok = ok && f8_wait(&c.sc.full[sl], (chunk >> 1) & 1, &c.abort, a);
                float sw[KP][SEG];
#pragma unroll
                for (int p = 0; p < KP; p++) {  // (a block behind the last: what is there is not used)
                    const float sx = c.sc.tok[sl][k + p][r];
#pragma unroll
                    for (int i = 0; i < SEG; i++) sw[p][i] = sx * c.sc.wt[sl][k + p][MODE == kF8GateUp ? i : wsel];
                }
                ok = ok && f8_wait(&c.dfull[b], (ph >> 1) & 1, &c.abort, a);
                __syncwarp();
                tc_fence_after();
#pragma unroll
                for (int p = 0; p < KP; p++) {
                    if (p > 0 && kb + p >= nkb) break;
                    const uint32_t t0 = taddr + (b * KP + p) * NB;
                    uint32_t v[2][16];
                    tmem_ld16(t0, v[0]);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 2 * SEG; i++) {  // the next sixteen columns are read while these are added
                        if (i + 1 < 2 * SEG) tmem_ld16(t0 + (i + 1) / 2 * SEGSTEP + ((i + 1) & 1) * 16, v[(i + 1) & 1]);
#pragma unroll
                        for (int j = 0; j < 16; j++) {
                            float& d = acc[i / 2][(i & 1) * 16 + j];
                            d = fmaf(__uint_as_float(v[i & 1][j]), sw[p][i / 2], d);
                        }
                        if (i + 1 < 2 * SEG) tmem_wait_ld();
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&c.dempty[b]);
                if (KP == 2 || k == 1 || kb + 1 == nkb) {
                    if (lane == 0) mbar_arrive(&c.sc.empty[sl]);
                    chunk++;
                }
            }
            const bool live = r < grp.rows;
            const size_t slot = (size_t)grp.row0 + r;
            if (MODE == kF8GateUp) {
                uint32_t top = 0;
#pragma unroll
                for (int j = 0; j < 32; j++) {
                    acc[0][j] = swiglu_f32(acc[0][j], acc[SEG - 1][j]);
                    const uint32_t t = __float_as_uint(acc[0][j]) & 0x7fffffffu;
                    top = max(top, t < 0x7f800000u ? t : 0u);
                }
                c.top[quarter][r] = top;
                named_bar_sync(1, kManyEpi * 32);
                top = max(max(c.top[0][r], c.top[1 % (sizeof(c.top) / sizeof(c.top[0]))][r]),
                          max(c.top[2 % (sizeof(c.top) / sizeof(c.top[0]))][r], c.top[3 % (sizeof(c.top) / sizeof(c.top[0]))][r]));
                named_bar_sync(1, kManyEpi * 32);  // read before the next item writes
                const uint32_t se = f8_scale_exp(top);
                const float inv = f8_inverse(se);
                const int f0 = n * 128 + quarter * 32;
                if (live && f0 < a.N) {  // F is a multiple of 64
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        const uint2 lo = f8_pack8(reinterpret_cast<const float(&)[8]>(acc[0][16 * j]), inv, true);
                        const uint2 hi = f8_pack8(reinterpret_cast<const float(&)[8]>(acc[0][16 * j + 8]), inv, true);
                        reinterpret_cast<uint4*>(a.aq + slot * a.N + f0)[j] = make_uint4(lo.x, lo.y, hi.x, hi.y);
                    }
                }
                if (live && quarter == 0) a.as[slot * a.nb + n] = __uint_as_float(se << 23);
            } else {
                const int rows = min(32, grp.rows - q * 32);  // of this warp
                const bool f32 = MODE == kF8Down || a.out_f32;
                const size_t row0 = (size_t)grp.row0 + q * 32;
#pragma unroll
                for (int i = 0; i < SEG; i++) {
                    const int n0 = n * NB + quarter * (NB / 4) + i * 32;
                    if (rows <= 0) break;
                    if (f32) turn_store<true>(turn, acc[i], a.out, row0, n0, a.N, rows);
                    else turn_store<false>(turn, acc[i], a.out, row0, n0, a.N, rows);
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kManyEpi + 1) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

}  // namespace moe
