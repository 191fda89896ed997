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
//   few rows   P = 128 weight rows (lanes), Q = 16..64 token rows: each weight byte is loaded once, by
//              TMA straight to the tensor core's shared memory, whatever the number of tokens.  A cluster
//              of CTAs splits the inner dimension and adds its partial sums, in order, through distributed
//              shared memory: enough loads are in flight with few tiles, and no sum depends on timing.
//   many rows  P = 128 token rows, Q = 256 (or 128) weight rows, one persistent CTA an SM.
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
    int M, N;                // dense: tokens; weight rows of a matrix (dense N, gate/up F, down H)
    const F8Group* groups;   // experts: token groups
    const int* n_groups;     //   and their number (device); dense: null
    const int32_t* perm;     // gate/up: token of each slot
    void* out;               // dense: [M, N]; down: y [slots, N] fp32
    int out_f32;
    uint8_t* aq;             // gate/up: quantised activations [slots, N]
    float* as;               //   and their scales [slots, nb]
    uint32_t* err;
    uint64_t timeout_ns;
};

// Bounded wait of all lanes (or of one thread): the clock is read only where the first try fails.
__device__ __forceinline__ bool f8_wait(uint64_t* bar, uint32_t parity, int* abort, const F8Gemm& a) {
    if (mbar_try_wait(bar, parity)) return true;
    const uint64_t t0 = globaltimer_ns();
    while (!mbar_try_wait_sleep(bar, parity, 20000u)) {
        if (*(volatile int*)abort) return false;
        if (globaltimer_ns() - t0 > a.timeout_ns) {
            *(volatile int*)abort = 1;
            atomicOr(a.err, kErrTimeout);
            return false;
        }
    }
    return true;
}

// Four 128-byte rows r0..r3 at byte column x of a [rows, cols] byte matrix (boxes one row high).
__device__ __forceinline__ void tma_gather4(void* dst, const CUtensorMap* map, int x, int4 r, uint64_t* bar, uint64_t policy) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes.L2::cache_hint [%0], "
        "[%1, {%3, %4, %5, %6, %7}], [%2], %8;" ::"r"(smem_u32(dst)),
        "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(r.x), "r"(r.y), "r"(r.z), "r"(r.w), "l"(policy)
        : "memory");
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
    const uint64_t t0 = globaltimer_ns();
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
        if (globaltimer_ns() - t0 > a.timeout_ns) {
            *(volatile int*)abort = 1;
            atomicOr(a.err, kErrTimeout);
            return false;
        }
    }
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
    return MODE == kF8Dense ? (a.M + height - 1) / height : __ldg(a.n_groups);
}
// Scales of the 128-row weight block `block` of the matrix a group uses (gate/up: g = 0 gate, 1 up).
template <int MODE>
__device__ __forceinline__ const float* f8_wscale(const F8Gemm& a, int expert, int g, int block) {
    const int mat = MODE == kF8GateUp ? expert * 2 + g : expert;
    return a.ws + ((size_t)mat * a.nb + block) * a.nkb;
}

// ---------------------------------------------------------------- few rows

template <int MODE, int NQ>
struct FewCfg {
    static constexpr int WB = MODE == kF8GateUp ? 2 : 1;  // weight tiles a stage: gate and up, or one
    static constexpr int kStage = WB * 16384 + NQ * 128;
    // two CTAs an SM; one where 64 rows of gate and up sums fill the registers
    static constexpr int kMinCtas = NQ == 64 && WB == 2 ? 1 : 2;
    static constexpr int kRed = NQ == 64 && WB == 2 ? 0 : WB * NQ * 128 * 4;  // partial sums of a cluster (none: no split)
    static constexpr int kBudget = (kMinCtas == 2 ? 112 : 224) * 1024 - 2048;
    static constexpr int kStages = (kBudget - kRed) / kStage > 8 ? 8 : (kBudget - kRed) / kStage;
    static constexpr int kTmemCols = 2 * WB * NQ < 32 ? 32 : 2 * WB * NQ;
    static constexpr int kSmem = kStages * kStage + kRed + 1024;  // 1 KB: alignment of the ring
    static_assert(kStages >= 2 && kSmem + 1024 <= 227 * 1024 / kMinCtas, "stages");
};

constexpr int kFewThreads = 192;  // 4 epilogue warps, the TMA warp, the MMA warp

template <int NQ>
struct FewCtrl {
    uint64_t full[8], empty[8], dfull[2], dempty[2], red_full, red_free, done;
    uint32_t tmem;
    int abort;
    float sq[2][NQ];         // token scales of a block
    float top[4][NQ];        // per-warp maxima of the activations
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
    if (tid == 0) {
        for (int s = 0; s < S; s++) mbar_init(&c.full[s], 1), mbar_init(&c.empty[s], 1);
        for (int b = 0; b < 2; b++) mbar_init(&c.dfull[b], 1), mbar_init(&c.dempty[b], 4);
        mbar_init(&c.red_full, 4 * CS);
        mbar_init(&c.red_free, 4 * CS);
        mbar_init(&c.done, 1);
        c.abort = 0;
        fence_mbar_init();
    }
    if (warp == 5) tmem_alloc(&c.tmem, C::kTmemCols);
    tc_fence_before();
    __syncthreads();
    if (CS > 1) cluster_sync_all();  // every CTA's barriers are initialised before another arrives on them
    tc_fence_after();
    const uint32_t tmem = c.tmem;
    griddep_launch_dependents();
    if (MODE != kF8Dense) griddep_wait();
    const int items = f8_groups<MODE>(a, NQ) * a.nt;

    if (warp == 4) {
        uint32_t g = 0;
        bool ok = true;
        const uint64_t pol_w = l2_evict_first(), pol_x = l2_evict_last();
        if (MODE == kF8Dense) griddep_wait();
        for (int item = cid; ok && item < items; item += n_clusters) {
            const int n = item % a.nt;
            const F8Group grp = f8_group<MODE>(a, item / a.nt, NQ);
            int4 rows = make_int4(0, 0, 0, 0);
            if (MODE == kF8GateUp && lane < NQ / 4) {  // the tokens of four slots; the first slot's again behind the last
                const int c0 = 4 * lane;
                const int32_t* p = a.perm + grp.row0;
                rows = make_int4(__ldg(p + (c0 < grp.rows ? c0 : 0)), __ldg(p + (c0 + 1 < grp.rows ? c0 + 1 : 0)),
                                 __ldg(p + (c0 + 2 < grp.rows ? c0 + 2 : 0)), __ldg(p + (c0 + 3 < grp.rows ? c0 + 3 : 0)));
            }
            for (int kb = kb0; kb < kb1; kb++, g++) {
                const int s = g % S;
                if (g >= (uint32_t)S) ok = f8_wait(&c.empty[s], ((g / S) & 1) ^ 1, &c.abort, a);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                unsigned char* st = ring + (size_t)s * C::kStage;
                if (lane == 0) {
                    mbar_arrive_expect_tx(&c.full[s], C::kStage);
                    if (MODE == kF8GateUp) {
                        tma_load_3d(st, &map_w, kb * 128, n * 128, grp.expert * 2, &c.full[s], pol_w);
                        tma_load_3d(st + 16384, &map_w, kb * 128, n * 128, grp.expert * 2 + 1, &c.full[s], pol_w);
                    } else {
                        tma_load_3d(st, &map_w, kb * 128, n * 128, grp.expert, &c.full[s], pol_w);
                        tma_load_2d(st + 16384, &map_x, kb * 128, grp.row0, &c.full[s], pol_x);
                    }
                }
                if (MODE == kF8GateUp) {
                    __syncwarp();
                    if (lane < NQ / 4) tma_gather4(st + 32768 + lane * 512, &map_x, kb * 128, rows, &c.full[s], pol_x);
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
        if (lane == 0) {
            constexpr uint32_t idesc = f8_idesc(NQ);
            uint32_t g = 0;
            bool ok = true;
            for (int item = cid; ok && item < items; item += n_clusters) {
                for (int kb = kb0; kb < kb1; kb++, g++) {
                    const int s = g % S, b = g & 1;
                    if (g >= 2) ok = f8_wait(&c.dempty[b], ((g >> 1) & 1) ^ 1, &c.abort, a);
                    ok = ok && f8_wait(&c.full[s], (g / S) & 1, &c.abort, a);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t sw = smem_u32(ring + (size_t)s * C::kStage), sx = sw + WB * 16384;
#pragma unroll
                    for (int kk = 0; kk < 4; kk++)
#pragma unroll
                        for (int h = 0; h < WB; h++)
                            umma_f8(tmem + (b * WB + h) * NQ, sw128_desc(sw + h * 16384 + kk * 32), sw128_desc(sx + kk * 32),
                                    idesc, kk > 0);
                    umma_commit(&c.empty[s]);
                    umma_commit(&c.dfull[b]);
                }
            }
            if (*(volatile int*)&c.abort) {  // MMAs that no warp waited for
                umma_commit(&c.done);
                const uint64_t t0 = globaltimer_ns();
                while (!mbar_try_wait(&c.done, 0))
                    if (globaltimer_ns() - t0 > a.timeout_ns) break;
            }
        }
        __syncwarp();
    } else {
        // epilogue: warp w holds weight rows [32 w, 32 w + 32) of the tile, one a lane, all token columns
        const uint32_t taddr = tmem + ((uint32_t)(warp * 32) << 16);
        uint32_t g = 0, it = 0;
        bool ok = true;
        if (MODE == kF8Dense) griddep_wait();
        for (int item = cid; item < items; item += n_clusters, it++) {
            const int n = item % a.nt;
            const F8Group grp = f8_group<MODE>(a, item / a.nt, NQ);
            const float* wsp[WB];
#pragma unroll
            for (int h = 0; h < WB; h++) wsp[h] = f8_wscale<MODE>(a, grp.expert, h, n);
            const float* xsp = nullptr;  // scales of token column tid
            if (tid < NQ && tid < grp.rows)
                xsp = a.xs + (size_t)(MODE == kF8GateUp ? __ldg(a.perm + grp.row0 + tid) : grp.row0 + tid) * a.nkb;
            float acc[WB][NQ];
#pragma unroll
            for (int h = 0; h < WB; h++)
#pragma unroll
                for (int j = 0; j < NQ; j++) acc[h][j] = 0.f;
            if (tid < NQ) c.sq[g & 1][tid] = xsp && kb0 < kb1 ? __ldg(xsp + kb0) : 0.f;
            float sw[WB];
#pragma unroll
            for (int h = 0; h < WB; h++) sw[h] = kb0 < kb1 ? __ldg(wsp[h] + kb0) : 0.f;
            for (int kb = kb0; kb < kb1; kb++, g++) {
                const int b = g & 1;
                const float next = xsp && kb + 1 < kb1 ? __ldg(xsp + kb + 1) : 0.f;
                float sw_next[WB];
#pragma unroll
                for (int h = 0; h < WB; h++) sw_next[h] = kb + 1 < kb1 ? __ldg(wsp[h] + kb + 1) : 0.f;
                ok = ok && f8_wait(&c.dfull[b], (g >> 1) & 1, &c.abort, a);
                named_bar_sync(1, 128);  // the block's token scales are in c.sq[b]; its last readers are past it
                tc_fence_after();
#pragma unroll
                for (int j0 = 0; j0 < NQ; j0 += 16) {
                    uint32_t v[WB][16];
                    __syncwarp();
#pragma unroll
                    for (int h = 0; h < WB; h++) tmem_ld16(taddr + (b * WB + h) * NQ + j0, v[h]);
                    tmem_wait_ld();
#pragma unroll
                    for (int j = 0; j < 16; j += 4) {
                        const float4 q = *reinterpret_cast<const float4*>(&c.sq[b][j0 + j]);
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
                if (tid < NQ) c.sq[b ^ 1][tid] = next;
#pragma unroll
                for (int h = 0; h < WB; h++) sw[h] = sw_next[h];
            }
            // columns this CTA finishes: j -> token rank + CS j
            int mine = grp.rows;
            if (C::kRed && CS > 1) {
                const int per = NQ / CS;
                mine = grp.rows > rank ? (grp.rows - rank + CS - 1) / CS : 0;
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
#pragma unroll
                for (int j = 0; j < NQ / 2; j++)  // CS >= 2
                    if (j < mine)
#pragma unroll
                        for (int h = 0; h < WB; h++) {
                            float v = 0.f;
                            for (int r = 0; r < CS; r++) v += red[((r * per + j) * WB + h) * 128 + tid];
                            acc[h][j] = v;
                        }
                __syncwarp();
                if (lane < CS) mbar_arrive_cluster(cluster_map(smem_u32(&c.red_free), lane));
            }
            const int step = C::kRed && CS > 1 ? CS : 1, first = C::kRed && CS > 1 ? rank : 0;
            const int i = n * 128 + tid;  // weight row
            if (MODE == kF8GateUp) {
#pragma unroll
                for (int j = 0; j < NQ; j++)
                    if (j < mine) {
                        const float v = swiglu_f32(acc[0][j], acc[WB - 1][j]);
                        acc[0][j] = v;
                        uint32_t t = __float_as_uint(v) & 0x7fffffffu;
                        t = __reduce_max_sync(0xffffffffu, t < 0x7f800000u ? t : 0u);
                        if (lane == 0) c.top[warp][j] = __uint_as_float(t);
                    }
                named_bar_sync(1, 128);
#pragma unroll
                for (int j = 0; j < NQ; j++)
                    if (j < mine) {
                        const float t = fmaxf(fmaxf(c.top[0][j], c.top[1][j]), fmaxf(c.top[2][j], c.top[3][j]));
                        const uint32_t se = f8_scale_exp(__float_as_uint(t));
                        const size_t slot = (size_t)grp.row0 + first + step * j;
                        if (i < a.N) a.aq[slot * a.N + i] = (uint8_t)f8_pack1(acc[0][j], f8_inverse(se));
                        if (tid == 0) a.as[slot * a.nb + n] = __uint_as_float(se << 23);
                    }
                // the next item's first barrier comes before c.top is written again
            } else if (i < a.N) {
#pragma unroll
                for (int j = 0; j < NQ; j++)
                    if (j < mine) {
                        const size_t at = ((size_t)grp.row0 + first + step * j) * a.N + i;
                        if (MODE == kF8Down || a.out_f32) static_cast<float*>(a.out)[at] = acc[0][j];
                        else static_cast<uint16_t*>(a.out)[at] = f8_bf16(acc[0][j]);
                    }
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

template <int MODE, int NB>
struct ManyCfg {
    static constexpr int kStage = 16384 + NB * 128;
    static constexpr int kStages = NB == 256 ? 4 : 6;
    static constexpr int kSmem = kStages * kStage + 1024;
    static_assert(MODE == kF8Dense || NB == 256, "the expert products use 256-row tiles");
};

constexpr int kManyThreads = 384;  // 8 epilogue warps, the TMA warp, the MMA warp, two idle ones

struct ManyCtrl {
    uint64_t full[6], empty[6], dfull[2], dempty[2], done;
    uint32_t tmem;
    int abort;
    uint32_t top[2][128];  // gate/up: row maxima of the two column halves
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

template <int MODE, int NB>
__global__ void __launch_bounds__(kManyThreads, 1)
    f8_many_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const F8Gemm a) {
    using C = ManyCfg<MODE, NB>;
    constexpr int S = C::kStages;
    extern __shared__ __align__(1024) unsigned char f8_smem[];
    __shared__ ManyCtrl c;
    unsigned char* ring = reinterpret_cast<unsigned char*>(((uintptr_t)f8_smem + 1023) & ~(uintptr_t)1023);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int s = 0; s < S; s++) mbar_init(&c.full[s], 1), mbar_init(&c.empty[s], 1);
        for (int b = 0; b < 2; b++) mbar_init(&c.dfull[b], 1), mbar_init(&c.dempty[b], 8);
        mbar_init(&c.done, 1);
        c.abort = 0;
        fence_mbar_init();
    }
    if (warp == 9) tmem_alloc(&c.tmem, 2 * NB);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = c.tmem;
    griddep_launch_dependents();
    griddep_wait();
    const int groups = f8_groups<MODE>(a, 128), items = groups * a.nt, nkb = a.nkb;

    if (warp >= 8) {
        setmaxnreg_dec<72>();
        if (warp == 8) {
            uint32_t g = 0;
            bool ok = true;
            const uint64_t pol_w = MODE == kF8Dense ? l2_evict_last() : l2_evict_first(), pol_x = l2_evict_last();
            for (int item = blockIdx.x; ok && item < items; item += gridDim.x) {
                int gi, n;
                many_tile<MODE>(a, item, groups, gi, n);
                const F8Group grp = f8_group<MODE>(a, gi, 128);
                int4 rows = make_int4(0, 0, 0, 0);
                if (MODE == kF8GateUp) {
                    const int c0 = 4 * lane;
                    const int32_t* p = a.perm + grp.row0;
                    rows = make_int4(__ldg(p + (c0 < grp.rows ? c0 : 0)), __ldg(p + (c0 + 1 < grp.rows ? c0 + 1 : 0)),
                                     __ldg(p + (c0 + 2 < grp.rows ? c0 + 2 : 0)), __ldg(p + (c0 + 3 < grp.rows ? c0 + 3 : 0)));
                }
                for (int kb = 0; kb < nkb; kb++, g++) {
                    const int s = g % S;
                    if (g >= (uint32_t)S) ok = f8_wait(&c.empty[s], ((g / S) & 1) ^ 1, &c.abort, a);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    unsigned char* st = ring + (size_t)s * C::kStage;
                    unsigned char* sw = st + 16384;
                    if (lane == 0) {
                        mbar_arrive_expect_tx(&c.full[s], C::kStage);
                        if (MODE == kF8GateUp) {
                            tma_load_3d(sw, &map_w, kb * 128, n * 128, grp.expert * 2, &c.full[s], pol_w);
                            tma_load_3d(sw + 16384, &map_w, kb * 128, n * 128, grp.expert * 2 + 1, &c.full[s], pol_w);
                        } else {
                            tma_load_2d(st, &map_x, kb * 128, grp.row0, &c.full[s], pol_x);
#pragma unroll
                            for (int h = 0; h < NB / 128; h++)
                                tma_load_3d(sw + h * 16384, &map_w, kb * 128, n * NB + h * 128, grp.expert, &c.full[s], pol_w);
                        }
                    }
                    if (MODE == kF8GateUp) {
                        __syncwarp();
                        tma_gather4(st + lane * 512, &map_x, kb * 128, rows, &c.full[s], pol_x);
                    }
                }
            }
            if (lane == 0) {
                const uint64_t t0 = globaltimer_ns();
                for (uint32_t q = g > (uint32_t)S ? g - S : 0; q < g; q++)
                    while (!mbar_try_wait(&c.full[q % S], (q / S) & 1))
                        if (globaltimer_ns() - t0 > a.timeout_ns) break;
            }
            __syncwarp();
        } else if (warp == 9) {
            if (lane == 0) {
                constexpr uint32_t idesc = f8_idesc(NB);
                uint32_t g = 0;
                bool ok = true;
                for (int item = blockIdx.x; ok && item < items; item += gridDim.x) {
                    for (int kb = 0; kb < nkb; kb++, g++) {
                        const int s = g % S, b = g & 1;
                        if (g >= 2) ok = f8_wait(&c.dempty[b], ((g >> 1) & 1) ^ 1, &c.abort, a);
                        ok = ok && f8_wait(&c.full[s], (g / S) & 1, &c.abort, a);
                        if (!ok) break;
                        tc_fence_after();
                        const uint32_t sx = smem_u32(ring + (size_t)s * C::kStage), sw = sx + 16384;
#pragma unroll
                        for (int kk = 0; kk < 4; kk++)
                            umma_f8(tmem + b * NB, sw128_desc(sx + kk * 32), sw128_desc(sw + kk * 32), idesc, kk > 0);
                        umma_commit(&c.empty[s]);
                        umma_commit(&c.dfull[b]);
                    }
                }
                if (*(volatile int*)&c.abort) {
                    umma_commit(&c.done);
                    const uint64_t t0 = globaltimer_ns();
                    while (!mbar_try_wait(&c.done, 0))
                        if (globaltimer_ns() - t0 > a.timeout_ns) break;
                }
            }
            __syncwarp();
        }
    } else {
        setmaxnreg_inc<216>();
        // epilogue: warp w holds token rows [32 (w % 4), ..), one a lane, and half the columns: segments of 64
        constexpr int SEG = NB / 128;
        const int q = warp & 3, half = warp >> 2, r = q * 32 + lane;
        int col[SEG];
#pragma unroll
        for (int i = 0; i < SEG; i++) col[i] = MODE == kF8GateUp ? i * 128 + half * 64 : (half * SEG + i) * 64;
        const uint32_t taddr = tmem + ((uint32_t)(q * 32) << 16);
        uint32_t g = 0;
        bool ok = true;
        for (int item = blockIdx.x; item < items; item += gridDim.x) {
            int gi, n;
            many_tile<MODE>(a, item, groups, gi, n);
            const F8Group grp = f8_group<MODE>(a, gi, 128);
            const bool live = r < grp.rows;
            const int slot = grp.row0 + (live ? r : 0);
            const float* xsp = a.xs + (size_t)(MODE == kF8GateUp ? __ldg(a.perm + slot) : slot) * nkb;
            const float* wsp[SEG];
#pragma unroll
            for (int i = 0; i < SEG; i++) {
                const int block = MODE == kF8GateUp ? n : min((n * NB + col[i]) / 128, a.nb - 1);
                wsp[i] = f8_wscale<MODE>(a, grp.expert, i, block);
            }
            f32x2 acc[SEG][32];
#pragma unroll
            for (int i = 0; i < SEG; i++)
#pragma unroll
                for (int j = 0; j < 32; j++) acc[i][j] = 0ull;
            float sx = __ldg(xsp), sw[SEG];
#pragma unroll
            for (int i = 0; i < SEG; i++) sw[i] = __ldg(wsp[i]);
            for (int kb = 0; kb < nkb; kb++, g++) {
                const int b = g & 1;
                f32x2 s[SEG];
#pragma unroll
                for (int i = 0; i < SEG; i++) s[i] = pack_f32x2(sx * sw[i], sx * sw[i]);
                if (kb + 1 < nkb) {
                    sx = __ldg(xsp + kb + 1);
#pragma unroll
                    for (int i = 0; i < SEG; i++) sw[i] = __ldg(wsp[i] + kb + 1);
                }
                ok = ok && f8_wait(&c.dfull[b], (g >> 1) & 1, &c.abort, a);
                __syncwarp();
                tc_fence_after();
                uint32_t v[2][32];
                tmem_ld32(taddr + b * NB + col[0], v[0]);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 2 * SEG; i++) {  // chunks of 32 columns; the next one is read while this one is added
                    if (i + 1 < 2 * SEG) tmem_ld32(taddr + b * NB + col[(i + 1) / 2] + ((i + 1) & 1) * 32, v[(i + 1) & 1]);
#pragma unroll
                    for (int j = 0; j < 16; j++)
                        acc[i / 2][(i & 1) * 16 + j] =
                            ffma2(pack_f32x2(__uint_as_float(v[i & 1][2 * j]), __uint_as_float(v[i & 1][2 * j + 1])), s[i / 2],
                                  acc[i / 2][(i & 1) * 16 + j]);
                    if (i + 1 < 2 * SEG) tmem_wait_ld();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&c.dempty[b]);
            }
            if (MODE == kF8GateUp) {
                uint32_t top = 0;
#pragma unroll
                for (int j = 0; j < 32; j++) {
                    float g0, g1, u0, u1;
                    unpack_f32x2(acc[0][j], g0, g1);
                    unpack_f32x2(acc[SEG - 1][j], u0, u1);
                    const float v0 = swiglu_f32(g0, u0), v1 = swiglu_f32(g1, u1);
                    acc[0][j] = pack_f32x2(v0, v1);
                    const uint32_t t0 = __float_as_uint(v0) & 0x7fffffffu, t1 = __float_as_uint(v1) & 0x7fffffffu;
                    top = max(top, t0 < 0x7f800000u ? t0 : 0u);
                    top = max(top, t1 < 0x7f800000u ? t1 : 0u);
                }
                c.top[half][r] = top;
                named_bar_sync(1, 256);
                top = max(c.top[0][r], c.top[1][r]);
                named_bar_sync(1, 256);  // read before the next item writes
                const uint32_t se = f8_scale_exp(top);
                const float inv = f8_inverse(se);
                const int f0 = n * 128 + half * 64;
                if (live) {
                    uint8_t* dst = a.aq + (size_t)slot * a.N + f0;
#pragma unroll
                    for (int j = 0; j < 4; j++) {  // sixteen values at a time (F is a multiple of 64)
                        float v[16];
#pragma unroll
                        for (int i = 0; i < 8; i++) unpack_f32x2(acc[0][8 * j + i], v[2 * i], v[2 * i + 1]);
                        const uint2 lo = f8_pack8(reinterpret_cast<const float(&)[8]>(v[0]), inv);
                        const uint2 hi = f8_pack8(reinterpret_cast<const float(&)[8]>(v[8]), inv);
                        if (f0 < a.N) reinterpret_cast<uint4*>(dst)[j] = make_uint4(lo.x, lo.y, hi.x, hi.y);
                    }
                    if (half == 0) a.as[(size_t)slot * a.nb + n] = __uint_as_float(se << 23);
                }
            } else if (live) {
#pragma unroll
                for (int i = 0; i < SEG; i++) {
                    const int n0 = n * NB + col[i];
                    const size_t at = (size_t)slot * a.N + n0;
                    if (MODE == kF8Down || a.out_f32) {
                        float* dst = static_cast<float*>(a.out) + at;
                        if (n0 + 64 <= a.N && a.N % 4 == 0) {
#pragma unroll
                            for (int j = 0; j < 16; j++)
                                reinterpret_cast<ulonglong2*>(dst)[j] = make_ulonglong2(acc[i][2 * j], acc[i][2 * j + 1]);
                        } else {
#pragma unroll
                            for (int j = 0; j < 32; j++) {
                                float v0, v1;
                                unpack_f32x2(acc[i][j], v0, v1);
                                if (n0 + 2 * j < a.N) dst[2 * j] = v0;
                                if (n0 + 2 * j + 1 < a.N) dst[2 * j + 1] = v1;
                            }
                        }
                    } else {
                        uint16_t* dst = static_cast<uint16_t*>(a.out) + at;
                        if (n0 + 64 <= a.N && a.N % 8 == 0) {
#pragma unroll
                            for (int j = 0; j < 8; j++) {
                                uint32_t o[4];
#pragma unroll
                                for (int k = 0; k < 4; k++) {
                                    float v0, v1;
                                    unpack_f32x2(acc[i][4 * j + k], v0, v1);
                                    o[k] = f8_bf16x2(v0, v1);
                                }
                                reinterpret_cast<uint4*>(dst)[j] = make_uint4(o[0], o[1], o[2], o[3]);
                            }
                        } else {
#pragma unroll
                            for (int j = 0; j < 32; j++) {
                                float v0, v1;
                                unpack_f32x2(acc[i][j], v0, v1);
                                if (n0 + 2 * j < a.N) dst[2 * j] = f8_bf16(v0);
                                if (n0 + 2 * j + 1 < a.N) dst[2 * j + 1] = f8_bf16(v1);
                            }
                        }
                    }
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        tc_fence_after();
        tmem_dealloc(tmem, 2 * NB);
    }
}

}  // namespace moe
