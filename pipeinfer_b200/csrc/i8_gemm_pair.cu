// i8_gemm_pair.cu -- 8-bit integer weights with a scale for each output times the tokens of long prompts: tcgen05 kind::i8 on pairs of SMs (cta_group::2).
//
// A pair forms 256 tokens x 256 outputs, tokens as M: each CTA brings its own 128 tokens and half of the weight rows, the tensor cores of both read both halves.
//   warp 0      streams a block of both operands by TMA through a ring; both CTAs' copies complete on the first CTA's barrier
//   warp 1      of the first CTA issues the MMAs of both; a tile is one accumulator over the whole of K, two of them take turns
//   warps 2..9  a thread owns a token (lane) and half of the tile's outputs, scaled and stored while the next tile's products run
// What bounds it: the tensor cores and, in a longer run, the power that they may take: 28672 x 8192 with 1,999 tokens 293 us in a single launch (3.2e15 operations a second, its tensor pipe 87 % busy),
// 366 to 375 in a loop with the rounding launch.
// Every wait is bounded (tc_common.cuh).
#include "i8_block.cuh"
#include "tc_common.cuh"

#include <algorithm>

#define IP_THREADS 320
#define IP_TILE    (128 * 128)
#define IP_STAGE   (2 * IP_TILE)
#define IP_STAGES  6
#define IP_RING    (IP_STAGES * IP_STAGE)
#define IP_BARS    (2 * IP_STAGES + 4)
#define IP_SMEM    ((size_t) IP_RING + IP_BARS * 8 + 32 + 1024)

// both operands of a block; called by a converged warp, one elected lane issues.  The first CTA (expect) announces the bytes of both CTAs' copies
__device__ __forceinline__ void ip_load(uint32_t dst, const CUtensorMap * xmap, const CUtensorMap * wmap, uint32_t bar, int m, int kb, int wrow, uint32_t expect, uint32_t own_bar) {
    asm volatile("{\n\t.reg .pred q, e;\n\telect.sync _|q, 0xffffffff;\n\tsetp.ne.and.b32 e, %8, 0, q;\n\t"
                 "@e mbarrier.arrive.expect_tx.shared::cta.b64 _, [%9], %10;\n\t"
                 "@q cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%2, {%11, %5, %6}], [%4];\n\t"
                 "@q cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%1], [%3, {%11, %7}], [%4];\n\t}"
                 ::"r"(dst), "r"(dst + IP_TILE), "l"(xmap), "l"(wmap), "r"(bar), "r"(m), "r"(kb), "r"(wrow), "r"(expect), "r"(own_bar), "r"(2 * IP_STAGE), "r"(0) : "memory");
}
// a block: four MMAs of K 32, 32 bytes further along both operands each; the commit hands the operands back in both CTAs
#define IP_MMA(A, B, ACC) "@q tcgen05.mma.cta_group::2.kind::i8 [%0], " A ", " B ", %3, {%4, %4, %4, %4, %4, %4, %4, %4}, " ACC ";\n\t"
#define IP_NEXT(D)        "add.s64 a, %1, " D ";\n\tadd.s64 b, %2, " D ";\n\t"
#define IP_COMMIT         "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 "
__device__ __forceinline__ void ip_step(uint32_t tmem_d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t bar_e, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p, q;\n\t.reg .b64 a, b;\n\telect.sync _|q, 0xffffffff;\n\tsetp.ne.b32 p, %7, 0;\n\t"
                 IP_MMA("%1", "%2", "p") IP_NEXT("2") IP_MMA("a", "b", "1") IP_NEXT("4") IP_MMA("a", "b", "1") IP_NEXT("6") IP_MMA("a", "b", "1")
                 "@q " IP_COMMIT "[%5], %6;\n\t}"
                 ::"r"(tmem_d), "l"(a), "l"(b), "r"(idesc), "r"(0u), "r"(bar_e), "h"((uint16_t) 3), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void ip_done(uint32_t bar_t) {
    asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\t@q " IP_COMMIT "[%0], %1;\n\t}" ::"r"(bar_t), "h"((uint16_t) 3) : "memory");
}

struct ip_args {
    int b, KB, NB, tiles_m, tiles, wide;             // wide: rows that stores of eight floats may take
    int64_t N;
    const float * ws, * ad;
    float * y;
    int * err;
};

__global__ void __launch_bounds__(IP_THREADS, 1)
i8_gemm_pair_kernel(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap wmap, const __grid_constant__ ip_args A) {
    extern __shared__ __align__(1024) uint8_t ip_dsm[];
    uint8_t *  sm  = ip_dsm + ((1024u - (dt_smem(ip_dsm) & 1023u)) & 1023u);
    uint64_t * bar = reinterpret_cast<uint64_t *>(sm + IP_RING);          // operands there[S], read[S], accumulator there[2], read[2]
    uint32_t * tmem_slot = reinterpret_cast<uint32_t *>(bar + IP_BARS);
    volatile int * abort_s = reinterpret_cast<volatile int *>(tmem_slot + 1);
    const uint32_t bar_f = dt_smem(bar), bar_e = bar_f + IP_STAGES * 8, bar_t = bar_e + IP_STAGES * 8, bar_r = bar_t + 16, sm0 = dt_smem(sm);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rank = (int) dt_cluster_rank(), pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

    if (threadIdx.x == 0) {
        for (int s = 0; s < IP_STAGES; s++) { dt_mbar_init(bar_f + s * 8, 1); dt_mbar_init(bar_e + s * 8, 1); }
        for (int a = 0; a < 2; a++) { dt_mbar_init(bar_t + a * 8, 1); dt_mbar_init(bar_r + a * 8, 16); }
        *abort_s = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dt_smem(tmem_slot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    dt_fence_before();
    __syncthreads();
    dt_cluster_sync();                                           // the other CTA's barriers and tensor memory are there
    dt_fence_after();
    const uint32_t tmem = *tmem_slot, lead_f = dt_mapa(bar_f, 0), lead_r = dt_mapa(bar_r, 0);
    pib_pdl_wait();
    pib_pdl_trigger();
    bool ok = true;

    if (warp == 0) {
        int s = 0;
        uint32_t ph = 1;                                         // the first round finds its stages free
        for (int tile = pair; tile < A.tiles && ok; tile += pairs) {
            const int m0 = tile % A.tiles_m * 256 + rank * 128, nb = tile / A.tiles_m * 2 + rank;
            for (int kb = 0; kb < A.KB; kb++) {
                ok = __all_sync(0xffffffffu, dt_mbar_wait(bar_e + s * 8, ph, abort_s));
                if (!ok) break;
                ip_load(sm0 + s * IP_STAGE, &xmap, &wmap, lead_f + s * 8, m0, kb, (nb * A.KB + kb) * 128, rank == 0, bar_f + s * 8);
                if (++s == IP_STAGES) { s = 0; ph ^= 1; }
            }
        }
    } else if (warp == 1) {
        if (rank == 0) {
            const uint32_t idesc = (2u << 4) | (1u << 7) | (1u << 10) | (256u >> 3 << 17) | (256u >> 4 << 24);     // 32-bit integer accumulators, int8 x int8, both K-major, 256 x 256
            const uint64_t d0 = dt_desc(sm0);
            int  s = 0, a = 0;
            uint32_t ph = 0, aph = 1;
            for (int tile = pair; tile < A.tiles && ok; tile += pairs) {
                ok = __all_sync(0xffffffffu, dt_mbar_wait(bar_r + a * 8, aph, abort_s));
                for (int kb = 0; kb < A.KB && ok; kb++) {
                    ok = __all_sync(0xffffffffu, dt_mbar_wait(bar_f + s * 8, ph, abort_s));
                    if (!ok) break;
                    dt_fence_after();
                    const uint64_t ad = d0 + (uint64_t) (s * IP_STAGE >> 4);
                    ip_step(tmem + a * 256, ad, ad + (IP_TILE >> 4), idesc, bar_e + s * 8, kb > 0);
                    if (++s == IP_STAGES) { s = 0; ph ^= 1; }
                }
                if (!ok) break;
                ip_done(bar_t + a * 8);
                if (++a == 2) { a = 0; aph ^= 1; }
            }
        }
    } else {
        const int q4 = warp & 3, hf = (warp - 2) >> 2;           // 128 columns: one weight block
        const uint32_t at = tmem + ((uint32_t) (q4 * 32) << 16) + hf * 128;
        int a = 0;
        uint32_t aph = 0;
        for (int tile = pair; tile < A.tiles && ok; tile += pairs) {
            const int     tk = tile % A.tiles_m * 256 + rank * 128 + q4 * 32 + lane;
            const int64_t n0 = (int64_t) (tile / A.tiles_m * 2 + hf) * 128;
            const bool    in = tk < A.b && n0 < A.N;
            const float   d = in ? __ldg(A.ad + tk) : 0.f;
            float *       y = A.y + (int64_t) tk * A.N + n0;
            const int     left = (int) max((int64_t) 0, min((int64_t) 128, A.N - n0));
            ok = __all_sync(0xffffffffu, dt_mbar_wait(bar_t + a * 8, aph, abort_s));
            if (!ok) break;
            dt_fence_after();
#pragma unroll
            for (int c = 0; c < 128; c += 32) {
                uint32_t v[32];
                dt_ld32(at + a * 256 + c, v);
                dt_wait_ld();
                if (c == 96) {                                   // all read: the accumulator goes back in front of the last stores
                    dt_fence_before();
                    __syncwarp();
                    // relaxed: no memory is handed over with it
                    if (lane == 0) asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(lead_r + a * 8) : "memory");
                }
                if (!in) continue;
                if (A.wide && left == 128) {
#pragma unroll
                    for (int j = 0; j < 32; j += 8) {
                        const float4 s0 = __ldg(reinterpret_cast<const float4 *>(A.ws + n0 + c + j)), s1 = __ldg(reinterpret_cast<const float4 *>(A.ws + n0 + c + j) + 1);
                        const float o[8] = { i8_out((int) v[j], d, s0.x), i8_out((int) v[j + 1], d, s0.y), i8_out((int) v[j + 2], d, s0.z), i8_out((int) v[j + 3], d, s0.w),
                                             i8_out((int) v[j + 4], d, s1.x), i8_out((int) v[j + 5], d, s1.y), i8_out((int) v[j + 6], d, s1.z), i8_out((int) v[j + 7], d, s1.w) };
                        asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(y + c + j), "f"(o[0]), "f"(o[1]), "f"(o[2]), "f"(o[3]), "f"(o[4]), "f"(o[5]), "f"(o[6]), "f"(o[7]) : "memory");
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 32; j++) if (c + j < left) y[c + j] = i8_out((int) v[j], d, __ldg(A.ws + n0 + c + j));
                }
            }
            if (++a == 2) { a = 0; aph ^= 1; }
        }
    }
    __syncwarp();
    dt_fence_before();
    __syncthreads();
    if (*abort_s) {
        // a wait ran out: say so, give copies and MMAs still in flight time to land (bounded), then free the tensor memory
        if (threadIdx.x == 0) atomicExch(A.err, 1 + (int) blockIdx.x);
        for (int i = 0; i < 2000; i++) __nanosleep(1000);
        __syncthreads();
    }
    dt_cluster_sync();                                           // both CTAs have read their accumulators, nothing arrives at a barrier any more
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

int pib_i8_gemm_pair(const pib_weight * w, const void * act, int b, float * y, int * err, cudaStream_t st) {
    const pib_i8_act L = pib_i8_act_of(w->K, b);
    ip_args A;
    A.b = b; A.KB = L.KB; A.NB = (int) pib_f8_blocks(w->N); A.N = w->N; A.y = y; A.err = err;
    A.ws = (const float *) w->d; A.ad = (const float *) ((const uint8_t *) act + L.d_off);
    A.wide = w->N % 8 == 0 && !((uintptr_t) y & 31);
    A.tiles_m = (b + 255) / 256;
    A.tiles = (A.NB + 1) / 2 * A.tiles_m;
    CUtensorMap xmap;
    int rc;
    if ((rc = pib_f8_map3(&xmap, act, b, L.KB, (int64_t) b * PIB_F8_BLOCK, 128, 1)) != PIB_OK) return rc;
    static pib_per_device attrs;
    PIB_CHECK(attrs.once([&] { return cudaFuncSetAttribute(i8_gemm_pair_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int) IP_SMEM); }));
    PIB_CHECK(pib_launch_cluster(i8_gemm_pair_kernel, dim3((unsigned) (2 * std::min(A.tiles, pib_num_sms() / 2))), dim3(IP_THREADS), dim3(2, 1, 1), IP_SMEM, st, xmap, ((const pib_f8_maps *) w->map)->block, A));
    return PIB_OK;
}
