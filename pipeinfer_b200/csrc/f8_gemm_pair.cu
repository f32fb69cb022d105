// f8_gemm_pair.cu -- 8-bit floating point weights with block scales times the tokens of long prompts: tcgen05 kind::f8f6f4 on pairs of SMs (cta_group::2).
//
//   y[t][n] = sum over kb of (d[kb][t] s[n/128][kb]) P_kb[t][n],  P_kb = the product of the block's 128 columns
//
// A pair forms 256 tokens x 256 outputs, tokens as M: each CTA brings its own 128 tokens and half of the weight rows, the tensor cores of both read both halves.
//   warp 0       streams a block of both operands by TMA through a ring; both CTAs' copies complete on the first CTA's barrier
//   warp 1       of the first CTA issues the MMAs of both: a block is one accumulator, two of them take turns
//   warp 2       makes the factors f = d s of a block's tokens and both weight blocks
//   warps 3..18  a thread owns a token (lane) and half of the outputs of one weight block: acc[c] += P[c] f with ONE factor f = d s for its 64 outputs
// That the factor is one number per thread is why the tokens are M here (f8_gemm.cu has them as N: a factor per column, whose product costs as much as the sum).
// What bounds it: an accumulator's round -- MMAs, their commit to both CTAs, reading it, handing it back -- with two of them in tensor memory, and the sums between the reads: 28672 x 8192 at
// 1 999 tokens takes 526 us (1.79 PFLOP/s) in a short burst, 404 without sums, 292 without reads.  Eight warps of 128 columns, which hold 128 sums a thread, take 562; four accumulators of
// 128 columns 562, since MMAs that narrow read the tokens twice.
// Every wait is bounded (tc_common.cuh).
#include "f8_block.cuh"
#include "tc_common.cuh"

#include <algorithm>

#define FP_THREADS 608
#define FP_FRING   8                          // factor rows under way
#define FP_TILE    (128 * 128)
#define FP_STAGE   (2 * FP_TILE)
#define FP_STAGES  6
#define FP_RING    (FP_STAGES * FP_STAGE)
#define FP_BARS    (2 * FP_STAGES + 4 + 2 * FP_FRING)
#define FP_SMEM    ((size_t) FP_RING + FP_FRING * 1024 + FP_BARS * 8 + 32 + 1024)

// both operands of a block; called by a converged warp, one elected lane issues.  The first CTA (expect) announces the bytes of both CTAs' copies
__device__ __forceinline__ void fp_load(uint32_t dst, const CUtensorMap * xmap, const CUtensorMap * wmap, uint32_t bar, int m, int kb, int wrow, uint32_t expect, uint32_t own_bar) {
    asm volatile("{\n\t.reg .pred q, e;\n\telect.sync _|q, 0xffffffff;\n\tsetp.ne.and.b32 e, %8, 0, q;\n\t"
                 "@e mbarrier.arrive.expect_tx.shared::cta.b64 _, [%9], %10;\n\t"
                 "@q cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%2, {%11, %5, %6}], [%4];\n\t"
                 "@q cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%1], [%3, {%11, %7}], [%4];\n\t}"
                 ::"r"(dst), "r"(dst + FP_TILE), "l"(xmap), "l"(wmap), "r"(bar), "r"(m), "r"(kb), "r"(wrow), "r"(expect), "r"(own_bar), "r"(2 * FP_STAGE), "r"(0) : "memory");
}
// a block: four MMAs of K 32, 32 bytes further along both operands each, the first one starting the accumulator; commits hand the operands back and the accumulator over, in both CTAs
#define FP_MMA(A, B, ACC) "@q tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], " A ", " B ", %3, {%4, %4, %4, %4, %4, %4, %4, %4}, " ACC ";\n\t"
#define FP_NEXT(D)        "add.s64 a, %1, " D ";\n\tadd.s64 b, %2, " D ";\n\t"
#define FP_COMMIT         "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 "
__device__ __forceinline__ void fp_step(uint32_t tmem_d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t bar_e, uint32_t bar_t) {
    asm volatile("{\n\t.reg .pred q;\n\t.reg .b64 a, b;\n\telect.sync _|q, 0xffffffff;\n\t"
                 FP_MMA("%1", "%2", "0") FP_NEXT("2") FP_MMA("a", "b", "1") FP_NEXT("4") FP_MMA("a", "b", "1") FP_NEXT("6") FP_MMA("a", "b", "1")
                 FP_COMMIT "[%5], %7;\n\t" FP_COMMIT "[%6], %7;\n\t}"
                 ::"r"(tmem_d), "l"(a), "l"(b), "r"(idesc), "r"(0u), "r"(bar_e), "r"(bar_t), "h"((uint16_t) 3) : "memory");
}
__device__ __forceinline__ unsigned long long fp_fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
    unsigned long long d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ unsigned long long fp_pack(uint32_t lo, uint32_t hi) { return (unsigned long long) hi << 32 | lo; }

__device__ __forceinline__ void fp_ld16(uint32_t at, uint32_t * v) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]),
                   "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]) : "r"(at) : "memory");
}
struct fp_args {
    int b, KB, NB, bp, tiles_m, tiles, wide;         // wide: rows that stores of eight floats may take
    int64_t N;
    const float * ws, * ad;
    float * y;
    int * err;
};

__global__ void __launch_bounds__(FP_THREADS, 1)
f8_gemm_pair_kernel(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap wmap, const __grid_constant__ fp_args A) {
    extern __shared__ __align__(1024) uint8_t fp_dsm[];
    uint8_t *  sm  = fp_dsm + ((1024u - (dt_smem(fp_dsm) & 1023u)) & 1023u);
    uint64_t * bar = reinterpret_cast<uint64_t *>(sm + FP_RING + FP_FRING * 1024);          // operands there[S], read[S], accumulator there[2], read[2], factors there[F], read[F]
    float *    fac = reinterpret_cast<float *>(sm + FP_RING);             // [F][2 weight blocks][128 tokens]
    uint32_t * tmem_slot = reinterpret_cast<uint32_t *>(bar + FP_BARS);
    volatile int * abort_s = reinterpret_cast<volatile int *>(tmem_slot + 1);
    const uint32_t bar_f = dt_smem(bar), bar_e = bar_f + FP_STAGES * 8, bar_t = bar_e + FP_STAGES * 8, bar_r = bar_t + 16, bar_d = bar_r + 16, bar_g = bar_d + FP_FRING * 8, sm0 = dt_smem(sm);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rank = (int) dt_cluster_rank(), pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

    if (threadIdx.x == 0) {
        for (int s = 0; s < FP_STAGES; s++) { dt_mbar_init(bar_f + s * 8, 1); dt_mbar_init(bar_e + s * 8, 1); }
        for (int a = 0; a < 2; a++) { dt_mbar_init(bar_t + a * 8, 1); dt_mbar_init(bar_r + a * 8, 32); }
        for (int f = 0; f < FP_FRING; f++) { dt_mbar_init(bar_d + f * 8, 1); dt_mbar_init(bar_g + f * 8, 16); }
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
                fp_load(sm0 + s * FP_STAGE, &xmap, &wmap, lead_f + s * 8, m0, kb, (nb * A.KB + kb) * 128, rank == 0, bar_f + s * 8);
                if (++s == FP_STAGES) { s = 0; ph ^= 1; }
            }
        }
    } else if (warp == 1) {
        if (rank == 0) {
            const uint32_t idesc = (1u << 4) | (256u >> 3 << 17) | (256u >> 4 << 24);     // fp32 accumulators, e4m3 x e4m3, both K-major, 256 x 256
            const uint64_t d0 = dt_desc(sm0);
            int  s = 0, a = 0;
            uint32_t ph = 0, aph = 1;
            for (int tile = pair; tile < A.tiles && ok; tile += pairs)
                for (int kb = 0; kb < A.KB; kb++) {
                    ok = __all_sync(0xffffffffu, dt_mbar_wait(bar_r + a * 8, aph, abort_s) && dt_mbar_wait(bar_f + s * 8, ph, abort_s));
                    if (!ok) break;
                    dt_fence_after();
                    const uint64_t ad = d0 + (uint64_t) (s * FP_STAGE >> 4);
                    fp_step(tmem + a * 256, ad, ad + (FP_TILE >> 4), idesc, bar_e + s * 8, bar_t + a * 8);
                    if (++s == FP_STAGES) { s = 0; ph ^= 1; }
                    if (++a == 2) { a = 0; aph ^= 1; }
                }
        }
    } else if (warp == 2) {
        // four tokens a lane, four blocks under way in registers that keep their places
        int fs = 0;
        uint32_t fph = 1;
        for (int tile = pair; tile < A.tiles && ok; tile += pairs) {
            const int    m = tile % A.tiles_m * 256 + rank * 128 + lane * 4, nb = tile / A.tiles_m * 2;
            const bool   in = m < A.bp, two = nb + 1 < A.NB;
            const float * ad = A.ad + m, * w0 = A.ws + (int64_t) nb * A.KB, * w1 = w0 + (two ? A.KB : 0);
            float4 d[4];
            float  wa[4], wb[4];
            auto ask = [&](int kb, int u) {
                const bool there = kb < A.KB;
                d[u] = there && in ? __ldg(reinterpret_cast<const float4 *>(ad + (int64_t) kb * A.bp)) : make_float4(0.f, 0.f, 0.f, 0.f);
                wa[u] = there ? __ldg(w0 + kb) : 0.f; wb[u] = there ? __ldg(w1 + kb) : 0.f;
            };
#pragma unroll
            for (int u = 0; u < 4; u++) ask(u, u);
            for (int kb0 = 0; kb0 < A.KB && ok; kb0 += 4)
#pragma unroll
                for (int u = 0; u < 4; u++)
                    if (kb0 + u < A.KB && ok) {
                        ok = __all_sync(0xffffffffu, dt_mbar_wait(bar_g + fs * 8, fph, abort_s));
                        if (ok) {
                            float4 * o = reinterpret_cast<float4 *>(fac + fs * 256) + lane;
                            o[0]  = make_float4(d[u].x * wa[u], d[u].y * wa[u], d[u].z * wa[u], d[u].w * wa[u]);
                            o[32] = make_float4(d[u].x * wb[u], d[u].y * wb[u], d[u].z * wb[u], d[u].w * wb[u]);
                            __syncwarp();
                            if (lane == 0) dt_arrive(bar_d + fs * 8);
                            ask(kb0 + u + 4, u);
                            if (++fs == FP_FRING) { fs = 0; fph ^= 1; }
                        }
                    }
        }
    } else {
        const int q4 = warp & 3, part = (warp - 3) >> 2, hf = part >> 1;       // 64 columns
        const uint32_t at = tmem + ((uint32_t) (q4 * 32) << 16) + part * 64;
        unsigned long long acc[32];
        int a = 0, fs = 0;
        uint32_t aph = 0, fph = 0;
        for (int tile = pair; tile < A.tiles && ok; tile += pairs) {
            const int  tk = tile % A.tiles_m * 256 + rank * 128 + q4 * 32 + lane, nb = tile / A.tiles_m * 2 + hf;
            const bool in = tk < A.b && nb < A.NB;
#pragma unroll
            for (int c = 0; c < 32; c++) acc[c] = 0;
            for (int kb = 0; kb < A.KB; kb++) {
                ok = __all_sync(0xffffffffu, dt_mbar_wait(bar_d + fs * 8, fph, abort_s));
                if (!ok) break;
                const uint32_t f = __float_as_uint(fac[fs * 256 + hf * 128 + q4 * 32 + lane]);
                const unsigned long long ff = fp_pack(f, f);
                ok = __all_sync(0xffffffffu, dt_mbar_wait(bar_t + a * 8, aph, abort_s));
                if (!ok) break;
                dt_fence_after();
                uint32_t v[16];
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    fp_ld16(at + a * 256 + c * 16, v);
                    dt_wait_ld();
                    if (c == 3) {                                // all read: the accumulator goes back in front of the last sums
                        dt_fence_before();
                        __syncwarp();
                        // relaxed: no memory is handed over with it (a release at cluster scope in its place took twice the time)
                        if (lane == 0) {
                            asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(lead_r + a * 8) : "memory");
                            dt_arrive(bar_g + fs * 8);
                        }
                    }
#pragma unroll
                    for (int j = 0; j < 8; j++) acc[c * 8 + j] = fp_fma2(fp_pack(v[2 * j], v[2 * j + 1]), ff, acc[c * 8 + j]);
                }
                if (++a == 2) { a = 0; aph ^= 1; }
                if (++fs == FP_FRING) { fs = 0; fph ^= 1; }
            }
            if (!ok) break;
            if (!in) continue;
            const int64_t n0 = (int64_t) nb * 128 + (part & 1) * 64;
            float * y = A.y + (int64_t) tk * A.N + n0;
            const int left = (int) min((int64_t) 64, A.N - n0);
            if (A.wide && left == 64) {
#pragma unroll
                for (int c = 0; c < 32; c += 4)
                    asm volatile("st.global.v4.b64 [%0], {%1, %2, %3, %4};" ::"l"(y + c * 2), "l"(acc[c]), "l"(acc[c + 1]), "l"(acc[c + 2]), "l"(acc[c + 3]) : "memory");
            } else {
#pragma unroll
                for (int c = 0; c < 32; c++) {
                    if (2 * c < left)     y[2 * c]     = __uint_as_float((uint32_t) acc[c]);
                    if (2 * c + 1 < left) y[2 * c + 1] = __uint_as_float((uint32_t) (acc[c] >> 32));
                }
            }
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

int pib_f8_gemm_pair(const pib_weight * w, const void * act, int b, float * y, int * err, cudaStream_t st) {
    const pib_f8_act L = pib_f8_act_of(w->K, b);
    fp_args A;
    A.b = b; A.KB = L.KB; A.NB = (int) pib_f8_blocks(w->N); A.bp = L.bp; A.N = w->N; A.y = y; A.err = err;
    A.ws = (const float *) w->d; A.ad = (const float *) ((const uint8_t *) act + L.d_off);
    A.wide = w->N % 8 == 0 && !((uintptr_t) y & 31);
    A.tiles_m = (b + 255) / 256;
    A.tiles = (A.NB + 1) / 2 * A.tiles_m;
    CUtensorMap xmap;
    int rc;
    if ((rc = pib_f8_map3(&xmap, act, b, L.KB, (int64_t) b * PIB_F8_BLOCK, 128, 1)) != PIB_OK) return rc;
    static pib_per_device attrs;
    PIB_CHECK(attrs.once([&] { return cudaFuncSetAttribute(f8_gemm_pair_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int) FP_SMEM); }));
    PIB_CHECK(pib_launch_cluster(f8_gemm_pair_kernel, dim3((unsigned) (2 * std::min(A.tiles, pib_num_sms() / 2))), dim3(FP_THREADS), dim3(2, 1, 1), FP_SMEM, st, xmap, ((const pib_f8_maps *) w->map)->block, A));
    return PIB_OK;
}
