// f8_gemm.cu -- 8-bit floating point weights with block scales times up to 128 tokens (f8_gemm_pair.cu beyond) on tcgen05 (kind::f8f6f4), fp32 accumulation.
//
//   y[t][n] = sum over kb of (s[n/128][kb] d[kb][t]) P_kb[n][t],  P_kb = the product of the block's 128 columns
//
// The scales change from block to block, so a block's product is one accumulator in tensor memory (four MMAs of K 32) that is read back, scaled and added up in fp32 registers, while the
// tensor core works on the next blocks' accumulators.
//   warp 0       streams blocks of both operands by TMA (a row's 128 bytes are a line of the 128-byte swizzle) through a ring
//   warp 10      streams the blocks' activation scales through a ring of their own
//   warp 1       issues the MMAs; a commit hands the operands back, another says that the accumulator is there
//   warps 2..9   two groups of four, half of the columns each: a thread owns a weight row (lane) and adds acc[c] += P[c] (s d[c])
// The CTAs walk tiles of up to 128 rows, all the tokens wide (NB: 16 .. 128, the smallest that holds them), each CTA a part of the rows (ft_grain).  Where the tiles leave most SMs idle, 2, 4 or 8
// CTAs of a cluster take a share of the blocks each and add their sums up through distributed shared memory, in share order.  (Clusters that share every tile of a longer walk lose: a meeting
// costs 3 us, 21 999 x 5700 with 13 tokens takes 36 us on pairs and 41 on fours instead of 29.)
// What bounds it: up to 48 tokens the weights' way from memory and an uneven last tile (57344 x 8192, 13 tokens: 88 us, 0.83 of the copy rate; 10240 x 8192, 40 tokens: 23 us on 80 SMs, 19 without
// any sums); beyond, reading the accumulators and adding them up (28672 x 8192, 128 tokens: 70 us, 1 000 clocks a block, of which the MMAs take 256).
// Every wait is bounded (tc_common.cuh).
#include "f8_block.cuh"
#include "tc_common.cuh"

#include <algorithm>

#define FT_THREADS 352
#define FT_BM      128
#define FT_A_TILE  (FT_BM * 128)
#define FT_RING    (192 * 1024)
#define FT_STAGES  10                       // at most
#define FT_KPS     2                        // blocks of a stage, and of a hand-over between the warps: fewer and larger ones (57344 x 8192, 4 tokens: 133 us with 1, 89 with 2)
#define FT_DRING   8                        // stages whose scale rows are under way
#define FT_BARS    (2 * FT_STAGES + 2 * FT_DRING + 2 * 16)
#define FT_SMEM    ((size_t) FT_RING + FT_DRING * FT_KPS * 512 + FT_BARS * 8 + 32 + 1024)

__device__ __forceinline__ void ft_mma(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc) {
    // a block: four MMAs of K 32, 32 bytes further along both operands each; the first one starts the accumulator
    asm volatile("{\n\t.reg .pred q;\n\t.reg .b64 a, b;\n\telect.sync _|q, 0xffffffff;\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, {%4, %4, %4, %4}, 0;\n\t"
                 "add.s64 a, %1, 2;\n\tadd.s64 b, %2, 2;\n\t@q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a, b, %3, {%4, %4, %4, %4}, 1;\n\t"
                 "add.s64 a, %1, 4;\n\tadd.s64 b, %2, 4;\n\t@q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a, b, %3, {%4, %4, %4, %4}, 1;\n\t"
                 "add.s64 a, %1, 6;\n\tadd.s64 b, %2, 6;\n\t@q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a, b, %3, {%4, %4, %4, %4}, 1;\n\t}"
                 ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(0u) : "memory");
}
__device__ __forceinline__ void ft_tma_2d(uint32_t dst, const CUtensorMap * map, uint32_t bar, int x, int y) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void ft_tma_4d(uint32_t dst, const CUtensorMap * map, uint32_t bar, int y, int z, int u) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst), "l"(map), "r"(bar), "r"(0), "r"(y), "r"(z), "r"(u) : "memory");
}
__device__ __forceinline__ void ft_tma_3d(uint32_t dst, const CUtensorMap * map, uint32_t bar, int y, int z) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst), "l"(map), "r"(bar), "r"(0), "r"(y), "r"(z) : "memory");
}
__device__ __forceinline__ void ft_bulk(uint32_t dst, const void * src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
template <int N> __device__ __forceinline__ void ft_ld(uint32_t at, uint32_t (&v)[N]) {
    if constexpr (N == 32) dt_ld32(at, v);
    else if constexpr (N == 16)
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                     : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]),
                       "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]) : "r"(at) : "memory");
    else
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]) : "r"(at) : "memory");
}
// M x N outputs of e4m3 x e4m3, fp32 accumulators, both operands K-major
__host__ __device__ constexpr uint32_t ft_idesc(int M, int N) { return (1u << 4) | ((uint32_t) (N >> 3) << 17) | ((uint32_t) (M >> 4) << 24); }

struct ft_args {
    int b, KB, bp, runs, shares;                                 // runs: of 32 rows, in all
    int64_t N;
    const float * ws, * ad;
    float * y;
    int * err;
};

// A CTA's rows begin at a multiple of so many runs of 32.  One divides the rows more evenly, four leave the weights' scales the same in all warps.  us with 1, with 4:
//   21 999 x 5700, 13 tokens  29.6  32.4      28 672 x 8192, 64 tokens  52  49      10 240 x 8192, 40 tokens  23.9  23.0      28 672 x 8192, 128 tokens  73  69
__host__ __device__ constexpr int ft_grain(int NB) { return NB <= 32 ? 1 : 4; }
template <int NB>
__global__ void __launch_bounds__(FT_THREADS, 1)
f8_gemm_kernel(const __grid_constant__ pib_f8_runs wmaps, const __grid_constant__ CUtensorMap xmap, const __grid_constant__ ft_args A) {
    constexpr int KPS = FT_KPS, STAGE = KPS * (FT_A_TILE + NB * 128), STAGES = FT_RING / STAGE < FT_STAGES ? FT_RING / STAGE : FT_STAGES, PITCH = NB <= 16 ? 16 : NB <= 32 ? 32 : NB <= 64 ? 64 : 128, ACCS = 512 / (KPS * PITCH), HALF = NB / 2, GRAIN = ft_grain(NB);
    extern __shared__ __align__(1024) uint8_t ft_dsm[];
    uint8_t *  sm  = ft_dsm + ((1024u - (dt_smem(ft_dsm) & 1023u)) & 1023u);
    float *    dsc = reinterpret_cast<float *>(sm + FT_RING);                            // scale rows, KPS of 128 floats a place
    uint64_t * bar = reinterpret_cast<uint64_t *>(sm + FT_RING + FT_DRING * FT_KPS * 512);       // operands there / read, scales there / read, accumulator there / read
    uint32_t * tmem_slot = reinterpret_cast<uint32_t *>(bar + FT_BARS);
    volatile int * abort_s = reinterpret_cast<volatile int *>(tmem_slot + 1);
    const uint32_t bar_f = dt_smem(bar), bar_e = bar_f + FT_STAGES * 8, bar_d = bar_e + FT_STAGES * 8, bar_g = bar_d + FT_DRING * 8, bar_t = bar_g + FT_DRING * 8, bar_r = bar_t + 16 * 8;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, S = A.shares, share = S > 1 ? (int) dt_cluster_rank() : 0;
    // the rows of a CTA (cluster) are neighbours, in runs of 32; its tiles take up to four runs each, as alike as can be
    const int unit = blockIdx.x / S, units = gridDim.x / S;
    const int grains = (A.runs + GRAIN - 1) / GRAIN, r0 = (int) ((int64_t) grains * unit / units) * GRAIN;
    const int runs = min(A.runs, (int) ((int64_t) grains * (unit + 1) / units) * GRAIN) - r0, tiles = (runs + 3) / 4, each = runs / tiles, more = runs % tiles;
    // a tile's first run, and how many; where rows go by blocks of four runs no tile reaches into the next
    auto run_of  = [&](int tile) { return r0 + (GRAIN == 4 ? tile * 4 : tile * each + min(tile, more)); };
    auto runs_of = [&](int tile) { return GRAIN == 4 ? min(4, runs - tile * 4) : each + (tile < more); };
    const int k0 = (int) ((int64_t) A.KB * share / S), nk = (int) ((int64_t) A.KB * (share + 1) / S) - k0;
    const uint32_t sm0 = dt_smem(sm);

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; s++) { dt_mbar_init(bar_f + s * 8, 1); dt_mbar_init(bar_e + s * 8, 1); }
        for (int s = 0; s < FT_DRING; s++) { dt_mbar_init(bar_d + s * 8, 1); dt_mbar_init(bar_g + s * 8, 8); }
        for (int a = 0; a < ACCS; a++) { dt_mbar_init(bar_t + a * 8, 1); dt_mbar_init(bar_r + a * 8, 8); }
        *abort_s = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dt_smem(tmem_slot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    dt_fence_before();
    __syncthreads();
    dt_fence_after();
    const uint32_t tmem = *tmem_slot;
    pib_pdl_wait();
    pib_pdl_trigger();
    bool ok = true;

    if (warp == 0) {
        int s = 0;
        uint32_t ph = 1;                                         // the first round finds its places free
        for (int tile = 0; tile < tiles && ok && lane == 0; tile++) {
            // rows of the tile in one block of the weights' layout, and in the next
            const int t0 = run_of(tile), n = runs_of(tile), n1 = GRAIN == 4 ? n : min(n, 4 - (t0 & 3)), n2 = n - n1;
            for (int kt = 0; kt < nk; kt += KPS) {
                ok = dt_mbar_wait(bar_e + s * 8, ph, abort_s);
                if (!ok) break;
                const int      ks = n1 == 4 ? KPS : min(KPS, nk - kt);         // (what a share's last copies take of the next block is not used)
                const uint32_t to = sm0 + s * STAGE;
                dt_mbar_expect_tx(bar_f + s * 8, ks * n * 4096 + KPS * NB * 128);
                static_assert(KPS == 2, "a copy of whole blocks");
                if (n1 == 4) ft_tma_2d(to, &wmaps.m[4], bar_f + s * 8, 0, (t0 / 4 * A.KB + k0 + kt) * 128);
                else for (int j = 0; j < ks; j++) {
                    ft_tma_4d(to + j * FT_A_TILE, &wmaps.m[n1 - 1], bar_f + s * 8, t0 % 4 * 32, k0 + kt + j, t0 / 4);
                    if (n2) ft_tma_4d(to + j * FT_A_TILE + n1 * 4096, &wmaps.m[n2 - 1], bar_f + s * 8, 0, k0 + kt + j, t0 / 4 + 1);
                }
                ft_tma_3d(to + KPS * FT_A_TILE, &xmap, bar_f + s * 8, 0, k0 + kt);
                if (++s == STAGES) { s = 0; ph ^= 1; }
            }
        }
        __syncwarp();
    } else if (warp == 10) {
        int ds = 0;
        uint32_t dph = 1;
        const uint32_t dbytes = (uint32_t) min(NB, A.bp) * 4;
        for (int tile = 0; tile < tiles && ok && lane == 0; tile++) {
            for (int kt = 0; kt < nk; kt += KPS) {
                ok = dt_mbar_wait(bar_g + ds * 8, dph, abort_s);
                if (!ok) break;
                const int n = min(KPS, nk - kt);
                dt_mbar_expect_tx(bar_d + ds * 8, n * dbytes);
                for (int j = 0; j < n; j++) ft_bulk(dt_smem(dsc + (ds * KPS + j) * 128), A.ad + (int64_t) (k0 + kt + j) * A.bp, dbytes, bar_d + ds * 8);
                if (++ds == FT_DRING) { ds = 0; dph ^= 1; }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        const uint64_t d0 = dt_desc(sm0);
        int s = 0, a = 0;
        uint32_t ph = 0, aph = 1;
        for (int tile = 0; tile < tiles && ok; tile++)
            for (int kt = 0; kt < nk; kt += KPS) {
                ok = __all_sync(0xffffffffu, dt_mbar_wait(bar_r + a * 8, aph, abort_s) && dt_mbar_wait(bar_f + s * 8, ph, abort_s));
                if (!ok) break;
                dt_fence_after();
#pragma unroll
                for (int j = 0; j < KPS; j++) {
                    const uint64_t ad = d0 + (uint64_t) ((s * STAGE + j * FT_A_TILE) >> 4), bd = d0 + (uint64_t) ((s * STAGE + KPS * FT_A_TILE + j * NB * 128) >> 4);
                    if (kt + j < nk) ft_mma(tmem + (a * KPS + j) * PITCH, ad, bd, ft_idesc(FT_BM, NB));
                }
                dt_commit(bar_t + a * 8);
                dt_commit(bar_e + s * 8);
                if (++s == STAGES) { s = 0; ph ^= 1; }
                if (++a == ACCS) { a = 0; aph ^= 1; }
            }
    } else {
        const int q4 = warp & 3, hf = (warp - 2) >> 2;
        const uint32_t lanes = (uint32_t) (q4 * 32) << 16;
        float acc[HALF];
        int a = 0, ds = 0;
        uint32_t aph = 0, dph = 0;
        for (int tile = 0; tile < tiles && ok; tile++) {
            const int  t0 = run_of(tile), run = t0 + q4;      // the warp's rows
            const bool in  = q4 < runs_of(tile);
            const int64_t n = (int64_t) run * 32 + lane;
            int m0 = hf * HALF;
            asm volatile("" : "+r"(m0));                         // keeps the outputs' addresses from being made, and held, ahead of the tiles
            // (a warp without rows goes along: a branch of its own in front of tcgen05.ld costs the others a tenth)
            const float * ws = A.ws + (int64_t) (GRAIN == 4 ? t0 / 4 : in ? run / 4 : 0) * A.KB + k0;
#pragma unroll
            for (int c = 0; c < HALF; c++) acc[c] = 0.f;
            for (int kt = 0; kt < nk; kt += KPS) {
                float w[KPS];
#pragma unroll
                for (int j = 0; j < KPS; j++) w[j] = kt + j < nk ? __ldg(ws + kt + j) : 0.f;
                ok = __all_sync(0xffffffffu, dt_mbar_wait(bar_d + ds * 8, dph, abort_s) && dt_mbar_wait(bar_t + a * 8, aph, abort_s));
                if (!ok) break;
                dt_fence_after();
                constexpr int STEP = HALF % 32 == 0 ? 32 : HALF % 16 == 0 ? 16 : 8;
#pragma unroll
                for (int j = 0; j < KPS; j++) {
                    if (kt + j >= nk) break;
                    const float4 * dv = reinterpret_cast<const float4 *>(dsc + (ds * KPS + j) * 128 + hf * HALF);
                    const uint32_t at = tmem + lanes + (a * KPS + j) * PITCH + hf * HALF;
#pragma unroll
                    for (int c0 = 0; c0 < HALF; c0 += STEP) {
                        uint32_t v[STEP];
                        ft_ld<STEP>(at + c0, v);
                        dt_wait_ld();
#pragma unroll
                        for (int c = 0; c < STEP; c += 4) {
                            const float4 d = dv[(c0 + c) / 4];
                            acc[c0 + c]     = fmaf(__uint_as_float(v[c]), w[j] * d.x, acc[c0 + c]);
                            acc[c0 + c + 1] = fmaf(__uint_as_float(v[c + 1]), w[j] * d.y, acc[c0 + c + 1]);
                            acc[c0 + c + 2] = fmaf(__uint_as_float(v[c + 2]), w[j] * d.z, acc[c0 + c + 2]);
                            acc[c0 + c + 3] = fmaf(__uint_as_float(v[c + 3]), w[j] * d.w, acc[c0 + c + 3]);
                        }
                    }
                }
                dt_fence_before();
                __syncwarp();
                if (lane == 0) { dt_arrive(bar_r + a * 8); dt_arrive(bar_g + ds * 8); }
                if (++a == ACCS) { a = 0; aph ^= 1; }
                if (++ds == FT_DRING) { ds = 0; dph ^= 1; }
            }
            if (!ok) break;
            if (S == 1) {
                if (in && n < A.N)
#pragma unroll
                    for (int c = 0; c < HALF; c++) if (m0 + c < A.b) A.y[(int64_t) (m0 + c) * A.N + n] = acc[c];
            } else {
                // a share's sums, [token][row]: its MMAs have completed, the ring is free (one tile per cluster)
                float * part = reinterpret_cast<float *>(sm);
#pragma unroll
                for (int c = 0; c < HALF; c++) part[(hf * HALF + c) * FT_BM + q4 * 32 + lane] = acc[c];
            }
        }
    }
    __syncwarp();
    if (S > 1) {
        dt_cluster_sync();
        if (warp >= 2 && warp < 10 && !*abort_s) {
            const int q4 = warp & 3, hf = (warp - 2) >> 2;
            const int64_t n = (int64_t) (r0 + q4) * 32 + lane;
            for (int c = share * 2 + hf; c < NB && c < A.b; c += S * 2) {
                float v = 0.f;
                for (int sh = 0; sh < S; sh++) {
                    float o;
                    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(o) : "r"(dt_mapa(sm0 + (uint32_t) (c * FT_BM + q4 * 32 + lane) * 4, (uint32_t) sh)) : "memory");
                    v += o;
                }
                if (q4 < runs && n < A.N) A.y[(int64_t) c * A.N + n] = v;
            }
        }
    }
    dt_fence_before();
    __syncthreads();
    if (*abort_s) {
        // a wait ran out: say so, give copies and MMAs still in flight time to land (bounded), then free the tensor memory
        if (threadIdx.x == 0) atomicExch(A.err, 1 + (int) blockIdx.x);
        for (int i = 0; i < 2000; i++) __nanosleep(1000);
        __syncthreads();
    }
    if (S > 1) dt_cluster_sync();                                // the shares' sums have been read
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

// ---- host side --------------------------------------------------------------------------------------------------------------------
static int ft_map(CUtensorMap * map, const void * base, int dims, const cuuint64_t * size, const cuuint64_t * stride, const cuuint32_t * box) {
    dt_encode_fn enc = pib_tma_encoder();
    if (!enc) { pib_set_error("tensor map: cuTensorMapEncodeTiled not available"); return PIB_ERR_UNSUPP; }
    const cuuint32_t es[4] = { 1, 1, 1, 1 };
    const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, (cuuint32_t) dims, const_cast<void *>(base), size, stride, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                           CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) { pib_set_error("tensor map: cuTensorMapEncodeTiled failed (%d)", (int) r); return PIB_ERR_UNSUPP; }
    return PIB_OK;
}
int pib_f8_map(CUtensorMap * map, const void * base, int64_t rows, int box) {
    const cuuint64_t size[2] = { 128, (cuuint64_t) rows }, stride[1] = { 128 };
    const cuuint32_t bx[2] = { 128, (cuuint32_t) box };
    return ft_map(map, base, 2, size, stride, bx);
}
int pib_f8_map3(CUtensorMap * map, const void * base, int64_t rows, int64_t groups, int64_t group_bytes, int box_rows, int box_groups) {
    const cuuint64_t size[3] = { 128, (cuuint64_t) rows, (cuuint64_t) groups }, stride[2] = { 128, (cuuint64_t) group_bytes };
    const cuuint32_t bx[3] = { 128, (cuuint32_t) box_rows, (cuuint32_t) box_groups };
    return ft_map(map, base, 3, size, stride, bx);
}
int pib_f8_map4(CUtensorMap * map, const void * base, int64_t KB, int64_t NB, int box_rows, int box_kb) {
    const cuuint64_t size[4] = { 128, 128, (cuuint64_t) KB, (cuuint64_t) NB }, stride[3] = { 128, 128 * 128, (cuuint64_t) KB * 128 * 128 };
    const cuuint32_t bx[4] = { 128, (cuuint32_t) box_rows, (cuuint32_t) box_kb, 1 };
    return ft_map(map, base, 4, size, stride, bx);
}

template <int NB> static int ft_launch(const pib_f8_runs & wmaps, const CUtensorMap & xmap, ft_args A, cudaStream_t st) {
    static pib_per_device attrs;
    PIB_CHECK(attrs.once([&] { return cudaFuncSetAttribute(f8_gemm_kernel<NB>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int) FT_SMEM); }));
    const int units = A.shares > 1 ? (A.runs + 3) / 4 : std::min((A.runs + ft_grain(NB) - 1) / ft_grain(NB), pib_num_sms());
    PIB_CHECK(pib_launch_cluster(f8_gemm_kernel<NB>, dim3((unsigned) (units * A.shares)), dim3(FT_THREADS), dim3((unsigned) A.shares, 1, 1), FT_SMEM, st, wmaps, xmap, A));
    return PIB_OK;
}

int pib_f8_gemm(const pib_weight * w, const void * act, int b, float * y, cudaStream_t st) {
    int rc = pib_f8_rows_ok("pib_gemm", w, act, y, b, PIB_F8_MAX_ROWS);
    if (rc != PIB_OK) return rc;
    if ((uintptr_t) act & 15) { pib_set_error("pib_gemm: act_dev needs 16-byte alignment"); return PIB_ERR_ARG; }
    const pib_f8_act L = pib_f8_act_of(w->K, b);
    int * err = pib_tc_error_word(st);
    if (!err) { pib_set_error("pib_gemm: no memory for the error word"); return PIB_ERR_NOMEM; }
    if (b > 128) return pib_f8_gemm_pair(w, act, b, y, err, st);
    const int NB = b <= 16 ? 16 : b <= 32 ? 32 : b <= 48 ? 48 : b <= 64 ? 64 : b <= 96 ? 96 : 128;
    ft_args A;
    A.b = b; A.KB = L.KB; A.bp = L.bp; A.N = w->N; A.y = y;
    A.ws = (const float *) w->d; A.ad = (const float *) ((const uint8_t *) act + L.d_off);
    A.runs = (int) ((w->N + 31) / 32);
    const int tiles = (A.runs + 3) / 4;
    A.shares = 1;
    while (A.shares < 8 && tiles * A.shares * 2 <= pib_num_sms() && A.KB >= A.shares * 4) A.shares *= 2;
    A.err = err;
    const pib_f8_runs & wmaps = ((const pib_f8_maps *) w->map)->runs;
    CUtensorMap xmap;
    if ((rc = pib_f8_map3(&xmap, act, b, L.KB, (int64_t) b * PIB_F8_BLOCK, NB, FT_KPS)) != PIB_OK) return rc;
    switch (NB) {
        case 16:  return ft_launch<16>(wmaps, xmap, A, st);
        case 32:  return ft_launch<32>(wmaps, xmap, A, st);
        case 48:  return ft_launch<48>(wmaps, xmap, A, st);
        case 64:  return ft_launch<64>(wmaps, xmap, A, st);
        case 96:  return ft_launch<96>(wmaps, xmap, A, st);
        default:  return ft_launch<128>(wmaps, xmap, A, st);
    }
}
