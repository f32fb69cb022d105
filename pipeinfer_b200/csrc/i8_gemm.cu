// i8_gemm.cu -- 8-bit integer weights with a scale for each output times up to 128 tokens (i8_gemm_pair.cu beyond) on tcgen05 (kind::i8), 32-bit integer accumulators.
//
//   y[t][n] = fp32(sum over k of q[n][k] a[t][k]) * fp32(d[t] s[n])
//
// A tile of up to 128 rows, all the tokens wide (NB: 16 .. 128, the smallest that holds them), is one accumulator in tensor memory over the whole of K; two of them take turns, so that a tile's
// outputs leave while the next one's products run.
//   warp 0       streams blocks of both operands by TMA (a row's 128 bytes are a line of the 128-byte swizzle) through a ring; the first stages' weights start ahead of the launch wait
//   warp 1       issues the MMAs; a commit hands the operands back, a tile's last one says that the accumulator is there
//   warps 2..9   two groups of four, half of the columns each: a thread owns a weight row (lane)
// The CTAs walk runs of 32 neighbouring rows, as many each as can be, in tiles of up to four.  Where the tiles leave most SMs idle, 2, 4 or 8 CTAs of a cluster take a share of the blocks
// each and add their sums up through distributed shared memory: whole numbers, any order.
// What bounds it: the weights' way from memory, at what one ring an SM asks for, and its start and end: 28672 x 8192 with 64 tokens 39 us (6.1 TB/s), 21999 x 5700 with 40 25.3
// (5.0 TB/s: 688 runs on 148 SMs are 4 or 5, and tiles begin inside row blocks; 18944 rows, four runs each, 5.5).  One accumulator over the whole of K is what whole numbers allow: there is nothing to add up between blocks.
// Every wait is bounded (tc_common.cuh).
#include "i8_block.cuh"
#include "tc_common.cuh"

#include <algorithm>

#define IT_THREADS 320
#define IT_BM      128
#define IT_A_TILE  (IT_BM * 128)
#define IT_RING    (192 * 1024)
#define IT_STAGES  10                       // at most
#define IT_KPS     2                        // blocks of a stage
#define IT_BARS    (2 * IT_STAGES + 4)
#define IT_SMEM    ((size_t) IT_RING + 512 + IT_BARS * 8 + 32 + 1024)

__device__ __forceinline__ void it_mma(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    // a block: four MMAs of K 32, 32 bytes further along both operands each
    asm volatile("{\n\t.reg .pred p, q;\n\t.reg .b64 a, b;\n\telect.sync _|q, 0xffffffff;\n\tsetp.ne.b32 p, %5, 0;\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, {%4, %4, %4, %4}, p;\n\t"
                 "add.s64 a, %1, 2;\n\tadd.s64 b, %2, 2;\n\t@q tcgen05.mma.cta_group::1.kind::i8 [%0], a, b, %3, {%4, %4, %4, %4}, 1;\n\t"
                 "add.s64 a, %1, 4;\n\tadd.s64 b, %2, 4;\n\t@q tcgen05.mma.cta_group::1.kind::i8 [%0], a, b, %3, {%4, %4, %4, %4}, 1;\n\t"
                 "add.s64 a, %1, 6;\n\tadd.s64 b, %2, 6;\n\t@q tcgen05.mma.cta_group::1.kind::i8 [%0], a, b, %3, {%4, %4, %4, %4}, 1;\n\t}"
                 ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(0u), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void it_tma_2d(uint32_t dst, const CUtensorMap * map, uint32_t bar, int x, int y) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void it_tma_4d(uint32_t dst, const CUtensorMap * map, uint32_t bar, int y, int z, int u) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst), "l"(map), "r"(bar), "r"(0), "r"(y), "r"(z), "r"(u) : "memory");
}
template <int N> __device__ __forceinline__ void it_ld(uint32_t at, uint32_t (&v)[N]) {
    if constexpr (N == 32) dt_ld32(at, v);
    else if constexpr (N == 16)
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                     : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]),
                       "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]) : "r"(at) : "memory");
    else
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]) : "r"(at) : "memory");
}
// M x N outputs of int8 x int8, 32-bit integer accumulators, both operands K-major
__host__ __device__ constexpr uint32_t it_idesc(int M, int N) { return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t) (N >> 3) << 17) | ((uint32_t) (M >> 4) << 24); }

struct it_args {
    int b, KB, runs, shares;                                     // runs: of 32 rows, in all
    int64_t N;
    const float * ws, * ad;
    float * y;
    int * err;
};

template <int NB>
__global__ void __launch_bounds__(IT_THREADS, 1)
i8_gemm_kernel(const __grid_constant__ pib_f8_runs wmaps, const __grid_constant__ CUtensorMap xmap, const __grid_constant__ it_args A) {
    constexpr int KPS = IT_KPS, STAGE = KPS * (IT_A_TILE + NB * 128), STAGES = IT_RING / STAGE < IT_STAGES ? IT_RING / STAGE : IT_STAGES, PITCH = NB <= 32 ? 32 : NB <= 64 ? 64 : 128, HALF = NB / 2;
    extern __shared__ __align__(1024) uint8_t it_dsm[];
    uint8_t *  sm  = it_dsm + ((1024u - (dt_smem(it_dsm) & 1023u)) & 1023u);
    float *    dsc = reinterpret_cast<float *>(sm + IT_RING);                            // the tokens' scales
    uint64_t * bar = reinterpret_cast<uint64_t *>(sm + IT_RING + 512);                   // operands there / read, accumulator there / read
    uint32_t * tmem_slot = reinterpret_cast<uint32_t *>(bar + IT_BARS);
    volatile int * abort_s = reinterpret_cast<volatile int *>(tmem_slot + 1);
    const uint32_t bar_f = dt_smem(bar), bar_e = bar_f + IT_STAGES * 8, bar_t = bar_e + IT_STAGES * 8, bar_r = bar_t + 16;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, S = A.shares, share = S > 1 ? (int) dt_cluster_rank() : 0;
    // the rows of a CTA (cluster) are neighbours, in runs of 32; its tiles take up to four runs each, as alike as can be
    const int unit = blockIdx.x / S, units = gridDim.x / S;
    const int r0 = (int) ((int64_t) A.runs * unit / units), runs = (int) ((int64_t) A.runs * (unit + 1) / units) - r0, tiles = (runs + 3) / 4, each = runs / tiles, more = runs % tiles;
    auto run_of  = [&](int tile) { return r0 + tile * each + min(tile, more); };         // a tile's first run, and how many
    auto runs_of = [&](int tile) { return each + (tile < more); };
    const int k0 = (int) ((int64_t) A.KB * share / S), nk = (int) ((int64_t) A.KB * (share + 1) / S) - k0, steps = (nk + KPS - 1) / KPS;
    const uint32_t sm0 = dt_smem(sm);

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; s++) { dt_mbar_init(bar_f + s * 8, 1); dt_mbar_init(bar_e + s * 8, 1); }
        for (int a = 0; a < 2; a++) { dt_mbar_init(bar_t + a * 8, 1); dt_mbar_init(bar_r + a * 8, 8); }
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
    bool ok = true;

    if (warp == 0) {
        if (lane == 0) {
            auto weights = [&](int s, int t0, int n, int kt) {
                // rows of the tile in one block of the weights' layout, and in the next
                const int      n1 = min(n, 4 - (t0 & 3)), n2 = n - n1, ks = n1 == 4 ? KPS : min(KPS, nk - kt);         // (what a share's last copies take of the next block is not used)
                const uint32_t to = sm0 + s * STAGE;
                dt_mbar_expect_tx(bar_f + s * 8, ks * n * 4096 + KPS * NB * 128);
                static_assert(KPS == 2, "a copy of whole blocks");
                if (n1 == 4) it_tma_2d(to, &wmaps.m[4], bar_f + s * 8, 0, (t0 / 4 * A.KB + k0 + kt) * 128);
                else for (int j = 0; j < ks; j++) {
                    it_tma_4d(to + j * IT_A_TILE, &wmaps.m[n1 - 1], bar_f + s * 8, t0 % 4 * 32, k0 + kt + j, t0 / 4);
                    if (n2) it_tma_4d(to + j * IT_A_TILE + n1 * 4096, &wmaps.m[n2 - 1], bar_f + s * 8, 0, k0 + kt + j, t0 / 4 + 1);
                }
            };
            auto tokens = [&](int s, int kt) { dt_tma_3d(sm0 + s * STAGE + KPS * IT_A_TILE, &xmap, bar_f + s * 8, 0, 0, k0 + kt); };
            // the weights of the first round are on their way while the launch in front still runs
            const int ahead = min(STAGES, tiles * steps);
            for (int i = 0; i < ahead; i++) { const int tile = i / steps; weights(i, run_of(tile), runs_of(tile), (i - tile * steps) * KPS); }
            pib_pdl_wait();
            for (int i = 0; i < ahead; i++) tokens(i, i % steps * KPS);
            int s = ahead % STAGES, i = 0;
            uint32_t ph = 0;
            for (int tile = 0; tile < tiles && ok; tile++) {
                const int t0 = run_of(tile), n = runs_of(tile);
                for (int kt = 0; kt < nk; kt += KPS, i++) {
                    if (i < ahead) continue;
                    ok = dt_mbar_wait(bar_e + s * 8, ph, abort_s);
                    if (!ok) break;
                    weights(s, t0, n, kt);
                    tokens(s, kt);
                    if (++s == STAGES) { s = 0; ph ^= 1; }
                }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        const uint64_t d0 = dt_desc(sm0);
        int s = 0, a = 0;
        uint32_t ph = 0, aph = 1;
        for (int tile = 0; tile < tiles && ok; tile++) {
            ok = __all_sync(0xffffffffu, dt_mbar_wait(bar_r + a * 8, aph, abort_s));
            for (int kt = 0; kt < nk && ok; kt += KPS) {
                ok = __all_sync(0xffffffffu, dt_mbar_wait(bar_f + s * 8, ph, abort_s));
                if (!ok) break;
                dt_fence_after();
#pragma unroll
                for (int j = 0; j < KPS; j++) {
                    const uint64_t ad = d0 + (uint64_t) ((s * STAGE + j * IT_A_TILE) >> 4), bd = d0 + (uint64_t) ((s * STAGE + KPS * IT_A_TILE + j * NB * 128) >> 4);
                    if (kt + j < nk) it_mma(tmem + a * PITCH, ad, bd, it_idesc(IT_BM, NB), kt + j > 0);
                }
                dt_commit(bar_e + s * 8);
                if (++s == STAGES) { s = 0; ph ^= 1; }
            }
            if (!ok) break;
            dt_commit(bar_t + a * 8);
            if (++a == 2) { a = 0; aph ^= 1; }
        }
    } else {
        pib_pdl_wait();
        pib_pdl_trigger();
        for (int c = threadIdx.x - 64; c < NB; c += IT_THREADS - 64) dsc[c] = c < A.b ? A.ad[c] : 0.f;
        asm volatile("bar.sync 1, 256;" ::: "memory");
        const int q4 = warp & 3, hf = (warp - 2) >> 2;
        const uint32_t lanes = (uint32_t) (q4 * 32) << 16;
        int a = 0;
        uint32_t aph = 0;
        constexpr int STEP = HALF % 32 == 0 ? 32 : HALF % 16 == 0 ? 16 : 8;
        for (int tile = 0; tile < tiles && ok; tile++) {
            const bool    in = q4 < runs_of(tile);
            const int64_t n  = (int64_t) (run_of(tile) + q4) * 32 + lane;
            const float   ws = in && n < A.N ? __ldg(A.ws + n) : 0.f;
            ok = __all_sync(0xffffffffu, dt_mbar_wait(bar_t + a * 8, aph, abort_s));
            if (!ok) break;
            dt_fence_after();
            int * part = reinterpret_cast<int *>(sm);            // a share's sums, [token][row]: its MMAs have completed, the ring is free (one tile per cluster)
#pragma unroll
            for (int c0 = 0; c0 < HALF; c0 += STEP) {
                uint32_t v[STEP];
                it_ld<STEP>(tmem + lanes + a * PITCH + hf * HALF + c0, v);
                dt_wait_ld();
                if (c0 + STEP == HALF) {                         // all read: the accumulator goes back
                    dt_fence_before();
                    __syncwarp();
                    if (lane == 0) dt_arrive(bar_r + a * 8);
                }
                if (S > 1) {
#pragma unroll
                    for (int c = 0; c < STEP; c++) part[(hf * HALF + c0 + c) * IT_BM + q4 * 32 + lane] = (int) v[c];
                } else if (in && n < A.N) {
#pragma unroll
                    for (int c = 0; c < STEP; c++) {
                        const int t = hf * HALF + c0 + c;
                        if (t < A.b) A.y[(int64_t) t * A.N + n] = i8_out((int) v[c], dsc[t], ws);
                    }
                }
            }
            if (++a == 2) { a = 0; aph ^= 1; }
        }
    }
    __syncwarp();
    if (S > 1) {
        dt_cluster_sync();
        if (warp >= 2 && !*abort_s) {
            const int q4 = warp & 3, hf = (warp - 2) >> 2;
            const int64_t n = (int64_t) (r0 + q4) * 32 + lane;
            const float  ws = q4 < runs && n < A.N ? __ldg(A.ws + n) : 0.f;
            for (int c = share * 2 + hf; c < NB && c < A.b; c += S * 2) {
                int v = 0;
                for (int sh = 0; sh < S; sh++) {
                    int o;
                    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(o) : "r"(dt_mapa(sm0 + (uint32_t) (c * IT_BM + q4 * 32 + lane) * 4, (uint32_t) sh)) : "memory");
                    v += o;
                }
                if (q4 < runs && n < A.N) A.y[(int64_t) c * A.N + n] = i8_out(v, dsc[c], ws);
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
template <int NB> static int it_launch(const pib_f8_runs & wmaps, const CUtensorMap & xmap, it_args A, cudaStream_t st) {
    static pib_per_device attrs;
    PIB_CHECK(attrs.once([&] { return cudaFuncSetAttribute(i8_gemm_kernel<NB>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int) IT_SMEM); }));
    const int units = A.shares > 1 ? (A.runs + 3) / 4 : std::min(A.runs, pib_num_sms());
    PIB_CHECK(pib_launch_cluster(i8_gemm_kernel<NB>, dim3((unsigned) (units * A.shares)), dim3(IT_THREADS), dim3((unsigned) A.shares, 1, 1), IT_SMEM, st, wmaps, xmap, A));
    return PIB_OK;
}

int pib_i8_gemm(const pib_weight * w, const void * act, int b, float * y, cudaStream_t st) {
    int rc = pib_f8_rows_ok("pib_gemm", w, act, y, b, PIB_I8_MAX_ROWS);
    if (rc != PIB_OK) return rc;
    if ((uintptr_t) act & 15) { pib_set_error("pib_gemm: act_dev needs 16-byte alignment"); return PIB_ERR_ARG; }
    const pib_i8_act L = pib_i8_act_of(w->K, b);
    int * err = pib_tc_error_word(st);
    if (!err) { pib_set_error("pib_gemm: no memory for the error word"); return PIB_ERR_NOMEM; }
    // pairs of SMs or this kernel, us at 96 and 128 tokens: 2560 x 2048 11.5 and 11.9 / 8.2 and 9.3, 4096 x 14336 39.5 and 40.1 / 16.6 and 18.0, 28672 x 8192 51.2 and 52.1 / 44.0 and 47.3.
    // Beyond 128 tokens this kernel would read the weights once for each 128: that is slower where the pairs have tiles for most SMs, and faster where they have not (4096 x 14336, 129 to 256 tokens: 38 on 16 of
    // 74 pairs, twice 15 here), of which the rule takes no notice
    if (b > 128) return pib_i8_gemm_pair(w, act, b, y, err, st);
    const int NB = b <= 16 ? 16 : b <= 32 ? 32 : b <= 48 ? 48 : b <= 64 ? 64 : b <= 96 ? 96 : 128;
    it_args A;
    A.b = b; A.KB = L.KB; A.N = w->N; A.y = y; A.err = err;
    A.ws = (const float *) w->d; A.ad = (const float *) ((const uint8_t *) act + L.d_off);
    A.runs = (int) ((w->N + 31) / 32);
    const int tiles = (A.runs + 3) / 4;
    A.shares = 1;
    // one / several shares, us at 16 tokens: 1024 x 2048 4.9 / 4.7, 2560 x 2048 5.5 / 4.8, 4096 x 14336 21.4 / 12.6
    while (A.shares < 8 && tiles * A.shares * 2 <= pib_num_sms() && A.KB >= A.shares * 4) A.shares *= 2;
    const pib_f8_runs & wmaps = ((const pib_f8_maps *) w->map)->runs;
    CUtensorMap xmap;
    if ((rc = pib_f8_map3(&xmap, act, b, L.KB, (int64_t) b * PIB_F8_BLOCK, NB, IT_KPS)) != PIB_OK) return rc;
    switch (NB) {
        case 16:  return it_launch<16>(wmaps, xmap, A, st);
        case 32:  return it_launch<32>(wmaps, xmap, A, st);
        case 48:  return it_launch<48>(wmaps, xmap, A, st);
        case 64:  return it_launch<64>(wmaps, xmap, A, st);
        case 96:  return it_launch<96>(wmaps, xmap, A, st);
        default:  return it_launch<128>(wmaps, xmap, A, st);
    }
}
