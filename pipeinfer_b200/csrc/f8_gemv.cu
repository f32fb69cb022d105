// f8_gemv.cu -- 8-bit floating point weights with block scales times 1..8 tokens (decode and verification batches; f8_gemm.cu beyond).
//
//   y[t][n] = sum over kb of d[kb][t] s[n/128][kb] (sum over k of the block of q[n][k] a[t][k])
//
// mma.m16n8k32 on e4m3 operands, rows of W as M, tokens as N; a block's 128 products per output are summed by the tensor core (fp32), scaled and added up in fp32 registers.  Which k a
// lane holds is free as long as both operands agree: lane t of a row takes 16 neighbouring bytes of 64, the operands of two MMAs.
//
// One CTA per SM walks a run of tiles of 16 rows (neighbouring ones: every gridDim-th tile instead takes 84.5 us for 57344 x 8192 and 4 tokens, runs 73.2, 0.99 of the copy rate).  A producer warp streams the rows by TMA, a stage being 16 blocks of the tile (one copy of 16 pieces of 2 KB, 128-byte swizzle), through a ring that
// runs on across tiles and starts ahead of the launch wait.  Of the 16 consumer warps warp w takes block w of a stage, and they meet in shared memory at the tile's end, in warp order.
// What bounds it: the weights' way from memory.  (Copies are few and large for the producer's sake: eight copies for 16 KB took 92 us for 57344 x 8192 without any products.)  The activations lie in shared memory for the whole launch, quantised there by every CTA itself in the fused form (FG_PRO >= 0) or copied
// (FG_RES); where they do not fit beside the ring they come with the weights of each stage (FG_RING).
#include "f8_block.cuh"
#include "tc_common.cuh"

#include <algorithm>

#define FG_WARPS 16
#define FG_THREADS (FG_WARPS * 32 + 32)
#define FG_RES  -1
#define FG_RING -2
#define FG_STAGE (32 * 1024)
#define FG_SMEM  (225 * 1024)

__device__ __forceinline__ void fg_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// the consumers meet; true in all of them if it is in one: they leave together or not at all
__device__ __forceinline__ bool fg_bar_or(bool v) {
    uint32_t any;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, 1, 512, p;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(any) : "r"((uint32_t) v) : "memory");
    return any != 0;
}
// the row of a swizzled tile that MMA row (or column) g stands for: the rows of neighbouring g lie in different halves of the banks
__device__ __forceinline__ int fg_perm(int g) { return (g >> 1) | (g & 1) << 2; }

__device__ __forceinline__ void fg_tma_3d(uint32_t dst, const CUtensorMap * map, uint32_t bar, int x, int y, int z) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z) : "memory");
}
__device__ __forceinline__ void fg_tma_4d(uint32_t dst, const CUtensorMap * map, uint32_t bar, int y, int z, int u) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst), "l"(map), "r"(bar), "r"(0), "r"(y), "r"(z), "r"(u) : "memory");
}

struct fg_args {
    const float * ws; int64_t Kp; int KB, tiles, stages; int64_t N, K;
    const uint8_t * a; const float * ad; int bp;                            // activations quantised before
    const float * x, * x2, * addend; float * sum_out; int64_t xs; float eps; int vec;
    int b; float * y; int * err;
};
// a value of the row that the prologue makes: 0 x, 1 rmsnorm(x + addend) * x2 (rs the row's 1 / rms), 2 silu(x) * x2
template <int PRO> __device__ __forceinline__ float fg_value(const fg_args & A, float v, float o, float add, float rs) {
    if (PRO == 1) return (v + add) * rs * o;
    if (PRO == 2) return v / (1.0f + expf(-v)) * o;
    return v;
}
// 16 values of token tk from k on
template <int PRO> __device__ __forceinline__ void fg_row16(const fg_args & A, int tk, int64_t k, float rs, float (&v)[16]) {
    const float * p = A.x + (int64_t) tk * A.xs + k, * q = PRO == 2 ? A.x2 + (int64_t) tk * A.xs + k : PRO == 1 ? A.x2 + k : nullptr, * r = PRO == 1 && A.addend ? A.addend + (int64_t) tk * A.K + k : nullptr;
    if (A.vec && k + 16 <= A.K) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float4 f = reinterpret_cast<const float4 *>(p)[j];
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f), d = o;
            if (PRO) o = reinterpret_cast<const float4 *>(q)[j];
            if (PRO == 1 && r) d = reinterpret_cast<const float4 *>(r)[j];
            v[4 * j] = fg_value<PRO>(A, f.x, o.x, d.x, rs); v[4 * j + 1] = fg_value<PRO>(A, f.y, o.y, d.y, rs);
            v[4 * j + 2] = fg_value<PRO>(A, f.z, o.z, d.z, rs); v[4 * j + 3] = fg_value<PRO>(A, f.w, o.w, d.w, rs);
        }
    } else
#pragma unroll
        for (int j = 0; j < 16; j++) v[j] = k + j < A.K ? fg_value<PRO>(A, p[j], PRO ? q[j] : 0.f, PRO == 1 && r ? r[j] : 0.f, rs) : 0.f;
}

template <int PRO>
__global__ void __launch_bounds__(FG_THREADS, 1) f8_gemv_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap amap, const __grid_constant__ fg_args A) {
    constexpr bool RING = PRO == FG_RING;
    constexpr int  STAGE = RING ? FG_STAGE + 16 * 1024 : FG_STAGE;
    extern __shared__ __align__(1024) uint8_t fg_dsm[];
    uint8_t * sm = fg_dsm + ((1024u - (dt_smem(fg_dsm) & 1023u)) & 1023u);
    __shared__ float    red[FG_WARPS][8][17];
    __shared__ float    part[FG_WARPS], rms[8];
    __shared__ uint64_t bars[2 * 14];
    __shared__ int      abort_w;
    volatile int * abort_s = &abort_w;
    const int      lane = threadIdx.x & 31, warp = threadIdx.x >> 5, stages = A.stages, steps = (A.KB + 15) / 16;
    const int      tile0 = (int) ((int64_t) A.tiles * blockIdx.x / gridDim.x), tile1 = (int) ((int64_t) A.tiles * (blockIdx.x + 1) / gridDim.x);
    const uint32_t bar_f = dt_smem(bars), bar_e = bar_f + 14 * 8, sm0 = dt_smem(sm);
    uint8_t *      acts = sm + stages * STAGE;                              // [KB][2][b][64]: lane (g, t) of block kb, half c takes 16 bytes of token g
    const int      sb = (A.b + 1) & ~1;
    float *        dsc  = reinterpret_cast<float *>(acts + (size_t) A.b * A.Kp);      // [KB][sb]
    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; s++) { dt_mbar_init(bar_f + s * 8, 1); dt_mbar_init(bar_e + s * 8, FG_WARPS); }
        abort_w = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    if (warp == FG_WARPS) {
        // producer: one lane; the weights do not wait for the launch before this one, the activations do
        if (lane == 0) {
            int s = 0;
            uint32_t ph = 1;
            bool waited = false, ok = true;
            for (int tile = tile0; tile < tile1 && ok; tile++)
                for (int st = 0; st < steps; st++) {
                    if (RING && !waited) { pib_pdl_wait(); waited = true; }
                    ok = dt_mbar_wait(bar_e + s * 8, ph, abort_s);
                    if (!ok) break;
                    // a tile's last copy finds zeros behind the last block
                    dt_mbar_expect_tx(bar_f + s * 8, STAGE);
                    fg_tma_4d(sm0 + s * STAGE, &wmap, bar_f + s * 8, (tile & 7) * 16, st * 16, tile >> 3);
                    if (RING) fg_tma_3d(sm0 + s * STAGE + FG_STAGE, &amap, bar_f + s * 8, 0, 0, st * 16);
                    if (++s == stages) { s = 0; ph ^= 1; }
                }
            if (!waited) pib_pdl_wait();
        }
        __syncwarp();
    } else {
        pib_pdl_wait();
        pib_pdl_trigger();
        const int g = lane >> 2, t = lane & 3, gp = fg_perm(g);
        if (PRO == FG_RES) {
            for (int u = threadIdx.x; u < A.b * A.KB * 8; u += FG_WARPS * 32) {
                const int k = u & 7, row = u >> 3, kb = row / A.b, tk = row - kb * A.b;
                *reinterpret_cast<int4 *>(acts + ((kb * 2 + (k >> 2)) * A.b + tk) * 64 + (k & 3) * 16) = *reinterpret_cast<const int4 *>(A.a + (size_t) u * 16);
            }
            for (int u = threadIdx.x; u < A.KB * sb; u += FG_WARPS * 32) dsc[u] = u % sb < A.b ? A.ad[(int64_t) (u / sb) * A.bp + u % sb] : 0.f;
        } else if (!RING) {
            if (PRO == 1)
                for (int tk = 0; tk < A.b; tk++) {
                    float s = 0.f;
                    for (int64_t k = threadIdx.x; k < A.K; k += FG_WARPS * 32) {
                        float v = A.x[(int64_t) tk * A.xs + k];
                        if (A.addend) v += A.addend[(int64_t) tk * A.K + k];
                        if (A.sum_out && blockIdx.x == 0) A.sum_out[(int64_t) tk * A.K + k] = v;
                        s = fmaf(v, v, s);
                    }
                    s = warp_sum(s);
                    if (lane == 0) part[warp] = s;
                    asm volatile("bar.sync 1, 512;" ::: "memory");
                    s = 0.f;
                    for (int i = 0; i < FG_WARPS; i++) s += part[i];
                    if (threadIdx.x == 0) rms[tk] = 1.0f / sqrtf(s / (float) A.K + A.eps);
                    asm volatile("bar.sync 1, 512;" ::: "memory");
                }
            // eight lanes per block of a token, 16 values each
            for (int u0 = warp * 4; u0 < A.b * A.KB; u0 += FG_WARPS * 4) {
                const int u = u0 + (lane >> 3), tk = u / A.KB, kb = u % A.KB, k = (lane & 7) * 16;
                const bool in = u < A.b * A.KB;
                float v[16], amax = 0.f;
                if (in) fg_row16<PRO < 0 ? 0 : PRO>(A, tk, (int64_t) kb * PIB_F8_BLOCK + k, PRO == 1 ? rms[tk] : 1.f, v);
                else
#pragma unroll
                    for (int j = 0; j < 16; j++) v[j] = 0.f;
#pragma unroll
                for (int j = 0; j < 16; j++) amax = fmaxf(amax, fabsf(v[j]));
#pragma unroll
                for (int o = 1; o < 8; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
                const float d = f8_scale(amax);
                if (in) {
                    *reinterpret_cast<int4 *>(acts + ((size_t) (kb * 2 + (k >> 6)) * A.b + tk) * 64 + (k & 63)) =
                        make_int4((int) f8_pack4(v[0], v[1], v[2], v[3], d), (int) f8_pack4(v[4], v[5], v[6], v[7], d), (int) f8_pack4(v[8], v[9], v[10], v[11], d), (int) f8_pack4(v[12], v[13], v[14], v[15], d));
                    if ((lane & 7) == 0) dsc[kb * sb + tk] = d;
                }
            }
        }
        if (!RING) asm volatile("bar.sync 1, 512;" ::: "memory");
        // columns of tokens that are not there repeat token 0; nothing reads their sums
        const int acol = (g < A.b ? g : 0) * 64 + t * 16;
        int tc[2];
#pragma unroll
        for (int j = 0; j < 2; j++) { const int tk = RING ? fg_perm(t * 2 + j) : t * 2 + j; tc[j] = tk < A.b ? tk : 0; }
        // scales are asked for ahead, a load's latency being longer than a stage's turn: those of the weights for 32 steps of a tile, one a lane; those of a token that are not resident a step
        auto scale32 = [&](int tile, int st0) { const int kb = (st0 + lane) * 16 + warp; return tile < tile1 && kb < A.KB ? __ldg(A.ws + (int64_t) (tile >> 3) * A.KB + kb) : 0.f; };
        auto token_scale = [&](int kb, int j) { return kb < A.KB ? __ldg(A.ad + (int64_t) kb * A.bp + tc[j]) : 0.f; };
        float w32 = scale32(tile0, 0), r0 = RING ? token_scale(warp, 0) : 0.f, r1 = RING ? token_scale(warp, 1) : 0.f;
        int s = 0;
        uint32_t ph = 0;
        bool ok = true;
        for (int tile = tile0; tile < tile1 && ok; tile++) {
            float acc[4] = { 0.f, 0.f, 0.f, 0.f };
            const float w32_next = steps > 32 ? 0.f : scale32(tile + 1, 0);
#pragma unroll 1
            for (int st = 0; st < steps; st++) {
                const int  kb = st * 16 + warp;
                const bool in = kb < A.KB;
                if (steps > 32 && (st & 31) == 0) w32 = scale32(tile, st);
                const float w = __shfl_sync(0xffffffffu, w32, st & 31), s0 = RING ? r0 : in ? dsc[kb * sb + tc[0]] : 0.f, s1 = RING ? r1 : in ? dsc[kb * sb + tc[1]] : 0.f;
                if (RING) { const int next = st + 1 < steps ? kb + 16 : warp; r0 = token_scale(next, 0); r1 = token_scale(next, 1); }
                ok = __all_sync(0xffffffffu, dt_mbar_wait(bar_f + s * 8, ph, abort_s));
                if (!ok) break;
                if (in) {
                    const uint8_t * tw = sm + s * STAGE + warp * 2048 + gp * 128, * ta = sm + s * STAGE + FG_STAGE + warp * 1024 + gp * 128;
                    int4 wa[2][2], ba[2];
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        const int at = ((c * 4 + t) ^ gp) * 16;
                        wa[0][c] = *reinterpret_cast<const int4 *>(tw + at);
                        wa[1][c] = *reinterpret_cast<const int4 *>(tw + 1024 + at);
                        ba[c]    = RING ? *reinterpret_cast<const int4 *>(ta + at) : *reinterpret_cast<const int4 *>(acts + (size_t) (kb * 2 + c) * A.b * 64 + acol);
                    }
                    float c[2][4] = { { 0.f, 0.f, 0.f, 0.f }, { 0.f, 0.f, 0.f, 0.f } };      // two short chains
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        fg_mma(c[h], wa[0][h].x, wa[1][h].x, wa[0][h].y, wa[1][h].y, ba[h].x, ba[h].y);
                        fg_mma(c[h], wa[0][h].z, wa[1][h].z, wa[0][h].w, wa[1][h].w, ba[h].z, ba[h].w);
                    }
#pragma unroll
                    for (int j = 0; j < 4; j++) acc[j] = fmaf(c[0][j] + c[1][j], w * (j & 1 ? s1 : s0), acc[j]);
                }
                __syncwarp();
                if (lane == 0) dt_arrive(bar_e + s * 8);
                if (++s == stages) { s = 0; ph ^= 1; }
            }
#pragma unroll
            for (int j = 0; j < 4; j++) red[warp][RING ? fg_perm(t * 2 + (j & 1)) : t * 2 + (j & 1)][gp + (j >> 1) * 8] = acc[j];
            if (fg_bar_or(*abort_s)) break;
            if (steps <= 32) w32 = w32_next;
            for (int e = threadIdx.x; e < A.b * 16; e += FG_WARPS * 32) {
                const int     tk = e >> 4;
                const int64_t n  = (int64_t) tile * 16 + (e & 15);
                float v = 0.f;
#pragma unroll
                for (int i = 0; i < FG_WARPS; i++) v += red[i][tk][e & 15];
                if (n < A.N) A.y[(int64_t) tk * A.N + n] = v;
            }
            asm volatile("bar.sync 1, 512;" ::: "memory");       // the sums have been read
        }
    }
    __syncthreads();
    if (*abort_s) {                                              // a wait ran out: say so, give copies still in flight time to land (bounded)
        if (threadIdx.x == 0) atomicExch(A.err, 1 + (int) blockIdx.x);
        for (int i = 0; i < 2000; i++) __nanosleep(1000);
    }
}

// shared memory: the ring, and beside it the activations and their scales where they are resident
static size_t fg_resident(int b, int64_t Kp) { return (size_t) b * Kp + (size_t) (Kp / PIB_F8_BLOCK) * ((b + 1) & ~1) * 4; }

static int fg_of(fg_args & A, const pib_weight * w, int b, float * y, cudaStream_t st) {
    memset(&A, 0, sizeof(A));
    A.KB = (int) pib_f8_blocks(w->K);
    A.Kp = (int64_t) A.KB * PIB_F8_BLOCK;
    A.tiles = (int) ((w->N + 15) / 16);
    A.ws = (const float *) w->d; A.N = w->N; A.K = w->K; A.b = b; A.y = y;
    if (!(A.err = pib_tc_error_word(st))) { pib_set_error("pib_gemv: no memory for the error word"); return PIB_ERR_NOMEM; }
    return PIB_OK;
}
template <int PRO> static int fg_launch(const CUtensorMap & wmap, const CUtensorMap & amap, fg_args A, cudaStream_t st) {
    const size_t stage = PRO == FG_RING ? FG_STAGE + 16 * 1024 : FG_STAGE, fixed = FG_WARPS * 8 * 17 * 4 + 512 + 1024, res = PRO == FG_RING ? 0 : fg_resident(A.b, A.Kp);
    A.stages = (int) ((FG_SMEM - fixed - res) / stage);
    static pib_per_device attrs;
    PIB_CHECK(attrs.once([&] { return cudaFuncSetAttribute(f8_gemv_kernel<PRO>, cudaFuncAttributeMaxDynamicSharedMemorySize, FG_SMEM - (int) fixed + 1024); }));
    PIB_CHECK(pib_launch(f8_gemv_kernel<PRO>, dim3((unsigned) std::min(A.tiles, pib_num_sms())), dim3(FG_THREADS), A.stages * stage + res + 1024, st, wmap, amap, A));
    return PIB_OK;
}

int pib_f8_gemv(const pib_weight * w, const void * act, int b, float * y, cudaStream_t st) {
    int rc = pib_f8_rows_ok("pib_gemv", w, act, y, b, PIB_MAX_BATCH);
    if (rc != PIB_OK) return rc;
    if ((uintptr_t) act & 15) { pib_set_error("pib_gemv: act_dev needs 16-byte alignment"); return PIB_ERR_ARG; }
    const pib_f8_act L = pib_f8_act_of(w->K, b);
    if (b > 8) return pib_f8_gemm(w, act, b, y, st);
    fg_args A;
    const CUtensorMap & wmap = ((const pib_f8_maps *) w->map)->stage;
    CUtensorMap amap;
    if ((rc = fg_of(A, w, b, y, st)) != PIB_OK) return rc;
    A.a = (const uint8_t *) act; A.ad = (const float *) (A.a + L.d_off); A.bp = L.bp;
    // resident activations leave room for three stages at least
    if (fg_resident(b, A.Kp) <= 104 * 1024) return fg_launch<FG_RES>(wmap, wmap, A, st);
    if ((rc = pib_f8_map3(&amap, act, b, A.KB, (int64_t) b * PIB_F8_BLOCK, 8, 16)) != PIB_OK) return rc;
    return fg_launch<FG_RING>(wmap, amap, A, st);
}

int pib_fused_rows_ok(const pib_weight * w, int pro, const float * x, const float * x2, const float * addend, const float * sum_out, int64_t xstride, int b, const float * y) {
    const int64_t xs = xstride ? xstride : w->K;
    if (xs < 0) { pib_set_error("pib_gemv_fused: bad arguments"); return PIB_ERR_ARG; }
    auto over = [&](const float * o, int64_t n, const float * in, int64_t stride) {            // n floats at o, rows of K at in
        for (int t = 0; t < b; t++) if (o && in && o < in + t * stride + w->K && in + t * stride < o + n) return true;
        return false;
    };
    const float * out[2] = { y, pro == 1 ? sum_out : nullptr };
    for (int i = 0; i < 2; i++) {
        const int64_t n = b * (i ? w->K : w->N);
        if (over(out[i], n, x, xs) || (pro && over(out[i], n, x2, pro == 2 ? xs : 0)) || (pro == 1 && over(out[i], n, addend, w->K))) {
            pib_set_error("pib_gemv_fused: an output lies over an input that other blocks still read");
            return PIB_ERR_ARG;
        }
    }
    if (((uintptr_t) x | (uintptr_t) x2 | (uintptr_t) addend | (uintptr_t) sum_out | (uintptr_t) y) & 3) { pib_set_error("pib_gemv_fused: fp32 rows need 4-byte alignment"); return PIB_ERR_ARG; }
    return PIB_OK;
}

int pib_f8_gemv_fused(const pib_weight * w, int pro, const float * x, const float * x2, const float * addend, float * sum_out, int64_t xstride, float eps, int b, float * y, cudaStream_t st) {
    if (b < 1 || b > 8 || w->K > 8192) { pib_set_error("pib_gemv_fused: unsupported matrix / batch"); return PIB_ERR_UNSUPP; }
    int rc = pib_fused_rows_ok(w, pro, x, x2, addend, sum_out, xstride, b, y);
    if (rc != PIB_OK) return rc;
    fg_args A;
    const CUtensorMap & wmap = ((const pib_f8_maps *) w->map)->stage;
    if ((rc = fg_of(A, w, b, y, st)) != PIB_OK) return rc;
    A.x = x; A.x2 = pro ? x2 : nullptr; A.addend = pro == 1 ? addend : nullptr; A.sum_out = pro == 1 ? sum_out : nullptr;
    A.xs = xstride ? xstride : w->K; A.eps = eps;
    A.vec = w->K % 4 == 0 && A.xs % 4 == 0 && !(((uintptr_t) A.x | (uintptr_t) A.x2 | (uintptr_t) A.addend) & 15);
    switch (pro) {
        case 0:  return fg_launch<0>(wmap, wmap, A, st);
        case 1:  return fg_launch<1>(wmap, wmap, A, st);
        default: return fg_launch<2>(wmap, wmap, A, st);
    }
}
