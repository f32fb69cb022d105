// i8_gemv.cu -- 8-bit integer weights with a scale for each output times 1..8 tokens (decode and verification batches; i8_gemm.cu beyond).
//
// mma.m16n8k32 on int8 operands, rows of W as M, tokens as N; whole sums stay in 32-bit integer registers, both scales meet them once at a tile's end.  Which k a lane holds is free as long
// as both operands agree: lane t of a row takes 16 neighbouring bytes of 64, the operands of two MMAs.
//
// One CTA per SM walks a run of neighbouring tiles of 16 rows.  A producer warp streams the rows by TMA, a stage being 16 blocks of 128 columns of the tile (one copy of 16 pieces of 2 KB,
// 128-byte swizzle), through a ring that runs on across tiles and starts ahead of the launch wait.  Of the 16 consumer warps warp w takes block w of a stage, and they meet in shared memory at the
// tile's end.  The activations lie in shared memory for the whole launch, rounded there by every CTA itself in the fused form (IG_PRO >= 0: the largest magnitude of each token first, then the
// values; what a thread read first stays in its registers between) or copied (IG_RES); where they do not fit beside the ring they come with the weights of each stage (IG_RING).
// What bounds it: the weights' way from memory, and for small matrices the start: 57344 x 8192 with four tokens 81 us (5.8 TB/s of 6.56 that a copy reaches), 2560 x 2048 with one 3.9 on the device.
#include "i8_block.cuh"
#include "tc_common.cuh"

#include <algorithm>

#define IG_WARPS 16
#define IG_THREADS (IG_WARPS * 32 + 32)
#define IG_RES  -1
#define IG_RING -2
#define IG_STAGE (32 * 1024)
#define IG_SMEM  (225 * 1024)

__device__ __forceinline__ void ig_mma(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// the consumers meet; true in all of them if it is in one: they leave together or not at all
__device__ __forceinline__ bool ig_bar_or(bool v) {
    uint32_t any;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, 1, 512, p;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(any) : "r"((uint32_t) v) : "memory");
    return any != 0;
}
__device__ __forceinline__ void ig_bar() { asm volatile("bar.sync 1, 512;" ::: "memory"); }
// the row of a swizzled tile that MMA row (or column) g stands for: the rows of neighbouring g lie in different halves of the banks
__device__ __forceinline__ int ig_perm(int g) { return (g >> 1) | (g & 1) << 2; }

__device__ __forceinline__ void ig_tma_4d(uint32_t dst, const CUtensorMap * map, uint32_t bar, int y, int z, int u) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst), "l"(map), "r"(bar), "r"(0), "r"(y), "r"(z), "r"(u) : "memory");
}

struct ig_args {
    const float * ws; int64_t Kp; int KB, tiles, stages; int64_t N, K;
    const uint8_t * a; const float * ad;                                    // activations rounded before
    const float * x, * x2, * addend; float * sum_out; int64_t xs; float eps; int vec;
    int b; float * y; int * err;
};
// a value of the row that the prologue makes: 0 x, 1 rmsnorm(x + addend) * x2 (rs the row's 1 / rms), 2 silu(x) * x2
template <int PRO> __device__ __forceinline__ float ig_value(float v, float o, float add, float rs) {
    if (PRO == 1) return (v + add) * rs * o;
    if (PRO == 2) return v / (1.0f + expf(-v)) * o;
    return v;
}
// 16 values of token tk from k on
template <int PRO> __device__ __forceinline__ void ig_row16(const ig_args & A, int tk, int64_t k, float rs, float (&v)[16]) {
    const float * p = A.x + (int64_t) tk * A.xs + k, * q = PRO == 2 ? A.x2 + (int64_t) tk * A.xs + k : PRO == 1 ? A.x2 + k : nullptr, * r = PRO == 1 && A.addend ? A.addend + (int64_t) tk * A.K + k : nullptr;
    if (A.vec && k + 16 <= A.K) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float4 f = reinterpret_cast<const float4 *>(p)[j];
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f), d = o;
            if (PRO) o = reinterpret_cast<const float4 *>(q)[j];
            if (PRO == 1 && r) d = reinterpret_cast<const float4 *>(r)[j];
            v[4 * j] = ig_value<PRO>(f.x, o.x, d.x, rs); v[4 * j + 1] = ig_value<PRO>(f.y, o.y, d.y, rs);
            v[4 * j + 2] = ig_value<PRO>(f.z, o.z, d.z, rs); v[4 * j + 3] = ig_value<PRO>(f.w, o.w, d.w, rs);
        }
    } else
#pragma unroll
        for (int j = 0; j < 16; j++) v[j] = k + j < A.K ? ig_value<PRO>(p[j], PRO ? q[j] : 0.f, PRO == 1 && r ? r[j] : 0.f, rs) : 0.f;
}

template <int PRO>
__global__ void __launch_bounds__(IG_THREADS, 1) i8_gemv_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap amap, const __grid_constant__ ig_args A) {
    constexpr bool RING = PRO == IG_RING;
    constexpr int  STAGE = RING ? IG_STAGE + 16 * 1024 : IG_STAGE;
    extern __shared__ __align__(1024) uint8_t ig_dsm[];
    uint8_t * sm = ig_dsm + ((1024u - (dt_smem(ig_dsm) & 1023u)) & 1023u);
    __shared__ int      red[IG_WARPS][8][17];
    __shared__ float    part[IG_WARPS], rms[8], dsc[8];
    __shared__ uint32_t top[8];
    __shared__ uint64_t bars[2 * 14];
    __shared__ int      abort_w;
    volatile int * abort_s = &abort_w;
    const int      lane = threadIdx.x & 31, warp = threadIdx.x >> 5, stages = A.stages, steps = (A.KB + 15) / 16;
    const int      tile0 = (int) ((int64_t) A.tiles * blockIdx.x / gridDim.x), tile1 = (int) ((int64_t) A.tiles * (blockIdx.x + 1) / gridDim.x);
    const uint32_t bar_f = dt_smem(bars), bar_e = bar_f + 14 * 8, sm0 = dt_smem(sm);
    uint8_t *      acts = sm + stages * STAGE;                              // [KB][2][b][64]: lane (g, t) of block kb, half c takes 16 bytes of token g
    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; s++) { dt_mbar_init(bar_f + s * 8, 1); dt_mbar_init(bar_e + s * 8, IG_WARPS); }
        abort_w = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (threadIdx.x < 8) top[threadIdx.x] = 0;
    __syncthreads();
    if (warp == IG_WARPS) {
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
                    ig_tma_4d(sm0 + s * STAGE, &wmap, bar_f + s * 8, (tile & 7) * 16, st * 16, tile >> 3);
                    if (RING) dt_tma_3d(sm0 + s * STAGE + IG_STAGE, &amap, bar_f + s * 8, 0, 0, st * 16);
                    if (++s == stages) { s = 0; ph ^= 1; }
                }
            if (!waited) pib_pdl_wait();
        }
        __syncwarp();
    } else {
        pib_pdl_wait();
        pib_pdl_trigger();
        const int g = lane >> 2, t = lane & 3, gp = ig_perm(g);
        if (PRO == IG_RES) {
            for (int u = threadIdx.x; u < A.b * A.KB * 8; u += IG_WARPS * 32) {
                const int k = u & 7, row = u >> 3, kb = row / A.b, tk = row - kb * A.b;
                *reinterpret_cast<int4 *>(acts + ((kb * 2 + (k >> 2)) * A.b + tk) * 64 + (k & 3) * 16) = *reinterpret_cast<const int4 *>(A.a + (size_t) u * 16);
            }
        } else if (!RING) {
            if (PRO == 1)
                for (int tk = 0; tk < A.b; tk++) {
                    float s = 0.f;
                    for (int64_t k = threadIdx.x; k < A.K; k += IG_WARPS * 32) {
                        float v = A.x[(int64_t) tk * A.xs + k];
                        if (A.addend) v += A.addend[(int64_t) tk * A.K + k];
                        if (A.sum_out && blockIdx.x == 0) A.sum_out[(int64_t) tk * A.K + k] = v;
                        s = fmaf(v, v, s);
                    }
                    s = warp_sum(s);
                    if (lane == 0) part[warp] = s;
                    ig_bar();
                    s = 0.f;
                    for (int i = 0; i < IG_WARPS; i++) s += part[i];
                    if (threadIdx.x == 0) rms[tk] = 1.0f / sqrtf(s / (float) A.K + A.eps);
                    ig_bar();
                }
            // units of 16 values, neighbouring ones in neighbouring lanes: a warp's eight lanes of a block are of one token
            const int per = A.KB * 8, units = A.b * per;
            auto load = [&](int u, float (&v)[16]) { const int tk = u / per, k = (u - tk * per) * 16; ig_row16<PRO < 0 ? 0 : PRO>(A, tk, k, PRO == 1 ? rms[tk] : 1.f, v); };
            auto largest = [&](int u, const float (&v)[16]) {
                uint32_t m = 0;
#pragma unroll
                for (int j = 0; j < 16; j++) m = max(m, i8_bits(v[j]));
#pragma unroll
                for (int o = 1; o < 8; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
                if ((lane & 7) == 0 && u < units) atomicMax(&top[u / per], m);
            };
            float first[16];
#pragma unroll
            for (int j = 0; j < 16; j++) first[j] = 0.f;
            if ((int) threadIdx.x < units) load(threadIdx.x, first);
            largest(threadIdx.x, first);
            for (int u0 = IG_WARPS * 32 + warp * 32; u0 < units; u0 += IG_WARPS * 32) {
                float v[16];
#pragma unroll
                for (int j = 0; j < 16; j++) v[j] = 0.f;
                if (u0 + lane < units) load(u0 + lane, v);
                largest(u0 + lane, v);
            }
            ig_bar();
            auto store = [&](int u, const float (&v)[16]) {
                const int   tk = u / per, i = u - tk * per, kb = i >> 3, k = (i & 7) * 16;
                const float d = i8_scale(top[tk]);
                *reinterpret_cast<int4 *>(acts + ((size_t) (kb * 2 + (k >> 6)) * A.b + tk) * 64 + (k & 63)) =
                    make_int4((int) i8_pack4(v[0], v[1], v[2], v[3], d), (int) i8_pack4(v[4], v[5], v[6], v[7], d), (int) i8_pack4(v[8], v[9], v[10], v[11], d), (int) i8_pack4(v[12], v[13], v[14], v[15], d));
            };
            if ((int) threadIdx.x < units) store(threadIdx.x, first);
            for (int u = IG_WARPS * 32 + threadIdx.x; u < units; u += IG_WARPS * 32) { float v[16]; load(u, v); store(u, v); }
        }
        if ((int) threadIdx.x < A.b) dsc[threadIdx.x] = PRO < 0 ? A.ad[threadIdx.x] : i8_scale(top[threadIdx.x]);
        ig_bar();
        // columns of tokens that are not there repeat token 0; nothing reads their sums
        const int acol = (g < A.b ? g : 0) * 64 + t * 16;
        int s = 0;
        uint32_t ph = 0;
        bool ok = true;
        for (int tile = tile0; tile < tile1 && ok; tile++) {
            int c[2][4] = { { 0, 0, 0, 0 }, { 0, 0, 0, 0 } };              // two chains
            // the scale of the output that this thread writes, asked for ahead of the products
            const int64_t nw = (int64_t) tile * 16 + (threadIdx.x & 15);
            const float   ws = nw < A.N ? __ldg(A.ws + nw) : 0.f;
#pragma unroll 1
            for (int st = 0; st < steps; st++) {
                const int kb = st * 16 + warp;
                ok = __all_sync(0xffffffffu, dt_mbar_wait(bar_f + s * 8, ph, abort_s));
                if (!ok) break;
                if (kb < A.KB) {
                    const uint8_t * tw = sm + s * STAGE + warp * 2048 + gp * 128, * ta = sm + s * STAGE + IG_STAGE + warp * 1024 + gp * 128;
                    int4 wa[2][2], ba[2];
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const int at = ((h * 4 + t) ^ gp) * 16;
                        wa[0][h] = *reinterpret_cast<const int4 *>(tw + at);
                        wa[1][h] = *reinterpret_cast<const int4 *>(tw + 1024 + at);
                        ba[h]    = RING ? *reinterpret_cast<const int4 *>(ta + at) : *reinterpret_cast<const int4 *>(acts + (size_t) (kb * 2 + h) * A.b * 64 + acol);
                    }
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        ig_mma(c[h], wa[0][h].x, wa[1][h].x, wa[0][h].y, wa[1][h].y, ba[h].x, ba[h].y);
                        ig_mma(c[h], wa[0][h].z, wa[1][h].z, wa[0][h].w, wa[1][h].w, ba[h].z, ba[h].w);
                    }
                }
                __syncwarp();
                if (lane == 0) dt_arrive(bar_e + s * 8);
                if (++s == stages) { s = 0; ph ^= 1; }
            }
#pragma unroll
            for (int j = 0; j < 4; j++) red[warp][RING ? ig_perm(t * 2 + (j & 1)) : t * 2 + (j & 1)][gp + (j >> 1) * 8] = c[0][j] + c[1][j];
            if (ig_bar_or(*abort_s)) break;
            if ((int) threadIdx.x < A.b * 16) {
                const int tk = threadIdx.x >> 4;
                int v = 0;
#pragma unroll
                for (int i = 0; i < IG_WARPS; i++) v += red[i][tk][threadIdx.x & 15];
                if (nw < A.N) A.y[(int64_t) tk * A.N + nw] = i8_out(v, dsc[tk], ws);
            }
            ig_bar();                                            // the sums have been read
        }
    }
    __syncthreads();
    if (*abort_s) {                                              // a wait ran out: say so, give copies still in flight time to land (bounded)
        if (threadIdx.x == 0) atomicExch(A.err, 1 + (int) blockIdx.x);
        for (int i = 0; i < 2000; i++) __nanosleep(1000);
    }
}

// shared memory: the ring, and beside it the activations where they are resident
static int ig_of(ig_args & A, const pib_weight * w, int b, float * y, cudaStream_t st) {
    memset(&A, 0, sizeof(A));
    A.KB = (int) pib_f8_blocks(w->K);
    A.Kp = (int64_t) A.KB * PIB_F8_BLOCK;
    A.tiles = (int) ((w->N + 15) / 16);
    A.ws = (const float *) w->d; A.N = w->N; A.K = w->K; A.b = b; A.y = y;
    if (!(A.err = pib_tc_error_word(st))) { pib_set_error("pib_gemv: no memory for the error word"); return PIB_ERR_NOMEM; }
    return PIB_OK;
}
template <int PRO> static int ig_launch(const CUtensorMap & wmap, const CUtensorMap & amap, ig_args A, cudaStream_t st) {
    const size_t stage = PRO == IG_RING ? IG_STAGE + 16 * 1024 : IG_STAGE, fixed = IG_WARPS * 8 * 17 * 4 + 1024 + 1024, res = PRO == IG_RING ? 0 : (size_t) A.b * A.Kp;
    A.stages = (int) ((IG_SMEM - fixed - res) / stage);
    static pib_per_device attrs;
    PIB_CHECK(attrs.once([&] { return cudaFuncSetAttribute(i8_gemv_kernel<PRO>, cudaFuncAttributeMaxDynamicSharedMemorySize, IG_SMEM - (int) fixed + 1024); }));
    PIB_CHECK(pib_launch(i8_gemv_kernel<PRO>, dim3((unsigned) std::min(A.tiles, pib_num_sms())), dim3(IG_THREADS), A.stages * stage + res + 1024, st, wmap, amap, A));
    return PIB_OK;
}

int pib_i8_gemv(const pib_weight * w, const void * act, int b, float * y, cudaStream_t st) {
    int rc = pib_f8_rows_ok("pib_gemv", w, act, y, b, PIB_MAX_BATCH);
    if (rc != PIB_OK) return rc;
    if ((uintptr_t) act & 15) { pib_set_error("pib_gemv: act_dev needs 16-byte alignment"); return PIB_ERR_ARG; }
    const pib_i8_act L = pib_i8_act_of(w->K, b);
    // here / in i8_gemm.cu, us at 8 tokens: 2560 x 2048 3.9 / 4.5, 4096 x 14336 11.2 / 12.2, 10240 x 8192 15.1 / 15.8, 28672 x 8192 38.0 / 36.3; wider tiles than eight columns are that kernel's
    if (b > 8) return pib_i8_gemm(w, act, b, y, st);
    ig_args A;
    const CUtensorMap & wmap = ((const pib_f8_maps *) w->map)->stage;
    CUtensorMap amap;
    if ((rc = ig_of(A, w, b, y, st)) != PIB_OK) return rc;
    A.a = (const uint8_t *) act; A.ad = (const float *) (A.a + L.d_off);
    // resident activations leave room for three stages at least
    if ((size_t) b * A.Kp <= 104 * 1024) return ig_launch<IG_RES>(wmap, wmap, A, st);
    if ((rc = pib_f8_map3(&amap, act, b, A.KB, (int64_t) b * PIB_F8_BLOCK, 8, 16)) != PIB_OK) return rc;
    return ig_launch<IG_RING>(wmap, amap, A, st);
}

int pib_i8_gemv_fused(const pib_weight * w, int pro, const float * x, const float * x2, const float * addend, float * sum_out, int64_t xstride, float eps, int b, float * y, cudaStream_t st) {
    if (b < 1 || b > 8 || w->K > 8192) { pib_set_error("pib_gemv_fused: unsupported matrix / batch"); return PIB_ERR_UNSUPP; }
    int rc = pib_fused_rows_ok(w, pro, x, x2, addend, sum_out, xstride, b, y);
    if (rc != PIB_OK) return rc;
    ig_args A;
    const CUtensorMap & wmap = ((const pib_f8_maps *) w->map)->stage;
    if ((rc = ig_of(A, w, b, y, st)) != PIB_OK) return rc;
    A.x = x; A.x2 = pro ? x2 : nullptr; A.addend = pro == 1 ? addend : nullptr; A.sum_out = pro == 1 ? sum_out : nullptr;
    A.xs = xstride ? xstride : w->K; A.eps = eps;
    A.vec = w->K % 4 == 0 && A.xs % 4 == 0 && !(((uintptr_t) A.x | (uintptr_t) A.x2 | (uintptr_t) A.addend) & 15);
    switch (pro) {
        case 0:  return ig_launch<0>(wmap, wmap, A, st);
        case 1:  return ig_launch<1>(wmap, wmap, A, st);
        default: return ig_launch<2>(wmap, wmap, A, st);
    }
}
