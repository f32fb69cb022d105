// f8_gemv.cu -- 8-bit floating point weights with block scales times 1..16 tokens (decode and verification batches).
//
//   y[t][n] = sum over kb of d[kb][t] s[n/128][kb] (sum over k of the block of q[n][k] a[t][k])
//
// mma.m16n8k32 on e4m3 operands, rows of W as M, tokens as N; a block's 128 products per output are summed by the tensor core (fp32), scaled and added up in fp32 registers.  Which k a
// lane holds is free as long as both operands agree: lane t of a row takes 16 neighbouring bytes of 64, the operands of two MMAs, so both matrices are read as they lie, 16 bytes a load.
// The eight warps of a CTA take every eighth block of its rows and meet in shared memory, in warp order.
#include "f8_block.cuh"

#define FG_WARPS 8
#define FG_ACT  -1

__device__ __forceinline__ void fg_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

struct fg_args {
    const uint8_t * w; const float * ws; int64_t Kp; int KB; int64_t N, K;
    const uint8_t * a; const float * ad; int bp;                            // activations quantised before
    const float * x, * x2, * addend; float * sum_out; int64_t xs; float eps; int vec;
    int b; float * y;
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

template <int NT, int MT, int PRO>
__global__ void __launch_bounds__(FG_WARPS * 32) f8_gemv_kernel(const __grid_constant__ fg_args A) {
    __shared__ float red[FG_WARPS][NT * 8][MT * 16 + 1];
    __shared__ float rms[8], part[FG_WARPS];
    const int  lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int64_t n0 = (int64_t) blockIdx.x * (MT * 16);
    const uint8_t * wp = A.w + (n0 + g) * A.Kp + t * 16;
    const float *   ws = A.ws + n0 / PIB_F8_BLOCK * A.KB;
    pib_pdl_wait();
    pib_pdl_trigger();
    float rs = 1.f;
    if (PRO == 1) {
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
            __syncthreads();
            if (threadIdx.x == 0) {
                s = 0.f;
                for (int i = 0; i < FG_WARPS; i++) s += part[i];
                rms[tk] = 1.0f / sqrtf(s / (float) A.K + A.eps);
            }
            __syncthreads();
        }
        rs = rms[g < A.b ? g : 0];
    }
    float acc[NT][MT][4];
#pragma unroll
    for (int i = 0; i < NT; i++)
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int j = 0; j < 4; j++) acc[i][m][j] = 0.f;
#pragma unroll 2
    for (int kb = warp; kb < A.KB; kb += FG_WARPS) {
        int4 wa[MT][2][2], ba[NT][2];
        float2 s[NT];
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int c = 0; c < 2; c++) wa[m][h][c] = ld_stream_v4(wp + (int64_t) (m * 16 + h * 8) * A.Kp + kb * PIB_F8_BLOCK + c * 64);
        const float w = __ldg(ws + kb);
        if (PRO == FG_ACT) {
#pragma unroll
            for (int i = 0; i < NT; i++) {
                const int tk = i * 8 + g, tc = i * 8 + t * 2;
#pragma unroll
                for (int c = 0; c < 2; c++)
                    ba[i][c] = tk < A.b ? *reinterpret_cast<const int4 *>(A.a + (int64_t) tk * A.Kp + kb * PIB_F8_BLOCK + c * 64 + t * 16) : make_int4(0, 0, 0, 0);
                s[i] = tc < A.b ? *reinterpret_cast<const float2 *>(A.ad + (int64_t) kb * A.bp + tc) : make_float2(0.f, 0.f);
            }
        } else {
            float v[2][16];
            float amax = 0.f;
#pragma unroll
            for (int c = 0; c < 2; c++) {
                if (g < A.b) fg_row16<PRO>(A, g, (int64_t) kb * PIB_F8_BLOCK + c * 64 + t * 16, rs, v[c]);
                else
#pragma unroll
                    for (int j = 0; j < 16; j++) v[c][j] = 0.f;
#pragma unroll
                for (int j = 0; j < 16; j++) amax = fmaxf(amax, fabsf(v[c][j]));
            }
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
            const float d = f8_scale(amax);
#pragma unroll
            for (int c = 0; c < 2; c++)
                ba[0][c] = make_int4((int) f8_pack4(v[c][0], v[c][1], v[c][2], v[c][3], d), (int) f8_pack4(v[c][4], v[c][5], v[c][6], v[c][7], d),
                                     (int) f8_pack4(v[c][8], v[c][9], v[c][10], v[c][11], d), (int) f8_pack4(v[c][12], v[c][13], v[c][14], v[c][15], d));
            s[0] = make_float2(__shfl_sync(0xffffffffu, d, t * 8), __shfl_sync(0xffffffffu, d, t * 8 + 4));
        }
#pragma unroll
        for (int i = 0; i < NT; i++)
#pragma unroll
            for (int m = 0; m < MT; m++) {
                float c[4] = { 0.f, 0.f, 0.f, 0.f };
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    fg_mma(c, wa[m][0][h].x, wa[m][1][h].x, wa[m][0][h].y, wa[m][1][h].y, ba[i][h].x, ba[i][h].y);
                    fg_mma(c, wa[m][0][h].z, wa[m][1][h].z, wa[m][0][h].w, wa[m][1][h].w, ba[i][h].z, ba[i][h].w);
                }
                const float s0 = w * s[i].x, s1 = w * s[i].y;
                acc[i][m][0] = fmaf(c[0], s0, acc[i][m][0]);
                acc[i][m][1] = fmaf(c[1], s1, acc[i][m][1]);
                acc[i][m][2] = fmaf(c[2], s0, acc[i][m][2]);
                acc[i][m][3] = fmaf(c[3], s1, acc[i][m][3]);
            }
    }
#pragma unroll
    for (int i = 0; i < NT; i++)
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int j = 0; j < 4; j++) red[warp][i * 8 + t * 2 + (j & 1)][m * 16 + g + (j >> 1) * 8] = acc[i][m][j];
    __syncthreads();
    for (int e = threadIdx.x; e < A.b * MT * 16; e += FG_WARPS * 32) {
        const int tk = e / (MT * 16), r = e % (MT * 16);
        float v = 0.f;
#pragma unroll
        for (int i = 0; i < FG_WARPS; i++) v += red[i][tk][r];
        if (n0 + r < A.N) A.y[(int64_t) tk * A.N + n0 + r] = v;
    }
}

static fg_args fg_of(const pib_weight * w, int b, float * y) {
    fg_args A;
    memset(&A, 0, sizeof(A));
    A.KB = (int) pib_f8_blocks(w->K);
    A.Kp = (int64_t) A.KB * PIB_F8_BLOCK;
    A.w = w->qs; A.ws = (const float *) w->d; A.N = w->N; A.K = w->K; A.b = b; A.y = y;
    return A;
}
template <int PRO> static int fg_launch(const fg_args & A, cudaStream_t st) {
    const bool two = A.N > 16LL * 4 * pib_num_sms();
    const dim3 grid((unsigned) ((A.N + (two ? 31 : 15)) / (two ? 32 : 16))), block(FG_WARPS * 32);
    if (PRO == FG_ACT && A.b > 8) {
        if (two) PIB_CHECK(pib_launch(f8_gemv_kernel<2, 2, FG_ACT>, grid, block, 0, st, A));
        else     PIB_CHECK(pib_launch(f8_gemv_kernel<2, 1, FG_ACT>, grid, block, 0, st, A));
    } else if (two) PIB_CHECK(pib_launch(f8_gemv_kernel<1, 2, PRO>, grid, block, 0, st, A));
    else            PIB_CHECK(pib_launch(f8_gemv_kernel<1, 1, PRO>, grid, block, 0, st, A));
    return PIB_OK;
}

int pib_f8_gemv(const pib_weight * w, const void * act, int b, float * y, cudaStream_t st) {
    const int ok = pib_f8_rows_ok("pib_gemv", w, act, y, b, PIB_MAX_BATCH);
    if (ok != PIB_OK) return ok;
    const pib_f8_act L = pib_f8_act_of(w->K, b);
    fg_args A = fg_of(w, b, y);
    A.a = (const uint8_t *) act; A.ad = (const float *) (A.a + L.d_off); A.bp = L.bp;
    return fg_launch<FG_ACT>(A, st);
}

int pib_f8_gemv_fused(const pib_weight * w, int pro, const float * x, const float * x2, const float * addend, float * sum_out, int64_t xstride, float eps, int b, float * y, cudaStream_t st) {
    if (b < 1 || b > 8 || w->K > 8192) { pib_set_error("pib_gemv_fused: unsupported matrix / batch"); return PIB_ERR_UNSUPP; }
    if (pro == 1 && sum_out && (sum_out == x || sum_out == addend)) { pib_set_error("pib_gemv_fused: sum_out_dev is an input that other blocks still read"); return PIB_ERR_ARG; }
    fg_args A = fg_of(w, b, y);
    A.x = x; A.x2 = pro ? x2 : nullptr; A.addend = pro == 1 ? addend : nullptr; A.sum_out = pro == 1 ? sum_out : nullptr;
    A.xs = xstride ? xstride : w->K; A.eps = eps;
    A.vec = w->K % 4 == 0 && A.xs % 4 == 0 && !(((uintptr_t) A.x | (uintptr_t) A.x2 | (uintptr_t) A.addend) & 15);
    switch (pro) {
        case 0:  return fg_launch<0>(A, st);
        case 1:  return fg_launch<1>(A, st);
        default: return fg_launch<2>(A, st);
    }
}
