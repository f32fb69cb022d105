// moe_few.cu -- a whole mixture layer for 1..16 tokens in two launches.
//
//   z = R x;  chosen: the `top` largest score + correction;  h_e = silu(G_e x) * U_e x;  y = residual + sum_e w_e D_e h_e   (shared experts: w = 1)
//
// moe_logits_kernel   a block per router output, all tokens; also clears the counters of the second launch
// moe_few_kernel      every block chooses the experts by itself (fewer steps than sharing the choice would take), then takes items by ticket: first the up items (expert, 16 gate rows and
//                     their 16 up rows), behind them the down items (expert, 32 output rows).  A down item waits for its expert's up items, which have lower tickets: whoever holds one is running
//                     and waits for nothing behind it, so the waits end however few blocks the GPU runs at a time.  The block that finishes the last expert of 32 output rows
//                     adds the experts up, in the order of the token's choices: no sum depends on which block came first.
//
// Products: mma.m16n8k16, expert rows as M, the expert's tokens as N.  Weights enter exactly: e4m3 as fp16 (times the block's scale in fp32 behind the block's sum), bfloat16 as it
// is.  The fp32 activations enter as parts: two fp16 (of the block's values times a power of two that brings the largest to 2^14 .. 2^15: 22 bits) with e4m3 weights, three bfloat16 (24
// bits) with bfloat16 ones; a line of 128 bytes of a weight row is summed by the tensor core and then added up in fp32.  Lane t of a row takes 16 neighbouring bytes of 64 (f8_gemv.cu).
#include <cuda_bf16.h>

#include "f8_block.cuh"
#include "hybrid.cuh"

#include <algorithm>

#define MF_WARPS 8
#define MF_SPIN  (1u << 22)

struct pib_moe {
    pib_moe_shape s;
    int   dev, KB1, KB2, T1, T2;         // lines of 128 bytes in a row of W1, W2; up and down items of an expert
    uint8_t * base;
    float * router, * corr;              // corr: null without a correction
    uint8_t * w1, * w2;                  // [experts + shared][T1][16 gate rows, 16 up rows][KB1 * 128 bytes], [..][T2 * 32 rows][KB2 * 128 bytes], zero behind the matrices
    float * s1, * s2;                    // F8: [..][gate, up][rows / 128][KB1], [..][rows / 128][KB2]
};
struct mf_args {
    int b, E, shared, top, score, renorm, has_corr, T1, T2, KB1, KB2, nb1, nb2, vec;
    float scale;
    int64_t D, F, Fk, Dr;
    const float * corr, * z;
    const uint8_t * w1, * w2;
    const float * s1, * s2;
    const float * x, * res; int64_t ldx, ldr, ldy;
    float * y, * h, * part;
    int * cnt, * err;                    // cnt: ticket, abort, up items done per active expert, experts done per 32 output rows
};
struct mf_layout { size_t z, h, part, total; int64_t Fk, Dr; int n_cnt; };
static mf_layout mf_of(const pib_moe * m, int b) {
    const int64_t P = (int64_t) b * (m->s.top + m->s.shared);
    auto al = [](size_t v) { return (v + 255) & ~(size_t) 255; };
    mf_layout L;
    L.Fk = (m->s.ff + 15) / 16 * 16; L.Dr = (int64_t) m->T2 * 32;
    L.n_cnt = 2 + m->s.experts + m->s.shared + m->T2;
    L.z = al((size_t) L.n_cnt * 4);
    L.h = L.z + al((size_t) b * m->s.experts * 4);
    L.part = L.h + al((size_t) (P * L.Fk) * 4);
    L.total = L.part + al((size_t) (P * L.Dr) * 4);
    return L;
}

// ---- router logits ------------------------------------------------------------------------------------------------------------------
template <int NT> __global__ void __launch_bounds__(256) moe_logits_kernel(const float * __restrict__ R, const float * __restrict__ x, int64_t ldx, int b, int E, int64_t D, int vec, float * __restrict__ z,
                                                                           int * __restrict__ cnt, int n_cnt) {
    __shared__ float red[8][NT];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float * r = R + (int64_t) blockIdx.x * D;
    pib_pdl_wait();
    pib_pdl_trigger();
    if (blockIdx.x == 0) for (int i = threadIdx.x; i < n_cnt; i += 256) cnt[i] = 0;
    float acc[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) acc[t] = 0.f;
    if (vec) {
        for (int64_t k = threadIdx.x * 4; k < D; k += 1024) {
            const float4 w = *reinterpret_cast<const float4 *>(r + k);
#pragma unroll
            for (int t = 0; t < NT; t++)
                if (t < b) {
                    const float4 v = *reinterpret_cast<const float4 *>(x + t * ldx + k);
                    acc[t] = fmaf(w.x, v.x, fmaf(w.y, v.y, fmaf(w.z, v.z, fmaf(w.w, v.w, acc[t]))));
                }
        }
    } else {
        for (int64_t k = threadIdx.x; k < D; k += 256) {
            const float w = r[k];
#pragma unroll
            for (int t = 0; t < NT; t++) if (t < b) acc[t] = fmaf(w, x[t * ldx + k], acc[t]);
        }
    }
#pragma unroll
    for (int t = 0; t < NT; t++) {
        acc[t] = warp_sum(acc[t]);
        if (lane == 0) red[warp][t] = acc[t];
    }
    __syncthreads();
    if (threadIdx.x < b) {
        float s = 0.f;
        for (int i = 0; i < 8; i++) s += red[i][threadIdx.x];
        z[threadIdx.x * E + blockIdx.x] = s;
    }
}

// ---- the layer ----------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void mf_mma_h(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mf_mma_b(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// two e4m3 as two fp16, exact
__device__ __forceinline__ uint32_t mf_half2(uint32_t q, int hi) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t) (hi ? q >> 16 : q), __NV_E4M3);
    return (uint32_t) h.x | (uint32_t) h.y << 16;
}
__device__ __forceinline__ uint32_t mf_pack_h(float a, float b) { const __half2 h = __floats2half2_rn(a, b); return *reinterpret_cast<const uint32_t *>(&h); }
__device__ __forceinline__ float2   mf_unpack_h(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2 *>(&u)); }
__device__ __forceinline__ uint32_t mf_pack_b(float a, float b) { const __nv_bfloat162 h = __floats2bfloat162_rn(a, b); return *reinterpret_cast<const uint32_t *>(&h); }
__device__ __forceinline__ float2   mf_unpack_b(uint32_t u) { return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u)); }

// N floats from p on, of which those behind `left` are zero; p is written by other blocks of this launch: cached in L2 only
template <int N> __device__ __forceinline__ void mf_row(const float * p, int64_t left, int vec, float (&v)[N]) {
    if (vec && left >= N) {
#pragma unroll
        for (int j = 0; j < N / 4; j++) {
            const float4 f = __ldcg(reinterpret_cast<const float4 *>(p) + j);
            v[4 * j] = f.x; v[4 * j + 1] = f.y; v[4 * j + 2] = f.z; v[4 * j + 3] = f.w;
        }
    } else
#pragma unroll
        for (int j = 0; j < N; j++) v[j] = j < left ? __ldcg(p + j) : 0.f;
}

// acc[column tile][half][..] = 32 rows of W (two tiles of 16; lines kb of this warp) times the columns' rows.  row: the lane's weight row (g) and 16 bytes (t) of it, Kp bytes a row;
// src: the lane's column's values or null, K of them; sa, sb: scales of the two tiles' blocks
template <bool F8, int NT>
__device__ __forceinline__ void mf_product(const uint8_t * __restrict__ row, int64_t Kp, int KB, int warp, int t, const float * const (&src)[NT], int64_t K, int vec, const float * __restrict__ sa,
                                           const float * __restrict__ sb, float (&acc)[NT][2][4]) {
    constexpr int LINE = F8 ? 128 : 64;                          // values of a line
#pragma unroll
    for (int i = 0; i < NT; i++)
#pragma unroll
        for (int m = 0; m < 2; m++)
#pragma unroll
            for (int j = 0; j < 4; j++) acc[i][m][j] = 0.f;
#pragma unroll 1
    for (int kb = warp; kb < KB; kb += MF_WARPS) {
        int4 w[2][2][2];
#pragma unroll
        for (int m = 0; m < 2; m++)
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int c = 0; c < 2; c++) w[m][h][c] = ld_stream_v4(row + (int64_t) (m * 16 + h * 8) * Kp + kb * 128 + c * 64);
        const float wa = F8 ? __ldg(sa + kb) : 1.f, wb = F8 ? __ldg(sb + kb) : 1.f;
#pragma unroll
        for (int i = 0; i < NT; i++) {
            float v[2][LINE / 8];
#pragma unroll
            for (int c = 0; c < 2; c++) {
                const int64_t k = (int64_t) kb * LINE + c * (LINE / 2) + t * (LINE / 8);
                mf_row(src[i] + k, src[i] ? K - k : 0, vec, v[c]);
            }
            float c[2][4];
#pragma unroll
            for (int m = 0; m < 2; m++)
#pragma unroll
                for (int j = 0; j < 4; j++) c[m][j] = 0.f;
            if (F8) {
                float amax = 0.f;
#pragma unroll
                for (int j = 0; j < 32; j++) amax = fmaxf(amax, fabsf(v[j / 16][j % 16]));
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
                const int   e  = min(253, 268 - (int) (__float_as_uint(amax) >> 23));
                const float up = __uint_as_float((uint32_t) e << 23), down = __uint_as_float((uint32_t) (254 - e) << 23);
#pragma unroll
                for (int q = 0; q < 8; q++) {                    // 16 values of k each
                    const float * p = &v[q / 4][q % 4 * 4];
                    const float p0 = p[0] * up, p1 = p[1] * up, p2 = p[2] * up, p3 = p[3] * up;
                    const uint32_t h0 = mf_pack_h(p0, p1), h1 = mf_pack_h(p2, p3);
                    const float2 f0 = mf_unpack_h(h0), f1 = mf_unpack_h(h1);
                    const uint32_t l0 = mf_pack_h(p0 - f0.x, p1 - f0.y), l1 = mf_pack_h(p2 - f1.x, p3 - f1.y);
#pragma unroll
                    for (int m = 0; m < 2; m++) {
                        const uint32_t r0 = (uint32_t) (&w[m][0][q / 4].x)[q % 4], r1 = (uint32_t) (&w[m][1][q / 4].x)[q % 4];
                        const uint32_t a0 = mf_half2(r0, 0), a1 = mf_half2(r1, 0), a2 = mf_half2(r0, 1), a3 = mf_half2(r1, 1);
                        mf_mma_h(c[m], a0, a1, a2, a3, h0, h1);
                        mf_mma_h(c[m], a0, a1, a2, a3, l0, l1);
                    }
                }
                const float d0 = __shfl_sync(0xffffffffu, down, t * 8), d1 = __shfl_sync(0xffffffffu, down, t * 8 + 4);
#pragma unroll
                for (int m = 0; m < 2; m++) {
                    const float s0 = (m ? wb : wa) * d0, s1 = (m ? wb : wa) * d1;
                    acc[i][m][0] = fmaf(c[m][0], s0, acc[i][m][0]);
                    acc[i][m][1] = fmaf(c[m][1], s1, acc[i][m][1]);
                    acc[i][m][2] = fmaf(c[m][2], s0, acc[i][m][2]);
                    acc[i][m][3] = fmaf(c[m][3], s1, acc[i][m][3]);
                }
            } else {
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    float p[4];
#pragma unroll
                    for (int j = 0; j < 4; j++) p[j] = v[q / 2][q % 2 * 4 + j];
#pragma unroll
                    for (int part = 0; part < 3; part++) {
                        const uint32_t b0 = mf_pack_b(p[0], p[1]), b1 = mf_pack_b(p[2], p[3]);
                        const float2 f0 = mf_unpack_b(b0), f1 = mf_unpack_b(b1);
                        p[0] -= f0.x; p[1] -= f0.y; p[2] -= f1.x; p[3] -= f1.y;
#pragma unroll
                        for (int m = 0; m < 2; m++) {
                            const uint32_t * r0 = reinterpret_cast<const uint32_t *>(&w[m][0][q / 2]) + q % 2 * 2, * r1 = reinterpret_cast<const uint32_t *>(&w[m][1][q / 2]) + q % 2 * 2;
                            mf_mma_b(c[m], r0[0], r1[0], r0[1], r1[1], b0, b1);
                        }
                    }
                }
#pragma unroll
                for (int m = 0; m < 2; m++)
#pragma unroll
                    for (int j = 0; j < 4; j++) acc[i][m][j] += c[m][j];
            }
        }
    }
}

struct mf_shared {
    float    wts[16][16];
    int      ids[16][16], at[16][16];     // chosen experts of a token; its row of h and of the experts' outputs
    uint32_t mask[PIB_MOE_MAX_EXPERTS + 16];
    int      slot[PIB_MOE_MAX_EXPERTS + 16], act[256], base[257], n_act, ticket, next, last;
    float    red[MF_WARPS][16][33];       // also the choice values of a warp's token
};
static_assert(sizeof(((mf_shared *) 0)->red) >= MF_WARPS * PIB_MOE_MAX_EXPERTS * 4, "choice values");

// the choice, by every block for itself
__device__ __forceinline__ void mf_route(const mf_args & A, mf_shared & S, int warp, int lane) {
    const int E = A.E;
    float * cv = &S.red[0][0][0] + warp * PIB_MOE_MAX_EXPERTS;
    for (int tk = warp; tk < A.b; tk += MF_WARPS) {
        const float * z = A.z + tk * E;
        float mx = -INFINITY, sum = 0.f;
        for (int i = lane; i < E; i += 32) mx = fmaxf(mx, z[i]);
        mx = warp_max(mx);
        for (int i = lane; i < E; i += 32) { const float s = A.score == PIB_MOE_SIGMOID ? 1.0f / (1.0f + expf(-z[i])) : expf(z[i] - mx); cv[i] = s; sum += s; }
        sum = warp_sum(sum);
        // softmax without a correction is chosen by the logits themselves: no two of them become equal on the way
        const bool by_z = !A.has_corr;
        for (int i = lane; i < E; i += 32) cv[i] = by_z ? z[i] : (A.score == PIB_MOE_SIGMOID ? cv[i] : cv[i] / sum) + A.corr[i];
        float tot = 0.f, mine = 0.f;
        int   id = 0;
        for (int k = 0; k < A.top; k++) {
            float bv = -INFINITY;
            int   bi = 0x7fffffff;
            for (int i = lane; i < E; i += 32) { const float v = cv[i]; if (v > bv || (v == bv && v > -INFINITY && i < bi)) { bv = v; bi = i; } }      // a lane reads back only what it wrote
            for (int o = 16; o > 0; o >>= 1) {
                const float ov = __shfl_xor_sync(0xffffffffu, bv, o);
                const int   oi = __shfl_xor_sync(0xffffffffu, bi, o);
                if (ov > bv || (ov == bv && oi < bi)) { bv = ov; bi = oi; }
            }
            if (bi >= E) {                                       // nothing comparable is left (logits that are no numbers): the first output that is not chosen yet
                for (bi = 0; __any_sync(0xffffffffu, lane < k && id == bi); bi++) {}
            }
            if ((bi & 31) == lane) cv[bi] = -INFINITY;
            const float s = A.score == PIB_MOE_SIGMOID ? 1.0f / (1.0f + expf(-z[bi])) : expf(z[bi] - mx) / sum;
            if (lane == k) { id = bi; mine = s; }
            tot += s;
        }
        if (lane < A.top) { S.ids[tk][lane] = id; S.wts[tk][lane] = A.scale * (A.renorm ? mine / (tot + 1e-20f) : mine); }
        else if (lane < A.top + A.shared) { S.ids[tk][lane] = E + lane - A.top; S.wts[tk][lane] = 1.f; }
    }
    const int all = E + A.shared, per = A.top + A.shared;
    for (int i = threadIdx.x; i < all; i += MF_WARPS * 32) S.mask[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < A.b * per; i += MF_WARPS * 32) atomicOr(&S.mask[S.ids[i / per][i % per]], 1u << i / per);
    __syncthreads();
    if (warp == 0) {                                             // the experts with tokens, in order; the first row of each one's tokens
        int n = 0, rows = 0;
        for (int i0 = 0; i0 < all; i0 += 32) {
            const uint32_t m = i0 + lane < all ? S.mask[i0 + lane] : 0;
            const unsigned has = __ballot_sync(0xffffffffu, m != 0), before = has & ((1u << lane) - 1);
            int r = __popc(m), s = r;
            for (int o = 1; o < 32; o <<= 1) { const int p = __shfl_up_sync(0xffffffffu, s, o); if (lane >= o) s += p; }
            if (m) { const int a = n + __popc(before); S.act[a] = i0 + lane; S.base[a] = rows + s - r; S.slot[i0 + lane] = a; }
            n += __popc(has);
            rows += __shfl_sync(0xffffffffu, s, 31);
        }
        if (lane == 0) S.n_act = n;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < A.b * per; i += MF_WARPS * 32) {
        const int tk = i / per, e = S.ids[tk][i % per];
        S.at[tk][i % per] = S.base[S.slot[e]] + __popc(S.mask[e] & ((1u << tk) - 1));
    }
    __syncthreads();
}

__device__ __forceinline__ int mf_nth_bit(uint32_t m, int n) {
    for (; n > 0; n--) m &= m - 1;
    return __ffs((int) m) - 1;
}

template <bool F8, int NT>
__device__ __forceinline__ void mf_item(const mf_args & A, mf_shared & S, bool up, int a, int i, int warp, int lane) {
    const int g = lane >> 2, t = lane & 3, e = S.act[a], base = S.base[a];
    const uint32_t mask = S.mask[e];
    const int n = __popc(mask);
    const float * src[NT];
#pragma unroll
    for (int j = 0; j < NT; j++) {
        const int c = j * 8 + g;
        src[j] = c >= n ? nullptr : up ? A.x + mf_nth_bit(mask, c) * A.ldx : A.h + (int64_t) (base + c) * A.Fk;
    }
    float acc[NT][2][4];
    if (up) {
        const float * s = A.s1 + ((int64_t) e * 2 * A.nb1 + i / 8) * A.KB1;
        mf_product<F8, NT>(A.w1 + (((int64_t) e * A.T1 + i) * 32 + g) * (A.KB1 * 128LL) + t * 16, A.KB1 * 128LL, A.KB1, warp, t, src, A.D, A.vec, s, s + (int64_t) A.nb1 * A.KB1, acc);
    } else {
        const float * s = A.s2 + ((int64_t) e * A.nb2 + i / 4) * A.KB2;
        mf_product<F8, NT>(A.w2 + (((int64_t) e * A.T2 + i) * 32 + g) * (A.KB2 * 128LL) + t * 16, A.KB2 * 128LL, A.KB2, warp, t, src, A.Fk, 1, s, s, acc);
    }
#pragma unroll
    for (int j = 0; j < NT; j++)
#pragma unroll
        for (int m = 0; m < 2; m++)
#pragma unroll
            for (int q = 0; q < 4; q++) S.red[warp][j * 8 + t * 2 + (q & 1)][m * 16 + g + (q >> 1) * 8] = acc[j][m][q];
    __syncthreads();
    if (up) {
        for (int q = threadIdx.x; q < n * 16; q += MF_WARPS * 32) {
            const int c = q >> 4, r = q & 15;
            float gt = 0.f, u = 0.f;
#pragma unroll
            for (int w = 0; w < MF_WARPS; w++) { gt += S.red[w][c][r]; u += S.red[w][c][16 + r]; }
            __stcg(A.h + (int64_t) (base + c) * A.Fk + i * 16 + r, gt / (1.0f + expf(-gt)) * u);
        }
    } else {
        for (int q = threadIdx.x; q < n * 32; q += MF_WARPS * 32) {
            const int c = q >> 5, r = q & 31;
            float v = 0.f;
#pragma unroll
            for (int w = 0; w < MF_WARPS; w++) v += S.red[w][c][r];
            __stcg(A.part + (int64_t) (base + c) * A.Dr + i * 32 + r, v);
        }
    }
}

template <bool F8>
__global__ void __launch_bounds__(MF_WARPS * 32, 2) moe_few_kernel(const __grid_constant__ mf_args A) {
    __shared__ mf_shared S;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    pib_pdl_wait();
    pib_pdl_trigger();
    if (threadIdx.x == 0) S.next = atomicAdd(A.cnt, 1);
    mf_route(A, S, warp, lane);
    const int per = A.top + A.shared, ups = S.n_act * A.T1, items = ups + S.n_act * A.T2;
    int * done_up = A.cnt + 2, * done_rows = done_up + A.E + A.shared;
    for (;;) {
        const int item = S.next;
        __syncthreads();
        if (item >= items) break;
        int next = 0;
        if (threadIdx.x == 0) next = atomicAdd(A.cnt, 1);
        const bool up = item < ups;
        const int  a = up ? item / A.T1 : (item - ups) / A.T2, i = up ? item % A.T1 : (item - ups) % A.T2;
        if (!up) {
            if (threadIdx.x == 0) {
                int ok = 0;
                for (uint32_t it = 0; it < MF_SPIN && !ok; it++) {
                    int v, stop;
                    asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(done_up + a) : "memory");
                    ok = v >= A.T1;
                    if (!ok && (it & 63) == 63) {
                        asm volatile("ld.relaxed.gpu.global.s32 %0, [%1];" : "=r"(stop) : "l"(A.cnt + 1) : "memory");
                        if (stop) break;
                    }
                }
                if (!ok) { atomicExch(A.cnt + 1, 1); atomicExch(A.err, 1 + (int) blockIdx.x); }
                S.last = ok;
            }
            __syncthreads();
            if (!S.last) break;                                  // a wait ran out: every block gives up at its own
        }
        if (__popc(S.mask[S.act[a]]) > 8) mf_item<F8, 2>(A, S, up, a, i, warp, lane);
        else                              mf_item<F8, 1>(A, S, up, a, i, warp, lane);
        __threadfence();
        __syncthreads();
        if (threadIdx.x == 0) {
            if (up) atomicAdd(done_up + a, 1);
            else    S.last = atomicAdd(done_rows + i, 1) == S.n_act - 1;
            S.next = next;
            __threadfence();
        }
        __syncthreads();
        if (!up && S.last) {
            for (int q = threadIdx.x; q < A.b * 32; q += MF_WARPS * 32) {
                const int tk = q >> 5;
                const int64_t row = i * 32 + (q & 31);
                if (row >= A.D) continue;
                float v = A.res ? A.res[tk * A.ldr + row] : 0.f;
                for (int k = 0; k < per; k++) v = fmaf(S.wts[tk][k], __ldcg(A.part + (int64_t) S.at[tk][k] * A.Dr + row), v);
                A.y[tk * A.ldy + row] = v;
            }
        }
    }
}

// ---- host side ----------------------------------------------------------------------------------------------------------------------
// rows of `bytes` bytes into rows of Kp, zero behind them; with `pairs` the source rows are tiles of 16 that land 32 apart (behind `off`)
static __global__ void mf_pack_kernel(const uint8_t * __restrict__ src, uint8_t * __restrict__ dst, int64_t rows, int64_t bytes, int64_t rows_p, int64_t Kp, int64_t dst_rows, int pairs, int off, int64_t n) {
    for (int64_t u = (int64_t) blockIdx.x * blockDim.x + threadIdx.x; u < n; u += (int64_t) gridDim.x * blockDim.x) {
        const int64_t k = u % (Kp / 16) * 16, r = u / (Kp / 16) % rows_p, e = u / (Kp / 16) / rows_p;
        __align__(16) uint8_t v[16];
        const uint8_t * p = src + (e * rows + r) * bytes + k;
#pragma unroll
        for (int j = 0; j < 16; j++) v[j] = r < rows && k + j < bytes ? p[j] : 0;
        *reinterpret_cast<int4 *>(dst + (e * dst_rows + (pairs ? r / 16 * 32 + off + r % 16 : r)) * Kp + k) = *reinterpret_cast<const int4 *>(v);
    }
}
static cudaError_t mf_pack(const void * src, uint8_t * dst, int64_t E, int64_t rows, int64_t bytes, int64_t rows_p, int64_t Kp, int64_t dst_rows, int pairs, int off) {
    const int64_t n = E * rows_p * (Kp / 16);
    mf_pack_kernel<<<(unsigned) std::min<int64_t>((n + 255) / 256, 1 << 16), 256>>>((const uint8_t *) src, dst, rows, bytes, rows_p, Kp, dst_rows, pairs, off, n);
    return cudaGetLastError();
}

extern "C" pib_moe * pib_moe_from_device(const pib_moe_shape * sh, const float * router, const float * correction, const void * gate, const float * gate_scales, const void * up,
                                         const float * up_scales, const void * down, const float * down_scales) {
    const bool f8 = sh && sh->type == PIB_TYPE_F8;
    if (!sh || !router || !gate || !up || !down || (!f8 && sh->type != PIB_TYPE_BF16) || (f8 && (!gate_scales || !up_scales || !down_scales)) || sh->experts < 1 || sh->experts > PIB_MOE_MAX_EXPERTS ||
        sh->top < 1 || sh->top > sh->experts || sh->shared < 0 || sh->shared > PIB_MOE_MAX_TOP || sh->top + sh->shared > PIB_MOE_MAX_TOP || (sh->score != PIB_MOE_SOFTMAX && sh->score != PIB_MOE_SIGMOID) ||
        sh->width < 1 || sh->ff < 1 || sh->width > (1 << 20) || sh->ff > (1 << 20)) {
        pib_set_error("pib_moe_from_device: bad arguments");
        return nullptr;
    }
    const int64_t E = sh->experts + sh->shared, D = sh->width, F = sh->ff;
    const int     eb = f8 ? 1 : 2;
    pib_moe * m = (pib_moe *) calloc(1, sizeof(pib_moe));
    if (!m) { pib_set_error("pib_moe_from_device: no host memory"); return nullptr; }
    m->s = *sh;
    m->KB1 = (int) ((D * eb + 127) / 128); m->KB2 = (int) ((F * eb + 127) / 128);
    m->T1 = (int) ((F + 15) / 16); m->T2 = (int) ((D + 31) / 32);
    auto al = [](size_t v) { return (v + 255) & ~(size_t) 255; };
    const size_t n_r = al((size_t) (sh->experts * D) * 4), n_c = al((size_t) sh->experts * 4), n_1 = (size_t) E * m->T1 * 32 * m->KB1 * 128, n_2 = (size_t) E * m->T2 * 32 * m->KB2 * 128;
    const size_t n_s1 = f8 ? al((size_t) (E * 2 * pib_f8_blocks(F) * m->KB1) * 4) : 0, n_s2 = f8 ? al((size_t) (E * pib_f8_blocks(D) * m->KB2) * 4) : 0;
    if (cudaGetDevice(&m->dev) != cudaSuccess || cudaMalloc(&m->base, n_r + n_c + n_1 + n_2 + n_s1 + n_s2) != cudaSuccess) {
        pib_set_error("pib_moe_from_device: cudaMalloc of %zu bytes failed", n_r + n_c + n_1 + n_2 + n_s1 + n_s2);
        cudaGetLastError();
        free(m);
        return nullptr;
    }
    m->router = (float *) m->base;
    m->corr = correction ? (float *) (m->base + n_r) : nullptr;
    m->w1 = m->base + n_r + n_c; m->w2 = m->w1 + n_1;
    m->s1 = (float *) (m->w2 + n_2); m->s2 = (float *) (m->w2 + n_2 + n_s1);
    cudaError_t e = cudaMemcpyAsync(m->router, router, (size_t) (sh->experts * D) * 4, cudaMemcpyDeviceToDevice, 0);
    if (e == cudaSuccess && correction) e = cudaMemcpyAsync(m->corr, correction, (size_t) sh->experts * 4, cudaMemcpyDeviceToDevice, 0);
    if (e == cudaSuccess) e = mf_pack(gate, m->w1, E, F, D * eb, m->T1 * 16LL, m->KB1 * 128LL, m->T1 * 32LL, 1, 0);
    if (e == cudaSuccess) e = mf_pack(up, m->w1, E, F, D * eb, m->T1 * 16LL, m->KB1 * 128LL, m->T1 * 32LL, 1, 16);
    if (e == cudaSuccess) e = mf_pack(down, m->w2, E, D, F * eb, m->T2 * 32LL, m->KB2 * 128LL, m->T2 * 32LL, 0, 0);
    if (f8) {
        const size_t row1 = (size_t) pib_f8_blocks(F) * m->KB1 * 4;                      // gate and up scales of an expert become neighbours
        if (e == cudaSuccess) e = cudaMemcpy2DAsync(m->s1, 2 * row1, gate_scales, row1, row1, (size_t) E, cudaMemcpyDeviceToDevice, 0);
        if (e == cudaSuccess) e = cudaMemcpy2DAsync((uint8_t *) m->s1 + row1, 2 * row1, up_scales, row1, row1, (size_t) E, cudaMemcpyDeviceToDevice, 0);
        if (e == cudaSuccess) e = cudaMemcpyAsync(m->s2, down_scales, (size_t) (E * pib_f8_blocks(D) * m->KB2) * 4, cudaMemcpyDeviceToDevice, 0);
    }
    if (e == cudaSuccess) e = cudaStreamSynchronize(0);
    if (e != cudaSuccess) {
        pib_set_error("pib_moe_from_device: %s", cudaGetErrorString(e));
        cudaGetLastError();
        pib_moe_free(m);
        return nullptr;
    }
    return m;
}

extern "C" void pib_moe_free(pib_moe * m) {
    if (!m) return;
    if (m->base) cudaFree(m->base);
    free(m);
}

extern "C" size_t pib_moe_scratch_bytes(const pib_moe * m, int b) { return m && b >= 1 && b <= PIB_MAX_BATCH ? mf_of(m, b).total : 0; }

extern "C" int pib_moe_forward(const pib_moe * m, const float * x, int64_t ldx, int b, const float * residual, int64_t ldr, float * y, int64_t ldy, void * scratch, pib_stream s) {
    if (!m || !x || !y || !scratch || b < 1 || b > PIB_MAX_BATCH || (const float *) y == x || ((uintptr_t) scratch & 255)) {
        pib_set_error("pib_moe_forward: bad arguments (b = %d, limit %d)", b, PIB_MAX_BATCH);
        return PIB_ERR_ARG;
    }
    const int64_t D = m->s.width;
    if (b > 1 && (ldx < D || ldy < D || (residual && ldr < D))) { pib_set_error("pib_moe_forward: rows overlap (ldx %lld, ldr %lld, ldy %lld, width %lld)", (long long) ldx, (long long) ldr, (long long) ldy, (long long) D); return PIB_ERR_ARG; }
    if (residual == y && ldr != ldy && b > 1) { pib_set_error("pib_moe_forward: y_dev is residual_dev with another distance of rows"); return PIB_ERR_ARG; }
    int dev = -1;
    PIB_CHECK(cudaGetDevice(&dev));
    if (dev != m->dev) { pib_set_error("pib_moe_forward: the layer is on device %d, the current device is %d", m->dev, dev); return PIB_ERR_ARG; }
    const cudaStream_t st = (cudaStream_t) s;
    const mf_layout L = mf_of(m, b);
    uint8_t * sc = (uint8_t *) scratch;
    mf_args A;
    memset(&A, 0, sizeof(A));
    A.b = b; A.E = m->s.experts; A.shared = m->s.shared; A.top = m->s.top; A.score = m->s.score; A.renorm = m->s.renorm; A.scale = m->s.scale; A.has_corr = m->corr != nullptr; A.corr = m->corr;
    A.T1 = m->T1; A.T2 = m->T2; A.KB1 = m->KB1; A.KB2 = m->KB2; A.nb1 = (int) pib_f8_blocks(m->s.ff); A.nb2 = (int) pib_f8_blocks(D);
    A.D = D; A.F = m->s.ff; A.Fk = L.Fk; A.Dr = L.Dr;
    A.vec = ldx % 4 == 0 && !((uintptr_t) x & 15);
    A.w1 = m->w1; A.w2 = m->w2; A.s1 = m->s1; A.s2 = m->s2;
    A.x = x; A.res = residual; A.ldx = ldx; A.ldr = ldr; A.ldy = ldy; A.y = y;
    A.cnt = (int *) sc; A.z = (const float *) (sc + L.z); A.h = (float *) (sc + L.h); A.part = (float *) (sc + L.part);
    if (!(A.err = pib_tc_error_word(st))) { pib_set_error("pib_moe_forward: no memory for the error word"); return PIB_ERR_NOMEM; }
    const dim3 rg((unsigned) A.E), rb(256);
    const int  rv = A.vec && D % 4 == 0;
    float *    z = (float *) (sc + L.z);
    if (b == 1)      PIB_CHECK(pib_launch(moe_logits_kernel<1>, rg, rb, 0, st, m->router, x, ldx, b, A.E, D, rv, z, A.cnt, L.n_cnt));
    else if (b <= 4) PIB_CHECK(pib_launch(moe_logits_kernel<4>, rg, rb, 0, st, m->router, x, ldx, b, A.E, D, rv, z, A.cnt, L.n_cnt));
    else             PIB_CHECK(pib_launch(moe_logits_kernel<16>, rg, rb, 0, st, m->router, x, ldx, b, A.E, D, rv, z, A.cnt, L.n_cnt));
    const dim3 grid((unsigned) (2 * pib_num_sms())), block(MF_WARPS * 32);
    if (m->s.type == PIB_TYPE_F8) PIB_CHECK(pib_launch(moe_few_kernel<true>, grid, block, 0, st, A));
    else                          PIB_CHECK(pib_launch(moe_few_kernel<false>, grid, block, 0, st, A));
    return PIB_OK;
}
