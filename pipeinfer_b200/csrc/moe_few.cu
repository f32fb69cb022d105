// moe_few.cu -- a whole mixture layer for 1..16 tokens in two launches.
//
//   z = R x;  chosen: the `top` largest score + correction;  h_e = silu(G_e x) * U_e x;  y = residual + sum_e w_e D_e h_e   (shared experts: w = 1)
//
// moe_logits_kernel   a block per router output, all tokens; one per token that splits its row into parts (below); also clears the counters of the second launch
// moe_few_kernel      every block chooses the experts by itself (fewer steps than sharing the choice would take), then takes items by ticket: first the up items (expert, 16 gate rows and
//                     their 16 up rows), behind them the down items (expert, 32 output rows).  A down item waits for its expert's up items, which have lower tickets: whoever holds one is running
//                     and waits for nothing behind it, so the waits end however few blocks the GPU runs at a time.  The block that finishes the last expert of 32 output rows
//                     adds the experts up, in the order of the token's choices: no sum depends on which block came first.
//
//   producer warp     takes the tickets and streams the items' rows in pieces of up to 24 KB (6 lines of 128 bytes of 32 rows, in one piece of memory) through a ring that runs on across
//                     items, a down item's weights ahead of its wait
//   six consumer warps take a line of a piece each and meet in shared memory at the item's end, in warp order
//   publisher warp    makes an item's results known to the other blocks and adds up finished rows: fences and atomics that the consumers would stand still for
//
// Products: mma.m16n8k16, expert rows as M, the expert's tokens as N.  Weights enter exactly: e4m3 as fp16 (times the block's scale in fp32 behind the sum), bfloat16 as it is.  The fp32
// activations enter as parts: with e4m3 weights two fp16 of the values times a power of two that brings the largest of them to 2^14 .. 2^15 (22 bits, down to 2^-39 of the largest), with bfloat16
// weights three bfloat16 (24 bits).  x has a power of two a row; h is split where it is made, 16 values of a row, so each such tile has its own: the k of one MMA, whose sum is scaled by it.
// (A bound of the row, which is there before the row is, in its place: where an expert's rows differ by a factor of 300 that left 2^-12 of the layer's output.)
// Half a line's sums (F8 with h: a tile's) are made by the tensor core, scaled and added up in fp32.  Four tokens' two parts (eight tokens' one of three) share the eight columns of one MMA; an
// expert with more tokens stands in the list of active ones once for each four (eight) of them, next to each other: its weights come from L2 again, which costs less than a second form of the
// kernel (registers).  Which k a lane holds is free as long as both operands agree: the weights' columns are permuted within a line when they are packed, so that 16 bytes of
// a row (lane t) are four values each of four (two) neighbouring tiles of 16, the k of an MMA, and the parts lie in that order too.
// What bounds it: at 16 tokens of 128 experts (4096 x 1536, 8 each) the weights, 1.56 GB in 322 us (0.75 of the copy rate; the choice takes some 8 us of it, a power of two for each tile of h 11, the
// turns of 48 KB down items the rest).  At one token (64 experts, 6 and 2 shared, 2048 x 1408: 30 us, the copies alone 11) latency: 6 us for the logits, 4 for the choice, then two rounds of items that are one
// way to memory and back each.  Sharing the choice among the blocks would save none of it: the launch's first 4 us are mostly the way of its code into the caches.
#include <cuda_bf16.h>

#include "f8_block.cuh"
#include "tc_common.cuh"

#include <algorithm>

#define MF_WARPS   6                          // consumers; with the producer and the publisher eight warps, and 128 registers a thread in two blocks per SM
#define MF_LT      4                          // tokens of a block of router outputs, where there are several
#define MF_THREADS (MF_WARPS * 32 + 64)
#define MF_SPIN    (1u << 22)
#define MF_LINE    4096                       // 128 bytes of 32 rows
#define MF_STAGE   (MF_WARPS * MF_LINE)
#define MF_STAGES  3
// the consumers meet; true in all of them if it is in one: they leave together or not at all
__device__ __forceinline__ bool mf_bar_or(bool v) {
    uint32_t any;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, 1, 192, p;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(any) : "r"((uint32_t) v) : "memory");
    return any != 0;
}

struct pib_moe {
    pib_moe_shape s;
    int   dev, KB1, KB2, T1, T2;         // lines of 128 bytes in a row of W1, W2; up and down items of an expert
    uint8_t * base;
    float * router, * corr;              // corr: null without a correction
    uint8_t * w1, * w2;                  // [experts + shared][T1][KB1][16 gate rows, 16 up rows][128 bytes], [..][T2][KB2][32 rows][128 bytes], zero behind the matrices; the 16-byte pieces of a row
                                         // lie at their number xor (row & 7): lanes of neighbouring rows read different banks
    float * s1, * s2;                    // F8: [..][gate, up][rows / 128][KB1], [..][rows / 128][KB2]
};
struct mf_args {
    int b, E, shared, top, score, renorm, has_corr, T1, T2, KB1, KB2, nb1, nb2;
    float scale;
    int64_t D, Dr;
    const float * corr, * z;
    const uint8_t * w1, * w2;
    const float * s1, * s2;
    const float * res; int64_t ldr, ldy;
    const uint16_t * xp; const float * xm;                   // parts of the tokens' rows, their largest |x|
    uint16_t * hp, * hx;                                     // parts of the pairs' rows of h; F8: the power of two that brings a tile of 16 back, its upper half
    float * y, * part;
    int * cnt, * err;                    // cnt: ticket, abort, up items done per entry of the list, entries done per 32 output rows
};
struct mf_layout { size_t z, xm, xp, hp, hx, part, total; int64_t Dr; int n_cnt; };
// a row's parts: [part][line][lane t][tile of the line][4] 16-bit numbers; 64 (F8) or 32 bytes per line, part and lane
__host__ __device__ static inline int64_t mf_row_of(bool f8, int KB) { return (int64_t) KB * (f8 ? 2 * 128 : 3 * 64); }
static mf_layout mf_of(const pib_moe * m, int b) {
    const int64_t P = (int64_t) b * (m->s.top + m->s.shared);
    const bool    f8 = m->s.type == PIB_TYPE_F8;
    auto al = [](size_t v) { return (v + 255) & ~(size_t) 255; };
    mf_layout L;
    L.Dr = (int64_t) m->T2 * 32;
    L.n_cnt = 2 + (int) P + m->T2;
    L.xm = al((size_t) L.n_cnt * 4);
    L.z = L.xm + al((size_t) b * 4);
    L.xp = L.z + al((size_t) b * m->s.experts * 4);
    L.hp = L.xp + al((size_t) (b * mf_row_of(f8, m->KB1)) * 2);
    L.hx = L.hp + al((size_t) (P * mf_row_of(f8, m->KB2)) * 2);
    L.part = L.hx + (f8 ? al((size_t) P * m->KB2 * 16) : 0);
    L.total = L.part + al((size_t) (P * L.Dr) * 4);
    return L;
}

__device__ __forceinline__ void mf_mma_h(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// two fp32 at a time
__device__ __forceinline__ uint64_t mf_pair(float lo, float hi) { return (uint64_t) __float_as_uint(hi) << 32 | __float_as_uint(lo); }
__device__ __forceinline__ uint64_t mf_mul2(uint64_t a, uint64_t b) { uint64_t d; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b)); return d; }
__device__ __forceinline__ uint64_t mf_fma2(uint64_t a, uint64_t b, uint64_t c) { uint64_t d; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c)); return d; }
// mf_mma_h without sums before it
__device__ __forceinline__ void mf_mma_h0(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mf_mma_b(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// two e4m3 as two fp16, exact
__device__ __forceinline__ uint32_t mf_half2(uint32_t q, int hi) {
    uint32_t h;
    asm volatile("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((unsigned short) (hi ? q >> 16 : q)));
    return h;
}
// the exponent field of the power of two that brings a number to 2^14 .. 2^15; 254 less it is the inverse's
__device__ __forceinline__ int mf_exponent(float v) { return min(253, 268 - (__float_as_int(v) >> 23 & 255)); }
__device__ __forceinline__ float mf_pow2(int field) { return __uint_as_float((uint32_t) field << 23); }
// parts of value v times `up` (F8), to place r of tile `tile` of a row
template <bool F8> __device__ __forceinline__ void mf_store(float v, float up, int tile, int r, int KB, uint16_t * row) {
    constexpr int Q = F8 ? 8 : 4;
    const int plane = KB * Q * 16, at = ((tile / Q * 4 + (r >> 2)) * Q + tile % Q) * 4 + (r & 3);
    if (F8) {
        const float  p  = v * up;
        const __half hi = __float2half_rn(p), lo = __float2half_rn(p - __half2float(hi));
        __stcg(row + at, __half_as_ushort(hi));
        __stcg(row + plane + at, __half_as_ushort(lo));
    } else {
#pragma unroll
        for (int part = 0; part < 3; part++) {
            const __nv_bfloat16 h = __float2bfloat16_rn(v);
            v -= __bfloat162float(h);
            __stcg(row + part * plane + at, __bfloat16_as_ushort(h));
        }
    }
}

// ---- router logits, parts of the tokens ---------------------------------------------------------------------------------------------
template <bool F8, int NT> __global__ void __launch_bounds__(256) moe_logits_kernel(const float * __restrict__ R, const float * __restrict__ x, int64_t ldx, int b, int E, int64_t D, int vec,
                                                                                    float * __restrict__ z, int * __restrict__ cnt, int n_cnt, int KB, uint16_t * __restrict__ xp, float * __restrict__ xm) {
    __shared__ float red[8][NT];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int out = blockIdx.x % E, t0 = blockIdx.x / E * NT, groups = (b + NT - 1) / NT;
    const bool split = (int) blockIdx.x >= groups * E;
    const float * r = R + (int64_t) out * D;
    if (!split) for (int64_t k = (int64_t) threadIdx.x * 32; k < D; k += 256 * 32) asm volatile("prefetch.global.L2 [%0];" ::"l"(r + k));     // the layer's own, ahead of the wait
    pib_pdl_wait();
    pib_pdl_trigger();
    if (blockIdx.x == 0) for (int i = threadIdx.x; i < n_cnt; i += 256) cnt[i] = 0;
    if (split) {
        const int t = blockIdx.x - groups * E;
        float up = 1.f;
        if (F8) {
            float m = 0.f;
            for (int64_t k = threadIdx.x; k < D; k += 256) m = fmaxf(m, fabsf(x[t * ldx + k]));
            m = warp_max(m);
            if (lane == 0) red[warp][0] = m;
            __syncthreads();
            for (int i = 0; i < 8; i++) m = fmaxf(m, red[i][0]);
            up = mf_pow2(mf_exponent(m));
            if (threadIdx.x == 0) xm[t] = m;
        }
        for (int u = threadIdx.x; u < KB * (F8 ? 128 : 64); u += 256) mf_store<F8>(u < D ? x[t * ldx + u] : 0.f, up, u >> 4, u & 15, KB, xp + t * mf_row_of(F8, KB));
        return;
    }
    // a token behind the last is the last one again: no branch between the loads (with one per token a row of 4096 took 12 us for 16 tokens)
    float acc[NT];
    const float * xt[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) { acc[t] = 0.f; xt[t] = x + min(t0 + t, b - 1) * ldx; }
    if (vec) {
        for (int64_t k = threadIdx.x * 4; k < D; k += 1024) {
            const float4 w = *reinterpret_cast<const float4 *>(r + k);
#pragma unroll
            for (int t = 0; t < NT; t++) {
                const float4 v = *reinterpret_cast<const float4 *>(xt[t] + k);
                acc[t] = fmaf(w.x, v.x, fmaf(w.y, v.y, fmaf(w.z, v.z, fmaf(w.w, v.w, acc[t]))));
            }
        }
    } else {
        for (int64_t k = threadIdx.x; k < D; k += 256) {
            const float w = r[k];
#pragma unroll
            for (int t = 0; t < NT; t++) acc[t] = fmaf(w, xt[t][k], acc[t]);
        }
    }
#pragma unroll
    for (int t = 0; t < NT; t++) {
        acc[t] = warp_sum(acc[t]);
        if (lane == 0) red[warp][t] = acc[t];
    }
    __syncthreads();
    if (threadIdx.x < NT && t0 + threadIdx.x < b) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 8; i++) s += red[i][threadIdx.x];
        z[(t0 + threadIdx.x) * E + out] = s;
    }
}

// ---- the layer ----------------------------------------------------------------------------------------------------------------------
struct mf_shared {
    float    wts[16][16];
    int      px[16];                      // the exponent field of a token's power of two
    int      ids[16][16], at[16][16];     // chosen experts of a token; its row of h and of the experts' outputs
    uint32_t mask[PIB_MOE_MAX_EXPERTS + 16], tokens[256];        // of an expert, of an entry of the list
    int      slot[PIB_MOE_MAX_EXPERTS + 16], act[256], base[256], n_act, item[MF_STAGES], pub[2], abort;
    uint64_t bars[2 * MF_STAGES + 4];     // a piece there / read, an item's results written / published
    float    red[2][MF_WARPS][9][33];     // two items' turns
};
static_assert(MF_STAGES * MF_STAGE >= MF_THREADS / 32 * PIB_MOE_MAX_EXPERTS * 4, "a token's logits for every warp");
#define MF_RING (((int) sizeof(mf_shared) + 127) & ~127)          // behind it the ring
#define MF_SMEM ((size_t) MF_RING + MF_STAGES * MF_STAGE)
extern __shared__ __align__(128) uint8_t mf_dsm[];               // named here, so that the compiler knows a shared address in every function

struct mf_place { int s; uint32_t ph; };       // a place of the ring and its phase

// order-preserving key of a choice value; what is no number comes last, a chosen one is 0
__device__ __forceinline__ uint32_t mf_key(float v) { const uint32_t u = __float_as_uint(v + 0.0f); return v != v ? 1u : u & 0x80000000u ? ~u : u | 0x80000000u; }

// the choice, by every block for itself
template <bool F8> __device__ __forceinline__ void mf_route(const mf_args & A, mf_shared & S, uint8_t * ring, int warp, int lane) {
    constexpr int COLS = F8 ? 4 : 8;                             // tokens of an entry of the list
    const int E = A.E;
    float * sv = reinterpret_cast<float *>(ring) + warp * PIB_MOE_MAX_EXPERTS;             // the token's logits
    for (int tk = warp; tk < A.b; tk += MF_THREADS / 32) {
        const float * z = A.z + tk * E;
        __syncwarp();                                            // the last token's logits have been read
        const float xmax = F8 ? __ldcg(A.xm + tk) : 0.f;
        float mx = -INFINITY, sum = 1.f;
        for (int i = lane; i < E; i += 32) { const float v = __ldcg(z + i); sv[i] = v; mx = fmaxf(mx, v); }
        if (A.score == PIB_MOE_SOFTMAX) {
            mx = warp_max(mx);
            sum = 0.f;
            for (int i = lane; i < E; i += 32) { const float v = expf(sv[i] - mx); sum += v; }
            sum = warp_sum(sum);
        }
        auto score = [&](float v) { return A.score == PIB_MOE_SIGMOID ? 1.0f / (1.0f + expf(-v)) : expf(v - mx) / sum; };
        // Without a correction chosen by the logits themselves: no two of them become equal on the way.  Keys of outputs lane + 32 j stay in registers, 0 once chosen; the
        // tests on E are the same in all lanes
        constexpr int PL = PIB_MOE_MAX_EXPERTS / 32;
        uint32_t key[PL], best = 0;
        int      at = 0x7fffffff;
#pragma unroll
        for (int j = 0; j < PL; j++) {
            key[j] = 0;
            if (j * 32 >= E) break;
            const int i = j * 32 + lane;
            if (i < E) key[j] = mf_key(A.has_corr ? score(sv[i]) + __ldg(A.corr + i) : sv[i]);
            if (key[j] > best) { best = key[j]; at = i; }
        }
        int id = 0;
        for (int k = 0; k < A.top; k++) {
            const uint32_t top = __reduce_max_sync(0xffffffffu, best);
            const int bi = __reduce_min_sync(0xffffffffu, best == top ? at : 0x7fffffff);
            if (lane == k) id = bi;
            const bool mine = at == bi;
            if (mine) { best = 0; at = 0x7fffffff; }
#pragma unroll
            for (int j = 0; j < PL; j++) {
                if (j * 32 >= E) break;
                const int i = j * 32 + lane;
                if (i == bi) key[j] = 0;
                if (mine && key[j] > best) { best = key[j]; at = i; }
            }
        }
        if (lane >= A.top) id = E + lane - A.top;
        __syncwarp();                                            // other lanes' logits, read below, are there
        const bool has = lane < A.top + A.shared;
        const float mine = lane < A.top ? score(sv[id]) : 0.f, tot = warp_sum(mine);
        if (has) {
            S.ids[tk][lane] = id;
            S.wts[tk][lane] = lane < A.top ? A.scale * (A.renorm ? mine / (tot + 1e-20f) : mine) : 1.f;
            if (F8 && lane == 0) S.px[tk] = mf_exponent(xmax);
        }
    }
    const int all = E + A.shared, per = A.top + A.shared;
    for (int i = threadIdx.x; i < all; i += MF_THREADS) S.mask[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < A.b * per; i += MF_THREADS) atomicOr(&S.mask[S.ids[i / per][i % per]], 1u << i / per);
    __syncthreads();
    if (warp == 0) {                                             // the experts with tokens, in order; the first row of each one's tokens
        int n = 0, rows = 0;
        for (int i0 = 0; i0 < all; i0 += 32) {
            const uint32_t m = i0 + lane < all ? S.mask[i0 + lane] : 0;
            const unsigned has = __ballot_sync(0xffffffffu, m != 0);
            if (!has) continue;
            const int r = __popc(m), k = (r + COLS - 1) / COLS;
            int s = r | k << 16;
            for (int o = 1; o < 32; o <<= 1) { const int p = __shfl_up_sync(0xffffffffu, s, o); if (lane >= o) s += p; }
            if (m) {
                int      a = n + (s >> 16) - k, row = rows + (s & 0xffff) - r;
                uint32_t left = m;
                S.slot[i0 + lane] = a;
                for (; left; a++) {
                    uint32_t few = 0;
                    for (int j = 0; j < COLS && left; j++) { few |= left & (0u - left); left &= left - 1; }
                    S.act[a] = i0 + lane; S.base[a] = row; S.tokens[a] = few;
                    row += __popc(few);
                }
            }
            s = __shfl_sync(0xffffffffu, s, 31);
            n += s >> 16;
            rows += s & 0xffff;
        }
        if (lane == 0) S.n_act = n;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < A.b * per; i += MF_THREADS) {
        const int tk = i / per, e = S.ids[tk][i % per];
        S.at[tk][i % per] = S.base[S.slot[e]] + __popc(S.mask[e] & ((1u << tk) - 1));
    }
}

__device__ __forceinline__ int mf_nth_bit(uint32_t m, int n) {
    for (; n > 0; n--) m &= m - 1;
    return __ffs((int) m) - 1;
}
__device__ __forceinline__ uint4 mf_ld(const uint16_t * p) { return __ldcg(reinterpret_cast<const uint4 *>(p)); }

// What a lane holds of a line's activations: the row of column g (F8: of token g & 3, part g >> 2), three parts of it with bfloat16
template <bool F8> struct mf_b {
    static constexpr int PARTS = F8 ? 1 : 3, WORDS = F8 ? 4 : 2;
    uint4 v[PARTS][WORDS];
};
template <bool F8> __device__ __forceinline__ void mf_ask(mf_b<F8> & B, const uint16_t * row, int plane, int kb, int t) {
    constexpr int P = mf_b<F8>::PARTS, W = mf_b<F8>::WORDS;
#pragma unroll
    for (int part = 0; part < P; part++)
#pragma unroll
        for (int w = 0; w < W; w++) B.v[part][w] = row ? mf_ld(row + part * plane + (kb * 4 + t) * (W * 8) + w * 8) : make_uint4(0, 0, 0, 0);
}
// Half c of a line of a piece times eight columns: acc[tile of 16 rows].  f: what a sum of the tile of rows is worth, per column that the lane holds; x: what the sums of four
// tiles of k are multiplied with besides (F8 with h), 16 bits each
template <bool F8, bool UP> __device__ __forceinline__ void mf_half(const uint8_t * line, int c, int lane, const mf_b<F8> & B, const float (&f)[2][2], const uint2 (&x)[2], uint64_t (&acc)[2][2]) {
    constexpr int P = mf_b<F8>::PARTS;
    const int g = lane >> 2, t = lane & 3, gp = (g >> 1) | (g & 1) << 2;
    int4  w[2][2];
    float s[2][4];
#pragma unroll
    for (int m = 0; m < 2; m++) {
#pragma unroll
        for (int h = 0; h < 2; h++) w[m][h] = *reinterpret_cast<const int4 *>(line + (m * 16 + h * 8 + gp) * 128 + ((c * 4 + t) ^ gp) * 16);
#pragma unroll
        for (int j = 0; j < 4; j++) s[m][j] = 0.f;
    }
    if (F8) {
#pragma unroll
        for (int q = 0; q < 4; q++) {                            // 16 values of k each
            const uint4    b = B.v[0][c * 2 + (q >> 1)];
            const uint32_t b0 = q & 1 ? b.z : b.x, b1 = q & 1 ? b.w : b.y;
            uint64_t d = 0;
            if (!UP) {
                const uint32_t x0 = q < 2 ? x[0].x : x[0].y, x1 = q < 2 ? x[1].x : x[1].y;
                d = mf_mul2(mf_pair(f[0][0], f[0][1]), mf_pair(__uint_as_float(q & 1 ? x0 & 0xffff0000u : x0 << 16), __uint_as_float(q & 1 ? x1 & 0xffff0000u : x1 << 16)));
            }
#pragma unroll
            for (int m = 0; m < 2; m++) {
                const uint32_t r0 = (uint32_t) (q == 0 ? w[m][0].x : q == 1 ? w[m][0].y : q == 2 ? w[m][0].z : w[m][0].w), r1 = (uint32_t) (q == 0 ? w[m][1].x : q == 1 ? w[m][1].y : q == 2 ? w[m][1].z : w[m][1].w);
                const uint32_t a0 = mf_half2(r0, 0), a1 = mf_half2(r1, 0), a2 = mf_half2(r0, 1), a3 = mf_half2(r1, 1);
                if (UP) mf_mma_h(s[m], a0, a1, a2, a3, b0, b1);
                else {
                    mf_mma_h0(s[m], a0, a1, a2, a3, b0, b1);
                    acc[m][0] = mf_fma2(mf_pair(s[m][0], s[m][1]), d, acc[m][0]);
                    acc[m][1] = mf_fma2(mf_pair(s[m][2], s[m][3]), d, acc[m][1]);
                }
            }
        }
        if (!UP) return;
    } else {
#pragma unroll
        for (int part = P - 1; part >= 0; part--) {              // the small ones first
            const uint4 b = B.v[part][c];
#pragma unroll
            for (int m = 0; m < 2; m++) {
                mf_mma_b(s[m], w[m][0].x, w[m][1].x, w[m][0].y, w[m][1].y, b.x, b.y);
                mf_mma_b(s[m], w[m][0].z, w[m][1].z, w[m][0].w, w[m][1].w, b.z, b.w);
            }
        }
    }
#pragma unroll
    for (int m = 0; m < 2; m++)
#pragma unroll
        for (int j = 0; j < 2; j++) acc[m][j] = mf_fma2(mf_pair(s[m][2 * j], s[m][2 * j + 1]), F8 ? mf_pair(f[m][0], f[m][1]) : mf_pair(1.f, 1.f), acc[m][j]);
}

// An item, by the consumers: the warp's lines of its pieces, the meeting, the results.  turn: the item's turn at the places of the sums.  False: the block gives up
template <bool F8, bool UP>
__device__ __forceinline__ bool mf_item(const mf_args & A, mf_shared & S, const uint8_t * ring, uint32_t bar_f, uint32_t bar_e, mf_place & at, int turn, int a, int i) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, e = S.act[a], base = S.base[a], KB = UP ? A.KB1 : A.KB2;
    const uint32_t mask = S.tokens[a];
    const int n = __popc(mask), stride = (int) mf_row_of(F8, KB), plane = KB * (F8 ? 128 : 64);
    // row of a column, -1: none
    auto row_of = [&](int c) { c = F8 ? c & 3 : c; return c >= n ? -1 : UP ? mf_nth_bit(mask, c) : base + c; };
    const int r = row_of(g);
    const uint16_t * row = r < 0 ? nullptr : (UP ? A.xp : A.hp) + (int64_t) r * stride + (F8 && g >= 4 ? plane : 0);
    // of the lane's two columns: the inverse of x's power of two, and where those of h's tiles lie
    float d[2] = { 1.f, 1.f };
    const uint16_t * hx[2] = { nullptr, nullptr };
    if (F8)
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const int rc = row_of(t * 2 + k);
            if (UP && rc >= 0) d[k] = mf_pow2(254 - S.px[rc]);
            if (!UP) hx[k] = rc < 0 ? nullptr : A.hx + (int64_t) rc * (KB * 8);
        }
    const float * sa = nullptr, * sb = nullptr;
    if (F8) {
        sa = UP ? A.s1 + ((int64_t) e * 2 * A.nb1 + i / 8) * A.KB1 : A.s2 + ((int64_t) e * A.nb2 + i / 4) * A.KB2;
        sb = UP ? sa + (int64_t) A.nb1 * A.KB1 : sa;
    }
    // the scales of 32 of the warp's lines, one a lane
    float ha = 0.f, hb = 0.f;
    auto scales = [&](int j) {
        const int kb = (j + lane) * MF_WARPS + warp;
        ha = kb < KB ? __ldg(sa + kb) : 0.f;
        hb = UP && kb < KB ? __ldg(sb + kb) : 0.f;
    };
    if (F8) scales(0);
    uint64_t acc[2][2] = { { 0, 0 }, { 0, 0 } };
#pragma unroll 1
    for (int st = 0; st < KB; st += MF_WARPS) {
        const int  kb = st + warp;
        const bool in = kb < KB;
        mf_b<F8> B;
        uint4 x[2] = { make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0) };
        float wa = 1.f, wb = 1.f;
        if (F8) {
            const int j = st / MF_WARPS;
            if (j && (j & 31) == 0) scales(j);
            wa = __shfl_sync(0xffffffffu, ha, j & 31);
            wb = UP ? __shfl_sync(0xffffffffu, hb, j & 31) : wa;
        }
        if (in) {                                                // ahead of the wait
            mf_ask<F8>(B, row, plane, kb, t);
            if (F8 && !UP)
#pragma unroll
                for (int k = 0; k < 2; k++) if (hx[k]) x[k] = mf_ld(hx[k] + kb * 8);
        }
        if (!__all_sync(0xffffffffu, dt_mbar_wait(bar_f + at.s * 8, at.ph, (volatile int *) &S.abort))) break;
        if (in) {
            const uint8_t * line = ring + at.s * MF_STAGE + warp * MF_LINE;
            const float f[2][2] = { { wa * d[0], wa * d[1] }, { wb * d[0], wb * d[1] } };
            mf_half<F8, UP>(line, 0, lane, B, f, { make_uint2(x[0].x, x[0].y), make_uint2(x[1].x, x[1].y) }, acc);
            mf_half<F8, UP>(line, 1, lane, B, f, { make_uint2(x[0].z, x[0].w), make_uint2(x[1].z, x[1].w) }, acc);
        }
        __syncwarp();
        if (lane == 0) dt_arrive(bar_e + at.s * 8);
        if (++at.s == MF_STAGES) { at.s = 0; at.ph ^= 1; }
    }
    const int gp = (g >> 1) | (g & 1) << 2;
    auto & red = S.red[turn];
#pragma unroll
    for (int m = 0; m < 2; m++)
#pragma unroll
        for (int q = 0; q < 4; q++) red[warp][t * 2 + (q & 1)][m * 16 + gp + (q >> 1) * 8] = __uint_as_float((uint32_t) (acc[m][q >> 1] >> (q & 1) * 32));
    if (mf_bar_or(*(volatile int *) &S.abort)) return false;
    auto sum = [&](int c, int k) {
        float x = 0.f;
#pragma unroll
        for (int w = 0; w < MF_WARPS; w++) x += F8 ? red[w][c][k] + red[w][c + 4][k] : red[w][c][k];
        return x;
    };
    if (UP) {
        const int last = i == A.T1 - 1 ? A.KB2 * (F8 ? 8 : 4) : i + 1;           // behind the last tile zeros, to the end of its line
        for (int q = threadIdx.x; q < n * 16; q += MF_WARPS * 32) {
            const int c = q >> 4, k = q & 15;
            const float gt = sum(c, k), u = sum(c, 16 + k), h = gt / (1.0f + expf(-gt)) * u;
            uint16_t *  hrow = A.hp + (int64_t) (base + c) * mf_row_of(F8, A.KB2);
            uint16_t *  hx = A.hx + (int64_t) (base + c) * (A.KB2 * 8);
            int field = 127;
            if (F8) {                                            // 16 neighbouring lanes hold the tile
                float m = fabsf(h);
#pragma unroll
                for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffu << (lane & 16), m, o));
                field = mf_exponent(m);
                if (k == 0) __stcg(hx + i, (uint16_t) ((254 - field) << 7));
            }
            mf_store<F8>(h, mf_pow2(field), i, k, A.KB2, hrow);
            for (int z = i + 1; z < last; z++) {
                mf_store<F8>(0.f, 1.f, z, k, A.KB2, hrow);
                if (F8 && k == 0) __stcg(hx + z, (uint16_t) (127 << 7));
            }
        }
    } else
        for (int q = threadIdx.x; q < n * 32; q += MF_WARPS * 32) __stcg(A.part + (int64_t) (base + (q >> 5)) * A.Dr + i * 32 + (q & 31), sum(q >> 5, q & 31));
    return true;
}

template <bool F8>
__global__ void __launch_bounds__(MF_THREADS, 2) moe_few_kernel(const __grid_constant__ mf_args A) {
    mf_shared & S = *reinterpret_cast<mf_shared *>(mf_dsm);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint8_t * ring = mf_dsm + MF_RING;
    const uint32_t bar_f = dt_smem(S.bars), bar_e = bar_f + MF_STAGES * 8, bar_w = bar_e + MF_STAGES * 8, bar_p = bar_w + 16;
    volatile int * abort_s = (volatile int *) &S.abort;
    if (threadIdx.x == 0) {
        for (int s = 0; s < MF_STAGES; s++) { dt_mbar_init(bar_f + s * 8, 2); dt_mbar_init(bar_e + s * 8, MF_WARPS); }
        for (int s = 0; s < 2; s++) { dt_mbar_init(bar_w + s * 8, MF_WARPS); dt_mbar_init(bar_p + s * 8, 1); }
        S.abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    pib_pdl_wait();
    pib_pdl_trigger();
    int ticket = 0;
    if (warp == MF_WARPS && lane == 0) ticket = atomicAdd(A.cnt, 1);
    mf_route<F8>(A, S, ring, warp, lane);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // the choice's values in the ring lie ahead of the copies
    __syncthreads();
    const int per = A.top + A.shared, ups = S.n_act * A.T1, items = ups + S.n_act * A.T2;
    int * done_up = A.cnt + 2, * done_rows = done_up + A.b * per;
    if (warp == MF_WARPS) {
        if (lane == 0) {
            int s = 0, item = ticket;
            uint32_t ph = 1;
            bool ok = true;
            while (item < items && ok) {
                const int  next = atomicAdd(A.cnt, 1);
                const bool up = item < ups;
                const int  a = up ? item / A.T1 : (item - ups) / A.T2, i = up ? item % A.T1 : (item - ups) % A.T2, KB = up ? A.KB1 : A.KB2;
                const uint8_t * src = up ? A.w1 + ((int64_t) S.act[a] * A.T1 + i) * KB * MF_LINE : A.w2 + ((int64_t) S.act[a] * A.T2 + i) * KB * MF_LINE;
                for (int st = 0; st < KB; st += MF_WARPS) {
                    ok = dt_mbar_wait(bar_e + s * 8, ph, abort_s);
                    if (!ok) break;
                    const uint32_t bytes = (uint32_t) min(MF_WARPS, KB - st) * MF_LINE;
                    S.item[s] = item;
                    dt_mbar_expect_tx(bar_f + s * 8, bytes);
                    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                                 ::"r"(dt_smem(ring) + s * MF_STAGE), "l"(src + (int64_t) st * MF_LINE), "r"(bytes), "r"(bar_f + s * 8) : "memory");
                    // the second arrival says that what a down item multiplies with is there
                    if (!up && st == 0) {
                        ok = false;
                        for (uint32_t it = 0; it < MF_SPIN && !ok; it++) {
                            int v, stop;
                            asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(done_up + a) : "memory");
                            ok = v >= A.T1;
                            if (!ok && (it & 63) == 63) {
                                asm volatile("ld.relaxed.gpu.global.s32 %0, [%1];" : "=r"(stop) : "l"(A.cnt + 1) : "memory");
                                if (stop || *abort_s) break;
                            }
                        }
                        if (!ok) { *abort_s = 1; atomicExch(A.cnt + 1, 1); break; }
                    }
                    dt_arrive(bar_f + s * 8);
                    if (++s == MF_STAGES) { s = 0; ph ^= 1; }
                }
                item = next;
            }
            if (ok && dt_mbar_wait(bar_e + s * 8, ph, abort_s)) { S.item[s] = -1; dt_arrive(bar_f + s * 8); dt_arrive(bar_f + s * 8); }
        }
    } else if (warp == MF_WARPS + 1) {
        // publisher: in the order of the block's items
        int turn = 0;
        uint32_t ph = 0;
        for (;;) {
            if (!__all_sync(0xffffffffu, dt_mbar_wait(bar_w + turn * 8, ph, abort_s))) break;
            const int item = S.pub[turn];
            if (item < 0) break;
            const bool up = item < ups;
            const int  i = (item - ups) % A.T2;
            bool last = false;
            if (lane == 0) {
                __threadfence();                                 // the consumers' writes too: they lie in front of their arrivals
                if (up) atomicAdd(done_up + item / A.T1, 1);
                else    last = atomicAdd(done_rows + i, 1) == S.n_act - 1;
                dt_arrive(bar_p + turn * 8);
            }
            if (__shfl_sync(0xffffffffu, last, 0)) {
                __threadfence();
                const int64_t row = i * 32 + lane;
                if (row < A.D)
                    for (int tk = 0; tk < A.b; tk++) {
                        float v = A.res ? A.res[tk * A.ldr + row] : 0.f, p[PIB_MOE_MAX_TOP];
#pragma unroll
                        for (int k = 0; k < PIB_MOE_MAX_TOP; k++) p[k] = k < per ? __ldcg(A.part + (int64_t) S.at[tk][k] * A.Dr + row) : 0.f;
#pragma unroll
                        for (int k = 0; k < PIB_MOE_MAX_TOP; k++) if (k < per) v = fmaf(S.wts[tk][k], p[k], v);
                        A.y[tk * A.ldy + row] = v;
                    }
            }
            if (turn ^= 1) continue;
            ph ^= 1;
        }
    } else {
        int turn = 0;
        mf_place at = { 0, 0 };
        uint32_t pph = 1;                                        // the first two turns find their places free
        for (;;) {
            bool ok = __all_sync(0xffffffffu, dt_mbar_wait(bar_f + at.s * 8, at.ph, abort_s) && dt_mbar_wait(bar_p + turn * 8, pph, abort_s));
            const int item = ok ? S.item[at.s] : items;             // a wait that ran out: through the barrier with the others, then out
            if (item < 0) {
                __syncwarp();
                if (lane == 0) { if (warp == 0) S.pub[turn] = -1; dt_arrive(bar_w + turn * 8); }
                mf_bar_or(false);                                // a warp whose wait ran out stands in mf_item's
                break;
            }
            const bool up = item < ups;
            const int  a = !ok ? 0 : up ? item / A.T1 : (item - ups) / A.T2, i = !ok ? 0 : up ? item % A.T1 : (item - ups) % A.T2;
            const bool go = up ? mf_item<F8, true>(A, S, ring, bar_f, bar_e, at, turn, a, i) : mf_item<F8, false>(A, S, ring, bar_f, bar_e, at, turn, a, i);
            if (!go) break;
            __syncwarp();
            if (lane == 0) { if (warp == 0) S.pub[turn] = item; dt_arrive(bar_w + turn * 8); }
            if (!(turn ^= 1)) pph ^= 1;
        }
    }
    __syncthreads();
    if (*abort_s) {                                              // say so, give copies still in flight time to land (bounded)
        if (threadIdx.x == 0) { atomicExch(A.cnt + 1, 1); atomicExch(A.err, 1 + (int) blockIdx.x); }
        for (int i = 0; i < 2000; i++) __nanosleep(1000);
    }
}

// ---- host side ----------------------------------------------------------------------------------------------------------------------
// rows of `bytes` bytes into the items' lines; with `pairs` an item holds 16 of them, behind `off`, else 32.  A thread per 16 bytes: lane t, four (two) tiles
static __global__ void mf_pack_kernel(const uint8_t * __restrict__ src, uint8_t * __restrict__ dst, int64_t rows, int64_t bytes, int64_t rows_p, int KB, int eb, int pairs, int off, int64_t n) {
    for (int64_t u = (int64_t) blockIdx.x * blockDim.x + threadIdx.x; u < n; u += (int64_t) gridDim.x * blockDim.x) {
        const int64_t j = u & 7, kb = (u >> 3) % KB, r = (u >> 3) / KB % rows_p, e = (u >> 3) / KB / rows_p;
        const int     t = (int) (j & 3), tiles = 4 / eb;         // of half a line
        __align__(16) uint8_t v[16];
        const uint8_t * p = src + (e * rows + r) * bytes;
#pragma unroll
        for (int q = 0; q < 16; q++) {
            const int64_t k = (kb * (128 / eb) + ((j >> 2) * tiles + q / (4 * eb)) * 16 + t * 4) * eb + q % (4 * eb);
            v[q] = r < rows && k < bytes ? p[k] : 0;
        }
        const int     per = pairs ? 16 : 32, in = (int) (r % per) + off;
        const int64_t tile = e * (rows_p / per) + r / per;
        *reinterpret_cast<int4 *>(dst + (tile * KB + kb) * MF_LINE + in * 128 + ((j ^ (in & 7)) * 16)) = *reinterpret_cast<const int4 *>(v);
    }
}
static cudaError_t mf_pack(const void * src, uint8_t * dst, int64_t E, int64_t rows, int64_t bytes, int64_t rows_p, int KB, int eb, int pairs, int off) {
    const int64_t n = E * rows_p * KB * 8;
    mf_pack_kernel<<<(unsigned) std::min<int64_t>((n + 255) / 256, 1 << 16), 256>>>((const uint8_t *) src, dst, rows, bytes, rows_p, KB, eb, pairs, off, n);
    return cudaGetLastError();
}

extern "C" pib_moe * pib_moe_from_device(const pib_moe_shape * sh, const float * router, const float * correction, const void * gate, const float * gate_scales, const void * up,
                                         const float * up_scales, const void * down, const float * down_scales) {
    const bool f8 = sh && sh->type == PIB_TYPE_F8;
    if (!sh || !router || !gate || !up || !down || (!f8 && sh->type != PIB_TYPE_BF16) || (f8 && (!gate_scales || !up_scales || !down_scales)) || sh->experts < 1 || sh->experts > PIB_MOE_MAX_EXPERTS ||
        sh->top < 1 || sh->top > sh->experts || sh->shared < 0 || sh->shared > PIB_MOE_MAX_TOP || sh->top + sh->shared > PIB_MOE_MAX_TOP || (sh->score != PIB_MOE_SOFTMAX && sh->score != PIB_MOE_SIGMOID) ||
        sh->width < 1 || sh->ff < 1 || sh->width > (1 << 20) || sh->ff > (1 << 20) ||
        (((uintptr_t) router | (uintptr_t) correction | (f8 ? (uintptr_t) gate_scales | (uintptr_t) up_scales | (uintptr_t) down_scales : 0)) & 3)) {
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
    if (e == cudaSuccess) e = mf_pack(gate, m->w1, E, F, D * eb, m->T1 * 16LL, m->KB1, eb, 1, 0);
    if (e == cudaSuccess) e = mf_pack(up, m->w1, E, F, D * eb, m->T1 * 16LL, m->KB1, eb, 1, 16);
    if (e == cudaSuccess) e = mf_pack(down, m->w2, E, D, F * eb, m->T2 * 32LL, m->KB2, eb, 0, 0);
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
    if (!m || !x || !y || !scratch || b < 1 || b > PIB_MAX_BATCH || (const float *) y == x || ((uintptr_t) scratch & 255) || (((uintptr_t) x | (uintptr_t) residual | (uintptr_t) y) & 3)) {
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
    A.D = D; A.Dr = L.Dr;
    A.w1 = m->w1; A.w2 = m->w2; A.s1 = m->s1; A.s2 = m->s2;
    A.res = residual; A.ldr = ldr; A.ldy = ldy; A.y = y;
    float *    z = (float *) (sc + L.z);
    float *    xm = (float *) (sc + L.xm);
    uint16_t * xp = (uint16_t *) (sc + L.xp);
    A.cnt = (int *) sc; A.z = z; A.xp = xp; A.xm = xm; A.hp = (uint16_t *) (sc + L.hp); A.hx = (uint16_t *) (sc + L.hx); A.part = (float *) (sc + L.part);
    if (!(A.err = pib_tc_error_word(st))) { pib_set_error("pib_moe_forward: no memory for the error word"); return PIB_ERR_NOMEM; }
    const int  vec = ldx % 4 == 0 && !((uintptr_t) x & 15) && D % 4 == 0, nt = b == 1 ? 1 : MF_LT;
    const dim3 rg((unsigned) (A.E * ((b + nt - 1) / nt) + b)), rb(256);
    const bool f8 = m->s.type == PIB_TYPE_F8;
#define MF_LOGITS(F8, NT) PIB_CHECK(pib_launch(moe_logits_kernel<F8, NT>, rg, rb, 0, st, m->router, x, ldx, b, A.E, D, vec, z, A.cnt, L.n_cnt, A.KB1, xp, xm))
    if (f8) { if (b == 1) MF_LOGITS(true, 1); else MF_LOGITS(true, MF_LT); }
    else    { if (b == 1) MF_LOGITS(false, 1); else MF_LOGITS(false, MF_LT); }
#undef MF_LOGITS
    const dim3 grid((unsigned) (2 * pib_num_sms())), block(MF_THREADS);
    static pib_per_device attrs;
    PIB_CHECK(attrs.once([&] {
        const cudaError_t e = cudaFuncSetAttribute(moe_few_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int) MF_SMEM);
        return e != cudaSuccess ? e : cudaFuncSetAttribute(moe_few_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int) MF_SMEM);
    }));
    if (f8) PIB_CHECK(pib_launch(moe_few_kernel<true>, grid, block, MF_SMEM, st, A));
    else    PIB_CHECK(pib_launch(moe_few_kernel<false>, grid, block, MF_SMEM, st, A));
    return PIB_OK;
}
