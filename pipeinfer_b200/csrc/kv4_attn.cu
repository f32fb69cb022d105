// kv4_attn.cu -- attention of ragged sequences over a key / value cache in 4 bits (kv4.cuh): one pass over the keys with the running maximum and sum.
#include "kv4_attn.cuh"

#include <algorithm>

__device__ __forceinline__ void ka_mma(float (&c)[4], uint4 a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
// the first product of a sum
__device__ __forceinline__ void ka_mma0(float (&c)[4], uint4 a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1), "f"(0.f));
}
// ---- decode and verification batches --------------------------------------------------------------------------------------------------
// All (sequence, tile, key / value head, page) units lie in one row, which the warps of the GPU divide evenly whatever the sequences' lengths; a warp walks its units alone, with the running maximum and
// sum of each row in registers.  Lane 0 streams the pages' records (keys' half, values' half) by bulk copies through the warp's ring of STAGES halves.
//   scores   mma.m16n8k16, rows as M, eight keys as N: lane (g, t) has 16 or 32 neighbouring channels of key g, one load and one step and lowest value, four of them a product's k
//   outputs  weights straight from the scores' registers as first operand, 16 keys as k; lane (g, t) has D / 8 neighbouring channels of four keys
// fp32 rows enter as fp16 part and remainder: rows 0..7 of a product's sixteen the parts, 8..15 the remainders, so that a row's sum is the sum of two registers of a lane.  bfloat16 rows are
// one fp16 number, as their weights, and take all sixteen.
// An item that lies in one warp's run is written at once, pieces of others go to scratch and kv4_join_kernel adds them up, in the order of the keys.
template <typename T, int D, int MT> struct ka_cfg {
    static constexpr bool SPLIT = sizeof(T) == 4;
    static constexpr int  RPM = SPLIT ? 8 : 16, RT = MT * RPM, NR = SPLIT ? 1 : 2, KS = D / 16, W = D / 32, NT = D / 8;
    static constexpr int  WARPS = 8;
    static constexpr bool QS = MT * KS >= 8;                       // the queries' operands lie in shared memory
    static constexpr int  HALF = kv4_half(D), Q_BYTES = QS ? WARPS * MT * KS * 512 : 0;
    static constexpr int  PIECE = RT * (D + 2);                   // floats
};

template <typename T, int D, int MT>
static __global__ void __launch_bounds__(ka_cfg<T, D, MT>::WARPS * 32, 1) kv4_decode_kernel(const __grid_constant__ ka_args A) {
    using C = ka_cfg<T, D, MT>;
    extern __shared__ __align__(128) uint8_t ka_dsm[];
    __shared__ uint64_t bars[C::WARPS * 16];
    __shared__ int64_t  part[C::WARPS];
    __shared__ int      abort_w;
    volatile int * abort_s = &abort_w;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3, NST = A.stages;
    uint8_t *  ring = ka_dsm + warp * NST * C::HALF;
    uint4 *    qsm  = reinterpret_cast<uint4 *>(ka_dsm + C::WARPS * NST * C::HALF) + warp * MT * C::KS * 32 + lane;
    int64_t *  prefix = reinterpret_cast<int64_t *>(ka_dsm + C::WARPS * NST * C::HALF + C::Q_BYTES);         // [seqs + 1]
    ka_seq *   seq  = reinterpret_cast<ka_seq *>(prefix + A.seqs + 1);
    const uint32_t bar0 = dt_smem(bars + warp * 16), ring0 = dt_smem(ring);
    if (lane == 0) for (int i = 0; i < NST; i++) dt_mbar_init(bar0 + i * 8, 1);
    if (threadIdx.x == 0) abort_w = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    pib_pdl_wait();
    pib_pdl_trigger();

    const int64_t U = ka_prefix<C::RT, 0, C::WARPS * 32>(A, prefix, part, [&](int s, ka_seq q) { seq[s] = q; });
    const int64_t warps = min((int64_t) gridDim.x * C::WARPS, U), me = (int64_t) warp * gridDim.x + blockIdx.x;
    ka_leave_plan<C::WARPS * 32>(A, prefix, warps);
    auto seq_of = [&](int s) { return seq[s]; };
    bool ok = true;
    if (me < warps) {
        const int64_t u0 = U * me / warps, u1 = U * (me + 1) / warps;
        ka_place at = ka_find<C::RT, 0>(A, prefix, seq_of, u0);
        // the stream of halves: 2 (u1 - u0) of them, the first NST ahead
        ka_place is = at;
        int64_t  iu = u0;
        int      ihalf = 0, ist = 0, id_s = -1, id_base = 0, ids = 0, id = 0;
        uint32_t there = 0;                                      // of each stage: whether its page is one of the cache's
        auto issue = [&]() {
            if (iu >= u1) return;
            if (!ihalf) {
                const int pg = is.first + is.p;
                if (is.s != id_s || pg < id_base || pg >= id_base + 32) {
                    id_s = is.s; id_base = pg;
                    ids = pg + lane < A.max_pages ? A.table[(int64_t) is.s * A.max_pages + pg + lane] : -1;
                }
                id = __shfl_sync(0xffffffffu, ids, pg - id_base);
            }
            const bool in = id >= 0 && id < A.pages;
            if (lane == 0) {
                if (in) {
                    dt_mbar_expect_tx(bar0 + ist * 8, C::HALF);
                    ka_bulk(ring0 + ist * C::HALF, A.base + ((int64_t) id * A.kvh + is.h) * kv4_record(D) + ihalf * C::HALF, C::HALF, bar0 + ist * 8);
                } else dt_arrive(bar0 + ist * 8);
            }
            there = in ? there | 1u << ist : there & ~(1u << ist);
            if (++ist == NST) ist = 0;
            if (ihalf) { iu++; if (iu < u1) ka_next<C::RT, 0>(A, prefix, seq_of, is); }
            ihalf ^= 1;
        };
        for (int i = 0; i < NST; i++) issue();

        int st = 0;
        uint32_t ph = 0;
        int64_t u = u0;
        while (u < u1 && ok) {
            // ---- an item, or the piece of it in this warp's run
            const ka_seq  q = seq[at.s];
            const int     rows = (int) min((int64_t) C::RT, (int64_t) q.n * A.rep - (int64_t) at.r * C::RT), pages = (int) min((int64_t) (at.np - at.p), u1 - u);
            const bool    whole = at.p == 0 && pages == at.np;
            const int     slot = 2 * (int) me + (at.p > 0 ? 0 : 1);
            const int64_t tok0 = min(max(A.starts[at.s], 0), A.tokens);
            const int     row0 = at.r * C::RT;
            float qs[MT][C::NR], m[MT][C::NR], l[MT][C::NR], O[MT][C::NT][4];
            int   lo[MT][C::NR], hi[MT][C::NR];
            uint4 qf[C::QS ? 1 : MT][C::QS ? 1 : C::KS];
            int   all_lo = 0, all_hi = 0x7fffffff;               // keys that all rows see
#pragma unroll
            for (int mt = 0; mt < MT; mt++) {
                uint32_t w[2][C::KS][2];                         // [row or part][product][k low, k high]
#pragma unroll
                for (int nr = 0; nr < C::NR; nr++) {
                    const int ri = mt * C::RPM + nr * 8 + g, rc = row0 + min(ri, rows - 1), tk = rc / A.rep, pos = q.len - q.n + tk;
                    hi[mt][nr] = pos;
                    lo[mt][nr] = A.window > 0 ? max(0, pos - A.window + 1) : 0;
                    const T * p = (const T *) A.q + (tok0 + tk) * A.ldq + (int64_t) (at.h * A.rep + rc % A.rep) * D + t * (D / 4);
                    float v[D / 4], top = 0.f;
                    ka_load<T, D / 4>(p, A.wide_q, v);
#pragma unroll
                    for (int c = 0; c < D / 4; c++) { v[c] *= A.scale * KA_LOG2E; top = fmaxf(top, fabsf(v[c])); }
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    const ka_power pw = ka_power_of(top);
                    qs[mt][nr] = pw.back;
#pragma unroll
                    for (int k = 0; k < C::KS; k++)
#pragma unroll
                        for (int b = 0; b < 2; b++) {            // product k of word k / 2 takes channels 2 (k % 2) + b and four further
                            const int   c = (k >> 1) * 8 + (k & 1) * 2 + b;
                            const float x = v[c] * pw.down, y = v[c + 4] * pw.down;
                            w[nr][k][b] = ka_pack(x, y);
                            if (C::SPLIT) w[1][k][b] = ka_rest(x, y, w[nr][k][b]);
                        }
                    m[mt][nr] = -INFINITY; l[mt][nr] = 0.f;
                }
#pragma unroll
                for (int k = 0; k < C::KS; k++) {
                    const uint4 f = make_uint4(w[0][k][0], w[1][k][0], w[0][k][1], w[1][k][1]);
                    if (C::QS) qsm[(mt * C::KS + k) * 32] = f; else qf[C::QS ? 0 : mt][C::QS ? 0 : k] = f;
                }
#pragma unroll
                for (int i = 0; i < C::NT; i++)
#pragma unroll
                    for (int c = 0; c < 4; c++) O[mt][i][c] = 0.f;
            }
            all_hi = q.len - q.n + row0 / A.rep;                                     // the first token's last key, the last token's first one
            all_lo = A.window > 0 ? q.len - q.n + (row0 + rows - 1) / A.rep - A.window + 1 : 0;

            for (int i = 0; i < pages && ok; i++) {
                const int key0 = (at.first + at.p + i) * KV4_P;
                const bool in = there >> st & 1;
                const uint32_t kst = st, kph = ph;
                if (++st == NST) { st = 0; ph ^= 1; }
                const uint32_t vst = st, vph = ph;
                if (++st == NST) { st = 0; ph ^= 1; }
                uint8_t * kp = ring + kst * C::HALF, * vp = ring + vst * C::HALF;
                const bool edge = key0 < all_lo || key0 + KV4_P - 1 > all_hi;
                ok = __all_sync(0xffffffffu, dt_mbar_wait(bar0 + kst * 8, kph, abort_s));
                if (!ok) break;
                if (!in) {                                       // no page: nothing was copied
                    issue();
                    ok = __all_sync(0xffffffffu, dt_mbar_wait(bar0 + vst * 8, vph, abort_s));
                    if (ok) issue();
                    continue;
                }
#pragma unroll 1
                for (int kb = 0; kb < 2; kb++) {
                    float S[4][MT][4];
                    uint32_t wv[4][C::W];
                    __half2  dm[4];
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const int r = kb * 32 + j * 8 + g;
                        dm[j] = *reinterpret_cast<const __half2 *>(kp + kv4_steps(D) + (r * C::W + (t * C::W >> 2)) * 4);
                        if constexpr (D == 128) { const uint4 x = *reinterpret_cast<const uint4 *>(kp + r * 64 + t * 16); wv[j][0] = x.x; wv[j][1] = x.y; wv[j][2] = x.z; wv[j][3] = x.w; }
                        else                    { const uint2 x = *reinterpret_cast<const uint2 *>(kp + r * 32 + t * 8); wv[j][0] = x.x; wv[j][1] = x.y; }
                    }
#pragma unroll
                    for (int w = 0; w < C::W; w++) {
                        uint4 f[MT][2];
#pragma unroll
                        for (int mt = 0; mt < MT; mt++)
#pragma unroll
                            for (int e = 0; e < 2; e++) f[mt][e] = C::QS ? qsm[(mt * C::KS + 2 * w + e) * 32] : qf[C::QS ? 0 : mt][C::QS ? 0 : 2 * w + e];
                        uint32_t o[4][4];
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            kv4_pairs(wv[j][w], __low2half2(dm[j]), __high2half2(dm[j]), o[j]);
#pragma unroll
                            for (int mt = 0; mt < MT; mt++)
                                if (w == 0) ka_mma0(S[j][mt], f[mt][0], o[j][0], o[j][1]); else ka_mma(S[j][mt], f[mt][0], o[j][0], o[j][1]);
                        }
#pragma unroll
                        for (int j = 0; j < 4; j++)
#pragma unroll
                            for (int mt = 0; mt < MT; mt++) ka_mma(S[j][mt], f[mt][1], o[j][2], o[j][3]);
                    }
                    if (kb == 1) {                               // the keys have been read
                        __syncwarp();
                        issue();
                    } else {
                        ok = __all_sync(0xffffffffu, dt_mbar_wait(bar0 + vst * 8, vph, abort_s));
                        if (!ok) break;
                    }
                    if (C::SPLIT)
#pragma unroll
                        for (int j = 0; j < 4; j++)
#pragma unroll
                            for (int mt = 0; mt < MT; mt++) { S[j][mt][0] += S[j][mt][2]; S[j][mt][1] += S[j][mt][3]; }
                    if (edge) {
#pragma unroll
                        for (int mt = 0; mt < MT; mt++)
#pragma unroll
                            for (int nr = 0; nr < C::NR; nr++)
#pragma unroll
                                for (int j = 0; j < 4; j++)
#pragma unroll
                                    for (int c = 0; c < 2; c++) {
                                        const int key = key0 + kb * 32 + j * 8 + t * 2 + c;
                                        if (key < lo[mt][nr] || key > hi[mt][nr]) S[j][mt][nr * 2 + c] = -INFINITY;
                                    }
                        if (kb == 0) {
                            // values that are none, on a page of which some row does not see all: the rows that see one are none in the channels of its group, and it takes part as zeros
                            bool bad = false;
                            for (int k = lane; k < KV4_P * C::W; k += 32) bad |= __hisnan(__high2half(*reinterpret_cast<const __half2 *>(vp + kv4_steps(D) + k * 4)));
                            if (__any_sync(0xffffffffu, bad)) {
                                for (int k = 0; k < KV4_P; k++)
                                    if (__hisnan(__high2half(*reinterpret_cast<const __half2 *>(vp + kv4_steps(D) + (kv4_row(k) * C::W + (t * C::W >> 2)) * 4))))
#pragma unroll
                                        for (int mt = 0; mt < MT; mt++)
#pragma unroll
                                            for (int nr = 0; nr < C::NR; nr++)
                                                if (key0 + k >= lo[mt][nr] && key0 + k <= hi[mt][nr])
#pragma unroll
                                                    for (int n = 0; n < C::NT; n++) { O[mt][n][nr * 2] = __uint_as_float(0x7fc00000u); O[mt][n][nr * 2 + 1] = __uint_as_float(0x7fc00000u); }
                                __syncwarp();
                                for (int k = lane; k < KV4_P * C::W; k += 32) {
                                    __half2 * dm = reinterpret_cast<__half2 *>(vp + kv4_steps(D) + k * 4);
                                    if (__hisnan(__high2half(*dm))) *dm = kv4_bits(0);
                                }
                                dt_fence_async();                // the ring's next copy comes behind these stores
                                __syncwarp();
                            }
                        }
                    }
                    // ---- weights: the rows' maxima, exponentials, sums
                    uint4 P[2][MT];
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) {
#pragma unroll
                        for (int nr = 0; nr < C::NR; nr++) {
                            float top = -INFINITY;
#pragma unroll
                            for (int j = 0; j < 4; j++) top = fmaxf(top, fmaxf(S[j][mt][nr * 2], S[j][mt][nr * 2 + 1]));
                            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2)) * qs[mt][nr];
                            if (__any_sync(0xffffffffu, top > m[mt][nr] + KA_LAZY)) {
                                const float mn = top > m[mt][nr] + KA_LAZY ? top : m[mt][nr], a = mn == m[mt][nr] ? 1.f : ka_exp2(m[mt][nr] - mn);
                                m[mt][nr] = mn;
                                l[mt][nr] *= a;
#pragma unroll
                                for (int n = 0; n < C::NT; n++) {
                                    O[mt][n][nr * 2] *= a; O[mt][n][nr * 2 + 1] *= a;
                                    if (C::SPLIT) { O[mt][n][2] *= a; O[mt][n][3] *= a; }
                                }
                            }
                            const float base = KA_LIFT - (m[mt][nr] == -INFINITY ? 0.f : m[mt][nr]);
#pragma unroll
                            for (int j = 0; j < 4; j++) {
                                const float x = ka_exp2(fmaf(S[j][mt][nr * 2], qs[mt][nr], base)), y = ka_exp2(fmaf(S[j][mt][nr * 2 + 1], qs[mt][nr], base));
                                l[mt][nr] += x + y;
                                const uint32_t h = ka_pack(x, y);
                                uint32_t & at0 = j & 1 ? P[j >> 1][mt].z : P[j >> 1][mt].x, & at1 = j & 1 ? P[j >> 1][mt].w : P[j >> 1][mt].y;
                                if (C::SPLIT) { at0 = h; at1 = ka_rest(x, y, h); }
                                else if (nr == 0) at0 = h;
                                else at1 = h;
                            }
                        }
                    }
                    // ---- outputs
#pragma unroll
                    for (int i2 = 0; i2 < 2; i2++) {
                        uint32_t a[2][C::W / 2], b[2][C::W / 2];               // this lane's channels of keys 2 t and 2 t + 1 of both groups of eight
                        __half2  d2[2], m2[2];
#pragma unroll
                        for (int f = 0; f < 2; f++) {
                            const int ra = kb * 32 + i2 * 16 + f * 8 + t, rb = ra + 4;         // kv4_row of the places 2 t and 2 t + 1
                            const __half2 da = *reinterpret_cast<const __half2 *>(vp + kv4_steps(D) + (ra * C::W + (g * C::W >> 3)) * 4);
                            const __half2 db = *reinterpret_cast<const __half2 *>(vp + kv4_steps(D) + (rb * C::W + (g * C::W >> 3)) * 4);
                            d2[f] = __lows2half2(da, db); m2[f] = __highs2half2(da, db);
                            if constexpr (D == 128) {
                                const uint2 x = *reinterpret_cast<const uint2 *>(vp + ra * 64 + ((g * 8) ^ kv4_flip(D, ra))), y = *reinterpret_cast<const uint2 *>(vp + rb * 64 + ((g * 8) ^ kv4_flip(D, rb)));
                                a[f][0] = x.x; a[f][1] = x.y; b[f][0] = y.x; b[f][1] = y.y;
                            } else { a[f][0] = *reinterpret_cast<const uint32_t *>(vp + ra * 32 + g * 4); b[f][0] = *reinterpret_cast<const uint32_t *>(vp + rb * 32 + g * 4); }
                        }
#pragma unroll
                        for (int w = 0; w < C::W / 2; w++)
#pragma unroll
                            for (int e = 0; e < 2; e++) {
                                uint32_t x[4], y[4];
                                kv4_pairs(ka_prmt(a[0][w], b[0][w], e ? 0x7632 : 0x5410), d2[0], m2[0], x);
                                kv4_pairs(ka_prmt(a[1][w], b[1][w], e ? 0x7632 : 0x5410), d2[1], m2[1], y);
#pragma unroll
                                for (int n = 0; n < 4; n++)
#pragma unroll
                                    for (int mt = 0; mt < MT; mt++) ka_mma(O[mt][w * 8 + e * 4 + n], P[i2][mt], x[n], y[n]);
                            }
                    }
                }
                if (!ok) break;
                __syncwarp();
                issue();                                         // the values have been read
            }
            if (!ok) break;
            // ---- rows out: lane (g, t) has D / 4 neighbouring channels of its rows
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int nr = 0; nr < C::NR; nr++) {
                    float sum = l[mt][nr];
                    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                    const int ri = mt * C::RPM + nr * 8 + g;
                    if (ri >= rows) continue;
                    float v[D / 4];
#pragma unroll
                    for (int n = 0; n < C::NT; n++) {
                        v[n]         = C::SPLIT ? O[mt][n][0] + O[mt][n][2] : O[mt][n][nr * 2];
                        v[n + C::NT] = C::SPLIT ? O[mt][n][1] + O[mt][n][3] : O[mt][n][nr * 2 + 1];
                    }
                    if (whole) {
                        const float inv = sum > 0.f ? 1.f / sum : sum;           // a row that saw nothing: zeros; a sum that is none stays so
#pragma unroll
                        for (int c = 0; c < D / 4; c++) v[c] *= inv;
                        const int rc = row0 + ri;
                        ka_store<T, D / 4>((T *) A.out + (tok0 + rc / A.rep) * A.ldo + (int64_t) (at.h * A.rep + rc % A.rep) * D + t * (D / 4), A.wide_o, v);
                    } else {
                        float * p = A.pieces + (int64_t) slot * C::PIECE;
                        ka_store<float, D / 4>(p + ri * D + t * (D / 4), true, v);
                        if (t == 0) { p[C::RT * D + ri] = m[mt][nr]; p[C::RT * D + C::RT + ri] = sum; }
                    }
                }
            u += pages;
            at.p += pages - 1;
            if (u < u1) ka_next<C::RT, 0>(A, prefix, seq_of, at);
        }
    }
    __syncthreads();
    if (*abort_s) {                                              // a wait ran out: say so, give copies still in flight time to land (bounded)
        if (threadIdx.x == 0) atomicExch(A.err, 1 + (int) blockIdx.x);
        for (int i = 0; i < 2000; i++) __nanosleep(1000);
    }
}

// A block per (token, query head): rows of items that lay in several warps' runs get their pieces' sum, rows of items without pages zeros; the others are written already.
template <typename T, int D, int MT>
static __global__ void __launch_bounds__(256) kv4_join_kernel(const __grid_constant__ ka_args A) {
    using C = ka_cfg<T, D, MT>;
    pib_pdl_wait();
    pib_pdl_trigger();
    __shared__ int   found;
    __shared__ float sm_m[8], sm_l[8], sm_o[8][D];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, heads = A.kvh * A.rep, t = blockIdx.x / heads, hq = blockIdx.x % heads, h = hq / A.rep;
    if (threadIdx.x == 0) found = -1;
    __syncthreads();
    for (int s = threadIdx.x; s < A.seqs; s += 256) if (A.starts[s] <= t && t < A.starts[s + 1]) atomicMax(&found, s);
    __syncthreads();
    const int s = found;
    if (s < 0) return;
    const ka_seq q = ka_load_seq(A, s);
    const int tl = t - min(max(A.starts[s], 0), A.tokens), idx = tl * A.rep + hq % A.rep, r = idx / C::RT, ri = idx % C::RT;
    if (tl >= q.n) return;
    int     first;
    int64_t ib = A.plan->prefix[s];
    for (int i = 0; i < r; i++) ib += (int64_t) ka_pages<C::RT>(A, q, i, first) * A.kvh;
    const int np = ka_pages<C::RT>(A, q, r, first);
    ib += (int64_t) h * np;
    T * out = (T *) A.out + (int64_t) t * A.ldo + (int64_t) hq * D;
    if (np == 0) {
        if (threadIdx.x < D) out[threadIdx.x] = (T) 0.f;
        return;
    }
    const int64_t U = A.plan->prefix[A.seqs], W = A.plan->runs, wa = ((ib + 1) * W + U - 1) / U - 1, wb = ((ib + np) * W + U - 1) / U - 1;
    if (wa == wb) return;
    constexpr int CH = D / 32;
    float m = -INFINITY, l = 0.f, o[CH];
#pragma unroll
    for (int c = 0; c < CH; c++) o[c] = 0.f;
    // a warp takes every eighth piece, 32 of them at a time: their maxima and sums, a piece a lane, then their rows, whose loads wait for nothing
    for (int64_t w0 = wa + warp; w0 <= wb; w0 += 256) {
        const int n = (int) min((int64_t) 32, (wb - w0) / 8 + 1);
        auto piece = [&](int k) { const int64_t w = w0 + 8 * k; return A.pieces + (2 * w + (w == wa ? 1 : 0)) * (int64_t) C::PIECE; };
        float pm = -INFINITY, pl = 0.f;
        if (lane < n) { pm = piece(lane)[C::RT * D + ri]; pl = piece(lane)[C::RT * D + C::RT + ri]; }
        const float mn = fmaxf(m, warp_max(pm)), a = m == mn ? 1.f : exp2f(m - mn), f = pm == mn ? 1.f : exp2f(pm - mn);
        m = mn; l = l * a + warp_sum(lane < n ? pl * f : 0.f);
#pragma unroll
        for (int c = 0; c < CH; c++) o[c] *= a;
#pragma unroll 8
        for (int k = 0; k < n; k++) {
            const float * p = piece(k) + ri * D;
            const float   fk = __shfl_sync(0xffffffffu, f, k);
            if constexpr (CH == 4) { const float4 v = *reinterpret_cast<const float4 *>(p + lane * 4); o[0] = fmaf(v.x, fk, o[0]); o[1] = fmaf(v.y, fk, o[1]); o[2] = fmaf(v.z, fk, o[2]); o[3] = fmaf(v.w, fk, o[3]); }
            else                   { const float2 v = *reinterpret_cast<const float2 *>(p + lane * 2); o[0] = fmaf(v.x, fk, o[0]); o[1] = fmaf(v.y, fk, o[1]); }
        }
    }
    if (lane == 0) { sm_m[warp] = m; sm_l[warp] = l; }
#pragma unroll
    for (int c = 0; c < CH; c++) sm_o[warp][lane * CH + c] = o[c];
    __syncthreads();
    if (threadIdx.x >= D) return;
    m = sm_m[0];
    for (int i = 1; i < 8; i++) m = fmaxf(m, sm_m[i]);
    float v = 0.f;
    l = 0.f;
    for (int i = 0; i < 8; i++) {
        const float a = sm_m[i] == m ? 1.f : exp2f(sm_m[i] - m);
        l += sm_l[i] * a; v += sm_o[i][threadIdx.x] * a;
    }
    out[threadIdx.x] = (T) (l > 0.f ? v / l : l != l ? l : 0.f);
}

// ---- host side --------------------------------------------------------------------------------------------------------------------
static int ka_batch_ok(const char * who, const pib_kv4 * kv, const pib_kv4_batch * b) {
    const bool ok = kv && b && kv4_type_size(b->type) && b->heads >= 1 && b->heads <= PIB_KV4_MAX_HEADS && b->heads % kv->heads == 0 && b->tokens >= 0 && b->tokens <= PIB_KV4_MAX_TOKENS && b->seqs >= 0 &&
                    b->seqs <= PIB_KV4_MAX_SEQS && b->max_tokens >= 0 && b->max_pages >= 0 && b->window >= 0 && b->scale == b->scale && fabsf(b->scale) <= 3.4e38f;
    if (ok) return PIB_OK;
    if (!b) pib_set_error("%s: bad arguments", who);
    else pib_set_error("%s: bad batch (type %d, %d heads, %d tokens, %d sequences, %d pages, window %d, scale %g)", who, b->type, b->heads, b->tokens, b->seqs, b->max_pages, b->window, b->scale);
    return PIB_ERR_ARG;
}
// whether rows of n bytes at a, lda bytes apart, and rows at b, ldb bytes apart, have a byte in common
static bool ka_overlap(const uint8_t * a, int64_t lda, const uint8_t * b, int64_t ldb, int64_t n, int64_t rows) {
    if (a + (rows - 1) * lda + n <= b || b + (rows - 1) * ldb + n <= a) return false;
    if (lda == ldb) {                                            // columns of the same rows may lie beside each other
        const int64_t off = ((b - a) % lda + lda) % lda;
        return !(off >= n && off + n <= lda);
    }
    return true;
}

// rows (token, head of the group) of the longest portion: up to one or two products' rows by the decode kernels, more than KA_FEW on tcgen05
#define KA_FEW 64
static int64_t ka_rows(const pib_kv4 * kv, const pib_kv4_batch * b) { return (int64_t) (b->max_tokens ? std::min(b->max_tokens, b->tokens) : b->tokens) * (b->heads / kv->heads); }
static int ka_mt(const pib_kv4 * kv, const pib_kv4_batch * b) { return ka_rows(kv, b) > (b->type == PIB_TYPE_F32 ? 8 : 16) ? 2 : 1; }
static size_t ka_pieces(const pib_kv4 * kv, const pib_kv4_batch * b) {
    const size_t rows = ka_rows(kv, b) > KA_FEW ? KP_ROWS : (size_t) 8 * ka_mt(kv, b) * (b->type == PIB_TYPE_F32 ? 8 : 16);
    return (size_t) 2 * pib_num_sms() * rows * (kv->dim + 2) * 4;
}
extern "C" size_t pib_kv4_attn_scratch_bytes(const pib_kv4 * kv, const pib_kv4_batch * b) {
    if (ka_batch_ok("pib_kv4_attn_scratch_bytes", kv, b) != PIB_OK) return 0;
    return (ka_pieces(kv, b) + sizeof(ka_plan) + 255) & ~(size_t) 255;
}

template <typename T, int D, int MT> static int ka_go(ka_args A, cudaStream_t st) {
    using C = ka_cfg<T, D, MT>;
    const size_t table = ((size_t) (A.seqs + 1) * 8 + (size_t) A.seqs * sizeof(ka_seq) + 127) & ~(size_t) 127, most = 224 * 1024;
    A.stages = (int) std::min<size_t>(8, (most - C::Q_BYTES - table) / (C::WARPS * C::HALF));
    static pib_per_device attrs;
    PIB_CHECK(attrs.once([&] { return cudaFuncSetAttribute(kv4_decode_kernel<T, D, MT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int) most); }));
    PIB_CHECK(pib_launch(kv4_decode_kernel<T, D, MT>, dim3((unsigned) pib_num_sms()), dim3(C::WARPS * 32), (size_t) C::WARPS * A.stages * C::HALF + C::Q_BYTES + table, st, A));
    PIB_CHECK(pib_launch(kv4_join_kernel<T, D, MT>, dim3((unsigned) ((int64_t) A.tokens * A.kvh * A.rep)), dim3(256), 0, st, A));
    return PIB_OK;
}

extern "C" int pib_kv4_attn(const pib_kv4 * kv, const pib_kv4_batch * b, const void * q, int64_t ldq, const int32_t * starts, const int32_t * lens, const int32_t * pages, void * out, int64_t ldo,
                            void * scratch, pib_stream s) {
    int rc = kv4_ok("pib_kv4_attn", kv);
    if (rc != PIB_OK || (rc = ka_batch_ok("pib_kv4_attn", kv, b)) != PIB_OK) return rc;
    if (!b->tokens || !b->seqs) return PIB_OK;
    const int     size = kv4_type_size(b->type);
    const int64_t row = (int64_t) b->heads * kv->dim;
    if (!q || !out || !starts || !lens || (!pages && b->max_pages) || !scratch || ldq < row || ldo < row || (((uintptr_t) q | (uintptr_t) out) & (size - 1)) ||
        (((uintptr_t) starts | (uintptr_t) lens | (uintptr_t) pages) & 3) || ((uintptr_t) scratch & 255)) {
        pib_set_error("pib_kv4_attn: bad arguments (rows %lld and %lld apart)", (long long) ldq, (long long) ldo);
        return PIB_ERR_ARG;
    }
    if (ka_overlap((const uint8_t *) q, ldq * size, (const uint8_t *) out, ldo * size, row * size, b->tokens)) { pib_set_error("pib_kv4_attn: out lies over q"); return PIB_ERR_ARG; }
    ka_args A;
    A.base = kv->base; A.pages = kv->pages; A.kvh = kv->heads; A.rep = b->heads / kv->heads; A.dim = kv->dim;
    A.starts = starts; A.lens = lens; A.table = pages; A.tokens = b->tokens; A.seqs = b->seqs; A.max_pages = b->max_pages; A.window = b->window; A.scale = b->scale;
    A.q = q; A.out = out; A.ldq = ldq; A.ldo = ldo;
    A.wide_q = ((uintptr_t) q & 15) == 0 && ldq * size % 16 == 0;
    A.wide_o = ((uintptr_t) out & 15) == 0 && ldo * size % 16 == 0;
    A.pieces = (float *) scratch; A.plan = (ka_plan *) ((uint8_t *) scratch + ka_pieces(kv, b));
    A.stages = 0;
    if (!(A.err = pib_tc_error_word((cudaStream_t) s))) { pib_set_error("pib_kv4_attn: no memory for the error word"); return PIB_ERR_NOMEM; }
    const cudaStream_t st = (cudaStream_t) s;
    if (ka_rows(kv, b) > KA_FEW) return pib_kv4_prompt(A, size == 4, st);
    const int form = (size == 4 ? 4 : 0) + (kv->dim == 128 ? 2 : 0) + (ka_mt(kv, b) == 2 ? 1 : 0);
    switch (form) {
        case 0:  return ka_go<__nv_bfloat16, 64, 1>(A, st);
        case 1:  return ka_go<__nv_bfloat16, 64, 2>(A, st);
        case 2:  return ka_go<__nv_bfloat16, 128, 1>(A, st);
        case 3:  return ka_go<__nv_bfloat16, 128, 2>(A, st);
        case 4:  return ka_go<float, 64, 1>(A, st);
        case 5:  return ka_go<float, 64, 2>(A, st);
        case 6:  return ka_go<float, 128, 1>(A, st);
        default: return ka_go<float, 128, 2>(A, st);
    }
}
