// kv4_attn.cu -- attention of ragged sequences over a key / value cache in 4 bits (kv4.cuh): one pass over the keys with the running maximum and sum.  Decode and verification batches; prompts: kv4_prompt.cu.
#include "kv4_attn.cuh"

#include <algorithm>

// c += a b: 16 x 16 by 16 x 8 in fp16, fp32 sums (not volatile: the order is the compiler's)
__device__ __forceinline__ void ka_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint2 b) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b.x), "r"(b.y));
}
// the first product of a sum
__device__ __forceinline__ void ka_mma0(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint2 b) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b.x), "r"(b.y), "f"(0.f));
}
// an 8 x 8 matrix of 16-bit numbers, two of a row a lane, turned
__device__ __forceinline__ uint32_t ka_turn(uint32_t v) { uint32_t r; asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v)); return r; }

// All (sequence, tile of rows, key / value head, page) units lie in one row, which the blocks of the GPU divide evenly whatever the sequences' lengths (with an item's start and end counted as pages), and a block's warps its run; a warp walks its units
// alone, with the running maximum and sum of each row in registers.  Lane 0 streams the pages' records (keys' half, values' half) by bulk copies through the warp's ring of STAGES halves.
//   scores   turned, S' = K Q': mma.m16n8k16, 16 keys as M, eight rows as N, keys straight from nibbles in registers: lane (g, t) has 16 or 32 neighbouring channels of keys g and g + 8, one load and one step
//            and lowest value each, four of them a product's k
//   outputs  O' = V' P': 16 channels as M, weights (turned once more by movmatrix) as N, 16 keys as k; lane (g, t) has D / 8 neighbouring channels of four keys
// The tensor core cuts off what it adds to a sum, always towards zero: of fp32 rows the rests' scores have sums of their own, and each product of weights begins at zero and is added with rounding.
// Rows as N cost what is there in steps of eight (as M, eight rows are a product of sixteen).  Queries of fp32 rows enter as fp16 part and remainder, two products, those of bfloat16 rows as one fp16 number.
// Weights are two products beside either: as one fp16 number they move one of eleven bfloat16 outputs to its neighbour (now one of 2,000), for 4 % of the time.
// An item that lies in one warp's units is written at once.  Pieces of others meet in shared memory at the end, in the order of the keys; what then is not a whole item goes to scratch, two pieces a block at
// most, and kv4_join_kernel adds those up.
// What bounds it: two warps an SM quarter, each a chain of conversions, products, the rows' maxima and exponentials; of 64 / 8 heads of 128 one bfloat16 token behind 131,071 keys takes 61 us (its records'
// bytes 26), 32 ragged fp32 sequences 47 (13), 16 x 4 bfloat16 tokens 41 (4: two pages a warp, so the start, queries, pieces and the join are most of it, and that kernel spills 248 bytes of its registers).
// Captured calls' times, here and below.  Warps of a block: registers (217 to 255 a thread) allow no more
#define KA_WARPS 8
// Pages after which a warp's sums leave its registers.  They are added to those of the same item before, fp32 rows' with compensation, and begin anew: additions with rounding (fp32 rows, one for each 16 keys)
// and those of a tensor core that cuts (bfloat16 rows) are chains of 256 whatever the item's length.  (Without, fp32 outputs behind 64,000 keys whose values are one were off by 3e-6, bfloat16 ones behind
// 131,072 keys low by 0.9e-3)
#define KA_FOLD 64
template <typename T, int D, int NR> struct ka_cfg {                 // NR: tiles of eight rows
    static constexpr bool SPLIT = sizeof(T) == 4;
    static constexpr int  RT = 8 * NR, PARTS = SPLIT ? 2 : 1, KS = D / 16, W = D / 32, MT = D / 16, C8 = D / 8;
    static constexpr int  WARPS = KA_WARPS;
    // keys of which the scores are in registers at once.  bfloat16, 8 rows, 131,071 keys: 61.4 us with 64, 65.1 with 32; 32 ragged sequences 67.1 and 71.6; 16 rows 40.7 and 41.2.  fp32 has registers for 32
    static constexpr int  KB = NR <= 2 && !SPLIT ? 64 : 32;
    static constexpr bool QS = NR > 1;                               // the queries' operands lie in shared memory
    // an item's start and end (queries, sums out, its piece's place), in pages' time.  With these and without: 16 x 4 tokens behind 300 to 8,190 keys 99 and 106 us, 32 such single ones 67 and 71, fp32 79 and 83
    static constexpr int  EXTRA = NR == 4 ? 3 : NR == 2 && SPLIT ? 1 : 2;
    static constexpr int  HALF = kv4_half(D), Q_BYTES = QS ? WARPS * NR * PARTS * KS * 256 : 0;
    static constexpr int  PIECE = RT * (D + 2);                      // floats
    // a warp's sums that have left its registers, in four floats: of each tile outputs, and {maxima, denominators}; of fp32 rows behind them what additions to those rounded away
    static constexpr int  REST = NR * (MT + 1) * 32, SUMS = SPLIT ? 2 * REST : REST;
};

// what happens once an item is a call: the loop over pages is long enough
template <int RT> __device__ __noinline__ ka_place ka_find_call(const ka_args & A, const int64_t * prefix, ka_seq_table seq, int64_t u) { return ka_find<RT, 0>(A, prefix, seq, u); }
template <int RT, int EXTRA> __device__ __noinline__ int64_t ka_cut_call(const ka_args & A, const int64_t * prefix, const int * items, ka_seq_table seq, int64_t w) { return ka_cut<RT, EXTRA>(A, prefix, items, seq, w); }
template <int RT> __device__ __noinline__ ka_place ka_next_call(const ka_args & A, const int64_t * prefix, ka_seq_table seq, ka_place c) { ka_next_item<RT, 0>(A, prefix, seq, c); return c; }
template <int RT> __device__ __forceinline__ void ka_next(const ka_args & A, const int64_t * prefix, ka_seq_table seq, ka_place & c) { if (++c.p >= c.np) c = ka_next_call<RT>(A, prefix, seq, c); }
// two or four neighbouring channels
__device__ __forceinline__ void ka_get(const float * p, float (&v)[2]) { const float2 f = *reinterpret_cast<const float2 *>(p); v[0] = f.x; v[1] = f.y; }
__device__ __forceinline__ void ka_get(const float * p, float (&v)[4]) { const float4 f = *reinterpret_cast<const float4 *>(p); v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w; }
__device__ __forceinline__ void ka_put(float * p, const float (&v)[2]) { *reinterpret_cast<float2 *>(p) = make_float2(v[0], v[1]); }
__device__ __forceinline__ void ka_put(float * p, const float (&v)[4]) { *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]); }
// a warp's piece of an item: sums of the rows that there are, their maxima and denominators
template <typename C, int NR>
__device__ __forceinline__ void ka_leave(float * p, int rows, int g, int t, const float (&O)[NR][C::MT][4], const float (&m)[NR][2], const float (&l)[NR][2]) {
#pragma unroll
    for (int n = 0; n < NR; n++)
#pragma unroll
        for (int r = 0; r < 2; r++) {
            const int ri = n * 8 + 2 * t + r;
            if (ri >= rows) continue;
            float v[C::C8];
#pragma unroll
            for (int c = 0; c < C::C8; c++) v[c] = O[n][c >> 1][2 * (c & 1) + r];
            ka_store<float, C::C8>(p + ri * (C::C8 * 8) + g * C::C8, true, v);
            if (g == 0) { p[C::RT * C::C8 * 8 + ri] = m[n][r]; p[C::RT * C::C8 * 8 + C::RT + ri] = l[n][r]; }
        }
}
// row ri of an item from its sums over all keys, D / 32 channels a lane
template <typename T, int D> __device__ __forceinline__ void ka_row_out(const ka_args & A, const ka_open & it, int ri, int lane, const float (&o)[D / 32], float l) {
    const int   rc = it.row0 + ri, tk = ka_over(A, rc);
    const float inv = l > 0.f ? 1.f / l : l;
    T * out = (T *) A.out + (it.tok0 + tk) * A.ldo + (int64_t) (it.h * A.rep + rc - tk * A.rep) * D + lane * (D / 32);
#pragma unroll
    for (int c = 0; c < D / 32; c++) out[c] = (T) (o[c] * inv);
}

template <typename T, int D, int NR>
static __global__ void __launch_bounds__(ka_cfg<T, D, NR>::WARPS * 32, 1) kv4_decode_kernel(const __grid_constant__ ka_args A) {
    using C = ka_cfg<T, D, NR>;
    extern __shared__ __align__(128) uint8_t ka_dsm[];
    __shared__ uint64_t bars[C::WARPS * 8];
    __shared__ int64_t  part[2 * C::WARPS];
    __shared__ ka_open  items[C::WARPS], last_item[C::WARPS];
    __shared__ int      flags[C::WARPS];
    __shared__ float    backs[C::WARPS][C::RT];
    __shared__ int      abort_w;
    volatile int * abort_s = &abort_w;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3, NST = A.stages;
    uint8_t *  ring = ka_dsm + warp * NST * C::HALF;
    uint2 *    qsm  = reinterpret_cast<uint2 *>(ka_dsm + C::WARPS * NST * C::HALF) + warp * NR * C::PARTS * C::KS * 32 + lane;
    int64_t *  prefix = reinterpret_cast<int64_t *>(ka_dsm + C::WARPS * NST * C::HALF + C::Q_BYTES);         // [seqs + 1]
    ka_seq *   seq  = reinterpret_cast<ka_seq *>(prefix + A.seqs + 1);
    float *    back = backs[warp];
    const uint32_t bar0 = dt_smem(bars + warp * 8), ring0 = dt_smem(ring);
    if (lane == 0) for (int i = 0; i < NST; i++) dt_mbar_init(bar0 + i * 8, 1);
    if (threadIdx.x == 0) abort_w = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    pib_pdl_wait();
    pib_pdl_trigger();
    int *         count = reinterpret_cast<int *>(seq + A.seqs);     // [seqs + 1]
    const int64_t units = ka_prefix<C::RT, 0, C::WARPS * 32, ka_seq_table>(A, prefix, part, { seq }, count), U = units + (int64_t) C::EXTRA * count[A.seqs];
    const int     runs = (int) min((int64_t) gridDim.x, U);
    const ka_seq_table seq_of = { seq };
    const int64_t w0 = blockIdx.x < runs ? U * blockIdx.x / runs : 0, w1 = blockIdx.x < runs ? U * (blockIdx.x + 1) / runs : 0;
    // (both ends at once, a lane each)
    const int64_t cut = w0 < w1 ? ka_cut_call<C::RT, C::EXTRA>(A, prefix, count, seq_of, lane & 1 ? min(w1, U - 1) : w0) : 0;
    const int64_t c0 = __shfl_sync(0xffffffffu, cut, 0), to = __shfl_sync(0xffffffffu, cut, 1), c1 = w0 < w1 && w1 == U ? units : to;
    ka_zero_rows<C::RT, C::WARPS * 32, T>(A, seq_of, D);
    bool ok = true;
    // the warp's pieces of items that lie in several warps' units: one that ends here (in scratch), one that does not (in registers)
    bool    ends = false, goes = false, begins = false;
    ka_place at = { 0, 0, 0, 0, 0, 0 };
    float qs[NR][2], m[NR][2], l[NR][2], O[NR][C::MT][4];            // of rows 2 t and 2 t + 1 of each tile
    // A warp begins where an item does if that is a page away: items of few pages stay with one warp.  Not further: the longest warp is the block's time (a quarter of the warp's pages: 32 fp32 sequences 89 us
    // for 79, 131,071 keys 65 for 61; never: level)
    if (c0 < c1) {
        const int64_t raw = c0 + (c1 - c0) * warp / C::WARPS;
        const int     near = 1;
        at = ka_find_call<C::RT>(A, prefix, seq_of, raw);
        int64_t u = raw;
        if (warp > 0) {
            if (at.p <= near && at.p <= at.np - at.p) { if (raw - at.p >= c0) { u -= at.p; at.p = 0; } }     // (not into the block before)
            else if (at.np - at.p <= near) { u += at.np - at.p; if (u < c1) { at.p = at.np - 1; ka_next<C::RT>(A, prefix, seq_of, at); } }
        }
        if (lane == 0) part[warp] = min(u, c1);
    }
    __syncthreads();
    const int64_t u0 = c0 < c1 ? part[warp] : 0, u1 = c0 < c1 ? (warp + 1 < C::WARPS ? part[warp + 1] : c1) : 0;
    if (u0 < u1) {
        // the stream of halves: 2 (u1 - u0) of them, the first NST ahead
        ka_place is = at;
        int      left = (int) (u1 - u0), todo = left;            // units to ask for, units to do
        int      ihalf = 0, ist = 0, id_s = -1, id_base = 0, ids = 0, id = 0;
        uint32_t there = 0;                                      // of each stage: whether its page is one of the cache's
        auto issue = [&]() {
            if (left == 0) return;
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
            if (ihalf) { left--; if (left) ka_next<C::RT>(A, prefix, seq_of, is); }
            ihalf ^= 1;
        };
        int st = 0;
        uint32_t ph = 0;
        bool begun = false;
#pragma unroll 1
        while (todo && ok) {
            // ---- an item, or the piece of it in this warp's run
            const ka_seq  q = seq[at.s];
            const int     rows = (int) min((int64_t) C::RT, (int64_t) q.n * A.rep - (int64_t) at.r * C::RT), pages = min(at.np - at.p, todo);
            const bool    whole = at.p == 0 && pages == at.np;
            const int     t0 = at.r * C::RT / A.rep, row0 = at.r * C::RT - t0 * A.rep, pos0 = q.len - q.n + t0;      // rows counted from the first token that has some
            const int64_t tok0 = q.start + t0;
            uint2 qf[C::QS ? 1 : C::PARTS][C::QS ? 1 : C::KS];
            // as the products' second operand a lane has row g: the channels of its t.  The next tile's are on their way meanwhile
            uint32_t raw[D / 4 * sizeof(T) / 4];
            auto fetch = [&](int n) {
                const int rc = row0 + min(n * 8 + g, rows - 1), tk = ka_over(A, rc);
                ka_fetch<T, D / 4>((const T *) A.q + (tok0 + tk) * A.ldq + (int64_t) (at.h * A.rep + rc - tk * A.rep) * D + t * (D / 4), ka_here(A.wide_q), raw);
            };
            fetch(0);
            if (!begun) {                                        // (behind the first queries' loads: both are on their way together)
                begun = true;
#pragma unroll 1
                for (int i = 0; i < NST; i++) issue();
            }
#pragma unroll 1
            for (int n = 0; n < NR; n++) {
                float v[D / 4], top = 0.f;
#pragma unroll
                for (int c = 0; c < D / 4; c++) { v[c] = C::SPLIT ? ka_value<T>(raw, c) * (A.scale * KA_LOG2E) : ka_value<T>(raw, c); top = fmaxf(top, fabsf(v[c])); }
                if (n + 1 < NR) fetch(n + 1);
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const ka_power pw = ka_power_of<C::SPLIT>(top, A.scale);
                if (C::QS) { if (t == 0) back[n * 8 + g] = pw.back; }
                else
#pragma unroll
                    for (int r = 0; r < 2; r++) qs[0][r] = __shfl_sync(0xffffffffu, pw.back, (2 * t + r) * 4);
#pragma unroll
                for (int k = 0; k < C::KS; k++) {                // product k of word k / 2 takes channels 2 (k % 2), 2 (k % 2) + 1 and four further
                    const int   c = (k >> 1) * 8 + (k & 1) * 2;
                    const float x0 = v[c] * pw.down, x1 = v[c + 4] * pw.down, y0 = v[c + 1] * pw.down, y1 = v[c + 5] * pw.down;
                    const uint2 hi = make_uint2(ka_pack(x0, x1), ka_pack(y0, y1));
                    if (C::QS) qsm[(n * C::PARTS * C::KS + k) * 32] = hi; else qf[0][C::QS ? 0 : k] = hi;
                    if (C::SPLIT) {
                        const uint2 lo = make_uint2(ka_rest(x0, x1, hi.x), ka_rest(y0, y1, hi.y));
                        if (C::QS) qsm[((n * C::PARTS + 1) * C::KS + k) * 32] = lo; else qf[C::QS || !C::SPLIT ? 0 : 1][C::QS ? 0 : k] = lo;
                    }
                }
            }
            if (C::QS) __syncwarp();
#pragma unroll
            for (int n = 0; n < NR; n++) {
#pragma unroll
                for (int r = 0; r < 2; r++) { if (C::QS) qs[n][r] = back[n * 8 + 2 * t + r]; m[n][r] = -INFINITY; l[n][r] = 0.f; }
#pragma unroll
                for (int i = 0; i < C::MT; i++)
#pragma unroll
                    for (int c = 0; c < 4; c++) O[n][i][c] = 0.f;
            }
            if (C::QS) __syncwarp();                             // (the next item's may come)
            int huge = 0;                                        // bfloat16, of each tile: whether a row's maximum is beyond KA_HUGE
            // keys that all rows see: from the last token's first one to the first token's last
            const int all_hi = pos0, all_lo = max(0, pos0 + ka_over(A, row0 + rows - 1) - ka_window(A) + 1);
            // the last key that row r of the tiles sees, and the first
            auto high = [&](int r) { return pos0 + ka_over(A, row0 + min(r, rows - 1)); };
            auto low  = [&](int r) { return max(0, high(r) - ka_window(A) + 1); };

#pragma unroll 1
            for (int p0 = 0; p0 < pages; p0 += KA_FOLD) {
#pragma unroll 1
            for (int i = p0; i < min(p0 + KA_FOLD, pages) && ok; i++) {
                const int key0 = (at.first + at.p + i) * KV4_P;
                const bool in = there >> st & 1;
                const uint32_t kst = st, kph = ph;
                if (++st == NST) { st = 0; ph ^= 1; }
                const uint32_t vst = st, vph = ph;
                if (++st == NST) { st = 0; ph ^= 1; }
                uint8_t * kp = ring + kst * C::HALF, * vp = ring + vst * C::HALF;
                ok = __all_sync(0xffffffffu, ka_wait(bar0 + kst * 8, kph, abort_s));
                if (!ok) break;
                if (!in) {                                       // no page: nothing was copied
                    issue();
                    ok = __all_sync(0xffffffffu, ka_wait(bar0 + vst * 8, vph, abort_s));
                    if (ok) issue();
                    continue;
                }
                const bool edge = key0 < all_lo || key0 + KV4_P - 1 > all_hi;
#pragma unroll 1
                for (int kb = 0; kb < KV4_P; kb += C::KB) {
                    float S[C::KB / 16][NR][4];                  // keys g and g + 8 of 16, rows 2 t and 2 t + 1
#pragma unroll
                    for (int j = 0; j < C::KB / 16; j++) {
                        uint32_t wv[2][C::W];
                        __half2  d2[2], m2[2];
                        float    rest[C::SPLIT ? NR : 1][4];     // of fp32 rows: the tensor core cuts what it adds to a sum, so small products have one of their own
#pragma unroll
                        for (int x = 0; x < 2; x++) {
                            const int r = kb + j * 16 + x * 8 + g;
                            const __half2 dm = *reinterpret_cast<const __half2 *>(kp + kv4_steps(D) + (r * C::W + (t * C::W >> 2)) * 4);
                            d2[x] = kv4_keep(__low2half2(dm)); m2[x] = kv4_keep(__high2half2(dm));
                            if constexpr (D == 128) { const uint4 v = *reinterpret_cast<const uint4 *>(kp + r * 64 + t * 16); wv[x][0] = v.x; wv[x][1] = v.y; wv[x][2] = v.z; wv[x][3] = v.w; }
                            else                    { const uint2 v = *reinterpret_cast<const uint2 *>(kp + r * 32 + t * 8); wv[x][0] = v.x; wv[x][1] = v.y; }
                        }
#pragma unroll
                        for (int w = 0; w < C::W; w++) {
                            uint32_t o[2][4];
#pragma unroll
                            for (int x = 0; x < 2; x++) kv4_pairs(wv[x][w], d2[x], m2[x], o[x]);
#pragma unroll
                            for (int n = 0; n < NR; n++)
#pragma unroll
                                for (int e = 0; e < 2; e++)
#pragma unroll
                                    for (int pt = 0; pt < C::PARTS; pt++) {
                                        const uint2 b = C::QS ? qsm[((n * C::PARTS + pt) * C::KS + 2 * w + e) * 32] : qf[C::QS ? 0 : pt][C::QS ? 0 : 2 * w + e];
                                        float (&to)[4] = pt ? rest[C::SPLIT ? n : 0] : S[j][n];
                                        if (w == 0 && e == 0) ka_mma0(to, o[0][0], o[1][0], o[0][1], o[1][1], b);
                                        else ka_mma(to, o[0][2 * e], o[1][2 * e], o[0][2 * e + 1], o[1][2 * e + 1], b);
                                    }
                        }
                        if (C::SPLIT)
#pragma unroll
                            for (int n = 0; n < NR; n++)
#pragma unroll
                                for (int c = 0; c < 4; c++) S[j][n][c] += rest[C::SPLIT ? n : 0][c];
                    }
                    if (kb == 0) {
                        ok = __all_sync(0xffffffffu, ka_wait(bar0 + vst * 8, vph, abort_s));
                        if (!ok) break;
                    }
                    if (kb + C::KB == KV4_P) {                   // the keys have been read
                        __syncwarp();
                        issue();
                    }
                    if (edge) {
#pragma unroll
                        for (int n = 0; n < NR; n++)
#pragma unroll
                            for (int r = 0; r < 2; r++) {
                                const int a = low(n * 8 + 2 * t + r) - key0 - kb - g, b = high(n * 8 + 2 * t + r) - key0 - kb - g;
#pragma unroll
                                for (int j = 0; j < C::KB / 16; j++)
#pragma unroll
                                    for (int x = 0; x < 2; x++) if (j * 16 + x * 8 < a || j * 16 + x * 8 > b) S[j][n][2 * x + r] = -INFINITY;
                            }
                        if (kb == 0) {
                            // values that are none, on a page of which some row does not see all: the rows that see one are none in the channels of its group, and it takes part as zeros
                            bool bad = false;
#pragma unroll 1
                            for (int k = lane; k < KV4_P * C::W; k += 32) bad |= __hisnan(__high2half(*reinterpret_cast<const __half2 *>(vp + kv4_steps(D) + k * 4)));
                            if (__any_sync(0xffffffffu, bad)) {
#pragma unroll
                                for (int n = 0; n < NR; n++)
#pragma unroll
                                    for (int r = 0; r < 2; r++) {
                                        const int a = low(n * 8 + 2 * t + r) - key0, b = high(n * 8 + 2 * t + r) - key0;
                                        bool sees = false;
#pragma unroll 1
                                        for (int k = max(a, 0); k <= min(b, KV4_P - 1); k++)
                                            sees |= __hisnan(__high2half(*reinterpret_cast<const __half2 *>(vp + kv4_steps(D) + (kv4_row(k) * C::W + (g * C::W >> 3)) * 4)));
                                        if (sees)
#pragma unroll
                                            for (int i3 = 0; i3 < C::MT; i3++) { O[n][i3][r] = __uint_as_float(0x7fc00000u); O[n][i3][2 + r] = __uint_as_float(0x7fc00000u); }
                                    }
                                __syncwarp();
#pragma unroll 1
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
                    uint2 P[C::KB / 16][NR][2];              // and what fp16 took away of them
#pragma unroll
                    for (int n = 0; n < NR; n++) {
                        float top[2];
#pragma unroll
                        for (int r = 0; r < 2; r++) {
                            top[r] = fmaxf(S[0][n][r], S[0][n][2 + r]);
#pragma unroll
                            for (int j = 1; j < C::KB / 16; j++) top[r] = fmaxf(top[r], fmaxf(S[j][n][r], S[j][n][2 + r]));
                        }
#pragma unroll
                        for (int o = 4; o < 32; o <<= 1) { top[0] = fmaxf(top[0], __shfl_xor_sync(0xffffffffu, top[0], o)); top[1] = fmaxf(top[1], __shfl_xor_sync(0xffffffffu, top[1], o)); }
                        top[0] *= qs[n][0]; top[1] *= qs[n][1];
                        if (__any_sync(0xffffffffu, top[0] > m[n][0] + ka_lazy<C::SPLIT> || top[1] > m[n][1] + ka_lazy<C::SPLIT>)) {
                            float a[2];
#pragma unroll
                            for (int r = 0; r < 2; r++) {
                                const float mn = top[r] > m[n][r] + ka_lazy<C::SPLIT> ? top[r] : m[n][r];
                                a[r] = mn == m[n][r] ? 1.f : ka_exp2(m[n][r] - mn);
                                m[n][r] = mn;
                                l[n][r] *= a[r];
                            }
#pragma unroll
                            for (int i3 = 0; i3 < C::MT; i3++) { O[n][i3][0] *= a[0]; O[n][i3][1] *= a[1]; O[n][i3][2] *= a[0]; O[n][i3][3] *= a[1]; }
                            if (!C::SPLIT) huge = (huge & ~(1 << n)) | (__any_sync(0xffffffffu, fmaxf(fabsf(m[n][0]), fabsf(m[n][1])) > KA_HUGE) ? 1 << n : 0);
                        }
                        float q0 = qs[n][0], q1 = qs[n][1];
                        if (!C::SPLIT && (huge >> n & 1)) {
#pragma unroll
                            for (int j = 0; j < C::KB / 16; j++) { S[j][n][0] *= q0; S[j][n][1] *= q1; S[j][n][2] *= q0; S[j][n][3] *= q1; }
                            q0 = q1 = 1.f;
                        }
                        const float base0 = ka_base<C::SPLIT>(m[n][0]), base1 = ka_base<C::SPLIT>(m[n][1]);
#pragma unroll
                        for (int j = 0; j < C::KB / 16; j++) {
                            uint32_t h[2], r[2];
#pragma unroll
                            for (int x = 0; x < 2; x++) {
                                const float a = ka_exp2(fmaf(S[j][n][2 * x], q0, base0)), b = ka_exp2(fmaf(S[j][n][2 * x + 1], q1, base1));
                                l[n][0] += a; l[n][1] += b;
                                h[x] = ka_pack(a, b);
                                r[x] = ka_turn(ka_rest(a, b, h[x]));
                                h[x] = ka_turn(h[x]);
                            }
                            P[j][n][0] = make_uint2(h[0], h[1]);
                            P[j][n][1] = make_uint2(r[0], r[1]);
                        }
                    }
                    // ---- outputs
#pragma unroll
                    for (int j = 0; j < C::KB / 16; j++) {
                        uint32_t a[2][C::W / 2], b[2][C::W / 2];               // this lane's channels of keys 2 t and 2 t + 1 of both groups of eight
                        __half2  d2[2], m2[2];
#pragma unroll
                        for (int f = 0; f < 2; f++) {
                            const int ra = kb + j * 16 + f * 8 + t, rb = ra + 4;               // kv4_row of the places 2 t and 2 t + 1
                            const __half2 da = *reinterpret_cast<const __half2 *>(vp + kv4_steps(D) + (ra * C::W + (g * C::W >> 3)) * 4);
                            const __half2 db = *reinterpret_cast<const __half2 *>(vp + kv4_steps(D) + (rb * C::W + (g * C::W >> 3)) * 4);
                            d2[f] = kv4_keep(__lows2half2(da, db)); m2[f] = kv4_keep(__highs2half2(da, db));
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
                                // rows g and g + 8 of a product are two neighbouring channels
#pragma unroll
                                for (int n = 0; n < NR; n++)
#pragma unroll
                                    for (int c = 0; c < 2; c++) {
                                        float (&to)[4] = O[n][w * 4 + e * 2 + c];
                                        if (C::SPLIT) {          // the rests' product, while the sum is small; then fp32 adds, with rounding
                                            float own[4];
                                            ka_mma0(own, x[2 * c], x[2 * c + 1], y[2 * c], y[2 * c + 1], P[j][n][1]);
                                            ka_mma(own, x[2 * c], x[2 * c + 1], y[2 * c], y[2 * c + 1], P[j][n][0]);
#pragma unroll
                                            for (int k = 0; k < 4; k++) to[k] += own[k];
                                        } else {
                                            ka_mma(to, x[2 * c], x[2 * c + 1], y[2 * c], y[2 * c + 1], P[j][n][1]);
                                            ka_mma(to, x[2 * c], x[2 * c + 1], y[2 * c], y[2 * c + 1], P[j][n][0]);
                                        }
                                    }
                            }
                    }
                }
                if (!ok) break;
                __syncwarp();
                issue();                                         // the values have been read
            }
            if (!ok) break;
            const bool last = p0 + KA_FOLD >= pages;
            if (p0 > 0 || !last) {                               // what has left the registers, relative to the maxima of then (they never fall), and this portion's
                float4 * sums = reinterpret_cast<float4 *>(A.sums) + (int64_t) (blockIdx.x * C::WARPS + warp) * C::SUMS + lane;
#pragma unroll
                for (int n = 0; n < NR; n++) {
                    float4 * ml = sums + (NR * C::MT + n) * 32;
                    float4   before = make_float4(m[n][0], m[n][1], 0.f, 0.f), e = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (p0 > 0) { before = *ml; if (C::SPLIT) e = ml[C::REST]; }
                    const float f0 = before.x == m[n][0] ? 1.f : ka_exp2(before.x - m[n][0]), f1 = before.y == m[n][1] ? 1.f : ka_exp2(before.y - m[n][1]);
                    e.x *= f0; e.y *= f1;
                    l[n][0] = ka_sum(before.z * f0, l[n][0], e.x); l[n][1] = ka_sum(before.w * f1, l[n][1], e.y);
                    if (last) { if (C::SPLIT) { l[n][0] += e.x; l[n][1] += e.y; } }
                    else { *ml = make_float4(m[n][0], m[n][1], l[n][0], l[n][1]); if (C::SPLIT) ml[C::REST] = e; l[n][0] = l[n][1] = 0.f; }
#pragma unroll
                    for (int k = 0; k < C::MT; k++) {
                        float4 * at = sums + (n * C::MT + k) * 32;
                        float4   o = make_float4(O[n][k][0], O[n][k][1], O[n][k][2], O[n][k][3]);
                        e = make_float4(0.f, 0.f, 0.f, 0.f);
                        if (p0 > 0) { if (C::SPLIT) e = ka_times(at[C::REST], f0, f1); o = ka_sum(ka_times(*at, f0, f1), o, e); }
                        if (!last) { *at = o; if (C::SPLIT) at[C::REST] = e; o = e = make_float4(0.f, 0.f, 0.f, 0.f); }
                        O[n][k][0] = o.x; O[n][k][1] = o.y; O[n][k][2] = o.z; O[n][k][3] = o.w;
                        if (C::SPLIT) { O[n][k][0] += e.x; O[n][k][1] += e.y; O[n][k][2] += e.z; O[n][k][3] += e.w; }
                    }
                }
            }
            }
            if (!ok) break;
            // ---- rows out: lane (g, t) has D / 8 neighbouring channels of rows 2 t and 2 t + 1 of each tile
#pragma unroll
            for (int n = 0; n < NR; n++)
#pragma unroll
                for (int r = 0; r < 2; r++)
#pragma unroll
                    for (int o = 4; o < 32; o <<= 1) l[n][r] += __shfl_xor_sync(0xffffffffu, l[n][r], o);
            todo -= pages;
            if (whole) {
#pragma unroll
                for (int n = 0; n < NR; n++)
#pragma unroll
                    for (int r = 0; r < 2; r++) {
                        const int ri = n * 8 + 2 * t + r;
                        if (ri >= rows) continue;
                        const float inv = l[n][r] > 0.f ? 1.f / l[n][r] : l[n][r];     // a row that saw nothing: zeros; a sum that is none stays so
                        float v[C::C8];
#pragma unroll
                        for (int c = 0; c < C::C8; c++) v[c] = O[n][c >> 1][2 * (c & 1) + r] * inv;
                        const int rc = row0 + ri, tk = ka_over(A, rc);
                        ka_store<T, C::C8>((T *) A.out + (tok0 + tk) * A.ldo + (int64_t) (at.h * A.rep + rc - tk * A.rep) * D + g * C::C8, ka_here(A.wide_o), v);
                    }
            } else if (at.p + pages == at.np) {
                ends = true;
                ka_leave<C, NR>(A.heads + (int64_t) (blockIdx.x * C::WARPS + warp) * C::PIECE, rows, g, t, O, m, l);
                if (lane == 0) items[warp] = { 0, 0, row0, rows, at.h, tok0 };
            } else { goes = true; begins = at.p == 0; if (lane == 0) last_item[warp] = { 0, 0, row0, rows, at.h, tok0 }; }
            at.p += pages - 1;
            if (todo) ka_next<C::RT>(A, prefix, seq_of, at);
        }
    }
    if (lane == 0) flags[warp] = (ends ? 1 : 0) | (goes ? 2 : 0) | (begins ? 4 : 0);
    __syncthreads();                                                 // nobody reads a ring or queries any more
    float * pieces = reinterpret_cast<float *>(ka_dsm);
    if (goes) ka_leave<C, NR>(pieces + warp * C::PIECE, C::RT, g, t, O, m, l);
    __syncthreads();
    if (!*abort_s && c0 < c1) {
        // Chains of pieces: each ends with the piece of a warp whose item ends there, the last one goes on behind the block.  A row of a chain a warp, lanes its channels: maxima and sums of the pieces a lane
        // each, then their rows; loads wait for nothing but these
        constexpr int CH = D / 32;
        const int fl = lane < C::WARPS ? flags[lane] : 0;
        const uint32_t all_ends = __ballot_sync(0xffffffffu, fl & 1), all_goes = __ballot_sync(0xffffffffu, fl & 2), all_begins = __ballot_sync(0xffffffffu, fl & 4);
        int my_end = C::WARPS;                                       // of the chain that has the lane's number; the last chain: none
        { uint32_t b = all_ends;
#pragma unroll 1
            for (int k = 0; b; k++, b &= b - 1) if (k == lane) my_end = __ffs(b) - 1; }
        constexpr int MANY = NR == 1 ? 1 : NR == 2 ? 2 : 4;                        // neighbouring rows of a chain at a time
        const int tasks = (__popc(all_ends) + 1) * C::RT;
#pragma unroll 1
        for (int task0 = warp * MANY; task0 < tasks; task0 += C::WARPS * MANY) {
            const int r0 = task0 % C::RT, chain = task0 / C::RT, from = __shfl_sync(0xffffffffu, my_end, max(chain - 1, 0) & 31), end = __shfl_sync(0xffffffffu, my_end, chain & 31);
            // pieces in shared memory (the warp where the chain before ends may begin this one); the one of warp `end` is in scratch
            const uint32_t span = ((1u << end) - 1) & ~((1u << (chain ? from : 0)) - 1), mine = all_goes & span;
            const bool ours = (all_begins & span) != 0, closed = end < C::WARPS, take = (mine >> lane & 1) || (closed && lane == end);
            const int  n = min(MANY, closed ? items[end].rows - r0 : mine ? MANY : 0);       // (rows of an open chain that are none are read by nobody)
            if (n <= 0) continue;
            const float * last = A.heads + (int64_t) (blockIdx.x * C::WARPS + (closed ? end : 0)) * C::PIECE, * p = closed && lane == end ? last : pieces + lane * C::PIECE;
            float ao[MANY][CH], f[MANY], am[MANY], al[MANY];
#pragma unroll
            for (int k = 0; k < MANY; k++) {
                const int ri = r0 + min(k, n - 1);
                if (closed) ka_get(last + ri * D + lane * CH, ao[k]);
                else
#pragma unroll
                    for (int c = 0; c < CH; c++) ao[k][c] = 0.f;
                am[k] = take ? p[C::RT * D + ri] : -INFINITY;
                al[k] = take ? p[C::RT * D + C::RT + ri] : 0.f;
            }
#pragma unroll
            for (int k = 0; k < MANY; k++) {
                const float pm = am[k];
                am[k] = warp_max(pm);
                f[k]  = pm == am[k] ? 1.f : exp2f(pm - am[k]);
                al[k] = warp_sum(al[k] * f[k]);
                const float fe = __shfl_sync(0xffffffffu, f[k], end & 31);
#pragma unroll
                for (int c = 0; c < CH; c++) ao[k][c] *= closed ? fe : 0.f;
            }
#pragma unroll 1
            for (uint32_t rest = mine; rest; rest &= rest - 1) {
                const int w = __ffs(rest) - 1;
#pragma unroll
                for (int k = 0; k < MANY; k++) {
                    const float fw = __shfl_sync(0xffffffffu, f[k], w);
                    float v[CH];
                    ka_get(pieces + w * C::PIECE + (r0 + min(k, n - 1)) * D + lane * CH, v);
#pragma unroll
                    for (int c = 0; c < CH; c++) ao[k][c] = fmaf(v[c], fw, ao[k][c]);
                }
            }
            float * q = A.pieces + (int64_t) (2 * blockIdx.x + (ours ? 1 : 0)) * C::PIECE;
#pragma unroll
            for (int k = 0; k < MANY; k++) {
                if (k >= n) break;
                const int ri = r0 + k;
                if (closed && ours) ka_row_out<T, D>(A, items[end], ri, lane, ao[k], al[k]);
                else {
                    ka_put(q + ri * D + lane * CH, ao[k]);
                    if (lane == 0) { q[C::RT * D + ri] = am[k]; q[C::RT * D + C::RT + ri] = al[k]; }
                }
            }
        }
    }
    // the last warp with units knows whether the run's last item goes on
    if (blockIdx.x < runs && u1 == c1 && u0 < u1 && lane == 0) {
        ka_open o = last_item[warp];
        bool ours = begins;                                          // of a chain through several warps: where it began
#pragma unroll 1
        for (int w = warp - 1; w >= 0 && !ours; w--) {               // (warps without units in between have no flags)
            if (flags[w] & 4) ours = true;
            if (flags[w] & 1) break;
        }
        o.runs = goes && ours;
        o.last = goes ? (int) ((ka_work<C::RT, C::EXTRA>(A, prefix, count, seq_of, at) * runs + U - 1) / U - 1) : 0;
        A.open[blockIdx.x] = o;
    }
    if (threadIdx.x == 0 && c0 >= c1) A.open[blockIdx.x].runs = 0;
    __syncthreads();
    if (*abort_s) {                                              // a wait ran out: say so, give copies still in flight time to land (bounded)
        if (threadIdx.x == 0) atomicExch(A.err, 1 + (int) blockIdx.x);
#pragma unroll 1
        for (int i = 0; i < 2000; i++) __nanosleep(1000);
    }
}

// Blocks (run, tile of eight rows): an item that begins in the run and does not end there gets its pieces' sum, a row a warp, lanes its channels.
template <typename T, int D, int NR>
static __global__ void __launch_bounds__(256) kv4_join_kernel(const __grid_constant__ ka_args A) {
    using C = ka_cfg<T, D, NR>;
    constexpr int CH = D / 32;
    pib_pdl_wait();
    pib_pdl_trigger();
    const int     lane = threadIdx.x & 31, wa = blockIdx.x, ri = blockIdx.y * 8 + (threadIdx.x >> 5);
    const ka_open it = A.open[wa];
    if (!it.runs || ri >= it.rows) return;
    float m = -INFINITY, l = 0.f, o[CH];
#pragma unroll
    for (int c = 0; c < CH; c++) o[c] = 0.f;
    auto piece = [&](int w) { return A.pieces + (2 * w + (w == wa ? 1 : 0)) * (int64_t) C::PIECE; };
    // 32 pieces at a time: their maxima and sums, a piece a lane, then their rows, whose loads wait for nothing
    for (int w0 = wa; w0 <= it.last; w0 += 32) {
        const int n = min(32, it.last - w0 + 1);
        float pm = -INFINITY, pl = 0.f;
        if (lane < n) { pm = piece(w0 + lane)[C::RT * D + ri]; pl = piece(w0 + lane)[C::RT * D + C::RT + ri]; }
        const float mn = fmaxf(m, warp_max(pm)), a = m == mn ? 1.f : exp2f(m - mn), f = pm == mn ? 1.f : exp2f(pm - mn);
        m = mn; l = l * a + warp_sum(lane < n ? pl * f : 0.f);
#pragma unroll
        for (int c = 0; c < CH; c++) o[c] *= a;
#pragma unroll 8
        for (int k = 0; k < n; k++) {
            const float * p = piece(w0 + k) + ri * D;
            const float   fk = __shfl_sync(0xffffffffu, f, k);
            float v[CH];
            ka_get(p + lane * CH, v);
#pragma unroll
            for (int c = 0; c < CH; c++) o[c] = fmaf(v[c], fk, o[c]);
        }
    }
    ka_row_out<T, D>(A, it, ri, lane, o, l);
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

// Rows (token, head of the group) of the longest portion: more than these go on tcgen05, which takes 256 rows in the time of one.  us here (a walk over the keys for each 32 rows, fp32 16) and there:
//   16 x 3,000 keys: bfloat16 32 rows 64 / 92, 48 rows 101 / 93; fp32 48 rows 108 / 127, 64 rows 138 / 128.  60,000 keys: bfloat16 71 / 109, 114 / 110; fp32 124 / 143, 162 / 144
static int ka_few(int type) { return type == PIB_TYPE_F32 ? 48 : 32; }
static int64_t ka_rows(const pib_kv4 * kv, const pib_kv4_batch * b) { return (int64_t) (b->max_tokens ? std::min(b->max_tokens, b->tokens) : b->tokens) * (b->heads / kv->heads); }
// tiles of eight rows that a warp takes at once; four only of bfloat16, whose queries' operands are half as large
static int ka_tiles_of(const pib_kv4 * kv, const pib_kv4_batch * b) { const int64_t r = ka_rows(kv, b); return r <= 8 ? 1 : r <= 16 || b->type == PIB_TYPE_F32 ? 2 : 4; }
// the scratch: two pieces a block; decode: one of each warp and the sums that have left its registers, prompts: a block's sums; then the tables
struct ka_space { size_t heads, sums, plan, open, total; };
static ka_space ka_space_of(const pib_kv4 * kv, const pib_kv4_batch * b) {
    const int    n = ka_tiles_of(kv, b), sms = pib_num_sms();
    const bool   few = ka_rows(kv, b) <= ka_few(b->type);
    const size_t piece = (size_t) (few ? n * 8 : KP_ROWS) * (kv->dim + 2) * 4;
    auto up = [](size_t v) { return (v + 255) & ~(size_t) 255; };
    ka_space s;
    s.heads = up(2 * sms * piece);
    s.sums  = s.heads + (few ? up((size_t) sms * KA_WARPS * piece) : 0);
    s.plan  = s.sums + up((size_t) sms * (few ? (size_t) KA_WARPS * n * (kv->dim / 16 + 1) * (b->type == PIB_TYPE_F32 ? 1024 : 512) : kp_sums(b->type == PIB_TYPE_F32, kv->dim) * 4));
    s.open  = s.plan + up(sizeof(ka_plan));
    s.total = s.open + up(sms * sizeof(ka_open));
    return s;
}
extern "C" size_t pib_kv4_attn_scratch_bytes(const pib_kv4 * kv, const pib_kv4_batch * b) {
    if (ka_batch_ok("pib_kv4_attn_scratch_bytes", kv, b) != PIB_OK) return 0;
    return ka_space_of(kv, b).total;
}

template <typename T, int D, int NR> static int ka_go(ka_args A, cudaStream_t st) {
    using C = ka_cfg<T, D, NR>;
    const size_t table = ((size_t) (A.seqs + 1) * 12 + (size_t) A.seqs * sizeof(ka_seq) + 127) & ~(size_t) 127;
    constexpr size_t most = 224 * 1024;
    A.stages = (int) std::min<size_t>(8, (most - C::Q_BYTES - table) / (C::WARPS * C::HALF));
    static_assert((most - C::Q_BYTES - (PIB_KV4_MAX_SEQS + 1) * 12 - PIB_KV4_MAX_SEQS * sizeof(ka_seq) - 128) / (C::WARPS * C::HALF) >= 2, "keys and values of a page");
    static_assert(C::PIECE * 4 <= 2 * C::HALF + C::Q_BYTES / C::WARPS, "pieces in the rings' and queries' place");
    static_assert(C::SUMS * 16 == NR * (D / 16 + 1) * (C::SPLIT ? 1024 : 512), "sums in the scratch");
    static pib_per_device attrs;
    PIB_CHECK(attrs.once([&] { return cudaFuncSetAttribute(kv4_decode_kernel<T, D, NR>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int) most); }));
    PIB_CHECK(pib_launch(kv4_decode_kernel<T, D, NR>, dim3((unsigned) pib_num_sms()), dim3(C::WARPS * 32), (size_t) C::WARPS * A.stages * C::HALF + C::Q_BYTES + table, st, A));
    PIB_CHECK(pib_launch(kv4_join_kernel<T, D, NR>, dim3((unsigned) pib_num_sms(), NR), dim3(256), 0, st, A));
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
    A.base = kv->base; A.pages = kv->pages; A.kvh = kv->heads; A.rep = b->heads / kv->heads; A.dim = kv->dim; A.part = (1u << 21) / A.rep + 1;
    A.starts = starts; A.lens = lens; A.table = pages; A.tokens = b->tokens; A.seqs = b->seqs; A.max_pages = b->max_pages; A.window = b->window; A.scale = b->scale;
    A.q = q; A.out = out; A.ldq = ldq; A.ldo = ldo;
    A.wide_q = ((uintptr_t) q & 15) == 0 && ldq * size % 16 == 0;
    A.wide_o = ((uintptr_t) out & 15) == 0 && ldo * size % 16 == 0;
    const ka_space sp = ka_space_of(kv, b);
    uint8_t * sc = (uint8_t *) scratch;
    A.pieces = (float *) sc; A.heads = (float *) (sc + sp.heads); A.sums = (float *) (sc + sp.sums); A.plan = (ka_plan *) (sc + sp.plan); A.open = (ka_open *) (sc + sp.open);
    A.stages = 0;
    if (!(A.err = pib_tc_error_word((cudaStream_t) s))) { pib_set_error("pib_kv4_attn: no memory for the error word"); return PIB_ERR_NOMEM; }
    const cudaStream_t st = (cudaStream_t) s;
    if (ka_rows(kv, b) > ka_few(b->type)) return pib_kv4_prompt(A, size == 4, st);
    const int n = ka_tiles_of(kv, b);
    if (size == 4) {
        if (kv->dim == 64) return n == 1 ? ka_go<float, 64, 1>(A, st) : ka_go<float, 64, 2>(A, st);
        return n == 1 ? ka_go<float, 128, 1>(A, st) : ka_go<float, 128, 2>(A, st);
    }
    if (kv->dim == 64) return n == 1 ? ka_go<__nv_bfloat16, 64, 1>(A, st) : n == 2 ? ka_go<__nv_bfloat16, 64, 2>(A, st) : ka_go<__nv_bfloat16, 64, 4>(A, st);
    return n == 1 ? ka_go<__nv_bfloat16, 128, 1>(A, st) : n == 2 ? ka_go<__nv_bfloat16, 128, 2>(A, st) : ka_go<__nv_bfloat16, 128, 4>(A, st);
}
