// kv4_prompt.cu -- attention of portions of prompts over a key / value cache in 4 bits (kv4.cuh) on tcgen05, scores, weights and outputs in tensor memory.
//
// A block takes 256 rows (token, head of the group) of one key / value head as two groups of 128 and walks the pages they see; pages of all such items lie in one row that the blocks of the GPU (one an
// SM) divide evenly, whatever the sequences' lengths (kv4_attn.cuh).  An item that lies in one block's run is written at once; pieces of others go to scratch and kv4_prompt_join_kernel adds them up.
//   warp 2        writes down the run's items
//   warp 0        brings pages' records (keys and values in 4 bits) by bulk copies through a ring
//   warps 4..7    write two pages' keys [128][dim] and their values, turned, [dim][128] as fp16 into tiles of the 128-byte swizzle
//   warp 1        issues the MMAs: a group's O += P V when its weights are there, its scores S = Q K' of the next two pages when that product is done; then the other group's, while the first forms weights
//   warps 8..15   a thread owns a row: scores from tensor memory, mask, running maximum (it moves once 2^ka_lazy behind), weights as fp16 into the scores' place, from where they enter the second product
// The tensor core cuts off what it adds to a sum instead of rounding it, always towards zero, some 2^-24 of it each time: of fp32 rows the rests' products come first, while the sum is small, and the outputs'
// sums go to scratch every FOLD steps (fp32: 256 keys, bfloat16: 4,096), are added there with rounding, and begin anew; of fp32 rows those go on to a second sum, with compensation, every KP_FOLDS times.
// Outputs of long items that a block takes whole, all values one: fp32 within 4.2e-7 behind 64,000 keys and a million, bfloat16 low by 3e-5 beside their rounding at any length (without: 0.9e-3 behind 131,072
// keys).  fp32 portions of 1,999 and 1,200 tokens of up to 4,100 keys: 700 us without, 868 at 2 steps, 1,065 at 1.  Denominators are added up step by step, with compensation.
// Queries of fp32 rows enter as fp16 part and remainder, two products, those of bfloat16 rows as one fp16 number.  Weights are two products beside either: as one fp16 number they move one of eleven
// bfloat16 outputs to its neighbour (now one of 400), for 478 instead of 540 us (portions of 1,999 tokens of two sequences of up to 4,100 keys, 64 / 8 heads of 128).
// What bounds it: no unit is full; a row's scores, weights and the two products follow one another, and two groups of rows are what tensor memory holds.  The portions above 545 us, in fp32 799; their operations at
// the measured bfloat16 rate 155, at four products for two 310.
// Every wait is bounded (tc_common.cuh).
#include "kv4_attn.cuh"

#include <algorithm>

#define KP_THREADS 512
#define KP_LEAD    8           // an item's start and end, in pages (4, 8, 12: bfloat16 portions of 1,999 and 1,200 tokens 584, 588, 597 us, fp32 878, 868, 883; 32 tokens behind 4,096 keys 36, 36, 42; 1,999 fp32 tokens alone 188, 174, 182)
#define KP_BARS    32
#define KP_FOLDS   16          // fp32 rows: times after which the sums in scratch go on to a second one (an addition of less than 2^-25 of a sum is lost: behind one large weight those of up to 4,096 keys)

// an item, or the piece of it in a run: its rows, pages [page, page + pages) of its sequence; keys hi and below, lo and above all its rows see; whether that is all of it, where its piece goes
struct kp_item { int s, h, row0, rows, tok0, pos0, page, pages, hi, lo, whole, slot; };
#define KP_ITEMS 4

template <typename T, int D> struct kp_cfg {
    static constexpr bool SPLIT = sizeof(T) == 4;
    static constexpr int  W = D / 32, NC = D / 64, STG = SPLIT ? 1 : 2;               // groups; 64-wide column chunks of a head; tiles of keys and of values
    static constexpr int  FOLD = SPLIT ? 2 : 32;                                     // steps after which the outputs' sums leave tensor memory
    static constexpr int  Q_CHUNK = 128 * 128, Q_PART = 2 * NC * Q_CHUNK;            // both groups' rows: [group][chunk][128 rows][128 bytes]
    static constexpr int  Q_BYTES = Q_PART * (SPLIT ? 2 : 1), K_CHUNK = 128 * 128, K_TILE = NC * K_CHUNK, V_CHUNK = D * 128, V_TILE = 2 * V_CHUNK;
    static constexpr int  TILES = Q_BYTES + STG * (K_TILE + V_TILE), REC = kv4_record(D);
    static constexpr int  PIECE = KP_ROWS * (D + 2);                                 // floats
    static constexpr size_t FIXED = (size_t) TILES + KP_BARS * 8 + 512 + 1024;          // without records and the table
};

// A in tensor memory, B in shared memory; called by a converged warp
__device__ __forceinline__ void kp_mma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p, q;\n\telect.sync _|q, 0xffffffff;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n\t}"
                 ::"r"(tmem_d), "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(0u) : "memory");
}
__device__ __forceinline__ void kp_st16(uint32_t taddr, const uint32_t * v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
                 ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]),
                   "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]) : "memory");
}
__device__ __forceinline__ void kp_add(float4 & o, float4 a, float f) { o.x = fmaf(a.x, f, o.x); o.y = fmaf(a.y, f, o.y); o.z = fmaf(a.z, f, o.z); o.w = fmaf(a.w, f, o.w); }
// fp16 x fp16, fp32 accumulators, both K-major, M x N outputs
__host__ __device__ constexpr uint32_t kp_idesc(int M, int N) { return (1u << 4) | ((uint32_t) (N >> 3) << 17) | ((uint32_t) (M >> 4) << 24); }

// N neighbouring values of a row in registers
template <typename T, int N> struct kp_row {
    uint32_t r[N * sizeof(T) / 4];
    __device__ __forceinline__ void load(const T * p, bool wide) {
        if (wide) {
#pragma unroll
            for (int i = 0; i < (int) (N * sizeof(T) / 16); i++) { const uint4 f = reinterpret_cast<const uint4 *>(p)[i]; r[4 * i] = f.x; r[4 * i + 1] = f.y; r[4 * i + 2] = f.z; r[4 * i + 3] = f.w; }
        } else if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < N; i++) r[i] = __float_as_uint(p[i]);
        } else {
#pragma unroll
            for (int i = 0; i < N / 2; i++) r[i] = (uint32_t) __bfloat16_as_ushort(p[2 * i]) | (uint32_t) __bfloat16_as_ushort(p[2 * i + 1]) << 16;
        }
    }
    __device__ __forceinline__ float at(int i) const { return sizeof(T) == 4 ? __uint_as_float(r[i]) : __uint_as_float(i & 1 ? r[i / 2] & 0xffff0000u : r[i / 2] << 16); }
    __device__ __forceinline__ float top() const {
        float m = 0.f;
#pragma unroll
        for (int i = 0; i < N; i++) m = fmaxf(m, fabsf(at(i)));
        return m;
    }
};

template <typename T, int D>
__global__ void __launch_bounds__(KP_THREADS, 1) kv4_prompt_kernel(const __grid_constant__ ka_args A) {
    using C = kp_cfg<T, D>;
    extern __shared__ __align__(1024) uint8_t kp_dsm[];
    uint8_t *  sQ   = kp_dsm + ((1024u - (dt_smem(kp_dsm) & 1023u)) & 1023u);
    const int  RAW = A.stages;                                   // records under way: 2 or 3
    uint8_t *  sK   = sQ + C::Q_BYTES, * sV = sK + C::STG * C::K_TILE, * raw = sV + C::STG * C::V_TILE;
    uint64_t * bar  = reinterpret_cast<uint64_t *>(raw + RAW * C::REC);
    uint32_t * tmem_slot = reinterpret_cast<uint32_t *>(bar + KP_BARS);
    volatile int * abort_s = reinterpret_cast<volatile int *>(tmem_slot + 1);
    volatile int * raw_in = reinterpret_cast<volatile int *>(tmem_slot + 2);         // [RAW] whether the record's page is one of the cache's
    volatile unsigned long long * v_none = reinterpret_cast<volatile unsigned long long *>(tmem_slot + 12);      // [STG][2][W] places of a page whose values are none, of each group
    int64_t *  prefix = reinterpret_cast<int64_t *>(reinterpret_cast<uint8_t *>(bar) + KP_BARS * 8 + 512);       // [seqs + 1]
    __shared__ int64_t part[KP_THREADS / 32];
    // barriers: records there / read; key tiles written / read, value tiles written / read; of each group queries written, scores there, weights written, product done
    kp_item *  list = reinterpret_cast<kp_item *>(tmem_slot + 48);                   // [KP_ITEMS]
    const uint32_t b0 = dt_smem(bar), bar_if = b0 + 192, bar_ie = b0 + 224, bar_rf = b0, bar_re = b0 + 32, bar_kf = b0 + 64, bar_ke = b0 + 80, bar_vf = b0 + 96, bar_ve = b0 + 112, bar_q = b0 + 128, bar_s = b0 + 144, bar_p = b0 + 160, bar_o = b0 + 176;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < RAW; i++) { dt_mbar_init(bar_rf + 8 * i, 1); dt_mbar_init(bar_re + 8 * i, 4); }
        // an item has been taken by the loader, the issuer, four warps of tiles and eight of rows
        for (int i = 0; i < KP_ITEMS; i++) { dt_mbar_init(bar_if + 8 * i, 1); dt_mbar_init(bar_ie + 8 * i, 14); }
        for (int i = 0; i < 2; i++) {
            dt_mbar_init(bar_kf + 8 * i, 4); dt_mbar_init(bar_vf + 8 * i, 4);
            for (uint32_t b : { bar_ke, bar_ve, bar_s, bar_o }) dt_mbar_init(b + 8 * i, 1);
            dt_mbar_init(bar_q + 8 * i, 4); dt_mbar_init(bar_p + 8 * i, 4);
        }
        *abort_s = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dt_smem(tmem_slot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    pib_pdl_wait();
    pib_pdl_trigger();
    dt_fence_before();
    const int64_t U = ka_prefix<KP_ROWS, KP_LEAD, KP_THREADS, ka_seq_none>(A, prefix, part, {});
    dt_fence_after();
    // (runs of less than an item's start and end are not worth their pieces)
    const int64_t runs = min((int64_t) gridDim.x, (U + KP_LEAD - 1) / KP_LEAD), me = blockIdx.x;
    ka_leave_plan<KP_THREADS>(A, prefix, runs);
    const uint32_t tmem = *tmem_slot, tm_o = tmem + 256;          // columns: scores of two pages, 64 each, of both groups; the weights take their scores' place; outputs 256..383 and 384..511
    ka_zero_rows<KP_ROWS, KP_THREADS, T>(A, ka_seq_call{ &A }, D);
    const int64_t u0 = me < runs ? U * me / runs : 0, u1 = me < runs ? U * (me + 1) / runs : 0;
    // whether some row of the item does not see all of a page
    auto edge_of = [&](const kp_item & it, int key0) { return key0 < it.lo || key0 + KV4_P - 1 > it.hi; };
    // a role takes the run's items as warp 2 writes them down, until one has no pages: f(item) says whether to go on
    auto items = [&](auto f) {
        int at = 0;
        uint32_t ph = 0;
#pragma unroll 1
        for (;;) {
            if (!__all_sync(0xffffffffu, ka_wait(bar_if + 8 * at, ph, abort_s))) return;
            const kp_item it = list[at];
            __syncwarp();
            if (lane == 0) dt_arrive(bar_ie + 8 * at);
            if (++at == KP_ITEMS) { at = 0; ph ^= 1; }
            if (it.pages == 0 || !f(it)) return;
        }
    };

    // registers go where the rows are: 512 x 128 at launch, 128 x (96 + 112 + 152 + 152) from here
    if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
    if (warp == 0) {
        int st = 0;
        uint32_t ph = 1;                                         // the first round finds its places free
        items([&](const kp_item & it) {
            int ids = 0;
#pragma unroll 1
            for (int i = 0; i < it.pages; i++) {
                const int pg = it.page + i;
                if ((i & 31) == 0) ids = pg + lane < A.max_pages ? A.table[(int64_t) it.s * A.max_pages + pg + lane] : -1;
                const int  id = __shfl_sync(0xffffffffu, ids, i & 31);
                const bool in = id >= 0 && id < A.pages;
                if (!__all_sync(0xffffffffu, ka_wait(bar_re + 8 * st, ph, abort_s))) return false;
                if (lane == 0) {
                    raw_in[st] = in;
                    if (in) {
                        dt_mbar_expect_tx(bar_rf + 8 * st, C::REC);
                        ka_bulk(dt_smem(raw + st * C::REC), A.base + ((int64_t) id * A.kvh + it.h) * C::REC, C::REC, bar_rf + 8 * st);
                    } else dt_arrive(bar_rf + 8 * st);
                }
                if (++st == RAW) { st = 0; ph ^= 1; }
            }
            return true;
        });
    } else if (warp == 2) {
        const ka_seq_call seq_of = { &A };
        int at = 0;
        uint32_t ph = 1;
        auto put = [&](const kp_item & it) {
            if (!__all_sync(0xffffffffu, ka_wait(bar_ie + 8 * at, ph, abort_s))) return false;
            if (lane == 0) { list[at] = it; dt_arrive(bar_if + 8 * at); }
            __syncwarp();
            if (++at == KP_ITEMS) { at = 0; ph ^= 1; }
            return true;
        };
        bool go = true;
        if (u0 < u1) {
            ka_place c = ka_find<KP_ROWS, KP_LEAD>(A, prefix, seq_of, u0);
#pragma unroll 1
            for (int64_t u = u0; u < u1 && go;) {
                const ka_seq q = seq_of(c.s);
                const int    units = (int) min((int64_t) (c.np - c.p), u1 - u), p0 = max(c.p - KP_LEAD, 0), pages = c.p + units - KP_LEAD - p0;
                if (pages > 0) {
                    kp_item it;
                    it.s = c.s; it.h = c.h; it.row0 = c.r * KP_ROWS; it.rows = (int) min((int64_t) KP_ROWS, (int64_t) q.n * A.rep - it.row0);
                    it.tok0 = q.start; it.pos0 = q.len - q.n;
                    it.page = c.first + p0; it.pages = pages;
                    it.hi = it.pos0 + it.row0 / A.rep;
                    it.lo = max(0, it.pos0 + (it.row0 + it.rows - 1) / A.rep - ka_window(A) + 1);
                    it.whole = p0 == 0 && pages == c.np - KP_LEAD; it.slot = p0 > 0 ? 0 : 1;
                    go = put(it);
                }
                u += units;
                c.p += units;
                if (u < u1 && c.p >= c.np) ka_next_item<KP_ROWS, KP_LEAD>(A, prefix, seq_of, c);
            }
        }
        kp_item end = {};
        if (go) put(end);
    } else if (warp == 1) {
        constexpr uint32_t id_o = kp_idesc(128, D);
        const uint64_t dq = dt_desc(dt_smem(sQ)), dk = dt_desc(dt_smem(sK)), dv = dt_desc(dt_smem(sV));
        int      j = 0, n_q[2] = { 0, 0 }, n_p[2] = { 0, 0 };     // steps of two pages; queries and weights that have entered
        auto wait = [&](uint32_t b, uint32_t ph) { return __all_sync(0xffffffffu, ka_wait(b, ph & 1, abort_s)) != 0; };
        auto scores = [&](int w, int jj, int two) {
            const uint32_t id_s = two ? kp_idesc(128, 128) : kp_idesc(128, 64);
            const uint64_t a0 = dq + (uint64_t) (w * C::NC * C::Q_CHUNK >> 4), k0 = dk + (uint64_t) (jj % C::STG * C::K_TILE >> 4);
            dt_fence_after();
#pragma unroll
            for (int r = 0; r < (C::SPLIT ? 2 : 1); r++)                                   // the rests first, while the sum is small
#pragma unroll
                for (int c = 0; c < C::NC; c++)
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        dt_mma(tmem + 128 * w, a0 + (((C::SPLIT ? 1 - r : 0) * C::Q_PART + c * C::Q_CHUNK) >> 4) + 2 * k, k0 + (c * C::K_CHUNK >> 4) + 2 * k, id_s, (r | c | k) != 0);
            dt_commit(bar_s + 8 * w);
        };
        auto outputs = [&](int w, int two, bool add) {
            const uint64_t v0 = dv + (uint64_t) (j % C::STG * C::V_TILE >> 4);
            dt_fence_after();
#pragma unroll 1
            for (int r = 0; r < 2; r++)
#pragma unroll 1
                for (int h = 0; h <= two; h++)
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        kp_mma_ts(tm_o + 128 * w, tmem + 128 * w + 64 * h + 32 - 32 * r + 8 * k, v0 + (uint64_t) (h * C::V_CHUNK >> 4) + 2 * k, id_o, add || (r | h | k) != 0);
            dt_commit(bar_o + 8 * w);
        };
        items([&](const kp_item & it) {
            const int pages = it.pages, groups = it.rows > 128 ? 2 : 1, steps = (pages + 1) / 2;
            if (!wait(bar_kf + 8 * (j % C::STG), j / C::STG)) return false;
            for (int w = 0; w < groups; w++) {
                if (!wait(bar_q + 8 * w, n_q[w]++)) return false;
                scores(w, j, pages > 1);
            }
            dt_commit(bar_ke + 8 * (j % C::STG));
#pragma unroll 1
            for (int i = 0; i < steps; i++, j++) {
                // a group at a time, its next scores right behind its outputs: the other one forms its weights meanwhile.  (Both groups' outputs, then both groups' scores, or a warp for each group's products, take a
                // tenth longer: the groups fall into step, share the exponentials, then wait together)
#pragma unroll 1
                for (int w = 0; w < groups; w++) {
                    if (!wait(bar_p + 8 * w, n_p[w]) || (w == 0 && !wait(bar_vf + 8 * (j % C::STG), j / C::STG))) return false;
                    outputs(w, 2 * i + 1 < pages, i % C::FOLD != 0);
                    n_p[w]++;
                    if (w == groups - 1) dt_commit(bar_ve + 8 * (j % C::STG));
                    if (i + 1 == steps) continue;
                    // (the weights lie where the scores go, and MMAs of different accumulators may overtake each other)
                    if ((w == 0 && !wait(bar_kf + 8 * ((j + 1) % C::STG), (j + 1) / C::STG)) || !wait(bar_o + 8 * w, n_p[w] + 1)) return false;
                    scores(w, j + 1, 2 * i + 3 < pages);
                    if (w == groups - 1) dt_commit(bar_ke + 8 * ((j + 1) % C::STG));
                }
            }
            return true;
        });
    }
    } else if (warp < 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 112;");
        // ---- a page's tiles, by 128 threads
        const int tid = threadIdx.x - 128;
        int       j = 0, st = 0;
        uint32_t  ph = 0;
        items([&](const kp_item & it) {
            const int pages = it.pages;
#pragma unroll 1
            for (int i = 0; i < pages; i += 2, j++) {
                const int two = i + 1 < pages, sg = j % C::STG;
                const uint32_t free_ph = (j / C::STG & 1) ^ 1;
                if (!__all_sync(0xffffffffu, ka_wait(bar_ke + 8 * sg, free_ph, abort_s))) return false;
                int      s1 = st;
                uint32_t p1 = ph;
#pragma unroll 1
                for (int h = 0; h <= two; h++) {
                    // keys: a thread has 32 channels (two times) of one key; of a group's four words the lanes start with different ones, for the banks
                    if (!__all_sync(0xffffffffu, ka_wait(bar_rf + 8 * s1, p1, abort_s))) return false;
                    const bool in = raw_in[s1] != 0;
                    const uint8_t * rec = raw + s1 * C::REC;
                    uint8_t * to = sK + sg * C::K_TILE + h * 64 * 128;
                    const int key = tid & 63, half = tid >> 6;
#pragma unroll
                    for (int x = 0; x < C::W / 2; x++) {
                        const int     cc = D == 128 ? (2 * half + x + (key >> 1)) & 3 : half;
                        const uint4   n = *reinterpret_cast<const uint4 *>(rec + key * (D / 2) + cc * 16);
                        const __half2 dm = *reinterpret_cast<const __half2 *>(rec + kv4_steps(D) + (key * C::W + cc) * 4);
                        const __half2 d2 = kv4_keep(__low2half2(dm)), m2 = kv4_keep(__high2half2(dm));
                        const uint32_t wv[4] = { n.x, n.y, n.z, n.w };
#pragma unroll
                        for (int w = 0; w < 4; w++) {
                            uint32_t o[4];
                            kv4_pairs(wv[w], d2, m2, o);
                            *reinterpret_cast<uint4 *>(to + (cc >> 1) * C::K_CHUNK + key * 128 + ((((cc & 1) * 4 + w) ^ (key & 7)) << 4)) = in ? make_uint4(o[0], o[1], o[2], o[3]) : make_uint4(0, 0, 0, 0);
                        }
                    }
                    if (++s1 == RAW) { s1 = 0; p1 ^= 1; }
                }
                dt_fence_async();
                __syncwarp();
                if (lane == 0) dt_arrive(bar_kf + 8 * sg);
                if (!__all_sync(0xffffffffu, ka_wait(bar_ve + 8 * sg, free_ph, abort_s))) return false;
#pragma unroll 1
                for (int h = 0; h <= two; h++) {
                    // values: a thread has eight keys (an octet, a piece of 16 bytes in the turned tile) of eight (heads of 64: four) neighbouring channels
                    const bool in = raw_in[st] != 0;
                    const uint8_t * vr = raw + st * C::REC + kv4_half(D);
                    uint8_t * to = sV + sg * C::V_TILE + h * C::V_CHUNK;
                    const int oct = tid & 7, o8 = D == 128 ? ((tid >> 5) * 4 + (lane >> 3) + 2 * oct) & 15 : (tid >> 3) & 7;
                    uint32_t n[8];
                    __half2  dm[8];
#pragma unroll
                    for (int k = 0; k < 8; k++) {
                        const int r = kv4_row(oct * 8 + k);
                        n[k]  = *reinterpret_cast<const uint32_t *>(vr + r * (D / 2) + ((o8 * 4) ^ kv4_flip(D, r)));
                        dm[k] = *reinterpret_cast<const __half2 *>(vr + kv4_steps(D) + (r * C::W + (o8 >> 2)) * 4);
                    }
                    if (edge_of(it, (it.page + i + h) * KV4_P)) {
                        // values that are none, on a page of which some row does not see all: they take part as zeros, and the rows that see one are told
                        if (tid < C::W) {
                            unsigned long long none = 0;
#pragma unroll 1
                            for (int k = 0; k < KV4_P; k++)
                                if (in && __hisnan(__high2half(*reinterpret_cast<const __half2 *>(vr + kv4_steps(D) + (kv4_row(k) * C::W + tid) * 4)))) none |= 1ull << k;
                            v_none[(sg * 2 + h) * C::W + tid] = none;
                        }
#pragma unroll
                        for (int k = 0; k < 8; k++) if (__hisnan(__high2half(dm[k]))) dm[k] = kv4_bits(0);
                    }
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        if (D == 64 && e != tid >> 6) continue;
                        uint32_t v[4][4];
#pragma unroll
                        for (int a = 0; a < 4; a++) kv4_pairs(ka_prmt(n[2 * a], n[2 * a + 1], e ? 0x7632 : 0x5410), __lows2half2(dm[2 * a], dm[2 * a + 1]), __highs2half2(dm[2 * a], dm[2 * a + 1]), v[a]);
#pragma unroll
                        for (int c = 0; c < 4; c++) {
                            const int row = o8 * 8 + e * 4 + c;
                            *reinterpret_cast<uint4 *>(to + row * 128 + ((oct ^ (row & 7)) << 4)) = in ? make_uint4(v[0][c], v[1][c], v[2][c], v[3][c]) : make_uint4(0, 0, 0, 0);
                        }
                    }
                    __syncwarp();
                    if (lane == 0) dt_arrive(bar_re + 8 * st);
                    if (++st == RAW) { st = 0; ph ^= 1; }
                }
                dt_fence_async();
                __syncwarp();
                if (lane == 0) dt_arrive(bar_vf + 8 * sg);
            }
            return true;
        });
    } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 152;");
        // ---- a row a thread
        const int w = (warp - 8) >> 2, q4 = warp & 3, rt = q4 * 32 + lane;
        const uint32_t lanes = (uint32_t) (q4 * 32) << 16, tm_s = tmem + lanes + 128 * w, tm_w = tm_o + lanes + 128 * w;
        int j = 0, n = 0;                                        // steps of the run, and those of which this group has scores
        auto wait = [&](uint32_t b, uint32_t ph) { return __all_sync(0xffffffffu, ka_wait(b, ph & 1, abort_s)) != 0; };
        items([&](const kp_item & it) {
            const int     pages = it.pages, rows = it.rows, ri = w * 128 + rt, rc = it.row0 + min(ri, rows - 1), tk = rc / A.rep, hi = it.pos0 + tk, lo = max(0, hi - ka_window(A) + 1);
            const int64_t tok = it.tok0 + tk, head = it.h * A.rep + rc % A.rep;
            const bool    on = w == 0 || rows > 128;
            if (!on) { j += (pages + 1) / 2; return true; }
            auto some = [&](int pg) { return pg + lane < A.max_pages ? A.table[(int64_t) it.s * A.max_pages + pg + lane] : -1; };
            int ids = some(it.page);
            float qs;
            {
                // the row as ka_power says, [0, 4, 1, 5, 2, 6, 3, 7] of eight channels as the keys have them.  Heads' rows of bfloat16 stay in registers between the passes
                const T * p = (const T *) A.q + tok * A.ldq + head * D;
                constexpr int N = C::SPLIT ? 32 : D;
                kp_row<T, N> v;
                float top = 0.f;
#pragma unroll 1
                for (int c = 0; c < D; c += N) { v.load(p + c, ka_here(A.wide_q)); top = fmaxf(top, v.top()); }
                const ka_power pw = ka_power_of<C::SPLIT>(C::SPLIT ? top * fabsf(A.scale * KA_LOG2E) : top, A.scale);
                qs = pw.back;
                uint8_t * to = sQ + w * C::NC * C::Q_CHUNK + rt * 128;
#pragma unroll 1
                for (int c = 0; c < D; c += N) {
                    if (N < D) v.load(p + c, ka_here(A.wide_q));
#pragma unroll
                    for (int i = 0; i < N / 8; i++) {
                        const int at16 = (N < D ? c >> 6 : i >> 3) * C::Q_CHUNK + (((N < D ? ((c & 63) >> 3) + i : i & 7) ^ (rt & 7)) << 4);
                        float x[8];
#pragma unroll
                        for (int k = 0; k < 8; k++) x[k] = (C::SPLIT ? v.at(8 * i + k) * (A.scale * KA_LOG2E) : v.at(8 * i + k)) * pw.down;
                        const uint4 h = make_uint4(ka_pack(x[0], x[4]), ka_pack(x[1], x[5]), ka_pack(x[2], x[6]), ka_pack(x[3], x[7]));
                        *reinterpret_cast<uint4 *>(to + at16) = h;
                        if (C::SPLIT)
                            *reinterpret_cast<uint4 *>(to + C::Q_PART + at16) = make_uint4(ka_rest(x[0], x[4], h.x), ka_rest(x[1], x[5], h.y), ka_rest(x[2], x[6], h.z), ka_rest(x[3], x[7], h.w));
                    }
                }
                dt_fence_async();
            }
            __syncwarp();
            if (lane == 0) dt_arrive(bar_q + 8 * w);
            float    m = -INFINITY, l = 0.f, l_low = 0.f;        // l_low: what additions to l rounded away
            bool     huge = false;
            // what has left tensor memory, [D / 4][rows] of four channels each, of fp32 rows three times (the sum, the second sum, what additions to that rounded away); then the maxima to which they are relative
            auto sums = [&]() { return reinterpret_cast<float4 *>(A.sums + me * kp_sums(C::SPLIT, D)) + ka_here(ri); };
            auto sums_m = [&](int level) -> float & { return (A.sums + me * kp_sums(C::SPLIT, D))[(C::SPLIT ? 3 : 1) * KP_ROWS * D + level * KP_ROWS + ka_here(ri)]; };
            uint32_t none = 0;                                   // groups of channels of which this row sees a value that is none
#pragma unroll 1
            for (int i0 = 0; i0 < pages; i0 += 2 * C::FOLD) {
                if (i0 > 0) {                                    // (the next scores come behind the end of the product before)
                    if (!wait(bar_s + 8 * w, n)) return false;
                    dt_fence_after();
                    const int   k = i0 / 2 / C::FOLD;            // the k-th time
                    float4 *    acc = sums();
                    const bool  have = C::SPLIT ? (k - 1) % KP_FOLDS != 0 : k > 1;
                    const float ma = have ? sums_m(0) : m, f = ma == m ? 1.f : ka_exp2(ma - m);
#pragma unroll 1
                    for (int c = 0; c < D; c += 32) {
                        uint32_t v[32];
                        dt_ld32(tm_w + c, v);
                        dt_wait_ld();
#pragma unroll
                        for (int x = 0; x < 32; x += 4) {
                            float4 * a = acc + (c + x) / 4 * KP_ROWS;
                            float4   o = make_float4(__uint_as_float(v[x]), __uint_as_float(v[x + 1]), __uint_as_float(v[x + 2]), __uint_as_float(v[x + 3]));
                            if (have) kp_add(o, *a, f);
                            *a = o;
                        }
                    }
                    sums_m(0) = m;
                    if (C::SPLIT && k % KP_FOLDS == 0) {         // on to the second sum
                        const float mb = k > KP_FOLDS ? sums_m(1) : m, fb = mb == m ? 1.f : ka_exp2(mb - m);
                        float4 *    sum = acc + KP_ROWS * D / 4, * low = sum + KP_ROWS * D / 4;
#pragma unroll 1
                        for (int c = 0; c < D / 4; c++) {
                            float4 o = acc[c * KP_ROWS], e = make_float4(0.f, 0.f, 0.f, 0.f);
                            if (k > KP_FOLDS) { e = ka_times(low[c * KP_ROWS], fb, fb); o = ka_sum(ka_times(sum[c * KP_ROWS], fb, fb), o, e); }
                            sum[c * KP_ROWS] = o;
                            low[c * KP_ROWS] = e;
                        }
                        sums_m(1) = m;
                    }
                }
#pragma unroll 1
            for (int i = i0; i < min(i0 + 2 * C::FOLD, pages); i += 2, j++, n++) {
                const int two = i + 1 < pages;
                if (i > 0 && (i & 31) == 0) ids = some(it.page + i);
                const int  id0 = __shfl_sync(0xffffffffu, ids, i & 31), id1 = __shfl_sync(0xffffffffu, ids, (i + 1) & 31);
                if (!wait(bar_s + 8 * w, n)) return false;
                dt_fence_after();
                uint32_t t[64];
                // a page's scores; keys that the row does not see are at -inf
                auto load = [&](int h) {
                    dt_ld32(tm_s + 64 * h, t);
                    dt_ld32(tm_s + 64 * h + 32, t + 32);
                    dt_wait_ld();
                    const int  key0 = (it.page + i + h) * KV4_P, id = h ? id1 : id0;
                    const bool in = id >= 0 && id < A.pages;
                    if (!in || edge_of(it, key0)) {
                        const int a = in ? lo - key0 : 64, b = hi - key0;
#pragma unroll
                        for (int x = 0; x < 64; x++) if (x < a || x > b) t[x] = 0xff800000u;
                    }
                };
                float top = -INFINITY;
#pragma unroll 1
                for (int h = 0; h <= two; h++) {
                    load(h);
#pragma unroll
                    for (int x = 0; x < 64; x++) top = fmaxf(top, __uint_as_float(t[x]));
                    const int  key0 = (it.page + i + h) * KV4_P, id = h ? id1 : id0;
                    if (id >= 0 && id < A.pages && edge_of(it, key0)) {
                        const int a = lo - key0, b = hi - key0;
                        if (!wait(bar_vf + 8 * (j % C::STG), j / C::STG)) return false;
                        if (b >= 0 && a < 64) {
                            const unsigned long long seen = (b >= 63 ? ~0ull : (1ull << (b + 1)) - 1) & ~(a > 0 ? (1ull << a) - 1 : 0ull);
#pragma unroll
                            for (int g = 0; g < C::W; g++) if (v_none[((j % C::STG) * 2 + h) * C::W + g] & seen) none |= 1u << g;
                        }
                    }
                }
                top *= qs;
                const bool grow = top > m + ka_lazy<C::SPLIT>;
                const bool rescale = __any_sync(0xffffffffu, grow);
                float f = 1.f;
                if (grow) { f = ka_exp2(m - top); m = top; l *= f; l_low *= f; huge = !C::SPLIT && fabsf(m) > KA_HUGE; }
                const float base = ka_base<C::SPLIT>(m);
                if (i > i0 && rescale) {
#pragma unroll 1
                    for (int c = 0; c < D; c += 32) {
                        uint32_t v[32];
                        dt_ld32(tm_w + c, v);
                        dt_wait_ld();
#pragma unroll
                        for (int x = 0; x < 32; x++) v[x] = __float_as_uint(__uint_as_float(v[x]) * f);
                        dt_st32(tm_w + c, v);
                    }
                }
                // the last page's scores are in registers still
                uint64_t ll = 0;
#pragma unroll 1
                for (int h = two; h >= 0; h--) {
                    if (h != two) load(h);
                    float q = qs;
                    if (!C::SPLIT && __any_sync(0xffffffffu, huge)) {
                        const float k = huge ? qs : 1.f;
#pragma unroll
                        for (int x = 0; x < 64; x++) t[x] = __float_as_uint(__uint_as_float(t[x]) * k);
                        if (huge) q = 1.f;
                    }
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        uint32_t e[16], r[16];
#pragma unroll
                        for (int x = 0; x < 16; x++) {
                            const float2 z = ka_each(ka_fma2(ka_two(__uint_as_float(t[32 * c + 2 * x]), __uint_as_float(t[32 * c + 2 * x + 1])), ka_two(q, q), ka_two(base, base)));
                            const uint64_t w2 = ka_two(ka_exp2(z.x), ka_exp2(z.y));
                            ll = ka_add2(ll, w2);
                            const float2 wf = ka_each(w2);
                            e[x] = ka_pack(wf.x, wf.y);
                            const float2 hf = ka_float2(e[x]);
                            const float2 rf = ka_each(ka_sub2(w2, ka_two(hf.x, hf.y)));
                            r[x] = ka_pack(rf.x, rf.y);
                        }
                        // in the page's scores' place, parts behind each other
                        kp_st16(tm_s + 64 * h + 16 * c, e);
                        kp_st16(tm_s + 64 * h + 32 + 16 * c, r);
                    }
                }
                dt_wait_st();
                dt_fence_before();
                __syncwarp();
                if (lane == 0) dt_arrive(bar_p + 8 * w);
                const float2 l2 = ka_each(ll);
                l = ka_sum(l, l2.x + l2.y, l_low);
            }
            }
            // ---- the row out, behind the last product
            if (!wait(bar_o + 8 * w, n + 1)) return false;
            dt_fence_after();
            const bool    whole = it.whole;
            const float   sum = l + l_low, inv = sum > 0.f ? 1.f / sum : sum;           // a row that saw nothing: zeros; a sum that is none stays so
            float *       piece = A.pieces + (2 * me + it.slot) * (int64_t) C::PIECE;
            const int     folds = (pages - 1) / 2 / C::FOLD;     // how often sums have left
            const float4 * acc = sums();
            const bool    have = !C::SPLIT ? folds > 0 : folds % KP_FOLDS != 0, more = C::SPLIT && folds >= KP_FOLDS;
            const float   ma = have ? sums_m(0) : m, f = ma == m ? 1.f : ka_exp2(ma - m), mb = more ? sums_m(1) : m, fb = mb == m ? 1.f : ka_exp2(mb - m);
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
                float v[32];
                dt_ld32(tm_w + c, reinterpret_cast<uint32_t *>(v));
                dt_wait_ld();
                if (folds)
#pragma unroll
                    for (int x = 0; x < 32; x += 4) {
                        float4 o = make_float4(v[x], v[x + 1], v[x + 2], v[x + 3]);
                        if (have) kp_add(o, acc[(c + x) / 4 * KP_ROWS], f);
                        if (more) { kp_add(o, acc[(c + x) / 4 * KP_ROWS + KP_ROWS * D / 2], fb); kp_add(o, acc[(c + x) / 4 * KP_ROWS + KP_ROWS * D / 4], fb); }
                        v[x] = o.x; v[x + 1] = o.y; v[x + 2] = o.z; v[x + 3] = o.w;
                    }
                const float k = none >> (c >> 5) & 1 ? __uint_as_float(0x7fc00000u) : whole ? inv : 1.f;
#pragma unroll
                for (int x = 0; x < 32; x++) v[x] *= k;
                if (!whole)                                      // [D / 4][rows] of four channels each: a warp's stores are neighbours
#pragma unroll
                    for (int x = 0; x < 32; x += 4) reinterpret_cast<float4 *>(piece)[(c + x) / 4 * KP_ROWS + ri] = make_float4(v[x], v[x + 1], v[x + 2], v[x + 3]);
                else if (ri < rows) ka_store<T, 32>((T *) A.out + tok * A.ldo + head * D + c, ka_here(A.wide_o), v);
                __syncwarp();                                    // (the next columns are loaded by the warp as one)
            }
            if (!whole) { piece[KP_ROWS * D + ri] = m; piece[KP_ROWS * D + KP_ROWS + ri] = sum; }
            dt_fence_before();
            return true;
        });
    }
    __syncwarp();
    dt_fence_before();
    __syncthreads();
    if (*abort_s) {
        // a wait ran out: say so, give copies and MMAs still in flight time to land (bounded), then free the tensor memory
        if (threadIdx.x == 0) atomicExch(A.err, 1 + (int) blockIdx.x);
#pragma unroll 1
        for (int i = 0; i < 2000; i++) __nanosleep(1000);
        __syncthreads();
    }
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

// Blocks (run, eighth of the rows): an item whose pages begin in the run and do not end there gets its pieces' sum, a lane a row, a warp an eighth of the channels.
template <typename T, int D>
static __global__ void __launch_bounds__(256) kv4_prompt_join_kernel(const __grid_constant__ ka_args A) {
    using C = kp_cfg<T, D>;
    pib_pdl_wait();
    pib_pdl_trigger();
    const int     lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t runs = A.plan->runs, wa = blockIdx.x;
    if (wa + 1 >= runs) return;
    const int64_t * prefix = A.plan->prefix;
    const int64_t U = prefix[A.seqs], u0 = U * wa / runs, u1 = U * (wa + 1) / runs;
    const ka_seq_call seq_of = { &A };
    const ka_place at = ka_find<KP_ROWS, KP_LEAD>(A, prefix, seq_of, u1 - 1);
    const int64_t  ib = u1 - 1 - at.p + KP_LEAD, ie = ib - KP_LEAD + at.np;         // its pages' units
    if (ib < u0 || ib >= u1 || ie <= u1) return;
    const ka_seq  q = seq_of(at.s);
    const int     row0 = at.r * KP_ROWS, rows = (int) min((int64_t) KP_ROWS, (int64_t) q.n * A.rep - row0);
    const int64_t wb = (ie * runs + U - 1) / U - 1, tok0 = q.start;
    constexpr int CH = D / 8;
    const int ri = blockIdx.y * 32 + lane;
    if (ri >= rows) return;
    auto piece = [&](int64_t w) { return A.pieces + (2 * w + (w == wa ? 1 : 0)) * (int64_t) C::PIECE; };
    float m = -INFINITY, l = 0.f, o[CH];
#pragma unroll
    for (int c = 0; c < CH; c++) o[c] = 0.f;
#pragma unroll 4
    for (int64_t w = wa; w <= wb; w++) m = fmaxf(m, piece(w)[KP_ROWS * D + ri]);
#pragma unroll 2
    for (int64_t w = wa; w <= wb; w++) {
        const float * p = piece(w);
        const float   pm = p[KP_ROWS * D + ri], f = pm == m ? 1.f : exp2f(pm - m);
        l = fmaf(p[KP_ROWS * D + KP_ROWS + ri], f, l);
#pragma unroll
        for (int c = 0; c < CH; c += 4) {
            const float4 v = reinterpret_cast<const float4 *>(p)[(warp * CH + c) / 4 * KP_ROWS + ri];
            o[c] = fmaf(v.x, f, o[c]); o[c + 1] = fmaf(v.y, f, o[c + 1]); o[c + 2] = fmaf(v.z, f, o[c + 2]); o[c + 3] = fmaf(v.w, f, o[c + 3]);
        }
    }
    const int rc = row0 + ri;
    const float inv = l > 0.f ? 1.f / l : l;
#pragma unroll
    for (int c = 0; c < CH; c++) o[c] *= inv;
    ka_store<T, CH>((T *) A.out + (tok0 + rc / A.rep) * A.ldo + (int64_t) (at.h * A.rep + rc % A.rep) * D + warp * CH, A.wide_o, o);
}

// ---- host side --------------------------------------------------------------------------------------------------------------------
template <typename T, int D> static int kp_go(ka_args A, cudaStream_t st) {
    using C = kp_cfg<T, D>;
    // three records under way where the sequences' table leaves room for them
    constexpr size_t most = 226 * 1024;
    const size_t need = C::FIXED + (size_t) (A.seqs + 1) * 8;
    static_assert(C::FIXED + (PIB_KV4_MAX_SEQS + 1) * 8 + 2 * C::REC <= most, "shared memory");
    A.stages = need + 3 * C::REC <= most ? 3 : 2;
    const size_t smem = need + (size_t) A.stages * C::REC;
    static pib_per_device attrs;
    PIB_CHECK(attrs.once([&] { return cudaFuncSetAttribute(kv4_prompt_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int) most); }));
    PIB_CHECK(pib_launch(kv4_prompt_kernel<T, D>, dim3((unsigned) pib_num_sms()), dim3(KP_THREADS), smem, st, A));
    PIB_CHECK(pib_launch(kv4_prompt_join_kernel<T, D>, dim3((unsigned) pib_num_sms(), KP_ROWS / 32), dim3(256), 0, st, A));
    return PIB_OK;
}
int pib_kv4_prompt(ka_args A, bool f32, cudaStream_t st) {
    if (f32) return A.dim == 64 ? kp_go<float, 64>(A, st) : kp_go<float, 128>(A, st);
    return A.dim == 64 ? kp_go<__nv_bfloat16, 64>(A, st) : kp_go<__nv_bfloat16, 128>(A, st);
}
