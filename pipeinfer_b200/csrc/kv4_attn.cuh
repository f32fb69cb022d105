// kv4_attn.cuh -- what the kernels of attention over a 4-bit cache share (kv4_attn.cu: decode and verification batches; kv4_prompt.cu: prompts): the work's division, rows in and out.
#pragma once

#include "kv4.cuh"
#include "tc_common.cuh"

#define KA_LOG2E 1.4426950408889634f

struct ka_args {
    const uint8_t * base; int64_t pages; int kvh, rep, dim; uint32_t part;                  // part: ka_over
    const int32_t * starts, * lens, * table; int tokens, seqs, max_pages, window; float scale;
    const void * q; void * out; int64_t ldq, ldo; bool wide_q, wide_o;       // rows that 16-byte loads and stores may take
    int stages; float * pieces, * heads, * sums; struct ka_plan * plan; struct ka_open * open; int * err;
};

// x / rep, x up to rep + 31 and rep up to 1024: a product, where a division in each row's place were a tenth of the decode kernel's code
__device__ __forceinline__ int ka_over(const ka_args & A, int x) { return (int) ((uint32_t) x * A.part >> 21); }
// a condition that stays where it is written: of one that holds for a whole loop the compiler makes two loops (of three, eight: 200 KB of code, which no instruction cache holds)
__device__ __forceinline__ int ka_here(int v) { asm volatile("" : "+r"(v)); return v; }
// dt_mbar_wait in few instructions: there is one at every turn, and the loops' code has to stay near
__device__ __forceinline__ bool ka_wait(uint32_t bar, uint32_t parity, volatile int * abort_s) {
    uint32_t ok = 0;
#pragma unroll 1
    for (uint32_t it = 0; it < DT_SPIN; it++) {
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
        if (ok) return true;
        if ((it & 63) == 63 && *abort_s) return false;
    }
    *abort_s = 1;
    return false;
}

// A row's queries enter over the power of two that brings the largest to 2^14 .. 2^15.  fp32 rows, times scale log2 e before: two fp16 numbers hold 22 bits of a channel down to 2^-17 of the row's largest and
// 2^-39 of the largest below; what scores are multiplied with is the power of two, exact, and so is the running maximum.  bfloat16 rows: one fp16 number holds every channel as it is down to 2^-30 of the
// largest, so |scale| log2 e is left to the factor that scores are multiplied with (never 0: what is not seen stands at -inf); a maximum beyond KA_HUGE is rounded too far for one fused operation, and its
// row's scores are then multiplied, and rounded, first
#define KA_HUGE 1048576.f
struct ka_power { float down, back; };
template <bool SPLIT> __device__ __forceinline__ ka_power ka_power_of(float top, float scale) {
    const uint32_t e = min(max((int) (__float_as_uint(top) >> 23) - 14, 1), 240);
    const float    down = __uint_as_float((254u - e) << 23), back = __uint_as_float(e << 23);
    if (SPLIT) return { down, back };
    return { copysignf(down, scale), fminf(fmaxf(back * fabsf(scale) * KA_LOG2E, 1.17549435e-38f), 3.4e38f) };
}

// n neighbouring values as floats, n a multiple of 8
template <typename T, int N> __device__ __forceinline__ void ka_fetch(const T * p, bool wide, uint32_t (&r)[N * sizeof(T) / 4]) {
    if (wide) {
#pragma unroll
        for (int i = 0; i < N * (int) sizeof(T) / 4; i += 4) { const uint4 f = reinterpret_cast<const uint4 *>(p)[i / 4]; r[i] = f.x; r[i + 1] = f.y; r[i + 2] = f.z; r[i + 3] = f.w; }
    } else
#pragma unroll
        for (int i = 0; i < N * (int) sizeof(T) / 4; i++) {
            if constexpr (sizeof(T) == 4) r[i] = __float_as_uint(p[i]);
            else                          r[i] = __bfloat16_as_ushort(p[2 * i]) | (uint32_t) __bfloat16_as_ushort(p[2 * i + 1]) << 16;
        }
}
template <typename T> __device__ __forceinline__ float ka_value(const uint32_t * r, int c) {
    if constexpr (sizeof(T) == 4) return __uint_as_float(r[c]);
    else                          return __uint_as_float(c & 1 ? r[c >> 1] & 0xffff0000u : r[c >> 1] << 16);
}
template <typename T, int N> __device__ __forceinline__ void ka_store(T * p, bool wide, const float (&v)[N]) {
    if constexpr (sizeof(T) == 4) {
        if (wide) {
#pragma unroll
            for (int i = 0; i < N; i += 4) *reinterpret_cast<float4 *>(p + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
        } else
#pragma unroll
            for (int i = 0; i < N; i++) p[i] = v[i];
    } else {
        if (wide) {
#pragma unroll
            for (int i = 0; i < N; i += 8) {
                __nv_bfloat162 h[4];
#pragma unroll
                for (int j = 0; j < 4; j++) h[j] = __floats2bfloat162_rn(v[i + 2 * j], v[i + 2 * j + 1]);
                *reinterpret_cast<uint4 *>(p + i) = *reinterpret_cast<const uint4 *>(h);
            }
        } else
#pragma unroll
            for (int i = 0; i < N; i++) p[i] = __float2bfloat16_rn(v[i]);
    }
}

// the window as a distance: none is one that reaches everything
__device__ __forceinline__ int ka_window(const ka_args & A) { return A.window > 0 ? min(A.window, 0x7fff0000) : 0x7fff0000; }
// ---- which keys a tile of rows sees ---------------------------------------------------------------------------------------------------
// A sequence's rows, (token, head of the group) with the heads next to each other, are taken in tiles of RT; a tile of one key / value head is an item, its pages the units of work
struct ka_seq { int n, len, start; };               // query tokens and keys, both >= 0; the first token's row
__device__ __forceinline__ ka_seq ka_load_seq(const ka_args & A, int s) {
    const int a = min(max(A.starts[s], 0), A.tokens), b = min(max(A.starts[s + 1], 0), A.tokens);
    return { max(b - a, 0), max(A.lens[s], 0), a };
}
// pages [first, first + count) of tile r; keys behind the table's row are not there
template <int RT> __device__ __forceinline__ int ka_pages(const ka_args & A, ka_seq q, int r, int & first) {
    const int t0 = r * RT / A.rep, t1 = min(q.n - 1, ((r + 1) * RT - 1) / A.rep), p0 = q.len - q.n + t0, p1 = q.len - q.n + t1;
    const int top = min(p1 < 0 ? -1 : p1 / KV4_P, A.max_pages - 1);
    first = max(0, p0 - ka_window(A) + 1) / KV4_P;
    return max(0, top - first + 1);
}
template <int RT> __device__ __forceinline__ int ka_tiles(const ka_args & A, ka_seq q) { return (int) (((int64_t) q.n * A.rep + RT - 1) / RT); }

// a + b, and what the addition rounds away comes on top of e
__device__ __forceinline__ float ka_sum(float a, float b, float & e) { const float t = a + b, z = t - a; e += (a - (t - z)) + (b - z); return t; }
__device__ __forceinline__ float4 ka_sum(float4 a, float4 b, float4 & e) { return make_float4(ka_sum(a.x, b.x, e.x), ka_sum(a.y, b.y, e.y), ka_sum(a.z, b.z, e.z), ka_sum(a.w, b.w, e.w)); }
__device__ __forceinline__ float4 ka_times(float4 a, float f, float g) { return make_float4(a.x * f, a.y * g, a.z * f, a.w * g); }

// what both kernels know of the work: behind the pieces in the scratch
struct ka_plan { int64_t runs, prefix[PIB_KV4_MAX_SEQS + 1]; };           // prompts: runs of units; units in front of each sequence
// decode: of each run whether an item begins there and does not end there; the run where it does, its first row counted from the first token in it (tok0), its rows
struct ka_open { int runs, last, row0, rows, h; int64_t tok0; };

// a sequence's tokens and keys from a table in shared memory, or from the call's
struct ka_seq_table { ka_seq * p; __device__ __forceinline__ ka_seq operator()(int s) const { return p[s]; } __device__ __forceinline__ void operator()(int s, ka_seq q) const { p[s] = q; } };
struct ka_seq_none  { __device__ __forceinline__ void operator()(int, ka_seq) const {} };
struct ka_seq_call  { const ka_args * a; __device__ __forceinline__ ka_seq operator()(int s) const { return ka_load_seq(*a, s); } };
// A place among the units: unit p of np, page first + p - LEAD, of head h, of tile r, of sequence s.  prefix: units in front of each sequence; seq(s): its tokens and keys.  An item has LEAD units in front
// of its pages: what its start and end cost, in pages
struct ka_place { int s, r, h, p, np, first; };
template <int RT, int LEAD> __device__ __forceinline__ int ka_units(const ka_args & A, ka_seq q, int r, int & first) { const int n = ka_pages<RT>(A, q, r, first); return n ? n + LEAD : 0; }
template <int RT, int LEAD, typename Seq> __device__ __forceinline__ void ka_enter(const ka_args & A, const Seq & seq, ka_place & c) { c.np = ka_units<RT, LEAD>(A, seq(c.s), c.r, c.first); }
// the item behind c's; only called where there is one
template <int RT, int LEAD, typename Seq> __device__ __forceinline__ void ka_next_item(const ka_args & A, const int64_t * prefix, const Seq & seq, ka_place & c) {
    c.p = 0;
    if (++c.h < A.kvh) return;
    c.h = 0;
#pragma unroll 1
    do {
        if (++c.r >= ka_tiles<RT>(A, seq(c.s))) {
            c.r = 0;
#pragma unroll 1
            do c.s++; while (prefix[c.s + 1] == prefix[c.s]);
        }
        ka_enter<RT, LEAD>(A, seq, c);
    } while (c.np == 0);
}
// unit u < prefix[seqs]
template <int RT, int LEAD, typename Seq> __device__ __forceinline__ ka_place ka_find(const ka_args & A, const int64_t * prefix, const Seq & seq, int64_t u) {
    int lo = 0, hi = A.seqs;                                     // the last sequence with prefix <= u: it has units
#pragma unroll 1
    while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (prefix[mid] <= u) lo = mid; else hi = mid; }
    int64_t  rest = u - prefix[lo];
    ka_place c;
    c.s = lo; c.r = 0;
#pragma unroll 1
    for (ka_enter<RT, LEAD>(A, seq, c); rest >= (int64_t) c.np * A.kvh; ka_enter<RT, LEAD>(A, seq, c)) { rest -= (int64_t) c.np * A.kvh; c.r++; }
    c.h = (int) (rest / c.np); c.p = (int) (rest % c.np);
    return c;
}
// Units in front of each sequence (and items, if asked for), by all THREADS threads of a block: a thread's neighbouring sequences, then warps, then the block.  part: THREADS / 32 numbers (twice that).  Ends with a barrier; the first block leaves
// them in the plan
template <int RT, int LEAD, int THREADS, typename Keep> __device__ __forceinline__ int64_t ka_prefix(const ka_args & A, int64_t * prefix, int64_t * part, Keep keep, int * items = nullptr) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, per = (A.seqs + THREADS - 1) / THREADS, s0 = threadIdx.x * per;
    int64_t sum = 0;
    int     count = 0;
#pragma unroll 1
    for (int s = s0; s < min(s0 + per, A.seqs); s++) {
        const ka_seq q = ka_load_seq(A, s);
        keep(s, q);
        prefix[s] = sum;
        if (items) items[s] = count;
        int first;
#pragma unroll 1
        for (int r = 0; r < ka_tiles<RT>(A, q); r++) { const int n = ka_units<RT, LEAD>(A, q, r, first); sum += (int64_t) n * A.kvh; count += n ? A.kvh : 0; }
    }
    int64_t before = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int64_t v = __shfl_up_sync(0xffffffffu, before, o); if (lane >= o) before += v; }
    int items_before = count;
    if (items)
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const int v = __shfl_up_sync(0xffffffffu, items_before, o); if (lane >= o) items_before += v; }
    if (lane == 31) { part[warp] = before; if (items) part[THREADS / 32 + warp] = items_before; }
    before -= sum;
    items_before -= count;
    __syncthreads();
    int64_t all = 0;
    int     all_items = 0;
#pragma unroll 1
    for (int i = 0; i * 32 * per < A.seqs; i++) {
        if (i < warp) before += part[i];
        all += part[i];
        if (items) { const int v = (int) part[THREADS / 32 + i]; if (i < warp) items_before += v; all_items += v; }
    }           // (warps without sequences add nothing)
#pragma unroll 1
    for (int s = s0; s < min(s0 + per, A.seqs); s++) { prefix[s] += before; if (items) items[s] += items_before; }
    if (threadIdx.x == 0) { prefix[A.seqs] = all; if (items) items[A.seqs] = all_items; }
    __syncthreads();
    return all;
}
// Decode: runs are shares of work, of which an item's start and end are EXTRA pages' worth.  The first unit (page) behind share w of prefix[seqs] + EXTRA * items[seqs]
template <int RT, int EXTRA, typename Seq> __device__ __forceinline__ int64_t ka_cut(const ka_args & A, const int64_t * prefix, const int * items, const Seq & seq, int64_t w) {
    int lo = 0, hi = A.seqs;
#pragma unroll 1
    while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (prefix[mid] + (int64_t) EXTRA * items[mid] <= w) lo = mid; else hi = mid; }
    int64_t rest = w - prefix[lo] - (int64_t) EXTRA * items[lo], u = prefix[lo];
    int n, first;
#pragma unroll 1
    for (int r = 0; (n = ka_pages<RT>(A, seq(lo), r, first)) == 0 || rest >= (int64_t) (n + EXTRA) * A.kvh; r++) if (n) { rest -= (int64_t) (n + EXTRA) * A.kvh; u += (int64_t) n * A.kvh; }
    return u + rest / (n + EXTRA) * n + max((int) (rest % (n + EXTRA)) - EXTRA, 0);
}
// the work up to an item's end
template <int RT, int EXTRA, typename Seq> __device__ __forceinline__ int64_t ka_work(const ka_args & A, const int64_t * prefix, const int * items, const Seq & seq, const ka_place & c) {
    int64_t w = prefix[c.s] + (int64_t) EXTRA * items[c.s] + (int64_t) (c.h + 1) * (c.np + EXTRA);
    int first;
#pragma unroll 1
    for (int r = 0; r < c.r; r++) { const int n = ka_pages<RT>(A, seq(c.s), r, first); if (n) w += (int64_t) (n + EXTRA) * A.kvh; }
    return w;
}
// zeros into the rows of tiles without pages; sequences by blocks
template <int RT, int THREADS, typename T, typename Seq> __device__ __forceinline__ void ka_zero_rows(const ka_args & A, const Seq & seq, int D) {
#pragma unroll 1
    for (int s = blockIdx.x; s < A.seqs; s += gridDim.x) {
        const ka_seq  q = seq(s);
        const int64_t tok0 = q.start;
#pragma unroll 1
        for (int r = 0; r < ka_tiles<RT>(A, q); r++) {
            int first;
            if (ka_pages<RT>(A, q, r, first)) continue;
            const int row0 = r * RT, rows = (int) min((int64_t) RT, (int64_t) q.n * A.rep - row0);
#pragma unroll 1
            for (int i = threadIdx.x; i < rows * A.kvh * D; i += THREADS) {          // at most 256 * 1024 * 128
                const int c = i % D, h = i / D % A.kvh, rc = row0 + i / D / A.kvh;
                ((T *) A.out)[(tok0 + rc / A.rep) * A.ldo + (int64_t) (h * A.rep + rc % A.rep) * D + c] = (T) 0.f;
            }
        }
    }
}
template <int THREADS> __device__ __forceinline__ void ka_leave_plan(const ka_args & A, const int64_t * prefix, int64_t runs) {
    if (blockIdx.x != 0) return;
    if (threadIdx.x == 0) A.plan->runs = runs;
#pragma unroll 1
    for (int s = threadIdx.x; s <= A.seqs; s += THREADS) A.plan->prefix[s] = prefix[s];
}

// Weights are e^(s - m) 2^lift, where m follows the running maximum once that is 2^lazy ahead: 2^15 at most.  Part and remainder in fp16 hold them down to 2^-25, that is 2^-32 (fp32 rows: 2^-39) of a row's
// largest weight: less is nothing in the products, and a million keys of which each loses 2^-39 are 2^-19.  With a lazy maximum few blocks of keys rescale the sums, and bfloat16 outputs do not see what is lost
template <bool SPLIT> constexpr float ka_lift = SPLIT ? 14.f : 7.f;
template <bool SPLIT> constexpr float ka_lazy = SPLIT ? 1.f : 8.f;
// what exponents get beside their score: lift - m, rounded down, since maxima from 2^25 on have no such numbers between their own, and weights of more than 2^15 are none in fp16
template <bool SPLIT> __device__ __forceinline__ float ka_base(float m) { return __fsub_rd(ka_lift<SPLIT>, m == -INFINITY ? 0.f : m); }

// within 2^-22 of 2^x
__device__ __forceinline__ float ka_exp2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ uint32_t ka_pack(float a, float b) { const __half2 h = __floats2half2_rn(a, b); return *reinterpret_cast<const uint32_t *>(&h); }
__device__ __forceinline__ float2 ka_float2(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2 *>(&v)); }
// two floats in one operation each
__device__ __forceinline__ uint64_t ka_two(float a, float b) { uint64_t r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ float2 ka_each(uint64_t v) { float2 f; asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v)); return f; }
__device__ __forceinline__ uint64_t ka_fma2(uint64_t a, uint64_t b, uint64_t c) { uint64_t r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }
__device__ __forceinline__ uint64_t ka_add2(uint64_t a, uint64_t b) { uint64_t r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ uint64_t ka_sub2(uint64_t a, uint64_t b) { uint64_t r; asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
// what the rounding to fp16 took away
__device__ __forceinline__ uint32_t ka_rest(float a, float b, uint32_t hi) { const float2 f = ka_float2(hi); return ka_pack(a - f.x, b - f.y); }
__device__ __forceinline__ uint32_t ka_prmt(uint32_t a, uint32_t b, uint32_t sel) { uint32_t r; asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(sel)); return r; }
__device__ __forceinline__ void ka_bulk(uint32_t dst, const void * src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

// kv4_prompt.cu: launches; rows of a block; floats of a block's sums that have left tensor memory
#define KP_ROWS 256
__host__ __device__ constexpr size_t kp_sums(bool f32, int dim) { return (size_t) KP_ROWS * (f32 ? 3 * dim + 2 : dim + 1); }
int    pib_kv4_prompt(ka_args A, bool f32, cudaStream_t st);
