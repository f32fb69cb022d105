// sample_draw.cu -- a token of each row of logits: top-k, top-p, min-p, temperature, drawn with a given number.
//
// A row's tokens are ordered by (logit descending, id ascending); every truncation keeps a run from the front of that order, so it is one threshold in it, and nothing is sorted.  With
// w = e^(l - l_max), formed in fp64 to 2^-37 of itself and rounded to a multiple of 2^-44: sums of up to 2^18 such numbers are exact in 64-bit integers, so no result depends on which thread or
// block added first.  (Below e^-31 a weight is 0: such a token is kept, and counted, but never drawn.)
//   top-k   the threshold is the k-th token of the order
//   top-p   the first token at which the running sum of w reaches top_p times that of what top-k left
//   min-p   w >= min_p
//   draw    weights e^((l - l_max) / temp) of what is kept, the first id at which their running sum exceeds u times the total
// A row is divided over the P blocks of a thread-block cluster in slices of neighbouring ids; the blocks meet through distributed shared memory.  A slice is walked in chunks of 256 ids, eight
// neighbours a lane (32 bytes of fp32, 16 of bfloat16, aligned wherever the row begins), two chunks of a warp under way; the row comes from memory once and from L2 after that:
//   1  the maximum (behind it the cluster's blocks are known to have started)
//   2  a histogram of l_max - l in 8192 bins 1/256 wide: counts alone, since the tokens of a bin weigh the same up to a factor of e^(1/256).  For top-p also the exact sum of all weights,
//      in registers
//   3  top-k: the tokens up to the bin of the k-th are gathered, and all that follows happens among them.  top-p: with the bounds that the counts give, the threshold lies in a few bins; their
//      tokens are gathered, and what lies ahead of those bins is summed exactly
//   4  the weights' sums of what is kept, per chunk, and the walk through one chunk (not where step 3 gathered everything that is kept)
// Among gathered tokens each finds what lies ahead of it by comparing with all.  Where a list would be too long (thousands of equal logits, say) sd_select narrows the threshold
// down by histograms over the order's own bits instead.
// What bounds it: the arithmetic and shared memory of an SM's walks over its slice, not the memory (64 rows of 128 256: 61 us with mixed settings, the bytes take 5).  64 rows of 128 256
// with a block each: greedy (one walk) 15 us, top-k 32, min-p 41, no truncation 54 (a dozen fp64 steps for a weight), top-p 130 (three walks that form weights, one with atomics beside it).
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include <limits.h>

#include "engine.cuh"
#include "sample_border.cuh"

#define SD_THREADS 512
#define SD_WARPS   (SD_THREADS / 32)
#define SD_BINS    2048                       // of a level of sd_select
#define SD_LIST    2048
#define SD_POW     1024
#define SD_SLICE   4096                       // ids of a block at least, where a row is divided
#define SD_CHUNK   256
#define SD_CHUNKS  (PIB_SAMPLE_MAX_VOCAB / SD_CHUNK + 1)

typedef unsigned long long sd_u64;

struct sd_range { sd_u64 mass; uint32_t count, bin; };
struct sd_shared {
    union {
        struct { uint32_t count[SD_BINS], lo[SD_BINS], hi[SD_BINS]; };      // a level's sums in two 32-bit parts: lo's carry goes to hi
        uint32_t fine[SD_FINE];
        sd_u64   w[SD_LIST];                                     // weights of the list
    };
    union { sd_u64 list[SD_LIST]; float tmax[SD_THREADS * 8]; };            // gathered tokens; the threads' maxima, in the first block
    sd_u64   chunk[SD_CHUNKS];
    double   pow[SD_POW];                                        // 2^(j / 1024)
    sd_u64   wsum[SD_WARPS], sum;                                // of a block's warps, of the block
    sd_u64   wbound[SD_WARPS], bound;
    uint32_t wcnt[SD_WARPS], cnt, n_list;
    float    bound_k;                                            // at least top_k tokens reach it
    float    wmax[SD_WARPS], max;
    int      warg[SD_WARPS], arg;
    sd_range own, found;                                         // a block's bins; the bin that holds the threshold, and what lies ahead of it
    uint32_t n_sub, res; sd_u64 pre;                             // sd_find
    uint32_t first, last, n_first, n_last;                       // bins between which the threshold lies; tokens ahead of them, and up to the last
    sd_u64   thr, thr_mass;                                      // the threshold in the order, and the mass up to it
};

__device__ __forceinline__ uint32_t sd_key(float v) { const uint32_t u = __float_as_uint(v + 0.0f); return u & 0x80000000u ? ~u : u | 0x80000000u; }
// place in the order: larger comes first
__device__ __forceinline__ sd_u64 sd_place(float v, int id) { return (sd_u64) sd_key(v) << 32 | (uint32_t) ~id; }
__device__ __forceinline__ float  sd_logit(sd_u64 place) { const uint32_t k = (uint32_t) (place >> 32); return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
// e^((v - l_max) / temp) 2^44 rounded to an integer: x = k ln2 / 1024 + r with |r| <= ln2 / 2048, e^r by its series up to r^2 / 2 (r^3 / 6 is 2^-37.1 and of either sign), 2^(k / 1024) from a table
// and the exponent.  x below -40 enters as about that, -inf too: it weighs nothing, without a branch or a choice.  (exp() in its place: 77 us for 64 rows of 128 256 without truncation, 30 with a
// table of 256 and a check of the range behind it.)
#define SD_BITS52 0x4330000000000000ull       // the bits of 2^52
struct sd_scale { double mx, inv; };
__device__ __forceinline__ sd_u64 sd_weight52(const double * pow, const sd_scale & e, float v) {      // with the bits of 2^52 added
    const double magic = 6755399441055744.0;                     // 1.5 2^52: the sum's last bits are the nearest integer
    double x = ((double) v - e.mx) * e.inv;
    x = __hiloint2double((int) min((uint32_t) __double2hiint(x), 0xc0440000u), __double2loint(x));
    const double t = fma(x, 1477.3197218702985, magic), k = t - magic, r = fma(k, -0.00067690154351557157, x);
    const int    n = __double2loint(t);
    const double p = fma(fma(r, 0.5, 1.0), r, 1.0) * pow[n & (SD_POW - 1)];
    const double w = __hiloint2double(__double2hiint(p) + ((n & ~(SD_POW - 1)) << 10) + (44 << 20), __double2loint(p));
    return (sd_u64) __double_as_longlong(w + 4503599627370496.0);
}
__device__ __forceinline__ sd_u64 sd_weight(const double * pow, const sd_scale & e, float v) { return sd_weight52(pow, e, v) - SD_BITS52; }
__device__ __forceinline__ sd_scale sd_scale_of(float mx, float temp) { return { (double) mx, 1.0 / fmin((double) temp, 1e30) }; }      // beyond 1e30: all alike
__device__ __forceinline__ sd_u64 sd_warp_sum(sd_u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ float sd_load(const float * p) { return __ldg(p); }
__device__ __forceinline__ float sd_load(const __nv_bfloat16 * p) { return __bfloat162float(__ldg(p)); }
__device__ __forceinline__ void sd_load8(const float * p, float (&v)[8]) {
    const float4 a = __ldg(reinterpret_cast<const float4 *>(p)), b = __ldg(reinterpret_cast<const float4 *>(p) + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void sd_load8(const __nv_bfloat16 * p, float (&v)[8]) {
    const uint4 a = __ldg(reinterpret_cast<const uint4 *>(p));
    const uint32_t u[4] = { a.x, a.y, a.z, a.w };
#pragma unroll
    for (int j = 0; j < 4; j++) { v[2 * j] = __uint_as_float(u[j] << 16); v[2 * j + 1] = __uint_as_float(u[j] & 0xffff0000u); }
}

namespace cg = cooperative_groups;

// a block's part of a row: ids lo .. hi, chunks c0 .. c1 (chunk c begins at id c * 256 - shift).  In a row whose maximum is +inf (alone), those that equal it take part
// alone, as zeros
template <typename T> struct sd_row {
    const T * l;
    int   lo, hi, V, P, part, c0, c1, shift;
    bool  alone;
    float mx;
    sd_scale one;                                                // temp 1
    __device__ __forceinline__ float see(float v) const { return !alone ? v : v == INFINITY ? 0.f : -INFINITY; }
    __device__ __forceinline__ float at(int i) const { return see(sd_load(l + i)); }
    // eight neighbours from id i on, -inf outside the row
    __device__ __forceinline__ void load(int i, float (&v)[8]) const {
        if (i >= 0 && i + 8 <= V) sd_load8(l + i, v);
        else
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = i + j >= 0 && i + j < V ? sd_load(l + i + j) : -INFINITY;
        if (alone)
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = see(v[j]);
    }
};
// f(chunk, first id of the lane, values) for the chunks of a warp, the next one under way
template <typename T, typename F> __device__ __forceinline__ void sd_walk(const sd_row<T> & R, int warp, int lane, F f) {
    int   c = R.c0 + warp, i = c * SD_CHUNK - R.shift + lane * 8;
    float a[8], b[8];
    if (c < R.c1) R.load(i, a);
    for (; c < R.c1; c += 2 * SD_WARPS, i += 2 * SD_WARPS * SD_CHUNK) {
        const bool more = c + SD_WARPS < R.c1;
        if (more) R.load(i + SD_WARPS * SD_CHUNK, b);
        f(c, i, a);
        if (c + 2 * SD_WARPS < R.c1) R.load(i + 2 * SD_WARPS * SD_CHUNK, a);
        if (more) f(c + SD_WARPS, i + SD_WARPS * SD_CHUNK, b);
    }
}

// members of a level: bin0 of l_max - l, and the order's leading bits
struct sd_level { int bin0, shift; sd_u64 prefix; };
__device__ __forceinline__ int sd_bin0(float l, float mx) { return (int) fminf((mx - l) * 64.0f, (float) (SD_BINS - 1)); }
__device__ __forceinline__ bool sd_member(float l, int i, float mx, const sd_level & L) {
    return l > -INFINITY && (L.bin0 < 0 || (sd_bin0(l, mx) == L.bin0 && (L.shift >= 64 || sd_place(l, i) >> L.shift == L.prefix)));
}

// blocks of a cluster, or the one block, meet
__device__ __forceinline__ void sd_sync(cg::cluster_group & cl, int P) { if (P > 1) cl.sync(); else __syncthreads(); }

// The place in the order of the last token that is kept: the `need`-th token (BY_MASS: the first at which the running sum reaches need_mass).  Returns it, and the sum up to and with it.
template <typename T, bool BY_MASS>
__device__ __noinline__ void sd_select(sd_shared & S, const sd_row<T> & R, cg::cluster_group & cl, uint32_t need, sd_u64 need_mass, bool want_mass, sd_u64 & thr, sd_u64 & thr_mass) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const bool mass = BY_MASS || want_mass;
    sd_level L = { -1, 64, 0 };
    sd_u64   ahead_mass = 0;
    uint32_t ahead = 0;
    // levels: bins of l_max - l; the place's bits [53..63], [42..52], [32..41], then the inverted id's [9..17], [0..8] (its bits above 17 are all set)
    for (int level = 0; level < 6; level++) {
        const int shift = level == 1 ? 53 : level == 2 ? 42 : level == 3 ? 32 : level == 4 ? 9 : 0;
        const int bins  = level < 3 ? SD_BINS : level == 3 ? 1024 : 512;
        for (int i = tid; i < SD_BINS; i += SD_THREADS) { S.count[i] = 0; S.lo[i] = 0; S.hi[i] = 0; }
        __syncthreads();
        for (int i = R.lo + tid; i < R.hi; i += SD_THREADS) {
            const float l = R.at(i);
            if (!sd_member(l, i, R.mx, L)) continue;
            // in falling order of the place: bin 0 comes first
            const int bin = level == 0 ? sd_bin0(l, R.mx) : bins - 1 - (int) (sd_place(l, i) >> shift & (bins - 1));
            atomicAdd(&S.count[bin], 1u);
            if (mass) {
                const sd_u64 w = sd_weight(S.pow, R.one, l);
                const uint32_t wl = (uint32_t) w, old = atomicAdd(&S.lo[bin], wl);
                const uint32_t wh = (uint32_t) (w >> 32) + (old + wl < old);
                if (wh) atomicAdd(&S.hi[bin], wh);
            }
        }
        cl.sync();
        // block `part` of the cluster adds up its share of the bins
        const int per = SD_BINS / R.P, b0 = R.part * per;
        uint32_t c = 0;
        sd_u64   m = 0;
        uint32_t tc[SD_BINS / SD_THREADS];
        sd_u64   tm[SD_BINS / SD_THREADS];
        const int each = max(1, per / SD_THREADS);               // neighbouring bins of a thread
#pragma unroll
        for (int j = 0; j < SD_BINS / SD_THREADS; j++) {
            tc[j] = 0; tm[j] = 0;
            const int b = b0 + tid * each + j;
            if (j < each && tid * each + j < per)
                for (int p = 0; p < R.P; p++) {
                    const sd_shared * o = cl.map_shared_rank(&S, p);
                    tc[j] += o->count[b];
                    if (mass) tm[j] += (sd_u64) o->hi[b] << 32;
                    if (mass) tm[j] += o->lo[b];
                }
            c += tc[j]; m += tm[j];
        }
        // running sums over the block's threads
        uint32_t sc = c;
        sd_u64   sm = m;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t pc = __shfl_up_sync(0xffffffffu, sc, o);
            const sd_u64   pm = __shfl_up_sync(0xffffffffu, sm, o);
            if (lane >= o) { sc += pc; sm += pm; }
        }
        if (lane == 31) { S.wcnt[warp] = sc; S.wsum[warp] = sm; }
        __syncthreads();
        uint32_t bc = 0;
        sd_u64   bm = 0;
        for (int w = 0; w < SD_WARPS; w++) {
            if (w < warp) { bc += S.wcnt[w]; bm += S.wsum[w]; }
        }
        sc += bc - c; sm += bm - m;                              // ahead of this thread's bins, in this block
        if (tid == SD_THREADS - 1) { S.own.count = sc + c; S.own.mass = sm + m; }
        if (tid == 0) S.found.bin = 0xffffffffu;
        cl.sync();
        for (int p = 0; p < R.part; p++) { const sd_shared * o = cl.map_shared_rank(&S, p); sc += o->own.count; sm += o->own.mass; }
        sc += ahead; sm += ahead_mass;
#pragma unroll
        for (int j = 0; j < SD_BINS / SD_THREADS; j++) {
            const bool here = BY_MASS ? sm < need_mass && sm + tm[j] >= need_mass : sc < need && sc + tc[j] >= need;
            if (here)
                for (int p = 0; p < R.P; p++) {
                    sd_shared * o = cl.map_shared_rank(&S, p);
                    o->found.bin = (uint32_t) (b0 + tid * each + j); o->found.count = sc; o->found.mass = sm; o->cnt = tc[j];
                }
            sc += tc[j]; sm += tm[j];
        }
        if (tid == 0) S.n_list = 0;
        cl.sync();
        const uint32_t bin = S.found.bin, n = S.cnt;
        ahead = S.found.count; ahead_mass = S.found.mass;
        if (level == 0) L.bin0 = (int) bin;
        else {
            const int width = level < 3 ? 11 : level == 3 ? 10 : 9;
            // behind the logit's bits stand the id's bits above 17, all set
            L.prefix = level == 1 ? (sd_u64) (bins - 1 - bin) : level == 4 ? (L.prefix << 14 | 0x3fffu) << width | (bins - 1 - bin) : L.prefix << width | (bins - 1 - bin);
            L.shift  = shift;
        }
        if (n <= SD_LIST || level == 5) {
            // the tokens of the bin to the first block's list, in any order
            sd_shared * lead = cl.map_shared_rank(&S, 0);
            for (int i = R.lo + tid; i < R.hi; i += SD_THREADS) {
                const float l = R.at(i);
                if (sd_member(l, i, R.mx, L)) { const uint32_t at = atomicAdd(&lead->n_list, 1u); if (at < SD_LIST) lead->list[at] = sd_place(l, i); }
            }
            cl.sync();
            if (R.part == 0) {
                if (mass) {                                      // their weights in the histogram's place, which every block has read
                    for (uint32_t j = tid; j < n; j += SD_THREADS) {
                        const sd_u64 w = sd_weight(S.pow, R.one, sd_logit(S.list[j]));
                        S.lo[j] = (uint32_t) w; S.hi[j] = (uint32_t) (w >> 32);
                    }
                    __syncthreads();
                }
                for (uint32_t j = tid; j < n; j += SD_THREADS) {
                    const sd_u64 me = S.list[j];
                    uint32_t r = ahead;
                    sd_u64   s = ahead_mass;
                    for (uint32_t o = 0; o < n; o++)
                        if (S.list[o] > me) {
                            r++;
                            if (mass) s += (sd_u64) S.hi[o] << 32 | S.lo[o];
                        }
                    const sd_u64 w = mass ? (sd_u64) S.hi[j] << 32 | S.lo[j] : 0;
                    if (BY_MASS ? s < need_mass && s + w >= need_mass : r == need - 1)
                        for (int p = 0; p < R.P; p++) { sd_shared * o = cl.map_shared_rank(&S, p); o->thr = me; o->thr_mass = s + w; }
                }
            }
            cl.sync();
            thr = S.thr; thr_mass = S.thr_mass;
            return;
        }
        cl.sync();                                               // found and cnt have been read
    }
}

// the least sum that reaches top_p of all
__device__ __forceinline__ sd_u64 sd_need(float top_p, sd_u64 mass) {
    const sd_u64 n = (sd_u64) ceil((double) top_p * (double) mass);
    return n < 1 ? 1 : n > mass ? mass : n;
}
// what a block has in all its warps: S.own
__device__ __forceinline__ void sd_block_sum(sd_shared & S, int warp, int lane, uint32_t n, sd_u64 m) {
    n = __reduce_add_sync(0xffffffffu, n);
    m = sd_warp_sum(m);
    if (lane == 0) { S.wcnt[warp] = n; S.wsum[warp] = m; }
    __syncthreads();
    if (threadIdx.x == 0) {
        uint32_t a = 0;
        sd_u64   b = 0;
        for (int w = 0; w < SD_WARPS; w++) { a += S.wcnt[w]; b += S.wsum[w]; }
        S.own.count = a; S.own.mass = b;
    }
}

// The entry of a list of m, with weights w(j), at which the running sum, in the order `ahead`, passes target: sums of 512 runs of that order (bucket), then the entries of one run among themselves.
template <typename W, typename B, typename O> __device__ __forceinline__ uint32_t sd_find(sd_shared & S, uint32_t m, sd_u64 target, W w, B bucket, O ahead) {
    static_assert(SD_THREADS == 512 && sizeof(S.fine) >= SD_LIST * 8 + 512 * 8 + SD_THREADS * 8 * 2, "room behind the weights");
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    uint32_t * lo = S.fine + SD_LIST * 2, * hi = lo + 512;
    uint16_t * sub = reinterpret_cast<uint16_t *>(hi + 512);
    lo[tid] = 0; hi[tid] = 0;
    if (tid == 0) { S.n_sub = 0; S.res = 0; }
    __syncthreads();
    for (uint32_t j = tid; j < m; j += SD_THREADS) {
        const sd_u64 v = w(j);
        if (v) {
            const int b = bucket(j);
            const uint32_t wl = (uint32_t) v, old = atomicAdd(&lo[b], wl), wh = (uint32_t) (v >> 32) + (old + wl < old);
            if (wh) atomicAdd(&hi[b], wh);
        }
    }
    __syncthreads();
    const sd_u64 mine = (sd_u64) hi[tid] << 32 | lo[tid];
    sd_u64 s = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const sd_u64 x = __shfl_up_sync(0xffffffffu, s, o); if (lane >= o) s += x; }
    if (lane == 31) S.wsum[warp] = s;
    __syncthreads();
    s -= mine;
    for (int x = 0; x < warp; x++) s += S.wsum[x];
    if (target >= s && target < s + mine) { S.found.bin = (uint32_t) tid; S.pre = s; }
    __syncthreads();
    const int at = (int) S.found.bin;
    for (uint32_t j = tid; j < m; j += SD_THREADS) if (w(j) && bucket(j) == at) sub[atomicAdd(&S.n_sub, 1u)] = (uint16_t) j;
    __syncthreads();
    const uint32_t n = S.n_sub;
    for (uint32_t a = tid; a < n; a += SD_THREADS) {
        const uint32_t j = sub[a];
        s = S.pre;
        for (uint32_t o = 0; o < n; o++) s += ahead(sub[o], j) ? w(sub[o]) : 0;
        if (target >= s && target < s + w(j)) S.res = j;
    }
    __syncthreads();
    return S.res;
}
// the other blocks' lists behind the first one's, by that; their sums of masses
__device__ __forceinline__ void sd_join(sd_shared & S, cg::cluster_group & cl, int P, uint32_t & m, sd_u64 & mass) {
    m = S.n_list;
    mass = S.own.mass;
#pragma unroll 1
    for (int p = 1; p < P; p++) {
        const sd_shared * o = cl.map_shared_rank(&S, p);
        const uint32_t n = o->n_list;
        for (uint32_t j = threadIdx.x; j < n; j += SD_THREADS) S.list[m + j] = o->list[j];
        m += n;
        mass += o->own.mass;
    }
    __syncthreads();
}

// how many tokens of the row take part
template <typename T> __device__ __noinline__ uint32_t sd_count(sd_shared & S, const sd_row<T> & R, cg::cluster_group & cl) {
    uint32_t n = 0;
    for (int i = R.lo + threadIdx.x; i < R.hi; i += SD_THREADS) n += R.at(i) > -INFINITY;
    __syncthreads();
    sd_block_sum(S, threadIdx.x >> 5, threadIdx.x & 31, n, 0);
    sd_sync(cl, R.P);
    n = 0;
    for (int p = 0; p < R.P; p++) n += cl.map_shared_rank(&S, p)->own.count;
    sd_sync(cl, R.P);
    return n;
}

template <typename T>
__global__ void __launch_bounds__(SD_THREADS, 2) sample_draw_kernel(const T * __restrict__ logits, int64_t ld, int V, const pib_sample_params * __restrict__ params, const float * __restrict__ us,
                                                                    int32_t * __restrict__ ids, float * __restrict__ ps, int32_t * __restrict__ kepts) {
    extern __shared__ __align__(16) uint8_t sd_dsm[];
    sd_shared & S = *reinterpret_cast<sd_shared *>(sd_dsm);
    cg::cluster_group cl = cg::this_cluster();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, row = blockIdx.x;
    sd_row<T> R;
    R.l = logits + row * ld; R.V = V; R.P = gridDim.y; R.part = blockIdx.y; R.alone = false;
    R.shift = (int) (((uintptr_t) R.l & (8 * sizeof(T) - 1)) / sizeof(T));
    const int chunks = (V + R.shift + SD_CHUNK - 1) / SD_CHUNK;
    R.c0 = chunks * R.part / R.P; R.c1 = chunks * (R.part + 1) / R.P;
    R.lo = max(0, R.c0 * SD_CHUNK - R.shift); R.hi = min(V, R.c1 * SD_CHUNK - R.shift);
    if (R.P > 1) cl.barrier_arrive();                            // this block has started: waited for ahead of the first store to another one's shared memory
    for (int j = tid; j < SD_POW; j += SD_THREADS) S.pow[j] = exp2((double) j / SD_POW);
    for (int i = tid; i < SD_FINE; i += SD_THREADS) S.fine[i] = 0;
    pib_pdl_wait();
    pib_pdl_trigger();
    const pib_sample_params q = params[row];
    const double u = (double) us[row];
    // 1: the row's maximum; per thread the first eight that hold it
    float mx = -INFINITY;
    int   arg = 0x7fffffff;
    sd_walk(R, warp, lane, [&](int, int i, const float (&v)[8]) {
        const float m = fmaxf(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])), fmaxf(fmaxf(v[4], v[5]), fmaxf(v[6], v[7])));
        if (m > mx) { mx = m; arg = i; }
    });
    const bool first = !(q.temp > 0.f) || q.top_k == 1 || q.min_p > 1.f || !(q.top_p > 0.f || q.top_p != q.top_p), by_k = q.top_k > 0 && q.top_k < V, by_p = q.top_p < 1.f;
    if (R.P > 1) cl.barrier_wait();
    if (by_k) cl.map_shared_rank(&S, 0)->tmax[R.part * SD_THREADS + tid] = mx;
    const float best = warp_max(mx);
    arg = __reduce_min_sync(0xffffffffu, mx == best ? arg : 0x7fffffff);
    if (lane == 0) { S.wmax[warp] = best; S.warg[warp] = arg; }
    __syncthreads();
    if (warp == 0) {
        const float v = lane < SD_WARPS ? S.wmax[lane] : -INFINITY, b = warp_max(v);
        const int   a = __reduce_min_sync(0xffffffffu, lane < SD_WARPS && v == b ? S.warg[lane] : 0x7fffffff);
        if (lane == 0) { S.max = b; S.arg = a; }
    }
    sd_sync(cl, R.P);
    mx = -INFINITY; arg = 0x7fffffff;
    for (int p = 0; p < R.P; p++) {
        const sd_shared * o = cl.map_shared_rank(&S, p);
        if (o->max > mx) { mx = o->max; arg = o->arg; }
    }
    const bool none = mx == -INFINITY;
    if (none || first) {
        if (R.part == 0 && tid == 0) {
            if (!none) while (arg < 0 || !(sd_load(R.l + arg) == mx)) arg++;         // the first of the eight
            ids[row] = none ? -1 : arg;
            if (ps) ps[row] = none ? 0.f : 1.f;
            if (kepts) kepts[row] = none ? 0 : 1;
        }
        sd_sync(cl, R.P);                                               // the other blocks have read this one's maximum
        return;
    }
    R.alone = mx == INFINITY;
    if (R.alone) mx = 0.f;
    const sd_scale tempered = sd_scale_of(mx, q.temp);
    R.one = sd_scale_of(mx, 1.f);
    R.mx = mx;
    // what is kept: logits above kl, and those equal to it up to id ki
    float kl = -INFINITY;
    int   ki = INT_MIN;
    if (q.min_p > 0.f) { kl = sd_min_p(q.min_p, mx); ki = 0x7fffffff; }
    auto kept = [&](float v, int i) { return v > kl || (v == kl && i <= ki); };
    auto by_id = [&](uint32_t a, uint32_t b) { return (uint32_t) S.list[a] > (uint32_t) S.list[b]; };           // inverted ids: larger is lower
    auto by_place = [&](uint32_t a, uint32_t b) { return S.list[a] > S.list[b]; };
    auto logit = [&](uint32_t j) { return sd_logit(S.list[j]); };
    auto weight_of = [&](uint32_t j) { return S.w[j]; };
    auto goal = [&](sd_u64 total) { const sd_u64 t = u > 0.0 ? (sd_u64) fmin(u * (double) total, 9.0e18) : 0; return t >= total ? total - 1 : t; };
    sd_u64 thr = 0, mass = 0;
    bool   summed = false;                                       // the chunks' sums are there
    uint32_t cnt = 0;
    sd_u64 need = 0;
    const bool bins = by_k ? q.top_k > R.P * SD_THREADS / 2 : by_p;
    if (bins) {
        // 2: counts of the bins; for top-p the sum of all weights
        uint32_t n = 0;
        sd_walk(R, warp, lane, [&](int, int, const float (&v)[8]) {
            sd_u64 s = 0;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                if (v[j] > -INFINITY) { n++; atomicAdd(&S.fine[sd_fine(v[j], mx)], 1u); }
                if (!by_k) s += sd_weight52(S.pow, R.one, fmaxf(v[j], -INFINITY));           // what is no number as -inf
            }
            if (!by_k) mass += s - 8 * SD_BITS52;
        });
        sd_block_sum(S, warp, lane, n, mass);
        sd_sync(cl, R.P);
        n = 0; mass = 0;
        for (int p = 0; p < R.P; p++) { const sd_shared * o = cl.map_shared_rank(&S, p); n += o->own.count; mass += o->own.mass; }
        // block `part` of the cluster adds up its share of the bins: counts, and the most that their tokens can weigh
        need = sd_need(q.top_p, mass);
        const uint32_t k = by_k ? min((uint32_t) q.top_k, n) : 0;
        const double want = (double) need;
        const int per = SD_FINE / R.P, each = per / SD_THREADS, b0 = R.part * per + tid * each;
        // a token of bin b weighs at most 2^44 e^(-b / 256), rounded: from bin to bin by a factor (a weight formed for each bin: 300 rows of 50 257 with top-p 142 us instead of 139).  The sums are
        // whole numbers: wherever a thread's or a block's bins begin they are the same, and one thread of the cluster finds each border
        const double fall = 0.99610136947011749, edge = by_k ? 0.0 : exp(-(double) b0 / 256.0) * 17592186044416.0;
        auto most_of = [&](double w, uint32_t c) { return (sd_u64) c * ((sd_u64) __double_as_longlong(w + (4503599627370496.0 + 1.0)) - SD_BITS52); };
        uint32_t sc = 0;
        sd_u64   sb = 0;
        // (loops that are not unrolled: most of a short row's time is code that runs once, and its way from memory)
        double w = edge;
#pragma unroll 1
        for (int b = b0; b < b0 + each; b += 2) {
            uint2 c = *reinterpret_cast<const uint2 *>(S.fine + b), o[8];
#pragma unroll
            for (int p = 0; p < 8; p++) o[p] = p < R.P && p != R.part ? *reinterpret_cast<const uint2 *>(cl.map_shared_rank(&S, p)->fine + b) : make_uint2(0, 0);
#pragma unroll
            for (int p = 0; p < 8; p++) { c.x += o[p].x; c.y += o[p].y; }
            *reinterpret_cast<uint2 *>(S.fine + b) = c;          // no other block reads this one's share here
            sc += c.x + c.y;
            sb += most_of(w, c.x);
            w *= fall;
            sb += most_of(w, c.y);
            w *= fall;
        }
        const uint32_t mine = sc;
        const sd_u64   mine_b = sb;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t pc = __shfl_up_sync(0xffffffffu, sc, o);
            const sd_u64   pb = __shfl_up_sync(0xffffffffu, sb, o);
            if (lane >= o) { sc += pc; sb += pb; }
        }
        __syncthreads();
        if (lane == 31) { S.wcnt[warp] = sc; S.wbound[warp] = sb; }
        __syncthreads();
        for (int w = 0; w < warp; w++) { sc += S.wcnt[w]; sb += S.wbound[w]; }
        if (tid == SD_THREADS - 1) { S.cnt = sc; S.bound = sb; }
        if (tid == 0) { S.first = S.last = SD_FINE; S.n_list = 0; S.n_first = S.n_last = 0; }
        sd_sync(cl, R.P);
        sc -= mine; sb -= mine_b;
        sd_u64 most = 0;
        for (int p = 0; p < R.P; p++) {
            const sd_shared * o = cl.map_shared_rank(&S, p);
            if (p < R.part) { sc += o->cnt; sb += o->bound; }
            most += o->bound;
        }
        // The bins between which the threshold lies.  What lies up to a bin weighs at most the sum of the bounds, `b`; at least e^(-1/256) of it, and at least all less the bounds behind it.
        // (4.1e-6: l_max - l is rounded to fp32, half a unit of 2^-19 at most; weights to integers, one unit for each of 2^18 tokens where the first alone weighs 2^44.  The last bin holds what lies
        // further away too, which weighs less than a unit each)
        auto least = [&](sd_u64 b) { return fmax((double) b * (0.99610136947 * (1.0 - 4.1e-6)), (double) mass - (double) (most - b) * (1.0 + 4.1e-6)); };
        const double reach = want * (1.0 - 4.1e-6);
        w = edge;
#pragma unroll 1
        for (int b = b0; b < b0 + each; b++, w *= fall) {
            const uint32_t c = S.fine[b];
            if (!c) continue;
            const sd_u64 nb = sb + most_of(w, c);
            const bool   f = by_k ? sc < k && sc + c >= k : (double) sb < reach && (double) nb >= reach, l = by_k ? f : (sc == 0 || least(sb) < want) && least(nb) >= want;
            if (f || l)
                for (int p = 0; p < R.P; p++) {
                    sd_shared * o = cl.map_shared_rank(&S, p);
                    if (f) { o->first = (uint32_t) b; o->n_first = sc; }
                    if (l) { o->last = (uint32_t) b; o->n_last = sc + c; }
                }
            sc += c; sb = nb;
        }
        sd_sync(cl, R.P);
    }
    if (by_k) {
        // otherwise 2: the k-th of the threads' maxima, which k tokens at least reach; as long as those are few, not many more do
        if (!bins) {
            if (tid == 0) { S.n_list = 0; S.bound_k = -INFINITY; }
            sd_sync(cl, R.P);
        } else if (tid == 0) S.bound_k = S.n_last <= SD_LIST ? sd_bin_floor((int) S.last, mx) : -INFINITY;
        if (!bins && R.part == 0) {
            const uint32_t m = (uint32_t) (R.P * SD_THREADS);
            uint32_t have = 0;
            if (R.alone) for (uint32_t j = tid; j < m; j += SD_THREADS) S.tmax[j] = R.see(S.tmax[j]);
            for (uint32_t j = tid; j < m; j += SD_THREADS) have += S.tmax[j] > -INFINITY;
            sd_block_sum(S, warp, lane, have, 0);
            __syncthreads();
            if ((uint32_t) q.top_k <= S.own.count) {
                const uint32_t j = sd_find(S, m, (sd_u64) q.top_k - 1, [&](uint32_t e) { return (sd_u64) (S.tmax[e] > -INFINITY); }, [&](uint32_t e) { return sd_fine(S.tmax[e], mx) * 512 / SD_FINE; },
                                           [&](uint32_t a, uint32_t b) { return S.tmax[a] > S.tmax[b] || (S.tmax[a] == S.tmax[b] && a < b); });
                if (tid == 0) for (int p = 0; p < R.P; p++) cl.map_shared_rank(&S, p)->bound_k = S.tmax[j];
            }
        }
        if (bins) __syncthreads(); else sd_sync(cl, R.P);
        // 3: gather them
        const float bound = S.bound_k;
        sd_walk(R, warp, lane, [&](int, int i, const float (&v)[8]) {
            uint32_t near = 0;
#pragma unroll
            for (int j = 0; j < 8; j++) near |= (uint32_t) (v[j] >= bound && v[j] > -INFINITY) << j;
            if (near) {
                uint32_t at = atomicAdd(&S.n_list, (uint32_t) __popc(near));
#pragma unroll
                for (int j = 0; j < 8; j++) if (near >> j & 1) { if (at < SD_LIST) S.list[at] = sd_place(v[j], i + j); at++; }
            }
        });
        __syncthreads();
        if (tid == 0) S.own.mass = 0;
        sd_sync(cl, R.P);
        uint32_t n = 0;
        for (int p = 0; p < R.P; p++) n += cl.map_shared_rank(&S, p)->n_list;
        const uint32_t k = min((uint32_t) q.top_k, n);
        if (n <= SD_LIST) {
            // everything that is kept lies in the list
            if (R.part == 0) {
                uint32_t m;
                sd_join(S, cl, R.P, m, mass);
                const int span = sd_fine(fmaxf(bound, -FLT_MAX), mx) + 1;
                auto run = [&](uint32_t e) { return sd_fine(logit(e), mx) * 512 / span; };
                if (m > k) thr = S.list[sd_find(S, m, k - 1, [&](uint32_t) { return (sd_u64) 1; }, run, by_place)];
                sd_u64 sum = 0;
                if (by_p) {
                    for (uint32_t j = tid; j < m; j += SD_THREADS) {
                        const sd_u64 w = S.list[j] >= thr ? sd_weight(S.pow, R.one, logit(j)) : 0;
                        S.w[j] = w;
                        sum += w;
                    }
                    sd_block_sum(S, warp, lane, 0, sum);
                    __syncthreads();
                    thr = S.list[sd_find(S, m, sd_need(q.top_p, S.own.mass) - 1, weight_of, run, by_place)];
                    sum = 0;
                }
                const float tl = sd_logit(thr);
                if (thr && !(kl > tl)) { kl = tl; ki = (int) ~(uint32_t) thr; }
                for (uint32_t j = tid; j < m; j += SD_THREADS) {
                    const float  l = logit(j);
                    const bool   in = kept(l, (int) ~(uint32_t) S.list[j]);
                    const sd_u64 w = in ? sd_weight(S.pow, tempered, l) : 0;
                    S.w[j] = w;
                    cnt += in; sum += w;
                }
                sd_block_sum(S, warp, lane, cnt, sum);
                __syncthreads();
                const sd_u64   total = S.own.mass;
                const uint32_t j = sd_find(S, m, goal(total), weight_of, [&](uint32_t e) { return (int) ((sd_u64) ~(uint32_t) S.list[e] * 512u / (uint32_t) V); }, by_id);
                if (tid == 0) {
                    ids[row] = (int32_t) ~(uint32_t) S.list[j];
                    if (ps) ps[row] = (float) ((double) S.w[j] / (double) total);
                    if (kepts) kepts[row] = (int32_t) S.own.count;
                }
            }
            sd_sync(cl, R.P);                                    // the first block has read the others' lists
            return;
        }
        // a long list is left to sd_select
        sd_select<T, false>(S, R, cl, min((uint32_t) q.top_k, sd_count(S, R, cl)), 0, by_p, thr, mass);
        __syncthreads();
        if (by_p) {
            sd_u64 t, tm;
            sd_select<T, true>(S, R, cl, 0, sd_need(q.top_p, mass), true, t, tm);
            thr = t > thr ? t : thr;
        }
    } else if (by_p) {
        const uint32_t b_first = S.first, b_last = S.last;
        if (b_first < SD_FINE && b_last < SD_FINE && S.n_last - S.n_first <= SD_LIST) {
            // 3: gather the tokens of those bins; of what lies ahead of them the sum, and the chunks' sums of its weights in the draw
            const bool same = q.temp == 1.f && !(kl > -INFINITY);
            const float near_v = sd_bin_floor(b_last, mx), far_v = b_first ? sd_bin_floor(b_first - 1, mx) : INFINITY;
            sd_u64 ahead = 0;
            sd_walk(R, warp, lane, [&](int c, int i, const float (&v)[8]) {
                uint32_t near = 0, far = 0, in = 0;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    far  |= (uint32_t) (v[j] >= far_v) << j;
                    near |= (uint32_t) (v[j] >= near_v && v[j] < far_v) << j;
                    in   |= (uint32_t) (v[j] >= far_v && kept(v[j], i + j)) << j;
                }
                if (near) {
                    uint32_t at = atomicAdd(&S.n_list, (uint32_t) __popc(near));
#pragma unroll
                    for (int j = 0; j < 8; j++) if (near >> j & 1) S.list[at++] = sd_place(v[j], i + j);
                }
                sd_u64 s = 0, d = 0;
                if (far) {
#pragma unroll
                    for (int j = 0; j < 8; j++) s += sd_weight52(S.pow, R.one, far >> j & 1 ? v[j] : -INFINITY);
                    s -= 8 * SD_BITS52;
                }
                if (same) d = s;
                else if (in) {
#pragma unroll
                    for (int j = 0; j < 8; j++) d += sd_weight52(S.pow, tempered, in >> j & 1 ? v[j] : -INFINITY);
                    d -= 8 * SD_BITS52;
                }
                ahead += s;
                cnt += __popc(in);
                d = sd_warp_sum(d);
                if (lane == 0) S.chunk[c - R.c0] = d;
            });
            sd_block_sum(S, warp, lane, cnt, ahead);
            sd_sync(cl, R.P);
            if (R.part == 0) {
                uint32_t m;
                sd_join(S, cl, R.P, m, ahead);
                for (uint32_t j = tid; j < m; j += SD_THREADS) S.w[j] = sd_weight(S.pow, R.one, logit(j));
                __syncthreads();
                thr = S.list[sd_find(S, m, need - 1 - ahead, weight_of, [&](uint32_t e) { return (sd_fine(logit(e), mx) - (int) b_first) * 512 / (int) (b_last - b_first + 1); }, by_place)];
                const float tl = sd_logit(thr);
                if (!(kl > tl)) { kl = tl; ki = (int) ~(uint32_t) thr; }
                // those of the list that are kept join their chunks
                cnt = 0;
                for (uint32_t j = tid; j < m; j += SD_THREADS) {
                    const int   i = (int) ~(uint32_t) S.list[j], c = (i + R.shift) / SD_CHUNK;
                    const float l = logit(j);
                    if (!kept(l, i)) continue;
                    cnt++;
                    int p = 0;
                    while (c >= chunks * (p + 1) / R.P) p++;
                    atomicAdd(&cl.map_shared_rank(&S, p)->chunk[c - chunks * p / R.P], sd_weight(S.pow, tempered, l));
                }
                cnt = __reduce_add_sync(0xffffffffu, cnt);
                if (lane == 0 && cnt) atomicAdd(&S.own.count, cnt);
                if (tid == 0) for (int p = 0; p < R.P; p++) cl.map_shared_rank(&S, p)->thr = thr;
            }
            sd_sync(cl, R.P);
            thr = S.thr;
            sd_u64 sum = 0;
            for (int c = tid; c < R.c1 - R.c0; c += SD_THREADS) sum += S.chunk[c];
            cnt = tid == 0 ? S.own.count : 0;
            __syncthreads();
            sd_block_sum(S, warp, lane, cnt, sum);
            summed = true;
        } else {
            sd_u64 tm;
            sd_select<T, true>(S, R, cl, 0, need, true, thr, tm);
        }
    }
    if (thr) {
        const float tl = sd_logit(thr);
        if (!(kl > tl)) { kl = tl; ki = (int) ~(uint32_t) thr; }     // min-p lets equal logits through together: the border is the other's
    }
    if (!summed) {
        // 4: weights of what is kept, per chunk
        sd_u64 sum = 0;
        cnt = 0;
        __syncthreads();
        sd_walk(R, warp, lane, [&](int c, int i, const float (&v)[8]) {
            sd_u64   s = 0;
            uint32_t any = 0;
#pragma unroll
            for (int j = 0; j < 8; j++) any |= (uint32_t) kept(v[j], i + j) << j;
            if (any) {
#pragma unroll
                for (int j = 0; j < 8; j++) s += sd_weight52(S.pow, tempered, any >> j & 1 ? v[j] : -INFINITY);
                s -= 8 * SD_BITS52;
            }
            cnt += __popc(any);
            s = sd_warp_sum(s);
            if (lane == 0) { S.chunk[c - R.c0] = s; sum += s; }
        });
        sd_block_sum(S, warp, lane, cnt, sum);
    }
    sd_sync(cl, R.P);
    sd_u64 total = 0, ahead = 0;
    cnt = 0;
    for (int p = 0; p < R.P; p++) {
        const sd_shared * o = cl.map_shared_rank(&S, p);
        if (p < R.part) ahead += o->own.mass;
        total += o->own.mass; cnt += o->own.count;
    }
    const sd_u64 target = goal(total);
    if (warp == 0 && target >= ahead && target < ahead + S.own.mass) {      // one warp of the cluster: the chunk, then the token
        for (int c0 = R.c0; c0 < R.c1; c0 += 32) {
            const sd_u64 w = c0 + lane < R.c1 ? S.chunk[c0 + lane - R.c0] : 0;
            sd_u64 s = w;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) { const sd_u64 x = __shfl_up_sync(0xffffffffu, s, o); if (lane >= o) s += x; }
            const unsigned over = __ballot_sync(0xffffffffu, ahead + s > target);
            if (!over) { ahead += __shfl_sync(0xffffffffu, s, 31); continue; }
            const int who = __ffs((int) over) - 1;
            ahead += __shfl_sync(0xffffffffu, s - w, who);
            const int i = (c0 + who) * SD_CHUNK - R.shift + lane * 8;
            float  v[8];
            sd_u64 x[8], mine = 0;
            R.load(i, v);
#pragma unroll
            for (int j = 0; j < 8; j++) { x[j] = kept(v[j], i + j) ? sd_weight(S.pow, tempered, v[j]) : 0; mine += x[j]; }
            s = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) { const sd_u64 y = __shfl_up_sync(0xffffffffu, s, o); if (lane >= o) s += y; }
            s += ahead - mine;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                if (target >= s && target < s + x[j]) {
                    ids[row] = i + j;
                    if (ps) ps[row] = (float) ((double) x[j] / (double) total);
                    if (kepts) kepts[row] = (int32_t) cnt;
                }
                s += x[j];
            }
            break;
        }
    }
    sd_sync(cl, R.P);                                                   // the sums have been read
}

template <typename T>
static int sd_launch(const void * logits, int64_t ld, int rows, int V, const pib_sample_params * params, const float * u, int32_t * ids, float * p, int32_t * kept, cudaStream_t st) {
    static pib_per_device attrs;
    PIB_CHECK(attrs.once([&] { return cudaFuncSetAttribute(sample_draw_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int) sizeof(sd_shared)); }));
    // Blocks of a row: as many as run at a time (two per SM), a slice holding 4096 ids or more.  us for 1, 2, 4, 8 blocks, top-p 0.9 and top-k 40:
    //   1 row of 32 000      47 34 27 24   15 15 14 16        64 rows of 128 256   130  80  69  97   32 27 26 46
    //   64 rows of 32 000    48 36 35 64   15 17 18 39        300 rows of 50 257   143 146 193 330   46 61 94 194
    //   40 rows of 8 000     28 25 28 53   11 14 17 36        100 rows of 128 256  132 108 111 163   35 33 47 81
    int P = 1;
    while (P < 8 && (int64_t) rows * P * 2 <= 2 * pib_num_sms() && V >= P * 2 * SD_SLICE) P <<= 1;
    for (int r0 = 0; r0 < rows; r0 += 1 << 20) {
        const int n = rows - r0 < 1 << 20 ? rows - r0 : 1 << 20;
        PIB_CHECK(pib_launch_cluster(sample_draw_kernel<T>, dim3((unsigned) n, (unsigned) P), dim3(SD_THREADS), dim3(1, (unsigned) P, 1), sizeof(sd_shared), st, (const T *) logits + r0 * ld, ld, V,
                                     params + r0, u + r0, ids + r0, p ? p + r0 : nullptr, kept ? kept + r0 : nullptr));
    }
    return PIB_OK;
}

extern "C" int pib_sample(int type, const void * logits, int64_t ld, int rows, int n_vocab, const pib_sample_params * params, const float * u, int32_t * ids, float * p, int32_t * kept, pib_stream s) {
    if (rows == 0) return PIB_OK;
    if ((type != PIB_TYPE_F32 && type != PIB_TYPE_BF16) || !logits || !params || !u || !ids || rows < 0 || n_vocab < 1 || n_vocab > PIB_SAMPLE_MAX_VOCAB || (rows > 1 && ld < n_vocab) ||
        ((uintptr_t) logits & (type == PIB_TYPE_F32 ? 3 : 1)) || (((uintptr_t) params | (uintptr_t) u | (uintptr_t) ids | (uintptr_t) p | (uintptr_t) kept) & 3)) {
        pib_set_error("pib_sample: bad arguments (type %d, %d rows of %d, %lld apart; at most %d tokens)", type, rows, n_vocab, (long long) ld, PIB_SAMPLE_MAX_VOCAB);
        return PIB_ERR_ARG;
    }
    if (type == PIB_TYPE_F32) return sd_launch<float>(logits, ld, rows, n_vocab, params, u, ids, p, kept, (cudaStream_t) s);
    return sd_launch<__nv_bfloat16>(logits, ld, rows, n_vocab, params, u, ids, p, kept, (cudaStream_t) s);
}
