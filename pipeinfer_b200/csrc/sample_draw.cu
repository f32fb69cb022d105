// sample_draw.cu -- a token of each row of logits: top-k, top-p, min-p, temperature, drawn with a given number.
//
// A row's tokens are ordered by (logit descending, id ascending); every truncation keeps a run from the front of that order, so it is one threshold in it, and nothing is sorted.  With
// w = e^(l - l_max) in 64 bits, rounded to a multiple of 2^-44: sums of up to 2^18 such numbers are exact in 64-bit integers, so no result depends on which thread or block added first.
//   top-k   the threshold is the k-th token of the order
//   top-p   the first token at which the running sum of w reaches top_p times that of what top-k left
//   min-p   w >= min_p
//   draw    weights e^((l - l_max) / temp) of what is kept, the first id at which their running sum exceeds u times the total
// A threshold is found in levels: a histogram (counts, and sums for top-p) over 2048 bins of l_max - l, 1/64 wide, gives the bin that holds it; the bin's tokens, if they are few, are gathered
// and each finds what lies ahead of it by comparing with all; if they are many, histograms over the order's own bits (11, 11 and 10 of the logit, 9 and 9 of the id) narrow it first.
// A row is divided over the P blocks of a thread-block cluster in slices of neighbouring ids; the blocks meet through distributed shared memory.
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include "engine.cuh"

#define SD_THREADS 512
#define SD_WARPS   (SD_THREADS / 32)
#define SD_BINS    2048
#define SD_LIST    2048
#define SD_ONE     17592186044416.0          // 2^44

typedef unsigned long long sd_u64;

struct sd_range { sd_u64 mass; uint32_t count, bin; };
struct sd_shared {
    uint32_t count[SD_BINS], lo[SD_BINS], hi[SD_BINS];           // sums in two 32-bit parts: lo's carry goes to hi
    sd_u64   list[SD_LIST];
    sd_u64   wsum[SD_WARPS], sum;                                // of a block's warps, of the block
    uint32_t wcnt[SD_WARPS], cnt, n_list;
    float    wmax[SD_WARPS], max;
    int      warg[SD_WARPS], arg;
    sd_range own, found;                                         // a block's bins; the bin that holds the threshold, and what lies ahead of it
    sd_u64   thr, thr_mass;                                      // the threshold in the order, and the mass up to it
};

__device__ __forceinline__ uint32_t sd_key(float v) { const uint32_t u = __float_as_uint(v + 0.0f); return u & 0x80000000u ? ~u : u | 0x80000000u; }
// place in the order: larger comes first
__device__ __forceinline__ sd_u64 sd_place(float v, int id) { return (sd_u64) sd_key(v) << 32 | (uint32_t) ~id; }
__device__ __forceinline__ sd_u64 sd_fixed(double w) { return (sd_u64) __double2ll_rn(w * SD_ONE); }
__device__ __forceinline__ double sd_rel(float l, float mx) { return l == mx ? 0.0 : (double) l - (double) mx; }
__device__ __forceinline__ sd_u64 sd_warp_sum(sd_u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// what is no number and, beside +inf, everything finite takes no part
__device__ __forceinline__ float sd_value(float v, float mx) { return v != v || (mx == INFINITY && v != mx) ? -INFINITY : v; }
__device__ __forceinline__ float sd_load(const float * p) { return __ldg(p); }
__device__ __forceinline__ float sd_load(const __nv_bfloat16 * p) { return __bfloat162float(__ldg(p)); }

namespace cg = cooperative_groups;

template <typename T> struct sd_row {
    const T * l;
    int   lo, hi, V, P, part;
    float mx;
    __device__ __forceinline__ float at(int i) const { return sd_value(sd_load(l + i), mx); }
};

// members of a level: bin0 of l_max - l, and the order's leading bits
struct sd_level { int bin0, shift; sd_u64 prefix; };
__device__ __forceinline__ int sd_bin0(float l, float mx) { return l == mx ? 0 : (int) fminf((mx - l) * 64.0f, (float) (SD_BINS - 1)); }
__device__ __forceinline__ bool sd_member(float l, int i, float mx, const sd_level & L) {
    return l > -INFINITY && (L.bin0 < 0 || (sd_bin0(l, mx) == L.bin0 && (L.shift >= 64 || sd_place(l, i) >> L.shift == L.prefix)));
}

// The place in the order of the last token that is kept: the `need`-th token (BY_MASS: the first at which the running sum reaches need_mass).  Returns it, and the sum up to and with it.
template <typename T, bool BY_MASS>
__device__ void sd_select(sd_shared & S, const sd_row<T> & R, cg::cluster_group & cl, uint32_t need, sd_u64 need_mass, bool want_mass, sd_u64 & thr, sd_u64 & thr_mass) {
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
                const sd_u64 w = sd_fixed(exp(sd_rel(l, R.mx)));
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
                        const uint32_t k = (uint32_t) (S.list[j] >> 32);
                        const sd_u64   w = sd_fixed(exp(sd_rel(__uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k), R.mx)));
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

template <typename T>
__global__ void __launch_bounds__(SD_THREADS) sample_draw_kernel(const T * __restrict__ logits, int64_t ld, int V, const pib_sample_params * __restrict__ params, const float * __restrict__ us,
                                                                 int32_t * __restrict__ ids, float * __restrict__ ps, int32_t * __restrict__ kepts) {
    extern __shared__ __align__(16) uint8_t sd_dsm[];
    sd_shared & S = *reinterpret_cast<sd_shared *>(sd_dsm);
    cg::cluster_group cl = cg::this_cluster();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, row = blockIdx.x;
    sd_row<T> R;
    R.l = logits + row * ld; R.V = V; R.P = gridDim.y; R.part = blockIdx.y;
    R.lo = (int) ((long long) V * R.part / R.P); R.hi = (int) ((long long) V * (R.part + 1) / R.P);
    R.mx = 0.f;
    pib_pdl_wait();
    pib_pdl_trigger();
    const pib_sample_params q = params[row];
    // the row's maximum and its first place
    float mx = -INFINITY;
    int   arg = 0x7fffffff;
    for (int i = R.lo + tid; i < R.hi; i += SD_THREADS) { const float v = sd_load(R.l + i); if (v > mx) { mx = v; arg = i; } }
    const float best = warp_max(mx);
    arg = __reduce_min_sync(0xffffffffu, mx == best ? arg : 0x7fffffff);
    if (lane == 0) { S.wmax[warp] = best; S.warg[warp] = arg; }
    __syncthreads();
    if (warp == 0) {
        const float v = lane < SD_WARPS ? S.wmax[lane] : -INFINITY, b = warp_max(v);
        const int   a = __reduce_min_sync(0xffffffffu, lane < SD_WARPS && v == b ? S.warg[lane] : 0x7fffffff);
        if (lane == 0) { S.max = b; S.arg = a; }
    }
    cl.sync();
    mx = -INFINITY; arg = 0x7fffffff;
    for (int p = 0; p < R.P; p++) {
        const sd_shared * o = cl.map_shared_rank(&S, p);
        if (o->max > mx) { mx = o->max; arg = o->arg; }
    }
    R.mx = mx;
    const bool none = mx == -INFINITY, first = !(q.temp > 0.f) || q.top_k == 1 || q.min_p > 1.f || !(q.top_p > 0.f || q.top_p != q.top_p);
    if (none || first) {
        if (R.part == 0 && tid == 0) {
            ids[row] = none ? -1 : arg;
            if (ps) ps[row] = none ? 0.f : 1.f;
            if (kepts) kepts[row] = none ? 0 : 1;
        }
        cl.sync();                                               // the other blocks have read this one's maximum
        return;
    }
    // what takes part: all, or fewer than top_k of them anyway
    const bool by_k = q.top_k > 0 && q.top_k < V, by_p = q.top_p < 1.f;
    sd_u64 thr = 0, mass = 0;
    if (by_k || by_p) {
        uint32_t n = 0;
        sd_u64   m = 0;
        for (int i = R.lo + tid; i < R.hi; i += SD_THREADS) {
            const float l = R.at(i);
            if (l > -INFINITY) { n++; if (by_p && !by_k) m += sd_fixed(exp(sd_rel(l, mx))); }
        }
        n = __reduce_add_sync(0xffffffffu, n);
        m = sd_warp_sum(m);
        if (lane == 0) { S.wcnt[warp] = n; S.wsum[warp] = m; }
        __syncthreads();
        if (tid == 0) {
            uint32_t a = 0;
            sd_u64   b = 0;
            for (int w = 0; w < SD_WARPS; w++) { a += S.wcnt[w]; b += S.wsum[w]; }
            S.own.count = a; S.own.mass = b;
        }
        cl.sync();
        n = 0;
        for (int p = 0; p < R.P; p++) { const sd_shared * o = cl.map_shared_rank(&S, p); n += o->own.count; mass += o->own.mass; }
        cl.sync();
        if (by_k) {
            const uint32_t k = (uint32_t) q.top_k;
            sd_select<T, false>(S, R, cl, k < n ? k : n, 0, by_p, thr, mass);
            __syncthreads();
        }
        if (by_p) {
            // the least sum that reaches top_p times the mass
            const double want = (double) q.top_p * (double) mass;
            sd_u64 need = (sd_u64) ceil(want), t, tm;
            need = need < 1 ? 1 : need > mass ? mass : need;
            sd_select<T, true>(S, R, cl, 0, need, true, t, tm);
            thr = t > thr ? t : thr;
        }
    }
    // weights of what is kept, per warp of neighbouring ids
    const double inv_t = 1.0 / (double) q.temp, min_p = q.min_p > 0.f ? (double) q.min_p : 0.0;
    const int    span = (R.hi - R.lo + SD_WARPS - 1) / SD_WARPS, w0 = R.lo + warp * span, w1 = min(R.hi, w0 + span);
    auto weight = [&](int i, bool & kept) -> sd_u64 {
        const float l = R.at(i);
        kept = l > -INFINITY && sd_place(l, i) >= thr;
        if (!kept) return 0;
        const double rel = sd_rel(l, mx);
        kept = min_p == 0.0 || rel == 0.0 || exp(rel) >= min_p;
        return kept ? sd_fixed(exp(rel * inv_t)) : 0;
    };
    sd_u64   sum = 0;
    uint32_t cnt = 0;
    for (int i = w0 + lane; i < w1; i += 32) {
        bool kept;
        sum += weight(i, kept);
        cnt += kept;
    }
    sum = sd_warp_sum(sum);
    cnt = __reduce_add_sync(0xffffffffu, cnt);
    __syncthreads();
    if (lane == 0) { S.wsum[warp] = sum; S.wcnt[warp] = cnt; }
    __syncthreads();
    if (tid == 0) {
        sd_u64   a = 0;
        uint32_t b = 0;
        for (int w = 0; w < SD_WARPS; w++) { a += S.wsum[w]; b += S.wcnt[w]; }
        S.sum = a; S.cnt = b;
    }
    cl.sync();
    sd_u64 total = 0, ahead = 0;
    cnt = 0;
    for (int p = 0; p < R.P; p++) {
        const sd_shared * o = cl.map_shared_rank(&S, p);
        if (p < R.part) ahead += o->sum;
        total += o->sum; cnt += o->cnt;
    }
    const double u = (double) us[row];
    sd_u64 target = u > 0.0 ? (sd_u64) fmin(u * (double) total, 9.0e18) : 0;
    if (target >= total) target = total - 1;
    for (int w = 0; w < warp; w++) ahead += S.wsum[w];
    if (target >= ahead && target < ahead + sum) {               // one warp of the cluster
        for (int i0 = w0; i0 < w1; i0 += 32) {
            bool kept;
            const sd_u64 w = i0 + lane < w1 ? weight(i0 + lane, kept) : 0;
            sd_u64 s = w;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) { const sd_u64 v = __shfl_up_sync(0xffffffffu, s, o); if (lane >= o) s += v; }
            const unsigned over = __ballot_sync(0xffffffffu, ahead + s > target);
            if (over) {
                if (lane == __ffs((int) over) - 1) {
                    ids[row] = i0 + lane;
                    if (ps) ps[row] = (float) ((double) w / (double) total);
                    if (kepts) kepts[row] = (int32_t) cnt;
                }
                break;
            }
            ahead += __shfl_sync(0xffffffffu, s, 31);
        }
    }
    cl.sync();                                                   // the sums have been read
}

template <typename T>
static int sd_launch(const void * logits, int64_t ld, int rows, int V, const pib_sample_params * params, const float * u, int32_t * ids, float * p, int32_t * kept, cudaStream_t st) {
    static pib_per_device attrs;
    PIB_CHECK(attrs.once([&] { return cudaFuncSetAttribute(sample_draw_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int) sizeof(sd_shared)); }));
    int P = 1;
    while (P < 8 && (int64_t) rows * P * 2 <= 2 * pib_num_sms() && V >= P * 4 * SD_THREADS) P <<= 1;
    for (int r0 = 0; r0 < rows; r0 += 1 << 20) {
        const int n = rows - r0 < 1 << 20 ? rows - r0 : 1 << 20;
        PIB_CHECK(pib_launch_cluster(sample_draw_kernel<T>, dim3((unsigned) n, (unsigned) P), dim3(SD_THREADS), dim3(1, (unsigned) P, 1), sizeof(sd_shared), st, (const T *) logits + r0 * ld, ld, V,
                                     params + r0, u + r0, ids + r0, p ? p + r0 : nullptr, kept ? kept + r0 : nullptr));
    }
    return PIB_OK;
}

extern "C" int pib_sample(int type, const void * logits, int64_t ld, int rows, int n_vocab, const pib_sample_params * params, const float * u, int32_t * ids, float * p, int32_t * kept, pib_stream s) {
    if (rows == 0) return PIB_OK;
    if ((type != PIB_TYPE_F32 && type != PIB_TYPE_BF16) || !logits || !params || !u || !ids || rows < 0 || n_vocab < 1 || n_vocab > PIB_SAMPLE_MAX_VOCAB || (rows > 1 && ld < n_vocab)) {
        pib_set_error("pib_sample: bad arguments (type %d, %d rows of %d, %lld apart; at most %d tokens)", type, rows, n_vocab, (long long) ld, PIB_SAMPLE_MAX_VOCAB);
        return PIB_ERR_ARG;
    }
    if (type == PIB_TYPE_F32) return sd_launch<float>(logits, ld, rows, n_vocab, params, u, ids, p, kept, (cudaStream_t) s);
    return sd_launch<__nv_bfloat16>(logits, ld, rows, n_vocab, params, u, ids, p, kept, (cudaStream_t) s);
}
