// kv4_cache.cu -- keys and values into the cells of a cache in 4 bits, and back.
//
//   m = fp16(min x), d = fp16((max x - m) / 15), n = rint((x - m) / d) in 0 .. 15; a channel stands for fp16(m + d n)
//
// A block per token: first its threads look whether a later token of the call has the same cell (the later one stays), then each takes eight neighbouring channels of a head's keys or values, four
// threads a group of 32.  What bounds it: the launch for the tokens of a decode step (2 us each way in a captured run of calls); for prompts instructions (79 % of issue slots, 11 % of memory): a block's
// start and end, a barrier, the rounding, and the look at all later cells, which grows with the square of the call's tokens.  8 heads of 128 in bfloat16: 4,000 tokens 14.9 us (memory 3.3), 8,000 31, 16,384
// 76; their values back 5.5, 9.8 and 24.5.
#include "kv4.cuh"

#include <algorithm>

#define KC_THREADS 256

template <typename T> __device__ __forceinline__ float kc_float(T v);
template <> __device__ __forceinline__ float kc_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float kc_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

// eight neighbouring values; wide: rows that 16-byte loads may take
template <typename T> __device__ __forceinline__ void kc_load8(const T * p, bool wide, float (&v)[8]) {
    if (wide) {
        if constexpr (sizeof(T) == 4) {
            const float4 a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        } else {
            const uint4 a = *reinterpret_cast<const uint4 *>(p);
            const uint32_t w[4] = { a.x, a.y, a.z, a.w };
#pragma unroll
            for (int j = 0; j < 4; j++) { v[2 * j] = __uint_as_float(w[j] << 16); v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u); }
        }
    } else
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = kc_float<T>(p[j]);
}

template <typename T, int dim>
static __global__ void __launch_bounds__(KC_THREADS) kv4_write_kernel(uint8_t * __restrict__ base, int64_t pages, int heads, const T * __restrict__ k, int64_t ldk, const T * __restrict__ v,
                                                                      int64_t ldv, const int32_t * __restrict__ cells, int n, bool wide) {
    pib_pdl_wait();
    pib_pdl_trigger();
    constexpr int per = dim / 8;
    const int t = blockIdx.x, all = 2 * heads * per;
    // (whole warps enter each round: heads * dim / 4 is a multiple of 16, lanes without work repeat the last octet's reading and store nothing)
    auto load = [&](int u0, float (&x)[8]) {
        const int u = min(u0 + (int) threadIdx.x, all - 1), values = u >= heads * per, w = u - values * heads * per;
        kc_load8<T>((values ? v + t * ldv : k + t * ldk) + (int64_t) (w / per) * dim + w % per * 8, wide, x);
    };
    // the first round's rows are on their way while the cells are looked through
    float x[8];
    load(0, x);
    const int cell = cells[t];
    if (cell < 0 || cell / KV4_P >= pages) return;
    bool later = false;
    if (((uintptr_t) cells & 15) == 0) {                             // four cells a load, the last ones one by one
        const int whole = n & ~3;
        for (int i = ((t + 1) & ~3) + 4 * threadIdx.x; i < whole; i += 4 * KC_THREADS) {
            const int4 c = *reinterpret_cast<const int4 *>(cells + i);
            later |= (c.x == cell && i > t) || (c.y == cell && i + 1 > t) || (c.z == cell && i + 2 > t) || (c.w == cell && i + 3 > t);
        }
        if ((int) threadIdx.x < n - whole) later |= cells[whole + threadIdx.x] == cell && whole + (int) threadIdx.x > t;
    } else
        for (int i = t + 1 + threadIdx.x; i < n; i += KC_THREADS) later |= cells[i] == cell;
    if (__syncthreads_or(later)) return;
    const int place = cell % KV4_P;
    for (int u0 = 0; u0 < all; u0 += KC_THREADS) {
        if (u0) load(u0, x);
        const int u = min(u0 + (int) threadIdx.x, all - 1), values = u >= heads * per, w = u - values * heads * per, head = w / per, o = w % per;
        float    lo = INFINITY, hi = -INFINITY;
        uint32_t big = 0;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            big  = max(big, __float_as_uint(x[j]) & 0x7fffffffu);
            x[j] = fminf(fmaxf(x[j], -60000.f), 60000.f);
            lo = fminf(lo, x[j]); hi = fmaxf(hi, x[j]);
        }
#pragma unroll
        for (int s = 1; s < 4; s <<= 1) {
            lo  = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, s));
            hi  = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, s));
            big = max(big, __shfl_xor_sync(0xffffffffu, big, s));
        }
        __half   m = __float2half_rn(lo);
        const float mf = __half2float(m);
        __half   d = __float2half_rn(__fdiv_rn(fmaxf(__fsub_rn(hi, mf), 0.f), 15.f));
        const float df = __half2float(d);
        uint32_t q = 0;
        // The quotient by a product with 1 / d is off by less than 2^-18; only where that lies next to a half does the division itself say which side it is on.  (Eight divisions a thread were the kernel's time)
        const float inv = __frcp_rn(df);
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float a = __fsub_rn(x[j], mf), p = a * inv;
            float       r = rintf(p);
            if (fabsf(p - r) > 0.49998f) r = rintf(__fdiv_rn(a, df));
            r = df > 0.f ? fminf(fmaxf(r, 0.f), 15.f) : 0.f;
            q |= (uint32_t) (int) r << (4 * j);
        }
        if (big >= 0x7f800000u) { d = __ushort_as_half(0); m = __ushort_as_half(0x7e00); q = 0; }
        if (u0 + (int) threadIdx.x >= all) continue;
        uint8_t * part = base + ((int64_t) (cell / KV4_P) * heads + head) * kv4_record(dim) + values * kv4_half(dim);
        const int row  = values ? kv4_row(place) : place;
        *reinterpret_cast<uint32_t *>(part + row * (dim / 2) + ((o * 4) ^ (values ? kv4_flip(dim, row) : 0))) = q;
        if ((o & 3) == 0) *reinterpret_cast<__half2 *>(part + kv4_steps(dim) + (row * (dim / 32) + (o >> 2)) * 4) = __halves2half2(d, m);
    }
}

template <typename T, int dim>
static __global__ void __launch_bounds__(KC_THREADS) kv4_read_kernel(const uint8_t * __restrict__ base, int64_t pages, int heads, T * __restrict__ k, int64_t ldk, T * __restrict__ v, int64_t ldv,
                                                                     const int32_t * __restrict__ cells, bool wide) {
    pib_pdl_wait();
    pib_pdl_trigger();
    constexpr int per = dim / 8;
    const int  t = blockIdx.x, cell = cells[t], place = cell & (KV4_P - 1);
    const bool there = cell >= 0 && cell / KV4_P < pages;
    for (int u = threadIdx.x; u < 2 * heads * per; u += KC_THREADS) {
        const int values = u >= heads * per, w = u - values * heads * per, head = w / per, o = w % per;
        T * out = (values ? v : k);
        if (!out) continue;
        out += (int64_t) t * (values ? ldv : ldk) + (int64_t) head * dim + o * 8;
        uint32_t p[4] = { 0, 0, 0, 0 };
        if (there) {
            const uint8_t * part = base + ((int64_t) (cell / KV4_P) * heads + head) * kv4_record(dim) + values * kv4_half(dim);
            const int       row = values ? kv4_row(place) : place;
            const __half2   dm = *reinterpret_cast<const __half2 *>(part + kv4_steps(dim) + (row * (dim / 32) + (o >> 2)) * 4);
            kv4_pairs(*reinterpret_cast<const uint32_t *>(part + row * (dim / 2) + ((o * 4) ^ (values ? kv4_flip(dim, row) : 0))), __low2half2(dm), __high2half2(dm), p);
        }
        float x[8];
#pragma unroll
        for (int j = 0; j < 4; j++) { const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&p[j])); x[j] = f.x; x[j + 4] = f.y; }
        if constexpr (sizeof(T) == 4) {
            if (wide) { reinterpret_cast<float4 *>(out)[0] = make_float4(x[0], x[1], x[2], x[3]); reinterpret_cast<float4 *>(out)[1] = make_float4(x[4], x[5], x[6], x[7]); }
            else
#pragma unroll
                for (int j = 0; j < 8; j++) out[j] = x[j];
        } else {
            __nv_bfloat162 h[4];
#pragma unroll
            for (int j = 0; j < 4; j++) h[j] = __floats2bfloat162_rn(x[2 * j], x[2 * j + 1]);
            if (wide) *reinterpret_cast<uint4 *>(out) = *reinterpret_cast<const uint4 *>(h);
            else
#pragma unroll
                for (int j = 0; j < 4; j++) { out[2 * j] = h[j].x; out[2 * j + 1] = h[j].y; }
        }
    }
}

// ---- host side --------------------------------------------------------------------------------------------------------------------
extern "C" pib_kv4 * pib_kv4_new(int64_t pages, int kv_heads, int head_dim) {
    // cells are counted in 32 bits
    if (pages < 1 || pages > 0x7fffffff / KV4_P || kv_heads < 1 || kv_heads > PIB_KV4_MAX_HEADS || (head_dim != 64 && head_dim != 128)) {
        pib_set_error("pib_kv4_new: %lld pages of %d heads of %d (up to %d heads, of 64 or 128)", (long long) pages, kv_heads, head_dim, PIB_KV4_MAX_HEADS);
        return nullptr;
    }
    pib_kv4 * kv = (pib_kv4 *) calloc(1, sizeof(pib_kv4));
    if (!kv) { pib_set_error("pib_kv4_new: no host memory"); return nullptr; }
    kv->heads = kv_heads; kv->dim = head_dim; kv->pages = pages;
    const size_t bytes = (size_t) pages * kv_heads * kv4_record(head_dim);
    cudaError_t  e = cudaGetDevice(&kv->device);
    if (e == cudaSuccess) e = cudaMalloc(&kv->base, bytes);
    if (e == cudaSuccess) e = cudaMemset(kv->base, 0, bytes);
    if (e == cudaSuccess) e = cudaStreamSynchronize(0);
    if (e == cudaSuccess) return kv;
    pib_set_error("pib_kv4_new: %zu bytes: %s", bytes, cudaGetErrorString(e));
    cudaGetLastError();
    cudaFree(kv->base);
    free(kv);
    return nullptr;
}
extern "C" void pib_kv4_free(pib_kv4 * kv) {
    if (!kv) return;
    cudaFree(kv->base);
    free(kv);
}
extern "C" size_t pib_kv4_bytes(const pib_kv4 * kv) { return kv ? (size_t) kv->pages * kv->heads * kv4_record(kv->dim) : 0; }

// rows that loads and stores of 16 bytes may take
static bool kc_wide(int size, const void * p, int64_t ld) { return !p || (((uintptr_t) p & 15) == 0 && ld * size % 16 == 0); }

extern "C" int pib_kv4_write(pib_kv4 * kv, int type, const void * k, int64_t ldk, const void * v, int64_t ldv, const int32_t * cells, int n, pib_stream s) {
    const int size = kv4_type_size(type), rc = kv4_ok("pib_kv4_write", kv);
    if (rc != PIB_OK) return rc;
    const int64_t row = (int64_t) kv->heads * kv->dim;
    if (!size || n < 0 || n > PIB_KV4_MAX_WRITE || (n > 0 && (!k || !v || !cells || ldk < row || ldv < row || (((uintptr_t) k | (uintptr_t) v) & (size - 1)) || ((uintptr_t) cells & 3)))) {
        pib_set_error("pib_kv4_write: bad arguments (type %d, n %d, rows %lld and %lld apart)", type, n, (long long) ldk, (long long) ldv);
        return PIB_ERR_ARG;
    }
    if (!n) return PIB_OK;
    const bool wide = kc_wide(size, k, ldk) && kc_wide(size, v, ldv);
    auto go = [&](auto kernel, auto * kp, auto * vp) { return pib_launch(kernel, dim3((unsigned) n), dim3(KC_THREADS), 0, (cudaStream_t) s, kv->base, kv->pages, kv->heads, kp, ldk, vp, ldv, cells, n, wide); };
    const float * kf = (const float *) k, * vf = (const float *) v;
    const __nv_bfloat16 * kb = (const __nv_bfloat16 *) k, * vb = (const __nv_bfloat16 *) v;
    if (kv->dim == 64) PIB_CHECK(size == 4 ? go(kv4_write_kernel<float, 64>, kf, vf) : go(kv4_write_kernel<__nv_bfloat16, 64>, kb, vb));
    else               PIB_CHECK(size == 4 ? go(kv4_write_kernel<float, 128>, kf, vf) : go(kv4_write_kernel<__nv_bfloat16, 128>, kb, vb));
    return PIB_OK;
}

extern "C" int pib_kv4_read(const pib_kv4 * kv, int type, const int32_t * cells, int n, void * k, int64_t ldk, void * v, int64_t ldv, pib_stream s) {
    const int size = kv4_type_size(type), rc = kv4_ok("pib_kv4_read", kv);
    if (rc != PIB_OK) return rc;
    const int64_t row = (int64_t) kv->heads * kv->dim;
    if (!size || n < 0 || (n > 0 && (!cells || (k && ldk < row) || (v && ldv < row) || (((uintptr_t) k | (uintptr_t) v) & (size - 1)) || ((uintptr_t) cells & 3)))) {
        pib_set_error("pib_kv4_read: bad arguments (type %d, n %d, rows %lld and %lld apart)", type, n, (long long) ldk, (long long) ldv);
        return PIB_ERR_ARG;
    }
    if (!n || (!k && !v)) return PIB_OK;
    const bool wide = kc_wide(size, k, ldk) && kc_wide(size, v, ldv);
    auto go = [&](auto kernel, auto * kp, auto * vp) { return pib_launch(kernel, dim3((unsigned) n), dim3(KC_THREADS), 0, (cudaStream_t) s, (const uint8_t *) kv->base, kv->pages, kv->heads, kp, ldk, vp, ldv, cells, wide); };
    float * kf = (float *) k, * vf = (float *) v;
    __nv_bfloat16 * kb = (__nv_bfloat16 *) k, * vb = (__nv_bfloat16 *) v;
    if (kv->dim == 64) PIB_CHECK(size == 4 ? go(kv4_read_kernel<float, 64>, kf, vf) : go(kv4_read_kernel<__nv_bfloat16, 64>, kb, vb));
    else               PIB_CHECK(size == 4 ? go(kv4_read_kernel<float, 128>, kf, vf) : go(kv4_read_kernel<__nv_bfloat16, 128>, kb, vb));
    return PIB_OK;
}
