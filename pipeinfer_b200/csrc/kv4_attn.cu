// kv4_attn.cu -- attention of ragged sequences over a key / value cache in 4 bits (kv4.cuh): a warp per query token and head, one pass over its keys with the running maximum and sum.
#include "kv4.cuh"

#include <algorithm>

#define KA_LOG2E 1.4426950408889634f

struct ka_args {
    const uint8_t * base; int64_t pages; int kvh, rep, dim;
    const int32_t * starts, * lens, * table; int tokens, seqs, max_pages, window; float scale;
    const void * q; void * out; int64_t ldq, ldo;
};

template <typename T, int D>
static __global__ void __launch_bounds__(128) kv4_attn_kernel(const __grid_constant__ ka_args A) {
    pib_pdl_wait();
    pib_pdl_trigger();
    __shared__ float sq[4][D];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, heads = A.kvh * A.rep;
    const int64_t row = (int64_t) blockIdx.x * 4 + warp;
    if (row >= (int64_t) A.tokens * heads) return;
    const int t = (int) (row / heads), h = (int) (row % heads), kvh = h / A.rep;
    // the last sequence that begins at or in front of t and has it
    int s = -1;
    for (int i = lane; i < A.seqs; i += 32) if (A.starts[i] <= t && t < A.starts[i + 1]) s = i;
    s = __reduce_max_sync(0xffffffffu, s);
    if (s < 0) return;
    const int pos = A.lens[s] - (A.starts[s + 1] - t), first = A.window > 0 ? max(0, pos - A.window + 1) : 0;
    const int last = min(pos, (int) min((int64_t) A.max_pages * KV4_P, (int64_t) 0x7fffffff) - 1);
    const T * q = (const T *) A.q + (int64_t) t * A.ldq + (int64_t) h * D;
    for (int c = lane; c < D; c += 32) sq[warp][c] = (float) q[c] * (A.scale * KA_LOG2E);
    __syncwarp();
    float m = -INFINITY, l = 0.f, o[D / 32] = {};
    for (int j0 = first; j0 <= last; j0 += 32) {
        const int j = j0 + lane;
        const uint8_t * rec = nullptr;
        float sc = -INFINITY;
        if (j <= last) {
            const int page = A.table[(int64_t) s * A.max_pages + j / KV4_P];
            if (page >= 0 && page < A.pages) {
                rec = A.base + ((int64_t) page * A.kvh + kvh) * kv4_record(D);
                sc = 0.f;
                for (int w = 0; w < D / 8; w++) {
                    const __half2 dm = *reinterpret_cast<const __half2 *>(rec + kv4_steps(D) + ((j % KV4_P) * (D / 32) + w / 4) * 4);
                    uint32_t p[4];
                    kv4_pairs(*reinterpret_cast<const uint32_t *>(rec + (j % KV4_P) * (D / 2) + w * 4), __low2half2(dm), __high2half2(dm), p);
                    for (int i = 0; i < 4; i++) { const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&p[i])); sc = fmaf(sq[warp][w * 8 + i], f.x, fmaf(sq[warp][w * 8 + i + 4], f.y, sc)); }
                }
            }
        }
        const float mn = fmaxf(m, warp_max(sc)), a = m == mn ? 1.f : exp2f(m - mn), p = rec ? exp2f(sc - mn) : 0.f;
        l = l * a + warp_sum(p);
        m = mn;
#pragma unroll
        for (int i = 0; i < D / 32; i++) o[i] *= a;
        for (int k = 0; k < 32; k++) {
            const uint8_t * r = (const uint8_t *) __shfl_sync(0xffffffffu, (unsigned long long) rec, k);
            const float pk = __shfl_sync(0xffffffffu, p, k);
            if (!r) continue;
            const int place = (j0 + k) % KV4_P;
            r += kv4_half(D);
#pragma unroll
            for (int i = 0; i < D / 32; i++) {
                const int c = i * 32 + lane;
                const __half2 dm = *reinterpret_cast<const __half2 *>(r + kv4_steps(D) + (place * (D / 32) + i) * 4);
                const uint8_t b = r[place * (D / 2) + ((c / 2) ^ kv4_flip(D, place))];
                o[i] = fmaf(pk, __half2float(__hfma(__int2half_rn(c & 1 ? b >> 4 : b & 15), __low2half(dm), __high2half(dm))), o[i]);
            }
        }
    }
    T * out = (T *) A.out + (int64_t) t * A.ldo + (int64_t) h * D;
#pragma unroll
    for (int i = 0; i < D / 32; i++) out[i * 32 + lane] = (T) (l > 0.f || l != l ? o[i] / l : 0.f);
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

extern "C" size_t pib_kv4_attn_scratch_bytes(const pib_kv4 * kv, const pib_kv4_batch * b) {
    return ka_batch_ok("pib_kv4_attn_scratch_bytes", kv, b) == PIB_OK ? 256 : 0;
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
    const dim3 grid((unsigned) (((int64_t) b->tokens * b->heads + 3) / 4));
    const cudaStream_t st = (cudaStream_t) s;
    if (size == 4) PIB_CHECK(pib_launch(kv->dim == 64 ? kv4_attn_kernel<float, 64> : kv4_attn_kernel<float, 128>, grid, dim3(128), 0, st, A));
    else           PIB_CHECK(pib_launch(kv->dim == 64 ? kv4_attn_kernel<__nv_bfloat16, 64> : kv4_attn_kernel<__nv_bfloat16, 128>, grid, dim3(128), 0, st, A));
    return PIB_OK;
}
