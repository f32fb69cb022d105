// i8_gemm.cu -- 8-bit integer weights with a scale for each output times any number of tokens: a warp per output and eight tokens, four products an instruction.
#include "i8_block.cuh"

#include <algorithm>

static __global__ void __launch_bounds__(256) i8_gemm_kernel(const uint8_t * __restrict__ qs, const float * __restrict__ ws, int64_t N, int KB, const uint8_t * __restrict__ a, const float * __restrict__ ad,
                                                             int b, float * __restrict__ y) {
    pib_pdl_wait();
    pib_pdl_trigger();
    const int     lane = threadIdx.x & 31;
    const int64_t n = (int64_t) blockIdx.x * 8 + (threadIdx.x >> 5);
    const int     t0 = blockIdx.y * 8;
    if (n >= N) return;
    int acc[8] = {};
    for (int u = lane; u < KB * 8; u += 32) {
        const int4 w = *reinterpret_cast<const int4 *>(qs + pib_f8_at(n, (int64_t) u * 16, KB));
#pragma unroll
        for (int t = 0; t < 8; t++)
            if (t0 + t < b) {
                const int4 v = *reinterpret_cast<const int4 *>(a + ((int64_t) (u >> 3) * b + t0 + t) * 128 + (u & 7) * 16);
                acc[t] = __dp4a(w.x, v.x, __dp4a(w.y, v.y, __dp4a(w.z, v.z, __dp4a(w.w, v.w, acc[t]))));
            }
    }
#pragma unroll
    for (int t = 0; t < 8; t++) {
        const int s = __reduce_add_sync(0xffffffffu, acc[t]);
        if (lane == t && t0 + t < b) y[(int64_t) (t0 + t) * N + n] = i8_out(s, ad[t0 + t], ws[n]);
    }
}

int pib_i8_gemm(const pib_weight * w, const void * act, int b, float * y, cudaStream_t st) {
    const int rc = pib_f8_rows_ok("pib_gemm", w, act, y, b, PIB_I8_MAX_ROWS);
    if (rc != PIB_OK) return rc;
    if ((uintptr_t) act & 15) { pib_set_error("pib_gemm: act_dev needs 16-byte alignment"); return PIB_ERR_ARG; }
    const pib_i8_act L = pib_i8_act_of(w->K, b);
    PIB_CHECK(pib_launch(i8_gemm_kernel, dim3((unsigned) ((w->N + 7) / 8), (unsigned) ((b + 7) / 8)), dim3(256), 0, st, w->qs, (const float *) w->d, w->N, L.KB, (const uint8_t *) act,
                         (const float *) ((const uint8_t *) act + L.d_off), b, y));
    return PIB_OK;
}
