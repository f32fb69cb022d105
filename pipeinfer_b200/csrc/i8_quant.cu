// i8_quant.cu -- 8-bit integers with a scale for each output and each token: weights into their layout and back, embedding rows, the activation quantiser.
#include "i8_block.cuh"

#include <string.h>

#include <algorithm>

// ---- weights ------------------------------------------------------------------------------------------------------------------------
static pib_weight * i8_alloc(int64_t N, int64_t K) {
    if (K > PIB_I8_MAX_K) { pib_set_error("pib_weight: 8-bit integer rows of %lld columns, limit %d", (long long) K, PIB_I8_MAX_K); return nullptr; }
    pib_weight * w = pib_tiles_alloc(PIB_TYPE_I8, N, K, N > 0 ? (size_t) N * 4 : 0);
    if (w) w->bytes = (size_t) N * K + (size_t) N * 4;
    return w;
}

extern "C" pib_weight * pib_weight_from_device_i8(const void * q_dev, const float * scales_dev, int64_t N, int64_t K) {
    if (!q_dev || !scales_dev || ((uintptr_t) scales_dev & 3)) { pib_set_error("pib_weight_from_device_i8: bad arguments"); return nullptr; }
    pib_weight * w = i8_alloc(N, K);
    if (!w) return nullptr;
    if (pib_tiles_fill(w, (const uint8_t *) q_dev, 0, pib_f8_blocks(N) * PIB_F8_BLOCK) != cudaSuccess || cudaMemcpyAsync(w->d, scales_dev, (size_t) N * 4, cudaMemcpyDeviceToDevice, 0) != cudaSuccess ||
        cudaStreamSynchronize(0) != cudaSuccess) {
        pib_set_error("pib_weight_from_device_i8: %s", cudaGetErrorString(cudaGetLastError()));
        pib_weight_free(w);
        return nullptr;
    }
    return w;
}

extern "C" pib_weight * pib_weight_upload_i8(const void * q_host, const float * scales_host, int64_t N, int64_t K) {
    if (!q_host || !scales_host) { pib_set_error("pib_weight_upload_i8: bad arguments"); return nullptr; }
    pib_weight * w = i8_alloc(N, K);
    if (!w) return nullptr;
    bool ok = pib_tiles_upload(w, (const uint8_t *) q_host) == cudaSuccess;
    ok = ok && cudaMemcpy(w->d, scales_host, (size_t) N * 4, cudaMemcpyHostToDevice) == cudaSuccess;
    if (ok) return w;
    pib_set_error("pib_weight_upload_i8: %s", cudaGetErrorString(cudaGetLastError()));
    pib_weight_free(w);
    return nullptr;
}

int pib_i8_row(const pib_weight * w, int64_t row, void * out) {
    const int rc = pib_tiles_row(w, row, out);
    if (rc != PIB_OK) return rc;
    PIB_CHECK(cudaMemcpy((uint8_t *) out + w->K, (const float *) w->d + row, 4, cudaMemcpyDeviceToHost));
    return PIB_OK;
}

static __global__ void i8_rows_kernel(const int8_t * __restrict__ qs, const float * __restrict__ d, int64_t N, int64_t K, int64_t KB, const int32_t * __restrict__ ids, float * __restrict__ out) {
    pib_pdl_wait();
    pib_pdl_trigger();
    const int64_t row = ids[blockIdx.x];
    for (int64_t k = (int64_t) blockIdx.y * blockDim.x + threadIdx.x; k < K; k += (int64_t) gridDim.y * blockDim.x)
        out[(int64_t) blockIdx.x * K + k] = row < 0 || row >= N ? 0.f : __fmul_rn((float) qs[pib_f8_at(row, k, KB)], d[row]);
}

int pib_i8_get_rows(const pib_weight * w, const int32_t * ids, int n, float * out, cudaStream_t st) {
    PIB_CHECK(pib_launch(i8_rows_kernel, dim3((unsigned) n, (unsigned) std::min<int64_t>((w->K + 255) / 256, 64)), dim3(256), 0, st, (const int8_t *) w->qs, (const float *) w->d, w->N, w->K,
                         pib_f8_blocks(w->K), ids, out));
    return PIB_OK;
}

// ---- activations --------------------------------------------------------------------------------------------------------------------
// A block per token, as a token's scale needs the whole row: eight values a thread and round, the first IQ_KEEP rounds stay in registers between the largest value's pass and the rounding's.
// NORM: the row's mean square first.  What bounds it: the launch up to a few hundred tokens; beyond that reading the floats (1,999 tokens of 8192: 66 MB).
#define IQ_THREADS 256
#define IQ_KEEP    4
template <bool NORM, bool VEC>
__global__ void __launch_bounds__(IQ_THREADS) i8_quant_kernel(const float * __restrict__ x, const float * __restrict__ nw, float eps, int b, int64_t K, int KB, uint8_t * __restrict__ qs,
                                                              float * __restrict__ d, float * __restrict__ xnorm) {
    pib_pdl_wait();
    pib_pdl_trigger();
    __shared__ float    part[IQ_THREADS / 32];
    __shared__ uint32_t top[IQ_THREADS / 32];
    const int      lane = threadIdx.x & 31, warp = threadIdx.x >> 5, units = KB * (PIB_F8_BLOCK / 8);
    const int64_t  row = blockIdx.x;
    const float *  p = x + row * K;
    float          rs = 1.f;
    if (NORM) {
        float s = 0.f;
        for (int64_t k = threadIdx.x; k < K; k += IQ_THREADS) s = fmaf(p[k], p[k], s);
        s = warp_sum(s);
        if (lane == 0) part[warp] = s;
        __syncthreads();
        s = 0.f;
        for (int i = 0; i < IQ_THREADS / 32; i++) s += part[i];
        rs = 1.0f / sqrtf(s / (float) K + eps);
    }
    auto load = [&](int u, float (&v)[8]) {
        const int64_t k = (int64_t) u * 8;
        if (VEC && k + 8 <= K) {
            const float4 f = reinterpret_cast<const float4 *>(p + k)[0], h = reinterpret_cast<const float4 *>(p + k)[1];
            v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w; v[4] = h.x; v[5] = h.y; v[6] = h.z; v[7] = h.w;
        } else
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = k + j < K ? p[k + j] : 0.f;
        if (NORM)
#pragma unroll
            for (int j = 0; j < 8; j++) if (k + j < K) v[j] = v[j] * rs * nw[k + j];
    };
    float    keep[IQ_KEEP][8];
    uint32_t m = 0;
    auto largest = [&](const float (&v)[8]) {
#pragma unroll
        for (int j = 0; j < 8; j++) m = max(m, i8_bits(v[j]));
    };
#pragma unroll
    for (int r = 0; r < IQ_KEEP; r++) {
        const int u = r * IQ_THREADS + threadIdx.x;
        if (u < units) { load(u, keep[r]); largest(keep[r]); }
    }
    for (int u = IQ_KEEP * IQ_THREADS + threadIdx.x; u < units; u += IQ_THREADS) { float v[8]; load(u, v); largest(v); }
    m = __reduce_max_sync(0xffffffffu, m);
    if (lane == 0) top[warp] = m;
    __syncthreads();
    m = 0;
    for (int i = 0; i < IQ_THREADS / 32; i++) m = max(m, top[i]);
    const float s = i8_scale(m);
    if (threadIdx.x == 0) d[row] = s;
    auto store = [&](int u, const float (&v)[8]) {
        if (NORM && xnorm)
#pragma unroll
            for (int j = 0; j < 8; j++) if ((int64_t) u * 8 + j < K) xnorm[row * K + (int64_t) u * 8 + j] = v[j];
        reinterpret_cast<uint2 *>(qs)[((int64_t) (u >> 4) * b + row) * 16 + (u & 15)] = make_uint2(i8_pack4(v[0], v[1], v[2], v[3], s), i8_pack4(v[4], v[5], v[6], v[7], s));
    };
#pragma unroll
    for (int r = 0; r < IQ_KEEP; r++) {
        const int u = r * IQ_THREADS + threadIdx.x;
        if (u < units) store(u, keep[r]);
    }
    for (int u = IQ_KEEP * IQ_THREADS + threadIdx.x; u < units; u += IQ_THREADS) { float v[8]; load(u, v); store(u, v); }
}

int pib_i8_quantize(const float * x, const float * norm_w, float eps, int b, int64_t K, void * act, float * xnorm, cudaStream_t st) {
    if (!x || !act || b < 1 || b > PIB_I8_MAX_ROWS || K < 1 || K > PIB_I8_MAX_K) {
        pib_set_error("act quantise: bad arguments (8-bit integers, b %d, K %lld)", b, (long long) K);
        return PIB_ERR_ARG;
    }
    if (((uintptr_t) act & 15) || (((uintptr_t) x | (uintptr_t) norm_w | (uintptr_t) xnorm) & 3)) {
        pib_set_error("act quantise: act_dev needs 16-byte alignment, fp32 rows 4-byte alignment");
        return PIB_ERR_ARG;
    }
    const pib_i8_act A = pib_i8_act_of(K, b);
    uint8_t * q = (uint8_t *) act;
    float *   d = (float *) (q + A.d_off);
    const bool vec = K % 4 == 0 && !((uintptr_t) x & 15);
    const dim3 grid((unsigned) b), block(IQ_THREADS);
    if (norm_w && vec) PIB_CHECK(pib_launch(i8_quant_kernel<true, true>, grid, block, 0, st, x, norm_w, eps, b, K, A.KB, q, d, xnorm));
    else if (norm_w)   PIB_CHECK(pib_launch(i8_quant_kernel<true, false>, grid, block, 0, st, x, norm_w, eps, b, K, A.KB, q, d, xnorm));
    else if (vec)      PIB_CHECK(pib_launch(i8_quant_kernel<false, true>, grid, block, 0, st, x, norm_w, eps, b, K, A.KB, q, d, xnorm));
    else               PIB_CHECK(pib_launch(i8_quant_kernel<false, false>, grid, block, 0, st, x, norm_w, eps, b, K, A.KB, q, d, xnorm));
    return PIB_OK;
}

int pib_i8_act_blocks(const void * act_dev, int b, int64_t K, void * out) {
    if (!act_dev || !out || b < 1 || b > PIB_I8_MAX_ROWS || K < 1 || K > PIB_I8_MAX_K) { pib_set_error("pib_act_to_blocks: bad arguments"); return PIB_ERR_ARG; }
    const pib_i8_act A = pib_i8_act_of(K, b);
    uint8_t * h = (uint8_t *) malloc(A.total);
    if (!h) { pib_set_error("pib_act_to_blocks: no host memory"); return PIB_ERR_NOMEM; }
    const cudaError_t e = cudaMemcpy(h, act_dev, A.total, cudaMemcpyDeviceToHost);
    if (e != cudaSuccess) { free(h); PIB_CHECK(e); }
    uint8_t * o = (uint8_t *) out;
    for (int64_t t = 0; t < b; t++, o += 4 + A.Kp) {
        memcpy(o, h + A.d_off + (size_t) t * 4, 4);
        for (int64_t kb = 0; kb < A.KB; kb++) memcpy(o + 4 + kb * PIB_F8_BLOCK, h + (size_t) (kb * b + t) * PIB_F8_BLOCK, PIB_F8_BLOCK);
    }
    free(h);
    return PIB_OK;
}

int pib_i8_gemm_host(const pib_weight * w, const float * x_host, int b, float * y_host) {
    const int ok = pib_f8_rows_ok("pib_gemm_host", w, x_host, y_host, b, PIB_I8_MAX_ROWS);
    if (ok != PIB_OK) return ok;
    const size_t xb = ((size_t) b * w->K * 4 + 255) & ~(size_t) 255, yb = ((size_t) b * w->N * 4 + 255) & ~(size_t) 255;
    uint8_t *    buf = nullptr;
    PIB_CHECK(cudaMalloc(&buf, xb + yb + pib_i8_act_of(w->K, b).total));
    int rc = PIB_OK;
    if (cudaMemcpy(buf, x_host, (size_t) b * w->K * 4, cudaMemcpyHostToDevice) != cudaSuccess) { rc = PIB_ERR_CUDA; pib_set_error("pib_gemm_host: %s", cudaGetErrorString(cudaGetLastError())); }
    if (rc == PIB_OK) rc = pib_i8_quantize((const float *) buf, nullptr, 0.f, b, w->K, buf + xb + yb, nullptr, nullptr);
    if (rc == PIB_OK) rc = pib_i8_gemm(w, buf + xb + yb, b, (float *) (buf + xb), nullptr);
    if (rc == PIB_OK) rc = pib_gemm_check(nullptr);
    if (rc == PIB_OK && cudaMemcpy(y_host, buf + xb, (size_t) b * w->N * 4, cudaMemcpyDeviceToHost) != cudaSuccess) { rc = PIB_ERR_CUDA; pib_set_error("pib_gemm_host: %s", cudaGetErrorString(cudaGetLastError())); }
    cudaFree(buf);
    return rc;
}
