// f8_quant.cu -- 8-bit floating point with block scales: weights into their layout and back, embedding rows, the activation quantiser.
#include "f8_block.cuh"

#include <string.h>

#include <algorithm>

// ---- weights ------------------------------------------------------------------------------------------------------------------------
// rows r0 .. r0 + rows of the padded plane, 16 bytes a thread; src holds those rows of the matrix, K bytes each (any alignment)
static __global__ void f8_pad_kernel(const uint8_t * __restrict__ src, uint8_t * __restrict__ dst, int64_t N, int64_t K, int64_t Kp, int64_t r0, int64_t rows) {
    for (int64_t i = (int64_t) blockIdx.x * blockDim.x + threadIdx.x; i < rows * (Kp / 16); i += (int64_t) gridDim.x * blockDim.x) {
        const int64_t r = i / (Kp / 16), k = i % (Kp / 16) * 16;
        __align__(16) uint8_t v[16];
#pragma unroll
        for (int j = 0; j < 16; j++) v[j] = r0 + r < N && k + j < K ? src[r * K + k + j] : 0;
        *reinterpret_cast<int4 *>(dst + pib_f8_at(r0 + r, k, Kp >> 7)) = *reinterpret_cast<const int4 *>(v);
    }
}

pib_weight * pib_tiles_alloc(int type, int64_t N, int64_t K, size_t scale_bytes) {
    // the rows of 128 bytes are counted in 32 bits
    if (N <= 0 || K <= 0 || N > 0x7fffff00 || K > 0x7fffff00 || pib_f8_blocks(N) * pib_f8_blocks(K) > 0x7fffffff / PIB_F8_BLOCK) {
        pib_set_error("pib_weight: bad shape %lld x %lld", (long long) N, (long long) K);
        return nullptr;
    }
    const int64_t NB = pib_f8_blocks(N), KB = pib_f8_blocks(K);
    pib_weight *  w  = (pib_weight *) calloc(1, sizeof(pib_weight));
    if (!w) { pib_set_error("pib_weight: no host memory"); return nullptr; }
    w->type = type;
    w->N = N; w->K = K;
    const size_t plane = (size_t) NB * KB * PIB_F8_BLOCK * PIB_F8_BLOCK;
    if (cudaMalloc(&w->base, plane + scale_bytes + 256) != cudaSuccess) {
        pib_set_error("pib_weight: cudaMalloc of %zu bytes failed", plane);
        cudaGetLastError();
        free(w);
        return nullptr;
    }
    w->qs   = (uint8_t *) w->base;
    w->d    = (uint16_t *) (w->qs + plane);
    w->owns = 1;
    pib_f8_maps * m = (pib_f8_maps *) aligned_alloc(64, (sizeof(pib_f8_maps) + 63) / 64 * 64);
    w->map = m;
    if (!m) pib_set_error("pib_weight: no host memory");
    int rc = m ? pib_f8_map(&m->block, w->qs, NB * KB * PIB_F8_BLOCK, PIB_F8_BLOCK) : PIB_ERR_NOMEM;
    if (rc == PIB_OK) rc = pib_f8_map4(&m->stage, w->qs, KB, NB, 16, 16);
    for (int i = 0; i < 4 && rc == PIB_OK; i++) rc = pib_f8_map4(&m->runs.m[i], w->qs, KB, NB, (i + 1) * 32, 1);
    if (rc == PIB_OK) rc = pib_f8_map(&m->runs.m[4], w->qs, NB * KB * PIB_F8_BLOCK, 2 * PIB_F8_BLOCK);
    if (rc != PIB_OK) { pib_weight_free(w); return nullptr; }
    return w;
}

cudaError_t pib_tiles_fill(pib_weight * w, const uint8_t * src, int64_t r0, int64_t rows) {
    const int64_t Kp = pib_f8_blocks(w->K) * PIB_F8_BLOCK, n = rows * (Kp / 16);
    f8_pad_kernel<<<(unsigned) std::min<int64_t>((n + 255) / 256, 1 << 16), 256>>>(src, w->qs, w->N, w->K, Kp, r0, rows);
    return cudaGetLastError();
}

cudaError_t pib_tiles_upload(pib_weight * w, const uint8_t * q_host) {
    // in pieces of whole rows, as the other formats: no second full-size buffer
    const int64_t N = w->N, K = w->K, Np = pib_f8_blocks(N) * PIB_F8_BLOCK, per = std::max<int64_t>(1, std::min<int64_t>(N, (int64_t) (256u << 20) / K));
    uint8_t *     stage = nullptr;
    cudaError_t   e = cudaMalloc(&stage, (size_t) per * K);
    for (int64_t r = 0; e == cudaSuccess && r < N; r += per) {
        const int64_t rows = std::min(per, N - r);
        if ((e = cudaMemcpy(stage, q_host + r * K, (size_t) (rows * K), cudaMemcpyHostToDevice)) != cudaSuccess) break;
        if ((e = pib_tiles_fill(w, stage, r, r + rows == N ? Np - r : rows)) != cudaSuccess) break;
        e = cudaStreamSynchronize(0);
    }
    cudaFree(stage);
    return e;
}

int pib_tiles_row(const pib_weight * w, int64_t row, void * out) {
    const int64_t KB = pib_f8_blocks(w->K);
    const size_t  full = (size_t) (w->K / PIB_F8_BLOCK), tail = (size_t) (w->K % PIB_F8_BLOCK);
    if (full) PIB_CHECK(cudaMemcpy2D(out, PIB_F8_BLOCK, w->qs + pib_f8_at(row, 0, KB), PIB_F8_BLOCK * PIB_F8_BLOCK, PIB_F8_BLOCK, full, cudaMemcpyDeviceToHost));
    if (tail) PIB_CHECK(cudaMemcpy((uint8_t *) out + full * PIB_F8_BLOCK, w->qs + pib_f8_at(row, (int64_t) full * PIB_F8_BLOCK, KB), tail, cudaMemcpyDeviceToHost));
    return PIB_OK;
}

static pib_weight * f8_alloc(int64_t N, int64_t K) {
    const size_t sb = N > 0 && K > 0 ? (size_t) pib_f8_blocks(N) * pib_f8_blocks(K) * 4 : 0;
    pib_weight * w  = pib_tiles_alloc(PIB_TYPE_F8, N, K, sb);
    if (w) w->bytes = (size_t) N * K + sb;
    return w;
}

extern "C" pib_weight * pib_weight_from_device_f8(const void * q_dev, const float * scales_dev, int64_t N, int64_t K) {
    if (!q_dev || !scales_dev) { pib_set_error("pib_weight_from_device_f8: bad arguments"); return nullptr; }
    pib_weight * w = f8_alloc(N, K);
    if (!w) return nullptr;
    const size_t sb = (size_t) pib_f8_blocks(N) * pib_f8_blocks(K) * 4;
    if (pib_tiles_fill(w, (const uint8_t *) q_dev, 0, pib_f8_blocks(N) * PIB_F8_BLOCK) != cudaSuccess || cudaMemcpyAsync(w->d, scales_dev, sb, cudaMemcpyDeviceToDevice, 0) != cudaSuccess ||
        cudaStreamSynchronize(0) != cudaSuccess) {
        pib_set_error("pib_weight_from_device_f8: %s", cudaGetErrorString(cudaGetLastError()));
        pib_weight_free(w);
        return nullptr;
    }
    return w;
}

extern "C" pib_weight * pib_weight_upload_f8(const void * q_host, const float * scales_host, int64_t N, int64_t K) {
    if (!q_host || !scales_host) { pib_set_error("pib_weight_upload_f8: bad arguments"); return nullptr; }
    pib_weight * w = f8_alloc(N, K);
    if (!w) return nullptr;
    const size_t sb = (size_t) pib_f8_blocks(N) * pib_f8_blocks(K) * 4;
    bool         ok = pib_tiles_upload(w, (const uint8_t *) q_host) == cudaSuccess;
    ok = ok && cudaMemcpy(w->d, scales_host, sb, cudaMemcpyHostToDevice) == cudaSuccess;
    if (!ok) pib_set_error("pib_weight_upload_f8: %s", cudaGetErrorString(cudaGetLastError()));
    if (!ok) { pib_weight_free(w); return nullptr; }
    return w;
}

int pib_f8_row(const pib_weight * w, int64_t row, void * out) {
    const int64_t KB = pib_f8_blocks(w->K);
    const int     rc = pib_tiles_row(w, row, out);
    if (rc != PIB_OK) return rc;
    PIB_CHECK(cudaMemcpy((uint8_t *) out + w->K, (const float *) w->d + row / PIB_F8_BLOCK * KB, (size_t) KB * 4, cudaMemcpyDeviceToHost));
    return PIB_OK;
}

__device__ __forceinline__ float f8_value(uint8_t q) { return __half2float(__half(__nv_cvt_fp8_to_halfraw(q, __NV_E4M3))); }

static __global__ void f8_rows_kernel(const uint8_t * __restrict__ qs, const float * __restrict__ d, int64_t N, int64_t K, int64_t KB, const int32_t * __restrict__ ids, float * __restrict__ out) {
    pib_pdl_wait();
    pib_pdl_trigger();
    const int64_t row = ids[blockIdx.x];
    for (int64_t k = (int64_t) blockIdx.y * blockDim.x + threadIdx.x; k < K; k += (int64_t) gridDim.y * blockDim.x)
        out[(int64_t) blockIdx.x * K + k] = row < 0 || row >= N ? 0.f : __fmul_rn(f8_value(qs[pib_f8_at(row, k, KB)]), d[row / PIB_F8_BLOCK * KB + k / PIB_F8_BLOCK]);
}

int pib_f8_get_rows(const pib_weight * w, const int32_t * ids, int n, float * out, cudaStream_t st) {
    PIB_CHECK(pib_launch(f8_rows_kernel, dim3((unsigned) n, (unsigned) std::min<int64_t>((w->K + 255) / 256, 64)), dim3(256), 0, st, w->qs, (const float *) w->d, w->N, w->K, pib_f8_blocks(w->K), ids, out));
    return PIB_OK;
}

// ---- activations --------------------------------------------------------------------------------------------------------------------
// A warp per 128 values: four a lane, the block's largest by shuffles, one 128-byte row out.  NORM: a block of threads per token forms the row's mean square first.
// What bounds it: the launch up to a few hundred tokens; beyond that reading the floats.
template <bool NORM, bool VEC>
__global__ void __launch_bounds__(256) f8_quant_kernel(const float * __restrict__ x, const float * __restrict__ nw, float eps, int b, int64_t K, int KB, uint8_t * __restrict__ qs,
                                                       float * __restrict__ d, int bp, float * __restrict__ xnorm) {
    pib_pdl_wait();
    pib_pdl_trigger();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float     rs = 1.f;
    int64_t   u = (int64_t) blockIdx.x * 8 + warp, end = (int64_t) b * KB, step = (int64_t) gridDim.x * 8;
    if (NORM) {
        __shared__ float part[8];
        const int64_t row = blockIdx.x;
        float s = 0.f;
        for (int64_t k = threadIdx.x; k < K; k += 256) { const float v = x[row * K + k]; s = fmaf(v, v, s); }
        s = warp_sum(s);
        if (lane == 0) part[warp] = s;
        __syncthreads();
        s = 0.f;
        for (int i = 0; i < 8; i++) s += part[i];
        rs = 1.0f / sqrtf(s / (float) K + eps);
        u = row * KB + warp; end = (row + 1) * KB; step = 8;
    }
    for (; u < end; u += step) {
        const int64_t row = u / KB, kb = u % KB, k = kb * PIB_F8_BLOCK + lane * 4;
        const float * p = x + row * K + k;
        float v[4];
        if (VEC && k + 3 < K) { const float4 f = *reinterpret_cast<const float4 *>(p); v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w; }
        else
#pragma unroll
            for (int j = 0; j < 4; j++) v[j] = k + j < K ? p[j] : 0.f;
        if (NORM)
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (k + j < K) {
                    v[j] = v[j] * rs * nw[k + j];
                    if (xnorm) xnorm[row * K + k + j] = v[j];
                }
        const float s = f8_scale(warp_max(fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])))));
        reinterpret_cast<uint32_t *>(qs)[(kb * b + row) * 32 + lane] = f8_pack4(v[0], v[1], v[2], v[3], s);
        if (lane == 0) d[kb * bp + row] = s;
    }
}

int pib_f8_quantize(const float * x, const float * norm_w, float eps, int b, int64_t K, void * act, float * xnorm, cudaStream_t st) {
    if (!x || !act || b < 1 || b > PIB_F8_MAX_ROWS || K < 1 || K > 0x7fffff00) {
        pib_set_error("act quantise: bad arguments (8-bit floating point, b %d, K %lld)", b, (long long) K);
        return PIB_ERR_ARG;
    }
    if (((uintptr_t) act & 15) || (((uintptr_t) x | (uintptr_t) norm_w | (uintptr_t) xnorm) & 3)) {
        pib_set_error("act quantise: act_dev needs 16-byte alignment, fp32 rows 4-byte alignment");
        return PIB_ERR_ARG;
    }
    const pib_f8_act A = pib_f8_act_of(K, b);
    uint8_t * q = (uint8_t *) act;
    float *   d = (float *) (q + A.d_off);
    const bool vec = K % 4 == 0 && !((uintptr_t) x & 15);
    if (norm_w) PIB_CHECK(pib_launch(f8_quant_kernel<true, false>, dim3((unsigned) b), dim3(256), 0, st, x, norm_w, eps, b, K, A.KB, q, d, A.bp, xnorm));
    else {
        const dim3 grid((unsigned) std::min<int64_t>(((int64_t) b * A.KB + 7) / 8, 1 << 20));
        if (vec) PIB_CHECK(pib_launch(f8_quant_kernel<false, true>, grid, dim3(256), 0, st, x, norm_w, eps, b, K, A.KB, q, d, A.bp, xnorm));
        else     PIB_CHECK(pib_launch(f8_quant_kernel<false, false>, grid, dim3(256), 0, st, x, norm_w, eps, b, K, A.KB, q, d, A.bp, xnorm));
    }
    return PIB_OK;
}

int pib_f8_act_blocks(const void * act_dev, int b, int64_t K, void * out) {
    if (!act_dev || !out || b < 1 || b > PIB_F8_MAX_ROWS || K < 1) { pib_set_error("pib_act_to_blocks: bad arguments"); return PIB_ERR_ARG; }
    const pib_f8_act A = pib_f8_act_of(K, b);
    uint8_t * h = (uint8_t *) malloc(A.total);
    if (!h) { pib_set_error("pib_act_to_blocks: no host memory"); return PIB_ERR_NOMEM; }
    const cudaError_t e = cudaMemcpy(h, act_dev, A.total, cudaMemcpyDeviceToHost);
    if (e != cudaSuccess) { free(h); PIB_CHECK(e); }
    uint8_t * o = (uint8_t *) out;
    for (int64_t t = 0; t < b; t++)
        for (int64_t kb = 0; kb < A.KB; kb++, o += 4 + PIB_F8_BLOCK) {
            memcpy(o, h + A.d_off + (size_t) (kb * A.bp + t) * 4, 4);
            memcpy(o + 4, h + (size_t) (kb * b + t) * PIB_F8_BLOCK, PIB_F8_BLOCK);
        }
    free(h);
    return PIB_OK;
}

int pib_f8_rows_ok(const char * who, const pib_weight * w, const void * in, const void * out, int b, int max_b) {
    if (w && in && out && b >= 1 && b <= max_b && !((uintptr_t) out & 3)) return PIB_OK;
    pib_set_error("%s: bad arguments (b = %d, limit %d; fp32 rows need 4-byte alignment)", who, b, max_b);
    return PIB_ERR_ARG;
}

int pib_f8_gemm_host(const pib_weight * w, const float * x_host, int b, float * y_host) {
    const int ok = pib_f8_rows_ok("pib_gemm_host", w, x_host, y_host, b, PIB_F8_MAX_ROWS);
    if (ok != PIB_OK) return ok;
    const size_t xb = ((size_t) b * w->K * 4 + 255) & ~(size_t) 255, yb = ((size_t) b * w->N * 4 + 255) & ~(size_t) 255;
    uint8_t *    buf = nullptr;
    PIB_CHECK(cudaMalloc(&buf, xb + yb + pib_f8_act_of(w->K, b).total));
    int rc = PIB_OK;
    if (cudaMemcpy(buf, x_host, (size_t) b * w->K * 4, cudaMemcpyHostToDevice) != cudaSuccess) rc = PIB_ERR_CUDA;
    if (rc == PIB_OK) rc = pib_f8_quantize((const float *) buf, nullptr, 0.f, b, w->K, buf + xb + yb, nullptr, nullptr);
    if (rc == PIB_OK) rc = pib_f8_gemm(w, buf + xb + yb, b, (float *) (buf + xb), nullptr);
    if (rc == PIB_OK) rc = pib_gemm_check(nullptr);
    if (rc == PIB_OK && cudaMemcpy(y_host, buf + xb, (size_t) b * w->N * 4, cudaMemcpyDeviceToHost) != cudaSuccess) { rc = PIB_ERR_CUDA; pib_set_error("pib_gemm_host: %s", cudaGetErrorString(cudaGetLastError())); }
    cudaFree(buf);
    return rc;
}
