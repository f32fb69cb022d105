// i8_block.cuh -- 8-bit integer matrices with a scale for each output, times activations with a scale for each token (PIB_TYPE_I8): layouts and the device code that their kernels share.
//
//   y[t][n] = fp32(sum over k of q[n][k] a[t][k]) * fp32(d[t] s[n])
//
// The sum is a whole number of 32 bits (K <= PIB_I8_MAX_K, 128 * 127 * K < 2^31), so it does not depend on the order of its terms: every kernel, tile and share gives the same bits.
//   weights      qs   int8 in the tiles of the 8-bit floating point matrices (f8_block.cuh): [Np / 128][Kp / 128][128 rows][128 bytes], zero behind the matrix
//                d    fp32 [N]
//   activations  int8 [Kp / 128][b][128], zero behind column K; behind them fp32 [b]
#pragma once

#include "f8_block.cuh"

struct pib_i8_act { int64_t Kp; int KB; size_t d_off, total; };
static inline pib_i8_act pib_i8_act_of(int64_t K, int b) {
    pib_i8_act a;
    a.KB = (int) pib_f8_blocks(K);
    a.Kp = (int64_t) a.KB * PIB_F8_BLOCK;
    a.d_off = ((size_t) b * a.Kp + 255) & ~(size_t) 255;
    a.total = a.d_off + (((size_t) b * 4 + 255) & ~(size_t) 255);
    return a;
}

int pib_i8_quantize(const float * x, const float * norm_w, float eps, int b, int64_t K, void * act, float * xnorm, cudaStream_t st);
int pib_i8_act_blocks(const void * act_dev, int b, int64_t K, void * out);
int pib_i8_row(const pib_weight * w, int64_t row, void * out);
int pib_i8_get_rows(const pib_weight * w, const int32_t * ids, int n, float * out, cudaStream_t st);
int pib_i8_gemv(const pib_weight * w, const void * act, int b, float * y, cudaStream_t st);
int pib_i8_gemv_fused(const pib_weight * w, int pro, const float * x, const float * x2, const float * addend, float * sum_out, int64_t xstride, float eps, int b, float * y, cudaStream_t st);
int pib_i8_gemm(const pib_weight * w, const void * act, int b, float * y, cudaStream_t st);
int pib_i8_gemm_pair(const pib_weight * w, const void * act, int b, float * y, int * err, cudaStream_t st);
int pib_i8_gemm_host(const pib_weight * w, const float * x_host, int b, float * y_host);

// a token's scale from the bits of its largest magnitude, which order infinities and what is no number behind all numbers: a row with one of those has a scale, and outputs, that are none
__device__ __forceinline__ float i8_scale(uint32_t amax) { return amax >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : __fmul_rn(fmaxf(__uint_as_float(amax), F8_MIN_AMAX), 1.0f / 127.0f); }
__device__ __forceinline__ uint32_t i8_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
// a value over the scale, rounded once, then to a whole number (nearest, even); quotients pass 127 by roundings only.  Of a scale that is none: 0
__device__ __forceinline__ int i8_value(float v, float d) {
    const float q = rintf(__fdiv_rn(v, d));
    return (int) fminf(fmaxf(q == q ? q : 0.f, -127.f), 127.f);
}
__device__ __forceinline__ uint32_t i8_pack4(float a, float b, float c, float e, float d) {
    return (uint32_t) (i8_value(a, d) & 255) | (uint32_t) (i8_value(b, d) & 255) << 8 | (uint32_t) (i8_value(c, d) & 255) << 16 | (uint32_t) (i8_value(e, d) & 255) << 24;
}
// sum and scales to an output
__device__ __forceinline__ float i8_out(int sum, float d, float s) { return __fmul_rn(__int2float_rn(sum), __fmul_rn(d, s)); }
