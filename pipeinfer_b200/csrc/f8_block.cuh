// f8_block.cuh -- 8-bit floating point matrices with a scale per 128 x 128 block (PIB_TYPE_F8): layouts and the device code that their kernels share.
//
//   weights      qs   e4m3 [Np / 128][Kp / 128][128 rows][128 bytes], N and K rounded up to 128, zero behind the matrix: a block is one piece of 16 KB, a row of it one line of a tile with
//                     128-byte swizzle
//                d    fp32 [Np / 128][Kp / 128]
//   activations  e4m3 [Kp / 128][b][128], zero behind column K; behind them fp32 [Kp / 128][bp], bp = b rounded up to 4: a block's values and scales of neighbouring tokens are neighbours
#pragma once

#include <cuda.h>
#include <cuda_fp8.h>

#include "pib_common.cuh"

#define F8_MIN_AMAX 7.888609052210118e-31f           // 2^-100: below it a block's values are as good as zero, and its scale would leave the normal numbers of fp32
#define F8_MAX      448.0f

// where element (r, k) of a matrix of KB blocks a row lies
__host__ __device__ static inline int64_t pib_f8_at(int64_t r, int64_t k, int64_t KB) { return (((r >> 7) * KB + (k >> 7)) << 14) + ((r & 127) << 7) + (k & 127); }
static inline int64_t pib_f8_blocks(int64_t n) { return (n + PIB_F8_BLOCK - 1) / PIB_F8_BLOCK; }
struct pib_f8_act { int64_t Kp; int KB, bp; size_t d_off, total; };
static inline pib_f8_act pib_f8_act_of(int64_t K, int b) {
    pib_f8_act a;
    a.KB = (int) pib_f8_blocks(K);
    a.Kp = (int64_t) a.KB * PIB_F8_BLOCK;
    a.bp = (b + 3) & ~3;
    a.d_off = ((size_t) b * a.Kp + 255) & ~(size_t) 255;
    a.total = a.d_off + (((size_t) a.KB * a.bp * 4 + 255) & ~(size_t) 255);
    return a;
}

int pib_f8_quantize(const float * x, const float * norm_w, float eps, int b, int64_t K, void * act, float * xnorm, cudaStream_t st);
int pib_f8_act_blocks(const void * act_dev, int b, int64_t K, void * out);
int pib_f8_row(const pib_weight * w, int64_t row, void * out);
int pib_f8_get_rows(const pib_weight * w, const int32_t * ids, int n, float * out, cudaStream_t st);
int pib_f8_gemv(const pib_weight * w, const void * act, int b, float * y, cudaStream_t st);
int pib_f8_gemv_fused(const pib_weight * w, int pro, const float * x, const float * x2, const float * addend, float * sum_out, int64_t xstride, float eps, int b, float * y, cudaStream_t st);
int pib_f8_gemm(const pib_weight * w, const void * act, int b, float * y, cudaStream_t st);
int pib_f8_gemm_pair(const pib_weight * w, const void * act, int b, float * y, int * err, cudaStream_t st);
int pib_f8_gemm_host(const pib_weight * w, const float * x_host, int b, float * y_host);
// the tensor maps of a matrix, made with it (pib_weight::map): boxes of 32, 64, 96 and 128 rows of a block, 128 rows of two blocks (f8_gemm.cu), 16 rows of 16 blocks (f8_gemv.cu), 128 rows (f8_gemm_pair.cu)
struct pib_f8_runs { CUtensorMap m[5]; };
struct pib_f8_maps { pib_f8_runs runs; CUtensorMap stage, block; };
int pib_f8_map(CUtensorMap * map, const void * base, int64_t rows, int box);                   // f8_gemm.cu: rows of 128 bytes, boxes of `box` rows, 128-byte swizzle (these three)
int pib_f8_map3(CUtensorMap * map, const void * base, int64_t rows, int64_t groups, int64_t group_bytes, int box_rows, int box_groups);      // groups of rows of 128 bytes
int pib_f8_map4(CUtensorMap * map, const void * base, int64_t KB, int64_t NB, int box_rows, int box_kb);      // the weights' blocks: boxes of some rows of some blocks of one row block
int pib_f8_rows_ok(const char * who, const pib_weight * w, const void * in, const void * out, int b, int max_b);

// a block's scale: its largest value times 1/448 as fp32 has it
__device__ __forceinline__ float f8_scale(float amax) { return __fmul_rn(fmaxf(amax, F8_MIN_AMAX), 1.0f / F8_MAX); }
// four values over the block's scale, each quotient rounded once, then to e4m3 (nearest, even); a quotient can pass 448 by roundings only, which does not change its e4m3
__device__ __forceinline__ uint32_t f8_pack4(float a, float b, float c, float d, float s) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(__fdiv_rn(a, s), __fdiv_rn(b, s)), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(__fdiv_rn(c, s), __fdiv_rn(d, s)), __NV_SATFINITE, __NV_E4M3);
    return lo | hi << 16;
}
