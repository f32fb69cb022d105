// kv4.cuh -- a layer's keys and values in 4 bits (kv4_cache.cu, kv4_attn.cu): where things lie, and the device code that the kernels share.
//
//   [page][key / value head] records of 80 * dim bytes, so that all that a page holds of a head is one copy:
//     keys    [64 places][dim / 2] bytes, channel c the nibble c % 2 of byte c / 2; behind them [64][dim / 32] pairs of fp16 {step d, lowest value m}
//     values  the same, with rows in another order: of eight places the even ones first (kv4_row), and with heads of 128 the 32-byte halves of a row change places where bit 1 of the row is set
//             (kv4_flip).  The lanes of a matrix product's second operand read quarters of the places 0, 2, 4, 6 at a time: so they lie in different banks
#pragma once

#include <cuda_bf16.h>

#include "pib_common.cuh"

#define KV4_P PIB_KV4_PAGE

struct pib_kv4 {
    int       device, heads, dim;
    int64_t   pages;
    uint8_t * base;
};

__host__ __device__ constexpr int kv4_record(int dim) { return 80 * dim; }
__host__ __device__ constexpr int kv4_half(int dim) { return 40 * dim; }          // the values' part begins here
__host__ __device__ constexpr int kv4_steps(int dim) { return 32 * dim; }         // of either part: its steps and lowest values
__host__ __device__ constexpr int kv4_row(int place) { return (place & ~7) | (place >> 1 & 3) | (place & 1) << 2; }
__host__ __device__ constexpr int kv4_flip(int dim, int row) { return dim == 128 ? (row >> 1 & 1) << 5 : 0; }

// the device's answer: a wrong handle is refused before any launch
static inline int kv4_ok(const char * who, const pib_kv4 * kv) {
    int dev = -1;
    if (!kv) { pib_set_error("%s: no cache", who); return PIB_ERR_ARG; }
    PIB_CHECK(cudaGetDevice(&dev));
    if (dev == kv->device) return PIB_OK;
    pib_set_error("%s: the cache is on device %d, the current one is %d", who, kv->device, dev);
    return PIB_ERR_ARG;
}
static inline int kv4_type_size(int type) { return type == PIB_TYPE_F32 ? 4 : type == PIB_TYPE_BF16 ? 2 : 0; }

// eight nibbles of a word as four pairs {n[i], n[i + 4]} of fp16 numbers.  A nibble or'ed into 1024's last bits is 1024 + n, into the bits above them 1024 + 16 n; both come off exactly.  (Constants by
// their bits: a conversion of theirs stays in the loops.)
__device__ __forceinline__ __half2 kv4_bits(uint32_t v) { return *reinterpret_cast<const __half2 *>(&v); }
// (one instruction for and + or: as two operators they stay two, 256 more for a page and warp)
__device__ __forceinline__ __half2 kv4_in(uint32_t w, uint32_t mask) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(w), "r"(mask), "r"(0x64006400u));
    return kv4_bits(r);
}
__device__ __forceinline__ __half2 kv4_low(uint32_t w)  { return __hadd2(kv4_in(w, 0x000f000fu), kv4_bits(0xe400e400u)); }
__device__ __forceinline__ __half2 kv4_high(uint32_t w) { return __hfma2(kv4_in(w, 0x00f000f0u), kv4_bits(0x2c002c00u), kv4_bits(0xd400d400u)); }
// a value that the compiler keeps instead of forming it again where it is used
__device__ __forceinline__ __half2 kv4_keep(__half2 v) {
    uint32_t r = *reinterpret_cast<const uint32_t *>(&v);
    asm volatile("" : "+r"(r));
    return kv4_bits(r);
}
__device__ __forceinline__ void kv4_pairs(uint32_t w, __half2 d, __half2 m, uint32_t (&o)[4]) {
    const __half2 a = __hfma2(kv4_low(w), d, m), b = __hfma2(kv4_high(w), d, m), c = __hfma2(kv4_low(w >> 8), d, m), e = __hfma2(kv4_high(w >> 8), d, m);
    o[0] = *reinterpret_cast<const uint32_t *>(&a); o[1] = *reinterpret_cast<const uint32_t *>(&b);
    o[2] = *reinterpret_cast<const uint32_t *>(&c); o[3] = *reinterpret_cast<const uint32_t *>(&e);
}
