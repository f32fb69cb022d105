// sample_border.cuh -- the smallest logit on the near side of a border (sample_draw.cu).  Plain C++ as well, so that it is tested without a device.
#pragma once

#include <float.h>
#include <math.h>
#include <stdint.h>
#include <string.h>

#ifdef __CUDACC__
#define SD_HD __host__ __device__ __forceinline__
#define SD_HD_CALL static __host__ __device__ __noinline__      // once in the kernel: code that runs once costs its way from memory
#else
#define SD_HD static inline
#define SD_HD_CALL static inline
#endif

#define SD_FINE    8192                       // bins of l_max - l
#define SD_PER     256.0f                     // for a difference of 1

// floats in their order as whole numbers: neighbours are one apart, the two zeros too
SD_HD uint32_t sd_rank(float v) { uint32_t u; memcpy(&u, &v, 4); return u & 0x80000000u ? ~u : u | 0x80000000u; }
SD_HD float    sd_of_rank(uint32_t r) { const uint32_t u = r & 0x80000000u ? r & 0x7fffffffu : ~r; float v; memcpy(&v, &u, 4); return v; }

// The smallest float with ok(v), where ok holds for every float above one that it holds for, holds for hi and does not for -inf.  From a guess by steps that double, until the border is
// passed, then by halves: two tests where the guess is right, 64 at most.  (Steps of one float do not end near 0: there a difference to l_max stays the same over 10^8 of them.)
template <typename F> SD_HD float sd_least(float guess, float hi, F ok) {
    uint32_t lo = sd_rank(-INFINITY), up = sd_rank(hi), g = sd_rank(guess);       // ok does not hold at lo, it holds at up
    if (g > lo) {
        const bool down = g >= up || ok(sd_of_rank(g));
        if (!down) lo = g; else if (g < up) up = g;
        for (uint32_t step = 1; step < up - lo; step <<= 1) {
            const uint32_t at = down ? up - step : lo + step;
            const bool is = ok(sd_of_rank(at));
            if (is) up = at; else lo = at;
            if (is != down) break;
        }
    }
    while (up - lo > 1) {
        const uint32_t at = lo + (up - lo) / 2;
        if (ok(sd_of_rank(at))) up = at; else lo = at;
    }
    return sd_of_rank(up);
}

SD_HD int sd_fine(float l, float mx) { return (int) fminf((mx - l) * SD_PER, (float) (SD_FINE - 1)); }
// the lowest logit of bin b of l_max - l: sd_fine does not grow with the logit
SD_HD_CALL float sd_bin_floor(int b, float mx) {
    if (b == SD_FINE - 1) return -FLT_MAX;
    return sd_least(mx - (float) (b + 1) / SD_PER, mx, [=](float l) { return sd_fine(l, mx) <= b; });
}

// the smallest logit with e^(l - l_max) >= min_p, 0 < min_p <= 1; the exponential is formed only where the logarithm leaves it open
SD_HD bool sd_enough(float l, float mx, double min_p, double log_p) {
    const double rel = (double) l - (double) mx;
    return rel >= log_p + 1e-12 || (rel > log_p - 1e-12 && exp(rel) >= min_p);
}
SD_HD_CALL float sd_min_p(float min_p, float mx) {
    const double p = (double) min_p, log_p = log(p);
    return sd_least((float) ((double) mx + log_p), mx, [=](float l) { return sd_enough(l, mx, p, log_p); });
}
