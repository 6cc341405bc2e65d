// logits.h -- logits as the operators over rows of them order and weigh them.
#pragma once

#include <math.h>

#include "common.h"

namespace qraf_hip {

// a logit as it is ordered and weighed: NaN counts as -inf, -0 as +0
__device__ __forceinline__ float clean_logit(float l) { return l == l ? l + 0.0f : -INFINITY; }

__device__ __forceinline__ uint32_t logit_key(float f) {  // a < b  <=>  key(a) < key(b)
    const uint32_t b = __float_as_uint(f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_logit(uint32_t key) {
    return __uint_as_float((key & 0x80000000u) ? (key & 0x7FFFFFFFu) : ~key);
}

// exp((l - m) / T) in 64 bits, within 1e-11 of it (m: the largest logit, not -inf): 2^y as 2^rint(y) times the
// series of 2^f, |f| <= 1/2, to its tenth power.  (The library's exponential, to the last bit: 28 us for the bins of
// 64 rows of 151,936 where this takes 20.)
__device__ __forceinline__ double weight64(float l, float m, double T) {
    const double y = fmax(((double)l - (double)m) * (1.4426950408889634074 / T), -1100.0), n = rint(y), f = y - n;
    double p = 7.0549116208011233e-9;
    p = __builtin_fma(p, f, 1.0178086009239699e-7);
    p = __builtin_fma(p, f, 1.3215486790144309e-6);
    p = __builtin_fma(p, f, 1.5252733804059841e-5);
    p = __builtin_fma(p, f, 1.5403530393381610e-4);
    p = __builtin_fma(p, f, 1.3333558146428443e-3);
    p = __builtin_fma(p, f, 9.6181291076284772e-3);
    p = __builtin_fma(p, f, 5.5504108664821580e-2);
    p = __builtin_fma(p, f, 2.4022650695910071e-1);
    p = __builtin_fma(p, f, 6.9314718055994531e-1);
    p = __builtin_fma(p, f, 1.0);
    p = ldexp(p, (int)n);
    return l == m ? 1.0 : l == -INFINITY || m == INFINITY ? 0.0 : p;
}

}  // namespace qraf_hip
