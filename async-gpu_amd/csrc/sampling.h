// Order of logits, shared by the sampling kernels.
#pragma once
#include "agpu_internal.h"

// Whole numbers in the order of the floats; NaN lowest.
__device__ __forceinline__ uint32_t order_key(float x) {
    if (x != x) return 0u;
    const uint32_t u = x == 0.0f ? 0u : __float_as_uint(x);  // -0.0 and 0.0 are one value
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__device__ __forceinline__ float key_value(uint32_t key) {
    return __uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key);
}
