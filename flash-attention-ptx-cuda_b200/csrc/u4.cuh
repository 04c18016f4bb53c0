// The 4-bit cache: 16 levels for every 64 elements of a row, value = offset + scale * code with scale and
// offset in fp16 (4.5 bits an element).
//
// A quarter of the 16-bit bytes is what attention over a long cache gains from 4 bits, so the format is chosen for
// the reader: codes are whole numbers, exact in either 16-bit type, and scale and offset stand outside the sum
// over the head dimension, sum_d q_d (z + s c_d) = s sum_d q_d c_d + z sum_d q_d, so no element is
// rounded on its way to the tensor core.  64 elements a pair cost 0.5 bits an element; 32 would cost 1 and
// two more sums a key.
//
// The reference has no cache.
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/fa_b200.h"
#include "cache_row.h"

namespace fa {

constexpr int kU4Group = 64;           // elements of a (scale, offset) pair
constexpr float kU4Max = 65504.0f;     // largest finite fp16

// Minimum and maximum that hand a NaN on.
__device__ __forceinline__ float min_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

template <bool BF16>
__device__ __forceinline__ float2 unpack16(uint32_t w) {
    if constexpr (BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
    else return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
    uint32_t r;
    if constexpr (BF16) {
        const __nv_bfloat162 x = __floats2bfloat162_rn(lo, hi);
        r = *reinterpret_cast<const uint32_t*>(&x);
    } else {
        const __half2 x = __floats2half2_rn(lo, hi);
        r = *reinterpret_cast<const uint32_t*>(&x);
    }
    return r;
}

}  // namespace fa
