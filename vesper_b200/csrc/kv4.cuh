// The 4-bit rows of a key / value cache: rounding 8 elements into a code word, and the value of a scale byte.
//
// Of 32 elements x: s = e4m3(max|x| / 7), c = sign(x) min(7, floor(|x| / s + 1/2)), stored as c + 8.  Every step is exact where it has to be:
//   * max|x| has at most 11 significant bits and the border between two scales at most 5, so that 7 times a border is a number the maximum can be: the fp32
//     quotient, correctly rounded, falls on the right side of each border, and on it only where the exact one does;
//   * |x| * (1 / s), with 1 / s rounded up, is at or above n + 1/2 where |x| / s is (both are fp32 numbers and rounding keeps order), and below it where
//     |x| / s is, since the next lower |x| is 2^-11 of it away.  Halves therefore go up in magnitude, on the device as in the definition.
#pragma once

#include "serving.h"

#include <cuda_fp8.h>

namespace vb200 {

__device__ __forceinline__ float scale_value(uint8_t s) {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw(s, __NV_E4M3)));
}

// the code word of 8 elements x * back and the scale byte of their group; `lanes`: the threads of the group
__device__ __forceinline__ uint32_t encode8(const float (&x)[8], float back, unsigned lanes, uint8_t& scale) {
    float y[8], m = 0.f, odd = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        y[i] = x[i] * back;
        m = fmaxf(m, fabsf(y[i]));
        odd += x[i] * 0.f;                  // 0, or NaN where an element is not finite
    }
#pragma unroll
    for (int o = 1; o <= 2; o <<= 1) {
        m = fmaxf(m, __shfl_xor_sync(lanes, m, o));
        odd += __shfl_xor_sync(lanes, odd, o);
    }
    scale = __nv_cvt_float_to_fp8(__fdiv_rn(m, 7.0f), __NV_SATFINITE, __NV_E4M3);
    if (odd != 0.f) scale = 0x7F;           // NaN
    const float s = scale_value(scale);
    const float r = s > 0.f ? __frcp_ru(s) : 0.f;
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int c = min(7, static_cast<int>(fmaf(fabsf(y[i]), r, 0.5f)));
        word |= static_cast<uint32_t>(8 + (y[i] < 0.f ? -c : c)) << (4 * i);
    }
    return word;
}

}  // namespace vb200
