// The 4-bit rows of a key / value cache: rounding 8 elements into a code word, and the value of a scale byte.
//
// Of 32 elements x: s = e4m3(max|x| / 7), c = sign(x) min(7, floor(|x| / s + 1/2)), stored as c + 8.  Every step is exact where it has to be:
//   * max|x| has at most 11 significant bits and the border between two scales at most 5, so that 7 times a border is a number the maximum can be: the fp32
//     quotient falls on the right side of each border as long as it is exact where the quotient is an fp32 number.  It is: the remainder of a first quotient is
//     exact, and a seventh of it added.
//   * |x| times something between 1 / s and (1 + 2^-20) / s is at or above n + 1/2 where |x| / s is (both are fp32 numbers and rounding keeps order), and below
//     it where |x| / s is, since the next lower |x| is 2^-11 of it away.  Halves therefore go up in magnitude, on the device as in the definition.
#pragma once

#include "serving.h"

#include <cuda_fp8.h>

namespace vb200 {

__device__ __forceinline__ float scale_value(uint8_t s) {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw(s, __NV_E4M3)));
}

// the code words of N elements x * back (a power of two) and the scale byte of their group; `lanes`: the 32 / N neighbouring threads that have the group
template <int N>
__device__ __forceinline__ void encode(float (&x)[N], float back, unsigned lanes, uint32_t (&words)[N / 8], uint8_t& scale) {
    float m = 0.f;                          // a NaN stays one
#pragma unroll
    for (int i = 0; i < N; ++i) asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(fabsf(x[i])));
#pragma unroll
    for (int o = 1; o < kKv4Group / N; o <<= 1) {
        const float other = __shfl_xor_sync(lanes, m, o);
        asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(other));
    }
    const bool finite = m < INFINITY;
    m = fminf(m * back, 1e30f);             // (far above the largest scale)
    constexpr float kSeventh = 1.0f / 7.0f;
    float q = m * kSeventh;
    q = fmaf(fmaf(-7.0f, q, m), kSeventh, q);
    scale = finite ? __nv_cvt_float_to_fp8(q, __NV_SATFINITE, __NV_E4M3) : 0x7F;      // NaN
    const float s = scale_value(scale);
    float r = s > 0.f ? __fdividef(1.0000005f, s) : 0.f;                              // (1 + 2^-21 and a little) / s, two units in the last place off at most
    if (m * r >= 7.5f) {                    // the largest scale, or one of the few small ones that lie far below a seventh: codes end at 7
        const float most = 7.0f * s / back;
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = fminf(fmaxf(x[i], -most), most);
    }
    r *= back;
#pragma unroll
    for (int w = 0; w < N / 8; ++w) {
        words[w] = 0x88888888u;
#pragma unroll
        for (int i = 0; i < 8; ++i) words[w] += static_cast<uint32_t>(static_cast<int>(fmaf(x[8 * w + i], r, copysignf(0.5f, x[8 * w + i])))) << (4 * i);
    }
}

}  // namespace vb200
