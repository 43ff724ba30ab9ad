// The 8-bit floating-point format of the cache, e4m3 (1 sign, 4 exponent bits with bias 7, 3 fraction bits, no infinities, 0x7f and
// 0xff no numbers), and the power-of-two scales that go with it.
#pragma once
#include "attn.h"

#define FP8_MAX 448.0f                       // the largest number, 1.75 * 2^8
#define FP8_MIN_SCALE 5.421010862427522e-20f // 2^-64, the smallest scale: that of a block of zeros
#define FP8_MAX_BLOCK 1024                   // tokens of a block at most (a multiple of 16)

// the smallest power of two from 2^-64 on that leaves amax / scale at most 448; amax is finite and not negative
__device__ __forceinline__ float fp8_scale_of(float amax) {
    // 2^e with e = exponent - 8, one more where the fraction is above 1.75: adding 0x1fffff to the fraction carries just then
    const int e = (int)((__float_as_uint(amax) + 0x1fffffu) >> 23) - 8;
    return __uint_as_float((uint32_t)max(e, 127 - 64) << 23);
}
// e4m3 codes of four numbers, nearest with ties to even, the first in the lowest byte; beyond +-448 (infinities too) the largest
// number, NaN stays NaN
__device__ __forceinline__ float fp8_clamp(float v) { return v != v ? v : fminf(fmaxf(v, -FP8_MAX), FP8_MAX); }
__device__ __forceinline__ uint32_t fp8_pack4(float a, float b, float c, float d) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(fp8_clamp(a), fp8_clamp(b), 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(fp8_clamp(c), fp8_clamp(d), w, true);
    return (uint32_t)w;
}
// the four numbers of a word times `scale`, as codes again
__device__ __forceinline__ uint32_t fp8_rescale4(uint32_t w, float scale) {
    const float2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    return fp8_pack4(lo.x * scale, lo.y * scale, hi.x * scale, hi.y * scale);
}
// eight codes as a matrix operand of 16-bit numbers (exact in both types)
template <typename T> __device__ __forceinline__ typename AttnT<T>::V8 fp8_widen8(uint32_t lo, uint32_t hi);
template <> __device__ __forceinline__ AttnT<__bf16>::V8 fp8_widen8<__bf16>(uint32_t lo, uint32_t hi) {
    return __builtin_bit_cast(AttnT<__bf16>::V8,
                              uint4_t{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false)),
                                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true)),
                                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false)),
                                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true))});
}
template <> __device__ __forceinline__ AttnT<half_t>::V8 fp8_widen8<half_t>(uint32_t lo, uint32_t hi) {
    return __builtin_bit_cast(AttnT<half_t>::V8,
                              uint4_t{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false)),
                                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true)),
                                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false)),
                                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true))});
}
