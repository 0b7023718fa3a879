// The 8-bit KV cache's format (gfx950): e4m3 codes in pools of the 16-bit
// layout [num_blocks, Hkv, block_size, D] and fp32 scales [num_blocks, Hkv, 2]
// (K's, V's), one per pool block and kv head. An entry stands for code * scale.
//
// A scale is a power of two, 2^e with e >= kFp8MinExp, and 0 for a block never
// written. e4m3 is a floating-point code (3 fraction bits, normal from 2^-6 to
// 448), so a finer scale would gain no precision; a power of two makes the
// value code * scale a number of the 16-bit model type itself (4 significant
// bits; a larger scale's codes of an older scale are exact but for
// subnormals), and lets the hardware's scaled conversions (8 -> 16 bits with an
// exponent added, two values an instruction) produce MFMA operands directly.
#pragma once

#include "mv_common.h"

namespace mv {
namespace {

constexpr int kFp8MinExp = -110;
constexpr float kFp8Max = 448.f;

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// The largest magnitude stored of a model type: 240 times the largest scale
// the type needs. The next code up, 256, would stand for a value past the
// type's largest.
template <int DTYPE>
__device__ __forceinline__ constexpr float fp8_limit() {
  return DTYPE == MV_DTYPE_F16 ? 61440.f : 240.f * 1.329227995784916e36f;  // 240 * 2^8, 240 * 2^120
}

// The exponent e of the smallest scale 2^e with amax <= 448 * 2^e = 1.75 *
// 2^(e + 8); kFp8MinExp for 0. amax_bits: the bits of a finite fp32 >= 0.
__device__ __forceinline__ int fp8_scale_exp(uint32_t amax_bits) {
  const int e = static_cast<int>(amax_bits >> 23) - 127 - 8 + ((amax_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return e < kFp8MinExp ? kFp8MinExp : e;
}
__device__ __forceinline__ float exp2i(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

// Four fp32 values as four codes (round to nearest even; |x| <= 448 or NaN).
__device__ __forceinline__ uint32_t fp8_pack(float x0, float x1, float x2, float x3) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(x0, x1, 0, false);
  r = __builtin_amdgcn_cvt_pk_fp8_f32(x2, x3, r, true);
  return static_cast<uint32_t>(r);
}

// Two codes (the low or high half of a word) times a scale, as two 16-bit
// floats of the model type: exact (see above).
template <int DTYPE, bool HI>
__device__ __forceinline__ uint32_t fp8_unpack2(uint32_t codes, float scale) {
  if constexpr (DTYPE == MV_DTYPE_BF16)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, HI));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, scale, HI));
}
// Four codes -> four 16-bit floats.
template <int DTYPE>
__device__ __forceinline__ u32x2 fp8_unpack4(uint32_t codes, float scale) {
  return u32x2{fp8_unpack2<DTYPE, false>(codes, scale), fp8_unpack2<DTYPE, true>(codes, scale)};
}

}  // namespace
}  // namespace mv
