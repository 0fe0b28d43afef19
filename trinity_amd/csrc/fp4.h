// 4-bit blocks of KV caches (OCP microscaling: e2m1 values, one power of two per 32 of them, stored as its exponent + 127)
// to and from the 16-bit element type.  The conversions are single instructions that take the power of two along; they
// round to nearest even, use the exponent of the scale only, and read and write 16-bit subnormals.
#include "common.h"

#if (defined(TRI_BF16) && !defined(TRI_FP4_H_BF16)) || (!defined(TRI_BF16) && !defined(TRI_FP4_H_F16))
#ifdef TRI_BF16
#define TRI_FP4_H_BF16
#else
#define TRI_FP4_H_F16
#endif

namespace tri {

constexpr int kFp4Block = 32;   // values that share a power of two
constexpr int kFp4MinExp = -110;
constexpr int kFp4Nan = 255;    // scale byte of a block that holds an infinity or NaN

__device__ __forceinline__ float fp4_scale(uint32_t byte) { return __uint_as_float(byte << 23); }  // (255: everything reads as NaN)

// eight values: `w` holds their codes, the first in its low four bits
__device__ __forceinline__ half8v fp4x8_to_half8(uint32_t w, float scale) {
#ifdef TRI_BF16
#define TRI_CVT_FP4(i) __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, i)
#else
#define TRI_CVT_FP4(i) __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, i)
#endif
  const auto p0 = TRI_CVT_FP4(0), p1 = TRI_CVT_FP4(1), p2 = TRI_CVT_FP4(2), p3 = TRI_CVT_FP4(3);
#undef TRI_CVT_FP4
  const half8v h = {(half_t)p0[0], (half_t)p0[1], (half_t)p1[0], (half_t)p1[1], (half_t)p2[0], (half_t)p2[1], (half_t)p3[0], (half_t)p3[1]};
  return h;
}

__device__ __forceinline__ uint32_t half8_to_fp4x8(half8v x, float scale) {
  uint32_t w = 0;
#ifdef TRI_BF16
#define TRI_CVT_FP4(i) w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, half2v{x[2 * i], x[2 * i + 1]}, scale, i)
#else
#define TRI_CVT_FP4(i) w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, half2v{x[2 * i], x[2 * i + 1]}, scale, i)
#endif
  TRI_CVT_FP4(0); TRI_CVT_FP4(1); TRI_CVT_FP4(2); TRI_CVT_FP4(3);
#undef TRI_CVT_FP4
  return w;
}

// scale byte of a block with this largest magnitude (its bits without the sign): the least power of two 2^e, e >= -110, of
// which the largest is less than seven - above six and a half it rounds to six, where a larger block's step is two
__device__ __forceinline__ uint32_t fp4_scale_byte(uint32_t amax_bits) {
  const uint32_t f = __float_as_uint((float)__builtin_bit_cast(half_t, (uint16_t)amax_bits));
  if (f >= 0x7F800000u) return kFp4Nan;
  const int e = (int)(f >> 23) - 127 - 2 + ((f & 0x7FFFFFu) >= 0x600000u ? 1 : 0);
  return (uint32_t)((e < kFp4MinExp ? kFp4MinExp : e) + 127);
}

}  // namespace tri

#endif  // once per element type
