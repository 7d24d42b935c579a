// The 4-bit cache format: e2m1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign), two a byte, the
// even dim in the low half, and one UE8M0 scale code for every 32 dims of a row (value 2^(s - 127);
// 0xFF: NaN, the whole group).
//
// Planes are head-major, codes [pages, kv_heads, page_size, dim / 2] and scales [pages, kv_heads,
// page_size, dim / 32]: a head's rows of a page lie side by side. Position-major, a row of 128 dims
// would be 64 bytes beside another head's, half of the cache line that a workgroup fetches for one
// head, and its four scale bytes an eighth of theirs.
#pragma once

#include "ayk_common.h"

namespace ayk {
namespace {

constexpr int kMxGroup = 32;

// Scale code of a group from the bits of its largest magnitude: the least e with amax <= 6 * 2^e,
// as e + 127. 6 * 2^e = 1.5 * 2^(e + 2), so with amax = m * 2^k, 1 <= m < 2, it is k - 2 up to m = 1.5
// and k - 1 above. Magnitudes over 1.5 * 2^127 count as that, so that every finite code stands for
// a finite value; tiny groups take e = -126, zeros code 0, infinities and NaN 0xFF.
__device__ inline uint32_t mx4_scale_code(uint32_t amax_bits) {
  if (amax_bits == 0) return 0;
  if (amax_bits >= 0x7F800000u) return 0xFF;
  const uint32_t b = amax_bits < 0x7F400000u ? amax_bits : 0x7F400000u;
  const int code = (int)(b >> 23) - 2 + ((b & 0x7FFFFFu) > 0x400000u ? 1 : 0);
  return code < 1 ? 1u : (uint32_t)code;
}

// Two values over the scale of `code` as e2m1 codes in one byte, rounded to nearest even and cut at 6.
// The hardware converter equals comparisons with the midpoints for every finite fp32 value
// (compared over all bit patterns on gfx950).
template <int BYTE>
__device__ inline uint32_t mx4_encode2(uint32_t into, float a, float b, uint32_t code) {
  return (uint32_t)__builtin_amdgcn_cvt_scalef32_pk_fp4_f32(into, a, b, u2f(code << 23), BYTE);
}
__device__ inline uint32_t mx4_encode8(const float* x, uint32_t code) {
  if (code == 0xFF) return 0;  // the group is NaN by its scale
  uint32_t w = mx4_encode2<0>(0u, x[0], x[1], code);
  w = mx4_encode2<1>(w, x[2], x[3], code);
  w = mx4_encode2<2>(w, x[4], x[5], code);
  return mx4_encode2<3>(w, x[6], x[7], code);
}

// Two codes (byte BYTE of w) times 2^(code - 127) as bf16, exactly: two significant bits and fp32's exponents.
// `scale` is code << 23; the converter takes 0 for 2^-127 and 0xFF for NaN.
template <int BYTE>
__device__ inline uint32_t mx4_widen2(uint32_t w, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, BYTE));
}
template <int BYTE>
__device__ inline void mx4_decode2(uint32_t w, float scale, float* x) {
  typedef float v2 __attribute__((ext_vector_type(2)));
  const v2 r = __builtin_bit_cast(v2, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, BYTE));
  x[0] = r.x;
  x[1] = r.y;
}
__device__ inline void mx4_decode8(uint32_t w, float scale, float* x) {
  mx4_decode2<0>(w, scale, x);
  mx4_decode2<1>(w, scale, x + 2);
  mx4_decode2<2>(w, scale, x + 4);
  mx4_decode2<3>(w, scale, x + 6);
}

}  // namespace
}  // namespace ayk
