// Fragments and small arithmetic of the attention kernels' matrix products (gfx950).
#pragma once

#include "ayk_common.h"

namespace ayk {
namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// Eight 16-bit elements of one lane times those of another: D[16][16] += A[16][32] B[32][16]
// (lane l: row or column l % 16, k slots 8 (l / 16) ..; D: column l % 16, rows 4 (l / 16) ..)
// and D[32][32] += A[32][16] B[16][32] (row or column l % 32, k slots 8 (l / 32) ..; D: column
// l % 32, element i at row 8 (i / 4) + 4 (l / 32) + i % 4).
template <int DT>
__device__ inline v4f mfma16(v4u a, v4u b, v4f c) {
  if constexpr (DT == AYK_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
template <int DT>
__device__ inline v16f mfma32(v4u a, v4u b, v16f c) {
  if constexpr (DT == AYK_BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Two fp32 values rounded to nearest even into one dword of 16-bit floats.
template <int DT>
__device__ inline uint32_t pack2(float a, float b) {
  if constexpr (DT == AYK_BF16) return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)a, (__bf16)b});
  else return __builtin_bit_cast(uint32_t, f16x2{(_Float16)a, (_Float16)b});
}

// Two of a dword's four fp8 codes (the low or high pair) widened to 16-bit floats, exactly.
template <int CT, int DT, bool HI>
__device__ inline uint32_t widen2(uint32_t w) {
  if constexpr (CT == AYK_E4M3) {
    if constexpr (DT == AYK_BF16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w, 1.0f, HI));
    else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.0f, HI));
  } else {
    if constexpr (DT == AYK_BF16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8((int)w, 1.0f, HI));
    else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_bf8((int)w, 1.0f, HI));
  }
}

// Four 16-bit elements of one column from LDS: of sixteen lanes that point at 8 bytes each,
// lanes 4 r .. 4 r + 3 at row r of a 4 x 16 block, lane i gets column i.
__device__ inline uint2 read_transposed(const uint8_t* lds) {
  typedef short v4s __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s*)lds));
}

__device__ inline float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// The largest of a lane's scores in one or two products' results, NaN losing to numbers. v_max3 is
// assembly, as fmaxf alone costs a canonicalization an operand. The compiler does not count the wait
// that a read of a matrix product's result needs for an assembly statement; so the chain, every
// link of which waits for the one before, begins with an fmaxf that reads both results.
template <int U>
__device__ inline float max_of_products(const v16f (&s)[U]) {
  static_assert(U == 1 || U == 2, "the first fmaxf reads every product's result");
  float top = fmaxf(s[0][14], s[U - 1][15]);
#pragma unroll
  for (int i = 0; i < 16; i += 3 - U)
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(top) : "v"(top), "v"(s[0][i]), "v"(U == 2 ? s[U - 1][i] : s[0][i + 1]));
  return top;
}

// Maximum and sum over the lanes l, l ^ 32, and over l, l ^ 16, l ^ 32, l ^ 48.
__device__ inline float max_halves(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(f2u(x), f2u(x), false, false);
  return fmaxf(u2f(r[0]), u2f(r[1]));
}
__device__ inline float sum_halves(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(f2u(x), f2u(x), false, false);
  return u2f(r[0]) + u2f(r[1]);
}
__device__ inline float max_quads(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(f2u(x), f2u(x), false, false);
  return max_halves(fmaxf(u2f(r[0]), u2f(r[1])));
}
__device__ inline float sum_quads(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(f2u(x), f2u(x), false, false);
  return sum_halves(u2f(r[0]) + u2f(r[1]));
}

// Sum over the wave, for every lane, and the sum up to each lane, of integers (DPP moves:
// within rows of 16, then across them).
template <int CTRL, int ROWS>
__device__ inline int dpp_int(int v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, false); }
__device__ inline int wave_scan(int v) {
  v += dpp_int<0x111, 0xF>(v);  // row_shr 1, 2, 4, 8
  v += dpp_int<0x112, 0xF>(v);
  v += dpp_int<0x114, 0xF>(v);
  v += dpp_int<0x118, 0xF>(v);
  v += dpp_int<0x142, 0xA>(v);  // the end of rows 0 and 2 to rows 1 and 3, then of row 1 to 2 and 3
  v += dpp_int<0x143, 0xC>(v);
  return v;
}
__device__ inline int wave_total(int v) { return __builtin_amdgcn_readlane(wave_scan(v), kWave - 1); }

// The largest over the wave, and the next lane's value (lane 63: 0), of integers of at least 0.
__device__ inline int wave_most(int v) {
  v = max(v, dpp_int<0x111, 0xF>(v));
  v = max(v, dpp_int<0x112, 0xF>(v));
  v = max(v, dpp_int<0x114, 0xF>(v));
  v = max(v, dpp_int<0x118, 0xF>(v));
  v = max(v, dpp_int<0x142, 0xA>(v));
  v = max(v, dpp_int<0x143, 0xC>(v));
  return __builtin_amdgcn_readlane(v, kWave - 1);
}
__device__ inline int next_lane(int v) { return __builtin_amdgcn_update_dpp(0, v, 0x130, 0xF, 0xF, false); }  // wave_shl 1

constexpr float kLog2e = 1.44269504088896340736f;

}  // namespace
}  // namespace ayk
