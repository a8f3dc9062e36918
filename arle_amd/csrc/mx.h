// Microscaled numbers: blocks of 32 consecutive numbers of a row that share a power of two.
//
// A block's scale is 2^(code - 127), code one byte; an element is e4m3 (8 bits, largest 448) or e2m1 (4 bits, largest 6, the
// number with the lower index in the lower half of a byte).  code is the smallest with which no number of the block is past the
// element type's largest: with amax = 2^e (1 + f), code = e - 8 (+ 1 if 1 + f > 1.75) for e4m3, e - 2 (+ 1 if 1 + f > 1.5) for e2m1,
// never under 0.  (The exponent of amax alone, without the carry, would cut the largest number of a block by up to an
// eighth, or a quarter; so it keeps the element's own half step.)  Elements round to nearest, ties to even: two of a floating type's
// steps are then what a block loses, and numbers under 2^-6 of the scale (e2m1: under 1/2, of which 1/4 and less become 0).  A block with a NaN or an
// infinity has code 255, a scale that is NaN, and elements of 0.  The codes come from the bits of amax, so that equal rows
// have equal codes whatever kernel makes them.
#pragma once
#include "common.h"

namespace arle {

constexpr int kMxBlock = 32;
constexpr int kMx8 = 8, kMx4 = 4;   // bits of an element, shared with the Python side

typedef int mx_i32x8 __attribute__((ext_vector_type(8)));
typedef int mx_i32x4 __attribute__((ext_vector_type(4)));
typedef float mx_f32x4 __attribute__((ext_vector_type(4)));
typedef float mx_f32x16 __attribute__((ext_vector_type(16)));

// The larger of the absolute values as bits: a NaN is past every number, so that no maximum loses it.
__device__ __forceinline__ uint32_t mx_abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t mx_max4(float4 v) {
  return max(max(mx_abs_bits(v.x), mx_abs_bits(v.y)), max(mx_abs_bits(v.z), mx_abs_bits(v.w)));
}
template <int CTRL>
__device__ __forceinline__ uint32_t row_move_bits(uint32_t v) {
  return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, 0xf, 0xf, true));
}
// Over 4 or 8 neighbouring lanes, the result in each of them.
template <int LANES>
__device__ __forceinline__ uint32_t mx_lanes_max(uint32_t v) {
  static_assert(LANES == 4 || LANES == 8, "the lanes that share a block");
  v = max(v, row_move_bits<0xB1>(v));                            // quad_perm [1, 0, 3, 2]
  v = max(v, row_move_bits<0x4E>(v));                            // quad_perm [2, 3, 0, 1]
  if constexpr (LANES == 8) v = max(v, row_move_bits<0x141>(v));  // row_half_mirror
  return v;
}

template <int BITS>
__device__ __forceinline__ uint32_t mx_code(uint32_t amax_bits) {
  constexpr int kExponent = BITS == kMx8 ? 8 : 2;
  constexpr uint32_t kFraction = BITS == kMx8 ? 0x600000u : 0x400000u;   // 1.75 and 1.5
  const int e = static_cast<int>(amax_bits >> 23);
  const int code = e - kExponent + ((amax_bits & 0x7fffffu) > kFraction ? 1 : 0);
  return e == 255 ? 255u : static_cast<uint32_t>(max(code, 0));
}
// The scale as a float; 2^-127 has no exponent field of its own.
__device__ __forceinline__ float mx_scale(uint32_t code) { return __uint_as_float(code == 0 ? 0x00400000u : (code == 255 ? 0x7fc00000u : code << 23)); }

// Four numbers as elements: e4m3 a whole register, e2m1 its lower half.  (The hardware divides by the scale's power of two.)
template <int BITS>
__device__ __forceinline__ uint32_t mx_pack4(float4 v, uint32_t code) {
  if (code == 255u) return 0u;
  const float s = mx_scale(code);
  if constexpr (BITS == kMx8) {
    typedef short s16x2 __attribute__((ext_vector_type(2)));
    s16x2 r = {0, 0};
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, v.x, v.y, s, false);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, v.z, v.w, s, true);
    return __builtin_bit_cast(uint32_t, r);
  } else {
    uint32_t r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, v.x, v.y, s, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v.z, v.w, s, 1);
    return r & 0xffffu;
  }
}
template <int BITS>
__device__ __forceinline__ void mx_store4(uint8_t* row, int col, uint32_t packed) {
  if constexpr (BITS == kMx8)
    *reinterpret_cast<uint32_t*>(row + col) = packed;
  else
    *reinterpret_cast<uint16_t*>(row + col / 2) = static_cast<uint16_t>(packed);
}

}  // namespace arle
