// tl_fp8.hpp -- fp32 values to E4M3 codes, and the scale of a row of them.
#pragma once

#include "tl_device.hpp"

namespace tl {

__device__ __forceinline__ float fp8_sat(float v) {
  const float c = __builtin_fminf(__builtin_fmaxf(v, -448.0f), 448.0f);
  return (v != v) ? v : c;
}
__device__ __forceinline__ uint32_t pack4_fp8(float a, float b, float c, float d) {
  uint32_t w = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(fp8_sat(a), fp8_sat(b), 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(fp8_sat(c), fp8_sat(d), (int)w, true);
}

// The scale of a row or group whose largest magnitude is amax (its bits:
// magnitudes order as unsigned integers, infinities and NaN last), and what
// its elements are multiplied by before they are rounded.  scale = amax / 448
// (fp8_gemm.cu:80-84).  A row without a scale that fp32 holds as a normal
// number (all zeros, or below 448 x 2^-126) is kept as zeros under scale 0; a
// row with an infinity or a NaN has the scale NaN, under which every code
// reads as NaN.
struct Fp8Scale {
  float scale, inv;
};
__device__ __forceinline__ Fp8Scale fp8_scale_of(uint32_t amax_bits) {
  if (amax_bits >= 0x7f800000u) return {__builtin_bit_cast(float, 0x7fc00000u), __builtin_bit_cast(float, 0x7fc00000u)};
  // The quotient by the constant, corrected by its exact remainder: the same
  // number as a / 448 for every a with a normal quotient; and the reciprocal
  // with one Newton step, within 2^-24 (checked on the CPU over whole binades
  // and the threshold's).  A division is about ten instructions, these are
  // three and four.
  constexpr float kInv = 1.0f / 448.0f;
  const float a = __builtin_bit_cast(float, amax_bits), q = a * kInv;
  const float s = __builtin_fmaf(__builtin_fmaf(-q, 448.0f, a), kInv, q);
  const float r = __builtin_amdgcn_rcpf(s), inv = __builtin_fmaf(__builtin_fmaf(-s, r, 1.0f), r, r);
  return s >= 1.17549435e-38f ? Fp8Scale{s, inv} : Fp8Scale{0.f, 0.f};
}
// Elements times the inverse of their own row's scale, which is a few parts in
// 2^23 above 448 at most and so rounds to it: not saturated.
__device__ __forceinline__ uint32_t pack4_fp8_found(float a, float b, float c, float d) {
  const uint32_t w = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, (int)w, true);
}
__device__ __forceinline__ uint32_t abs_bits(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7fffffffu; }

// A lane's bits of another lane of its row of 16 (a DPP control of tl_device.hpp).
template <int CTRL>
__device__ __forceinline__ uint32_t lane_bits(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xF, 0xF, true);
}
__device__ __forceinline__ uint32_t lanes_umax_16(uint32_t v) {   // with lane ^ 16
  const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  return max((uint32_t)r[0], (uint32_t)r[1]);
}
__device__ __forceinline__ uint32_t lanes_umax_32(uint32_t v) {   // with lane ^ 32
  const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return max((uint32_t)r[0], (uint32_t)r[1]);
}
// Max over the aligned group of LANES lanes that a lane is in.
template <int LANES>
__device__ __forceinline__ uint32_t lanes_umax(uint32_t v) {
  static_assert(LANES >= 1 && LANES <= 64 && (LANES & (LANES - 1)) == 0, "a power of two");
  if constexpr (LANES >= 2) v = max(v, lane_bits<kDppXor1>(v));
  if constexpr (LANES >= 4) v = max(v, lane_bits<kDppXor2>(v));
  if constexpr (LANES >= 8) v = max(v, lane_bits<kDppHalfMirror>(v));
  if constexpr (LANES >= 16) v = max(v, lane_bits<kDppMirror>(v));
  if constexpr (LANES >= 32) v = lanes_umax_16(v);
  if constexpr (LANES >= 64) v = lanes_umax_32(v);
  return v;
}

}  // namespace tl
