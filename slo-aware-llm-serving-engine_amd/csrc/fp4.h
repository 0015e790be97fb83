// The 4-bit KV format: E2M1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their
// negatives) with one E8M0 scale (a power of two, biased by 127) per 32
// channels of a (token, kv head) vector.  Two codes a byte, the even channel in
// the low half.  A page is stored head by head, [kv_heads, block_size, ...], so
// that a wavefront reading one head's tokens reads whole 128-byte lines (a
// token's codes are 64 bytes at head_dim 128; token by token, half of every
// line and seven eighths of every sector of scales would be another head's).
#pragma once
#include "common.h"

namespace slo {

constexpr int kFp4Group = 32;   // channels per scale
constexpr int kFp4MaxCode = 252;  // 6 * 2^(252 - 127) is the largest that stays finite

// Codes of this lane's 8 bf16 values (x) of a 32-channel group held by 4
// adjacent lanes.  The scale is the smallest power of two at which the group's
// largest magnitude is below 7 (at 7 rounding would leave the largest code):
// with the magnitude's bf16 bits b, adding 32 carries into the exponent from a
// mantissa of 1.75 on, and 4 <= 1.0 * 2^2 puts the exponent two below.  Codes
// are x / scale rounded to the nearest value, ties to even, saturating at 6
// (v_cvt_scalef32_pk_fp4_bf16; checked for every bf16 value on gfx950).
// Infinities and NaN count as the largest finite value of their sign.
__device__ __forceinline__ uint32_t e2m1_encode8(const u32x4& x, int floor_code, int& code) {
  uint32_t y[4], top = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t lo = min(x[j] & 0x7fffu, 0x7f7fu), hi = min((x[j] >> 16) & 0x7fffu, 0x7f7fu);
    top = max(top, max(lo, hi));
    y[j] = (x[j] & 0x80008000u) | lo | (hi << 16);
  }
  top = max(top, (uint32_t)__builtin_amdgcn_mov_dpp((int)top, 0xb1, 0xf, 0xf, false));  // quad_perm 1, 0, 3, 2
  top = max(top, (uint32_t)__builtin_amdgcn_mov_dpp((int)top, 0x4e, 0xf, 0xf, false));  // quad_perm 2, 3, 0, 1
  code = min(max((int)((top + 32) >> 7) - 2, floor_code), kFp4MaxCode);
  const float scale = __uint_as_float((uint32_t)code << 23);
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2, y[0]), scale, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2, y[1]), scale, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2, y[2]), scale, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2, y[3]), scale, 3);
}

// The two codes of byte SEL of w times scale (a power of two), as two bf16:
// exact, as a code has two significant bits.
template <int SEL>
__device__ __forceinline__ uint32_t e2m1_pair(uint32_t w, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, SEL));
}

// The 8 codes of a dword times scale, as bf16 in channel order.
__device__ __forceinline__ u32x4 e2m1_decode8(uint32_t w, float scale) {
  return u32x4{e2m1_pair<0>(w, scale), e2m1_pair<1>(w, scale), e2m1_pair<2>(w, scale), e2m1_pair<3>(w, scale)};
}

__device__ __forceinline__ float e8m0(uint32_t code) { return __uint_as_float(code << 23); }

}  // namespace slo
