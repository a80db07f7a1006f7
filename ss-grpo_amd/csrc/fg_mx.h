// Microscaled (MX) rows: 32 consecutive elements of a row are a block; its elements are codes of 8 bits (e4m3) or
// 4 bits (e2m1, two to a byte, the earlier element in the low half) and one byte s gives its scale X = 2^(s - 127)
// (255: the block is NaN). The scales of a [rows, cols] matrix lie as [ceil(cols / 128)][rows][4]: one dword holds
// the four blocks of 128 consecutive elements of a row, the dwords of neighbouring rows are neighbours, and bytes
// behind the last block are 0.
//
// A block that is quantised gets the smallest power of two X >= 2^-126 that holds its largest magnitude a without
// saturation, a <= F X (F = 448 = 1.75 * 2^8 for e4m3, 6 = 1.5 * 2^2 for e2m1), and codes RNE(v / X); a block
// that holds an infinity or a NaN gets s = 255. From the bits of a: its exponent field, plus one where the fraction
// is over that of F (the added constant carries into the exponent exactly then), less F's exponent. The common rule
// that only takes a's exponent saturates up to 1/8 (e4m3) or 1/4 (e2m1) of the largest elements' value; this one
// never does, at the cost of one exponent step for the blocks between.
#pragma once

#include "fg_common.h"

namespace fg {

enum MxFormat : int { kE4M3 = 0, kE2M1 = 1 };
constexpr int kMxBlock = 32;   // elements per scale
constexpr int kMxStep = 128;   // elements per dword of scales

template <int FMT>
FG_DEVICE uint32_t mx_scale_byte(uint32_t amax_bits) {  // amax_bits: of the largest magnitude (sign 0)
  constexpr uint32_t kCarry = FMT == kE4M3 ? 0x1fffffu : 0x3fffffu;
  constexpr int kTop = FMT == kE4M3 ? 8 : 2;
  const int s = (int)((amax_bits + kCarry) >> 23) - kTop;
  return amax_bits >= 0x7f800000u ? 255u : (uint32_t)max(s, 1);
}

// 2^(127 - s), the factor that takes a block's values to its codes' grid (exact: s in [1, 247]); 0 for a NaN block,
// whose codes are of no account.
FG_DEVICE float mx_inverse_scale(uint32_t s) { return __uint_as_float(s == 255u ? 0u : (254u - s) << 23); }

// 2^(s - 127), NaN for 255. s = 0, 2^-127, is a subnormal float.
FG_DEVICE float mx_scale(uint32_t s) {
  return __uint_as_float(s == 255u ? 0x7fc00000u : s == 0u ? 0x00400000u : s << 23);
}

// Eight values, already times mx_inverse_scale, to eight codes: 8 bytes (e4m3) or the low dword (e2m1).
template <int FMT>
FG_DEVICE uint2 mx_pack8(const float (&v)[8]) {
  uint2 r = make_uint2(0u, 0u);
  if constexpr (FMT == kE4M3) {
    int lo = 0, hi = 0;
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], lo, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], lo, true);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[4], v[5], hi, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[6], v[7], hi, true);
    r = make_uint2((uint32_t)lo, (uint32_t)hi);
  } else {
    uint32_t c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0], v[1], 1.0f, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], 1.0f, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], 1.0f, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], 1.0f, 3);
    r.x = c;
  }
  return r;
}

// The largest magnitude of eight values as bits: infinities and NaN are above every number.
FG_DEVICE uint32_t mx_amax8(const float (&v)[8]) {
  uint32_t a = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) a = max(a, __float_as_uint(v[j]) & 0x7fffffffu);  // (v_max3_u32 takes two)
  return a;
}

// Lane l of 16 that share a row's 128-element step holds elements 8l .. 8l + 7 (valid: they are in the row). Writes
// its codes and, from lane 0, the step's dword of scales. All 16 lanes take part.
template <int FMT>
FG_DEVICE void mx_store_step(const float (&v)[8], bool valid, int l, uint8_t* code, uint32_t* scale, bool row_ok) {
  uint32_t a = valid ? mx_amax8(v) : 0u;
  a = max(a, (uint32_t)__shfl_xor((int)a, 1, 64));
  a = max(a, (uint32_t)__shfl_xor((int)a, 2, 64));
  const uint32_t s = mx_scale_byte<FMT>(a);
  uint32_t d = valid ? s << (8 * (l >> 2)) : 0u;
  d |= (uint32_t)__shfl_xor((int)d, 4, 64);
  d |= (uint32_t)__shfl_xor((int)d, 8, 64);
  if (!row_ok) return;
  if (valid) {
    const float inv = mx_inverse_scale(s);
    float y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = v[j] * inv;
    const uint2 c = mx_pack8<FMT>(y);
    if constexpr (FMT == kE4M3)
      *(uint2*)code = c;
    else
      *(uint32_t*)code = c.x;
  }
  if (l == 0) *scale = d;
}

}  // namespace fg
