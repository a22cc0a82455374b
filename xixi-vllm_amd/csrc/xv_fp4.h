// MXFP4 helpers (OCP microscaling, e2m1 codes with one e8m0 scale per 32
// values) on the gfx950 conversion instructions: a code times its block's
// 2^(s - 127) is an exact bf16 value, and a bf16 value divided by the power
// of two and rounded to the nearest code, ties to even, past 6 to 6, is one
// instruction per pair.
#pragma once
#include "xv_common.h"

constexpr int kFp4Block = 32;       // values per scale
constexpr uint32_t kFp4Nan = 0xff;  // the scale byte of a block that held an infinity or NaN

// The fp32 scale operand of the conversions: they use its exponent field alone.
XV_INLINE float fp4_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

XV_INLINE uint32_t bf16x2_bits(xv_bf16x2 v) {
  uint32_t r;
  __builtin_memcpy(&r, &v, 4);
  return r;
}

// The eight codes of w times the scale, as bf16.
XV_INLINE void fp4x8_to_bf16(uint32_t w, float scale, uint32_t (&o)[4]) {
  o[0] = bf16x2_bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0));
  o[1] = bf16x2_bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1));
  o[2] = bf16x2_bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2));
  o[3] = bf16x2_bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3));
}

// The scale byte of a block from `top`, the bf16 bits of its largest magnitude
// (0x7f80 and above: an infinity or NaN among the values).  The exponent of
// the value rounded to one mantissa bit (1.75 and above carries), less 2:
// the largest code, 6, is then never below 6/7 of the largest value.  Kept
// within -126 .. 125, where 6 * 2^e is a finite bf16 and the scale itself a
// normal fp32.
XV_INLINE uint32_t fp4_block_scale(uint32_t top) {
  if (top >= 0x7f80u) return kFp4Nan;
  const int e = (int)((top + 0x20u) >> 7) - 2;
  return (uint32_t)min(max(e, 1), 252);
}

// A lane's 8 of the 32 values of a block that 4 neighbouring lanes hold (a
// DPP quad): the block's scale byte and this lane's 8 codes.
XV_INLINE uint32_t quantise_fp4(const Vec8& x, uint32_t& scale_byte) {
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  u16x2 m = {0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t a = x.w[i] & 0x7fff7fffu;
    u16x2 v;
    __builtin_memcpy(&v, &a, 4);
    m = __builtin_elementwise_max(m, v);
  }
  uint32_t top = max((uint32_t)m[0], (uint32_t)m[1]);
  top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x4E, 0xf, 0xf, false));  // quad_perm [2,3,0,1]
  top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0xB1, 0xf, 0xf, false));  // quad_perm [1,0,3,2]
  scale_byte = fp4_block_scale(top);
  if (scale_byte == kFp4Nan) return 0u;  // the codes of such a block are zero, whatever its values
  const float s = fp4_scale(scale_byte);
  xv_bf16x2 v[4];
  __builtin_memcpy(v, x.w, 16);
  uint32_t r = 0;
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, v[0], s, 0);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, v[1], s, 1);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, v[2], s, 2);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, v[3], s, 3);
  return r;
}

// LDS images of operand rows.  ds_read_b128 serves a wave in four phases, the
// first of lanes 0-3, 12-15 and 20-27, the second of 4-11, 16-19 and 28-31,
// the others 32 lanes on (measured: two lanes of one phase on one bank cost a
// cycle more).  A lane (g, i) of an operand reads row i's 16-byte piece c(g), so
// a phase holds rows 0-3 and 12-15 with one piece and 4-11 with the next: the
// swizzles below give those sixteen reads sixteen different bank groups
// (XOR with the row number alone collides pairwise: 8 cycles a read, not 4).
// Rows of 64 bytes (4 pieces): piece j of row r in slot j ^ swz4(r).
XV_INLINE int swz4(int r) { return (0x78 >> (2 * ((r >> 2) & 3))) & 3; }
// Rows of 128 bytes (8 pieces).
XV_INLINE int swz8p(int r) { return ((r >> 1) + 2) & 7; }
// Rows of 256 bytes and more, the pieces of neighbouring lane groups 1 or 4 apart (the low four bits of the piece).
XV_INLINE int swz16(int r) { return (r + 4) & 15; }
