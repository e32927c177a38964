// Codes and scales of the 8-bit operators (fstu_fp8.hip, fstu_fp8_gemm.hip).
//
// A block of 128 values shares a scale: v ~ scale * code, code an e4m3 value (4 exponent and 3 mantissa bits, largest 448, no
// infinity), scale = max(amax, 2^-100) / 448 in 32 bits, code = the nearest to v * 448 / max(amax, 2^-100), ties to the even one (fp8_cut: exactly
// that for bf16 values; for fp32 ones the quotient is off by up to 2^-23 of itself).  2^-100 keeps the quotients finite for
// blocks of zeros.  amax is the maximum of the values' bits without their sign, in which an infinity is above every number and a NaN
// above that: a block that holds either has a scale that is one too, and stands for nothing but NaN.
#pragma once
#include "fstu_common.h"

#define FP8_BLOCK 128
#define FP8_MOST 448.0f
#define FP8_LEAST 0x1p-100f

template <int CTRL>
__device__ __forceinline__ unsigned fp8_dpp(unsigned v) {
  return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
// The largest of 16 lanes (a DPP row), every lane active.
__device__ __forceinline__ unsigned fp8_max16(unsigned v) {
  v = max(v, fp8_dpp<0xB1>(v));    // quad_perm [1,0,3,2]
  v = max(v, fp8_dpp<0x4E>(v));    // quad_perm [2,3,0,1]
  v = max(v, fp8_dpp<0x141>(v));   // row_half_mirror
  return max(v, fp8_dpp<0x140>(v));   // row_mirror
}
__device__ __forceinline__ unsigned fp8_size(float v) { return __float_as_uint(v) & 0x7fffffffu; }
// A block's scale; an amax that is not a number keeps it from being one.
__device__ __forceinline__ float fp8_scale(float most) { return (most < FP8_LEAST ? FP8_LEAST : most) / FP8_MOST; }
// v * 448 / most as the conversion to a code takes it.  v times a rounded 448 / most is off by 1.5 units of its last place, enough to leave a tie on its wrong
// side, and of bf16 values every 200th quotient is one (of 1.8 M values, 9321 ties, 460 had the other code).  A block that is not finite: NaN throughout.
template <typename T> struct fp8_cut;
// Values of up to 16 bits: bf16, and products of two.  Ties have 5 bits, so that a quotient that is none is more than 2^-21 of itself, 4 units, away from
// one: |448 v - most t| is a whole number of steps in which most * t is below 2^21.  The factor a unit above its rounded value, a quotient is 0 to 3
// units too large, and without its last two bits on the tie or on its own side of it: one instruction a value.
template <> struct fp8_cut<bf16_t> {
  float times;
  __device__ __forceinline__ explicit fp8_cut(float most, bool ordinary = false) {      // ordinary: finite and at least 2^-100
    if (!ordinary && most < FP8_LEAST) most = FP8_LEAST;
    times = ordinary || most < __builtin_inff() ? __uint_as_float(__float_as_uint(FP8_MOST / most) + 1u) : __builtin_nanf("");
  }
  __device__ __forceinline__ float operator()(float v) const { return __uint_as_float(__float_as_uint(v * times) & ~3u); }
};
// fp32: the quotient, corrected by its remainder v * 448/512 - q * most/512, which is exact for values of up to 21 bits.
template <> struct fp8_cut<float> {
  float times, most, inv;
  __device__ __forceinline__ explicit fp8_cut(float m, bool ordinary = false) {
    if (!ordinary && m < FP8_LEAST) m = FP8_LEAST;
    times = ordinary || m < __builtin_inff() ? FP8_MOST / m : __builtin_nanf(""), most = m * (1.f / 512.f), inv = times * (512.f / FP8_MOST);
  }
  __device__ __forceinline__ float operator()(float v) const {
    const float q = v * times;
    return fmaf(-fmaf(q, most, v * (-FP8_MOST / 512.f)), inv, q);      // of this sign, so that a zero keeps its own
  }
};
// Four codes in a word, the first in its low byte.
__device__ __forceinline__ unsigned fp8_pack4(float a, float b, float c, float d) {
  int v = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, v, true);
}

// Whether what is written to rows of b (ldb elements apart, `bytes` each) leaves unread rows of a alone: they are the same rows, or share no byte.
inline bool fp8_same_or_apart(const void* a, int64_t lda, const void* b, int64_t ldb, int rows, int cols, int bytes) {
  if (a == b && (lda == ldb || rows == 1)) return true;
  const int64_t pa = (int64_t)(intptr_t)a, pb = (int64_t)(intptr_t)b, row = (int64_t)cols * bytes;
  const int64_t ra = lda * bytes, rb = ldb * bytes;
  if (pa + (rows - 1) * ra + row <= pb || pb + (rows - 1) * rb + row <= pa) return true;
  if (ra != rb || rows == 1) return false;
  const int64_t off = ((pb - pa) % ra + ra) % ra;      // columns of the same rows
  return off >= row && off + row <= ra;
}
