// Codes and scales of the 8-bit operators (fstu_fp8.hip, fstu_fp8_gemm.hip).
//
// A block of 128 values shares a scale: v ~ scale * code, code an e4m3 value (4 exponent and 3 mantissa bits, largest 448, no
// infinity), scale = max(amax, 2^-100) / 448 in 32 bits, code = v * (448 / max(amax, 2^-100)) to the nearest, ties to the even one:
// off by at most half a code's step and, where the reciprocal's rounding meets a tie, 2^-23 more.  2^-100 keeps the reciprocal finite for
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
// A block's scale and what its values are multiplied by; an amax that is not a number keeps both from being one.
__device__ __forceinline__ float fp8_scale(float most) { return (most < FP8_LEAST ? FP8_LEAST : most) / FP8_MOST; }
__device__ __forceinline__ float fp8_times(float most) { return FP8_MOST / (most < FP8_LEAST ? FP8_LEAST : most); }
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
