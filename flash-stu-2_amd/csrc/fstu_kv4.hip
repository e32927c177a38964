// The 4-bit ring cache: keys and values to codes as they are written, back to values, and the attention of one query a sequence over it.
#include "fstu_common.h"
#include "fstu_kv4.h"

namespace {

typedef float f32x2_t __attribute__((ext_vector_type(2)));

// The scale's byte for a block whose largest size has these bits: the smallest power of two with amax <= 7 * 2^e.  Its codes end at 6
// and steps beside that are 2 wide, so nothing is off by more than 2^e.  -120 <= e <= 125: every code's value is a normal bf16 (sizes beyond 7 * 2^125, 1.75 * 2^127,
// become 6 * 2^125 all the same, off by up to 2 * 2^125).
__device__ __forceinline__ unsigned kv4_scale(unsigned amax) {
  const unsigned ex = amax >> 23;
  if (ex == 255) return 255;
  const int b = (int)ex - ((amax & 0x7fffff) <= 0x600000 ? 2 : 1);
  return (unsigned)min(max(b, 7), 252);
}
__device__ __forceinline__ float kv4_scale_value(unsigned byte) { return __uint_as_float(byte << 23); }

template <typename T>
__device__ __forceinline__ void load8(const T* p, float* o) {
  if constexpr (sizeof(T) == 2) {
    const uint4 v = *(const uint4*)p;
    const unsigned w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { o[2 * i] = __uint_as_float(w[i] << 16); o[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
  } else {
    const float4 a = ((const float4*)p)[0], b = ((const float4*)p)[1];
    o[0] = a.x; o[1] = a.y; o[2] = a.z; o[3] = a.w;
    o[4] = b.x; o[5] = b.y; o[6] = b.z; o[7] = b.w;
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float* o) {
  if constexpr (sizeof(T) == 2) {
    *(uint4*)p = make_uint4(pack2_bf16(o[0], o[1]), pack2_bf16(o[2], o[3]), pack2_bf16(o[4], o[5]), pack2_bf16(o[6], o[7]));
  } else {
    ((float4*)p)[0] = make_float4(o[0], o[1], o[2], o[3]);
    ((float4*)p)[1] = make_float4(o[4], o[5], o[6], o[7]);
  }
}

// Where byte b of chunk c's (hd/16 dims) piece at slot i of eight lies: pieces of hd/4 bytes in planes of 16.
template <int HD>
__device__ __forceinline__ int value_at(int c, int i, int b) {
  const int at = i * (HD / 32) + b;
  return HD <= 64 ? c * (HD / 4) + at : (at & ~15) * 16 + c * 16 + (at & 15);
}
// Codes of dims 8u .. 8u + 7 of a value at one slot (a word, low nibble first).
template <int HD>
__device__ __forceinline__ void put_value(unsigned char* tile, int i, int u, unsigned code) {       // slot i of the eight at `tile`
  if constexpr (HD >= 128) *(unsigned*)(tile + value_at<HD>(u * 128 / HD, i, u * 4 % (HD / 32))) = code;
  else if constexpr (HD == 64) {
    *(unsigned short*)(tile + value_at<HD>(2 * u, i, 0)) = (unsigned short)code;
    *(unsigned short*)(tile + value_at<HD>(2 * u + 1, i, 0)) = (unsigned short)(code >> 16);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) tile[value_at<HD>(4 * u + e, i, 0)] = (unsigned char)(code >> (8 * e));
  }
}
template <int HD>
__device__ __forceinline__ unsigned get_value(const unsigned char* tile, int i, int u) {
  if constexpr (HD >= 128) return *(const unsigned*)(tile + value_at<HD>(u * 128 / HD, i, u * 4 % (HD / 32)));
  else if constexpr (HD == 64)
    return *(const unsigned short*)(tile + value_at<HD>(2 * u, i, 0)) | (unsigned)*(const unsigned short*)(tile + value_at<HD>(2 * u + 1, i, 0)) << 16;
  else {
    unsigned code = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) code |= (unsigned)tile[value_at<HD>(4 * u + e, i, 0)] << (8 * e);
    return code;
  }
}
// The same at all eight slots (hd up to 128), pieces of four, two or one byte a slot: 32 bytes beside each other, at hd 128 two halves of a plane each.
template <int HD>
__device__ __forceinline__ void eight_to_pieces(const unsigned* code, unsigned* w) {
  if constexpr (HD == 128) {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = code[i];
  } else if constexpr (HD == 64) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = __builtin_amdgcn_perm(code[2 * i + 1], code[2 * i], 0x05040100);
      w[4 + i] = __builtin_amdgcn_perm(code[2 * i + 1], code[2 * i], 0x07060302);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {                              // a 4 x 4 transposition of bytes
      const unsigned ab = __builtin_amdgcn_perm(code[4 * i + 1], code[4 * i], 0x05010400), cd = __builtin_amdgcn_perm(code[4 * i + 3], code[4 * i + 2], 0x05010400);
      const unsigned AB = __builtin_amdgcn_perm(code[4 * i + 1], code[4 * i], 0x07030602), CD = __builtin_amdgcn_perm(code[4 * i + 3], code[4 * i + 2], 0x07030602);
      w[0 + i] = __builtin_amdgcn_perm(cd, ab, 0x05040100);
      w[2 + i] = __builtin_amdgcn_perm(cd, ab, 0x07060302);
      w[4 + i] = __builtin_amdgcn_perm(CD, AB, 0x05040100);
      w[6 + i] = __builtin_amdgcn_perm(CD, AB, 0x07060302);
    }
  }
}
template <int HD>
__device__ __forceinline__ void pieces_to_eight(const unsigned* w, unsigned* code) {
  if constexpr (HD == 128) {
#pragma unroll
    for (int i = 0; i < 8; ++i) code[i] = w[i];
  } else if constexpr (HD == 64) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      code[2 * i] = __builtin_amdgcn_perm(w[4 + i], w[i], 0x05040100);
      code[2 * i + 1] = __builtin_amdgcn_perm(w[4 + i], w[i], 0x07060302);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const unsigned ab = __builtin_amdgcn_perm(w[2 + i], w[i], 0x05010400), cd = __builtin_amdgcn_perm(w[6 + i], w[4 + i], 0x05010400);
      const unsigned AB = __builtin_amdgcn_perm(w[2 + i], w[i], 0x07030602), CD = __builtin_amdgcn_perm(w[6 + i], w[4 + i], 0x07030602);
      code[4 * i] = __builtin_amdgcn_perm(cd, ab, 0x05040100);
      code[4 * i + 1] = __builtin_amdgcn_perm(cd, ab, 0x07060302);
      code[4 * i + 2] = __builtin_amdgcn_perm(CD, AB, 0x05040100);
      code[4 * i + 3] = __builtin_amdgcn_perm(CD, AB, 0x07060302);
    }
  }
}
template <int HD>
__device__ __forceinline__ unsigned char* kv4_scale_at(unsigned char* s, int64_t at, int slot, int blk) {      // at: the head's first slot
  return s + (at + (slot & ~7)) * (HD / 32) + blk * 8 + (slot & 7);
}

__device__ __forceinline__ unsigned quad_max(unsigned v) {     // over each four lanes
  v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, true));
  return max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, true));
}

// Four lanes to a block of 32 values: eight each, their largest size by three exchanges of bits (which order infinities and NaN behind all else).
__device__ __forceinline__ unsigned kv4_quantise(const float* x, unsigned* byte) {
  unsigned m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
  *byte = kv4_scale(quad_max(m));
  if (*byte == 255) return 0;
  const float s = kv4_scale_value(*byte);
  unsigned code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, x[0], x[1], s, 0);
  code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, x[2], x[3], s, 1);
  code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, x[4], x[5], s, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, x[6], x[7], s, 3);
}
__device__ __forceinline__ void kv4_values(unsigned code, unsigned byte, float* o) {
  const float s = kv4_scale_value(byte);
  const f32x2_t a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, s, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, s, 1);
  const f32x2_t c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, s, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, s, 3);
  o[0] = a.x; o[1] = a.y; o[2] = b.x; o[3] = b.y; o[4] = c.x; o[5] = c.y; o[6] = d.x; o[7] = d.y;
}

// Eight slots' worth of a sequence's new rows: the rows that go to slots sl .. sl + 7 of it, as far as there are such.
struct Eight {
  int s, at, len, t, slot, p;      // sequence, its first row and rows, the group's first row in it (or up to 7 in front of it), that one's slot, position
  bool whole;                      // eight rows and eight slots beside each other, from a multiple of 8 on
};
// Group number n: a sequence's groups begin at cu[s] / 8 + 2 s, which leaves room for a partial one at each end.
__device__ __forceinline__ Eight eight_of(const int* cu, const int* pos, int seqs, int rows, int cap, int n) {
  Eight g;
  g.s = fstu_last_where(seqs, [&](int i) { return max(cu[i], 0) / 8 + 2 * i <= n; });
  g.at = min(max(cu[g.s], 0), rows);
  g.len = min(max(cu[g.s + 1], g.at), rows) - g.at;
  g.p = pos[g.s];
  const int first = g.p < 0 ? 0 : g.p % cap;
  g.t = (n - (g.at / 8 + 2 * g.s)) * 8 - (first & 7);
  g.slot = (int)((unsigned)(first + g.t) % (unsigned)cap);
  g.whole = g.t >= 0 && g.t + 8 <= g.len && g.slot % 8 == 0 && g.slot + 8 <= cap;
  return g;
}

// A workgroup takes a group of eight slots (ONE: one row of a sequence), keys where y = 0 and values where y = 1; a thread eight dims of a head.  Each thread's
// eight rows are asked for together, and what it leaves is 32 bytes beside each other (keys: 4 in each of eight rows).  16384 rows of 16 x 128 in bf16, written and
// read back: 132 us with a row's eight dims to a thread, 76 so, 4.5 TB/s: bytes bound it, the bf16 rows 79 % of them; a token a row the launch and one trip to
// memory.
template <typename T, int HD, bool ONE>
__global__ void __launch_bounds__(256)
kv4_write_kernel(const T* k, const T* v, int64_t k_row, int64_t k_head, int64_t v_row, int64_t v_head, void* cache, const int* pos, const int* cu, int rows,
                 int seqs, int kvh, int cap) {
  constexpr int P = HD / 8, kPiece = HD == 128 ? 16 : 32, kPlane = HD == 128 ? 256 : 16;
  const Kv4 c = kv4_at(cache, (int64_t)seqs * kvh, HD, cap);
  const bool keys = blockIdx.y == 0;
  const T* const x = keys ? k : v;
  const int64_t x_row = keys ? k_row : v_row, x_head = keys ? k_head : v_head;
  if constexpr (ONE) {
    const int s = blockIdx.x, p = pos[s];
    if (p < 0) return;
    const int slot = p % cap;
    for (int e = threadIdx.x; e < kvh * P; e += blockDim.x) {
      const int h = e / P, u = e % P;
      const int64_t at = ((int64_t)s * kvh + h) * c.slots;
      float f[8];
      unsigned byte;
      load8(x + s * x_row + h * x_head + u * 8, f);
      const unsigned code = kv4_quantise(f, &byte);
      if (keys) *(unsigned*)(c.kc + (at + slot) * (HD / 2) + u * 4) = code;
      else put_value<HD>(c.vc + (at + (slot & ~7)) * (HD / 2), slot & 7, u, code);
      if ((u & 3) == 0) *kv4_scale_at<HD>(keys ? c.ks : c.vs, at, slot, u / 4) = (unsigned char)byte;
    }
    return;
  }
  const Eight g = eight_of(cu, pos, seqs, rows, cap, blockIdx.x);
  if (g.p < 0 || g.len == 0 || g.t >= g.len || g.t <= -8) return;
  const int from = max(0, g.len - cap);
  for (int e = threadIdx.x; e < kvh * P; e += blockDim.x) {
    const int h = e / P, u = e % P;
    const int64_t at = ((int64_t)g.s * kvh + h) * c.slots;
    const T* src = x + h * x_head + u * 8;
    float f[8][8];
    unsigned code[8], byte[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) load8(src + (g.at + min(max(g.t + i, 0), g.len - 1)) * x_row, f[i]);
#pragma unroll
    for (int i = 0; i < 8; ++i) code[i] = kv4_quantise(f[i], &byte[i]);
    if (g.whole && g.t >= from) {
      if (keys) {
        unsigned char* dst = c.kc + (at + g.slot) * (HD / 2) + u * 4;
#pragma unroll
        for (int i = 0; i < 8; ++i) *(unsigned*)(dst + i * (HD / 2)) = code[i];
      } else {
        unsigned char* tile = c.vc + (at + g.slot) * (HD / 2);
        if constexpr (HD <= 128) {
          unsigned w[8];
          eight_to_pieces<HD>(code, w);
          *(uint4*)(tile + u * kPiece) = make_uint4(w[0], w[1], w[2], w[3]);
          *(uint4*)(tile + u * kPiece + kPlane) = make_uint4(w[4], w[5], w[6], w[7]);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) put_value<HD>(tile, i, u, code[i]);
        }
      }
      if ((u & 3) == 0)
        *(uint2*)kv4_scale_at<HD>(keys ? c.ks : c.vs, at, g.slot, u / 4) = make_uint2(byte[0] | byte[1] << 8 | byte[2] << 16 | byte[3] << 24,
                                                                                    byte[4] | byte[5] << 8 | byte[6] << 16 | byte[7] << 24);
      continue;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (g.t + i < from || g.t + i >= g.len) continue;
      const int slot = (int)((unsigned)(g.slot + i) % (unsigned)cap);
      if (keys) *(unsigned*)(c.kc + (at + slot) * (HD / 2) + u * 4) = code[i];
      else put_value<HD>(c.vc + (at + (slot & ~7)) * (HD / 2), slot & 7, u, code[i]);
      if ((u & 3) == 0) *kv4_scale_at<HD>(keys ? c.ks : c.vs, at, slot, u / 4) = (unsigned char)byte[i];
    }
  }
}

template <typename T, int HD, bool ONE>
__global__ void __launch_bounds__(256)
kv4_read_kernel(const void* cache, T* k, T* v, const int* pos, const int* cu, int rows, int seqs, int kvh, int cap) {
  constexpr int P = HD / 8, kPiece = HD == 128 ? 16 : 32, kPlane = HD == 128 ? 256 : 16;
  const Kv4 c = kv4_at((void*)cache, (int64_t)seqs * kvh, HD, cap);
  const bool keys = blockIdx.y == 0;
  T* const y = keys ? k : v;
  const int64_t row = (int64_t)kvh * HD;
  if constexpr (ONE) {
    const int s = blockIdx.x, p = pos[s];
    const int slot = p < 0 ? 0 : p % cap;
    for (int e = threadIdx.x; e < kvh * P; e += blockDim.x) {
      const int h = e / P, u = e % P;
      const int64_t at = ((int64_t)s * kvh + h) * c.slots;
      float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (p >= 0)
        kv4_values(keys ? *(const unsigned*)(c.kc + (at + slot) * (HD / 2) + u * 4) : get_value<HD>(c.vc + (at + (slot & ~7)) * (HD / 2), slot & 7, u),
                   *kv4_scale_at<HD>(keys ? c.ks : c.vs, at, slot, u / 4), f);
      store8(y + s * row + e * 8, f);
    }
    return;
  }
  const int begin = min(max(cu[0], 0), rows), end = min(max(cu[seqs], begin), rows);
  for (int r = blockIdx.x; r < begin + rows - end; r += gridDim.x)               // rows of no sequence
    for (int e = threadIdx.x; e < kvh * P; e += blockDim.x) {
      const float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      store8(y + (r < begin ? r : end + r - begin) * row + e * 8, f);
    }
  const Eight g = eight_of(cu, pos, seqs, rows, cap, blockIdx.x);
  if (g.t >= g.len || g.t <= -8) return;
  for (int e = threadIdx.x; e < kvh * P; e += blockDim.x) {
    const int h = e / P, u = e % P;
    const int64_t at = ((int64_t)g.s * kvh + h) * c.slots;
    T* dst = y + (int64_t)(g.at + g.t) * row + e * 8;
    if (g.whole && g.p >= 0) {
      unsigned code[8];
      if (keys) {
        const unsigned char* src = c.kc + (at + g.slot) * (HD / 2) + u * 4;
#pragma unroll
        for (int i = 0; i < 8; ++i) code[i] = *(const unsigned*)(src + i * (HD / 2));
      } else {
        const unsigned char* tile = c.vc + (at + g.slot) * (HD / 2);
        if constexpr (HD <= 128) {
          const uint4 a = *(const uint4*)(tile + u * kPiece), b = *(const uint4*)(tile + u * kPiece + kPlane);
          const unsigned w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
          pieces_to_eight<HD>(w, code);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) code[i] = get_value<HD>(tile, i, u);
        }
      }
      const uint2 b = *(const uint2*)kv4_scale_at<HD>(keys ? c.ks : c.vs, at, g.slot, u / 4);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float f[8];
        kv4_values(code[i], ((i < 4 ? b.x : b.y) >> (8 * (i & 3))) & 255, f);
        store8(dst + i * row, f);
      }
      continue;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (g.t + i < 0 || g.t + i >= g.len) continue;
      const int slot = (int)((unsigned)(g.slot + i) % (unsigned)cap);
      float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (g.p >= 0)
        kv4_values(keys ? *(const unsigned*)(c.kc + (at + slot) * (HD / 2) + u * 4) : get_value<HD>(c.vc + (at + (slot & ~7)) * (HD / 2), slot & 7, u),
                   *kv4_scale_at<HD>(keys ? c.ks : c.vs, at, slot, u / 4), f);
      store8(dst + i * row, f);
    }
  }
}

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float floatx4_t __attribute__((ext_vector_type(4)));
typedef unsigned u32x2_t __attribute__((ext_vector_type(2)));
typedef unsigned u32x4_t __attribute__((ext_vector_type(4)));

// capA * tanh(x / softcap) of scale * s = x (fp32) or 2 log2(e) x (bf16: 1 - 2 / (exp(2x) + 1) on the hardware's exp and reciprocal, which is off by
// up to 2^-21 of capA, where the bf16 queries' own rounding moves a score by 2^-9 of itself; fstu_wide_cap where capA is so large that this would show)
template <typename T>
__device__ __forceinline__ float cap_scale(float softcap) { return (sizeof(T) == 2 ? 2.0f * 1.4426950408889634f : 1.0f) / softcap; }
template <typename T>
__device__ __forceinline__ void cap_scores(float (&s)[8], float scale, float capA) {
  if (sizeof(T) == 2) {
    if (capA <= FSTU_FAST_CAP * 1.4426950408889634f) {
#pragma unroll
      for (int j = 0; j < 8; ++j) s[j] = fmaf(-2.0f * capA, __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(s[j] * scale) + 1.0f), capA);
    } else {
      asm volatile("");
#pragma unroll
      for (int j = 0; j < 8; ++j) s[j] = fstu_wide_cap(s[j], scale, capA);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j] *= scale;
    fstu_tanh(s);
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j] *= capA;
  }
}

#define KV4_MOST_PARTS 64  // more: workgroups that all keys are dealt to
#define KV4_COLS 8        // query heads of a key head that a workgroup takes

template <bool STREAM, typename V>
__device__ __forceinline__ V load_from(const void* p) {
  if constexpr (STREAM) return __builtin_nontemporal_load((const V*)p);
  return *(const V*)p;
}
template <int N, bool STREAM>
__device__ __forceinline__ void load_words(unsigned* w, const unsigned char* p) {
  if constexpr (N == 1) w[0] = load_from<STREAM, unsigned>(p);
  else if constexpr (N == 2) { const u32x2_t v = load_from<STREAM, u32x2_t>(p); w[0] = v[0]; w[1] = v[1]; }
  else {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const u32x4_t v = load_from<STREAM, u32x4_t>(p + 16 * i);
#pragma unroll
      for (int e = 0; e < 4; ++e) w[4 * i + e] = v[e];
    }
  }
}
template <int SEL>
__device__ __forceinline__ unsigned two_values(unsigned word, float scale) {
  return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, SEL));
}
__device__ __forceinline__ bf16x8_t eight_values(unsigned word, float scale) {
  return __builtin_bit_cast(bf16x8_t, u32x4_t{two_values<0>(word, scale), two_values<1>(word, scale), two_values<2>(word, scale), two_values<3>(word, scale)});
}
// A scale for the conversions above, byte J of eight: they look at the exponent's bits of it and at nothing beside them, so that one shift does.
template <int J>
__device__ __forceinline__ float scale_of(u32x2_t bytes) {
  const unsigned w = bytes[J / 4];
  return __uint_as_float((J & 3) < 3 ? w << (23 - 8 * (J & 3)) : w >> 1);
}
template <int HD>      // dims 2b, 2b + 1 of a piece of hd/16 at slot j
__device__ __forceinline__ unsigned piece_pair(const unsigned* w, float scale, int j, int b) {
  const int byte = j * (HD / 32) + b;
  const unsigned word = w[byte >> 2];
  switch (byte & 3) {
    case 0: return two_values<0>(word, scale);
    case 1: return two_values<1>(word, scale);
    case 2: return two_values<2>(word, scale);
    default: return two_values<3>(word, scale);
  }
}

// What a lane reads of 32 slots: its keys' codes (two tiles of 16 keys) with their scales' bytes, its values' codes with theirs.
template <int HD>
struct Kv4Tile {
  static constexpr int KW = HD / 32, VW = HD / 16, KN = HD == 256 ? 2 : 1;
  unsigned k[2][KW], v[VW];
  u32x2_t ks[KN], vs;
  // STREAM: codes past the caches, which a ring of more than they hold would only push other data out of
  template <bool STREAM>
  __device__ __forceinline__ void load(const Kv4& c, int64_t slot0, int g, int col) {
    const unsigned char* kt = c.kc + slot0 * (HD / 2);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const unsigned at = (8 * (col >> 2) + 4 * t + (col & 3)) * (HD / 2) + g * (HD / 8 / KN);
#pragma unroll
      for (int n = 0; n < KN; ++n) load_words<KW / KN, STREAM>(k[t] + n * (KW / KN), kt + at + n * (HD / 4));
    }
    const unsigned char *kst = c.ks + slot0 * (HD / 32), *vst = c.vs + slot0 * (HD / 32);
#pragma unroll
    for (int n = 0; n < KN; ++n) ks[n] = *(const u32x2_t*)(kst + (col >> 2) * (HD / 4) + (g * (HD / KN) / 128 + 4 * n) * 8);
    const unsigned char* vt = c.vc + slot0 * (HD / 2) + g * (4 * HD);
    if constexpr (HD <= 64) load_words<VW, STREAM>(v, vt + col * (HD / 4));
    else {
#pragma unroll
      for (int n = 0; n < VW / 4; ++n) load_words<4, STREAM>(v + 4 * n, vt + n * 256 + col * 16);
    }
    vs = *(const u32x2_t*)(vst + g * (HD / 4) + (col * HD / 512) * 8);
  }
};

// The tiles of 32 slots that the query of a sequence at position p looks at: `count` of them from `start` on, around the ring's end.
struct Tiles {
  int slot, lim, start, count;       // the query's own slot, how far behind it the last key is
};
__device__ __forceinline__ Tiles tiles_of(int p, int cap, int window, int tiles) {
  Tiles t;
  t.slot = p < 0 ? 0 : p % cap;
  t.lim = p < 0 ? -1 : min(window, p);
  const int lo = t.slot - t.lim;
  t.start = (lo < 0 ? lo + cap : lo) / KV4_TILE;
  t.count = p < 0 ? 0 : lo < 0 ? min(tiles, tiles - t.start + t.slot / KV4_TILE + 1) : t.slot / KV4_TILE - t.start + 1;
  return t;
}

struct NewRows {               // the keys and values of the queries' own positions, or nothing: strides in elements
  const void *k, *v;
  int64_t k_row, k_head, v_row, v_head;
  int dtype;
};

// All sequences' tiles behind one another, `per_seq` groups (key heads, chunks of query heads) each: workgroup w of W takes per or per + 1 of them.
struct Plan {
  int total, per, more;
  __device__ __forceinline__ int begin(int w) const { return w * per + min(w, more); }
  __device__ __forceinline__ int owner(int x) const { return x < more * (per + 1) ? x / (per + 1) : more + (x - more * (per + 1)) / per; }
};
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_int(int v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false); }      // zero where there is no such lane
__device__ __forceinline__ int wave_prefix(int v) {          // inclusive: inside rows of 16 lanes, then their last lanes onto the rows behind
  v += dpp_int<0x111, 0xf>(v);
  v += dpp_int<0x112, 0xf>(v);
  v += dpp_int<0x114, 0xf>(v);
  v += dpp_int<0x118, 0xf>(v);
  v += dpp_int<0x142, 0xa>(v);
  return v + dpp_int<0x143, 0xc>(v);
}
__device__ __forceinline__ int tiles_behind(const int* pos, int seqs, int at, int cap, int window, int tiles) {      // of the lane's sequence
  const int b = at + ((int)threadIdx.x & 63);
  return b < seqs ? tiles_of(pos[b], cap, window, tiles).count : 0;
}
__device__ __forceinline__ Plan plan_of(const int* pos, int seqs, int cap, int window, int tiles, int per_seq, int W) {
  int n = 0;
  for (int at = 0; at < seqs; at += 64) n += __builtin_amdgcn_readlane(wave_prefix(tiles_behind(pos, seqs, at, cap, window, tiles)), 63);
  Plan p;
  p.total = n * per_seq;
  p.per = p.total / W;
  p.more = p.total - p.per * W;
  return p;
}
// The sequence whose tiles hold tile x (x < total), and where they begin.
__device__ __forceinline__ int sequence_of(const int* pos, int seqs, int cap, int window, int tiles, int per_seq, int x, int* begin, int* count) {
  int sum = 0, at = 0;
  for (;;) {
    const int n = tiles_behind(pos, seqs, at, cap, window, tiles), end = wave_prefix(n), all = __builtin_amdgcn_readlane(end, 63);
    if (x < (sum + all) * per_seq || at + 64 >= seqs) {
      const unsigned long long yes = __ballot((sum + end - n) * per_seq <= x && at + ((int)threadIdx.x & 63) < seqs);
      const int i = 63 - __builtin_clzll(yes | 1);
      *count = __builtin_amdgcn_readlane(n, i);
      *begin = (sum + __builtin_amdgcn_readlane(end - n, i)) * per_seq;
      return at + i;
    }
    sum += all;
    at += 64;
  }
}

// One query a sequence.  S^T = K Q^T over 32 slots at a time as two tiles of 16 keys, rows dealt so that lane (g, col) ends up with query col's scores of slots
// 8 g .. 8 g + 7, which is what it holds of the second product O^T = V^T P^T: no score crosses a lane, only the maxima do.  Codes become bf16 in registers (exact),
// probabilities go in as a bf16 head and, in the columns 8 further on, what its rounding left.  fp32: queries and probabilities in three such parts, 24 bits of them,
// since codes widen to bf16 at once and the fp32 instruction would take them at a sixteenth of the rate; in 2-norm 2.4e-7 to 8e-7 off (plain fp32 1.8e-7 to 1.7e-6,
// the more the longer the ring).
// PLAN: the tiles of all sequences are dealt evenly to the workgroups; without, a workgroup takes a key head of a sequence or one of gridDim.z parts of its tiles.
// kv4_join_kernel adds up what is in parts.
// Bytes bound it where there are many: 16 sequences of up to 32768 positions, 8 key heads of 128, 84 us, 5.5 TB/s (an instruction undoes two codes and applies
// their scale, a fourth of the vector ALUs' time; a look-up and a product for each would be more than memory takes), 32 of 1025 positions and 16 heads of 128
// 17 us, of which 4 are the launch and the first trip.  12 heads of 64 over 513 positions 6 us: the launch, the trip for the position, the trip for the codes,
// the join through LDS.
template <typename T, int HD, int NW, bool CAP, bool PLAN>
__global__ void __launch_bounds__(NW * 64, HD == 256 || NW == 8 ? 1 : HD == 128 ? 2 : 3)
kv4_attend_kernel(const T* q, int64_t q_row, int64_t q_head, const void* cache, T* out, float* ws, const int* pos, const float* slopes, int seqs, int heads,
                  int kvh, int cap, int window, float softcap, int chunks, NewRows fresh) {
  constexpr int KS = HD / 32, NV = HD / 16, QP = sizeof(T) == 2 ? 1 : 3;     // steps of a score's product, tiles of dims, bf16 parts of a query
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
  const int group = heads / kvh, per_seq = kvh * chunks;
  const Kv4 c = kv4_at((void*)cache, (int64_t)seqs * kvh, HD, cap);
  const int tiles = c.slots / KV4_TILE;
  const float kLog2e = 1.4426950408889634f, capA = softcap * kLog2e;
  const float scale = rsqrtf((float)HD) * (CAP ? cap_scale<T>(softcap) : kLog2e);
  const unsigned low_part = col < 8 ? 0u : 0xffffffffu;
  const unsigned turn = (8 * (col & 3) + 9) & 31;                // turns byte col & 3 to where a float has its exponent
  extern __shared__ float sm[];                                  // (NW, cols) maxima, sums, then (NW, cols, HD)
  float* const sl = sm + NW * KV4_COLS;
  float* const so = sl + NW * KV4_COLS;

  Plan plan;
  int x = 0, x_end = 1;
  if (PLAN) {
    plan = plan_of(pos, seqs, cap, window, tiles, per_seq, gridDim.x);
    x = plan.begin(blockIdx.x);
    x_end = plan.begin(blockIdx.x + 1);
  }
  while (x < x_end) {                                            // a stretch of one key head's tiles
    int b, y, first = 0, last, all;
    if (PLAN) {
      int begin;
      b = sequence_of(pos, seqs, cap, window, tiles, per_seq, x, &begin, &all);
      all = max(all, 1);                                         // (whatever becomes of pos meanwhile: an end, and no head that is not there)
      y = min(max((x - begin) / all, 0), per_seq - 1);
      first = max(x - begin - y * all, 0);
      last = min(all, first + x_end - x);
      x += max(last - first, 1);
    } else {
      b = blockIdx.y;
      y = blockIdx.x;
      x = x_end;
    }
    const Tiles tl = tiles_of(pos[b], cap, window, tiles);
    const int ps = tl.slot, lim = tl.lim, start = tl.start;
    const int parts = PLAN ? 1 : gridDim.z, part_no = PLAN ? 0 : blockIdx.z;
    if (!PLAN) {
      all = tl.count;
      const int per = all / parts, more = all - per * parts;     // the first `more` parts take one tile more
      first = per * part_no + min(part_no, more);
      last = first + per + (part_no < more ? 1 : 0);
    }
    const int hk = y / chunks, h0 = hk * group + y % chunks * KV4_COLS, cols = min(KV4_COLS, hk * group + group - h0);
    const int64_t head0 = ((int64_t)b * kvh + hk) * c.slots;
    if (!PLAN && fresh.k) {
      // this position's key and value first: each workgroup of the head leaves the same bytes, and reads what itself has left
      if (w < 2 && lane < HD / 8) {
        float f[8];
        unsigned byte;
        load8(w == 0 ? (const T*)fresh.k + b * fresh.k_row + hk * fresh.k_head + lane * 8 : (const T*)fresh.v + b * fresh.v_row + hk * fresh.v_head + lane * 8, f);
        const unsigned code = kv4_quantise(f, &byte);
        if (lim >= 0) {
          if (w == 0) *(unsigned*)(c.kc + (head0 + ps) * (HD / 2) + lane * 4) = code;
          else put_value<HD>(c.vc + (head0 + (ps & ~7)) * (HD / 2), ps & 7, lane, code);
          if ((lane & 3) == 0) *kv4_scale_at<HD>(w == 0 ? c.ks : c.vs, head0, ps, lane / 4) = (unsigned char)byte;
        }
      }
      __syncthreads();
    }

    // queries: column col and col + 8 are the same head
    const int h = h0 + min(col & 7, cols - 1);
    bf16x8_t qf[KS][QP];
    {
      const T* qr = q + b * q_row + h * q_head;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        float f[8];
        load8(qr + (HD == 256 ? (k >> 2) * 128 + g * 32 + (k & 3) * 8 : g * (HD / 4) + k * 8), f);
#pragma unroll
        for (int e = 0; e < QP; ++e) {
          u32x4_t part;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            part[i] = pack2_bf16(f[2 * i], f[2 * i + 1]);
            f[2 * i] -= __uint_as_float(part[i] << 16);
            f[2 * i + 1] -= __uint_as_float(part[i] & 0xffff0000u);
          }
          qf[k][e] = __builtin_bit_cast(bf16x8_t, part);
        }
      }
    }
    const float slope = slopes ? slopes[h] * kLog2e : 0.f;
    float m = -INFINITY, l = 0.f;
    floatx4_t o[NV];
#pragma unroll
    for (int t = 0; t < NV; ++t) o[t] = floatx4_t{0.f, 0.f, 0.f, 0.f};
    auto tile_at = [&](int i) { const int t = start + i; return t >= tiles ? t - tiles : t; };
    auto take = [&](const Kv4Tile<HD>& now, int i) {
      const int t0 = tile_at(i) * KV4_TILE;
      float s[8];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        floatx4_t d = {0.f, 0.f, 0.f, 0.f};
        float f[Kv4Tile<HD>::KN];
#pragma unroll
        for (int e = 0; e < Kv4Tile<HD>::KN; ++e) f[e] = __uint_as_float(__builtin_amdgcn_alignbit(now.ks[e][t], now.ks[e][t], turn));
#pragma unroll
        for (int x = 0; x < KS; ++x) {
          const bf16x8_t kf = eight_values(now.k[t][x], f[HD == 256 ? x >> 2 : 0]);
#pragma unroll
          for (int e = 0; e < QP; ++e) d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[x][e], d, 0, 0, 0);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) s[4 * t + r] = d[r];
      }
      // slot t0 + 8 g + j is score j of this lane
      const int far0 = t0 <= ps ? ps - t0 : ps + cap - t0;
      const bool whole = __builtin_amdgcn_readfirstlane(t0 + KV4_TILE <= cap && far0 <= lim && (t0 + KV4_TILE - 1 <= ps || t0 > ps)) != 0;      // wave-uniform
      const float tb = whole ? -slope * (float)(far0 - 8 * g) : 0.f;
      float vs[8] = {scale_of<0>(now.vs), scale_of<1>(now.vs), scale_of<2>(now.vs), scale_of<3>(now.vs),
                     scale_of<4>(now.vs), scale_of<5>(now.vs), scale_of<6>(now.vs), scale_of<7>(now.vs)};
      float top = -INFINITY;
      if (CAP) cap_scores<T>(s, scale, capA);
      if (whole) {
#pragma unroll
        for (int j = 0; j < 8; ++j) s[j] = fmaf(s[j], CAP ? 1.f : scale, slope * (float)j);
      } else {
        asm volatile("");                                          // a branch: most tiles need none of this
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int slot = t0 + 8 * g + j, far = slot <= ps ? ps - slot : ps + cap - slot;
          const bool seen = slot < cap && far <= lim;
          s[j] = seen ? fmaf(s[j], CAP ? 1.f : scale, -slope * (float)far) : -INFINITY;
          vs[j] = seen ? vs[j] : 1.f;                              // a scale of NaN times a weight of zero
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) top = fmaxf(top, s[j]);
      top += tb;
      if (__any(top > m)) {
        top = fmaxf(top, fstu_swz16(top));
        top = fmaxf(top, __shfl_xor(top, 32, FSTU_WAVE));
        const float mn = fmaxf(m, top), corr = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
        l *= corr;
#pragma unroll
        for (int t = 0; t < NV; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) o[t][r] *= corr;
        m = mn;
      }
      const float off = tb - (m == -INFINITY ? 0.f : m);
      // probabilities in bf16 parts: the columns of the upper half hold what the lower half's rounding left
      u32x4_t pf, pf2;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float a = __builtin_amdgcn_exp2f(s[2 * e] + off), z = __builtin_amdgcn_exp2f(s[2 * e + 1] + off);
        l += a + z;
        const unsigned head = pack2_bf16(a, z) & low_part;
        a -= __uint_as_float(head << 16);
        z -= __uint_as_float(head & 0xffff0000u);
        pf[e] = pack2_bf16(a, z);
        if (QP == 3) {                                             // and, for fp32, a third part beside the second
          a -= __uint_as_float(pf[e] << 16);
          z -= __uint_as_float(pf[e] & 0xffff0000u);
          pf2[e] = pack2_bf16(a, z) & low_part;
        }
      }
#pragma unroll
      for (int t = 0; t < NV / 2; ++t) {
        u32x4_t low, high;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const unsigned a = piece_pair<HD>(now.v, vs[2 * e], 2 * e, t), z = piece_pair<HD>(now.v, vs[2 * e + 1], 2 * e + 1, t);
          low[e] = __builtin_amdgcn_perm(z, a, 0x05040100);
          high[e] = __builtin_amdgcn_perm(z, a, 0x07060302);
        }
        o[2 * t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, low), __builtin_bit_cast(bf16x8_t, pf), o[2 * t], 0, 0, 0);
        o[2 * t + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, high), __builtin_bit_cast(bf16x8_t, pf), o[2 * t + 1], 0, 0, 0);
        if (QP == 3) {
          o[2 * t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, low), __builtin_bit_cast(bf16x8_t, pf2), o[2 * t], 0, 0, 0);
          o[2 * t + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, high), __builtin_bit_cast(bf16x8_t, pf2), o[2 * t + 1], 0, 0, 0);
        }
      }
    };
    // AHEAD tiles on their way at any time, each asked for without a branch (behind the last one the last again), so that a wait is for one tile and not for all
    constexpr int AHEAD = 2;
    Kv4Tile<HD> ring[AHEAD];
    int i = first + w;
    if (i < last) {
      const int end = i + (last - 1 - i) / NW * NW;
      auto ask = [&](Kv4Tile<HD>& t, int n) {
        t.template load<PLAN>(c, head0 + (int64_t)tile_at(min(n, end)) * KV4_TILE, g, col);
        __builtin_amdgcn_sched_barrier(0);
      };
#pragma unroll
      for (int a = 0; a < AHEAD; ++a) ask(ring[a], i + a * NW);
      for (bool more = true; more;) {
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
          take(ring[a], i);
          i += NW;
          if (i > end) { more = false; break; }
          ask(ring[a], i + (AHEAD - 1) * NW);
        }
      }
    }
    l += fstu_swz16(l);
    l += __shfl_xor(l, 32, FSTU_WAVE);
#pragma unroll
    for (int t = 0; t < NV; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) o[t][r] += fstu_dpp<0x128>(o[t][r]);       // row_ror:8: the other part's column
    if (col < cols) {
      if (g == 0) { sm[w * KV4_COLS + col] = m; sl[w * KV4_COLS + col] = l; }
      float* dst = so + (w * cols + col) * HD + 4 * g * NV;      // dim (4 g + r) * NV + t
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int t = 0; t < NV; ++t) dst[r * NV + t] = o[t][r];
    }
    __syncthreads();
    for (int e = threadIdx.x; e < cols * HD; e += NW * 64) {
      const int cc = e / HD, d = e % HD;
      float M = -INFINITY, L = 0.f, v = 0.f;
#pragma unroll
      for (int k = 0; k < NW; ++k) M = fmaxf(M, sm[k * KV4_COLS + cc]);
#pragma unroll
      for (int k = 0; k < NW; ++k) {
        const float f = sm[k * KV4_COLS + cc] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(sm[k * KV4_COLS + cc] - M);
        L = fmaf(sl[k * KV4_COLS + cc], f, L);
        v = fmaf(so[(k * cols + cc) * HD + d], f, v);
      }
      if (PLAN ? last - first == all : parts == 1) DT<T>::st(out + ((int64_t)b * heads + h0 + cc) * HD + d, all ? v / L : 0.f);
      else {
        // PLAN: one place to each pair of workgroup and key head that meet: both rise from one to the next
        const int64_t place = PLAN ? (int64_t)blockIdx.x + b * per_seq + y : ((int64_t)b * per_seq + y) * parts + part_no;
        float* part = ws + (place * KV4_COLS + cc) * (HD + 2);
        part[2 + d] = v;
        if (d == 0) { part[0] = M; part[1] = L; }
      }
    }
    if (PLAN) __syncthreads();
  }
}

// The parts of a query head, in the order of its keys: several to a thread row, joined through LDS.
template <typename T, int HD>
__global__ void __launch_bounds__(512)
kv4_join_kernel(const float* ws, T* out, const int* pos, int seqs, int heads, int kvh, int cap, int window, int chunks, int splits) {
  constexpr int R = 512 / HD;
  const int b = blockIdx.x / heads, h = blockIdx.x % heads, group = heads / kvh, hk = h / group, per_seq = kvh * chunks;
  const int y = hk * chunks + (h - hk * group) / KV4_COLS, cc = (h - hk * group) % KV4_COLS, d = threadIdx.x % HD, r = threadIdx.x / HD;
  const int tiles = kv4_slots(cap) / KV4_TILE, count = tiles_of(pos[b], cap, window, tiles).count;
  T* const dst = out + (int64_t)blockIdx.x * HD + d;
  if (count == 0) {
    if (r == 0) DT<T>::st(dst, 0.f);
    return;
  }
  int n = splits;
  int64_t place = ((int64_t)b * per_seq + y) * splits;
  if (splits > KV4_MOST_PARTS) {
    const Plan plan = plan_of(pos, seqs, cap, window, tiles, per_seq, splits);
    int before = 0;
    for (int at = 0; at < b; at += 64) before += __builtin_amdgcn_readlane(wave_prefix(tiles_behind(pos, b, at, cap, window, tiles)), 63);
    const int begin = min(before * per_seq + y * count, plan.total - 1), w0 = plan.owner(begin), w1 = min(plan.owner(begin + count - 1), splits - 1);
    if (w0 == w1) return;                                        // whole, and there already
    n = w1 - w0 + 1;
    place = (int64_t)w0 + b * per_seq + y;
  }
  const float* part = ws + (place * KV4_COLS + cc) * (HD + 2);
  constexpr int STEP = KV4_COLS * (HD + 2);
  float M = -INFINITY, L = 0.f, v = 0.f;
#pragma unroll 4
  for (int s = r; s < n; s += R) {
    const float m = part[(int64_t)s * STEP], l = part[(int64_t)s * STEP + 1], o = part[(int64_t)s * STEP + 2 + d];
    const float top = fmaxf(M, m), f = M == top ? 1.f : __builtin_amdgcn_exp2f(M - top), e = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);
    L = fmaf(L, f, l * e);
    v = fmaf(v, f, o * e);
    M = top;
  }
  __shared__ float sm[R], sl[R], so[R][HD];
  if (d == 0) { sm[r] = M; sl[r] = L; }
  so[r][d] = v;
  __syncthreads();
  if (r) return;
  M = -INFINITY;
  for (int s = 0; s < R; ++s) M = fmaxf(M, sm[s]);
  L = v = 0.f;
  for (int s = 0; s < R; ++s) {
    const float e = sm[s] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(sm[s] - M);
    const float ls = sl[s], os = so[s][d];
    L = fmaf(ls, e, L);
    v = fmaf(os, e, v);
  }
  DT<T>::st(dst, v / L);
}

int kv4_check(const char* name, const void* cache, int seqs, int kvh, int hd, int cap) {
  FSTU_REQUIRE(cache, FSTU_ENULL, "%s: null pointer", name);
  FSTU_REQUIRE(hd == 32 || hd == 64 || hd == 128 || hd == 256, FSTU_ESHAPE, "%s: head dim %d not in {32,64,128,256}", name, hd);
  FSTU_REQUIRE(seqs >= 1 && kvh >= 1 && cap >= 1 && cap <= (1 << 30) && (int64_t)seqs * kvh <= 0x7fffffff, FSTU_ESHAPE,
               "%s: bad shape sequences=%d key heads=%d capacity=%d", name, seqs, kvh, cap);
  FSTU_REQUIRE(fstu_aligned(cache, 16), FSTU_EALIGN, "%s: the cache must be 16-byte aligned", name);
  return FSTU_OK;
}

#define KV4_DISPATCH(dtype, hd, name, BODY)                                                                                     \
  do {                                                                                                                          \
    FSTU_REQUIRE(dtype == FSTU_F32 || dtype == FSTU_BF16, FSTU_EDTYPE, "%s: unknown dtype %d", name, dtype);                    \
    auto go = [&](auto t, auto w) { using T = decltype(t); constexpr int HD = decltype(w)::value; BODY; };                      \
    auto by_width = [&](auto t) {                                                                                               \
      if (hd == 32) go(t, std::integral_constant<int, 32>{});                                                                   \
      else if (hd == 64) go(t, std::integral_constant<int, 64>{});                                                              \
      else if (hd == 128) go(t, std::integral_constant<int, 128>{});                                                            \
      else go(t, std::integral_constant<int, 256>{});                                                                           \
    };                                                                                                                          \
    if (dtype == FSTU_F32) by_width(float{}); else by_width(bf16_t{});                                                          \
  } while (0)

// Whole waves over the dims of a row's heads, up to 256 threads.
int kv4_threads(int kvh, int hd) {
  const int64_t n = (int64_t)kvh * (hd / 8);
  return n > 192 ? 256 : (int)((n + 63) / 64 * 64);
}

}  // namespace

extern "C" int64_t fstu_kv4_bytes(int seqs, int kvh, int hd, int cap) {
  return (int64_t)seqs * kvh * kv4_slots(cap) * (hd + hd / 16);
}

extern "C" int fstu_kv4_write(const void* k, int64_t k_row, int64_t k_head, const void* v, int64_t v_row, int64_t v_head, void* cache, const int* pos,
                              const int* cu, int rows, int seqs, int kvh, int hd, int cap, int dtype, void* stream) {
  const int rc = kv4_check("fstu_kv4_write", cache, seqs, kvh, hd, cap);
  if (rc) return rc;
  FSTU_REQUIRE(k && v && pos, FSTU_ENULL, "fstu_kv4_write: null pointer");
  FSTU_REQUIRE(rows >= 0 && (cu || rows == seqs), FSTU_EARG, "fstu_kv4_write: %d rows for %d sequences", rows, seqs);
  const int size = dtype == FSTU_BF16 ? 2 : 4;
  FSTU_REQUIRE(fstu_heads_aligned(k, k_row, k_head, size) && fstu_heads_aligned(v, v_row, v_head, size), FSTU_EALIGN,
               "fstu_kv4_write: rows and heads of k and v must begin at multiples of 16 bytes");
  const int64_t groups = cu ? (int64_t)rows / 8 + 2 * (int64_t)seqs : rows;
  FSTU_REQUIRE(groups < 1 << 23, FSTU_ESHAPE, "fstu_kv4_write: %d rows of %d sequences are more than a launch takes", rows, seqs);
  if (rows == 0) return FSTU_OK;
  const int threads = kv4_threads(kvh, hd);
  KV4_DISPATCH(dtype, hd, "fstu_kv4_write", {
    auto run = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3((unsigned)groups, 2), dim3(threads), 0, (hipStream_t)stream, (const T*)k, (const T*)v, k_row, k_head, v_row, v_head, cache,
                         pos, cu, rows, seqs, kvh, cap);
    };
    cu ? run(kv4_write_kernel<T, HD, false>) : run(kv4_write_kernel<T, HD, true>);
  });
  FSTU_CHECK_LAUNCH("fstu_kv4_write");
  return FSTU_OK;
}

extern "C" int fstu_kv4_read(const void* cache, void* k, void* v, const int* pos, const int* cu, int rows, int seqs, int kvh, int hd, int cap, int dtype,
                             void* stream) {
  const int rc = kv4_check("fstu_kv4_read", cache, seqs, kvh, hd, cap);
  if (rc) return rc;
  FSTU_REQUIRE(k && v && pos, FSTU_ENULL, "fstu_kv4_read: null pointer");
  FSTU_REQUIRE(rows >= 0 && (cu || rows == seqs), FSTU_EARG, "fstu_kv4_read: %d rows for %d sequences", rows, seqs);
  FSTU_REQUIRE(fstu_aligned(k, 16) && fstu_aligned(v, 16), FSTU_EALIGN, "fstu_kv4_read: k and v must be 16-byte aligned");
  const int64_t groups = cu ? (int64_t)rows / 8 + 2 * (int64_t)seqs : rows;
  FSTU_REQUIRE(groups < 1 << 23, FSTU_ESHAPE, "fstu_kv4_read: %d rows of %d sequences are more than a launch takes", rows, seqs);
  if (rows == 0) return FSTU_OK;
  const int threads = kv4_threads(kvh, hd);
  KV4_DISPATCH(dtype, hd, "fstu_kv4_read", {
    auto run = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3((unsigned)groups, 2), dim3(threads), 0, (hipStream_t)stream, cache, (T*)k, (T*)v, pos, cu, rows, seqs, kvh, cap);
    };
    cu ? run(kv4_read_kernel<T, HD, false>) : run(kv4_read_kernel<T, HD, true>);
  });
  FSTU_CHECK_LAUNCH("fstu_kv4_read");
  return FSTU_OK;
}

// How a call's keys are cut: 1: a workgroup to each key head of a sequence; up to 64: that many parts of each; more: that many workgroups, to which all keys are
// dealt evenly.  Parts cost a second launch and its boundary, some 3 us, and pay where few heads leave compute units idle through more than a thousand positions;
// dealing evenly costs two looks at all positions besides, and pays where there is so much to do that an uneven end is more.  us, a workgroup to a head / parts (how
// many) / dealt to 256: 16 heads of 128 over 1025 positions 9.1 / 7.5 (16) / -, 700 7.9 / 7.4 (16), 2048 12.5 / 7.8 (16) / 9.9; 12 heads of 64 over 2048 9.9 /
// 7.6 (16) / 11.0; 4 of 128 over 32768 138 / 12.9 (64) / 14.9; 32 of 128 over 4200 23.8 / 11.8 (8) / 17.8; 8 of 256 over 700 12.7 / 8.8 (16); sequences of
// uneven length, 128 heads of 128: 8192 39 / 27 (2) / 31, 32768 155 / 106 (2) / 88; 512 of 128 over 4096 49 / - / 52.
// The even deal counts a call's tiles in an int: each sequence's window's, and one more where the ring's end cuts it.
static bool kv4_can_deal(int seqs, int heads, int kvh, int cap, int window) {
  const int64_t tiles = ((int64_t)(window < cap ? window : cap - 1) + 3 * KV4_TILE - 1) / KV4_TILE;
  return tiles * seqs * kvh * ((heads / kvh + KV4_COLS - 1) / KV4_COLS) <= 0x7fffffff;
}
extern "C" int fstu_kv4_attend_splits(int seqs, int heads, int kvh, int hd, int cap, int window) {
  if (seqs < 1 || kvh < 1 || heads < kvh || cap < 1 || window < 0) return 1;
  const int chunks = (heads / kvh + KV4_COLS - 1) / KV4_COLS;
  const int64_t tiles = ((int64_t)(window < cap ? window : cap - 1) + 2 * KV4_TILE - 1) / KV4_TILE, groups = (int64_t)seqs * kvh * chunks;
  if (groups * tiles >= 98304 && tiles >= 192 && kv4_can_deal(seqs, heads, kvh, cap, window)) return 256;
  int64_t parts = 256 / groups;
  if (parts > tiles / 3) parts = tiles / 3;
  return tiles < (hd == 256 ? 20 : 40) || parts < 2 ? 1 : (int)(parts < KV4_MOST_PARTS ? parts : KV4_MOST_PARTS);
}
extern "C" int64_t fstu_kv4_attend_ws(int seqs, int heads, int kvh, int hd, int splits) {
  if (seqs < 1 || kvh < 1 || heads < kvh || splits <= 1) return 0;
  const int64_t groups = (int64_t)seqs * kvh * ((heads / kvh + KV4_COLS - 1) / KV4_COLS);
  return (splits > KV4_MOST_PARTS ? groups + splits : groups * splits) * KV4_COLS * (hd + 2);
}

static int kv4_attend_call(const char* name, const void* q, int64_t q_row, int64_t q_head, NewRows fresh, void* cache, void* out, float* ws, int splits,
                           const int* pos, const float* slopes, int seqs, int heads, int kvh, int hd, int cap, int window, float softcap, int dtype, void* stream) {
  const int rc = kv4_check(name, cache, seqs, kvh, hd, cap);
  if (rc) return rc;
  FSTU_REQUIRE(q && out && pos, FSTU_ENULL, "%s: null pointer", name);
  FSTU_REQUIRE(heads >= 1 && heads % kvh == 0 && heads <= 65535 && seqs <= 65535 && (int64_t)seqs * heads <= 0x7fffffff, FSTU_ESHAPE, "%s: %d heads over %d key heads, %d sequences", name,
               heads, kvh, seqs);
  FSTU_REQUIRE(window >= 0 && window < cap, FSTU_EARG, "%s: window %d with a capacity of %d", name, window, cap);
  FSTU_REQUIRE(fstu_softcap_ok(softcap), FSTU_EARG, "%s: softcap must be zero (none) or a number from 2^-40 to 2^40", name);
  FSTU_REQUIRE(splits >= 1 && splits <= 65535 && (splits == 1 || ws), FSTU_EARG, "%s: %d splits need their workspace", name, splits);
  const int size = dtype == FSTU_BF16 ? 2 : 4;
  FSTU_REQUIRE(fstu_heads_aligned(q, q_row, q_head, size) && fstu_aligned(out, 16) && fstu_aligned(ws, 4), FSTU_EALIGN,
               "%s: rows and heads of q and out must begin at multiples of 16 bytes", name);
  FSTU_REQUIRE(dtype == FSTU_F32 || dtype == FSTU_BF16, FSTU_EDTYPE, "%s: unknown dtype %d", name, dtype);
  const int64_t n = (int64_t)seqs * heads * hd * size;
  FSTU_REQUIRE(!fstu_heads_touch(q, q_row, q_head, seqs, heads, hd, size, out, n) &&
                   !fstu_heads_touch(cache, fstu_kv4_bytes(seqs, kvh, hd, cap), 0, 2, 1, 0, 1, out, n),
               FSTU_EARG, "%s: out overlaps q or the cache", name);
  const int group = heads / kvh, chunks = (group + KV4_COLS - 1) / KV4_COLS;
  FSTU_REQUIRE((int64_t)seqs * heads < 1 << 23 &&
                   (splits > KV4_MOST_PARTS ? kv4_can_deal(seqs, heads, kvh, cap, window) : (int64_t)seqs * kvh * chunks * splits < 1 << 23), FSTU_ESHAPE,
               "%s: %d sequences of %d heads in %d parts are more than a launch takes", name, seqs, heads, splits);
  if (fresh.k) {
    FSTU_REQUIRE(fresh.dtype == FSTU_F32 || fresh.dtype == FSTU_BF16, FSTU_EDTYPE, "%s: unknown dtype %d of k and v", name, fresh.dtype);
    const int wide = fresh.dtype == FSTU_BF16 ? 2 : 4;
    FSTU_REQUIRE(fstu_heads_aligned(fresh.k, fresh.k_row, fresh.k_head, wide) && fstu_heads_aligned(fresh.v, fresh.v_row, fresh.v_head, wide), FSTU_EALIGN,
                 "%s: rows and heads of k and v must begin at multiples of 16 bytes", name);
    const int64_t held = fstu_kv4_bytes(seqs, kvh, hd, cap);
    FSTU_REQUIRE(!fstu_heads_touch(fresh.k, fresh.k_row, fresh.k_head, seqs, kvh, hd, wide, out, n) &&
                     !fstu_heads_touch(fresh.v, fresh.v_row, fresh.v_head, seqs, kvh, hd, wide, out, n) &&
                     !fstu_heads_touch(fresh.k, fresh.k_row, fresh.k_head, seqs, kvh, hd, wide, cache, held) &&
                     !fstu_heads_touch(fresh.v, fresh.v_row, fresh.v_head, seqs, kvh, hd, wide, cache, held),
                 FSTU_EARG, "%s: out or the cache overlaps k or v", name);
    // written by a launch of its own, once nothing is left to refuse: where keys are dealt evenly (a call that long does not feel a launch), or of another type
    if (splits > KV4_MOST_PARTS || fresh.dtype != dtype) {
      const int wrote = fstu_kv4_write(fresh.k, fresh.k_row, fresh.k_head, fresh.v, fresh.v_row, fresh.v_head, cache, pos, nullptr, seqs, seqs, kvh, hd, cap, fresh.dtype,
                                       stream);
      if (wrote) return wrote;
      fresh.k = nullptr;
    }
  }
  KV4_DISPATCH(dtype, hd, name, {
    auto run = [&](auto kernel, dim3 grid, int waves) {
      const unsigned lds = waves * (2 * KV4_COLS + (group < KV4_COLS ? group : KV4_COLS) * HD) * sizeof(float);
      hipLaunchKernelGGL(kernel, grid, dim3(waves * 64), lds, (hipStream_t)stream, (const T*)q, q_row, q_head, cache, (T*)out, ws, pos, slopes, seqs, heads, kvh,
                         cap, window, softcap, chunks, fresh);
    };
    constexpr int WIDE = HD == 256 ? 4 : 8;
    const dim3 grid(kvh * chunks, seqs, splits);
    if (splits > KV4_MOST_PARTS)
      softcap > 0.f ? run(kv4_attend_kernel<T, HD, WIDE, true, true>, dim3(splits), WIDE) : run(kv4_attend_kernel<T, HD, WIDE, false, true>, dim3(splits), WIDE);
    else if ((int64_t)seqs * kvh * chunks * splits <= 256)      // one to a compute unit: eight waves (12 heads of 64 over 513 positions 5.7 us, 6.6 with four)
      softcap > 0.f ? run(kv4_attend_kernel<T, HD, WIDE, true, false>, grid, WIDE) : run(kv4_attend_kernel<T, HD, WIDE, false, false>, grid, WIDE);
    else
      softcap > 0.f ? run(kv4_attend_kernel<T, HD, 4, true, false>, grid, 4) : run(kv4_attend_kernel<T, HD, 4, false, false>, grid, 4);
    if (splits > 1)
      hipLaunchKernelGGL((kv4_join_kernel<T, HD>), dim3(seqs * heads), dim3(512), 0, (hipStream_t)stream, ws, (T*)out, pos, seqs, heads, kvh, cap, window, chunks,
                         splits);
  });
  FSTU_CHECK_LAUNCH(name);
  return FSTU_OK;
}

extern "C" int fstu_kv4_attend(const void* q, int64_t q_row, int64_t q_head, const void* cache, void* out, float* ws, int splits, const int* pos,
                               const float* slopes, int seqs, int heads, int kvh, int hd, int cap, int window, float softcap, int dtype, void* stream) {
  return kv4_attend_call("fstu_kv4_attend", q, q_row, q_head, NewRows{}, (void*)cache, out, ws, splits, pos, slopes, seqs, heads, kvh, hd, cap, window, softcap, dtype,
                         stream);
}

extern "C" int fstu_kv4_step_of(const void* q, int64_t q_row, int64_t q_head, int dtype, const void* k, int64_t k_row, int64_t k_head, const void* v, int64_t v_row,
                                int64_t v_head, int kv_dtype, void* cache, void* out, float* ws, int splits, const int* pos, const float* slopes, int seqs, int heads,
                                int kvh, int hd, int cap, int window, float softcap, void* stream) {
  FSTU_REQUIRE(k && v, FSTU_ENULL, "fstu_kv4_step: null pointer");
  return kv4_attend_call("fstu_kv4_step", q, q_row, q_head, NewRows{k, v, k_row, k_head, v_row, v_head, kv_dtype}, cache, out, ws, splits, pos, slopes, seqs, heads,
                         kvh, hd, cap, window, softcap, dtype, stream);
}

// One launch with the write where a workgroup has its head to itself or shares it in parts: a step of one sequence, 12 heads of 64 over 513 positions 5.75 us,
// 7.6 in two and 5.15 without its write; 32 sequences of 16 heads of 128 over 1025 16.4, 18.6 and 15.8; called from Python 9.4, 14.7 and 8.3.
extern "C" int fstu_kv4_step(const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row, int64_t k_head, const void* v, int64_t v_row,
                             int64_t v_head, void* cache, void* out, float* ws, int splits, const int* pos, const float* slopes, int seqs, int heads, int kvh,
                             int hd, int cap, int window, float softcap, int dtype, void* stream) {
  return fstu_kv4_step_of(q, q_row, q_head, dtype, k, k_row, k_head, v, v_row, v_head, dtype, cache, out, ws, splits, pos, slopes, seqs, heads, kvh, hd, cap, window,
                          softcap, stream);
}
