// The 4-bit ring cache: keys and values to codes as they are written, back to values, and the attention of one query a sequence over it.
#include "fstu_common.h"
#include "fstu_kv4.h"

namespace {

typedef float f32x2_t __attribute__((ext_vector_type(2)));

// The scale's byte for a block whose largest size has these bits: the smallest power of two with amax <= 7 * 2^e.  Its codes end at 6
// and steps beside that are 2 wide, so nothing is off by more than 2^e.  -120 <= e <= 125: every code's value is a normal bf16.
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

// Codes of dims 8u .. 8u + 7 of a value at one slot (a word, low nibble first), in the pieces of hd/16 dims that the cache deals them to.
template <int HD>
__device__ __forceinline__ void put_value(unsigned char* tile, int i, int u, unsigned code) {       // slot i of the eight at `tile`
  constexpr int PB = HD / 32;                                  // bytes of a piece
  tile += i * PB;
  if constexpr (PB >= 4) *(unsigned*)(tile + (u * 4 / PB) * 8 * PB + (u * 4) % PB) = code;
  else if constexpr (PB == 2) {
    *(unsigned short*)(tile + (2 * u) * 16) = (unsigned short)code;
    *(unsigned short*)(tile + (2 * u + 1) * 16) = (unsigned short)(code >> 16);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) tile[(4 * u + e) * 8] = (unsigned char)(code >> (8 * e));
  }
}
template <int HD>
__device__ __forceinline__ unsigned get_value(const unsigned char* tile, int i, int u) {
  constexpr int PB = HD / 32;
  tile += i * PB;
  if constexpr (PB >= 4) return *(const unsigned*)(tile + (u * 4 / PB) * 8 * PB + (u * 4) % PB);
  else if constexpr (PB == 2) return *(const unsigned short*)(tile + (2 * u) * 16) | (unsigned)*(const unsigned short*)(tile + (2 * u + 1) * 16) << 16;
  else {
    unsigned code = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) code |= (unsigned)tile[(4 * u + e) * 8] << (8 * e);
    return code;
  }
}
// The same at all eight slots, as the 32 bytes beside each other that they are (hd up to 128): pieces of four, two or one byte a slot.
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
// read back: 134 us with a row's eight dims to a thread, WRITE_US now.
template <typename T, int HD, bool ONE>
__global__ void __launch_bounds__(256)
kv4_write_kernel(const T* k, const T* v, int64_t k_row, int64_t k_head, int64_t v_row, int64_t v_head, void* cache, const int* pos, const int* cu, int rows,
                 int seqs, int kvh, int cap) {
  constexpr int P = HD / 8;
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
          *(uint4*)(tile + u * 32) = make_uint4(w[0], w[1], w[2], w[3]);
          *(uint4*)(tile + u * 32 + 16) = make_uint4(w[4], w[5], w[6], w[7]);
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
  constexpr int P = HD / 8;
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
          const uint4 a = *(const uint4*)(tile + u * 32), b = *(const uint4*)(tile + u * 32 + 16);
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
// up to 2^-21 of capA, where the bf16 queries' own rounding moves a score by 2^-9 of itself)
template <typename T>
__device__ __forceinline__ float cap_scale(float softcap) { return (sizeof(T) == 2 ? 2.0f * 1.4426950408889634f : 1.0f) / softcap; }
template <typename T>
__device__ __forceinline__ float capped(float s, float scale, float capA) {
  if (sizeof(T) == 2) return fmaf(-2.0f * capA, __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(s * scale) + 1.0f), capA);
  return capA * tanhf(s * scale);
}

#define KV4_COLS 8        // query heads of a key head that a workgroup takes

template <int N>
__device__ __forceinline__ void load_words(unsigned* w, const unsigned char* p) {
  if constexpr (N == 1) w[0] = *(const unsigned*)p;
  else if constexpr (N == 2) { const u32x2_t v = *(const u32x2_t*)p; w[0] = v[0]; w[1] = v[1]; }
  else {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const u32x4_t v = ((const u32x4_t*)p)[i];
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
template <int SEL>
__device__ __forceinline__ float scale_of(u32x2_t bytes) { return kv4_scale_value((SEL < 4 ? bytes[0] >> (8 * SEL) : bytes[1] >> (8 * (SEL - 4))) & 255); }
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
  __device__ __forceinline__ void load(const Kv4& c, int64_t slot0, int g, int col) {
    const unsigned char* kt = c.kc + slot0 * (HD / 2);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const unsigned at = (8 * (col >> 2) + 4 * t + (col & 3)) * (HD / 2) + g * (HD / 8 / KN);
#pragma unroll
      for (int n = 0; n < KN; ++n) load_words<KW / KN>(k[t] + n * (KW / KN), kt + at + n * (HD / 4));
    }
    load_words<VW>(v, c.vc + slot0 * (HD / 2) + (g * 16 + col) * (HD / 4));
    const unsigned char *kst = c.ks + slot0 * (HD / 32), *vst = c.vs + slot0 * (HD / 32);
#pragma unroll
    for (int n = 0; n < KN; ++n) ks[n] = *(const u32x2_t*)(kst + (col >> 2) * (HD / 4) + (g * (HD / KN) / 128 + 4 * n) * 8);
    vs = *(const u32x2_t*)(vst + g * (HD / 4) + (col * HD / 512) * 8);
  }
};

template <typename T, int HD, int NW, bool CAP>
__global__ void __launch_bounds__(NW * 64)
kv4_attend_kernel(const T* q, int64_t q_row, int64_t q_head, const void* cache, T* out, float* ws, const int* pos, const float* slopes, int seqs, int heads,
                  int kvh, int cap, int window, float softcap, int chunks) {
  constexpr int KS = HD / 32, NV = HD / 16, QP = sizeof(T) == 2 ? 1 : 3;     // steps of a score's product, tiles of dims, bf16 parts of a query
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
  const int splits = gridDim.x, split = blockIdx.x, hk = blockIdx.y / chunks, chunk = blockIdx.y % chunks, b = blockIdx.z;
  const int group = heads / kvh, cols = min(KV4_COLS, group - chunk * KV4_COLS);
  const int h0 = hk * group + chunk * KV4_COLS;
  const Kv4 c = kv4_at((void*)cache, (int64_t)seqs * kvh, HD, cap);
  const int64_t head0 = ((int64_t)b * kvh + hk) * c.slots;
  const int p = pos[b], tiles = c.slots / KV4_TILE;
  const int ps = p < 0 ? 0 : p % cap, lim = p < 0 ? -1 : min(window, p);
  const int lo = ps - lim < 0 ? ps - lim + cap : ps - lim, start = lo / KV4_TILE;
  const int n = p < 0 ? 0 : ps - lim < 0 ? min(tiles, tiles - start + ps / KV4_TILE + 1) : ps / KV4_TILE - start + 1;
  const int first = (int)((int64_t)n * split / splits), last = (int)((int64_t)n * (split + 1) / splits);

  // queries: column col and col + 8 are the same head
  const int h = h0 + min(col & 7, cols - 1);
  bf16x8_t qf[KS][QP];
  {
    const T* qr = q + b * q_row + h * q_head;
#pragma unroll
    for (int x = 0; x < KS; ++x) {
      float f[8];
      load8(qr + (HD == 256 ? (x >> 2) * 128 + g * 32 + (x & 3) * 8 : g * (HD / 4) + x * 8), f);
#pragma unroll
      for (int e = 0; e < QP; ++e) {
        u32x4_t part;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          part[i] = pack2_bf16(f[2 * i], f[2 * i + 1]);
          f[2 * i] -= __uint_as_float(part[i] << 16);
          f[2 * i + 1] -= __uint_as_float(part[i] & 0xffff0000u);
        }
        qf[x][e] = __builtin_bit_cast(bf16x8_t, part);
      }
    }
  }
  const float kLog2e = 1.4426950408889634f, slope = slopes ? slopes[h] * kLog2e : 0.f, capA = softcap * kLog2e;
  const float scale = rsqrtf((float)HD) * (CAP ? cap_scale<T>(softcap) : kLog2e);
  const unsigned low_part = col < 8 ? 0u : 0xffffffffu;
  float m = -INFINITY, l = 0.f;
  floatx4_t o[NV];
#pragma unroll
  for (int t = 0; t < NV; ++t) o[t] = floatx4_t{0.f, 0.f, 0.f, 0.f};

  auto tile_at = [&](int i) { const int t = start + i; return t >= tiles ? t - tiles : t; };
  Kv4Tile<HD> now, next;
  int i = first + w;
  if (i < last) next.load(c, head0 + (int64_t)tile_at(i) * KV4_TILE, g, col);
  for (; i < last; i += NW) {
    now = next;
    const int t0 = tile_at(i) * KV4_TILE;
    if (i + NW < last) next.load(c, head0 + (int64_t)tile_at(i + NW) * KV4_TILE, g, col);
    float s[8];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      floatx4_t d = {0.f, 0.f, 0.f, 0.f};
      float f[Kv4Tile<HD>::KN];
#pragma unroll
      for (int e = 0; e < Kv4Tile<HD>::KN; ++e) f[e] = kv4_scale_value((now.ks[e][t] >> (8 * (col & 3))) & 255);
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
    const bool whole = t0 + KV4_TILE <= cap && far0 <= lim && (t0 + KV4_TILE - 1 <= ps || t0 > ps);      // wave-uniform
    const float tb = whole ? -slope * (float)(far0 - 8 * g) : 0.f;
    float vs[8] = {scale_of<0>(now.vs), scale_of<1>(now.vs), scale_of<2>(now.vs), scale_of<3>(now.vs),
                   scale_of<4>(now.vs), scale_of<5>(now.vs), scale_of<6>(now.vs), scale_of<7>(now.vs)};
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (CAP) s[j] = capped<T>(s[j], scale, capA);
      if (whole) s[j] = fmaf(s[j], CAP ? 1.f : scale, slope * (float)j);
    }
    if (!whole) {
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
      u32x4_t even, odd;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const unsigned a = piece_pair<HD>(now.v, vs[2 * e], 2 * e, t), z = piece_pair<HD>(now.v, vs[2 * e + 1], 2 * e + 1, t);
        even[e] = __builtin_amdgcn_perm(z, a, 0x05040100);
        odd[e] = __builtin_amdgcn_perm(z, a, 0x07060302);
      }
      o[2 * t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, even), __builtin_bit_cast(bf16x8_t, pf), o[2 * t], 0, 0, 0);
      o[2 * t + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, odd), __builtin_bit_cast(bf16x8_t, pf), o[2 * t + 1], 0, 0, 0);
      if (QP == 3) {
        o[2 * t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, even), __builtin_bit_cast(bf16x8_t, pf2), o[2 * t], 0, 0, 0);
        o[2 * t + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, odd), __builtin_bit_cast(bf16x8_t, pf2), o[2 * t + 1], 0, 0, 0);
      }
    }
  }
  l += fstu_swz16(l);
  l += __shfl_xor(l, 32, FSTU_WAVE);
  extern __shared__ float sm[];                                  // (NW, cols) maxima, sums, then (NW, cols, HD)
  float* const sl = sm + NW * KV4_COLS;
  float* const so = sl + NW * KV4_COLS;
#pragma unroll
  for (int t = 0; t < NV; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r) o[t][r] += fstu_dpp<0x128>(o[t][r]);         // row_ror:8: the other part's column
  if (col < cols) {
    if (g == 0) { sm[w * KV4_COLS + col] = m; sl[w * KV4_COLS + col] = l; }
    float* dst = so + (w * cols + col) * HD + 4 * g * NV;        // dim (4 g + r) * NV + t
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int t = 0; t < NV; ++t) dst[r * NV + t] = o[t][r];
  }
  __syncthreads();
  for (int e = threadIdx.x; e < cols * HD; e += NW * 64) {
    const int cc = e / HD, d = e % HD;
    float M = -INFINITY, L = 0.f, y = 0.f;
#pragma unroll
    for (int x = 0; x < NW; ++x) M = fmaxf(M, sm[x * KV4_COLS + cc]);
#pragma unroll
    for (int x = 0; x < NW; ++x) {
      const float f = sm[x * KV4_COLS + cc] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(sm[x * KV4_COLS + cc] - M);
      const float lx = sl[x * KV4_COLS + cc], yx = so[(x * cols + cc) * HD + d];
      L = fmaf(lx, f, L);
      y = fmaf(yx, f, y);
    }
    const int64_t row = (int64_t)b * heads + h0 + cc;
    if (splits == 1) DT<T>::st(out + row * HD + d, n ? y / L : 0.f);
    else {
      float* part = ws + (row * splits + split) * (HD + 2);
      part[2 + d] = y;
      if (d == 0) { part[0] = M; part[1] = L; }
    }
  }
}

// Splits of a query's keys, in their order.
template <typename T, int HD>
__global__ void __launch_bounds__(HD)
kv4_join_kernel(const float* ws, T* out, int splits) {
  const int64_t row = blockIdx.x;
  const float* part = ws + row * splits * (HD + 2);
  float M = -INFINITY, L = 0.f, y = 0.f;
  for (int s = 0; s < splits; ++s) M = fmaxf(M, part[s * (HD + 2)]);
  for (int s = 0; s < splits; ++s) {
    const float* ps = part + s * (HD + 2);
    const float f = ps[0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ps[0] - M);
    L = fmaf(ps[1], f, L);
    y = fmaf(ps[2 + threadIdx.x], f, y);
  }
  DT<T>::st(out + row * HD + threadIdx.x, L == 0.f ? 0.f : y / L);
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

#define KV4_WAVES 4

extern "C" int fstu_kv4_attend_splits(int seqs, int heads, int kvh, int hd, int cap, int window) {
  if (seqs < 1 || kvh < 1 || heads < kvh || cap < 1 || window < 0) return 1;
  const int chunks = (heads / kvh + KV4_COLS - 1) / KV4_COLS;
  const int64_t groups = (int64_t)seqs * kvh * chunks;
  const int tiles = (int)(((int64_t)(window < cap ? window : cap - 1) + 2 * KV4_TILE - 1) / KV4_TILE);
  int64_t splits = 1024 / groups;
  if (splits > tiles / (4 * KV4_WAVES)) splits = tiles / (4 * KV4_WAVES);
  return splits < 2 ? 1 : (int)(splits > 64 ? 64 : splits);
}

extern "C" int fstu_kv4_attend(const void* q, int64_t q_row, int64_t q_head, const void* cache, void* out, float* ws, int splits, const int* pos,
                               const float* slopes, int seqs, int heads, int kvh, int hd, int cap, int window, float softcap, int dtype, void* stream) {
  const int rc = kv4_check("fstu_kv4_attend", cache, seqs, kvh, hd, cap);
  if (rc) return rc;
  FSTU_REQUIRE(q && out && pos, FSTU_ENULL, "fstu_kv4_attend: null pointer");
  FSTU_REQUIRE(heads >= 1 && heads % kvh == 0 && heads <= 65535 && seqs <= 65535, FSTU_ESHAPE, "fstu_kv4_attend: %d heads over %d key heads, %d sequences", heads,
               kvh, seqs);
  FSTU_REQUIRE(window >= 0 && window < cap, FSTU_EARG, "fstu_kv4_attend: window %d with a capacity of %d", window, cap);
  FSTU_REQUIRE(softcap >= 0.f && softcap < INFINITY, FSTU_EARG, "fstu_kv4_attend: softcap must be zero (none) or a positive number");
  FSTU_REQUIRE(splits >= 1 && splits <= 65535 && (splits == 1 || ws), FSTU_EARG, "fstu_kv4_attend: %d splits need their workspace", splits);
  const int size = dtype == FSTU_BF16 ? 2 : 4;
  FSTU_REQUIRE(fstu_heads_aligned(q, q_row, q_head, size) && fstu_aligned(out, 16) && fstu_aligned(ws, 4), FSTU_EALIGN,
               "fstu_kv4_attend: rows and heads of q and out must begin at multiples of 16 bytes");
  const int64_t n = (int64_t)seqs * heads * hd * size;
  FSTU_REQUIRE(!fstu_heads_touch(q, q_row, q_head, seqs, heads, hd, size, out, n) &&
                   !fstu_heads_touch(cache, fstu_kv4_bytes(seqs, kvh, hd, cap), 0, 2, 1, 0, 1, out, n),
               FSTU_EARG, "fstu_kv4_attend: out overlaps q or the cache");
  const int group = heads / kvh, chunks = (group + KV4_COLS - 1) / KV4_COLS;
  KV4_DISPATCH(dtype, hd, "fstu_kv4_attend", {
    const unsigned lds = KV4_WAVES * (2 * KV4_COLS + (group < KV4_COLS ? group : KV4_COLS) * HD) * sizeof(float);
    auto run = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3(splits, kvh * chunks, seqs), dim3(KV4_WAVES * 64), lds, (hipStream_t)stream, (const T*)q, q_row, q_head, cache, (T*)out, ws,
                         pos, slopes, seqs, heads, kvh, cap, window, softcap, chunks);
    };
    softcap > 0.f ? run(kv4_attend_kernel<T, HD, KV4_WAVES, true>) : run(kv4_attend_kernel<T, HD, KV4_WAVES, false>);
    if (splits > 1) hipLaunchKernelGGL((kv4_join_kernel<T, HD>), dim3(seqs * heads), dim3(HD), 0, (hipStream_t)stream, ws, (T*)out, splits);
  });
  FSTU_CHECK_LAUNCH("fstu_kv4_attend");
  return FSTU_OK;
}
