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

// The sequence that row belongs to (the last one that begins at or in front of it), -1 where none does; *at: its first row, *len: its rows.
__device__ __forceinline__ int kv4_sequence(const int* cu, int seqs, int row, int* at, int* len) {
  int lo = 0, hi = seqs;              // cu[lo] <= row < cu[hi], as far as cu rises
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= row) lo = mid; else hi = mid;
  }
  const int a = cu[lo], b = cu[lo + 1];
  *at = a;
  *len = b - a;
  return row >= a && row < b ? lo : -1;
}

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

// Eight values of a key's or value's row, dims 8u..8u+7, in the cache: codes in a word, low nibble first.
template <int HD>
__device__ __forceinline__ void kv4_put_value(unsigned char* vc, int64_t head, int slots, int slot, int u, unsigned code) {
  constexpr int PB = HD / 32;                                  // bytes of a piece: hd/16 dims
  unsigned char* tile = vc + (head * slots + (slot & ~7)) * (HD / 2) + (slot & 7) * PB;
  if constexpr (PB >= 4) *(unsigned*)(tile + (u * 4 / PB) * 8 * PB + (u * 4) % PB) = code;
  else if constexpr (PB == 2) {
    *(unsigned short*)(tile + (2 * u) * 16) = (unsigned short)code;
    *(unsigned short*)(tile + (2 * u + 1) * 16) = (unsigned short)(code >> 16);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) tile[(4 * u + i) * 8] = (unsigned char)(code >> (8 * i));
  }
}
template <int HD>
__device__ __forceinline__ unsigned kv4_get_value(const unsigned char* vc, int64_t head, int slots, int slot, int u) {
  constexpr int PB = HD / 32;
  const unsigned char* tile = vc + (head * slots + (slot & ~7)) * (HD / 2) + (slot & 7) * PB;
  if constexpr (PB >= 4) return *(const unsigned*)(tile + (u * 4 / PB) * 8 * PB + (u * 4) % PB);
  else if constexpr (PB == 2) return *(const unsigned short*)(tile + (2 * u) * 16) | (unsigned)*(const unsigned short*)(tile + (2 * u + 1) * 16) << 16;
  else {
    unsigned code = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) code |= (unsigned)tile[(4 * u + i) * 8] << (8 * i);
    return code;
  }
}
template <int HD>
__device__ __forceinline__ unsigned char* kv4_scale_at(unsigned char* s, int64_t head, int slots, int slot, int blk) {
  return s + (head * slots + (slot & ~7)) * (HD / 32) + blk * 8 + (slot & 7);
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

// Eight values a thread; threads of y = 1 take the values, of y = 0 the keys.
template <typename T, int HD>
__global__ void __launch_bounds__(256)
kv4_write_kernel(const T* k, const T* v, int64_t k_row, int64_t k_head, int64_t v_row, int64_t v_head, void* cache, const int* pos, const int* cu,
                 int rows, int seqs, int kvh, int cap) {
  constexpr int P = HD / 8;
  const Kv4 c = kv4_at(cache, (int64_t)seqs * kvh, HD, cap);
  const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int u = (int)(idx % P), h = (int)(idx / P % kvh);
  const int64_t row = idx / P / kvh;
  if (row >= rows) return;
  int at = (int)row, len = 1, s = (int)row;
  if (cu) s = kv4_sequence(cu, seqs, (int)row, &at, &len);
  const int p = s < 0 ? -1 : pos[s], t = (int)row - at;
  if (p < 0 || t < len - cap) return;                         // four lanes of a block go together
  const int slot = (int)(((unsigned)p + (unsigned)t) % (unsigned)cap);
  const int64_t head = (int64_t)s * kvh + h;
  float x[8];
  unsigned byte;
  if (blockIdx.y == 0) {
    load8(k + row * k_row + h * k_head + u * 8, x);
    const unsigned code = kv4_quantise(x, &byte);
    *(unsigned*)(c.kc + (head * c.slots + slot) * (HD / 2) + u * 4) = code;
    if ((u & 3) == 0) *kv4_scale_at<HD>(c.ks, head, c.slots, slot, u / 4) = (unsigned char)byte;
  } else {
    load8(v + row * v_row + h * v_head + u * 8, x);
    const unsigned code = kv4_quantise(x, &byte);
    kv4_put_value<HD>(c.vc, head, c.slots, slot, u, code);
    if ((u & 3) == 0) *kv4_scale_at<HD>(c.vs, head, c.slots, slot, u / 4) = (unsigned char)byte;
  }
}

template <typename T, int HD>
__global__ void __launch_bounds__(256)
kv4_read_kernel(const void* cache, T* k, T* v, const int* pos, const int* cu, int rows, int seqs, int kvh, int cap) {
  constexpr int P = HD / 8;
  const Kv4 c = kv4_at((void*)cache, (int64_t)seqs * kvh, HD, cap);
  const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int u = (int)(idx % P), h = (int)(idx / P % kvh);
  const int64_t row = idx / P / kvh;
  if (row >= rows) return;
  int at = (int)row, len = 1, s = (int)row;
  if (cu) s = kv4_sequence(cu, seqs, (int)row, &at, &len);
  const int p = s < 0 ? -1 : pos[s];
  float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (p >= 0) {
    const int slot = (int)(((unsigned)p + (unsigned)((int)row - at)) % (unsigned)cap);
    const int64_t head = (int64_t)s * kvh + h;
    if (blockIdx.y == 0) kv4_values(*(const unsigned*)(c.kc + (head * c.slots + slot) * (HD / 2) + u * 4), *kv4_scale_at<HD>(c.ks, head, c.slots, slot, u / 4), x);
    else kv4_values(kv4_get_value<HD>(c.vc, head, c.slots, slot, u), *kv4_scale_at<HD>(c.vs, head, c.slots, slot, u / 4), x);
  }
  store8((blockIdx.y == 0 ? k : v) + idx * 8, x);
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
  const int64_t blocks = ((int64_t)rows * kvh * (hd / 8) + 255) / 256;
  FSTU_REQUIRE(blocks <= 0x7fffff, FSTU_ESHAPE, "fstu_kv4_write: %d rows of %d heads of %d are more than a launch takes", rows, kvh, hd);
  if (rows == 0) return FSTU_OK;
  KV4_DISPATCH(dtype, hd, "fstu_kv4_write",
               hipLaunchKernelGGL((kv4_write_kernel<T, HD>), dim3((unsigned)blocks, 2), dim3(256), 0, (hipStream_t)stream, (const T*)k, (const T*)v, k_row, k_head,
                                  v_row, v_head, cache, pos, cu, rows, seqs, kvh, cap));
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
  const int64_t blocks = ((int64_t)rows * kvh * (hd / 8) + 255) / 256;
  FSTU_REQUIRE(blocks <= 0x7fffff, FSTU_ESHAPE, "fstu_kv4_read: %d rows of %d heads of %d are more than a launch takes", rows, kvh, hd);
  if (rows == 0) return FSTU_OK;
  KV4_DISPATCH(dtype, hd, "fstu_kv4_read",
               hipLaunchKernelGGL((kv4_read_kernel<T, HD>), dim3((unsigned)blocks, 2), dim3(256), 0, (hipStream_t)stream, cache, (T*)k, (T*)v, pos, cu, rows, seqs,
                                  kvh, cap));
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
