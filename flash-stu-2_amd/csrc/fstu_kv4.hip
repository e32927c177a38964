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

// One query: 8 lanes to a key, 32 keys of a workgroup side by side, each group with a softmax of its own; joined through LDS.
template <typename T, int HD>
__global__ void __launch_bounds__(256)
kv4_attend_kernel(const T* q, int64_t q_row, int64_t q_head, const void* cache, T* out, const int* pos, const float* slopes, int seqs, int heads, int kvh,
                  int cap, int window, float softcap) {
  constexpr int DPL = HD / 8, NB = DPL < 8 ? 1 : DPL / 8, E = DPL < 8 ? DPL : 8;
  const Kv4 c = kv4_at((void*)cache, (int64_t)seqs * kvh, HD, cap);
  const int h = blockIdx.x, b = blockIdx.y, gl = threadIdx.x & 7, G = threadIdx.x >> 3;
  const int p = pos[b], n = p < 0 ? 0 : min(p, window) + 1;
  const int ps = p < 0 ? 0 : p % cap;
  const int64_t head = (int64_t)b * kvh + h / (heads / kvh);
  float qv[DPL], acc[DPL], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < DPL; ++i) {
    qv[i] = DT<T>::ld(q + b * q_row + h * q_head + gl * DPL + i);
    acc[i] = 0.f;
  }
  const float slope = slopes ? slopes[h] : 0.f, scale = rsqrtf((float)HD);
  for (int far = G; far < n; far += 32) {
    int slot = ps - far;
    slot = slot < 0 ? slot + cap : slot;
    float s = 0.f, x[8];
    const unsigned char* kr = c.kc + (head * c.slots + slot) * (HD / 2);
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int d = gl * DPL + i * 8;
      const unsigned code = *(const unsigned*)(kr + (d & ~7) / 2) >> ((d & 7) * 4);
      kv4_values(code, *kv4_scale_at<HD>(c.ks, head, c.slots, slot, d / 32), x);
#pragma unroll
      for (int e = 0; e < E; ++e) s = fmaf(qv[i * 8 + e], x[e], s);
    }
#pragma unroll
    for (int x = 1; x < 8; x *= 2) s += __shfl_xor(s, x);
    s *= scale;
    if (softcap > 0.f) s = softcap * tanhf(s / softcap);
    s -= slope * (float)far;
    const float mn = fmaxf(m, s), corr = __expf(m - mn), pr = __expf(s - mn);
    l = l * corr + pr;
    m = mn;
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int d = gl * DPL + i * 8;
      const unsigned code = kv4_get_value<HD>(c.vc, head, c.slots, slot, d / 8) >> ((d & 7) * 4);
      kv4_values(code, *kv4_scale_at<HD>(c.vs, head, c.slots, slot, d / 32), x);
#pragma unroll
      for (int e = 0; e < E; ++e) acc[i * 8 + e] = fmaf(pr, x[e], acc[i * 8 + e] * corr);
    }
  }
  __shared__ float sm[32], sl[32], sa[32][HD];
  if (gl == 0) { sm[G] = m; sl[G] = l; }
#pragma unroll
  for (int i = 0; i < DPL; ++i) sa[G][gl * DPL + i] = acc[i];
  __syncthreads();
  if ((int)threadIdx.x < HD) {
    float M = -INFINITY, L = 0.f, o = 0.f;
    for (int g = 0; g < 32; ++g) M = fmaxf(M, sm[g]);
    for (int g = 0; g < 32; ++g) {
      const float e = sm[g] == -INFINITY && sl[g] == 0.f ? 0.f : __expf(sm[g] - M);
      L = fmaf(sl[g], e, L);
      o = fmaf(sa[g][threadIdx.x], e, o);
    }
    DT<T>::st(out + ((int64_t)b * heads + h) * HD + threadIdx.x, n ? o / L : 0.f);
  }
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

extern "C" int fstu_kv4_attend(const void* q, int64_t q_row, int64_t q_head, const void* cache, void* out, const int* pos, const float* slopes, int seqs,
                               int heads, int kvh, int hd, int cap, int window, float softcap, int dtype, void* stream) {
  const int rc = kv4_check("fstu_kv4_attend", cache, seqs, kvh, hd, cap);
  if (rc) return rc;
  FSTU_REQUIRE(q && out && pos, FSTU_ENULL, "fstu_kv4_attend: null pointer");
  FSTU_REQUIRE(heads >= 1 && heads % kvh == 0 && heads <= 65535 && seqs <= 65535, FSTU_ESHAPE, "fstu_kv4_attend: %d heads over %d key heads, %d sequences", heads,
               kvh, seqs);
  FSTU_REQUIRE(window >= 0 && window < cap, FSTU_EARG, "fstu_kv4_attend: window %d with a capacity of %d", window, cap);
  FSTU_REQUIRE(softcap >= 0.f && softcap < INFINITY, FSTU_EARG, "fstu_kv4_attend: softcap must be zero (none) or a positive number");
  const int size = dtype == FSTU_BF16 ? 2 : 4;
  FSTU_REQUIRE(fstu_heads_aligned(q, q_row, q_head, size) && fstu_aligned(out, 16), FSTU_EALIGN,
               "fstu_kv4_attend: rows and heads of q and out must begin at multiples of 16 bytes");
  const int64_t n = (int64_t)seqs * heads * hd * size;
  FSTU_REQUIRE(!fstu_heads_touch(q, q_row, q_head, seqs, heads, hd, size, out, n) &&
                   !fstu_heads_touch(cache, fstu_kv4_bytes(seqs, kvh, hd, cap), 0, 2, 1, 0, 1, out, n),
               FSTU_EARG, "fstu_kv4_attend: out overlaps q or the cache");
  KV4_DISPATCH(dtype, hd, "fstu_kv4_attend",
               hipLaunchKernelGGL((kv4_attend_kernel<T, HD>), dim3(heads, seqs), dim3(256), 0, (hipStream_t)stream, (const T*)q, q_row, q_head, cache, (T*)out, pos,
                                  slopes, seqs, heads, kvh, cap, window, softcap));
  FSTU_CHECK_LAUNCH("fstu_kv4_attend");
  return FSTU_OK;
}
