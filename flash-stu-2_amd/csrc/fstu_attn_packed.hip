// Attention over whole prompts of different lengths packed behind one another: causal, an optional window, grouped heads.
//   s_ij = softcap * tanh(q_i . k_j * hd^-1/2 / softcap) - slope * (i - j),  0 <= i - j <= window,  o_i = sum_j softmax_j(s_ij) v_j
#include "fstu_common.h"

#ifndef PK_NW
#define PK_NW 4
#define PK_NQ 2
#endif

namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float floatx4_t __attribute__((ext_vector_type(4)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef unsigned u32x4_t __attribute__((ext_vector_type(4)));

struct Heads {                 // rows of heads: strides in elements
  const void* p;
  int64_t row, head;
};

// The sequence that row tile t (of `per` rows) belongs to, and its number there: sequence i has the tiles from cu[i] / per + i on, which are as many as it
// needs or one more (a sequence's rows begin anywhere), so that no count has to be added up on the way.
__device__ __forceinline__ int packed_tile(const int* cu, int seqs, int rows, int per, int t, int* at, int* len, int* first) {
  const int lo = fstu_last_where(seqs, [&](int i) { return max(cu[i], 0) / per + i <= t; });
  const int a = min(max(cu[lo], 0), rows), b = min(max(cu[lo + 1], a), rows);
  *at = a;
  *len = b - a;
  *first = (t - (a / per + lo)) * per;
  return lo;
}

// One query of one head by a wave, key by key: 8 lanes to a key, 8 keys side by side, each group with a softmax of its own.  i: the query's row in its sequence, which
// begins at row `at`.
template <typename T, int HD>
__device__ __forceinline__ void packed_one(const T* q, const T* kb, const T* vb, T* out, int64_t k_row, int64_t v_row, int i, int window, float slope,
                                           float softcap) {
  constexpr int DPL = HD / 8;
  const int lane = threadIdx.x & 63, gl = lane & 7, G = lane >> 3;
  float qv[DPL], acc[DPL], m = -INFINITY, l = 0.f;
  kb += gl * DPL;
  vb += gl * DPL;
#pragma unroll
  for (int e = 0; e < DPL; ++e) {
    qv[e] = DT<T>::ld(q + gl * DPL + e);
    acc[e] = 0.f;
  }
  const float scale = rsqrtf((float)HD);
  for (int j = max(0, i - window) + G; j <= i; j += 8) {
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < DPL; ++e) s = fmaf(qv[e], DT<T>::ld(kb + j * k_row + e), s);
#pragma unroll
    for (int x = 1; x < 8; x *= 2) s += __shfl_xor(s, x);
    s *= scale;
    if (softcap > 0.f) s = softcap * tanhf(s / softcap);
    s -= slope * (float)(i - j);
    const float mn = fmaxf(m, s), corr = __expf(m - mn), p = __expf(s - mn);
    l = l * corr + p;
    m = mn;
#pragma unroll
    for (int e = 0; e < DPL; ++e) acc[e] = fmaf(p, DT<T>::ld(vb + j * v_row + e), acc[e] * corr);
  }
  float M = m;
#pragma unroll
  for (int x = 8; x < 64; x *= 2) M = fmaxf(M, __shfl_xor(M, x));
  const float f = l == 0.f ? 0.f : __expf(m - M);
  l *= f;
#pragma unroll
  for (int x = 8; x < 64; x *= 2) l += __shfl_xor(l, x);
#pragma unroll
  for (int e = 0; e < DPL; ++e) {
    float a = acc[e] * f;
#pragma unroll
    for (int x = 8; x < 64; x *= 2) a += __shfl_xor(a, x);
    if (G == 0) DT<T>::st(out + gl * DPL + e, a / l);
  }
}

template <typename T, int HD>
__global__ void __launch_bounds__(256)
swa_packed_kernel(Heads q, Heads k, Heads v, T* out, const int* cu, const float* slopes, int rows, int seqs, int heads, int kvh, int window, float softcap) {
  const int h = blockIdx.y, hk = h / (heads / kvh);
  int at, len, first;
  packed_tile(cu, seqs, rows, 4, blockIdx.x, &at, &len, &first);
  const int i = first + (threadIdx.x >> 6);
  if (i < 0 || i >= len) return;
  packed_one<T, HD>((const T*)q.p + (at + i) * q.row + h * q.head, (const T*)k.p + at * k.row + hk * k.head, (const T*)v.p + at * v.row + hk * v.head,
                    out + ((int64_t)(at + i) * heads + h) * HD, k.row, v.row, i, window, slopes ? slopes[h] : 0.f, softcap);
}

template <int HD>
__device__ __forceinline__ int key_turn(int row) {
  return HD >= 128 ? (row & 3) | (row >> 3 & 3) << 2 : HD == 64 ? (row >> 1 & 1) | (row >> 3 & 3) << 1 : row >> 3 & 3;
}
template <int HD>
__device__ __forceinline__ int value_turn(int row) {
  return HD >= 128 ? (row & 3) | (row >> 3 & 1) << 2 : HD == 64 ? (row >> 1 & 1) | (row >> 3 & 1) << 1 : row >> 3 & 1;
}

// bf16 on the matrix cores: a wave owns NQ tiles of 16 queries of one head and walks their keys 32 at a time,
//   S^T (keys x queries) = K Q^T      rows dealt so that lane (g, c) ends up with query c's scores of keys 8 g .. 8 g + 7 of the 32, which is
//   O^T (dims x queries) = V^T P^T    what it holds of the second product: no score crosses a lane, only the maxima do.
// Tiles of KB keys and values go through LDS by way of registers, one barrier a tile; values are read back transposed.
template <int HD, int NW, int NQ, bool CAP, bool BIAS>
__global__ void __launch_bounds__(NW * 64, HD == 256 || NW == 8 ? 1 : 2)
swa_packed_mfma_kernel(Heads q, Heads k, Heads v, bf16_t* out, const int* cu, const float* slopes, int rows, int seqs, int heads, int kvh, int window,
                       float softcap) {
  constexpr int KB = HD == 256 ? 32 : 64, NS = KB / 32, CH = HD / 8, KS = HD / 32, ND = HD / 16, NT = NW * 64, WQ = NQ * 16;
  constexpr int PT = (KB * CH + NT - 1) / NT;                    // 16-byte pieces of a tile to a thread
  __shared__ u32x4_t k_two[2][KB * CH], v_two[2][KB * CH];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, g = lane >> 4;
  const int h = blockIdx.x % heads, hk = h / (heads / kvh);
  int at, len, first;
  packed_tile(cu, seqs, rows, NW * WQ, gridDim.x / heads - 1 - blockIdx.x / heads, &at, &len, &first);
  if (first < 0 || first >= len) return;
  const int qs = first + w * WQ;                                 // the wave's first query
  const bool on = qs < len;
  const int64_t k_row = k.row, v_row = v.row;
  const bf16_t* kb = (const bf16_t*)k.p + at * k_row + hk * k.head;
  const bf16_t* vb = (const bf16_t*)v.p + at * v_row + hk * v.head;
  const float kLog2e = 1.4426950408889634f, raw_slope = BIAS ? slopes[h] : 0.f, slope = raw_slope * kLog2e;
  const float scale = rsqrtf((float)HD) * (CAP ? 2.0f * kLog2e / softcap : kLog2e), capA = softcap * kLog2e;

  u32x4_t qf[NQ][KS];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const bf16_t* qr = (const bf16_t*)q.p + (at + min(qs + n * 16 + c, len - 1)) * q.row + h * q.head + g * 8;
#pragma unroll
    for (int s = 0; s < KS; ++s) qf[n][s] = *(const u32x4_t*)(qr + s * 32);
  }
  floatx4_t o[NQ][ND];
  float m[NQ], l[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    m[n] = -INFINITY;
    l[n] = 0.f;
#pragma unroll
    for (int d = 0; d < ND; ++d) o[n][d] = floatx4_t{0.f, 0.f, 0.f, 0.f};
  }
  // ALiBi of key 8 g + 4 t + r of 32: without a soft-cap what the scores' sums begin with, in units of theirs
  floatx4_t bias[2];
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r) bias[t][r] = BIAS ? slope * (float)(8 * g + 4 * t + r) / (CAP ? 1.f : scale) : 0.f;

  const int k_first = max(0, first - window) / KB * KB, k_last = min(len - 1, first + NW * WQ - 1);
  u32x4_t kr[PT], vr[PT];
  auto fetch = [&](int b) {
#pragma unroll
    for (int i = 0; i < PT; ++i) {
      const int e = min(tid + i * NT, KB * CH - 1);              // threads beyond the tile's pieces hold the last one too
      const int64_t row = min(b + e / CH, len - 1);              // rows behind the sequence: its last one, which no query of these sees
      kr[i] = *(const u32x4_t*)(kb + row * k_row + e % CH * 8);
      vr[i] = *(const u32x4_t*)(vb + row * v_row + e % CH * 8);
    }
  };
  // The 16-byte pieces of a row are XOR-ed with bits of it, so that what 16 lanes read together lies in different banks: 16 keys' rows one piece each (rows
  // differ in bits 0, 1, 3 and 4), four values' rows 32 bytes each (bits 0, 1 and 3: two blocks of lanes).
  auto store = [&](int buf) {
#pragma unroll
    for (int i = 0; i < PT; ++i) {
      const int e = min(tid + i * NT, KB * CH - 1), row = e / CH, ch = e % CH;
      k_two[buf][row * CH + (ch ^ key_turn<HD>(row))] = kr[i];
      v_two[buf][row * CH + (ch ^ value_turn<HD>(row) << 1)] = vr[i];
    }
  };
  int k_at[KS], v_at[ND];                                        // in pieces, and in elements
  {
    const int row = 8 * (c >> 2) + (c & 3), vrow = 8 * g + (c >> 2);
#pragma unroll
    for (int s = 0; s < KS; ++s) k_at[s] = row * CH + ((4 * s + g) ^ key_turn<HD>(row));
#pragma unroll
    for (int d = 0; d < ND; ++d) v_at[d] = vrow * HD + (d ^ value_turn<HD>(vrow)) * 16 + 4 * (c & 3);
  }
  fetch(k_first);
  store(0);
  if (k_first + KB <= k_last) fetch(k_first + KB);
  __syncthreads();
  int buf = 0;
  for (int b = k_first; b <= k_last; b += KB, buf ^= 1) {
    if (b > k_first) __syncthreads();                            // this tile is there, and the one before it has been read
    if (b + KB <= k_last) store(buf ^ 1);
    if (b + 2 * KB <= k_last) fetch(b + 2 * KB);
    if (!on) continue;
#pragma unroll
    for (int u = 0; u < NS; ++u) {
      const int b0 = b + 32 * u;
      if (b0 > qs + WQ - 1 || b0 + 31 < qs - window) continue;   // wave-uniform: the wave sees none of it
      const u32x4_t* kl = k_two[buf] + u * 32 * CH;
      const bf16_t* vl = (const bf16_t*)v_two[buf] + u * 32 * HD;
      floatx4_t s[NQ][2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int n = 0; n < NQ; ++n) s[n][t] = CAP || !BIAS ? floatx4_t{0.f, 0.f, 0.f, 0.f} : bias[t];
#pragma unroll
        for (int x = 0; x < KS; ++x) {
          const bf16x8_t f = __builtin_bit_cast(bf16x8_t, kl[k_at[x] + t * 4 * CH]);
#pragma unroll
          for (int n = 0; n < NQ; ++n) s[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f, __builtin_bit_cast(bf16x8_t, qf[n][x]), s[n][t], 0, 0, 0);
        }
      }
      const bool edge = b0 + 31 > qs || b0 < qs + WQ - 1 - window;     // wave-uniform: some key is not visible to some query
      u32x4_t pf[NQ];
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        const int far0 = qs + n * 16 + c - b0;                   // how far behind the lane's query key 0 of the 32 is
        const float base = -slope * (float)far0;
        if (CAP) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float r = __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(s[n][e >> 2][e & 3] * scale) + 1.0f);
            s[n][e >> 2][e & 3] = fmaf(-2.0f * capA, r, BIAS ? capA + bias[e >> 2][e & 3] : capA);
          }
        }
        if (edge) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int far = far0 - 8 * g - e;
            s[n][e >> 2][e & 3] = far >= 0 && far <= window ? s[n][e >> 2][e & 3] : -INFINITY;
          }
        }
        const float kk = CAP ? 1.f : scale;
        float top = fmaxf(fmaxf(s[n][0][0], s[n][0][1]), s[n][0][2]);
        top = fmaxf(fmaxf(top, s[n][0][3]), s[n][1][0]);
        top = fmaxf(fmaxf(top, s[n][1][1]), s[n][1][2]);
        top = fmaf(fmaxf(top, s[n][1][3]), kk, base);
        // Lanes exchange their maxima, and what was summed so far is rescaled, only where a score exceeds the running maximum by 2^8: a probability is up to 2^8
        // then, which costs neither the sums (fp32) nor its rounding to bf16 (relative) anything.
        if (__any(top > m[n] + 8.f)) {
          top = fmaxf(top, fstu_swz16(top));
          top = fmaxf(top, __shfl_xor(top, 32, FSTU_WAVE));
          const float mn = fmaxf(m[n], top), corr = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[n] - mn);
          l[n] *= corr;
#pragma unroll
          for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int r = 0; r < 4; ++r) o[n][d][r] *= corr;
          m[n] = mn;
        }
        const float off = base - (m[n] == -INFINITY ? 0.f : m[n]);
        float p[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x = s[n][e >> 2][e & 3];
          p[e] = __builtin_amdgcn_exp2f(CAP ? x + off : fmaf(x, scale, off));
          l[n] += p[e];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) pf[n][e] = pack2_bf16(p[2 * e], p[2 * e + 1]);
      }
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        struct { s16x4_t a, b; } f;
        f.a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t*)(vl + v_at[d]));
        f.b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t*)(vl + v_at[d] + 4 * HD));
#pragma unroll
        for (int n = 0; n < NQ; ++n)
          o[n][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, f), __builtin_bit_cast(bf16x8_t, pf[n]), o[n][d], 0, 0, 0);
      }
    }
  }
  if (!on) return;
  unsigned long long bad = 0;
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    l[n] += fstu_swz16(l[n]);
    l[n] += __shfl_xor(l[n], 32, FSTU_WAVE);
    const float inv = 1.0f / l[n];
    const int qi = qs + n * 16 + c;
    bool fine = true;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        o[n][d][r] *= inv;
        fine = fine && o[n][d][r] == o[n][d][r];
      }
    if (qi < len) {
      bf16_t* orow = out + ((int64_t)(at + qi) * heads + h) * HD + 4 * g;
#pragma unroll
      for (int d = 0; d < ND; ++d) *(uint2*)(orow + d * 16) = make_uint2(pack2_bf16(o[n][d][0], o[n][d][1]), pack2_bf16(o[n][d][2], o[n][d][3]));
    }
    unsigned long long here = __ballot(!fine && qi < len);
    here |= here >> 32;
    bad |= ((here | here >> 16) & 0xffffull) << (16 * n);
  }
  // A NaN comes from a row's own scores and values, or from a value that it does not see (0 * infinity): the wave forms such rows once more, key by key.
  while (bad) {
    const int i = qs + __builtin_ctzll(bad);
    bad &= bad - 1;
    packed_one<bf16_t, HD>((const bf16_t*)q.p + (at + i) * q.row + h * q.head, kb, vb, out + ((int64_t)(at + i) * heads + h) * HD, k_row, v_row, i, window,
                           raw_slope, softcap);
  }
}

}  // namespace

extern "C" int fstu_swa_packed(const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row, int64_t k_head, const void* v, int64_t v_row,
                               int64_t v_head, void* out, const int* cu, const float* slopes, int rows, int seqs, int heads, int kvh, int hd, int window,
                               float softcap, int dtype, void* stream) {
  FSTU_REQUIRE(q && k && v && out && cu, FSTU_ENULL, "fstu_swa_packed: null pointer");
  FSTU_REQUIRE(dtype == FSTU_F32 || dtype == FSTU_BF16, FSTU_EDTYPE, "fstu_swa_packed: unknown dtype %d", dtype);
  FSTU_REQUIRE(hd == 32 || hd == 64 || hd == 128 || hd == 256, FSTU_ESHAPE, "fstu_swa_packed: head dim %d not in {32,64,128,256}", hd);
  FSTU_REQUIRE(rows >= 0 && rows <= (1 << 30) && seqs >= 0 && seqs <= (1 << 30) && kvh >= 1 && heads >= 1 && heads % kvh == 0 && heads <= 65535, FSTU_ESHAPE,
               "fstu_swa_packed: bad shape rows=%d sequences=%d heads=%d key heads=%d", rows, seqs, heads, kvh);
  FSTU_REQUIRE(window >= 0, FSTU_EARG, "fstu_swa_packed: window<0");
  FSTU_REQUIRE(softcap >= 0.f && softcap < INFINITY, FSTU_EARG, "fstu_swa_packed: softcap must be zero (none) or a positive number");
  const int size = dtype == FSTU_BF16 ? 2 : 4;
  FSTU_REQUIRE(fstu_heads_aligned(q, q_row, q_head, size) && fstu_heads_aligned(k, k_row, k_head, size) && fstu_heads_aligned(v, v_row, v_head, size) &&
                   fstu_aligned(out, 16),
               FSTU_EALIGN, "fstu_swa_packed: rows and heads of q, k and v and out must begin at multiples of 16 bytes");
  const int64_t n = (int64_t)rows * heads * hd * size;
  FSTU_REQUIRE(!fstu_heads_touch(q, q_row, q_head, rows, heads, hd, size, out, n) && !fstu_heads_touch(k, k_row, k_head, rows, kvh, hd, size, out, n) &&
                   !fstu_heads_touch(v, v_row, v_head, rows, kvh, hd, size, out, n),
               FSTU_EARG, "fstu_swa_packed: out overlaps q, k or v");
  if (rows == 0 || seqs == 0) return FSTU_OK;
  const Heads hq{q, q_row, q_head}, hk{k, k_row, k_head}, hv{v, v_row, v_head};
  auto run = [&](auto w) {
    constexpr int HD = decltype(w)::value;
    if (dtype == FSTU_F32) {
      hipLaunchKernelGGL((swa_packed_kernel<float, HD>), dim3(rows / 4 + seqs, heads), dim3(256), 0, (hipStream_t)stream, hq, hk, hv, (float*)out, cu, slopes, rows,
                         seqs, heads, kvh, window, softcap);
      return;
    }
    auto bf16 = [&](auto nw, auto nq) {
      constexpr int NW = decltype(nw)::value, NQ = decltype(nq)::value;
      auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)(rows / (NW * NQ * 16) + seqs) * heads), dim3(NW * 64), 0, (hipStream_t)stream, hq, hk, hv, (bf16_t*)out, cu,
                           slopes, rows, seqs, heads, kvh, window, softcap);
      };
      if (softcap > 0.f) slopes ? go(swa_packed_mfma_kernel<HD, NW, NQ, true, true>) : go(swa_packed_mfma_kernel<HD, NW, NQ, true, false>);
      else slopes ? go(swa_packed_mfma_kernel<HD, NW, NQ, false, true>) : go(swa_packed_mfma_kernel<HD, NW, NQ, false, false>);
    };
    bf16(std::integral_constant<int, PK_NW>{}, std::integral_constant<int, HD == 256 ? 2 : PK_NQ>{});
  };
  if (hd == 32) run(std::integral_constant<int, 32>{});
  else if (hd == 64) run(std::integral_constant<int, 64>{});
  else if (hd == 128) run(std::integral_constant<int, 128>{});
  else run(std::integral_constant<int, 256>{});
  FSTU_CHECK_LAUNCH("fstu_swa_packed");
  return FSTU_OK;
}
