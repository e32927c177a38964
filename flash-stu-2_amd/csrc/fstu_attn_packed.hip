// Attention over whole prompts of different lengths packed behind one another: causal, an optional window, grouped heads.
//   s_ij = softcap * tanh(q_i . k_j * hd^-1/2 / softcap) - slope * (i - j),  0 <= i - j <= window,  o_i = sum_j softmax_j(s_ij) v_j
#include "fstu_common.h"

namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef float floatx16_t __attribute__((ext_vector_type(16)));
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

__device__ __forceinline__ float other_half(float v) { return __shfl_xor(v, 32, FSTU_WAVE); }

template <int HD, int NW, bool CAP, bool BIAS>
__global__ void __launch_bounds__(NW * 64, HD == 256 ? 1 : 2)
swa_packed_mfma_kernel(Heads q, Heads k, Heads v, bf16_t* out, const int* cu, const float* slopes, int rows, int seqs, int heads, int kvh, int window,
                       float softcap) {
  constexpr int KB = HD == 256 ? 32 : 64, NS = KB / 32, CH = HD / 8, KS = HD / 16, ND = HD / 32, NT = NW * 64;
  constexpr int PT = (KB * CH + NT - 1) / NT;                    // 16-byte pieces of a tile to a thread
  __shared__ u32x4_t k_two[2][KB * CH], v_two[2][KB * CH];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, c = lane & 31, hi = lane >> 5;
  const int h = blockIdx.x % heads, hk = h / (heads / kvh);
  int at, len, first;
  packed_tile(cu, seqs, rows, NW * 32, gridDim.x / heads - 1 - blockIdx.x / heads, &at, &len, &first);
  if (first < 0 || first >= len) return;
  const int qs = first + w * 32, qi = qs + c;                    // the wave's first query, this lane's
  const bool on = qs < len;
  const bf16_t* kb = (const bf16_t*)k.p + at * k.row + hk * k.head;
  const bf16_t* vb = (const bf16_t*)v.p + at * v.row + hk * v.head;
  const int64_t k_row = k.row, v_row = v.row;
  const float kLog2e = 1.4426950408889634f, raw_slope = BIAS ? slopes[h] : 0.f, slope = raw_slope * kLog2e;
  const float scale = rsqrtf((float)HD) * (CAP ? 2.0f * kLog2e / softcap : kLog2e), capA = softcap * kLog2e;

  u32x4_t qf[KS];
  {
    const bf16_t* qr = (const bf16_t*)q.p + (at + min(qi, len - 1)) * q.row + h * q.head + hi * 8;
#pragma unroll
    for (int s = 0; s < KS; ++s) qf[s] = *(const u32x4_t*)(qr + s * 16);
  }
  floatx16_t o[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[d][r] = 0.f;
  float bias[16];                                                // of row (r & 3) + 8 (r >> 2) + 4 hi of a tile of 32 keys
#pragma unroll
  for (int r = 0; r < 16; ++r) bias[r] = BIAS ? slope * (float)((r & 3) + 8 * (r >> 2) + 4 * hi) * (CAP ? 1.f : 1.f / scale) : 0.f;
  float m = -INFINITY, l = 0.f;

  const int k_first = max(0, first - window) / KB * KB, k_last = min(len - 1, first + NW * 32 - 1);
  u32x4_t kr[PT], vr[PT];
  auto fetch = [&](int b) {
#pragma unroll
    for (int i = 0; i < PT; ++i) {
      const int e = min(tid + i * NT, KB * CH - 1);
      const int64_t row = min(b + e / CH, len - 1);              // rows behind the sequence: its last one, which no query of these sees
      kr[i] = *(const u32x4_t*)(kb + row * k_row + e % CH * 8);
      vr[i] = *(const u32x4_t*)(vb + row * v_row + e % CH * 8);
    }
  };
  auto store = [&](int buf) {
#pragma unroll
    for (int i = 0; i < PT; ++i) {
      const int e = min(tid + i * NT, KB * CH - 1), row = e / CH, ch = e % CH;
      const int ks = HD >= 128 ? row & 15 : HD == 64 ? (row >> 1) & 7 : (row >> 2) & 3;
      const int vs = HD >= 128 ? (row & 3) << 2 : HD == 64 ? (row >> 1 & 1) << 2 : 0;
      k_two[buf][row * CH + (ch ^ ks)] = kr[i];
      v_two[buf][row * CH + (ch ^ vs)] = vr[i];
    }
  };
  fetch(k_first);
  store(0);
  if (k_first + KB <= k_last) fetch(k_first + KB);
  __syncthreads();
  const int ksw = HD >= 128 ? c & 15 : HD == 64 ? (c >> 1) & 7 : (c >> 2) & 3;
  const int li = lane & 15, vx = HD >= 128 ? (li >> 2) & 3 : HD == 64 ? (li >> 3) & 1 : 0;
  const int v_at = (4 * hi + (li >> 2)) * HD + 16 * (lane >> 4 & 1) + 4 * (li & 3);      // in elements, without the tile of 32 dims
  int buf = 0;
  for (int b = k_first; b <= k_last; b += KB, buf ^= 1) {
    if (b > k_first) __syncthreads();                            // this tile is there, and the one before it has been read
    if (b + KB <= k_last) store(buf ^ 1);
    if (b + 2 * KB <= k_last) fetch(b + 2 * KB);
    if (!on || b > qs + 31 || b + KB - 1 < qs - window) continue;     // wave-uniform: the wave sees none of it
    const u32x4_t* kl = k_two[buf];
    const bf16_t* vl = (const bf16_t*)v_two[buf];
    floatx16_t s[NS];
#pragma unroll
    for (int u = 0; u < NS; ++u) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[u][r] = CAP ? 0.f : bias[r];
#pragma unroll
      for (int x = 0; x < KS; ++x) {
        const u32x4_t f = kl[(u * 32 + c) * CH + ((2 * x + hi) ^ ksw)];
        s[u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, f), __builtin_bit_cast(bf16x8_t, qf[x]), s[u], 0, 0, 0);
      }
    }
    const float base = slope * (float)(b - qi);
    if (CAP) {
#pragma unroll
      for (int u = 0; u < NS; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          s[u][r] = fmaf(-2.0f * capA, __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(s[u][r] * scale) + 1.0f), capA + bias[r]);
    }
    if (b + KB - 1 > qs || b < qs + 31 - window) {               // wave-uniform: some key is not visible to some query
#pragma unroll
      for (int u = 0; u < NS; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int far = qi - b - u * 32 - ((r & 3) + 8 * (r >> 2) + 4 * hi);
          s[u][r] = far >= 0 && far <= window ? s[u][r] : -INFINITY;
        }
    }
    const float kk = CAP ? 1.f : scale;
    float top = -INFINITY;
#pragma unroll
    for (int u = 0; u < NS; ++u) {
      float t = s[u][0];
#pragma unroll
      for (int r = 1; r < 16; ++r) t = fmaxf(t, s[u][r]);
      top = fmaxf(top, fmaf(t, kk, base + slope * (float)(32 * u)));
    }
    if (__any(top > m + 8.f)) {
      top = fmaxf(top, other_half(top));
      const float mn = fmaxf(m, top);
      const float corr = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
      l *= corr;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] *= corr;
      m = mn;
    }
    const float off = base - (m == -INFINITY ? 0.f : m);
#pragma unroll
    for (int u = 0; u < NS; ++u) {
      const float ou = off + slope * (float)(32 * u);
      unsigned pk[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float a = CAP ? s[u][2 * e] + ou : fmaf(s[u][2 * e], scale, ou), bb = CAP ? s[u][2 * e + 1] + ou : fmaf(s[u][2 * e + 1], scale, ou);
        pk[e] = pack2_bf16(__builtin_amdgcn_exp2f(a), __builtin_amdgcn_exp2f(bb));
        l = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, pk[e]), __builtin_bit_cast(bf16x2_t, 0x3f803f80u), l, false);
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const u32x4_t pf = u32x4_t{pk[4 * t], pk[4 * t + 1], pk[4 * t + 2], pk[4 * t + 3]};
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          const bf16_t* va = vl + v_at + (u * 32 + t * 16) * HD + (d ^ vx) * 32;
          struct { s16x4_t a, b; } f;
          f.a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t*)va);
          f.b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t*)(va + 8 * HD));
          o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, f), __builtin_bit_cast(bf16x8_t, pf), o[d], 0, 0, 0);
        }
      }
    }
  }
  if (!on) return;
  l += other_half(l);
  const float inv = 1.0f / l;
  bool fine = true;
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      o[d][r] *= inv;
      fine = fine && o[d][r] == o[d][r];
    }
  if (qi < len) {
    bf16_t* orow = out + ((int64_t)(at + qi) * heads + h) * HD + 4 * hi;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        *(uint2*)(orow + d * 32 + e * 8) = make_uint2(pack2_bf16(o[d][4 * e], o[d][4 * e + 1]), pack2_bf16(o[d][4 * e + 2], o[d][4 * e + 3]));
  }
  // A NaN comes from a row's own scores and values, or from a value that it does not see (0 * infinity): the wave forms such rows once more, key by key.
  unsigned long long bad = __ballot(!fine && qi < len);
  bad = (bad | bad >> 32) & 0xffffffffull;
  while (bad) {
    const int i = qs + __builtin_ctzll(bad);
    bad &= bad - 1;
    packed_one<bf16_t, HD>((const bf16_t*)q.p + (at + i) * q.row + h * q.head, kb, vb, out + ((int64_t)(at + i) * heads + h) * HD, k.row, v.row, i, window,
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
    constexpr int NW = 4;
    auto go = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3((unsigned)(rows / (NW * 32) + seqs) * heads), dim3(NW * 64), 0, (hipStream_t)stream, hq, hk, hv, (bf16_t*)out, cu, slopes,
                         rows, seqs, heads, kvh, window, softcap);
    };
    if (softcap > 0.f) slopes ? go(swa_packed_mfma_kernel<HD, NW, true, true>) : go(swa_packed_mfma_kernel<HD, NW, true, false>);
    else slopes ? go(swa_packed_mfma_kernel<HD, NW, false, true>) : go(swa_packed_mfma_kernel<HD, NW, false, false>);
  };
  if (hd == 32) run(std::integral_constant<int, 32>{});
  else if (hd == 64) run(std::integral_constant<int, 64>{});
  else if (hd == 128) run(std::integral_constant<int, 128>{});
  else run(std::integral_constant<int, 256>{});
  FSTU_CHECK_LAUNCH("fstu_swa_packed");
  return FSTU_OK;
}
