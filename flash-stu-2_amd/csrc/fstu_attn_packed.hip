// Attention over whole prompts of different lengths packed behind one another: causal, an optional window, grouped heads.
//   s_ij = softcap * tanh(q_i . k_j * hd^-1/2 / softcap) - slope * (i - j),  0 <= i - j <= window,  o_i = sum_j softmax_j(s_ij) v_j
#include "fstu_common.h"

namespace {

// One wave to a query: 8 lanes to a key, 8 keys side by side, each group with a softmax of its own.
template <typename T, int HD>
__global__ void __launch_bounds__(256)
swa_packed_kernel(const T* q, const T* k, const T* v, T* out, const int* cu, const float* slopes, int64_t q_row, int64_t q_head, int64_t k_row, int64_t k_head,
                  int64_t v_row, int64_t v_head, int rows, int seqs, int heads, int kvh, int window, float softcap) {
  constexpr int DPL = HD / 8;
  const int h = blockIdx.y, lane = threadIdx.x & 63, gl = lane & 7, G = lane >> 3;
  const int row = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  int lo = 0, hi = seqs;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= row) lo = mid; else hi = mid;
  }
  const int at = max(cu[lo], 0);
  if (row < at || row >= cu[lo + 1]) return;                 // behind the last sequence
  const int first = window < row - at ? row - window : at;
  const T *kb = k + h / (heads / kvh) * k_head + gl * DPL, *vb = v + h / (heads / kvh) * v_head + gl * DPL;
  float qv[DPL], acc[DPL], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < DPL; ++i) {
    qv[i] = DT<T>::ld(q + row * q_row + h * q_head + gl * DPL + i);
    acc[i] = 0.f;
  }
  const float slope = slopes ? slopes[h] : 0.f, scale = rsqrtf((float)HD);
  for (int j = first + G; j <= row; j += 8) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < DPL; ++i) s = fmaf(qv[i], DT<T>::ld(kb + j * k_row + i), s);
#pragma unroll
    for (int x = 1; x < 8; x *= 2) s += __shfl_xor(s, x);
    s *= scale;
    if (softcap > 0.f) s = softcap * tanhf(s / softcap);
    s -= slope * (float)(row - j);
    const float mn = fmaxf(m, s), corr = __expf(m - mn), p = __expf(s - mn);
    l = l * corr + p;
    m = mn;
#pragma unroll
    for (int i = 0; i < DPL; ++i) acc[i] = fmaf(p, DT<T>::ld(vb + j * v_row + i), acc[i] * corr);
  }
  float M = m;
#pragma unroll
  for (int x = 8; x < 64; x *= 2) M = fmaxf(M, __shfl_xor(M, x));
  const float e = l == 0.f ? 0.f : __expf(m - M);
  l *= e;
#pragma unroll
  for (int x = 8; x < 64; x *= 2) l += __shfl_xor(l, x);
#pragma unroll
  for (int i = 0; i < DPL; ++i) {
    float a = acc[i] * e;
#pragma unroll
    for (int x = 8; x < 64; x *= 2) a += __shfl_xor(a, x);
    if (G == 0) DT<T>::st(out + ((int64_t)row * heads + h) * HD + gl * DPL + i, a / l);
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
  auto run = [&](auto t, auto w) {
    using T = decltype(t);
    constexpr int HD = decltype(w)::value;
    hipLaunchKernelGGL((swa_packed_kernel<T, HD>), dim3((rows + 3) / 4, heads), dim3(256), 0, (hipStream_t)stream, (const T*)q, (const T*)k, (const T*)v, (T*)out,
                       cu, slopes, q_row, q_head, k_row, k_head, v_row, v_head, rows, seqs, heads, kvh, window, softcap);
  };
  auto by_width = [&](auto t) {
    if (hd == 32) run(t, std::integral_constant<int, 32>{});
    else if (hd == 64) run(t, std::integral_constant<int, 64>{});
    else if (hd == 128) run(t, std::integral_constant<int, 128>{});
    else run(t, std::integral_constant<int, 256>{});
  };
  if (dtype == FSTU_F32) by_width(float{}); else by_width(bf16_t{});
  FSTU_CHECK_LAUNCH("fstu_swa_packed");
  return FSTU_OK;
}
