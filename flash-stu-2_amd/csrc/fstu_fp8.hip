// Activations and weights to 8-bit codes with scales: rows in blocks of 128 values, weights in blocks of 128 x 128, and the RMSNorm
// with the residual's addition whose result leaves as codes (the norm in front of the MLP, flash_stu/layers/stu_layer.py:95-96 and
// layers/attention_layer.py:58-62, where the MLP runs in 8 bits).
//
// A lane holds 8 consecutive values, the 16 lanes of a DPP row one block: its amax takes four lane exchanges, its codes leave as one
// line of 128 bytes.  All three read their operands once and keep them in registers: the bytes bound them.
#include <algorithm>
#include "fstu_fp8.h"

namespace {

// 16 bytes at an element's alignment
typedef unsigned u32x4_any_t __attribute__((ext_vector_type(4), aligned(2)));
typedef float floatx4_any_t __attribute__((ext_vector_type(4), aligned(4)));

// 8 consecutive values from column c of a row of d (fewer behind its end: zeros there).  VEC: rows of whole 8 values at 16-byte addresses;
// otherwise the 8 are read at whatever address they begin (one by one 16384 x 2047 took 124 us), those of a row's end one by one.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* p, int c, int d, float (&v)[8]) {
  if (VEC ? c < d : c + 8 <= d) {
    if constexpr (sizeof(T) == 4 && VEC) {
      const float4 a = *(const float4*)(p + c), b = *(const float4*)(p + c + 4);
      v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else if constexpr (sizeof(T) == 4) {
      const floatx4_any_t a = *(const floatx4_any_t*)(p + c), b = *(const floatx4_any_t*)(p + c + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = a[e], v[4 + e] = b[e];
    } else {
      unsigned u[4];
      if constexpr (VEC) {
        const uint4 x = *(const uint4*)(p + c);
        u[0] = x.x, u[1] = x.y, u[2] = x.z, u[3] = x.w;
      } else {
        const u32x4_any_t x = *(const u32x4_any_t*)(p + c);
        u[0] = x[0], u[1] = x[1], u[2] = x[2], u[3] = x[3];
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) v[2 * e] = __uint_as_float(u[e] << 16), v[2 * e + 1] = __uint_as_float(u[e] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.f;
    if (!VEC && c < d) {                                         // all of them asked for: behind a condition each waits for the one before
      float w[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = DT<T>::ld(p + min(c + e, d - 1));
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = c + e < d ? w[e] : 0.f;
    }
  }
}
// The same where few rows ever come: one by one in place of unaligned vectors, whose registers and code all other rows would pay for.
template <typename T, bool VEC>
__device__ __forceinline__ void again8(const T* p, int c, int d, float (&v)[8]) {
  if constexpr (VEC) {
    load8<T, true>(p, c, d, v);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = c + e < d ? DT<T>::ld(p + c + e) : 0.f;
  }
}
template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* p, int c, int d, const float (&v)[8]) {
  if (VEC ? c < d : c + 8 <= d) {
    if constexpr (sizeof(T) == 4) {
      if constexpr (VEC) {
        *(float4*)(p + c) = make_float4(v[0], v[1], v[2], v[3]);
        *(float4*)(p + c + 4) = make_float4(v[4], v[5], v[6], v[7]);
      } else {
        *(floatx4_any_t*)(p + c) = floatx4_any_t{v[0], v[1], v[2], v[3]};
        *(floatx4_any_t*)(p + c + 4) = floatx4_any_t{v[4], v[5], v[6], v[7]};
      }
    } else {
      const unsigned a = pack2_bf16(v[0], v[1]), b = pack2_bf16(v[2], v[3]), e = pack2_bf16(v[4], v[5]), f = pack2_bf16(v[6], v[7]);
      if constexpr (VEC) *(uint4*)(p + c) = make_uint4(a, b, e, f);
      else *(u32x4_any_t*)(p + c) = u32x4_any_t{a, b, e, f};
    }
  } else if (!VEC) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c + e < d) DT<T>::st(p + c + e, v[e]);
  }
}
__device__ __forceinline__ unsigned size8(const float (&v)[8]) {
  unsigned m = fp8_size(v[0]);
#pragma unroll
  for (int e = 1; e < 8; ++e) m = max(m, fp8_size(v[e]));
  return m;
}
template <typename T>
__device__ __forceinline__ uint2 codes8(const float (&v)[8], const fp8_cut<T>& cut) {
  return make_uint2(fp8_pack4(cut(v[0]), cut(v[1]), cut(v[2]), cut(v[3])), fp8_pack4(cut(v[4]), cut(v[5]), cut(v[6]), cut(v[7])));
}

// One block of a row per 16 lanes.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256)
fp8_rows_kernel(const T* __restrict__ x, long long ldx, uint8_t* __restrict__ codes, long long ldc, float* __restrict__ scales,
                long long ss, long long sb, long long units, int blocks, int d) {
  const long long u = (long long)blockIdx.x * 16 + (threadIdx.x >> 4);
  const long long row = u < units ? u / blocks : 0;              // every lane takes part in the exchange
  const int b = u < units ? (int)(u - row * blocks) : 0, c = b * FP8_BLOCK + (int)(threadIdx.x & 15) * 8;
  float v[8];
  load8<T, VEC>(x + row * ldx, c, d, v);
  const float most = __uint_as_float(fp8_max16(size8(v)));
  if (u >= units) return;
  if (c < d) *(uint2*)(codes + row * ldc + c) = codes8(v, fp8_cut<T>(most));
  if ((threadIdx.x & 15) == 0) scales[row * ss + b * sb] = fp8_scale(most);
}

// W waves to a row, NV groups of 8 values to a lane.  The codes do not go by the root mean square, which is the same factor in a
// block's values and in its amax: they are those of x * w, whose products are exact for bf16, and only the scale takes the factor.
template <typename T, bool VEC, int W, int NV>
__global__ void __launch_bounds__(W == 1 ? 256 : W * 64)
fp8_rmsnorm_kernel(const T* x, long long ldx, const T* delta, long long ldd, T* xo, long long ldo,
                   const T* __restrict__ w, float eps, uint8_t* __restrict__ codes, long long ldc, float* __restrict__ scales, long long ss,
                   long long sb, int rows, int d) {
  constexpr int ROWS = W == 1 ? 4 : 1;
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  const int row = (int)blockIdx.x * ROWS + (W == 1 ? wv : 0);
  if (row >= rows) return;                                       // W > 1: never
  const int c0 = (W == 1 ? 0 : wv * 512) + lane * 8;
  float v[NV][8], g[NV][8], sum = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) load8<T, VEC>(x + (size_t)row * ldx, c0 + i * W * 512, d, v[i]);
  if (delta) {
#pragma unroll
    for (int i = 0; i < NV; ++i) load8<T, VEC>(delta + (size_t)row * ldd, c0 + i * W * 512, d, g[i]);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i][e] = DT<T>::rnd(v[i][e] + g[i][e]);     // the stream is held in its own type
      store8<T, VEC>(xo + (size_t)row * ldo, c0 + i * W * 512, d, v[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) load8<T, VEC>(w, c0 + i * W * 512, d, g[i]);
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) sum = fmaf(v[i][e], v[i][e], sum), v[i][e] *= g[i][e];
  __shared__ float part[2][W];
  const auto join = [&](float s, int turn) __attribute__((always_inline)) {     // over the lanes and waves of the row
    s = wave_sum(s);
    if constexpr (W > 1) {
      if (lane == 0) part[turn][wv] = s;
      __syncthreads();
      s = 0.f;
#pragma unroll
      for (int i = 0; i < W; ++i) s += part[turn][i];
    }
    return s;
  };
  const T* const src = delta ? xo + (size_t)row * ldo : x + (size_t)row * ldx;     // what is normed: a lane has read, or written, all that it reads here again
  float up = 1.f;
  sum = join(sum, 0);
  if (__builtin_expect(sum == __builtin_inff(), 0)) {                                 // squares beyond fp32 (values of 1e17 and more): those of 2^-80 of the values
    up = 0x1p-80f, sum = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      again8<T, VEC>(src, c0 + i * W * 512, d, g[i]);
#pragma unroll
      for (int e = 0; e < 8; ++e) g[i][e] *= up, sum = fmaf(g[i][e], g[i][e], sum);
    }
    sum = join(sum, 1);
  }
  const float rms = 1.0f / sqrtf(sum / (float)d + eps * up * up);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = c0 + i * W * 512;
    const float most = __uint_as_float(fp8_max16(size8(v[i])));
    float norm = most * up * rms;                                // amax of the normed values: NaN where one of them is not a number
    uint2 out;
    const bool none = (c & ~(FP8_BLOCK - 1)) >= d;                // a block behind the row's end: nothing of it is stored
    if (__builtin_expect(none || (norm >= FP8_LEAST && most >= FP8_LEAST && most < __builtin_inff()), 1)) {
      out = codes8(v[i], fp8_cut<T>(most, true));
    } else {
      // next to nothing, not a number, or products x * w beyond fp32's range whose normed values are not: these themselves, from the row as it was read
      again8<T, VEC>(src, c, d, v[i]);
      again8<T, VEC>(w, c, d, g[i]);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i][e] = v[i][e] * up * rms * g[i][e];
      norm = __uint_as_float(fp8_max16(size8(v[i])));            // all of the 16 lanes are here
      out = codes8(v[i], fp8_cut<float>(norm));
    }
    if (c < d) *(uint2*)(codes + (size_t)row * ldc + c) = out;
    if ((lane & 15) == 0 && c < d) scales[row * ss + (c >> 7) * sb] = fp8_scale(norm);
  }
}

// One block of 128 x 128 per workgroup: 64 values to a lane.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256)
fp8_weight_kernel(const T* __restrict__ w, long long ldw, uint8_t* __restrict__ codes, long long ldc, float* __restrict__ scales,
                  long long ss, long long sb, int N, int K) {
  __shared__ unsigned part[4];
  const int c = (int)blockIdx.x * FP8_BLOCK + (int)(threadIdx.x & 15) * 8, r0 = (int)blockIdx.y * FP8_BLOCK + (int)(threadIdx.x >> 4);
  float v[8][8];
  unsigned m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = r0 + 16 * i;
    load8<T, VEC>(w + (size_t)min(r, N - 1) * ldw, c, r < N ? K : 0, v[i]);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, size8(v[i]));
  m = fp8_max16(m);
  m = max(m, __float_as_uint(fstu_swz16(__uint_as_float(m))));
  m = max((unsigned)__builtin_amdgcn_readlane((int)m, 0), (unsigned)__builtin_amdgcn_readlane((int)m, 32));
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = m;
  __syncthreads();
  const float most = __uint_as_float(max(max(part[0], part[1]), max(part[2], part[3])));
  const fp8_cut<T> cut(most);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = r0 + 16 * i;
    if (r < N && c < K) *(uint2*)(codes + (size_t)r * ldc + c) = codes8(v[i], cut);
  }
  if (threadIdx.x == 0) scales[blockIdx.y * ss + blockIdx.x * sb] = fp8_scale(most);
}

bool whole16(const void* p, int64_t ld, int elem) { return !p || (fstu_aligned(p, 16) && ld * elem % 16 == 0); }

template <typename T, bool VEC, int W, int NV>
void rmsnorm_launch(const void* x, int64_t ldx, const void* delta, int64_t ldd, void* xo, int64_t ldo, const void* w, float eps, uint8_t* codes,
                    int64_t ldc, float* scales, int64_t ss, int64_t sb, int rows, int d, hipStream_t s) {
  hipLaunchKernelGGL((fp8_rmsnorm_kernel<T, VEC, W, NV>), dim3(W == 1 ? (rows + 3) / 4 : rows), dim3(W == 1 ? 256 : W * 64), 0, s, (const T*)x, ldx,
                     (const T*)delta, ldd, (T*)xo, ldo, (const T*)w, eps, codes, ldc, scales, ss, sb, rows, d);
}
template <typename T, bool VEC>
void rmsnorm_pick(const void* x, int64_t ldx, const void* delta, int64_t ldd, void* xo, int64_t ldo, const void* w, float eps, uint8_t* codes,
                  int64_t ldc, float* scales, int64_t ss, int64_t sb, int rows, int d, hipStream_t s) {
  const auto go = [&](auto f) { f(x, ldx, delta, ldd, xo, ldo, w, eps, codes, ldc, scales, ss, sb, rows, d, s); };
  // A lane takes one group of 8, a row the waves that this needs: more groups to a lane left fewer waves in flight.  us, bf16 with the addition,
  // groups to a wave / one: 8 x 2048 four 5.7 / 3.3, 1024 x 2048 6.7 / 4.9, 16384 x 2048 42.3 / 38.0, 16384 x 4096 two 90 / 86, 16384 x 8192 four
  // 200 / 167 (5000 61 / 52).  Up to 1024 columns many rows have waves enough: 1024 x 768 two 4.2 / 3.6, 2048 4.7 / 4.6, 8192 10.9 / 10.7, x 1024 12.8 / 13.2.
  if (d <= 512) go(rmsnorm_launch<T, VEC, 1, 1>);
  else if (d <= 1024 && rows <= 1024) go(rmsnorm_launch<T, VEC, 2, 1>);
  else if (d <= 1024) go(rmsnorm_launch<T, VEC, 1, 2>);
  else if (d <= 2048) go(rmsnorm_launch<T, VEC, 4, 1>);
  else if (d <= 4096) go(rmsnorm_launch<T, VEC, 8, 1>);
  else if (d <= 8192) go(rmsnorm_launch<T, VEC, 16, 1>);
  else go(rmsnorm_launch<T, VEC, 16, 4>);
}

}  // namespace

#define FP8_CODES_OK(name, codes, ldc, cols)                                                                        \
  FSTU_REQUIRE(fstu_aligned(codes, 16) && (ldc) % 16 == 0 && (ldc) >= (cols), FSTU_EALIGN,                          \
               name ": rows of codes must be 16-byte aligned, a multiple of 16 bytes apart and at least %d (stride %lld)", (int)(cols), (long long)(ldc))

extern "C" int fstu_fp8_quantize_rows(const void* x, int64_t ldx, uint8_t* codes, int64_t ldc, float* scales, int64_t ss, int64_t sb, int rows,
                                      int d, int dtype, void* stream) {
  FSTU_REQUIRE(x && codes && scales, FSTU_ENULL, "fstu_fp8_quantize_rows: null pointer");
  FSTU_REQUIRE(rows >= 1 && d >= 1 && (rows == 1 || ldx >= d), FSTU_ESHAPE, "fstu_fp8_quantize_rows: rows=%d d=%d ldx=%lld", rows, d, (long long)ldx);
  FP8_CODES_OK("fstu_fp8_quantize_rows", codes, ldc, d);
  const int blocks = (d + FP8_BLOCK - 1) / FP8_BLOCK;
  const long long units = (long long)rows * blocks;
  FSTU_REQUIRE((units + 15) / 16 <= 0xffffff, FSTU_ESHAPE, "fstu_fp8_quantize_rows: rows=%d d=%d", rows, d);
  FSTU_DISPATCH_DTYPE(dtype, "fstu_fp8_quantize_rows", {
    const dim3 grid((unsigned)((units + 15) / 16));
    if (d % 8 == 0 && whole16(x, ldx, sizeof(T)))
      hipLaunchKernelGGL((fp8_rows_kernel<T, true>), grid, dim3(256), 0, (hipStream_t)stream, (const T*)x, ldx, codes, ldc, scales, ss, sb, units, blocks, d);
    else
      hipLaunchKernelGGL((fp8_rows_kernel<T, false>), grid, dim3(256), 0, (hipStream_t)stream, (const T*)x, ldx, codes, ldc, scales, ss, sb, units, blocks, d);
  });
  FSTU_CHECK_LAUNCH("fstu_fp8_quantize_rows");
  return FSTU_OK;
}

extern "C" int fstu_fp8_rmsnorm(const void* x, int64_t ldx, const void* delta, int64_t ldd, void* x_out, int64_t ldo, const void* w, float eps,
                                uint8_t* codes, int64_t ldc, float* scales, int64_t ss, int64_t sb, int rows, int d, int dtype, void* stream) {
  FSTU_REQUIRE(x && w && codes && scales, FSTU_ENULL, "fstu_fp8_rmsnorm: null pointer");
  FSTU_REQUIRE(!delta == !x_out, FSTU_EARG, "fstu_fp8_rmsnorm: delta and x_out go together");
  FSTU_REQUIRE(rows >= 1 && d >= 1 && d <= 32768 && (rows == 1 || (ldx >= d && (!delta || (ldd >= d && ldo >= d)))), FSTU_ESHAPE,
               "fstu_fp8_rmsnorm: rows=%d d=%d (1..32768) ldx=%lld", rows, d, (long long)ldx);
  FP8_CODES_OK("fstu_fp8_rmsnorm", codes, ldc, d);
  FSTU_REQUIRE((long long)rows * (d <= 1024 ? 64 : d <= 2048 ? 256 : d <= 4096 ? 512 : 1024) <= 0xff000000LL, FSTU_ESHAPE, "fstu_fp8_rmsnorm: rows=%d d=%d", rows, d);
  const int bytes = dtype == FSTU_F32 ? 4 : 2;
  FSTU_REQUIRE(!delta || (fp8_same_or_apart(x, ldx, x_out, ldo, rows, d, bytes) && fp8_same_or_apart(delta, ldd, x_out, ldo, rows, d, bytes)), FSTU_EARG,
               "fstu_fp8_rmsnorm: x_out overlaps x or delta and is not the same rows");
  FSTU_DISPATCH_DTYPE(dtype, "fstu_fp8_rmsnorm", {
    const bool vec = d % 8 == 0 && whole16(x, ldx, sizeof(T)) && whole16(delta, ldd, sizeof(T)) && whole16(x_out, ldo, sizeof(T)) && fstu_aligned(w, 16);
    if (vec) rmsnorm_pick<T, true>(x, ldx, delta, ldd, x_out, ldo, w, eps, codes, ldc, scales, ss, sb, rows, d, (hipStream_t)stream);
    else rmsnorm_pick<T, false>(x, ldx, delta, ldd, x_out, ldo, w, eps, codes, ldc, scales, ss, sb, rows, d, (hipStream_t)stream);
  });
  FSTU_CHECK_LAUNCH("fstu_fp8_rmsnorm");
  return FSTU_OK;
}

extern "C" int fstu_fp8_quantize_weight(const void* w, int64_t ldw, uint8_t* codes, int64_t ldc, float* scales, int64_t ss, int64_t sb, int N, int K,
                                        int dtype, void* stream) {
  FSTU_REQUIRE(w && codes && scales, FSTU_ENULL, "fstu_fp8_quantize_weight: null pointer");
  FSTU_REQUIRE(N >= 1 && K >= 1 && (N == 1 || ldw >= K) && N <= 65535 * FP8_BLOCK, FSTU_ESHAPE, "fstu_fp8_quantize_weight: N=%d K=%d ldw=%lld", N, K, (long long)ldw);
  FP8_CODES_OK("fstu_fp8_quantize_weight", codes, ldc, K);
  const dim3 grid((K + FP8_BLOCK - 1) / FP8_BLOCK, (N + FP8_BLOCK - 1) / FP8_BLOCK);
  FSTU_DISPATCH_DTYPE(dtype, "fstu_fp8_quantize_weight", {
    if (K % 8 == 0 && whole16(w, ldw, sizeof(T)))
      hipLaunchKernelGGL((fp8_weight_kernel<T, true>), grid, dim3(256), 0, (hipStream_t)stream, (const T*)w, ldw, codes, ldc, scales, ss, sb, N, K);
    else
      hipLaunchKernelGGL((fp8_weight_kernel<T, false>), grid, dim3(256), 0, (hipStream_t)stream, (const T*)w, ldw, codes, ldc, scales, ss, sb, N, K);
  });
  FSTU_CHECK_LAUNCH("fstu_fp8_quantize_weight");
  return FSTU_OK;
}
