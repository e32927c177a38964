// Products of 8-bit codes with a scale for each block of 128 (fstu_fp8.h):
//   y[m, n] = sum_b xs[m, b] ws[n / 128, b] sum_{k in block b} x[m, k] w[n, k]
// for activations x (M rows, K contiguous, a scale for each 128 values of a row) and weights w (N, K) (a scale for each 128 x 128).
// A block's inner sum starts from zero; its results times the block's two scales are added in fp32.  The weights are the A operand, so that
// a lane ends up with 4 consecutive features of one row: its results share one row's scale.  A lane's 32 bytes of an operand are the chunks
// of 16 bytes q and 4 + q of the block (q = lane / 16): any split will do that is the same for both operands.
// The inner sum goes by the type of the result:
//   bf16  one v_mfma_f32_16x16x128_f8f6f4.  Its products are exact and its sum is held in 32 bits, but the few products that one step of
//         it adds are first lined up with the largest of them and cut 13 bits below: 2^16 + 2^3 is kept, 2^16 + 2^2 is not, eight places apart
//         both are.  Measured on random codes: 1.4e-5 of the result (2-norm) where a block's values are of one size, 5e-5 where they differ by
//         orders; the result's own rounding is 1.7e-3, the codes' 2.6e-2.  v_mfma_f32_16x16x32_fp8_fp8 gives the same values at a third of the rate.
//   fp32  the codes widened to bf16, which holds them, and four v_mfma_f32_16x16x32_bf16: 1e-8 to 7e-8, at half the rate.
//   linear  y = T( acc + bias + residual )                 (down_proj and the add behind it, flash_stu/modules/swiglu.py:27)
//   glu     y = T( gelu_tanh(gate) * up )                  (swiglu.py:23-26), or codes and scales of that y (bf16), as
//           fstu_fp8_quantize_rows makes them of it
#include <algorithm>
#include "fstu_fp8.h"

namespace {

typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef int i32x8_t __attribute__((ext_vector_type(8)));
typedef float floatx4_t __attribute__((ext_vector_type(4)));
typedef unsigned u32x4_t __attribute__((ext_vector_type(4)));
struct Frag32 { u32x4_t lo, hi; };

// An operand: codes, and scales of stride sr between rows (weights: blocks of 128 rows) and sb between blocks of K.
struct Codes {
  const uint8_t* p;
  long long ld;
  const float* s;
  long long sr, sb;
};
// Where a product leaves: y; linear: bias and residual; glu: with s not null codes (y) and scales.
struct Leave {
  void* y;
  long long ldy;
  const void *bias, *res;
  long long ldr;
  float* s;
  long long sr, sb;
};

// Eight codes as bf16.
__device__ __forceinline__ bf16x8_t widen8(unsigned a, unsigned b) {
  const bf16x2_t v0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, false), v1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, true);
  const bf16x2_t v2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, false), v3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, true);
  return bf16x8_t{v0[0], v0[1], v1[0], v1[1], v2[0], v2[1], v3[0], v3[1]};
}
// A fragment as the instruction of the result's type takes it, and a block's inner sum.
template <typename T> struct Operand;
template <> struct Operand<bf16_t> {
  i32x8_t v;
  __device__ __forceinline__ explicit Operand(const Frag32& f) : v(__builtin_bit_cast(i32x8_t, f)) {}
  static __device__ __forceinline__ floatx4_t sum(const Operand& w, const Operand& x) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w.v, x.v, floatx4_t{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
  }
};
template <> struct Operand<float> {
  bf16x8_t v[4];
  __device__ __forceinline__ explicit Operand(const Frag32& f)
      : v{widen8(f.lo[0], f.lo[1]), widen8(f.lo[2], f.lo[3]), widen8(f.hi[0], f.hi[1]), widen8(f.hi[2], f.hi[3])} {}
  static __device__ __forceinline__ floatx4_t sum(const Operand& w, const Operand& x) {
    floatx4_t d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; ++i) d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.v[i], x.v[i], d, 0, 0, 0);
    return d;
  }
};
// The bytes of a 16-byte chunk that lie before the end: `left` of them (none where negative).
__device__ __forceinline__ u32x4_t cut16(u32x4_t v, int left) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int n = left - 4 * e;
    v[e] = n >= 4 ? v[e] : n <= 0 ? 0u : v[e] & ((1u << (8 * n)) - 1u);
  }
  return v;
}
// A chunk of 16 bytes from byte k of a row of K.  A row's last chunk is read whole: rows are 16-byte aligned, so that it lies in the
// 16 bytes whose first the row has.
__device__ __forceinline__ u32x4_t chunk16(const uint8_t* row, int k, int K) {
  if (k >= K) return u32x4_t{0, 0, 0, 0};
  return cut16(*(const u32x4_t*)(row + k), K - k);
}
// The tanh-approximated GELU, x (1 + tanh t) / 2 = x / (1 + exp(-2 t)), on the hardware exp and reciprocal.
__device__ __forceinline__ float gelu_tanh_exp(float x) {
  return x * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * fmaf(x * x, -0.10294324f, -2.3022082f)));
}

// 128 features x 64 rows per workgroup, 16 features (GLU: of both matrices) x 64 rows per wave; operands straight from global memory.
template <bool GLU, typename T>
__global__ void __launch_bounds__(512)
fp8_plain_kernel(Codes X, Codes W, Codes U, Leave o, int M, int N, int K) {
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, l16 = lane & 15, q = lane >> 4;
  const int n0 = (int)blockIdx.x * 128, m0 = (int)blockIdx.y * 64;
  const uint8_t* const wr = W.p + (size_t)min(n0 + wv * 16 + l16, N - 1) * W.ld;
  const uint8_t* const ur = GLU ? U.p + (size_t)min(n0 + wv * 16 + l16, N - 1) * U.ld : nullptr;
  floatx4_t acc[4], acu[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) acc[j] = acu[j] = floatx4_t{0.f, 0.f, 0.f, 0.f};
  const int nb = (K + 127) / 128;
  for (int b = 0; b < nb; ++b) {
    const int k = b * 128 + q * 16;
    const Operand<T> w(Frag32{chunk16(wr, k, K), chunk16(wr, k + 64, K)});
    const Operand<T> u(GLU ? Frag32{chunk16(ur, k, K), chunk16(ur, k + 64, K)} : Frag32{});
    const float sw = W.s[blockIdx.x * W.sr + b * W.sb], su = GLU ? U.s[blockIdx.x * U.sr + b * U.sb] : 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int m = min(m0 + j * 16 + l16, M - 1);
      const uint8_t* const xr = X.p + (size_t)m * X.ld;
      const Operand<T> x(Frag32{chunk16(xr, k, K), chunk16(xr, k + 64, K)});
      const float sx = X.s[m * X.sr + b * X.sb];
      const floatx4_t d = Operand<T>::sum(w, x);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[j][e] = fmaf(d[e], sx * sw, acc[j][e]);
      if constexpr (GLU) {
        const floatx4_t f = Operand<T>::sum(u, x);
#pragma unroll
        for (int e = 0; e < 4; ++e) acu[j][e] = fmaf(f[e], sx * su, acu[j][e]);
      }
    }
  }
  const int f0 = n0 + wv * 16 + q * 4;                    // this lane's features of row l16 of every row tile
  if constexpr (GLU) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[j][e] = f0 + e < N ? DT<T>::rnd(gelu_tanh_exp(acc[j][e]) * acu[j][e]) : 0.f;
    if (o.s) {
      __shared__ unsigned part[8][64];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        unsigned m = max(max(fp8_size(acc[j][0]), fp8_size(acc[j][1])), max(fp8_size(acc[j][2]), fp8_size(acc[j][3])));
        m = max(m, (unsigned)__shfl_xor((int)m, 16));
        m = max(m, (unsigned)__shfl_xor((int)m, 32));
        if (q == 0) part[wv][j * 16 + l16] = m;
      }
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        unsigned bits = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) bits = max(bits, part[i][j * 16 + l16]);
        const float most = __uint_as_float(bits), times = fp8_times(most);
        const int m = m0 + j * 16 + l16;
        if (m < M && f0 < N)                                // a row's codes lie in whole 16 bytes: zeros behind the last feature
          *(unsigned*)((uint8_t*)o.y + (size_t)m * o.ldy + f0) = fp8_pack4(acc[j][0] * times, acc[j][1] * times, acc[j][2] * times, acc[j][3] * times);
        if (m < M && wv == 0 && q == 0) o.s[m * o.sr + blockIdx.x * o.sb] = fp8_scale(most);
      }
      return;
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int m = m0 + j * 16 + l16;
    if (m >= M) continue;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int f = f0 + e;
      if (f >= N) break;
      float v = acc[j][e];
      if (!GLU && o.bias) v += DT<T>::ld((const T*)o.bias + f);
      if (!GLU && o.res) v += DT<T>::ld((const T*)o.res + (size_t)m * o.ldr + f);
      DT<T>::st((T*)o.y + (size_t)m * o.ldy + f, v);
    }
  }
}

}  // namespace

#define FP8_OPERAND(name, c, rows, what)                                                                                         \
  FSTU_REQUIRE((c).p && (c).s, FSTU_ENULL, name ": null pointer");                                                               \
  FSTU_REQUIRE(fstu_aligned((c).p, 16) && (c).ld % 16 == 0 && (c).ld >= ((rows) > 1 ? K : 0), FSTU_EALIGN,                       \
               name ": rows of " what " must be 16-byte aligned, a multiple of 16 bytes apart and at least K=%d (stride %lld)", K, (long long)(c).ld)

extern "C" int fstu_fp8_linear(const uint8_t* x, int64_t ldx, const float* xs, int64_t xs_row, int64_t xs_blk, const uint8_t* w, int64_t ldw,
                               const float* ws, int64_t ws_row, int64_t ws_blk, const void* bias, const void* res, int64_t ldr, void* y, int64_t ldy,
                               int M, int N, int K, int dtype, void* stream) {
  const Codes X = {x, ldx, xs, xs_row, xs_blk}, W = {w, ldw, ws, ws_row, ws_blk};
  FSTU_REQUIRE(y, FSTU_ENULL, "fstu_fp8_linear: null pointer");
  FSTU_REQUIRE(M >= 1 && N >= 1 && K >= 1 && M <= 65535 * 64, FSTU_ESHAPE, "fstu_fp8_linear: M=%d N=%d K=%d", M, N, K);
  FP8_OPERAND("fstu_fp8_linear", X, M, "x");
  FP8_OPERAND("fstu_fp8_linear", W, N, "w");
  FSTU_REQUIRE(M == 1 || (ldy >= N && (!res || ldr >= N)), FSTU_ESHAPE, "fstu_fp8_linear: N=%d ldy=%lld ldr=%lld", N, (long long)ldy, (long long)ldr);
  const Leave o = {y, ldy, bias, res, ldr, nullptr, 0, 0};
  FSTU_DISPATCH_DTYPE(dtype, "fstu_fp8_linear", {
    hipLaunchKernelGGL((fp8_plain_kernel<false, T>), dim3((N + 127) / 128, (M + 63) / 64), dim3(512), 0, (hipStream_t)stream, X, W, W, o, M, N, K);
  });
  FSTU_CHECK_LAUNCH("fstu_fp8_linear");
  return FSTU_OK;
}

extern "C" int fstu_fp8_glu(const uint8_t* x, int64_t ldx, const float* xs, int64_t xs_row, int64_t xs_blk, const uint8_t* gate, int64_t ldg,
                            const float* gs, int64_t gs_row, int64_t gs_blk, const uint8_t* up, int64_t ldu, const float* us, int64_t us_row,
                            int64_t us_blk, void* y, int64_t ldy, float* scales, int64_t ss, int64_t sb, int M, int N, int K, int dtype, void* stream) {
  const Codes X = {x, ldx, xs, xs_row, xs_blk}, W = {gate, ldg, gs, gs_row, gs_blk}, U = {up, ldu, us, us_row, us_blk};
  FSTU_REQUIRE(y, FSTU_ENULL, "fstu_fp8_glu: null pointer");
  FSTU_REQUIRE(M >= 1 && N >= 1 && K >= 1 && M <= 65535 * 64, FSTU_ESHAPE, "fstu_fp8_glu: M=%d N=%d K=%d", M, N, K);
  FP8_OPERAND("fstu_fp8_glu", X, M, "x");
  FP8_OPERAND("fstu_fp8_glu", W, N, "the gate");
  FP8_OPERAND("fstu_fp8_glu", U, N, "the up weight");
  FSTU_REQUIRE(M == 1 || ldy >= N, FSTU_ESHAPE, "fstu_fp8_glu: N=%d ldy=%lld", N, (long long)ldy);
  FSTU_REQUIRE(!scales || dtype == FSTU_BF16, FSTU_EDTYPE, "fstu_fp8_glu: codes are those of the bf16 result (dtype %d)", dtype);
  FSTU_REQUIRE(!scales || (fstu_aligned(y, 16) && ldy % 16 == 0 && ldy >= N), FSTU_EALIGN,
               "fstu_fp8_glu: rows of codes must be 16-byte aligned, a multiple of 16 bytes apart and at least %d (stride %lld)", N, (long long)ldy);
  const Leave o = {y, ldy, nullptr, nullptr, 0, scales, ss, sb};
  FSTU_DISPATCH_DTYPE(dtype, "fstu_fp8_glu", {
    hipLaunchKernelGGL((fp8_plain_kernel<true, T>), dim3((N + 127) / 128, (M + 63) / 64), dim3(512), 0, (hipStream_t)stream, X, W, U, o, M, N, K);
  });
  FSTU_CHECK_LAUNCH("fstu_fp8_glu");
  return FSTU_OK;
}
