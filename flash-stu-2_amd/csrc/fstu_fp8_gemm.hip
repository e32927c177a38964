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
#include <type_traits>
#include <utility>
#include "fstu_fp8.h"
#include "fstu_fp8_plan.h"

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
// A chunk of 16 bytes from byte k of a row of K (behind its end zeros, and its last chunk is read in their place).  A row's last chunk is
// read whole: rows are 16-byte aligned, so that it lies in the 16 bytes whose first the row has.
__device__ __forceinline__ u32x4_t chunk16(const uint8_t* row, int k, int K) {
  return cut16(*(const u32x4_t*)(row + min(k, max(K - 1, 0) & ~15)), K - k);
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
  for (int it = 0; it < nb + (K % 16 != 0); ++it) {      // a row's last chunk, where it is no whole one, by itself, as on the tiles
    const int b = min(it, nb - 1), end = it < nb ? K & ~15 : K, k = it < nb ? b * 128 + q * 16 : (K & ~15) + q * 16;
    const Operand<T> w(Frag32{chunk16(wr, k, end), chunk16(wr, k + 64, end)});
    const Operand<T> u(GLU ? Frag32{chunk16(ur, k, end), chunk16(ur, k + 64, end)} : Frag32{});
    const float sw = W.s[blockIdx.x * W.sr + b * W.sb], su = GLU ? U.s[blockIdx.x * U.sr + b * U.sb] : 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int m = min(m0 + j * 16 + l16, M - 1);
      const uint8_t* const xr = X.p + (size_t)m * X.ld;
      const Operand<T> x(Frag32{chunk16(xr, k, end), chunk16(xr, k + 64, end)});
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
        const float most = __uint_as_float(bits);
        const fp8_cut<bf16_t> cut(most);
        const int m = m0 + j * 16 + l16;
        if (m < M && f0 < N)                                // a row's codes lie in whole 16 bytes: zeros behind the last feature
          *(unsigned*)((uint8_t*)o.y + (size_t)m * o.ldy + f0) = fp8_pack4(cut(acc[j][0]), cut(acc[j][1]), cut(acc[j][2]), cut(acc[j][3]));
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


// ---------------------------------------------------------------- 256 x 256 tiles in two alternating wave groups
// Many rows, results in bf16.  A workgroup of 8 waves owns 256 features (glu: 128 of the gate and 128 of the up weight) x 256 rows, K in blocks
// of 128 through two LDS stages.  Waves 0-3 and 4-7 (one of each on every SIMD) run the same program half a phase apart: while one
// group multiplies, the other reads its next fragments and requests the blocks to come, so that a SIMD's matrix core always has one of its
// two waves to work for.  The halves of the weight tile (W0, W1: 128 features) and of the activation tile (X0, X1: 128 rows) are parts
// of 16 KB; a wave owns 32 features of each W half and 64 rows of each X half, and a block is two phases of 16
// v_mfma_f32_16x16x128_f8f6f4 (512 cycles), whose results are scaled and added (64 v_fma, 256 cycles) behind the next products:
//   phase  fragments read               multiplied      requested
//   0      W0, W1, X0 and scales of kt  (W0, W1) X0     X1 of kt + 1
//   1      X1 and its scales of kt      (W0, W1) X1     W0, W1, X0 and scales of kt + 2
// A part is requested in the first phase after its last readers have left it (their reads are complete before the barrier that ends a memory
// phase) and waited for three phases later: vmcnt(9) at the end of a memory phase leaves the two youngest requests (2 and 7
// instructions) in flight.  Scales have three stages, since a block's are read in both of its phases.
// LDS rows are 128 bytes with the 16-byte chunk index XOR-ed with bits of the row, so that neither fills nor fragment reads meet bank
// conflicts.  The W rows are dealt so that a lane ends up with 8 consecutive features of a row, which leave straight from the accumulators.
// Workgroup ids are dealt round-robin to the 8 XCDs; each XCD works through its own share of the tiles in panels of 8 feature tiles, and
// a workgroup requests the first blocks of its next tile before it stores this one.
// 16384 x 2048 x 24576 620 us (2.66 PFLOP/s; a library's 8-bit product of 8192^3 2.71), the pair 16384 x 2 x 24576 x 2048 1385 us (2.38), 4096 x 2 x 9216 x
// 768 64 to 70: the matrix cores are busy for 70 % of the cycles (pair 54 %: a tile's GELU takes 5.5 us) at the 1.8 GHz that the power leaves
// (all zeros 482 us instead of 620).  v_mfma_f32_32x32x64_f8f6f4, twice the products for the same fragments, behind sums of 16 registers: 686 and
// 72; a phase's last sums moved behind its barrier: 628 and 64; half of the GELU beside the last block's products: the pair 69.
#define F8_PANEL 8
#define F8_AHEAD 3                                // products that are on their way when one is scaled and added
#define F8_PART 16384u
#define F8_STAGE 65536u
#define F8_SCALES (2 * F8_STAGE)                  // three stages of 2 KB: by wave the scales of 32 rows, then the two weights' in wave 0's
#define F8_MAXIMA (F8_SCALES + 3 * 2048u)         // codes: the largest of a wave's 32 features of each row
#define F8_LDS(CODES) (F8_MAXIMA + ((CODES) ? 4096u : 0u))
#define F8_MAX_LD (1 << 23)                       // 256 rows of it are what a 32-bit offset covers

typedef __amdgpu_buffer_rsrc_t rsrc_t;
__device__ __forceinline__ rsrc_t make_rsrc(const void* p, size_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (unsigned)bytes, 0x00020000);
}
// 16 bytes per lane from global memory into 64 consecutive slots of LDS without a stop in registers; zeros behind the range
__device__ __forceinline__ void fill16(rsrc_t rs, unsigned voff, unsigned soff, void* l) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)l, 16, voff, soff, 0, 0);
}
__device__ __forceinline__ void fill4(const float* p, void* l) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)p, (__attribute__((address_space(3))) void*)l, 4, 0, 0);
}
__device__ __forceinline__ unsigned lds_addr(const void* p) { return (unsigned)(size_t)(const __attribute__((address_space(3))) void*)p; }
// LDS reads are written as asm: the compiler orders every one it knows of behind all outstanding fills.  Each is waited for below, before any use;
// that nothing (a spill, a copy) touches its registers before is held by a test of the built code (tests/test_fp8_registers_cpu.py).
template <int OFF>
__device__ __forceinline__ u32x4_t lds16(unsigned addr) {
  u32x4_t v;
  asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(v) : "v"(addr), "n"(OFF));
  return v;
}
template <int OFF>
__device__ __forceinline__ float lds4(unsigned addr) {
  float v;
  asm volatile("ds_read_b32 %0, %1 offset:%2" : "=v"(v) : "v"(addr), "n"(OFF));
  return v;
}

// 8 consecutive features of a row, at any element's alignment
typedef unsigned u32x4_any_t __attribute__((ext_vector_type(4), aligned(2)));
typedef float floatx4_any_t __attribute__((ext_vector_type(4), aligned(4)));
template <typename T> struct Put;
template <> struct Put<bf16_t> {
  typedef u32x4_any_t Eight;
  static __device__ __forceinline__ void put(bf16_t* p, const float (&v)[8]) {
    *(Eight*)p = Eight{pack2_bf16(v[0], v[1]), pack2_bf16(v[2], v[3]), pack2_bf16(v[4], v[5]), pack2_bf16(v[6], v[7])};
  }
  static __device__ __forceinline__ void add(float (&v)[8], Eight r) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[2 * e] += __uint_as_float(r[e] << 16), v[2 * e + 1] += __uint_as_float(r[e] & 0xffff0000u);
  }
};
template <> struct Put<float> {
  struct Eight { floatx4_any_t a, b; };
  static __device__ __forceinline__ void put(float* p, const float (&v)[8]) {
    *(floatx4_any_t*)p = floatx4_any_t{v[0], v[1], v[2], v[3]};
    *(floatx4_any_t*)(p + 4) = floatx4_any_t{v[4], v[5], v[6], v[7]};
  }
  static __device__ __forceinline__ void add(float (&v)[8], const Eight& r) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] += r.a[e], v[4 + e] += r.b[e];
  }
};
// the last features of a row, fewer than 8
__device__ __forceinline__ void put_some(bf16_t* p, const float (&v)[8], int left) {
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (e < left) p[e] = f32_to_bf16(v[e]);
}
__device__ __forceinline__ void add_some(float (&v)[8], const bf16_t* p, int left) {
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (e < left) v[e] += bf16_to_f32(p[e]);
}

// MODE 0 linear, 1 glu, 2 glu as codes.  K a multiple of 16; TAIL: not one of 128, the last block's chunks behind K are asked for behind the
// range, where a fill finds zeros.
template <int MODE, bool TAIL>
__global__ void __launch_bounds__(512)
fp8_large_kernel(Codes X, Codes W, Codes U, Leave o, int M, int N, int K, int mt, int nt, int share) {
  constexpr bool GLU = MODE != 0;
  constexpr int NF = GLU ? 128 : 256;
  extern __shared__ __align__(16) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int per_panel = mt * F8_PANEL, xcd = (int)(blockIdx.x & 7) * share, tiles = mt * nt;
  int idx = (int)(blockIdx.x >> 3);                    // this workgroup's next tile in its XCD's share
  if (idx >= share || xcd + idx >= tiles) return;
  const int nkt = (K + 127) >> 7;
  int m0, n0;
  unsigned wbytes, ubytes, xbytes;
  const uint8_t *wb, *ub, *xb;
  const float* sp;                                     // this lane's scale of block 0: a row's, or one of the two weights'
  const long long sstep = lane < 32 ? X.sb : GLU && (lane & 1) ? U.sb : W.sb;
  const auto open = [&]() __attribute__((always_inline)) {
    const int t = xcd + idx, panel = t / per_panel, in_panel = t - panel * per_panel, pw = min(F8_PANEL, nt - panel * F8_PANEL);
    m0 = in_panel / pw * 256;
    n0 = (panel * F8_PANEL + in_panel % pw) * NF;
    wbytes = (unsigned)(min(NF, N - n0) - 1) * (unsigned)W.ld + (unsigned)K;
    ubytes = GLU ? (unsigned)(min(NF, N - n0) - 1) * (unsigned)U.ld + (unsigned)K : wbytes;
    xbytes = (unsigned)(min(256, M - m0) - 1) * (unsigned)X.ld + (unsigned)K;
    wb = W.p + (size_t)n0 * W.ld;
    ub = GLU ? U.p + (size_t)n0 * U.ld : wb;
    xb = X.p + (size_t)m0 * X.ld;
    const int b = n0 >> 7, last = (N - 1) >> 7;
    sp = lane < 32 ? X.s + (long long)min(m0 + wv * 32 + lane, M - 1) * X.sr
                   : GLU ? (lane & 1 ? U.s + b * U.sr : W.s + b * W.sr) : W.s + min(b + (lane & 1), last) * W.sr;
  };
  const int wn = wv & 3, wm = wv >> 2;                 // 32-feature slice and 64-row slice of every half
  // ---- fills: a part is 128 rows x 128 bytes, a wave fills 16 of them with two instructions.  SPREAD: 8 rows of either half of it, so that what
  // differs between the two is the same for all lanes and goes into the descriptors, whose ranges end where the tile's rows do (a lane keeps one
  // offset for an operand instead of two; 16384 x 2048 x 2048 78.5 -> 77.6 us, x 2064 88.9 -> 84.8, the pair 4096 x 9216 x 784 91.5 -> 82.6).  The pair
  // in whole blocks has registers enough and is faster on 16 rows in line: 4096 x 9216 x 768 69.4 us, 71.0 spread.
  constexpr bool SPREAD = TAIL || !GLU;
  unsigned wvoff[2], uvoff[2], xvoff[2];
  bool wthere[2], xthere[2];                           // whether this lane's chunk of the last block is one of K's
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int row = SPREAD ? wv * 8 + (lane >> 3) : wv * 16 + j * 8 + (lane >> 3), feat = GLU ? row : (row & 31) + 2 * (row & 32);
    const unsigned wch = (unsigned)((lane & 7) ^ (((row >> 1) & 1) | ((row >> 2) & 6))) * 16u, xch = (unsigned)((lane & 7) ^ ((row >> 1) & 7)) * 16u;
    wvoff[j] = (unsigned)feat * (unsigned)W.ld + wch;
    uvoff[j] = GLU ? (unsigned)feat * (unsigned)U.ld + wch : wvoff[j];
    xvoff[j] = (unsigned)row * (unsigned)X.ld + xch;
    wthere[j] = (nkt - 1) * 128 + (int)wch < K, xthere[j] = (nkt - 1) * 128 + (int)xch < K;
  }
  unsigned char* const fill0 = smem + (unsigned)wv * (SPREAD ? 1024u : 2048u);
  constexpr unsigned SECOND = SPREAD ? 8192 : 1024;
  // beyond the last block the descriptors are empty and the scales the last block's: into stages that nobody reads
  const auto fetch = [&](int kt, const uint8_t* base, unsigned bytes, unsigned skip, unsigned voff, bool there, unsigned to) __attribute__((always_inline)) {
    const rsrc_t rs = make_rsrc(base + skip, kt < nkt && bytes > skip ? bytes - skip : 0);
    fill16(rs, TAIL && kt == nkt - 1 && !there ? 0x80000000u : voff, (unsigned)kt * 128u, fill0 + to);
  };
  const auto fetch_w = [&](int kt, unsigned stage) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < 2; ++j) fetch(kt, wb, wbytes, SPREAD ? (unsigned)(j * NF / 2) * (unsigned)W.ld : 0u, wvoff[j], wthere[j], stage + j * SECOND);
#pragma unroll
    for (int j = 0; j < 2; ++j)
      fetch(kt, ub, ubytes, !SPREAD ? 0u : GLU ? (unsigned)(j * 64) * (unsigned)U.ld : (unsigned)(j * 128 + 32) * (unsigned)W.ld, uvoff[j], wthere[j],
            stage + F8_PART + j * SECOND);
  };
  const auto fetch_x = [&](int kt, unsigned stage, int h) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
      fetch(kt, xb, xbytes, (unsigned)(h * 128 + (SPREAD ? j * 64 : 0)) * (unsigned)X.ld, xvoff[j], xthere[j], stage + (2 + h) * F8_PART + j * SECOND);
  };
  const auto fetch_s = [&](int kt, unsigned third) __attribute__((always_inline)) {
    fill4(sp + (long long)min(kt, nkt - 1) * sstep, smem + F8_SCALES + third + (unsigned)wv * 256u);
  };

  const int l16 = lane & 15, lq = lane >> 4;
  unsigned fw[2], fx[2];                               // fragment addresses of a block's two halves inside a part
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int rw = wn * 32 + 8 * (l16 >> 2) + (l16 & 3), rx = wm * 64 + l16, c = h * 4 + lq;
    fw[h] = lds_addr(smem) + (unsigned)rw * 128u + (unsigned)((c ^ (((rw >> 1) & 1) | ((rw >> 2) & 6))) << 4);
    fx[h] = lds_addr(smem) + 2 * F8_PART + (unsigned)rx * 128u + (unsigned)((c ^ ((rx >> 1) & 7)) << 4);
  }
  const unsigned fs = lds_addr(smem) + F8_SCALES + (unsigned)wm * 512u + (unsigned)l16 * 4u;    // rows 64 wm + l16: waves 2 wm and 2 wm + 1 filled them
  const unsigned fsw = lds_addr(smem) + F8_SCALES + 128u + (GLU ? 0u : (unsigned)(wn >> 1) * 4u);
  Frag32 wa[4], xf[4];                                 // [W half, feature tile], [row tile]
  float sx[4], sw, su = 0.f;
  floatx4_t acc[4][2][4];                              // [W half, feature tile][X half][row tile]
  bool young = false;
  constexpr int STORES = 8;                            // a whole tile's stores, at the least
  const auto landed = [&]() __attribute__((always_inline)) {    // all but the 9 youngest fills; the stores of the tile before are younger than what is waited for
    if (young) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(9 + STORES) : "memory");
    else asm volatile("s_waitcnt vmcnt(9)" ::: "memory");
  };
  const auto read_x = [&](unsigned stage, unsigned third, auto half) __attribute__((always_inline)) {
    constexpr int H = decltype(half)::value;
    xf[0] = Frag32{lds16<H * 16384>(fx[0] + stage), lds16<H * 16384>(fx[1] + stage)};
    xf[1] = Frag32{lds16<H * 16384 + 2048>(fx[0] + stage), lds16<H * 16384 + 2048>(fx[1] + stage)};
    xf[2] = Frag32{lds16<H * 16384 + 4096>(fx[0] + stage), lds16<H * 16384 + 4096>(fx[1] + stage)};
    xf[3] = Frag32{lds16<H * 16384 + 6144>(fx[0] + stage), lds16<H * 16384 + 6144>(fx[1] + stage)};
    sx[0] = lds4<H * 1024>(fs + third);
    sx[1] = lds4<H * 1024 + 64>(fs + third);
    sx[2] = lds4<H * 1024 + 256>(fs + third);
    sx[3] = lds4<H * 1024 + 320>(fs + third);
  };
  // end of a memory phase: this wave's reads are complete, its share of the parts that the next phase reads has landed
  const auto memory_end = [&]() __attribute__((always_inline)) {
    landed();
    asm volatile("s_waitcnt lgkmcnt(0)"
                 : "+v"(xf[0].lo), "+v"(xf[0].hi), "+v"(xf[1].lo), "+v"(xf[1].hi), "+v"(xf[2].lo), "+v"(xf[2].hi), "+v"(xf[3].lo), "+v"(xf[3].hi),
                   "+v"(wa[0].lo), "+v"(wa[0].hi), "+v"(wa[1].lo), "+v"(wa[1].hi), "+v"(wa[2].lo), "+v"(wa[2].hi), "+v"(wa[3].lo), "+v"(wa[3].hi),
                   "+v"(sx[0]), "+v"(sx[1]), "+v"(sx[2]), "+v"(sx[3]), "+v"(sw), "+v"(su)::"memory");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
  };
  const auto multiply = [&](auto half) __attribute__((always_inline)) {
    constexpr int H = decltype(half)::value;
    __builtin_amdgcn_s_setprio(1);
    float f[4], g[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = sx[j] * sw, g[j] = GLU ? sx[j] * su : f[j];
    floatx4_t d[16];
#pragma unroll
    for (int t = 0; t < 16 + F8_AHEAD; ++t) {
      if (t < 16) d[t] = Operand<bf16_t>::sum(Operand<bf16_t>(wa[t >> 2]), Operand<bf16_t>(xf[t & 3]));
      if (t >= F8_AHEAD) {
        const int p = t - F8_AHEAD, i = p >> 2, j = p & 3;
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][H][j][e] = fmaf(d[p][e], GLU && i >= 2 ? g[j] : f[j], acc[i][H][j][e]);
      }
      __builtin_amdgcn_sched_barrier(0);               // in this order: left to itself the compiler puts each sum right behind its product
    }
    __builtin_amdgcn_s_setprio(0);
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
  };
  const auto first = [&]() __attribute__((always_inline)) {
    fetch_w(0, 0), fetch_x(0, 0, 0), fetch_s(0, 0), fetch_x(0, 0, 1);
    fetch_w(1, F8_STAGE), fetch_x(1, F8_STAGE, 0), fetch_s(1, 2048);
  };
  open();
  first();
  for (;;) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[i][j >> 2][j & 3] = floatx4_t{0.f, 0.f, 0.f, 0.f};
    landed();                                          // W0, W1, X0 and scales of block 0
    __builtin_amdgcn_s_barrier();
    if (wm) __builtin_amdgcn_s_barrier();              // the second group runs half a phase later
    __builtin_amdgcn_sched_barrier(0);
    unsigned stage = 0, third = 0;
    for (int kt = 0; kt < nkt; ++kt) {
      const unsigned two = third == 0 ? 4096u : third - 2048u;       // the stage of block kt + 2's scales
      wa[0] = Frag32{lds16<0>(fw[0] + stage), lds16<0>(fw[1] + stage)};
      wa[1] = Frag32{lds16<512>(fw[0] + stage), lds16<512>(fw[1] + stage)};
      wa[2] = Frag32{lds16<16384>(fw[0] + stage), lds16<16384>(fw[1] + stage)};
      wa[3] = Frag32{lds16<16384 + 512>(fw[0] + stage), lds16<16384 + 512>(fw[1] + stage)};
      sw = lds4<0>(fsw + third);
      if constexpr (GLU) su = lds4<4>(fsw + third);
      read_x(stage, third, std::integral_constant<int, 0>{});
      fetch_x(kt + 1, F8_STAGE - stage, 1);
      memory_end();
      multiply(std::integral_constant<int, 0>{});
      young = false;
      read_x(stage, third, std::integral_constant<int, 1>{});
      fetch_w(kt + 2, stage), fetch_x(kt + 2, stage, 0), fetch_s(kt + 2, two);
      memory_end();
      multiply(std::integral_constant<int, 1>{});
      stage = F8_STAGE - stage;
      third = third == 4096u ? 0u : third + 2048u;
    }
    if (!wm) __builtin_amdgcn_s_barrier();
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the empty fills behind the last block
    __builtin_amdgcn_s_barrier();
    // every wave has left the stages: the next tile's first blocks are on their way while this one is stored
    const int em0 = m0, en0 = n0;
    const bool whole = en0 + NF <= N;                  // all of the tile's features are there
    // y may be the residual, so that no load passes a store: those of an X half are asked for together, the first ahead of the fills
    Put<bf16_t>::Eight res[GLU ? 1 : 8];
    const auto ask = [&](int h) __attribute__((always_inline)) {
      if (GLU || !o.res || !whole) return;
#pragma unroll
      for (int i = 0; i < (GLU ? 1 : 8); ++i)
        res[i] = *(const Put<bf16_t>::Eight*)((const bf16_t*)o.res + (size_t)min(em0 + h * 128 + wm * 64 + (i >> 1) * 16 + l16, M - 1) * o.ldr + en0 + wn * 64 +
                                              (i & 1) * 32 + 8 * lq);
    };
    ask(0);
    idx += (int)(gridDim.x >> 3);
    const bool more = idx < share && xcd + idx < tiles;
    if (more) {
      open();
      first();
    }
    asm volatile("" ::: "memory");
    // D of a 16x16 tile: lane l holds row l % 16, and of the two feature tiles of a W half features 8*(l/16) .. + 7 of its 32
    if constexpr (MODE == 2) {
      const unsigned fm = lds_addr(smem) + F8_MAXIMA + (unsigned)(wm * 64 + l16) * 16u;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          unsigned m = 0;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float a = DT<bf16_t>::rnd(gelu_tanh_exp(acc[e >> 2][h][j][e & 3]) * acc[2 + (e >> 2)][h][j][e & 3]);
            acc[e >> 2][h][j][e & 3] = en0 + wn * 32 + 8 * lq + e < N ? a : 0.f;
            m = max(m, fp8_size(acc[e >> 2][h][j][e & 3]));
          }
          m = max(m, (unsigned)__shfl_xor((int)m, 16));
          m = max(m, (unsigned)__shfl_xor((int)m, 32));
          if (lq == 0) asm volatile("ds_write_b32 %0, %1" ::"v"(fm + (unsigned)(h * 128 + j * 16) * 16u + (unsigned)wn * 4u), "v"(m) : "memory");
        }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          u32x4_t v = lds16<0>(fm + (unsigned)(h * 128 + j * 16) * 16u);
          asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(v)::"memory");
          const float most = __uint_as_float(max(max(v[0], v[1]), max(v[2], v[3])));
          const fp8_cut<bf16_t> cut(most);
          const int m = em0 + h * 128 + wm * 64 + j * 16 + l16, f = en0 + wn * 32 + 8 * lq;
          const floatx4_t a = acc[0][h][j], b = acc[1][h][j];
          if (m < M && f < N)                          // a row's codes lie in whole 16 bytes: zeros behind the last feature
            *(uint2*)((uint8_t*)o.y + (size_t)m * o.ldy + f) = make_uint2(fp8_pack4(cut(a[0]), cut(a[1]), cut(a[2]), cut(a[3])),
                                                                          fp8_pack4(cut(b[0]), cut(b[1]), cut(b[2]), cut(b[3])));
          if (m < M && wn == 0 && lq == 0) o.s[m * o.sr + (en0 >> 7) * o.sb] = fp8_scale(most);
        }
    } else {
      // whether all features are there is asked for the tile: the other form's branches are many, and a launch fetches its code anew
      const auto leave = [&](auto every) __attribute__((always_inline)) {
        constexpr bool ALL = decltype(every)::value;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (h) ask(1);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int m = em0 + h * 128 + wm * 64 + j * 16 + l16;
#pragma unroll
            for (int i = 0; i < (GLU ? 1 : 2); ++i) {
              const int f = en0 + wn * (GLU ? 32 : 64) + i * 32 + 8 * lq;
              float v[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const float a = acc[2 * i + (e >> 2)][h][j][e & 3];
                v[e] = GLU ? gelu_tanh_exp(a) * acc[2 + (e >> 2)][h][j][e & 3] : a;
              }
              bf16_t* const y = (bf16_t*)o.y + (size_t)m * o.ldy + f;
              if constexpr (ALL) {
                if (m < M) {
                  if (!GLU && o.bias) Put<bf16_t>::add(v, *(const Put<bf16_t>::Eight*)((const bf16_t*)o.bias + f));
                  if (!GLU && o.res) Put<bf16_t>::add(v, res[j * 2 + i]);
                  Put<bf16_t>::put(y, v);
                }
              } else if (m < M && f < N) {
                if (!GLU && o.bias) add_some(v, (const bf16_t*)o.bias + f, N - f);
                if (!GLU && o.res) add_some(v, (const bf16_t*)o.res + (size_t)m * o.ldr + f, N - f);
                put_some(y, v, N - f);
              }
            }
          }
        }
      };
      if (whole) leave(std::true_type{});
      else leave(std::false_type{});
    }
    young = em0 + 256 <= M && whole;
    if (!more) break;
  }
}

template <int MODE, bool TAIL>
int large_launch(const Codes& X, const Codes& W, const Codes& U, const Leave& o, int M, int N, int K, hipStream_t s, const char* name) {
  constexpr int NF = MODE ? 128 : 256;
  static fstu_lds_limit most;
  if (const int rc = fstu_need_lds((const void*)fp8_large_kernel<MODE, TAIL>, most, F8_LDS(MODE == 2), name)) return rc;
  const int mt = (M + 255) / 256, nt = (N + NF - 1) / NF, share = (int)(((long long)mt * nt + 7) / 8);
  hipLaunchKernelGGL((fp8_large_kernel<MODE, TAIL>), dim3(8u * (unsigned)std::min(share, fstu_cus() / 8)), dim3(512), F8_LDS(MODE == 2), s, X, W, U, o,
                     M, N, K, mt, nt, share);
  return 0;
}
template <int MODE>
int large(const Codes& X, const Codes& W, const Codes& U, const Leave& o, int M, int N, int K, hipStream_t s, const char* name) {
  return K % 128 ? large_launch<MODE, true>(X, W, U, o, M, N, K, s, name) : large_launch<MODE, false>(X, W, U, o, M, N, K, s, name);
}

// ---------------------------------------------------------------- few rows
// The weights' bytes bound these (8 rows, weights that come from memory: 2 x 24576 x 2048 20.3 us, 5.0 TB/s; 2048 x 24576 20.1, 2.5; 50304 x 768 12.3, 3.1; the
// same weight again and again, which the caches hold, 17.8, 13.4 and 9.8, as the figures below are): a wave takes 16 features
// (glu: of both weights; linear 16 F) x 16 R rows of every KH-th block of K, U blocks in
// flight at once in registers, and the KH waves of a feature tile join their sums in LDS.  A load is 8 rows of 128 bytes, whole lines;
// the fragments, 16 rows of 64 bytes, are taken through 2 KB of LDS that the wave has for itself (read straight as fragments, half a line to a row,
// one compute unit gets half as much: 768 x 9216 bytes over 48 of them 5.5 us, 2.9 so).  A workgroup has NT feature tiles, F of them to
// a wave; K may be cut into slices over the grid (linear), whose fp32 sums a second launch adds in their order.  A wave keeps P sums, of
// every P-th of its blocks: the pair's sums are those of every fourth block whether four waves form them or two, so that its codes are
// those of its bf16 result to the bit.
template <typename T, int MODE, int R, int F, int NT, int KH, int P, int U, bool TAIL>
__global__ void __launch_bounds__(64 * NT * KH)
fp8_skinny_kernel(Codes X, Codes W, Codes V, Leave o, float* __restrict__ partial, int M, int N, int K, int slices) {
  constexpr bool GLU = MODE != 0;
  constexpr int FT = GLU ? 1 : F, G = F * R;           // feature tiles side by side of a wave, its 16 x 16 sums
  static_assert(!GLU || F == 2, "gate and up");
  static_assert(R * FT <= KH, "one wave joins one tile's sums");
  static_assert(MODE != 2 || NT == 8, "the block of 128 features that shares a scale");
  static_assert(U % P == 0 && (!GLU || KH * P == 4), "sums by block");
  extern __shared__ __align__(16) unsigned char skinny_smem[];
  float* const red = (float*)skinny_smem;              // behind the loop: [P][KH][NT][G][64 lanes][4]
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, q = lane >> 4;
  const int nt = wv % NT, kh = wv / NT;
  const int n0 = ((int)blockIdx.x * NT + nt) * 16 * FT, m0 = (int)blockIdx.z * 16 * R;
  const int row8 = lane >> 3, ch = lane & 7;           // this lane's row (and row + 8) of a load, its chunk of a block
  const uint8_t *wr[F][2], *xr[R][2];
  const float *ws[F], *xs[R];
#pragma unroll
  for (int f = 0; f < F; ++f) {
    const Codes& c = GLU && f ? V : W;
    const int n = min(n0 + (GLU ? 0 : f * 16), N - 1);
#pragma unroll
    for (int h = 0; h < 2; ++h) wr[f][h] = c.p + (size_t)min(n + row8 + 8 * h, N - 1) * c.ld;
    ws[f] = c.s + (n >> 7) * c.sr;
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
#pragma unroll
    for (int h = 0; h < 2; ++h) xr[r][h] = X.p + (size_t)min(m0 + r * 16 + row8 + 8 * h, M - 1) * X.ld;
    xs[r] = X.s + (long long)min(m0 + r * 16 + l16, M - 1) * X.sr;
  }
  const int nb = (K + 127) >> 7, s = (int)blockIdx.y;
  const int b0 = (int)((unsigned)(nb * s) / (unsigned)slices), b1 = (int)((unsigned)(nb * (s + 1)) / (unsigned)slices);
  floatx4_t acc[P][F][R];
#pragma unroll
  for (int i = 0; i < P * G; ++i) acc[i / G][i % G / R][i % R] = floatx4_t{0.f, 0.f, 0.f, 0.f};
  const auto chunk = [&](const uint8_t* p, int k) __attribute__((always_inline)) { return TAIL ? chunk16(p, k, K) : *(const u32x4_t*)(p + k); };
  const bool both = R > 1 || M - m0 > 8;               // rows 8 .. 15 of the only row tile (what lies in LDS for them reaches nobody else's sum)
  // the chunk index is XOR-ed with bits of the row: neither the lines' writes nor the fragments' reads meet bank conflicts
  unsigned char* const own = skinny_smem + (size_t)wv * ((F + R) * 2048);
  unsigned char* const to = own + row8 * 128;
  const unsigned to0 = (unsigned)(ch ^ (row8 >> 1)) * 16u, to1 = 1024u + (unsigned)(ch ^ (4 + (row8 >> 1))) * 16u;
  const unsigned at0 = (unsigned)l16 * 128u + (unsigned)(q ^ (l16 >> 1)) * 16u, at1 = (unsigned)l16 * 128u + (unsigned)((4 + q) ^ (l16 >> 1)) * 16u;
  for (int b = b0 + kh; b < b1; b += KH * U) {
    u32x4_t w[U][F][2], x[U][R][2];
    float sw[U][F], sx[U][R];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int bb = b + u * KH, k = bb * 128 + ch * 16;
      if (bb < b1) {
#pragma unroll
        for (int f = 0; f < F; ++f) {
          w[u][f][0] = chunk(wr[f][0], k), w[u][f][1] = chunk(wr[f][1], k);
          sw[u][f] = ws[f][bb * (GLU && f ? V.sb : W.sb)];
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
          x[u][r][0] = chunk(xr[r][0], k);
          if (both) x[u][r][1] = chunk(xr[r][1], k);
          sx[u][r] = xs[r][bb * X.sb];
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (b + u * KH < b1) {
        __builtin_amdgcn_wave_barrier();               // a wave's LDS operations stay in order
#pragma unroll
        for (int t = 0; t < F + R; ++t) {
          *(u32x4_t*)(to + t * 2048 + to0) = t < F ? w[u][t < F ? t : 0][0] : x[u][t < F ? 0 : t - F][0];
          if (t < F || both) *(u32x4_t*)(to + t * 2048 + to1) = t < F ? w[u][t < F ? t : 0][1] : x[u][t < F ? 0 : t - F][1];
        }
        asm volatile("" ::: "memory");
        __builtin_amdgcn_wave_barrier();
        const auto fragment = [&](int t) __attribute__((always_inline)) {
          return Operand<T>(Frag32{*(const u32x4_t*)(own + t * 2048 + at0), *(const u32x4_t*)(own + t * 2048 + at1)});
        };
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const Operand<T> xo = fragment(F + r);
#pragma unroll
          for (int f = 0; f < F; ++f) {
            const floatx4_t d = Operand<T>::sum(fragment(f), xo);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[u % P][f][r][e] = fmaf(d[e], sx[u][r] * sw[u][f], acc[u % P][f][r][e]);
          }
        }
        asm volatile("" ::: "memory");
      }
  }
  __syncthreads();                                     // the sums take the place of what other waves have read
  // the sums of a tile, by the wave whose kh is its number
  floatx4_t* const mine = (floatx4_t*)red + ((size_t)(kh * NT + nt) * G) * 64 + lane;
#pragma unroll
  for (int i = 0; i < P * G; ++i) mine[((size_t)(i / G) * KH * NT * G + i % G) * 64] = acc[i / G][i % G / R][i % R];
  __syncthreads();
  const bool joins = kh < R * FT;
  const int r = kh % R, f = kh / R;                    // this wave's row tile and, linear, feature tile
  floatx4_t v = {0.f, 0.f, 0.f, 0.f}, w2 = v;
  if (joins) {
#pragma unroll
    for (int k = 0; k < KH * P; ++k) {
      const floatx4_t* const p = (const floatx4_t*)red + ((size_t)(k * NT + nt) * G) * 64 + lane;
      v += p[(f * R + r) * 64];
      if constexpr (GLU) w2 += p[(R + r) * 64];
    }
  }
  const int fe = n0 + f * 16 + q * 4, m = m0 + r * 16 + l16;
  if constexpr (GLU) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = fe + e < N ? DT<T>::rnd(gelu_tanh_exp(v[e]) * w2[e]) : 0.f;
  }
  if constexpr (MODE == 2) {
    __syncthreads();                                   // the sums have been read: the maxima take their place
    unsigned* const most = (unsigned*)red;             // [NT][16 R]
    if (joins) {
      unsigned a = max(max(fp8_size(v[0]), fp8_size(v[1])), max(fp8_size(v[2]), fp8_size(v[3])));
      a = max(a, (unsigned)__shfl_xor((int)a, 16));
      a = max(a, (unsigned)__shfl_xor((int)a, 32));
      if (q == 0) most[nt * 16 * R + r * 16 + l16] = a;
    }
    __syncthreads();
    if (joins && m < M) {
      unsigned a = 0;
#pragma unroll
      for (int i = 0; i < NT; ++i) a = max(a, most[i * 16 * R + r * 16 + l16]);
      const fp8_cut<bf16_t> cut(__uint_as_float(a));
      if (fe < N) *(unsigned*)((uint8_t*)o.y + (size_t)m * o.ldy + fe) = fp8_pack4(cut(v[0]), cut(v[1]), cut(v[2]), cut(v[3]));
      if (nt == 0 && q == 0) o.s[m * o.sr + blockIdx.x * o.sb] = fp8_scale(__uint_as_float(a));
    }
    return;
  }
  if (!joins || m >= M) return;
  if (!GLU && slices > 1) {
    float* const p = partial + ((size_t)s * M + m) * N + fe;
    if (N % 4 == 0 && fe < N) *(floatx4_t*)p = v;
    else
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (fe + e < N) p[e] = v[e];
    return;
  }
  T* const y = (T*)o.y + (size_t)m * o.ldy + fe;
  const T* const res = (const T*)o.res + (size_t)m * o.ldr + fe;
  float more[4] = {0.f, 0.f, 0.f, 0.f};                // y may be the residual, so that no load passes a store
  if constexpr (!GLU) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (o.bias && fe + e < N) more[e] = DT<T>::ld((const T*)o.bias + fe + e);
      if (o.bias) v[e] += more[e];
      if (o.res && fe + e < N) more[e] = DT<T>::ld(res + e);
    }
    if (o.res)
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += more[e];
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (fe + e < N) DT<T>::st(y + e, v[e]);
}

// fp32 slices (slices, M, N), added in order -> T( sum + bias + residual )
template <typename T>
__global__ void __launch_bounds__(256)
fp8_join_kernel(const float* __restrict__ partial, Leave o, int M, int N, int slices) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x, n = (long long)M * N;
  if (i >= n) return;
  const int m = (int)(i / N), f = (int)(i - (long long)m * N);
  float v = partial[i];
  for (int s = 1; s < slices; ++s) v += partial[s * n + i];
  if (o.bias) v += DT<T>::ld((const T*)o.bias + f);
  if (o.res) v += DT<T>::ld((const T*)o.res + (size_t)m * o.ldr + f);
  DT<T>::st((T*)o.y + (size_t)m * o.ldy + f, v);
}

template <typename T, int MODE, int R, int F, int NT, int KH, int P, int U, bool TAIL>
int skinny_launch(const Codes& X, const Codes& W, const Codes& V, const Leave& o, float* partial, int slices, int M, int N, int K, hipStream_t s,
                  const char* name) {
  constexpr int NF = 16 * NT * (MODE ? 1 : F);
  constexpr unsigned lds = KH * NT * std::max(P * F * R * 1024, (F + R) * 2048);
  static fstu_lds_limit most;
  if (const int rc = fstu_need_lds((const void*)fp8_skinny_kernel<T, MODE, R, F, NT, KH, P, U, TAIL>, most, lds, name)) return rc;
  hipLaunchKernelGGL((fp8_skinny_kernel<T, MODE, R, F, NT, KH, P, U, TAIL>), dim3((N + NF - 1) / NF, slices, (M + 16 * R - 1) / (16 * R)), dim3(64 * NT * KH),
                     lds, s, X, W, V, o, partial, M, N, K, slices);
  if (MODE == 0 && slices > 1)
    hipLaunchKernelGGL((fp8_join_kernel<T>), dim3((unsigned)(((long long)M * N + 255) / 256)), dim3(256), 0, s, partial, o, M, N, slices);
  return 0;
}
template <typename T, bool TAIL>
int skinny_linear(const Codes& X, const Codes& W, const Leave& o, float* partial, int slices, int M, int N, int K, hipStream_t s) {
  const char* const name = "fstu_fp8_linear";
  // eight waves to a tile, or four where the tiles are many or K is short: waves without a block of their own hold up the next workgroup.  us, 16 / 8 / 4
  // waves: 8 rows, 50304 x 768 34 / 12.5 / 9.0, 9216 x 768 7.3 / 3.7 / 3.4, 2048 x 2048 3.6 / 3.3 / 3.5, 768 x 9216 5.3 / 5.3 / 6.9 (fp32, whose codes are widened
  // beside the loads, 5.7 / 6.1 / 8.3, so sixteen); 32 rows, 50304 x 768 28 / 17 / 15, 2048 x 24576 in four slices 14.3 / 13.9 / 16.4, 768 x 9216 in four
  // 6.9 / 6.7 / 7.7; 300 x 2304 x 768 - / 7.5 / 6.4, 300 x 768 x 9216 - / 10.3 / 14.9.
  const int nb = ((K + 127) / 128 + slices - 1) / slices;
  const long long groups = skinny_groups(M, N, slices);
  if (M <= 16) {
    if (nb <= 8 || groups > 2 * fstu_cus()) return skinny_launch<T, 0, 1, 1, 1, 4, 1, 2, TAIL>(X, W, W, o, partial, slices, M, N, K, s, name);
    if constexpr (sizeof(T) == 4)
      if (nb > F8_LONG && groups <= fstu_cus()) return skinny_launch<T, 0, 1, 1, 1, 16, 1, 4, TAIL>(X, W, W, o, partial, slices, M, N, K, s, name);
    return skinny_launch<T, 0, 1, 1, 1, 8, 1, 2, TAIL>(X, W, W, o, partial, slices, M, N, K, s, name);
  }
  if (skinny_64(M, N, nb, slices)) return skinny_launch<T, 0, 4, 2, 1, 8, 1, 2, TAIL>(X, W, W, o, partial, slices, M, N, K, s, name);
  if (nb <= F8_LONG && groups > 2 * fstu_cus()) return skinny_launch<T, 0, 2, 2, 1, 4, 1, 2, TAIL>(X, W, W, o, partial, slices, M, N, K, s, name);
  return skinny_launch<T, 0, 2, 2, 1, 8, 1, 1, TAIL>(X, W, W, o, partial, slices, M, N, K, s, name);
}
template <typename T, bool TAIL>
int skinny_glu(const Codes& X, const Codes& W, const Codes& V, const Leave& o, int M, int N, int K, hipStream_t s) {
  const char* const name = "fstu_fp8_glu";
  if constexpr (std::is_same<T, bf16_t>::value) {
    // 16 waves of 16 rows: those of 32 rows had to spill (32 rows, 9216 x 768 12.1 us, so 6.4; 24576 x 2048 28 and 30)
    if (o.s) return skinny_launch<T, 2, 1, 2, 8, 2, 2, 2, TAIL>(X, W, V, o, nullptr, 1, M, N, K, s, name);
  }
  // us, 8 / 32 rows: 9216 x 768 two tiles of four waves 4.2 / 5.5, one 4.3 / 5.0
  if (M <= 16) return skinny_launch<T, 1, 1, 2, 2, 4, 1, 2, TAIL>(X, W, V, o, nullptr, 1, M, N, K, s, name);
  return skinny_launch<T, 1, 2, 2, 1, 4, 1, 2, TAIL>(X, W, V, o, nullptr, 1, M, N, K, s, name);
}

// ---------------------------------------------------------------- 128 x 128 tiles
// Products of too few 256 x 256 tiles, and those whose results are fp32.  The pair's codes in tiles of 64 rows and the 128 features that share a scale, a
// wave 32 of either weight's, in three stages of 41 KB.  Four waves, each 64 features (glu: 32 of the gate and 32 of the
// up weight) x 64 rows; K in blocks of 128 through STAGES LDS stages: two, and two workgroups to a compute unit, which cover each other's
// waits and ends (fp32: the widening of one's codes runs beside the other's products: 8192 x 2048 x 24576 849 us with four, 707 so;
// 4096 x 2048 x 2048 bf16 30 / 24), or four where there is no second one (4096 x 768 x 9216 51 with two, 39 so).  There fp32 takes two
// groups of four waves with two stages each, which halve K between them and add their sums through LDS: what stands in for the second workgroup
// (4096 x 768 x 9216 82 without, 66 so; 1000 x 2048 x 2048 24 / 21; below 7 blocks the sum costs more: 2000 x 768 x 768 13.2 / 14.3; bf16
// 39 / 42).  One wave of a group to a SIMD, so it does everything at once:
//   wait for the fragments of kt (this wave has left stage kt) and for its share of block kt + 1; barrier; multiply the fragments of kt and,
//   an instruction to three behind each product, request block kt + STAGES into stage kt and read the fragments of kt + 1 (bf16: with the first half of
//   the products, 4096 x 768 x 9216 39.8 -> 38.5 us)
// (all requests, then all reads, then the products: 0.75 us a block of the four-stage form, since a wave issues in order and the queues of
// both are short; 0.46 to 0.5 so, of which the products are 0.25).
// K may be cut into slices over the grid (linear), whose fp32 sums a second launch adds in their order.
template <int MODE>
struct Tl {                                            // MODE 0 linear, 1 glu, 2 glu codes: 64 rows x the 128 features that share a scale
  static constexpr int NF = MODE == 1 ? 64 : 128, ROWS = MODE == 2 ? 64 : 128;
  static constexpr int WJ = MODE == 2 ? 8 : 4, XJ = ROWS / 32, FILLS = WJ + XJ + 1;        // a wave's fills of a block, 8 rows each, and its scales
  static constexpr unsigned X = WJ * 4096u, SCALES = X + XJ * 4096u, STAGE = SCALES + 1024u;   // W | X | scales: by wave those of 32 rows, then the two weights'
};

template <class F, int... I>
__device__ __forceinline__ void steps16(F& step, std::integer_sequence<int, I...>) {
  (step(std::integral_constant<int, I>{}), ...);
}

// TAIL: 1 K is no multiple of 128 (chunks behind K are asked for behind the range, where a fill finds zeros), 2 nor one of 16 (the chunk with a
// row's end is left out as well and comes straight from global memory behind the loop; cut in LDS between two blocks it cost the fp32
// form 27 spilled registers: 4096 x 2048 x 2001 79 us)
template <typename T, int MODE, int TAIL, int STAGES, int GROUPS>
__global__ void __launch_bounds__(256 * GROUPS, 2)
fp8_tile_kernel(Codes X, Codes W, Codes U, Leave o, float* __restrict__ partial, int M, int N, int K, int mt, int nt, int share, int slices) {
  typedef Tl<MODE> L;
  constexpr bool GLU = MODE != 0;
  constexpr int NF = L::NF, WJ = L::WJ, XJ = L::XJ;
  extern __shared__ __align__(16) unsigned char smem[];
  const int group = GROUPS > 1 ? __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 8) : 0;
  const int tid = threadIdx.x & 255, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  unsigned char* const own = smem + (unsigned)group * (STAGES * L::STAGE);
  int t = (int)(blockIdx.x & 7) * share + (int)(blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= share || t >= mt * nt * slices) return;
  const int slice = t / (mt * nt);
  t -= slice * (mt * nt);
  const int per_panel = mt * F8_PANEL, panel = t / per_panel, in_panel = t - panel * per_panel, pw = min(F8_PANEL, nt - panel * F8_PANEL);
  const int m0 = in_panel / pw * L::ROWS, n0 = (panel * F8_PANEL + in_panel % pw) * NF;
  const int nb = (K + 127) >> 7, K16 = (K + 15) & ~15;
  // a slice's blocks; of two groups the first takes the first half of them, rounded up, and both as many steps
  const int s0 = (int)((unsigned)(nb * slice) / (unsigned)slices), s1 = (int)((unsigned)(nb * (slice + 1)) / (unsigned)slices);
  const int half = GROUPS > 1 ? (s1 - s0 + 1) >> 1 : s1 - s0, b0 = s0 + group * half, e1 = min(b0 + half, s1);
  const uint8_t* const wb = W.p + (size_t)n0 * W.ld;
  const uint8_t* const ub = GLU ? U.p + (size_t)n0 * U.ld : wb;
  const uint8_t* const xb = X.p + (size_t)m0 * X.ld;
  const unsigned wbytes = (unsigned)(min(NF, N - n0) - 1) * (unsigned)W.ld + (unsigned)K16;
  const unsigned ubytes = GLU ? (unsigned)(min(NF, N - n0) - 1) * (unsigned)U.ld + (unsigned)K16 : 0;
  const unsigned xbytes = (unsigned)(min(L::ROWS, M - m0) - 1) * (unsigned)X.ld + (unsigned)K16;
  const float* const sp = lane < 32 ? X.s + (long long)min(m0 + wv * 32 + lane, M - 1) * X.sr
                                    : GLU && (lane & 1) ? U.s + (n0 >> 7) * U.sr : W.s + (n0 >> 7) * W.sr;
  const long long sstep = lane < 32 ? X.sb : GLU && (lane & 1) ? U.sb : W.sb;
  // ---- fills: a wave fills a quarter of the rows of either part, 8 to an instruction (glu: waves 0 and 1 the gate's, 2 and 3 the up weight's)
  unsigned woff[WJ], xoff[XJ];
  bool wthere[WJ], xthere[XJ];                         // whether this lane's chunk of the last block is one of K's
#pragma unroll
  for (int j = 0; j < WJ; ++j) {
    const int row = wv * 8 * WJ + j * 8 + (lane >> 3), ch = ((lane & 7) ^ (((row >> 1) & 1) | ((row >> 2) & 6))) * 16;
    woff[j] = (unsigned)(GLU ? row & (NF - 1) : row) * (unsigned)(GLU && wv >= 2 ? U.ld : W.ld) + (unsigned)ch;
    wthere[j] = (nb - 1) * 128 + ch < (K & ~15);
  }
#pragma unroll
  for (int j = 0; j < XJ; ++j) {
    const int row = wv * 8 * XJ + j * 8 + (lane >> 3), ch = ((lane & 7) ^ ((row >> 1) & 7)) * 16;
    xoff[j] = (unsigned)row * (unsigned)X.ld + (unsigned)ch;
    xthere[j] = (nb - 1) * 128 + ch < (K & ~15);
  }
  unsigned char* const fill0 = own + (unsigned)wv * (WJ * 1024u), * const fillx = own + L::X + (unsigned)wv * (XJ * 1024u);
  const auto w_at = [&](int b, int j) __attribute__((always_inline)) { return TAIL && b == nb - 1 && !wthere[j] ? 0x80000000u : woff[j]; };
  const auto x_at = [&](int b, int j) __attribute__((always_inline)) { return TAIL && b == nb - 1 && !xthere[j] ? 0x80000000u : xoff[j]; };
  const auto fetch = [&](int b, unsigned stage) __attribute__((always_inline)) {   // beyond the last block nothing, into a stage that nobody reads
    const bool in = b < e1;
    const rsrc_t rw = make_rsrc(GLU && wv >= 2 ? ub : wb, in ? (GLU && wv >= 2 ? ubytes : wbytes) : 0), rx = make_rsrc(xb, in ? xbytes : 0);
#pragma unroll
    for (int j = 0; j < WJ; ++j) fill16(rw, w_at(b, j), (unsigned)b * 128u, fill0 + stage + j * 1024);
#pragma unroll
    for (int j = 0; j < XJ; ++j) fill16(rx, x_at(b, j), (unsigned)b * 128u, fillx + stage + j * 1024);
    fill4(sp + (long long)min(b, e1 - 1) * sstep, own + stage + L::SCALES + (unsigned)wv * 256u);
  };
  const int l16 = lane & 15, lq = lane >> 4, wn = MODE == 2 ? wv : wv & 1, wm = MODE == 2 ? 0 : wv >> 1;
  const int rw0 = (GLU ? 32 : 64) * wn + 8 * (l16 >> 2) + (l16 & 3);       // this lane's W row of the first feature tile; + 4, + 32 (glu: NF)
  unsigned fw[2], fx[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int rx = wm * 64 + l16, c = h * 4 + lq;
    fw[h] = lds_addr(own) + (unsigned)rw0 * 128u + (unsigned)((c ^ (((rw0 >> 1) & 1) | ((rw0 >> 2) & 6))) << 4);
    fx[h] = lds_addr(own) + L::X + (unsigned)rx * 128u + (unsigned)((c ^ ((rx >> 1) & 7)) << 4);
  }
  const unsigned fs = lds_addr(own) + L::SCALES + (unsigned)wm * 512u + (unsigned)l16 * 4u, fsw = lds_addr(own) + L::SCALES + 128u;
  struct Set {
    Frag32 w[4], x[4];
    float sx[4], sw, su;
  };
  Set a, b;
  // the I-th of 16 reads of a block's fragments (w first: a wave's products begin with w[0] and all of x)
  const auto read_one = [&](Set& f, unsigned stage, auto which) __attribute__((always_inline)) {
    constexpr int I = decltype(which)::value, H = I & 1, P = GLU ? NF * 128 : 4096;       // P: from the first pair of feature tiles to the second
    if constexpr (I < 8) {
      (H ? f.x[I >> 1].hi : f.x[I >> 1].lo) = lds16<(I >> 1) * 2048>(fx[H] + stage);
    } else {
      constexpr int J = (I - 8) >> 1;
      (H ? f.w[J].hi : f.w[J].lo) = lds16<(J >> 1) * P + (J & 1) * 512>(fw[H] + stage);
    }
    if constexpr (I < 4) f.sx[I] = lds4<(I & 1) * 64 + (I >> 1) * 256>(fs + stage);
    if constexpr (I == 4) f.sw = lds4<0>(fsw + stage);
    if constexpr (I == 5) f.su = GLU ? lds4<4>(fsw + stage) : 0.f;
  };
  const auto each16 = [](auto&& step) __attribute__((always_inline)) { steps16(step, std::make_integer_sequence<int, 16>{}); };
  // the fragments f of a block have come; this wave's share of the next one has landed
  const auto wait = [&](Set& f) __attribute__((always_inline)) {
    asm volatile("s_waitcnt vmcnt(%22) lgkmcnt(0)"
                 : "+v"(f.w[0].lo), "+v"(f.w[0].hi), "+v"(f.w[1].lo), "+v"(f.w[1].hi), "+v"(f.w[2].lo), "+v"(f.w[2].hi), "+v"(f.w[3].lo), "+v"(f.w[3].hi),
                   "+v"(f.x[0].lo), "+v"(f.x[0].hi), "+v"(f.x[1].lo), "+v"(f.x[1].hi), "+v"(f.x[2].lo), "+v"(f.x[2].hi), "+v"(f.x[3].lo), "+v"(f.x[3].hi),
                   "+v"(f.sx[0]), "+v"(f.sx[1]), "+v"(f.sx[2]), "+v"(f.sx[3]), "+v"(f.sw), "+v"(f.su)
                 : "n"(L::FILLS * (STAGES - 2))
                 : "memory");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
  };
  floatx4_t acc[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = floatx4_t{0.f, 0.f, 0.f, 0.f};
  // multiplies block f; behind its products block kt + STAGES is requested into stage cur and block kt + 1 is read from stage nxt into g
  const auto multiply = [&](Set& f, Set& g, int kt, unsigned cur, unsigned nxt) __attribute__((always_inline)) {
    const bool in = kt + STAGES < e1;
    const rsrc_t rw = make_rsrc(GLU && wv >= 2 ? ub : wb, in ? (GLU && wv >= 2 ? ubytes : wbytes) : 0), rx = make_rsrc(xb, in ? xbytes : 0);
    float s[4], u[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) s[j] = f.sx[j] * f.sw, u[j] = GLU ? f.sx[j] * f.su : s[j];
    const auto request = [&](auto which) __attribute__((always_inline)) {
      constexpr int I = decltype(which)::value;
      if constexpr (I < L::FILLS - 1) {
        constexpr bool TO_X = MODE == 2 ? I >= WJ : I & 1;
        constexpr int J = MODE == 2 ? I % WJ : I >> 1;
        if constexpr (TO_X) fill16(rx, x_at(kt + STAGES, J), (unsigned)(kt + STAGES) * 128u, fillx + cur + J * 1024);
        else fill16(rw, w_at(kt + STAGES, J), (unsigned)(kt + STAGES) * 128u, fill0 + cur + J * 1024);
      }
      if constexpr (I == L::FILLS - 1) fill4(sp + (long long)min(kt + STAGES, e1 - 1) * sstep, own + cur + L::SCALES + (unsigned)wv * 256u);
    };
    if constexpr (std::is_same<T, float>::value) {
      // widened fragments: x's at once, w's one after the other, so that what comes for the next block takes the place of what has been widened
      Operand<T> x[4] = {Operand<T>(f.x[0]), Operand<T>(f.x[1]), Operand<T>(f.x[2]), Operand<T>(f.x[3])};
      __builtin_amdgcn_sched_barrier(0);
      floatx4_t d[4];
      each16([&](auto which) __attribute__((always_inline)) {
        constexpr int I = decltype(which)::value, i = I >> 2, k = I & 3;
        const bf16x8_t w = k < 2 ? widen8(f.w[i].lo[2 * (k & 1)], f.w[i].lo[2 * (k & 1) + 1]) : widen8(f.w[i].hi[2 * (k & 1)], f.w[i].hi[2 * (k & 1) + 1]);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          d[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, x[j].v[k], k ? d[j] : floatx4_t{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
        request(which);
        read_one(g, nxt, which);
        if constexpr (k == 3) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(d[j][e], GLU && i >= 2 ? u[j] : s[j], acc[i][j][e]);
        }
        __builtin_amdgcn_sched_barrier(0);
      });
    } else {
      floatx4_t d[16];
      const auto add = [&](auto which) __attribute__((always_inline)) {
        constexpr int I = decltype(which)::value, i = I >> 2, j = I & 3;
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(d[I][e], GLU && i >= 2 ? u[j] : s[j], acc[i][j][e]);
      };
      each16([&](auto which) __attribute__((always_inline)) {
        constexpr int I = decltype(which)::value;
        d[I] = Operand<T>::sum(Operand<T>(f.w[I >> 2]), Operand<T>(f.x[I & 3]));
        if constexpr (I < 8) {
          read_one(g, nxt, std::integral_constant<int, 2 * I>{});
          read_one(g, nxt, std::integral_constant<int, 2 * I + 1>{});
        }
        request(which);
        if constexpr (I >= F8_AHEAD) add(std::integral_constant<int, I - F8_AHEAD>{});
        __builtin_amdgcn_sched_barrier(0);
      });
      add(std::integral_constant<int, 13>{}), add(std::integral_constant<int, 14>{}), add(std::integral_constant<int, 15>{});
      static_assert(F8_AHEAD == 3, "the last sums");
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  {
#pragma unroll
    for (int i = 0; i < STAGES; ++i) fetch(b0 + i, i * L::STAGE);
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(L::FILLS * (STAGES - 1)) : "memory");
    __builtin_amdgcn_s_barrier();
    each16([&](auto which) __attribute__((always_inline)) { read_one(a, 0, which); });
    unsigned cur = 0;                                  // the stage of block kt
    const auto next = [&](unsigned st) __attribute__((always_inline)) { return st == (STAGES - 1) * L::STAGE ? 0u : st + L::STAGE; };
    // blocks in pairs; behind an odd number comes one of zeros (what a fill finds behind the range), whose scales are the last block's: where
    // they are not finite, neither is the sum any more
    for (int kt = b0; kt < b0 + half; kt += 2) {
      unsigned nxt = next(cur);
      wait(a);
      multiply(a, b, kt, cur, nxt);
      cur = nxt, nxt = next(cur);
      wait(b);
      multiply(b, a, kt + 1, cur, nxt);
      cur = nxt;
    }
    wait(a);                                      // the last reads, of a block that is not there, have to have come in
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the empty fills behind the last block
  }
  const int fe = n0 + wn * (GLU ? 32 : 64) + 8 * lq;   // this lane's features: 8 of each pair of tiles
  if constexpr (TAIL == 2) {
    if (e1 == nb && b0 < e1) {
      const int k = K & ~15;
      const u32x4_t none = {0, 0, 0, 0};
      Frag32 w[4], x[4];
      float sx[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int f = wn * (GLU ? 32 : 64) + 8 * (l16 >> 2) + (l16 & 3) + 4 * (i & 1) + (GLU ? 0 : 16 * (i & 2)), m = min(wm * 64 + i * 16 + l16, M - 1 - m0);
        w[i] = Frag32{chunk16((GLU && i >= 2 ? ub : wb) + (size_t)min(f, N - 1 - n0) * (GLU && i >= 2 ? U.ld : W.ld), k, K), none};
        x[i] = Frag32{chunk16(xb + (size_t)m * X.ld, k, K), none};
        sx[i] = X.s[(m0 + m) * X.sr + (nb - 1) * X.sb];
      }
      const float sw = W.s[(n0 >> 7) * W.sr + (nb - 1) * W.sb], su = GLU ? U.s[(n0 >> 7) * U.sr + (nb - 1) * U.sb] : 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {                    // of the four chunks that the lanes of a row hold one is meant
        if (lq) w[i].lo = none, x[i].lo = none;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const floatx4_t d = Operand<T>::sum(Operand<T>(w[i]), Operand<T>(x[j]));
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(d[e], sx[j] * (GLU && i >= 2 ? su : sw), acc[i][j][e]);
        }
    }
  }
  if constexpr (MODE == 2) {
    unsigned* const most = (unsigned*)smem;            // [64 rows][4 waves]
    __syncthreads();                                   // every wave has left the stages
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      unsigned m = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float v = DT<T>::rnd(gelu_tanh_exp(acc[e >> 2][j][e & 3]) * acc[2 + (e >> 2)][j][e & 3]);
        acc[e >> 2][j][e & 3] = fe + e < N ? v : 0.f;
        m = max(m, fp8_size(acc[e >> 2][j][e & 3]));
      }
      m = max(m, (unsigned)__shfl_xor((int)m, 16));
      m = max(m, (unsigned)__shfl_xor((int)m, 32));
      if (lq == 0) most[(j * 16 + l16) * 4 + wn] = m;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint4 all = *(const uint4*)(most + (j * 16 + l16) * 4);
      const float amax = __uint_as_float(max(max(all.x, all.y), max(all.z, all.w)));
      const fp8_cut<bf16_t> cut(amax);
      const int m = m0 + j * 16 + l16;
      const floatx4_t a = acc[0][j], b = acc[1][j];
      if (m < M && fe < N)                             // a row's codes lie in whole 16 bytes: zeros behind the last feature
        *(uint2*)((uint8_t*)o.y + (size_t)m * o.ldy + fe) = make_uint2(fp8_pack4(cut(a[0]), cut(a[1]), cut(a[2]), cut(a[3])),
                                                                       fp8_pack4(cut(b[0]), cut(b[1]), cut(b[2]), cut(b[3])));
      if (m < M && wn == 0 && lq == 0) o.s[m * o.sr + (n0 >> 7) * o.sb] = fp8_scale(amax);
    }
    return;
  }
  // two groups: each hands the other half of its rows over and finishes the other half
  constexpr int RT = 4 / GROUPS;                       // this wave's row tiles from here on, the first at row mw
  const int mw = wm * 64 + group * 32;
  if constexpr (GROUPS > 1) {
    __syncthreads();                                   // every wave has left the stages
    floatx4_t* const there = (floatx4_t*)smem + ((1 - group) * 256 + tid);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < RT; ++j) there[(i * RT + j) * 512] = group ? acc[i][j] : acc[i][RT + j];
    __syncthreads();
    const floatx4_t* const here = (const floatx4_t*)smem + (group * 256 + tid);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < RT; ++j) {
        const floatx4_t other = here[(i * RT + j) * 512], mine = group ? acc[i][RT + j] : acc[i][j];
        acc[i][j] = group ? other + mine : mine + other;
      }
  }
  // straight from the accumulators where all of the tile's features are there, in rows of whole 16 bytes
  const bool sliced = !GLU && slices > 1;
  const long long apart = sliced ? 4LL * N : (o.ldy | (!GLU && o.res ? o.ldr : 0)) * (long long)sizeof(T);
  const size_t from = sliced ? 0 : (size_t)o.y | (GLU ? 0 : (size_t)o.res | (size_t)o.bias);
  if (n0 + NF <= N && (apart & 15) == 0 && (from & 15) == 0) {
    // y may be the residual, so that no load passes a store: all of them are asked for first (one behind the other they took 5 us)
    typename Put<T>::Eight res[GLU ? 1 : 2 * RT];
    if (!GLU && o.res && slices == 1) {
#pragma unroll
      for (int i = 0; i < (GLU ? 1 : 2 * RT); ++i)
        res[i] = *(const typename Put<T>::Eight*)((const T*)o.res + (size_t)min(m0 + mw + (i >> 1) * 16 + l16, M - 1) * o.ldr + fe + (i & 1) * 32);
    }
#pragma unroll
    for (int j = 0; j < RT; ++j) {
      const int m = m0 + mw + j * 16 + l16;
      if (m >= M) continue;
#pragma unroll
      for (int p = 0; p < (GLU ? 1 : 2); ++p) {
        const int f = fe + p * 32;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float g = acc[2 * p + (e >> 2)][j][e & 3];
          v[e] = GLU ? gelu_tanh_exp(g) * acc[2 + (e >> 2)][j][e & 3] : g;
        }
        if (!GLU && slices > 1) {
          Put<float>::put(partial + ((size_t)slice * M + m) * N + f, v);
          continue;
        }
        if (!GLU && o.bias) Put<T>::add(v, *(const typename Put<T>::Eight*)((const T*)o.bias + f));
        if (!GLU && o.res) Put<T>::add(v, res[2 * j + p]);
        Put<T>::put((T*)o.y + (size_t)m * o.ldy + f, v);
      }
    }
    return;
  }
  // features of any number and alignment: through LDS and one value at a time, whole lines of a row side by side
  __syncthreads();                                     // every wave has left the stages
  float* const rows = (float*)smem;                    // 128 rows of 132
#pragma unroll
  for (int j = 0; j < RT; ++j)
#pragma unroll
    for (int i = 0; i < (GLU ? 2 : 4); ++i) {
      floatx4_t v = acc[i][j];
      if constexpr (GLU)
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = gelu_tanh_exp(v[e]) * acc[2 + i][j][e];
      *(floatx4_t*)(rows + (mw + j * 16 + l16) * 132 + (fe - n0) + (i >> 1) * 32 + (i & 1) * 4) = v;
    }
  __syncthreads();
  const int f = n0 + (int)(threadIdx.x & (NF - 1));
  if (f >= N) return;
  float bias = -0.f;                                   // nothing: keeps the sign of a zero, which a code has too
  if (!GLU && o.bias && slices == 1) bias = DT<T>::ld((const T*)o.bias + f);
  constexpr int STEP = 256 * GROUPS / NF;
  const int end = min(128, M - m0);
  const T* const res = GLU || sliced ? nullptr : (const T*)o.res;
  for (int r0 = (int)threadIdx.x / NF; r0 < end; r0 += 16 * STEP) { // sixteen at a time, none behind a condition of its own: it would wait for each
    float v[16], more[16];
    if (res) {
#pragma unroll
      for (int i = 0; i < 16; ++i) more[i] = DT<T>::ld(res + (size_t)(m0 + min(r0 + i * STEP, end - 1)) * o.ldr + f);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = rows[min(r0 + i * STEP, end - 1) * 132 + f - n0] + bias;
    if (res) {
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] += more[i];
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int m = m0 + r0 + i * STEP;
      if (r0 + i * STEP >= end) break;
      if (sliced) partial[((size_t)slice * M + m) * N + f] = v[i];
      else DT<T>::st((T*)o.y + (size_t)m * o.ldy + f, v[i]);
    }
  }
}

template <typename T, int MODE, int TAIL, int STAGES, int GROUPS>
int tile_launch(const Codes& X, const Codes& W, const Codes& U, const Leave& o, float* partial, int slices, int M, int N, int K, hipStream_t s,
                const char* name) {
  typedef Tl<MODE> L;
  static fstu_lds_limit most;
  if (const int rc = fstu_need_lds((const void*)fp8_tile_kernel<T, MODE, TAIL, STAGES, GROUPS>, most, GROUPS * STAGES * L::STAGE, name)) return rc;
  const int mt = (M + L::ROWS - 1) / L::ROWS, nt = (N + L::NF - 1) / L::NF;
  const int share = (int)(((long long)mt * nt * slices + 7) / 8);
  hipLaunchKernelGGL((fp8_tile_kernel<T, MODE, TAIL, STAGES, GROUPS>), dim3(8u * share), dim3(256 * GROUPS), GROUPS * STAGES * L::STAGE, s, X, W, U, o, partial, M, N, K, mt, nt, share, slices);
  return 0;
}
template <typename T, bool GLU>
int tile(const Codes& X, const Codes& W, const Codes& U, const Leave& o, float* partial, int slices, int M, int N, int K, hipStream_t s, const char* name) {
  const long long tiles = (long long)((M + 127) / 128) * ((N + (GLU ? 63 : 127)) / (GLU ? 64 : 128)) * slices;
  const int tail = K % 16 ? 2 : K % 128 ? 1 : 0;
  const auto run = [&](auto t) {
    constexpr int TAIL = decltype(t)::value;
    if constexpr (sizeof(T) == 2) {
      if (tiles <= fstu_cus()) return tile_launch<T, GLU ? 1 : 0, TAIL, 4, 1>(X, W, U, o, partial, slices, M, N, K, s, name);
    } else if constexpr (!GLU) {
      if (tiles <= fstu_cus() && two_groups(K, slices)) return tile_launch<T, 0, TAIL, 2, 2>(X, W, U, o, partial, slices, M, N, K, s, name);
    }
    return tile_launch<T, GLU ? 1 : 0, TAIL, 2, 1>(X, W, U, o, partial, slices, M, N, K, s, name);
  };
  const int rc = tail == 2 ? run(std::integral_constant<int, 2>{}) : tail ? run(std::integral_constant<int, 1>{}) : run(std::integral_constant<int, 0>{});
  if (!rc && !GLU && slices > 1)
    hipLaunchKernelGGL((fp8_join_kernel<T>), dim3((unsigned)(((long long)M * N + 255) / 256)), dim3(256), 0, s, partial, o, M, N, slices);
  return rc;
}

// Offsets inside a tile are of 32 bits.
bool near_rows(const Codes& X, const Codes& W, const Codes& U) { return std::max(X.ld, std::max(W.ld, U.ld)) < F8_MAX_LD; }

}  // namespace

#define FP8_OPERAND(name, c, rows, what)                                                                                         \
  FSTU_REQUIRE((c).p && (c).s, FSTU_ENULL, name ": null pointer");                                                               \
  FSTU_REQUIRE(fstu_aligned((c).p, 16) && (c).ld % 16 == 0 && (c).ld >= ((rows) > 1 ? K : 0), FSTU_EALIGN,                       \
               name ": rows of " what " must be 16-byte aligned, a multiple of 16 bytes apart and at least K=%d (stride %lld)", K, (long long)(c).ld)

// Slices of K (1: none).
extern "C" int fstu_fp8_linear_slices(int M, int N, int K, int dtype) {
  if (M < 1 || N < 1 || K < 1 || (dtype != FSTU_F32 && dtype != FSTU_BF16)) return 1;
  return plan(M, N, K, dtype == FSTU_F32, false, false, 0).slices;
}

extern "C" int fstu_fp8_linear(const uint8_t* x, int64_t ldx, const float* xs, int64_t xs_row, int64_t xs_blk, const uint8_t* w, int64_t ldw,
                               const float* ws, int64_t ws_row, int64_t ws_blk, const void* bias, const void* res, int64_t ldr, void* y, int64_t ldy,
                               int M, int N, int K, int dtype, float* partial, int slices, void* stream) {
  const Codes X = {x, ldx, xs, xs_row, xs_blk}, W = {w, ldw, ws, ws_row, ws_blk};
  FSTU_REQUIRE(y, FSTU_ENULL, "fstu_fp8_linear: null pointer");
  FSTU_REQUIRE(M >= 1 && N >= 1 && K >= 1 && M <= 65535 * 64 && N <= 1 << 26 && K <= 1 << 30 && (M / 64 + 2LL) * (N / 64 + 2) <= 1 << 25, FSTU_ESHAPE,
               "fstu_fp8_linear: M=%d N=%d K=%d", M, N, K);
  FP8_OPERAND("fstu_fp8_linear", X, M, "x");
  FP8_OPERAND("fstu_fp8_linear", W, N, "w");
  FSTU_REQUIRE(M == 1 || (ldy >= N && (!res || ldr >= N)), FSTU_ESHAPE, "fstu_fp8_linear: N=%d ldy=%lld ldr=%lld", N, (long long)ldy, (long long)ldr);
  FSTU_REQUIRE(slices == 1 || (partial && fstu_aligned(partial, 16) && slices > 1 && slices <= std::min(64, (K + 127) / 128) && near_rows(X, W, W) && (long long)M * N < 1LL << 31),
               FSTU_EARG, "fstu_fp8_linear: slices=%d (M=%d N=%d K=%d, row strides %lld and %lld)", slices, M, N, K, (long long)ldx, (long long)ldw);
  FSTU_REQUIRE(!res || fp8_same_or_apart(res, ldr, y, ldy, M, N, dtype == FSTU_F32 ? 4 : 2), FSTU_EARG,
               "fstu_fp8_linear: y overlaps the residual and is not the same rows");
  const Leave o = {y, ldy, bias, res, ldr, nullptr, 0, 0};
  const Kind kind = plan(M, N, K, dtype == FSTU_F32, false, false, slices).kind;
  hipStream_t const s = (hipStream_t)stream;
  int rc = 0;
  FSTU_DISPATCH_DTYPE(dtype, "fstu_fp8_linear", {
    if (kind == SKINNY)
      rc = K % 128 ? skinny_linear<T, true>(X, W, o, partial, slices, M, N, K, s) : skinny_linear<T, false>(X, W, o, partial, slices, M, N, K, s);
    else if (!near_rows(X, W, W) && slices == 1)
      hipLaunchKernelGGL((fp8_plain_kernel<false, T>), dim3((N + 127) / 128, (M + 63) / 64), dim3(512), 0, s, X, W, W, o, M, N, K);
    else if (kind == LARGE)
      rc = large<0>(X, W, W, o, M, N, K, s, "fstu_fp8_linear");
    else
      rc = tile<T, false>(X, W, W, o, partial, slices, M, N, K, s, "fstu_fp8_linear");
  });
  if (rc) return rc;
  FSTU_CHECK_LAUNCH("fstu_fp8_linear");
  return FSTU_OK;
}

extern "C" int fstu_fp8_glu(const uint8_t* x, int64_t ldx, const float* xs, int64_t xs_row, int64_t xs_blk, const uint8_t* gate, int64_t ldg,
                            const float* gs, int64_t gs_row, int64_t gs_blk, const uint8_t* up, int64_t ldu, const float* us, int64_t us_row,
                            int64_t us_blk, void* y, int64_t ldy, float* scales, int64_t ss, int64_t sb, int M, int N, int K, int dtype, void* stream) {
  const Codes X = {x, ldx, xs, xs_row, xs_blk}, W = {gate, ldg, gs, gs_row, gs_blk}, U = {up, ldu, us, us_row, us_blk};
  FSTU_REQUIRE(y, FSTU_ENULL, "fstu_fp8_glu: null pointer");
  FSTU_REQUIRE(M >= 1 && N >= 1 && K >= 1 && M <= 65535 * 64 && N <= 1 << 26 && K <= 1 << 30 && (M / 64 + 2LL) * (N / 64 + 2) <= 1 << 25, FSTU_ESHAPE,
               "fstu_fp8_glu: M=%d N=%d K=%d", M, N, K);
  FP8_OPERAND("fstu_fp8_glu", X, M, "x");
  FP8_OPERAND("fstu_fp8_glu", W, N, "the gate");
  FP8_OPERAND("fstu_fp8_glu", U, N, "the up weight");
  FSTU_REQUIRE(M == 1 || ldy >= N, FSTU_ESHAPE, "fstu_fp8_glu: N=%d ldy=%lld", N, (long long)ldy);
  FSTU_REQUIRE(!scales || dtype == FSTU_BF16, FSTU_EDTYPE, "fstu_fp8_glu: codes are those of the bf16 result (dtype %d)", dtype);
  FSTU_REQUIRE(!scales || (fstu_aligned(y, 16) && ldy % 16 == 0 && ldy >= N), FSTU_EALIGN,
               "fstu_fp8_glu: rows of codes must be 16-byte aligned, a multiple of 16 bytes apart and at least %d (stride %lld)", N, (long long)ldy);
  const Leave o = {y, ldy, nullptr, nullptr, 0, scales, ss, sb};
  const Kind kind = plan(M, N, K, dtype == FSTU_F32, true, scales, 1).kind;
  hipStream_t const s = (hipStream_t)stream;
  int rc = 0;
  FSTU_DISPATCH_DTYPE(dtype, "fstu_fp8_glu", {
    if (kind == SKINNY)
      rc = K % 128 ? skinny_glu<T, true>(X, W, U, o, M, N, K, s) : skinny_glu<T, false>(X, W, U, o, M, N, K, s);
    else if (!near_rows(X, W, U) || (scales && K % 16))
      hipLaunchKernelGGL((fp8_plain_kernel<true, T>), dim3((N + 127) / 128, (M + 63) / 64), dim3(512), 0, s, X, W, U, o, M, N, K);
    else if (kind == LARGE)
      rc = scales ? large<2>(X, W, U, o, M, N, K, s, "fstu_fp8_glu") : large<1>(X, W, U, o, M, N, K, s, "fstu_fp8_glu");
    else if (scales)
      rc = K % 128 ? tile_launch<bf16_t, 2, 1, 3, 1>(X, W, U, o, nullptr, 1, M, N, K, s, "fstu_fp8_glu")
                   : tile_launch<bf16_t, 2, 0, 3, 1>(X, W, U, o, nullptr, 1, M, N, K, s, "fstu_fp8_glu");
    else
      rc = tile<T, true>(X, W, U, o, nullptr, 1, M, N, K, s, "fstu_fp8_glu");
  });
  if (rc) return rc;
  FSTU_CHECK_LAUNCH("fstu_fp8_glu");
  return FSTU_OK;
}
