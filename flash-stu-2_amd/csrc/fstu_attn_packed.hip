// Attention over whole prompts of different lengths packed behind one another: causal, an optional window, grouped heads.
//   s_ij = softcap * tanh(q_i . k_j * hd^-1/2 / softcap) - slope * (i - j),  0 <= i - j <= window,  o_i = sum_j softmax_j(s_ij) v_j
#include "fstu_common.h"

namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float floatx16_t __attribute__((ext_vector_type(16)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef unsigned u32x4_t __attribute__((ext_vector_type(4)));

struct Heads {                 // rows of heads: strides in elements
  const void* p;
  int64_t row, head;
};

// The tile of `per` rows that workgroup t of a head takes: its sequence's first row and length and the tile's first row there (behind the sequence: none).
// Where a call fills the card more than once (many), the tiles of the highest number within their sequences come first: they have the most keys to walk, and
// the short ones fill the gaps of the last round.  A sequence's tiles behind another's: two documents of 4096 and 8 heads of 256 318 us, so 284; 16000 rows of
// 8 prompts and 12 heads of 64 under a window of 512 68 and 63; two of 8192 and 16 heads of 128 711 and 715.  A wave looks for that number with a lane to each
// of 63 candidates, a sequence to a lane; more than 64 sequences, whose tiles are short or many, come one behind the other, and so do few tiles (58 rows of
// three sequences 5.3 us, 5.5 by that search).
#define PACKED_WAVES 2048                                        // that the card holds at once, two to a SIMD
__device__ __forceinline__ void packed_tile(const int* cu, int seqs, int rows, int per, int t, int tiles, bool many, int* at, int* len, int* first) {
  const int lane = (int)threadIdx.x & 63;
  if (many && seqs <= 64) {
    const int a = min(max(cu[min(lane, seqs - 1)], 0), rows), b = min(max(cu[min(lane, seqs - 1) + 1], a), rows);
    const int mine = lane < seqs ? (b - a + per - 1) / per : 0;  // tiles of the lane's sequence
    int stride = 1, level = 0, above;
    while (__any(mine > 63 * stride)) stride *= 63;
    for (;; stride /= 63) {                                      // above: the tiles of number level + lane * stride and more, which are all that come before
      above = 0;
      for (int i = 0; i < seqs; ++i) above += max(0, __builtin_amdgcn_readlane(mine, i) - (level + lane * stride));
      const int last = __builtin_popcountll(__ballot(above > t)) - 1;
      if (last < 0) {                                            // no such tile: the grid has one to spare for each sequence
        *at = *len = *first = 0;
        return;
      }
      level += last * stride;
      if (stride == 1) {
        const int rank = t - __builtin_amdgcn_readlane(above, last + 1);
        const unsigned long long with = __ballot(mine > level);
        const int seq = __builtin_ctzll(__ballot(mine > level && (int)__builtin_popcountll(with & ((1ull << lane) - 1)) == rank));
        *at = __builtin_amdgcn_readlane(a, seq);
        *len = __builtin_amdgcn_readlane(b, seq) - *at;
        *first = level * per;
        return;
      }
    }
  }
  // sequence i has the tiles from cu[i] / per + i on, which are as many as it needs or one more (a sequence's rows begin anywhere), so that no count has to be
  // added up on the way
  t = tiles - 1 - t;
  const int lo = fstu_last_where(seqs, [&](int i) { return max(cu[i], 0) / per + i <= t; });
  const int a = min(max(cu[lo], 0), rows), b = min(max(cu[lo + 1], a), rows);
  *at = a;
  *len = b - a;
  *first = (t - (a / per + lo)) * per;
}

// One query of one head by a wave, key by key: 8 lanes to a key, 8 keys side by side, each group with a softmax of its own.  i: the query's row in its
// sequence, which begins at row `at`.
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
    const float mn = fmaxf(m, s), off = mn == -INFINITY ? 0.f : mn, corr = __expf(m - off), p = __expf(s - off);      // no weight for scores of -infinity
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

typedef float floatx4_t __attribute__((ext_vector_type(4)));

// fp32: v_mfma_f32_16x16x4_f32, whose operands are one value a lane, so that rows come straight from memory and probabilities straight from their registers.
// A workgroup takes 16 queries of one head; its waves take 16 keys in turn, each with a softmax of its own, and add up through LDS in order.  The order of dims
// in the first product and of keys in the second is what lanes hold: lane (g, c) the dims g hd/4 .. of key c, scores of keys 4 g + r. us, a wave to a query /
// tiles of 32 queries on the 32x32x2 form / 16 queries, 32 keys a step / with values asked for before the products and a lane's dims beside each other / 16
// keys a step: 777 rows of 4 x 64 under a window of 129 12.7 / 13.1 / 9.8 / 9.3 / 8.7, 4096 of 8 x 64 under 512 267 / 76 / 74 / 65 / 61 (the L2's reads of keys
// and values, once for each 16 queries), of 8 x 128 - / - / 161 / 129 / 108.  Two workgroups to a compute unit at heads of 256 (251 rows of 50 sequences and 64
// heads 74 us, 127 with the registers of one; 2000 rows of 8 heads 145 and 129).
template <int HD, int NW, bool CAP>
__global__ void __launch_bounds__(NW * 64, 2)
swa_packed_f32_kernel(Heads q, Heads k, Heads v, float* out, const int* cu, const float* slopes, int rows, int seqs, int heads, int kvh, int window, float softcap) {
  constexpr int ND = HD / 16, PART = HD / 4;
  typedef float Dims __attribute__((ext_vector_type(ND)));         // a lane's dims of a value: ND c ..
  __shared__ float sm[NW][16], sl[NW][16], so[16][HD + 1];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
  const int h = blockIdx.x % heads, hk = h / (heads / kvh);
  int at, len, first;
  packed_tile(cu, seqs, rows, 16, blockIdx.x / heads, gridDim.x / heads, gridDim.x * NW > PACKED_WAVES, &at, &len, &first);
  if (first < 0 || first >= len) return;
  const int qi = first + c, last = min(len - 1, first + 15);
  const int64_t k_row = k.row, v_row = v.row;
  const float* kb = (const float*)k.p + at * k_row + hk * k.head;
  const float* vb = (const float*)v.p + at * v_row + hk * v.head;
  const float kLog2e = 1.4426950408889634f, raw_slope = slopes ? slopes[h] : 0.f, slope = raw_slope * kLog2e;
  const float scale = rsqrtf((float)HD) * (CAP ? 1.0f / softcap : kLog2e), capA = softcap * kLog2e;
  floatx4_t qf[PART / 4];
  {
    const float* qr = (const float*)q.p + (at + min(qi, len - 1)) * q.row + h * q.head + g * PART;
#pragma unroll
    for (int s = 0; s < PART / 4; ++s) qf[s] = *(const floatx4_t*)(qr + 4 * s);
  }
#pragma unroll
  for (int s = 0; s < PART / 4; ++s) asm volatile("" : "+v"(qf[s]));         // waited for here, not among the loop's requests
  floatx4_t o[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) o[d] = floatx4_t{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
  for (int b = max(0, first - window) / 16 * 16 + 16 * w; b <= last; b += 16 * NW) {
    // all of the step's keys and values before the first product; rows behind the sequence: its last one, which no query of these sees
    floatx4_t s = {0.f, 0.f, 0.f, 0.f}, kf[PART / 4];
    Dims vf[4];
#pragma unroll
    for (int x = 0; x < PART / 4; ++x) kf[x] = *(const floatx4_t*)(kb + min(b + c, len - 1) * k_row + g * PART + 4 * x);
#pragma unroll
    for (int e = 0; e < 4; ++e) vf[e] = *(const Dims*)(vb + min(b + 4 * g + e, len - 1) * v_row + c * ND);
    if (HD < 256) __builtin_amdgcn_sched_barrier(0);           // 4096 rows of 8 heads of 128 108 us, 142 without; 2000 rows of 8 of 256 158 and 146
#pragma unroll
    for (int x = 0; x < PART / 4; ++x)
#pragma unroll
      for (int e = 0; e < 4; ++e) s = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[x][e], qf[x][e], s, 0, 0, 0);
    float top = -INFINITY, y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = s[e] * scale;
    if (CAP) fstu_tanh(y);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int far = qi - b - (4 * g + e);
      const float x = (CAP ? capA * y[e] : y[e]) - slope * (float)far;
      s[e] = far >= 0 && far <= window ? x : -INFINITY;
      top = fmaxf(top, s[e]);
    }
    top = fmaxf(top, fstu_swz16(top));
    top = fmaxf(top, __shfl_xor(top, 32, FSTU_WAVE));
    if (__any(top > m)) {
      const float mn = fmaxf(m, top), corr = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
      l *= corr;
#pragma unroll
      for (int d = 0; d < ND; ++d) o[d] *= corr;
      m = mn;
    }
    const float off = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float p = __builtin_amdgcn_exp2f(s[e] - off);
      l += p;
#pragma unroll
      for (int d = 0; d < ND; ++d) o[d] = __builtin_amdgcn_mfma_f32_16x16x4f32(vf[e][d], p, o[d], 0, 0, 0);
    }
  }
  l += fstu_swz16(l);
  l += __shfl_xor(l, 32, FSTU_WAVE);
  if (g == 0) { sm[w][c] = m; sl[w][c] = l; }
  __syncthreads();
  float M = -INFINITY;
#pragma unroll
  for (int n = 0; n < NW; ++n) M = fmaxf(M, sm[n][c]);
  const float mine = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - M);
#pragma unroll
  for (int n = 0; n < NW; ++n) {
    if (w == n) {
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float& sum = so[c][(4 * g + r) * ND + d];
          sum = fmaf(o[d][r], mine, n ? sum : 0.f);
        }
    }
    __syncthreads();
  }
  for (int row = w; row < 16 && first + row < len; row += NW) {
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int n = 0; n < NW; ++n) top = fmaxf(top, sm[n][row]);
#pragma unroll
    for (int n = 0; n < NW; ++n) sum = fmaf(sl[n][row], sm[n][row] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(sm[n][row] - top), sum);
    bool fine = true;
#pragma unroll
    for (int d = lane; d < HD; d += 64) fine = fine && so[row][d] / sum == so[row][d] / sum;
    float* const dst = out + ((int64_t)(at + first + row) * heads + h) * HD;
    if (__all(fine)) {
#pragma unroll
      for (int d = lane; d < HD; d += 64) dst[d] = so[row][d] / sum;
    } else   // a NaN comes from the row's own scores and values, or from a value that it does not see (0 * infinity): once more, key by key
      packed_one<float, HD>((const float*)q.p + (at + first + row) * q.row + h * q.head, kb, vb, dst, k_row, v_row, first + row, window, raw_slope, softcap);
  }
}

constexpr int packed_dims(int hd) { return hd == 256 ? 2 : 1; }             // waves that share a query's dims

typedef __amdgpu_buffer_rsrc_t rsrc_t;
typedef unsigned u32x2_t __attribute__((ext_vector_type(2)));
struct Frag8 { u32x2_t lo, hi; };

// bf16 on the matrix cores: a wave owns 32 queries of one head and walks their keys 64 at a time in two halves,
//   S^T (keys x queries) = K Q^T      lane (c, hi) ends up with query c's scores of keys (r & 3) + 8 (r >> 2) + 4 hi of 32, which is
//   O^T (dims x queries) = V^T P^T    what it holds of the second product: no score crosses a lane, only the maxima do, between two lanes.
// Keys and values go to LDS by way of registers, which hold the next tile, one barrier a tile; values are read back transposed.  The second half's first
// product runs beside the first half's softmax, the first half's second product beside the second half's: the maximum that a probability is taken from is the
// one before these keys, and where a score exceeds it by more than 2^16 (the first keys, and hardly any after) that half is formed once more. Two documents of
// 8192 rows, 16 heads of 128 on 4 key heads: 0.70 ms, 1.0 PFLOP/s, which the power of both units bounds: at the 1.80 GHz that it leaves, matrix cores are busy
// 48 % of the time and vector ALUs 42 %.  Soft-cap and ALiBi (16383 rows of 16 heads of 128, window 1024: 202-221 us) take the vector ALUs to 52 %,
// three exp or rcp to a score, matrix cores 27 %.  Instructions of 16x16x32, memory straight to LDS, halves of a workgroup in opposite phases were 7 to 15 %
// slower.
// CAP: 0 no soft-cap, 1 up to FSTU_FAST_CAP, 2 a larger one (a branch on that inside costs the windowed prompts 50 % by the registers it spills).  1 is
// 1 - 2 / (exp(2x) + 1) on the hardware's exp and reciprocal, off by up to 2^-21 of the soft-cap (2e-5 at 50), where a bf16 query's own rounding moves a score by
// 2^-9 of itself; 2 keeps small scores exact (fstu_wide_cap).
// Registers: four waves to heads of 64 are held to three a SIMD and spill 1 to 6 of 168 with ALiBi, to heads of 128 1 or 2 of 256 with ALiBi and soft-cap (FINE: up
// to 16 and 9).
// Heads of 256 are shared by two waves, a half of the dims to each: 16 registers of scores' sums cross over LDS, and a wave has what it has with heads of 128.
// Two documents of 4096 and 8 heads 253 us, 301 with all dims in a wave, which fits only one to a SIMD; 1000 rows of two 8 heads with ALiBi 39 and 47 with 128
// queries a workgroup instead of 64, which leaves room for a second one beside it.  The next tile's first product beside this one's softmax spilled with ALiBi
// (a tenth slower).
// PARTS: 2 gives each half of 32 keys to a wave of its own, and adds the two up in the end.
// A probability goes into the second product as one bf16 value, which adds as much to the result's error as its own rounding does (in 2-norm 0.0017 to 0.0022 of it
// where fp32 probabilities leave 0.0016).  FINE: as a bf16 value and what its rounding left, two products, as the layers' attention has it (0.0016): that takes
// 4096 rows of 12 heads of 64 from 20.6 us to 22.2, 16383 of 16 heads of 128 under a window from 218 to 295, two documents of 8192 from 704 to 954.
template <int HD, int NQ, int PARTS, int CAP, bool BIAS, bool FINE>
__global__ void __launch_bounds__(NQ * PARTS * packed_dims(HD) * 64, HD <= 64 && NQ * PARTS == 4 ? 3 : 2)
swa_packed_mfma_kernel(Heads q, Heads k, Heads v, bf16_t* out, const int* cu, const float* slopes, int rows, int seqs, int heads, int kvh, int window,
                       float softcap) {
  constexpr int DIMS = packed_dims(HD), NW = NQ * PARTS * DIMS, KB = HD == 256 ? 32 : 64, CH = HD / 8, KS = HD / 16 / DIMS, ND = HD / 32 / DIMS;
  constexpr int TILE = KB * CH;                              // 16-byte pieces
  extern __shared__ u32x4_t lds[];                               // two tiles of keys, two of values
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 31, hi = lane >> 5;
  // neighbouring workgroups go to the eight XCDs in turn: the query heads of a key head to one of them, whose L2 then holds its keys and values
  const int hx = blockIdx.x % heads, h = heads % 8 ? hx : hx % 8 * (heads / 8) + hx / 8, hk = h / (heads / kvh);
  int at, len, first;
  packed_tile(cu, seqs, rows, NQ * 32, blockIdx.x / heads, gridDim.x / heads, gridDim.x * NW > PACKED_WAVES, &at, &len, &first);
  if (first < 0 || first >= len) return;
  const int part = PARTS == 1 ? 0 : w / NQ, share = DIMS == 1 ? 0 : w / NQ, wq = w - (part + share) * NQ,
            qs = first + wq * 32, qi = qs + c;                    // the wave's first query, this lane's
  const bool on = qs < len;
  const int64_t k_row = k.row, v_row = v.row;
  const bf16_t* kb = (const bf16_t*)k.p + at * k_row + hk * k.head;
  const bf16_t* vb = (const bf16_t*)v.p + at * v_row + hk * v.head;
  const float kLog2e = 1.4426950408889634f, raw_slope = BIAS ? slopes[h] : 0.f, slope = raw_slope * kLog2e;
  const float scale = rsqrtf((float)HD) * (CAP ? 2.0f * kLog2e / softcap : kLog2e), capA = softcap * kLog2e;

  u32x4_t qf[KS];
  {
    const bf16_t* qr = (const bf16_t*)q.p + (at + min(qi, len - 1)) * q.row + h * q.head + share * (HD / 2) + hi * 8;
#pragma unroll
    for (int s = 0; s < KS; ++s) qf[s] = *(const u32x4_t*)(qr + s * 16);
  }
  floatx16_t o[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[d][r] = 0.f;
  // ALiBi of a half's key: without a soft-cap what the scores' sums begin with, in units of theirs
  floatx16_t bias;
#pragma unroll
  for (int r = 0; r < 16; ++r) bias[r] = BIAS ? slope * (float)((r & 3) + 8 * (r >> 2) + 4 * hi) / (CAP ? 1.f : scale * DIMS) : 0.f;
  float m = -INFINITY, l = 0.f;

  const int k_first = max(0, first - window) / KB * KB, k_last = min(len - 1, first + NQ * 32 - 1);
  // A tile's rows through a buffer descriptor: what lies behind the sequence's last row reads as zeros.  The range is checked against the lane's offset, which
  // therefore holds the row; the scalar one takes no part in it (sums made in the loop and not kept in registers: 16383 rows of 16 heads of 128 221 us, 231 with them kept).
  constexpr int NT = NW * 64, PR = (TILE + NT - 1) / NT, STEP = NT / CH;      // 16-byte pieces of a tile to a thread, rows between them
  u32x4_t kr[PR], vr[PR];
  const int row0 = tid / CH, ch0 = tid % CH;
  const int k_off = (row0 * (int)k_row + ch0 * 8) * 2, v_off = (row0 * (int)v_row + ch0 * 8) * 2;
  auto fetch = [&](int b) {
    const int last = min(KB, len - b) - 1;
    const rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc((void*)(kb + b * k_row), 0, (unsigned)(last * (int)k_row + HD) * 2, 0x00020000);
    const rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc((void*)(vb + b * v_row), 0, (unsigned)(last * (int)v_row + HD) * 2, 0x00020000);
    int ks = STEP * (int)k_row * 2, vs = STEP * (int)v_row * 2;
    asm volatile("" : "+s"(ks), "+s"(vs));
#pragma unroll
    for (int i = 0; i < PR; ++i) {
      kr[i] = __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(rk, k_off + i * ks, 0, 0));
      vr[i] = __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(rv, v_off + i * vs, 0, 0));
    }
  };
  // The 16-byte pieces of a row are XOR-ed with bits of it, so that what 16 lanes read together lies in different banks
  auto store = [&](int buf) {
#pragma unroll
    for (int i = 0; i < PR; ++i) {
      const int row = row0 + i * STEP;
      const int ks = HD >= 128 ? row & 15 : HD == 64 ? (row >> 1) & 7 : (row >> 2) & 3;
      const int vs = HD >= 128 ? (row & 3) << 2 : HD == 64 ? (row >> 1 & 1) << 2 : 0;
      if (TILE % NT == 0 || row < KB) {
        lds[buf * TILE + row * CH + (ch0 ^ ks)] = kr[i];
        lds[(2 + buf) * TILE + row * CH + (ch0 ^ vs)] = vr[i];
      }
    }
  };
  int k_at[KS], v_at[ND];                                        // in pieces, and in elements
  {
    const int ksw = HD >= 128 ? c & 15 : HD == 64 ? (c >> 1) & 7 : (c >> 2) & 3;
    const int li = lane & 15, vx = HD >= 128 ? (li >> 2) & 3 : HD == 64 ? (li >> 3) & 1 : 0;
#pragma unroll
    for (int s = 0; s < KS; ++s) k_at[s] = c * CH + ((2 * (s + share * KS) + hi) ^ ksw);
#pragma unroll
    for (int d = 0; d < ND; ++d) v_at[d] = (4 * hi + (li >> 2)) * HD + 16 * (lane >> 4 & 1) + 4 * (li & 3) + ((d + share * ND) ^ vx) * 32;
  }
  // a half's scores in base 2 are s * unit + lift: capped ones without ALiBi stay 1 / (-1 - exp 2x), and the exponential's product and sum finish them
  // (two documents of 8192, 16 heads of 128, 883 us, so 870; of 64 581 and 560)
  constexpr bool FOLD = CAP == 1 && !BIAS;
  const float unit = FOLD ? 2.0f * capA : CAP ? 1.f : scale, lift = FOLD ? capA : 0.f;
  unsigned pk[8], rest[8];
  float add, top;
  struct Keys { u32x4_t f[KS]; };
  struct Values { Frag8 f[2][ND]; };
  auto get_keys = [&](int buf, int half) {
    Keys k;
#pragma unroll
    for (int x = 0; x < KS; ++x) k.f[x] = lds[buf * TILE + half * 32 * CH + k_at[x]];
    return k;
  };
  auto get_values = [&](int buf, int half) {
    const bf16_t* vl = (const bf16_t*)(lds + (2 + buf) * TILE) + half * 32 * HD;
    Values v;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        v.f[t][d].lo = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t*)(vl + t * 16 * HD + v_at[d])));
        v.f[t][d].hi = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t*)(vl + t * 16 * HD + v_at[d] + 8 * HD)));
      }
    return v;
  };
  auto scores = [&](const Keys& k) {                             // first product of a half
    floatx16_t s = bias;
    if (CAP || !BIAS)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
    for (int x = 0; x < KS; ++x)
      s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, k.f[x]), __builtin_bit_cast(bf16x8_t, qf[x]), s, 0, 0, 0);
    return s;
  };
  auto shape = [&](floatx16_t& s, int b0) {                      // soft-cap, and what the lane's query does not see
    if (CAP == 1) {
#pragma unroll
      for (int r = 0; r < 16; ++r)
        s[r] = FOLD ? __builtin_amdgcn_rcpf(-1.0f - __builtin_amdgcn_exp2f(s[r] * scale))
                    : fmaf(-2.0f * capA, __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(s[r] * scale) + 1.0f), capA + bias[r]);
    }
    if (CAP == 2) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = fstu_wide_cap(s[r], scale, capA) + (BIAS ? bias[r] : 0.f);
    }
    if (b0 + 31 > qs || b0 < qs + 31 - window) {                 // wave-uniform: some key is not visible to some query
      asm volatile("");
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int far = qi - b0 - ((r & 3) + 8 * (r >> 2) + 4 * hi);
        s[r] = far >= 0 && far <= window ? s[r] : -INFINITY;
      }
    }
  };
  auto weigh = [&](const floatx16_t& s, float base) {            // probabilities and their sum, by the maximum as it stands
    const float off = base + lift - (m == -INFINITY ? 0.f : m);
    add = 0.f;
    float t = fmaxf(s[0], s[1]);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float a = __builtin_amdgcn_exp2f(CAP && !FOLD ? s[2 * e] + off : fmaf(s[2 * e], unit, off));
      const float z = __builtin_amdgcn_exp2f(CAP && !FOLD ? s[2 * e + 1] + off : fmaf(s[2 * e + 1], unit, off));
      add += a;
      add += z;
      pk[e] = pack2_bf16(a, z);
      if (FINE) rest[e] = pack2_bf16(a - __uint_as_float(pk[e] << 16), z - __uint_as_float(pk[e] & 0xffff0000u));
      if (e) t = fmaxf(fmaxf(t, s[2 * e]), s[2 * e + 1]);
    }
    top = fmaf(t, unit, base + lift);
  };
  auto settle = [&](const floatx16_t& s, float base) {
    if (__any(top > m + 16.f)) {
      top = fmaxf(top, __shfl_xor(top, 32, FSTU_WAVE));
      const float mn = fmaxf(m, top), corr = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
      l *= corr;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] *= corr;
      m = mn;
      weigh(s, base);
    }
    l += add;
  };
  auto add_values = [&](const Values& v) {                       // second product of a half
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const u32x4_t pf = u32x4_t{pk[4 * t], pk[4 * t + 1], pk[4 * t + 2], pk[4 * t + 3]};
#pragma unroll
      for (int d = 0; d < ND; ++d)
        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, v.f[t][d]), __builtin_bit_cast(bf16x8_t, pf), o[d], 0, 0, 0);
      if constexpr (FINE) {
        const u32x4_t rf = u32x4_t{rest[4 * t], rest[4 * t + 1], rest[4 * t + 2], rest[4 * t + 3]};
#pragma unroll
        for (int d = 0; d < ND; ++d)
          o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, v.f[t][d]), __builtin_bit_cast(bf16x8_t, rf), o[d], 0, 0, 0);
      }
    }
  };
  // With ALiBi the largest scores are a query's latest keys': from those backwards the maximum settles at once (two documents of 8192, 16 heads of 128, 719 us, 785
  // forwards; 16383 rows of 16 heads of 128 under a window of 1024 218 and 229; 512 rows of 12 heads of 64 10.6 and 11.0).  Without it forwards, where the
  // workgroups of a document read the same keys at the same time (two of 4096, 8 heads of 256, 287 us, 297 backwards).
  const int b_first = BIAS ? k_last / KB * KB : k_first, b_step = BIAS ? -KB : KB;
  int left = (k_last - k_first) / KB;                            // tiles after this one: k_first is a multiple of KB
  fetch(b_first);
  // the queries are waited for here: left to their first use in the loop, that wait would be one for the loop's own requests too
#pragma unroll
  for (int s = 0; s < KS; ++s) asm volatile("" : "+v"(qf[s]));
  store(0);
  if (left > 0) fetch(b_first + b_step);
  auto tile = [&](int b, auto bufs) {
    constexpr int buf = decltype(bufs)::value;
    __syncthreads();                                             // this tile is there, and the one before it has been read
    if (left > 0) store(buf ^ 1);
    if (left > 1) fetch(b + 2 * b_step);
    if (PARTS == 2) b += 32 * part;
    const bool seen = on && b <= qs + 31 && b + KB / PARTS - 1 >= qs - window;      // wave-uniform: the wave sees some of it
    const float base = slope * (float)(b - qi);
    if constexpr (DIMS == 2) {
      floatx4_t* const across = (floatx4_t*)(lds + 4 * TILE) + lane;               // 16 values a lane, of each wave
      floatx16_t s0;
      if (seen) {
        s0 = scores(get_keys(buf, 0));
#pragma unroll
        for (int r = 0; r < 4; ++r) across[(w * 4 + r) * 64] = floatx4_t{s0[4 * r], s0[4 * r + 1], s0[4 * r + 2], s0[4 * r + 3]};
      }
      __syncthreads();
      if (!seen) return;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const floatx4_t x = across[((w ^ NQ) * 4 + r) * 64];
#pragma unroll
        for (int e = 0; e < 4; ++e) s0[4 * r + e] += x[e];
      }
      shape(s0, b);
      const Values v0 = get_values(buf, 0);
      weigh(s0, base);
      settle(s0, base);
      add_values(v0);
      return;
    }
    if (!seen) return;
    const Keys k0 = get_keys(buf, part);
    __builtin_amdgcn_sched_barrier(0);                           // all of them asked for before the first product waits for one
    if constexpr (KB / PARTS == 32) {
      floatx16_t s0 = scores(k0);
      shape(s0, b);
      weigh(s0, base);
      settle(s0, base);
      add_values(get_values(buf, part));
      return;
    }
    const float base1 = base + slope * 32.f;
    const Keys k1 = get_keys(buf, KB / 32 - 1);
    floatx16_t s0 = scores(k0);
    shape(s0, b);
    const Values v0 = get_values(buf, 0);
    floatx16_t s1 = scores(k1);
    weigh(s0, base);
    settle(s0, base);
    shape(s1, b + 32);
    const Values v1 = get_values(buf, KB / 32 - 1);
    add_values(v0);
    weigh(s1, base1);
    settle(s1, base1);
    add_values(v1);
  };
  for (int b = b_first;; b += 2 * b_step) {
    tile(b, std::integral_constant<int, 0>{});
    if (--left < 0) break;
    tile(b + b_step, std::integral_constant<int, 1>{});
    if (--left < 0) break;
  }
  l += __shfl_xor(l, 32, FSTU_WAVE);
  if constexpr (PARTS == 2) {
    constexpr int EACH = ND * 16 + 2;
    float* const theirs = (float*)lds + wq * EACH * 64 + lane;
    __syncthreads();
    if (part) {
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) theirs[(d * 16 + r) * 64] = o[d][r];
      theirs[(EACH - 2) * 64] = m;
      theirs[(EACH - 1) * 64] = l;
    }
    __syncthreads();
    if (part) return;
    const float other = theirs[(EACH - 2) * 64], mn = fmaxf(m, other), off = mn == -INFINITY ? 0.f : mn;
    const float mf = __builtin_amdgcn_exp2f(m - off), of = __builtin_amdgcn_exp2f(other - off);
    l = fmaf(l, mf, theirs[(EACH - 1) * 64] * of);
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[d][r] = fmaf(o[d][r], mf, theirs[(d * 16 + r) * 64] * of);
  }
  const float inv = 1.0f / l;
  bool fine = true;
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      o[d][r] *= inv;
      fine = fine && o[d][r] == o[d][r];
    }
  // A NaN comes from a row's own scores and values, or from a value that it does not see (0 * infinity): a wave forms such rows once more, key by key.
  unsigned long long both = __ballot(!fine && qi < len);
  unsigned bad = (unsigned)both | (unsigned)(both >> 32);
  if constexpr (DIMS == 2) {
    unsigned* const rows_of = (unsigned*)(lds + 4 * TILE);
    __syncthreads();
    if (lane == 0) rows_of[w] = bad;
    __syncthreads();
    bad |= rows_of[w ^ NQ];
  }
  if (!on) return;
  if (qi < len && !(bad >> c & 1)) {
    bf16_t* orow = out + ((int64_t)(at + qi) * heads + h) * HD + share * (HD / 2) + 4 * hi;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        *(uint2*)(orow + d * 32 + e * 8) = make_uint2(pack2_bf16(o[d][4 * e], o[d][4 * e + 1]), pack2_bf16(o[d][4 * e + 2], o[d][4 * e + 3]));
  }
  if (share) return;
  while (bad) {
    const int i = qs + __builtin_ctz(bad);
    bad &= bad - 1;
    packed_one<bf16_t, HD>((const bf16_t*)q.p + (at + i) * q.row + h * q.head, kb, vb, out + ((int64_t)(at + i) * heads + h) * HD, k_row, v_row, i, window,
                           raw_slope, softcap);
  }
}

int packed_call(const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row, int64_t k_head, const void* v, int64_t v_row, int64_t v_head, void* out,
                const int* cu, const float* slopes, int rows, int seqs, int heads, int kvh, int hd, int window, float softcap, bool two_parts, int dtype, void* stream) {
  FSTU_REQUIRE(q && k && v && out && cu, FSTU_ENULL, "fstu_swa_packed: null pointer");
  FSTU_REQUIRE(dtype == FSTU_F32 || dtype == FSTU_BF16, FSTU_EDTYPE, "fstu_swa_packed: unknown dtype %d", dtype);
  FSTU_REQUIRE(hd == 32 || hd == 64 || hd == 128 || hd == 256, FSTU_ESHAPE, "fstu_swa_packed: head dim %d not in {32,64,128,256}", hd);
  FSTU_REQUIRE(rows >= 0 && rows <= (1 << 30) && seqs >= 0 && seqs <= (1 << 30) && kvh >= 1 && heads >= 1 && heads % kvh == 0 && heads <= 65535, FSTU_ESHAPE,
               "fstu_swa_packed: bad shape rows=%d sequences=%d heads=%d key heads=%d", rows, seqs, heads, kvh);
  FSTU_REQUIRE(window >= 0, FSTU_EARG, "fstu_swa_packed: window<0");
  FSTU_REQUIRE(fstu_softcap_ok(softcap), FSTU_EARG, "fstu_swa_packed: softcap must be zero (none) or a number from 2^-40 to 2^40");
  const int size = dtype == FSTU_BF16 ? 2 : 4;
  FSTU_REQUIRE(fstu_heads_aligned(q, q_row, q_head, size) && fstu_heads_aligned(k, k_row, k_head, size) && fstu_heads_aligned(v, v_row, v_head, size) &&
                   fstu_aligned(out, 16),
               FSTU_EALIGN, "fstu_swa_packed: rows and heads of q, k and v and out must begin at multiples of 16 bytes");
  FSTU_REQUIRE(rows == 0 || (k_row < (1 << 23) && v_row < (1 << 23)), FSTU_ESHAPE, "fstu_swa_packed: rows of k and v 2^23 elements apart and more");
  // fp32: 16 threads a row; bf16: 2 or 4; up to 512 more a sequence
  FSTU_REQUIRE(((int64_t)rows * (dtype == FSTU_F32 ? 16 : hd == 256 ? 4 : 2) + (int64_t)seqs * 512) * heads < 1ll << 32, FSTU_ESHAPE, "fstu_swa_packed: %d rows of %d sequences and %d heads are more than a launch takes", rows, seqs, heads);
  const int64_t n = (int64_t)rows * heads * hd * size;
  FSTU_REQUIRE(!fstu_heads_touch(q, q_row, q_head, rows, heads, hd, size, out, n) && !fstu_heads_touch(k, k_row, k_head, rows, kvh, hd, size, out, n) &&
                   !fstu_heads_touch(v, v_row, v_head, rows, kvh, hd, size, out, n),
               FSTU_EARG, "fstu_swa_packed: out overlaps q, k or v");
  if (rows == 0 || seqs == 0) return FSTU_OK;
  int rc = FSTU_OK;
  const Heads hq{q, q_row, q_head}, hk{k, k_row, k_head}, hv{v, v_row, v_head};
  auto run = [&](auto w) {
    constexpr int HD = decltype(w)::value;
    if (dtype == FSTU_F32) {
      const dim3 grid((unsigned)(rows / 16 + seqs) * heads);
      auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid, dim3(256), 0, (hipStream_t)stream, hq, hk, hv, (float*)out, cu, slopes, rows, seqs, heads, kvh, window, softcap);
      };
      softcap > 0.f ? go(swa_packed_f32_kernel<HD, 4, true>) : go(swa_packed_f32_kernel<HD, 4, false>);
      return;
    }
    auto bf16 = [&](auto nq, auto parts) {
      constexpr int NQ = decltype(nq)::value, PARTS = decltype(parts)::value;
      auto form = [&](auto cap, auto bias, auto fine) {
        constexpr unsigned threads = NQ * PARTS * packed_dims(HD) * 64, lds = 4 * (HD == 256 ? 32 : 64) * HD * 2 + (HD == 256 ? threads * 64 : 0);
        const auto kernel = swa_packed_mfma_kernel<HD, NQ, PARTS, decltype(cap)::value, decltype(bias)::value, decltype(fine)::value>;
        if constexpr (lds > 65536) {
          static fstu_lds_limit most;
          rc = fstu_need_lds((const void*)kernel, most, lds, "fstu_swa_packed");
          if (rc != FSTU_OK) return;
        }
        // two tiles of keys and two of values; with heads of 256 the scores' sums besides, 16 a thread
        hipLaunchKernelGGL(kernel, dim3((unsigned)(rows / (NQ * 32) + seqs) * heads), dim3(threads), lds, (hipStream_t)stream, hq, hk, hv, (bf16_t*)out, cu, slopes, rows,
                           seqs, heads, kvh, window, softcap);
      };
      auto go = [&](auto cap, auto bias) { two_parts ? form(cap, bias, std::true_type{}) : form(cap, bias, std::false_type{}); };
      auto capped = [&](auto cap) { slopes ? go(cap, std::true_type{}) : go(cap, std::false_type{}); };
      if constexpr (NQ == (HD == 256 ? 2 : 4) && PARTS == 1)
        if (softcap > FSTU_FAST_CAP) return capped(std::integral_constant<int, 2>{});
      softcap > 0.f ? capped(std::integral_constant<int, 1>{}) : capped(std::integral_constant<int, 0>{});
    };
    typedef std::integral_constant<int, 1> One;
    typedef std::integral_constant<int, HD == 256 ? 2 : 4> Four;
    typedef std::integral_constant<int, 8> Eight;
    typedef std::integral_constant<int, 2> Pair;
    // Waves of 32 queries to a workgroup: eight share a tile of keys where documents are long and nothing but the products counts (two of 8192 and 16 heads of
    // 128 699 us, 722 with four; heads of 64 469 and 444; a window of 1024 253 and 238).  Where there are few workgroups a wave's chain of steps bounds them:
    // two waves of queries, each with a partner for half of its keys.  us, four waves / two and partners: heads of 64, window 512, 2048 rows of 12 20.0 / 16.1,
    // 4096 27.3 / 19.4, 6144 29.5 / 26.7, one document of 16 heads 4096 61 / 55.6, 6144 109 / 112; heads of 128, window 1024, 2048 rows of 16 26.4 / 22.2, 4096
    // 61.8 / 58, 5120 68 / 71; heads of 32 21.8 / 15.9, 77 / 75. Heads of 256: two waves of queries, two of dims.  Partners for quarters of the keys: 512 rows
    // of 12 heads of 64 10.9, 11.4 with halves, 58 rows 6.2 and 5.2, 2000 rows 21 and 17.  Soft-caps of no ordinary size have the kernel of four waves alone.
    const bool usual = softcap <= FSTU_FAST_CAP;
    if constexpr (HD == 128)
      if (usual && window >= 4096 && rows / seqs >= 4096) return bf16(Eight{}, One{});
    if constexpr (HD <= 128)
      if (usual && (int64_t)(rows / 128) * heads < (HD == 128 ? 576 : 768)) return bf16(Pair{}, Pair{});
    bf16(Four{}, One{});
  };
  if (hd == 32) run(std::integral_constant<int, 32>{});
  else if (hd == 64) run(std::integral_constant<int, 64>{});
  else if (hd == 128) run(std::integral_constant<int, 128>{});
  else run(std::integral_constant<int, 256>{});
  if (rc != FSTU_OK) return rc;
  FSTU_CHECK_LAUNCH("fstu_swa_packed");
  return FSTU_OK;
}

}  // namespace

extern "C" int fstu_swa_packed(const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row, int64_t k_head, const void* v, int64_t v_row,
                               int64_t v_head, void* out, const int* cu, const float* slopes, int rows, int seqs, int heads, int kvh, int hd, int window,
                               float softcap, int dtype, void* stream) {
  return packed_call(q, q_row, q_head, k, k_row, k_head, v, v_row, v_head, out, cu, slopes, rows, seqs, heads, kvh, hd, window, softcap, false, dtype, stream);
}

extern "C" int fstu_swa_packed_fine(const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row, int64_t k_head, const void* v, int64_t v_row,
                                    int64_t v_head, void* out, const int* cu, const float* slopes, int rows, int seqs, int heads, int kvh, int hd, int window,
                                    float softcap, int dtype, void* stream) {
  return packed_call(q, q_row, q_head, k, k_row, k_head, v, v_row, v_head, out, cu, slopes, rows, seqs, heads, kvh, hd, window, softcap, true, dtype, stream);
}
