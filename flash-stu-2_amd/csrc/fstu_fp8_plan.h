// Which kernel an 8-bit product runs on (fstu_fp8_gemm.hip): whole numbers and an estimate, no GPU code.  fstu_cus() is the number of compute units.
#pragma once
#include <algorithm>
#include <cmath>

namespace {

#define F8_LONG 24                                // blocks of K beyond which the compute units work in rounds of one tile
// Tiles of 16 rows and features, or of 32.
long long skinny_groups(int M, int N, int slices) {
  const int t = M <= 16 ? 16 : 32;
  return ((N + t - 1) / t) * (long long)((M + t - 1) / t) * slices;
}
// Tiles of 64 rows where K is long and 32 rows take a second round: 500 x 768 x 9216 18.4 us, 16.4 so (300 rows, one round, 10.3 and 15.6; 1000, three and two
// rounds, 26.4 and 30.8; short K 300 x 2304 x 768 6.4 and 9.8).
bool skinny_64(int M, int N, int nb, int slices) {
  return M > 32 && nb > F8_LONG && skinny_groups(M, N, slices) > fstu_cus() && ((N + 31) / 32) * (long long)((M + 63) / 64) * slices <= fstu_cus();
}
// fp32 in tiles that leave compute units over: two groups of waves, each with half of a slice's blocks in steps of two
bool two_groups(int K, int slices) { return (K + 127) / 128 >= 7 * slices; }

// Which kernel a product runs on, and in how many slices of K: the least of an estimate in us, fitted to products of 1 to 8192 rows, 128 to
// 24576 features and K = 256 to 24576.  Of 226 products timed on each kernel (profiles/fp8_plan.txt) the one chosen is within a tenth of the best for 211; the
// farthest, 1.2 to 1.6 times it, are pairs of K = 256 whose features are no multiple of 64, and 64 x 24576 x 2048 (23 us, tiles 15).  TILE is priced by rounds of workgroups over the
// compute units, each with a start and an end of its own, SKINNY by the longest of one workgroup's time, that of all of them at the chip's rate
// and the weights' bytes.
// us, skinny / tile / large.  Linear, rows x features x K: 500 x 768 x 768 5.2 / 8.3 / 15.7, 1000 6.5 / 8.3, 3000 - / 8.8 / 16; 200 x 2048 x 2048 6.4 / 12.8 /
// 26, 600 14.4 / 12.5 / 26, 4096 - / 23 / 29, 8192 - / 44 / 38; 500 x 768 x 9216 16 / 39 / 87, 1000 26 / 22, 2000 - / 29 / 87, 8192 - / 65 / 88; fp32 500 x
// 768 x 768 5.4 / 12.4, 1500 10.6 / 13.  Gated pair: 64 x 9216 x 768 7.4 / 6.8 / 10.5, 300 26 / 9.5 / 13.4, 500 - / 15.2 / 14.4, 1200 - / 26.8 / 27, 4096
// - / 79 / 69; 2000 x 24576 x 2048 - / 217 / 175.
enum Kind { SKINNY, TILE, LARGE };
struct Plan { Kind kind; int slices; double us; };
double estimate(Kind kind, int slices, int M, int N, int K, bool f32, bool glu) {
  const auto up = [](long long a, long long b) { return (a + b - 1) / b; };
  const long long nb = up(up(K, 128), slices), cus = fstu_cus();
  double us = slices > 1 ? (kind == SKINNY ? 0.4 + 0.37 * slices : 2.2) + (double)slices * M * N * 8 / 3e6 : 0.0;
  if (kind == SKINNY) {
    const bool one = M <= 16;
    const double groups = (double)skinny_groups(M, N, slices);
    const double bytes = 1.5 + (double)N * K / (5.3e6 * std::sqrt(std::sqrt(std::min(1.0, groups / cus))));     // fewer compute units draw less
    if (one)
      return us + std::max(bytes, std::max(f32 ? 2.7 + 0.04 * nb : 2.6 + 0.036 * nb, 2.0 + groups * (0.0011 + (f32 ? 0.0002 : 0.00017) * nb)));
    if (skinny_64(M, N, (int)nb, slices)) return us + std::max(bytes, 1.5 + (f32 ? 4.2 + 0.205 * nb : 4.2 + 0.15 * nb));
    if (nb > F8_LONG) return us + std::max(bytes, 1.5 + std::ceil(groups / cus) * (f32 ? 1.5 + 0.112 * nb : 1.6 + 0.098 * nb));
    return us + std::max(bytes, std::max(f32 ? 3.6 + 0.1 * nb : 3.4 + 0.08 * nb, 2.2 + groups * (0.0035 + (f32 ? 0.00044 : 0.00038) * nb)));
  }
  if (kind == TILE) {
    const long long tiles = up(N, glu ? 64 : 128) * up(M, 128) * slices;
    us += (N % (glu ? 64 : 128) ? 4.0 : 0.0) + (K % 16 ? 2.0 : 0.0);       // the ends by one value and one chunk at a time
    if (tiles <= cus) return us + (f32 ? (!glu && two_groups(K, slices) ? 9.5 + 0.78 * (double)(up(nb, 4) * 4) : 5.0 + 1.03 * nb) : 4.5 + 0.45 * nb);
    const long long rest = tiles % (2 * cus);
    const double rounds = (double)(tiles / (2 * cus)) + (rest == 0 ? 0.0 : rest <= cus ? 0.75 : 1.0);
    return us + 2.0 + rounds * (glu ? (f32 ? 4.0 + 1.73 * nb : 3.0 + 0.94 * nb) : f32 ? 10.0 + 1.73 * nb : 6.5 + 0.94 * nb);
  }
  const long long tiles = up(N, glu ? 128 : 256) * up(M, 256);
  // rows of no whole 16 bytes: 16384 x 2003 x 2048 132 instead of 79 (tiles, which pass them through LDS, 105)
  if (glu) return 1.0 + (double)up(tiles, cus) * (5.5 + 1.35 * nb) * (N % 8 ? 1.2 : 1.0);
  return 5.0 + (N % 8 ? 1.6 : 1.0) * (double)up(tiles, cus) * (2.5 + (1.1 + 0.5 * std::min(1.0, (double)tiles / cus)) * nb);
}
// slices: 0 as many as pay, otherwise that many
Plan plan(int M, int N, int K, bool f32, bool glu, bool codes, int slices) {
  const bool few = M <= (glu ? 32 : 64), big = !f32 && K % 16 == 0;
  if (glu && few) return {SKINNY, 1, 0.0};
  if (codes) {
    // tiles of 64 rows, one to a compute unit, or of 256.  us, 64 / 256: 64 x 9216 x 768 9.2 / 16.2, 100 9.5 / 16.6, 300 17.3 / 18.0, 500 26 / 19, 1000 42 / 35;
    // 64 x 24576 x 2048 20 / 31, 100 29 / 32, 200 43 / 33; 700 x 2304 x 768 9.9 / 17.3
    const long long nb = (K + 127) / 128, tiles = ((N + 127) / 128) * (long long)((M + 63) / 64);
    const double us = 1.3 + (double)((tiles + fstu_cus() - 1) / fstu_cus()) * (2.6 + 0.6 * nb) + (double)N * K * 6e-8;
    return {us < estimate(LARGE, 1, M, N, K, false, true) ? TILE : LARGE, 1, us};
  }
  // the pair of more rows adds its blocks in one order on all kernels, so that its codes are those of its bf16 result
  const int least = std::max(slices, 1);
  const bool skinny = !glu && M <= 65535 * 32;           // rows over the grid's third side
  Plan best = {TILE, least, estimate(TILE, least, M, N, K, f32, glu)};
  if (skinny) {
    const double us = estimate(SKINNY, least, M, N, K, f32, glu);
    if (few || us < best.us) best = {SKINNY, least, us};
  }
  const auto take = [&](Kind kind, int s) {
    // a slice's second launch and sums cost a caller's host what a short call takes as well: they have to gain a microsecond
    const double us = estimate(kind, s, M, N, K, f32, glu) + (slices == 0 && s > 1 ? 1.0 : 0.0);
    if (us < best.us) best = {kind, s, us};
  };
  const int nb = (K + 127) / 128;
  static const int counts[] = {2, 3, 4, 6, 8, 12, 16};
  if (slices <= 1 && big && !few) take(LARGE, 1);
  if (slices == 0 && !glu)
    for (const int s : counts) {
      if (s > nb) break;
      if (skinny) take(SKINNY, s);
      if (!few) take(TILE, s);
    }
  return best;
}

}  // namespace
