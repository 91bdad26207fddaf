// lbk_gated_plan.h — how the products of the dense gated FFN (lbk_gated.hip) run: plain host code on sizes.
#pragma once

#include <cstdint>
#include <initializer_list>

namespace lbk {

enum { EPI_STORE = 0, EPI_PART = 1, EPI_GATE = 2, EPI_GRAD = 3 };      // epilogues of gemm_kernel

constexpr int BK = 64;       // K of a stage

// Whether the weights are streamed: where the tokens' own reads, once a workgroup, do not outweigh the tiled
// kernel's idle columns.  us of a forward, streamed / tiled (33 tokens): 2048 / 8192 16 tokens 36 / 47, 32 tokens
// 51 / 47; 1024 / 4096 32 tokens 20 / 25; 4096 / 14336 16 tokens 93 / 95, 8 tokens 80.  Between 9 and 64 tokens either is far
// from the weights' 20 us at 2048 / 8192 (38 at 16, 50 at 32, 53 at 64): every workgroup of 16 features reads all tokens
// again here, and the tiled gate product has 128 workgroups for 256 CUs.
inline bool skinny(int64_t N, int64_t D, int64_t F) { return N <= 16 || (N <= 32 && D * F <= (int64_t)1 << 23); }

// How a product of M features, N columns and K (over all pairs) runs: output tiles of 256 or 128, K in
// `splits` shares.  The least of the estimated times in us: a 256 tile takes 1.75 a K stage and 8 more, one to
// a CU; a 128 tile 0.8 and 4 alone on a CU, 1.15 and 5 beside another; shares write their fp32 sums, and a
// second launch adds them up.  (Measured: 16384 x 1024, K 4096: 124 us with 256 tiles, 163 with 128 ones;
// 1024 x 4096, K 16384: 204 us with 128 tiles, 124 and the sums with 256 ones in four shares.)  EPI_GRAD's
// epilogue moves five times the results' bytes, which a 256 tile does not overlap with products of its own CU
// (16384 x 4096, K 1024: 293 us with 256 tiles, 301 with 128 ones; a training step of 4096 tokens: 429 and 422).
struct Plan {
  int tile, splits;
};
inline Plan plan(int64_t M, int64_t N, int64_t K, int parts, int epi, bool may_split) {
  Plan best{256, 1};
  double least = 1e30;
  const int64_t st = (K + BK - 1) / BK;
  for (int tile : {256, 128}) {
    const int64_t fm = epi == EPI_GATE ? tile / 2 : tile, t1 = (M + fm - 1) / fm * ((N + tile - 1) / tile) * parts;
    for (int s = 1; s <= 16 && (s == 1 || (may_split && st >= 4 * s)); s *= 2) {
      const int64_t t = t1 * s;
      const double k = (double)((st + s - 1) / s);
      double us;
      const bool grad = epi == EPI_GRAD;
      if (tile == 256) us = (double)((t + 255) / 256) * (1.75 * k + (grad ? 29 : 8)) + (grad ? 16 : 0);
      else us = t <= 256 ? 0.8 * k + (grad ? 13 : 4) : (double)((t + 511) / 512) * (1.15 * k + (grad ? 14 : 5));
      if (s > 1) us += 4 + (double)M * N * parts * (8 * s + 2) / 4.5e6;
      if (us < least) least = us, best = {tile, s};
    }
  }
  return best;
}

}  // namespace lbk
