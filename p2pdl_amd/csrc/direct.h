// A product on the 32-bit matrix instructions, for sizes where the tiles of
// gemm_tile.h would leave most of the chip idle and wait for copies: C[m, n] =
// sum over k of A(m, k) * B(n, k), operands of any type read where they lie,
// at any alignment and pitch, and multiplied as floats.
#pragma once
#include "train_common.h"

namespace p2p {

struct DirectArgs {
  const void *a, *b, *b2;
  int32_t a_type, b_type;  // of the operands; b_type also of out
  int64_t lda, ldb, ldb2;
  int64_t b_rows;  // lines of b; the further ones are b2's (INT64_MAX: b alone)
  int64_t M, N, K;
  int split;       // k-runs, whose sums go to partial[run][M][N] where that is given
  void* out[2];
  int64_t half;    // rows of out[0]; the further ones are out[1]'s (INT64_MAX: out[0] alone)
  const float* scale[2];
  float* partial;
};

// Whether a product of this size goes this way.  Forward and backward of the
// gated layer, direct / tiles, us.  Float32 (three planes in tiles): 32 x 512 x
// 512 46 / 82, 512 x 1024 x 1024 118 / 171, 1024 x 1024 x 1024 198 / 204, 1024 x
// 2048 x 1024 328 / 327, 2048 x 2048 x 2048 1153 / 673; few rows leave the tiles
// empty and pay for copies of all of B: 16 x 4096 x 8192 232 / 794.  bfloat16:
// 1 x 512 x 1000 28 / 35, 256 x 256 x 512 38 / 41, 90 x 512 x 1000 42 / 43, 512 x 256 x
// 1024 65 / 47 (the loss: 31 / 51, 44 / 55, 49 / 61, 65 / 61).  Up to 2^24 rows and
// columns: its 64 x 64 tiles and the rows of its epilogues then fit one dimension of a grid.
static inline bool direct_pays(int64_t M, int64_t N, int64_t K, int32_t dtype) {
  const double size = static_cast<double>(M) * static_cast<double>(N) * static_cast<double>(K);
  if (M > 1 << 24 || N > 1 << 24) return false;
  return dtype == P2P_DTYPE_F32 ? M <= 128 || size <= 4.0e9 : size <= 6.0e7;
}
// Its k-runs: enough blocks for every CU twice, at least two k-steps each.
P2P_INTERNAL int direct_split(int64_t M, int64_t N, int64_t K);

// AT / BT: the operand's lines are k (row-contiguous), else rows (k-contiguous).
P2P_INTERNAL int32_t direct_product(bool at, bool bt, const DirectArgs& g, hipStream_t st);

}  // namespace p2p
