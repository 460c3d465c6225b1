// A float32 product on the 32-bit matrix instructions, for sizes where the
// three-plane product (gemm_tile.h) would leave most of the chip idle and
// wait for its copies: C[m, n] = sum over k of A(m, k) * B(n, k), operands
// read where they lie, at any alignment and pitch.
#pragma once
#include "train_common.h"

namespace p2p {

struct DirectArgs {
  const float *a, *b, *b2;
  int64_t lda, ldb, ldb2;
  int64_t b_rows;  // lines of b; the further ones are b2's (INT64_MAX: b alone)
  int64_t M, N, K;
  int split;       // k-runs, whose sums go to partial[run][M][N] where that is given
  float* out[2];
  int64_t half;    // rows of out[0]; the further ones are out[1]'s (INT64_MAX: out[0] alone)
  const float* scale[2];
  float* partial;
};

// Whether a float32 product of this size goes this way.  Forward and backward
// of the gated layer, direct / planes: 32 x 512 x 512 46 / 82 us, 512 x 1024 x
// 1024 118 / 171, 1024 x 1024 x 1024 198 / 204, 1024 x 2048 x 1024 328 / 327,
// 2048 x 2048 x 2048 1153 / 673 us; 16 x 4096 x 8192 232 / 794 us.
// Few rows leave the planes' large tile empty and pay for copies of all of B.
static inline bool direct_pays(int64_t M, int64_t N, int64_t K) {
  return M <= 128 || static_cast<double>(M) * static_cast<double>(N) * static_cast<double>(K) <= 4.0e9;
}
// Its k-runs: enough blocks for every CU twice, at least two k-steps each.
P2P_INTERNAL int direct_split(int64_t M, int64_t N, int64_t K);

// AT / BT: the operand's lines are k (row-contiguous), else rows (k-contiguous).
P2P_INTERNAL int32_t direct_product(bool at, bool bt, const DirectArgs& g, hipStream_t st);

}  // namespace p2p
