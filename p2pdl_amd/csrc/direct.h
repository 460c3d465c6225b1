// A product on the 32-bit matrix instructions, for sizes where the tiles of
// gemm_tile.h would leave most of the chip idle and wait for copies: C[m, n] =
// sum over k of A(m, k) * B(n, k), operands of any type read where they lie,
// at any alignment and pitch, and multiplied as floats.
#pragma once
#include "train_common.h"

namespace p2p {

struct DirectArgs {
  const void *a, *b, *b2;
  int64_t lda, ldb, ldb2;
  int64_t b_rows;  // lines of b; the further ones are b2's (INT64_MAX: b alone)
  int64_t M, N, K;
  int split;       // k-runs, whose sums go to partial[run][M][N] where that is given
  void* out[2];
  int64_t half;    // rows of out[0]; the further ones are out[1]'s (INT64_MAX: out[0] alone)
  const float* scale[2];
  float* partial;
};

// Whether a product of this size (N of the gated layer: 2 units) goes this
// way.  Forward and backward together, direct / tiles, us.  Gated layer,
// float32 (three planes in tiles): 1024 x 1024 x 512 105 / 108, 512 x 1024 x 1024
// 101 / 112, 632 x 1800 x 873 195 / 164, 1024 x 1024 x 1024 180 / 147; bfloat16: 256 x
// 256 x 512 32 / 38, 90 x 512 x 1000 34 / 40, 512 x 256 x 1024 53 / 46.  Loss, float32:
// 632 x 1800 x 873 151 / 155, 1024 x 1024 x 1024 143 / 149, 384 x 1128 x 4734 259 / 215,
// 4040 x 1560 x 389 328 / 242; bfloat16: 128 x 512 x 1000 49 / 57, 200 x 512 x 1000 61 /
// 62, 512 x 256 x 1024 61 / 61.  Up to 64 rows 16-bit tiles are half empty: 64 x 1001
// x 3001 loss 66 / 76.  Up to 32 rows the time of either is the weight's: loss 16 x 1024
// x 4096 47 / 58, 8 x 2048 x 4096 60 / 60, 2 x 2048 x 8192 83 / 66; gated layer 25 x 2119 x
// 1210 45 / 62, 16 x 1024 x 4096 43 / 43, 8 x 2048 x 4096 63 / 51; rows that tiles have to
// copy first: loss 2 x 258 x 91984 float16 130 / 200.  Float32 pays for copies of
// all of B besides, whatever the weight up to 192 rows: loss 64 x 512 x 32000 136 / 303, 128
// x 4096 x 4096 226 / 258, 192 x 1024 x 8192 182 / 189, 256 x 1024 x 8192 231 / 205.
// Up to 2^24 rows and columns: its tiles and the rows of its epilogues then fit one
// dimension of a grid.
static inline bool direct_pays(int64_t M, int64_t N, int64_t K, int32_t dtype) {
  const double weight = static_cast<double>(N) * static_cast<double>(K), size = static_cast<double>(M) * weight;
  if (M > 1 << 24 || N > 1 << 24) return false;
  if (dtype == P2P_DTYPE_F32) return M <= 192 || size <= 1.3e9;
  return M <= 32 ? weight <= (K % 8 ? 3.0e7 : 9.0e6) : size <= (M <= 64 ? 2.0e8 : 1.0e8);
}
// Its k-runs, at least two k-steps each.  The forward pass joins them anyway:
// blocks for every CU four times, up to as many runs as a lane's loads take at
// once (sum_runs; 32 x 784 x 10 float32 19.1 us with up to 32 runs, 15.0 with 8, 16.9
// with 4; 632 x 1800 x 873 gated forward 89 us with two blocks per CU, 61 with four).
// Gradients: blocks for every CU twice, or four times where a run would
// still be 28 steps long (4 x 2608 x 96752 968 -> 830 us, but 512 x 1024 x 1024 60 ->
// 64), up to 128 runs (1 x 108 x 6640 bfloat16 24 us with 32, 13 with 128).
P2P_INTERNAL int direct_split(int64_t M, int64_t N, int64_t K, bool forward);

// A B^T, both operands' lines their rows, of one type.
P2P_INTERNAL int32_t direct_product(const DirectArgs& g, int32_t dtype, hipStream_t st);

}  // namespace p2p
