// The product of direct.h with its first operand in memory.
#include "direct_tile.h"

#include <algorithm>

namespace p2p {

template <typename T, int BM>
__global__ __launch_bounds__(256) void direct_kernel(DirectArgs g) {
  __shared__ __attribute__((aligned(16))) float lds[kDirectLds];
  const DirectLines<T> a{static_cast<const T*>(g.a), static_cast<const T*>(g.a), g.lda, g.lda, INT64_MAX};
  direct_tile<DirectLines<T>, T, false, false, BM>(g, a, blockIdx.x, blockIdx.y, lds);
}

int direct_split(int64_t M, int64_t N, int64_t K, bool forward) {
  const int64_t tiles = direct_tiles(M, N), steps = ceil_div(K, kDirectK);
  const int64_t blocks = forward || steps * tiles > 512 * 28 ? 1024 : 512, most = forward ? 8 : 128;
  return static_cast<int>(std::max<int64_t>(1, std::min({blocks / tiles, steps / 2, most})));
}

template <typename T>
static int32_t direct_run(const DirectArgs& g, hipStream_t st) {
  const int64_t tiles = direct_tiles(g.M, g.N);
  if (tiles >= (int64_t(1) << 23)) return P2P_ERR_UNSUPPORTED;
  const dim3 grid(static_cast<unsigned>(tiles), g.split);
  if (g.M <= 32) direct_kernel<T, 32><<<grid, dim3(256), 0, st>>>(g);
  else direct_kernel<T, 64><<<grid, dim3(256), 0, st>>>(g);
  return launch_status();
}

int32_t direct_product(const DirectArgs& g, int32_t dtype, hipStream_t st) {
  if (dtype == P2P_DTYPE_F32) return direct_run<float>(g, st);
  return dtype == P2P_DTYPE_F16 ? direct_run<f16>(g, st) : direct_run<bf16>(g, st);
}

}  // namespace p2p
