// The product of direct.h.
//
// Tile 64 x 64 (32 x 64 for few rows) x 32 in two LDS images of pitch 36
// floats, on which a fragment's 16 rows of four floats fall on all 64 banks
// once.  A lane reads four neighbouring k of a row at once and feeds them to
// four v_mfma_f32_16x16x4_f32; the order of k within a step is the same for both
// operands.  The next step's elements are on their way to registers while
// this one's are multiplied; four blocks share a CU.  Few tiles are cut along
// k (grid.y), their sums joined in run order by the caller.
#include "direct.h"

#include <algorithm>

namespace p2p {

using f4 = float __attribute__((ext_vector_type(4)));

constexpr int kDirectN = 64, kDirectK = 32, kDirectPitch = kDirectK + 4;

// EXT rows of an operand for one k-step: EXT / 8 floats per lane.
template <typename E, bool T, int EXT>
struct DirectLoader {
  static constexpr int VECS = EXT / 32;  // vectors of four elements per lane
  const E *p, *p2;
  int64_t ld, ld2, lines, rows, K;
  float v[VECS][4];

  __device__ __forceinline__ const E* line(int64_t i) const { return i < lines ? p + i * ld : p2 + (i - lines) * ld2; }

  __device__ __forceinline__ void load(int64_t row0, int64_t k0) {
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      const int q = i * 256 + threadIdx.x;
      if constexpr (!T) {
        const int64_t r = row0 + q / 8;
        if (r < rows) load_row<E, 4>(line(r), k0 + q % 8 * 4, K, v[i]);
        else v[i][0] = v[i][1] = v[i][2] = v[i][3] = 0.f;
      } else {
        const int64_t k = k0 + q / (EXT / 4);
        if (k < K) load_row<E, 4>(line(k), row0 + q % (EXT / 4) * 4, rows, v[i]);
        else v[i][0] = v[i][1] = v[i][2] = v[i][3] = 0.f;
      }
    }
  }
  __device__ __forceinline__ void store(float* image) const {
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      const int q = i * 256 + threadIdx.x;
      if constexpr (!T) {
        *reinterpret_cast<f4*>(image + q / 8 * kDirectPitch + q % 8 * 4) = f4{v[i][0], v[i][1], v[i][2], v[i][3]};
      } else {
        float* to = image + q % (EXT / 4) * 4 * kDirectPitch + q / (EXT / 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) to[e * kDirectPitch] = v[i][e];
      }
    }
  }
};

template <typename TA, typename TB, bool AT, bool BT, int BM>
__global__ __launch_bounds__(256) void direct_kernel(DirectArgs g) {
  constexpr int WM = BM / 32, WN = 4 / WM;                    // waves over the tile
  constexpr int MI = BM / WM / 16, NJ = kDirectN / WN / 16;   // 16 x 16 blocks of a wave
  __shared__ __attribute__((aligned(16))) float la[2][BM * kDirectPitch], lb[2][kDirectN * kDirectPitch];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / WN, wn = wave % WN;
  const int tiles_n = static_cast<int>(ceil_div(g.N, kDirectN));
  const int64_t m0 = static_cast<int64_t>(blockIdx.x / tiles_n) * BM, n0 = static_cast<int64_t>(blockIdx.x % tiles_n) * kDirectN;
  const int64_t steps = ceil_div(g.K, kDirectK);
  const int64_t first = steps * blockIdx.y / g.split, last = steps * (blockIdx.y + 1) / g.split;

  DirectLoader<TA, AT, BM> a;
  DirectLoader<TB, BT, kDirectN> b;
  a.p = a.p2 = static_cast<const TA*>(g.a), a.ld = a.ld2 = g.lda, a.lines = INT64_MAX, a.rows = g.M, a.K = g.K;
  b.p = static_cast<const TB*>(g.b), b.p2 = static_cast<const TB*>(g.b2), b.ld = g.ldb, b.ld2 = g.ldb2, b.lines = g.b_rows, b.rows = g.N, b.K = g.K;
  f4 acc[MI][NJ];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[i][j] = f4{0.f, 0.f, 0.f, 0.f};
  if (first < last) {
    a.load(m0, first * kDirectK);
    b.load(n0, first * kDirectK);
  }
  const int at = (lane & 15) * kDirectPitch + (lane >> 4) * 4;
  for (int64_t s = first; s < last; ++s) {
    float* ia = la[(s - first) & 1];
    float* ib = lb[(s - first) & 1];
    a.store(ia);
    b.store(ib);
    __syncthreads();  // this image is whole; the other one's readers were done before their last barrier's successor
    if (s + 1 < last) {
      a.load(m0, (s + 1) * kDirectK);
      b.load(n0, (s + 1) * kDirectK);
    }
#pragma unroll
    for (int h = 0; h < kDirectK / 16; ++h) {
      f4 fa[MI], fb[NJ];
#pragma unroll
      for (int i = 0; i < MI; ++i) fa[i] = *reinterpret_cast<const f4*>(ia + (wm * MI + i) * 16 * kDirectPitch + at + h * 16);
#pragma unroll
      for (int j = 0; j < NJ; ++j) fb[j] = *reinterpret_cast<const f4*>(ib + (wn * NJ + j) * 16 * kDirectPitch + at + h * 16);
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
          for (int j = 0; j < NJ; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(fb[j][e], fa[i][e], acc[i][j], 0, 0, 0);
    }
  }
  float alpha = 1.f;
  if (!g.partial) {
    if (g.scale[0]) alpha *= ldc(g.scale[0]);
    if (g.scale[1]) alpha *= ldc(g.scale[1]);
  }
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    const int64_t m = m0 + (wm * MI + i) * 16 + (lane & 15);
    if (m >= g.M) continue;
    float* sums = g.partial ? g.partial + (blockIdx.y * g.M + m) * g.N : nullptr;
    TB* row = m < g.half ? static_cast<TB*>(g.out[0]) + m * g.N : static_cast<TB*>(g.out[1]) + (m - g.half) * g.N;
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int64_t n = n0 + (wn * NJ + j) * 16 + (lane >> 4) * 4;
      const float v[4] = {acc[i][j][0] * alpha, acc[i][j][1] * alpha, acc[i][j][2] * alpha, acc[i][j][3] * alpha};
      if (n >= g.N) continue;
      if (sums) store_row<float, 4>(sums, n, g.N, v);
      else store_row<TB, 4>(row, n, g.N, v);
    }
  }
}

int direct_split(int64_t M, int64_t N, int64_t K) {
  const int64_t tiles = ceil_div(M, M <= 32 ? 32 : 64) * ceil_div(N, kDirectN), steps = ceil_div(K, kDirectK);
  return static_cast<int>(std::max<int64_t>(1, std::min({512 / tiles, steps / 2, int64_t(32)})));
}

template <typename TA, typename TB, bool AT, bool BT>
static int32_t direct_run(const DirectArgs& g, hipStream_t st) {
  const bool low = g.M <= 32;
  const int64_t tiles = ceil_div(g.M, low ? 32 : 64) * ceil_div(g.N, kDirectN);
  if (tiles >= (int64_t(1) << 23)) return P2P_ERR_UNSUPPORTED;
  const dim3 grid(static_cast<unsigned>(tiles), g.split);
  if (low) direct_kernel<TA, TB, AT, BT, 32><<<grid, dim3(256), 0, st>>>(g);
  else direct_kernel<TA, TB, AT, BT, 64><<<grid, dim3(256), 0, st>>>(g);
  return launch_status();
}

// The products used: x W^T, and d (always float) with W or, both row-contiguous, with x.
template <typename T>
static int32_t direct_typed(bool at, bool bt, const DirectArgs& g, hipStream_t st) {
  if (at) return direct_run<float, T, true, true>(g, st);
  return bt ? direct_run<float, T, false, true>(g, st) : direct_run<T, T, false, false>(g, st);
}

int32_t direct_product(bool at, bool bt, const DirectArgs& g, hipStream_t st) {
  if (g.a_type != (bt ? P2P_DTYPE_F32 : g.b_type) || (at && !bt)) return P2P_ERR_INVALID;
  if (g.b_type == P2P_DTYPE_F32) return direct_typed<float>(at, bt, g, st);
  return g.b_type == P2P_DTYPE_F16 ? direct_typed<f16>(at, bt, g, st) : direct_typed<bf16>(at, bt, g, st);
}

}  // namespace p2p
