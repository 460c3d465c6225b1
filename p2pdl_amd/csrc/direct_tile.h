// The tile of direct.h's product, over any source of its first operand.
//
// Tile 64 x 64 (32 x 64 for few rows) x 32 in two LDS images of pitch 36
// floats, on which a fragment's 16 rows of four floats fall on all 64 banks
// once.  A lane reads four neighbouring k of a row at once and feeds them to
// four v_mfma_f32_16x16x4_f32; the order of k within a step is the same for both
// operands.  The next step's elements are on their way to registers while
// this one's are multiplied (two steps ahead cost the fourth block of a CU its
// registers: 1024 x 1024 x 1024 float32 loss backward 98 us, 114); four blocks
// share a CU.  Few tiles are cut along k into runs, their sums joined in run
// order by the caller.
#pragma once
#include "direct.h"

namespace p2p {

using f4 = float __attribute__((ext_vector_type(4)));

constexpr int kDirectN = 64, kDirectK = 32, kDirectPitch = kDirectK + 4;
constexpr int kDirectLds = 2 * (64 + kDirectN) * kDirectPitch;  // floats

// Where four k (chunk k / 4) of a row lie in an image: on rows alone, a wave that stores 64 rows of 4 k transposed
// would meet itself four times on 16 banks (632 x 1800 x 873 float32 loss
// backward 107 us so, 99 with the chunks exchanged).
__device__ __forceinline__ int direct_at(int row, int chunk) { return row * kDirectPitch + ((chunk ^ (row >> 4 & 3)) << 2); }

// A source of an operand: fetch(i, c, cols) requests elements c .. c + 3 of
// line i (0 at and past `cols`), of(raw) makes them floats.  Between the two
// lies a step's products: a conversion at the load would wait for it there.

// A matrix in memory, of up to two parts.
template <typename E>
struct DirectLines {
  const E *p, *p2;
  int64_t ld, ld2, lines;  // lines of p; the further ones are p2's
  struct Raw4 {
    uint32_t w[sizeof(E)];
  };
  __device__ __forceinline__ Raw4 fetch(int64_t i, int64_t c, int64_t cols) const {
    const E* row = i < lines ? p + i * ld : p2 + (i - lines) * ld2;
    if (c + 4 <= cols) return __builtin_bit_cast(Raw4, load_pack<E, 4>(row + c));
    Pack<E, 4> v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v.v[e] = c + e < cols ? ldg(row + c + e) : static_cast<E>(0.f);
    return __builtin_bit_cast(Raw4, v);
  }
  __device__ __forceinline__ void of(const Raw4& r, float (&v)[4]) const {
    const Pack<E, 4> q = __builtin_bit_cast(Pack<E, 4>, r);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = static_cast<float>(q.v[e]);
  }
};

// EXT rows of an operand for one k-step: EXT / 8 elements per lane.  T: its lines are k, else rows.
template <class Src, bool T, int EXT>
struct DirectLoader {
  static constexpr int VECS = EXT / 32;  // vectors of four elements per lane
  const Src& src;
  int64_t rows, K;
  typename Src::Raw4 raw[VECS];

  __device__ __forceinline__ DirectLoader(const Src& s, int64_t r, int64_t k) : src(s), rows(r), K(k) {}
  __device__ __forceinline__ void load(int64_t row0, int64_t k0) {
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      const int q = i * 256 + threadIdx.x;
      const int64_t line = T ? k0 + q / (EXT / 4) : row0 + q / 8, c = T ? row0 + q % (EXT / 4) * 4 : k0 + q % 8 * 4;
      raw[i] = typename Src::Raw4{};
      if (line < (T ? K : rows)) raw[i] = src.fetch(line, c, T ? rows : K);
    }
  }
  __device__ __forceinline__ void store(float* image) const {
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      const int q = i * 256 + threadIdx.x;
      float v[4];
      src.of(raw[i], v);
      if constexpr (!T) {
        *reinterpret_cast<f4*>(image + direct_at(q / 8, q % 8)) = f4{v[0], v[1], v[2], v[3]};
      } else {
        const int row = q % (EXT / 4) * 4, k = q / (EXT / 4);
        float* to = image + direct_at(row, k / 4) + k % 4;
#pragma unroll
        for (int e = 0; e < 4; ++e) to[e * kDirectPitch] = v[e];
      }
    }
  }
};

// Tile `tile` of k-run `run` of the product g whose first operand is `sa`, by a block of 256.
template <class SA, typename TB, bool AT, bool BT, int BM>
__device__ __forceinline__ void direct_tile(const DirectArgs& g, const SA& sa, int tile, int run, float* lds) {
  constexpr int WM = BM / 32, WN = 4 / WM;                    // waves over the tile
  constexpr int MI = BM / WM / 16, NJ = kDirectN / WN / 16;   // 16 x 16 blocks of a wave
  constexpr int IMAGE_A = BM * kDirectPitch, IMAGE_B = kDirectN * kDirectPitch;
  static_assert(2 * (IMAGE_A + IMAGE_B) <= kDirectLds, "");
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / WN, wn = wave % WN;
  const int tiles_n = static_cast<int>(ceil_div(g.N, kDirectN));
  const int64_t m0 = static_cast<int64_t>(tile / tiles_n) * BM, n0 = static_cast<int64_t>(tile % tiles_n) * kDirectN;
  const int64_t steps = ceil_div(g.K, kDirectK);
  const int64_t first = steps * run / g.split, last = steps * (run + 1) / g.split;

  const DirectLines<TB> sb{static_cast<const TB*>(g.b), static_cast<const TB*>(g.b2), g.ldb, g.ldb2, g.b_rows};
  DirectLoader<SA, AT, BM> a(sa, g.M, g.K);
  DirectLoader<DirectLines<TB>, BT, kDirectN> b(sb, g.N, g.K);
  f4 acc[MI][NJ];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[i][j] = f4{0.f, 0.f, 0.f, 0.f};
  if (first < last) {
    a.load(m0, first * kDirectK);
    b.load(n0, first * kDirectK);
  }
  for (int64_t s = first; s < last; ++s) {
    float* ia = lds + ((s - first) & 1) * IMAGE_A;
    float* ib = lds + 2 * IMAGE_A + ((s - first) & 1) * IMAGE_B;
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
      for (int i = 0; i < MI; ++i) fa[i] = *reinterpret_cast<const f4*>(ia + direct_at((wm * MI + i) * 16 + (lane & 15), h * 4 + (lane >> 4)));
#pragma unroll
      for (int j = 0; j < NJ; ++j) fb[j] = *reinterpret_cast<const f4*>(ib + direct_at((wn * NJ + j) * 16 + (lane & 15), h * 4 + (lane >> 4)));
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
    float* sums = g.partial ? g.partial + (run * g.M + m) * g.N : nullptr;
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

// Both gradients of a linear layer out of d, in one launch: x.out = d B
// (x: lines of d are rows), then w.out = d^T B (w: lines of d are k), `sd`
// the source of d.  Two launches against one, us: gated layer 512 x 1024 x 1024
// float32 77.6 / 67.5, head 64 x 512 x 32000 114 / 97.
template <class SD, typename T>
__global__ __launch_bounds__(256) void direct_grads_kernel(DirectArgs x, DirectArgs w, SD sd, int x_tiles, int w_tiles) {
  __shared__ __attribute__((aligned(16))) float lds[kDirectLds];
  const int block = blockIdx.x, x_blocks = x_tiles * x.split;
  if (block < x_blocks) {
    if (x.M <= 32) direct_tile<SD, T, false, true, 32>(x, sd, block % x_tiles, block / x_tiles, lds);
    else direct_tile<SD, T, false, true, 64>(x, sd, block % x_tiles, block / x_tiles, lds);
  } else {
    const int b = block - x_blocks;
    if (w.M <= 32) direct_tile<SD, T, true, true, 32>(w, sd, b % w_tiles, b / w_tiles, lds);
    else direct_tile<SD, T, true, true, 64>(w, sd, b % w_tiles, b / w_tiles, lds);
  }
}
static inline int64_t direct_tiles(int64_t M, int64_t N) { return ceil_div(M, M <= 32 ? 32 : 64) * ceil_div(N, kDirectN); }
template <class SD, typename T>
static int32_t direct_grads(const DirectArgs& x, const DirectArgs& w, const SD& sd, hipStream_t st) {
  const int64_t tx = direct_tiles(x.M, x.N), tw = direct_tiles(w.M, w.N);
  if (tx * x.split + tw * w.split >= int64_t(1) << 23) return P2P_ERR_UNSUPPORTED;
  direct_grads_kernel<SD, T><<<dim3(static_cast<unsigned>(tx * x.split + tw * w.split)), dim3(256), 0, st>>>(
      x, w, sd, static_cast<int>(tx), static_cast<int>(tw));
  return launch_status();
}

}  // namespace p2p
