// K10 -- softmax cross entropy of a linear head over a large vocabulary, its
// logits kept by neither pass, with its gradient.
//
//   z = x W^T                                  x [T, H], W [V, H]
//   lse_t = log sum_v exp(z_tv),  loss = norm * sum_t (lse_t - z_t,target(t))
//   d_tv = exp(z_tv - lse_t) - [v = target(t)]
//   dx = s * d W,  dW = s * d^T x,  s = dloss * norm
// over the tokens whose target is not `ignore_index`; norm = 1 / their count
// (mean; 0 where there is none) or 1 (sum).
//
// Matrix-bound.  Forward: the product's epilogue keeps, per token and 256
// columns, the maximum and the sum of exponentials of its accumulators and
// the target's logit; a second kernel joins those in column order.
// Backward: the vocabulary in pieces, each piece's logits computed again
// (one product of then four), turned in the epilogue into d in the operand
// type, and read by the two gradient products out of one buffer of at most
// half a gigabyte.  dx is summed over the pieces in 32 bits; dW's rows belong
// to one piece each.
//
// d is rounded to x's type once (float32: not, three planes; small heads: not,
// floats), which the results' own rounding hides (RMS error of the pass 2.1e-4 in
// float16, 1.7e-3 in bfloat16, with d in 32 bits the same).  It lies in
// [-1, 1]; for float16 it is held times 2^14, else the 1 / V of a
// large vocabulary would sit among float16's subnormal numbers; s and 2^-14
// are applied to the 32-bit sums.  A target outside [0, V) that is not
// ignore_index makes the loss and both gradients NaN and reads nothing.
//
// Small heads take the product of direct.h, whose k-runs are joined by the
// kernel that reduces a token's row (forward) or makes d of it; they, and few
// tiles cut along k, write their logits to the workspace, at most half a
// gigabyte (forward and backward of 32 x 256 x 10 float32 75 us on tiles, 20 so; 1 x 512 x 1000
// bfloat16 51, 26).
#include <type_traits>

#include "direct_tile.h"
#include "gemm_tile.h"

namespace p2p {

constexpr int64_t kPieceBytes = int64_t(512) << 20;
constexpr float kHalfScale = 16384.f;
constexpr int kAloneTokens = 32, kAloneLogits = 16384;  // tokens and partial logits of one block alone

// Per token and tile of columns: (maximum, sum of exp(z - maximum)).
struct StatsEpi {
  float2* part;        // [column tile][T]
  float* at_target;    // [T]
  const int64_t* target;
  int64_t first;       // vocabulary index of column 0
  int precise;

  template <class Cfg>
  __device__ __forceinline__ void finish(f4 (&acc)[Cfg::MI][Cfg::NJ], const Place& p, const GemmArgs& g, char* lds) const {
    const int i16 = p.lane & 15;
    const int64_t n0 = p.n0 + (p.lane >> 4) * 4;  // this lane's columns: n0 + Cfg::col(j) + e
    const int cols = static_cast<int>(std::min<int64_t>(g.N - n0, Cfg::BN));  // left from n0
    const bool whole = p.n0 + Cfg::HN + 32 <= g.N;  // of the wave's columns none is past the end
    float2* rows = reinterpret_cast<float2*>(lds);  // [WN][BM]
    // in steps over all of the lane's rows, so that their loads and exchanges wait together
    int t[Cfg::MI];  // the target among the lane's columns
#pragma unroll
    for (int i = 0; i < Cfg::MI; ++i) {
      const int64_t m = p.m0 + Cfg::row(i) + i16;
      const int64_t y = m < g.M ? ldg(target + m) - first - n0 : -1;
      t[i] = y >= 0 && y < cols ? static_cast<int>(y) : -1;
    }
    if (!whole) {
#pragma unroll
      for (int i = 0; i < Cfg::MI; ++i)
#pragma unroll
        for (int j = 0; j < Cfg::NJ; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (Cfg::col(j) + e >= cols) acc[i][j][e] = -INFINITY;
    }
    float top[Cfg::MI], s[Cfg::MI];
#pragma unroll
    for (int i = 0; i < Cfg::MI; ++i) {
      top[i] = -INFINITY;
#pragma unroll
      for (int j = 0; j < Cfg::NJ; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) top[i] = fmaxf(top[i], acc[i][j][e]);  // passes over a NaN, which the sum below takes up
    }
#pragma unroll
    for (int o = 16; o <= 32; o *= 2)
#pragma unroll
      for (int i = 0; i < Cfg::MI; ++i) top[i] = fmaxf(top[i], __shfl_xor(top[i], o, 64));
#pragma unroll
    for (int i = 0; i < Cfg::MI; ++i) {
      if (__any(t[i] >= 0)) {  // few tiles hold a token's target
#pragma unroll
        for (int j = 0; j < Cfg::NJ; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (Cfg::col(j) + e == t[i]) stg(at_target + p.m0 + Cfg::row(i) + i16, acc[i][j][e]);
      }
    }
    // (a choice of exponential for each element would compute both)
    const auto sums = [&](auto exponential) {
#pragma unroll
      for (int i = 0; i < Cfg::MI; ++i) {
        const float base = top[i] == -INFINITY ? 0.f : top[i];  // -inf throughout: a sum of zeros
        s[i] = 0.f;
#pragma unroll
        for (int j = 0; j < Cfg::NJ; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[i] += exponential(acc[i][j][e] - base);  // a column past the end: exp(-inf)
      }
    };
    if (precise) sums([](float x) { return expf(x); });
    else sums([](float x) { return __expf(x); });
#pragma unroll
    for (int o = 16; o <= 32; o *= 2)
#pragma unroll
      for (int i = 0; i < Cfg::MI; ++i) s[i] += __shfl_xor(s[i], o, 64);
    if (p.lane < 16)
#pragma unroll
      for (int i = 0; i < Cfg::MI; ++i) rows[p.wn * Cfg::BM + p.wm * Cfg::QM + Cfg::row(i) + i16] = make_float2(top[i], s[i]);
    __syncthreads();
    for (int r = threadIdx.x; r < Cfg::BM; r += Cfg::THREADS) {
      const int64_t m = static_cast<int64_t>(p.tm) * Cfg::BM + r;
      if (m >= g.M) continue;
      float2 a = rows[r];
#pragma unroll
      for (int w = 1; w < Cfg::WN; ++w) a = join_stats(a, rows[w * Cfg::BM + r]);
      part[p.tn * g.M + m] = a;
    }
  }

  // A part without a finite logit is (-inf, 0) and adds nothing.
  static __device__ __forceinline__ float2 join_stats(float2 a, float2 b) {
    if (b.y == 0.f && b.x == -INFINITY) return a;
    if (a.y == 0.f && a.x == -INFINITY) return b;
    const float top = fmaxf(a.x, b.x);
    return make_float2(top, a.y * expf(a.x - top) + b.y * expf(b.x - top));
  }
};

// loss and norm, by one block of 1024 in a fixed order, in 64 bits.
struct LossOut {
  const int64_t* target;
  int64_t T, ignore;
  int mean;
  float *loss, *norm;
};
// at(t): the token's loss and whether it counts.
template <typename At>
__device__ __forceinline__ void ce_loss_of(const At& at, const LossOut& o) {
  __shared__ double sums[16];
  __shared__ int64_t counts[16];
  double s = 0.0;
  int64_t n = 0;
  for (int64_t t = threadIdx.x; t < o.T; t += 1024) {
    const float2 l = at(t);
    s += static_cast<double>(l.x);
    n += l.y != 0.f;
  }
#pragma unroll
  for (int h = 32; h > 0; h >>= 1) {
    s += __shfl_xor(s, h, 64);
    n += __shfl_xor(n, h, 64);
  }
  if ((threadIdx.x & 63) == 0) {
    sums[threadIdx.x / 64] = s;
    counts[threadIdx.x / 64] = n;
  }
  __syncthreads();
  if (threadIdx.x == 0)
    for (int w = 1; w < 16; ++w) {
      sums[0] += sums[w];
      counts[0] += counts[w];
    }
  if (threadIdx.x == 0) {
    const double f = !o.mean ? 1.0 : counts[0] ? 1.0 / static_cast<double>(counts[0]) : 0.0;
    *o.loss = static_cast<float>(o.mean && counts[0] ? sums[0] / static_cast<double>(counts[0]) : sums[0]);
    *o.norm = static_cast<float>(f);
  }
}
__device__ __forceinline__ void ce_loss_of_rows(const float* row_loss, const LossOut& o) {
  ce_loss_of([&](int64_t t) { return make_float2(row_loss[t], o.target[t] != o.ignore ? 1.f : 0.f); }, o);
}
__global__ __launch_bounds__(1024) void ce_loss_kernel(const float* row_loss, LossOut o) { ce_loss_of_rows(row_loss, o); }

// Joins the column tiles of a piece, and with what earlier pieces left in
// `state`; after the last piece, lse and the token's loss.  64 tokens per
// block, a wave for every sixteenth of the tiles; one block sums the losses itself.
__global__ __launch_bounds__(1024) void ce_join_kernel(const float2* part, int tiles, float2* state, int first, int last,
                                                       int64_t V, const float* at_target, float* lse, float* row_loss,
                                                       LossOut o, unsigned gx) {
  const int64_t T = o.T;
  __shared__ float2 groups[16][64];
  const int lane = threadIdx.x & 63, group = threadIdx.x >> 6;
  const int64_t t = tile_id(gx) * 64 + lane;
  float2 a = make_float2(-INFINITY, 0.f);
  if (t < T) {
    const int from = tiles * group / 16, to = tiles * (group + 1) / 16;
#pragma unroll 8
    for (int i = from; i < to; ++i) a = StatsEpi::join_stats(a, part[i * T + t]);
  }
  groups[group][lane] = a;
  __syncthreads();
  if (group == 0 && t < T) {
#pragma unroll
    for (int q = 1; q < 16; ++q) a = StatsEpi::join_stats(a, groups[q][lane]);
    if (!first) a = StatsEpi::join_stats(state[t], a);
    if (!last) {
      state[t] = a;
    } else {
      lse[t] = a.x + logf(a.y);
      const int64_t y = o.target[t];
      // z - max and log(sum) apart: lse - z would lose the digits of a large maximum
      row_loss[t] = y == o.ignore ? 0.f : (y < 0 || y >= V) ? NAN : logf(a.y) - (at_target[t] - a.x);
    }
  }
  if (last && T <= 64) {
    __syncthreads();
    ce_loss_of_rows(row_loss, o);
  }
}

// Four values of d as operands of type T: float32 in planes `plane` elements apart, float16 times kHalfScale.
template <typename T>
__device__ __forceinline__ void store_d(uint16_t* to, int64_t plane, f4 x) {
  if constexpr (sizeof(T) == 4) {
    Pack<uint16_t, 4> o[3];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const Planes s = split3(x[e]);
#pragma unroll
      for (int q = 0; q < 3; ++q) o[q].v[e] = s.p[q];
    }
#pragma unroll
    for (int q = 0; q < 3; ++q) store_pack<uint16_t, 4>(to + q * plane, o[q]);
  } else {
    store4(reinterpret_cast<T*>(to), 0, 4, std::is_same_v<T, f16> ? x * kHalfScale : x);
  }
}

// d of a piece into its buffer [T, pitch] (planes `plane` elements apart).
struct GradEpi {
  uint16_t* d;
  int64_t pitch, plane;
  const float* lse;
  const int64_t* target;
  int64_t first, vocab, ignore;
  int32_t dtype;

  template <class Cfg>
  __device__ __forceinline__ void finish(f4 (&acc)[Cfg::MI][Cfg::NJ], const Place& p, const GemmArgs& g, char* lds) const {
    const int64_t own = row_of_lane<Cfg>(p);
    const int64_t y = own < g.M ? ldg(target + own) : ignore;
    const int counted = y != ignore;
    const float l = !counted ? 0.f : y >= 0 && y < vocab ? ldg(lse + own) : NAN;
    const int64_t n0 = static_cast<int64_t>(p.tn) * Cfg::BN;
    const int at = y >= first + n0 && y < first + n0 + Cfg::BN ? static_cast<int>(y - first - n0) : -1;  // in the tile
    const auto rows = [&](auto exponential, auto put) {
      by_rows<Cfg>(acc, p, lds, [&](int r, int64_t m, int64_t n, f4 v) {
        const float lr = from_lane<Cfg>(l, r);
        const int t = from_lane<Cfg>(at, r) - static_cast<int>(n - n0), c = from_lane<Cfg>(counted, r);
        if (m >= g.M || n >= pitch) return;
        f4 x;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = !c || n + e >= g.N ? 0.f : exponential(v[e] - lr) - (e == t ? 1.f : 0.f);
        put(d + m * pitch + n, x);
      });
    };
    const auto fast = [](float x) { return __expf(x); };
    if (dtype == P2P_DTYPE_F32) rows([](float x) { return expf(x); }, [&](uint16_t* to, f4 x) { store_d<float>(to, plane, x); });
    else if (dtype == P2P_DTYPE_F16) rows(fast, [&](uint16_t* to, f4 x) { store_d<f16>(to, plane, x); });
    else rows(fast, [&](uint16_t* to, f4 x) { store_d<bf16>(to, plane, x); });
  }
};

// The direct product's logits in k-runs [runs][T, V], a token per TEAM of a block's 1024 lanes: lse and the
// token's loss.  A block alone with few tokens sums their losses itself.
template <int TEAM>
__global__ __launch_bounds__(1024) void ce_row_kernel(const float* parts, int runs, int64_t V, float* lse, float* row_loss,
                                                      LossOut o) {
  constexpr int TEAMS = 1024 / TEAM, LANES = TEAM < 64 ? TEAM : 64;
  __shared__ float2 stats[16], losses[kAloneTokens];
  __shared__ float found[16];
  const int64_t T = o.T;
  const bool alone = gridDim.x == 1 && T <= kAloneTokens;
  const int lane = threadIdx.x % TEAM;
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * TEAMS + threadIdx.x / TEAM; t < T;
       t += static_cast<int64_t>(gridDim.x) * TEAMS) {
    const int64_t y = ldg(o.target + t);
    float2 a = make_float2(-INFINITY, 0.f);
    float at = 0.f;
    for (int64_t n = lane * 4; n < V; n += TEAM * 4) {
      float z[4];
      sum_runs<4>(parts + t * V, T * V, runs, n, V, z);
      float2 b = make_float2(-INFINITY, 0.f);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < V) {
          b.x = fmaxf(b.x, z[e]);
          if (n + e == y) at = z[e];
        }
      const float base = b.x == -INFINITY ? 0.f : b.x;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < V) b.y += expf(z[e] - base);
      a = StatsEpi::join_stats(a, b);
    }
    float top = a.x;
#pragma unroll
    for (int h = LANES / 2; h > 0; h >>= 1) top = fmaxf(top, __shfl_xor(top, h, 64));
    a = make_float2(top, a.y * expf(a.x - (top == -INFINITY ? 0.f : top)));
#pragma unroll
    for (int h = LANES / 2; h > 0; h >>= 1) {
      a.y += __shfl_xor(a.y, h, 64);
      at += __shfl_xor(at, h, 64);
    }
    if constexpr (TEAM > 64) {  // the whole block is on this token
      __syncthreads();
      if ((threadIdx.x & 63) == 0) stats[threadIdx.x / 64] = a, found[threadIdx.x / 64] = at;
      __syncthreads();
      a = stats[0], at = found[0];
      for (int w = 1; w < TEAM / 64; ++w) a = StatsEpi::join_stats(a, stats[w]), at += found[w];
    }
    if (lane == 0) {
      lse[t] = a.x + logf(a.y);
      const float l = y == o.ignore ? 0.f : (y < 0 || y >= V) ? NAN : logf(a.y) - (at - a.x);
      if (alone) losses[t] = make_float2(l, y != o.ignore ? 1.f : 0.f);
      else row_loss[t] = l;
    }
  }
  if (alone) {
    __syncthreads();
    ce_loss_of([&](int64_t t) { return losses[t]; }, o);
  }
}

// The same of few tokens with long rows: (maximum, sum) of 1024 logits of a token per block, joined by
// ce_join_kernel (loss forward, a block per row / in chunks: 2 x 258 x 91984 float16 84 / 47 us, 64 x 512 x 32000
// float32 50 / 40, 16 x 512 x 5000 18.6 / 16.1).
constexpr int kChunk = 1024;
__global__ __launch_bounds__(256) void ce_chunk_kernel(const float* parts, int runs, int64_t T, int64_t V, const int64_t* target,
                                                       float2* stats, float* at_target) {
  __shared__ float2 waves[4];
  const int64_t t = blockIdx.y, n = static_cast<int64_t>(blockIdx.x) * kChunk + threadIdx.x * 4, y = ldg(target + t);
  float z[4] = {0.f, 0.f, 0.f, 0.f};
  if (n < V && runs <= 2) add_runs<2, 4>(parts + t * V, T * V, runs, n, V, z);
  else if (n < V) sum_runs<4>(parts + t * V, T * V, runs, n, V, z);
  float2 a = make_float2(-INFINITY, 0.f);
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (n + e < V) {
      a.x = fmaxf(a.x, z[e]);
      if (n + e == y) stg(at_target + t, z[e]);
    }
#pragma unroll
  for (int h = 32; h > 0; h >>= 1) a.x = fmaxf(a.x, __shfl_xor(a.x, h, 64));
  const float base = a.x == -INFINITY ? 0.f : a.x;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (n + e < V) a.y += expf(z[e] - base);
  a.y = wave_sum(a.y);
  if ((threadIdx.x & 63) == 0) waves[threadIdx.x / 64] = a;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int w = 1; w < 4; ++w) a = StatsEpi::join_stats(a, waves[w]);
    stats[blockIdx.x * T + t] = a;
  }
}

// d of the logits in k-runs, over the first run.
__global__ __launch_bounds__(kBlock) void ce_grad_kernel(float* parts, int runs, int64_t T, int64_t V, const float* lse,
                                                         const int64_t* target, int64_t ignore) {
  const int64_t per_row = (V + 3) / 4, all = T * per_row;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x; i < all;
       i += static_cast<int64_t>(gridDim.x) * kBlock) {
    const int64_t t = i / per_row, n = (i - t * per_row) * 4;
    const int64_t y = ldg(target + t);
    const float l = y >= 0 && y < V ? ldg(lse + t) : NAN;
    float z[4];
    sum_runs<4>(parts + t * V, T * V, runs, n, V, z);
#pragma unroll
    for (int e = 0; e < 4; ++e) z[e] = y == ignore ? 0.f : expf(z[e] - l) - (n + e == y ? 1.f : 0.f);
    store_row<float, 4>(parts + t * V, n, V, z);
  }
}

// d as the tiles' gradient products read it: T, or three planes, [T, pitch], zeros past the last class.
template <typename T>
__global__ __launch_bounds__(kBlock) void ce_d_kernel(const float* parts, int runs, int64_t tokens, int64_t V, const float* lse,
                                                      const int64_t* target, int64_t ignore, uint16_t* d, int64_t pitch,
                                                      int64_t plane) {
  const int64_t per_row = pitch / 4, all = tokens * per_row;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x; i < all;
       i += static_cast<int64_t>(gridDim.x) * kBlock) {
    const int64_t t = i / per_row, n = (i - t * per_row) * 4;
    const int64_t y = ldg(target + t);
    const float l = y >= 0 && y < V ? ldg(lse + t) : NAN;
    f4 x = {0.f, 0.f, 0.f, 0.f};
    if (n < V && y != ignore) {
      float z[4];
      sum_runs<4>(parts + t * V, tokens * V, runs, n, V, z);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = n + e < V ? expf(z[e] - l) - (n + e == y ? 1.f : 0.f) : 0.f;
    }
    store_d<T>(d + t * pitch + n, plane, x);
  }
}

// The same, made where the gradients' products read it (again for every 64
// columns of x, against a launch).
struct CeGrad {
  const float* parts;
  int runs;
  int64_t T, V;
  const float* lse;
  const int64_t* target;
  int64_t ignore;

  struct Raw4 {
    float z[4], l;
    int at, in;  // the target among the four; how many of them are classes (0: the token does not count)
  };
  __device__ __forceinline__ Raw4 fetch(int64_t t, int64_t n, int64_t) const {
    Raw4 r;
    const int64_t y = ldg(target + t);
    r.l = y >= 0 && y < V ? ldg(lse + t) : NAN;
    sum_runs<4>(parts + t * V, T * V, runs, n, V, r.z);
    r.at = y >= n && y < n + 4 ? static_cast<int>(y - n) : -1;
    r.in = y == ignore || n >= V ? 0 : static_cast<int>(V - n < 4 ? V - n : 4);
    return r;
  }
  __device__ __forceinline__ void of(const Raw4& r, float (&v)[4]) const {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = e < r.in ? expf(r.z[e] - r.l) - (e == r.at ? 1.f : 0.f) : 0.f;
  }
};

static int32_t ce_check(const p2p_linear_ce_t* a) {
  if (!a || !known_dtype(a->dtype) || a->tokens < 0 || a->hidden < 1 || a->vocab < 1 || a->ldx < a->hidden ||
      a->ldw < a->hidden)
    return P2P_ERR_INVALID;
  const int64_t most = (int64_t(1) << 31) - 256;
  if (a->hidden > kMaxPitch - 8 || a->vocab > most || a->tokens > most) return P2P_ERR_UNSUPPORTED;
  if (!a->w || (a->tokens > 0 && (!a->x || !a->target || !a->lse)) || !a->norm) return P2P_ERR_INVALID;
  const int s = dtype_bytes(a->dtype);
  if (!aligned_to(a->x, s) || !aligned_to(a->w, s) || !aligned_to(a->target, 8) || !aligned_to(a->lse, 4) ||
      !aligned_to(a->norm, 4))
    return P2P_ERR_ALIGN;
  return P2P_OK;
}

struct CeSpace {
  int64_t piece;      // vocabulary rows per piece
  uint16_t *x, *w;    // packed x; packed rows of one piece of W
  // forward
  float2 *part, *state;
  float *at_target, *row_loss;
  float* z;           // few tiles: the logits in k-runs
  Plan z_plan;
  // backward
  uint16_t* d;
  float* dx_parts;
  Plan dx_plan;
  int64_t dw_floats;
  float* dw_parts;
};

static Plan ce_dw_plan(const p2p_linear_ce_t& a, int64_t rows) {
  return gemm_plan(rows, a.hidden, ksteps(a.tokens, a.dtype == P2P_DTYPE_F32 ? 6 : 1), true);
}

static bool ce_direct(const p2p_linear_ce_t& a) {
  return direct_pays(a.tokens, a.vocab, a.hidden, a.dtype) && a.tokens * a.vocab * 4 <= kPieceBytes;
}
// Whether the direct forward pass takes a token's row in chunks: rows of one block each would leave the chip idle.
static bool ce_chunked(const p2p_linear_ce_t& a) { return a.tokens <= 64 && a.vocab > 4 * kChunk; }
// Whether the direct gradients make d where they read it.  Backward, us, so /
// out of the logits' buffer: 32 x 256 x 10 float32 9.4 / 12.5, 1 x 512 x 1000
// bfloat16 13.8 / 14.8, 64 x 256 x 512 float32 17.7 / 17.2, 64 x 512 x 1000 22.0 / 19.7.
static bool ce_made_in_place(const p2p_linear_ce_t& a) {
  return static_cast<double>(a.tokens) * static_cast<double>(a.vocab) * static_cast<double>(a.hidden) <= 8.0e6;
}
// The logits' tile and runs.  Few tiles over a long sum are cut along k like the gradients; the runs are joined by the
// kernel that reduces a token's row (forward) or makes d (backward).  Forward, whole / in runs, us: 64 x 4096 x 4096
// bfloat16 52.6 / 24.6, 512 x 4096 x 1024 54.3 / 28.4, 1298 x 3618 x 920 60.1 / 41.8, 512 x 4096 x 2048 float32 274 / 95.
static Plan ce_logits_plan(const p2p_linear_ce_t& a, int64_t piece) {
  const int64_t steps = ksteps(a.hidden, a.dtype == P2P_DTYPE_F32 ? 6 : 1);
  const Plan p = gemm_plan(a.tokens, piece, steps, piece == a.vocab);
  return p.split * a.tokens * piece * 4 <= kPieceBytes ? p : gemm_plan(a.tokens, piece, steps, false);
}
// What the reduction of rows of logits needs besides them.
static void ce_take_rows(const p2p_linear_ce_t& a, Carver* c, CeSpace* s) {
  s->row_loss = static_cast<float*>(c->take(a.tokens * 4));
  if (!ce_chunked(a)) return;
  s->part = static_cast<float2*>(c->take(ceil_div(a.vocab, kChunk) * a.tokens * 8));
  s->at_target = static_cast<float*>(c->take(a.tokens * 4));
}
static int64_t ce_carve(const p2p_linear_ce_t& a, bool backward, void* base, CeSpace* s) {
  Carver c{static_cast<char*>(base)};
  if (ce_direct(a)) {
    *s = CeSpace{};
    const int64_t runs = direct_split(a.tokens, a.vocab, a.hidden, true);
    s->d = static_cast<uint16_t*>(c.take(runs * a.tokens * a.vocab * 4));
    if (!backward) {
      ce_take_rows(a, &c, s);
      return c.used;
    }
    const int64_t sx = direct_split(a.tokens, a.hidden, a.vocab, false), sw = direct_split(a.vocab, a.hidden, a.tokens, false);
    if (sx > 1) s->dx_parts = static_cast<float*>(c.take(sx * a.tokens * a.hidden * 4));
    if (sw > 1) s->dw_parts = static_cast<float*>(c.take(sw * a.vocab * a.hidden * 4));
    return c.used;
  }
  const int planes = planes_of(a.dtype);
  const bool x_here = in_place(a.x, a.ldx, a.hidden, a.dtype), w_here = in_place(a.w, a.ldw, a.hidden, a.dtype);
  // pieces: the buffers that grow with one stay under kPieceBytes (one tile's columns at least).  By shape and type alone,
  // since the sums over pieces are rounded piece by piece: a weight that is copied for its address or pitch only is
  // copied whole with its piece, however large
  int64_t per_row = backward ? a.tokens * 2 * planes : ceil_div(a.tokens * 8, Small::BN);
  if (a.dtype == P2P_DTYPE_F32 || a.hidden % 8) per_row = std::max(per_row, line_pitch(a.hidden) * 2 * planes);
  int64_t piece = std::max<int64_t>(1, kPieceBytes / per_row / Big::BN) * Big::BN;
  if (piece >= a.vocab) piece = a.vocab;
  else piece = round_up(ceil_div(a.vocab, ceil_div(a.vocab, piece)), Big::BN);  // pieces of about one size
  s->piece = piece;
  s->x = x_here ? nullptr : static_cast<uint16_t*>(c.take(packed_bytes(a.tokens, a.hidden, a.dtype)));
  s->w = w_here ? nullptr : static_cast<uint16_t*>(c.take(packed_bytes(piece, a.hidden, a.dtype)));
  s->z_plan = ce_logits_plan(a, piece);
  s->z = s->z_plan.split > 1 ? static_cast<float*>(c.take(s->z_plan.split * a.tokens * a.vocab * 4)) : nullptr;
  if (s->z && !backward) {
    s->part = nullptr;
    ce_take_rows(a, &c, s);
    return c.used;
  }
  if (!backward) {
    s->part = static_cast<float2*>(c.take(ceil_div(piece, Small::BN) * a.tokens * 8));
    s->state = static_cast<float2*>(c.take(a.tokens * 8));
    s->at_target = static_cast<float*>(c.take(a.tokens * 4));
    s->row_loss = static_cast<float*>(c.take(a.tokens * 4));
    return c.used;
  }
  const int nseg = a.dtype == P2P_DTYPE_F32 ? 6 : 1;
  s->d = static_cast<uint16_t*>(c.take(a.tokens * line_pitch(piece) * 2 * planes));
  s->dx_plan = gemm_plan(a.tokens, a.hidden, ksteps(piece, nseg), true);
  const bool parts = s->dx_plan.split > 1 || piece < a.vocab;
  s->dx_parts = parts ? static_cast<float*>(c.take(s->dx_plan.split * a.tokens * a.hidden * 4)) : nullptr;
  s->dw_floats = 0;
  for (const int64_t rows : {piece, a.vocab - (ceil_div(a.vocab, piece) - 1) * piece}) {
    const Plan pw = ce_dw_plan(a, rows);
    if (pw.split > 1) s->dw_floats = std::max(s->dw_floats, pw.split * rows * a.hidden);
  }
  s->dw_parts = s->dw_floats ? static_cast<float*>(c.take(s->dw_floats * 4)) : nullptr;
  return c.used;
}

// x (with the first piece) and the rows [v0, v0 + rows) of W as the products read them.
static int32_t ce_operands(const p2p_linear_ce_t& a, const CeSpace& s, int64_t v0, int64_t rows, Mat* x, Mat* w,
                           hipStream_t st) {
  const char* p = static_cast<const char*>(a.w) + v0 * a.ldw * dtype_bytes(a.dtype);
  const PackJob jobs[2] = {{p, a.ldw, rows, a.hidden, s.w, 0}, {a.x, a.ldx, a.tokens, a.hidden, s.x, 0}};
  *w = mat_of(jobs[0], a.dtype);
  *x = mat_of(jobs[1], a.dtype);
  return pack_matrices(jobs, v0 ? 1 : 2, a.dtype, st);
}

static LossOut ce_out(const p2p_linear_ce_t& a) {
  return LossOut{a.target, a.tokens, a.ignore_index, a.mean, a.loss, a.norm};
}

static int32_t ce_direct_logits(const p2p_linear_ce_t& a, const CeSpace& s, int* runs, hipStream_t st) {
  *runs = direct_split(a.tokens, a.vocab, a.hidden, true);
  const DirectArgs g{a.x, a.w, a.w, a.ldx, a.ldw, a.ldw, INT64_MAX, a.tokens, a.vocab, a.hidden, *runs,
                     {nullptr, nullptr}, INT64_MAX, {nullptr, nullptr}, reinterpret_cast<float*>(s.d)};
  return direct_product(g, a.dtype, st);
}

// lse and the loss out of the logits in k-runs.
static int32_t ce_rows(const p2p_linear_ce_t& a, const CeSpace& s, const float* z, int runs, hipStream_t st) {
  int32_t rc;
  if (ce_chunked(a)) {
    const int chunks = static_cast<int>(ceil_div(a.vocab, kChunk));
    ce_chunk_kernel<<<dim3(chunks, static_cast<unsigned>(a.tokens)), dim3(256), 0, st>>>(z, runs, a.tokens, a.vocab, a.target,
                                                                                         s.part, s.at_target);
    if ((rc = launch_status()) != P2P_OK) return rc;
    ce_join_kernel<<<dim3(1), dim3(1024), 0, st>>>(s.part, chunks, nullptr, 1, 1, a.vocab, s.at_target, a.lse, s.row_loss,
                                                   ce_out(a), 1);
    return launch_status();
  }
  // a token per 16 lanes, wave or block by the length of its row; few tokens in one block, which saves the launch
  // of the sum.  Forward, us: 32 x 784 x 10 float32 15.1 with a wave per token, 10.8 so; 32 x 512 x 512, of 131072
  // partial logits, 16.1 in one block, 13.3 in two; 64 x 128 x 100 17.5, 12.6.
  const int team = a.vocab <= 64 ? 16 : a.vocab <= 1024 ? 64 : 1024;
  const bool alone = a.tokens <= kAloneTokens && runs * a.tokens * a.vocab <= kAloneLogits;
  const int64_t blocks = alone && team < 1024 ? 1 : ceil_div(a.tokens, 1024 / team);
  const auto kernel = team == 16 ? ce_row_kernel<16> : team == 64 ? ce_row_kernel<64> : ce_row_kernel<1024>;
  kernel<<<dim3(static_cast<unsigned>(blocks)), dim3(1024), 0, st>>>(z, runs, a.vocab, a.lse, s.row_loss, ce_out(a));
  if ((rc = launch_status()) != P2P_OK || (blocks == 1 && a.tokens <= kAloneTokens)) return rc;
  ce_loss_kernel<<<dim3(1), dim3(1024), 0, st>>>(s.row_loss, ce_out(a));
  return launch_status();
}

static int32_t ce_direct_fwd(const p2p_linear_ce_t& a, const CeSpace& s, hipStream_t st) {
  int runs;
  const int32_t rc = ce_direct_logits(a, s, &runs, st);
  return rc == P2P_OK ? ce_rows(a, s, reinterpret_cast<const float*>(s.d), runs, st) : rc;
}

// The logits of all classes in k-runs, by tiles.
static int32_t ce_tile_logits(const p2p_linear_ce_t& a, const CeSpace& s, const Mat& x, const Mat& w, hipStream_t st) {
  GemmArgs g{};
  add_pairs(&g, x, w, nullptr, a.dtype);
  g.lda = x.ld, g.ldb = w.ld;
  g.M = a.tokens, g.N = a.vocab, g.K = a.hidden;
  g.ksplit = s.z_plan.split;
  const StoreEpi e{{nullptr, nullptr}, 0, 0, a.vocab, a.dtype, {nullptr, nullptr}, 1.f, s.z, 0};
  return gemm_launch<false, false, false>(g, a.dtype == P2P_DTYPE_F16, s.z_plan.big, e, st);
}
template <typename T>
static int32_t ce_tile_d(const p2p_linear_ce_t& a, const CeSpace& s, int64_t pitch, int64_t plane, hipStream_t st) {
  const int64_t blocks = ceil_div(a.tokens * (pitch / 4), kBlock);
  ce_d_kernel<T><<<dim3(static_cast<unsigned>(std::min<int64_t>(blocks, 256 * 32))), dim3(kBlock), 0, st>>>(
      s.z, s.z_plan.split, a.tokens, a.vocab, a.lse, a.target, a.ignore_index, s.d, pitch, plane);
  return launch_status();
}

static int32_t ce_direct_bwd(const p2p_linear_ce_t& a, const CeSpace& s, hipStream_t st) {
  int runs;
  int32_t rc = ce_direct_logits(a, s, &runs, st);
  if (rc != P2P_OK) return rc;
  const int64_t nx = a.tokens * a.hidden, nw = a.vocab * a.hidden;
  const int sx = direct_split(a.tokens, a.hidden, a.vocab, false), sw = direct_split(a.vocab, a.hidden, a.tokens, false);
  // dx = d W, dW = d^T x
  const DirectArgs x{nullptr, a.w, a.w, 0, a.ldw, a.ldw, INT64_MAX, a.tokens, a.hidden, a.vocab, sx,
                     {a.dx, nullptr}, INT64_MAX, {a.norm, a.dloss}, sx > 1 ? s.dx_parts : nullptr};
  const DirectArgs w{nullptr, a.x, a.x, 0, a.ldx, a.ldx, INT64_MAX, a.vocab, a.hidden, a.tokens, sw,
                     {a.dw, nullptr}, INT64_MAX, {a.norm, a.dloss}, sw > 1 ? s.dw_parts : nullptr};
  float* z = reinterpret_cast<float*>(s.d);
  const auto grads = [&](const auto& d) {
    using D = std::decay_t<decltype(d)>;
    return a.dtype == P2P_DTYPE_F32   ? direct_grads<D, float>(x, w, d, st)
           : a.dtype == P2P_DTYPE_F16 ? direct_grads<D, f16>(x, w, d, st)
                                      : direct_grads<D, bf16>(x, w, d, st);
  };
  if (ce_made_in_place(a)) {
    rc = grads(CeGrad{z, runs, a.tokens, a.vocab, a.lse, a.target, a.ignore_index});
  } else {
    const int64_t blocks = ceil_div(a.tokens * ceil_div(a.vocab, 4), kBlock);
    ce_grad_kernel<<<dim3(static_cast<unsigned>(std::min<int64_t>(blocks, 256 * 32))), dim3(kBlock), 0, st>>>(
        z, runs, a.tokens, a.vocab, a.lse, a.target, a.ignore_index);
    if ((rc = launch_status()) != P2P_OK) return rc;
    rc = grads(DirectLines<float>{z, z, a.vocab, a.vocab, INT64_MAX});
  }
  if (rc == P2P_OK && sx > 1) rc = join_parts(s.dx_parts, sx, nx, nx, 0, a.norm, a.dloss, 1.f, a.dx, nullptr, a.dtype, st);
  if (rc == P2P_OK && sw > 1) rc = join_parts(s.dw_parts, sw, nw, nw, 0, a.norm, a.dloss, 1.f, a.dw, nullptr, a.dtype, st);
  return rc;
}

}  // namespace p2p

using namespace p2p;

extern "C" int64_t p2p_linear_ce_workspace(const p2p_linear_ce_t* a, int32_t backward) {
  const int32_t rc = ce_check(a);
  if (rc != P2P_OK) return rc;
  CeSpace s;
  return a->tokens ? ce_carve(*a, backward != 0, nullptr, &s) : 0;
}

extern "C" int32_t p2p_linear_ce_fwd(const p2p_linear_ce_t* a, void* workspace, int64_t workspace_bytes,
                                     p2p_stream_t stream) {
  int32_t rc = ce_check(a);
  if (rc != P2P_OK) return rc;
  if (!a->loss) return P2P_ERR_INVALID;
  if (!aligned_to(a->loss, 4)) return P2P_ERR_ALIGN;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (a->tokens == 0) {  // the empty sum
    ce_loss_kernel<<<dim3(1), dim3(1024), 0, st>>>(nullptr, ce_out(*a));
    return launch_status();
  }
  CeSpace s;
  if (ce_carve(*a, false, workspace, &s) > workspace_bytes || !workspace) return P2P_ERR_INVALID;
  if (!aligned_to(workspace, 16)) return P2P_ERR_ALIGN;
  if (ce_direct(*a)) return ce_direct_fwd(*a, s, st);
  Mat x, w;
  if (s.z) {
    if ((rc = ce_operands(*a, s, 0, a->vocab, &x, &w, st)) != P2P_OK) return rc;
    if ((rc = ce_tile_logits(*a, s, x, w, st)) != P2P_OK) return rc;
    return ce_rows(*a, s, s.z, s.z_plan.split, st);
  }
  for (int64_t v0 = 0; v0 < a->vocab; v0 += s.piece) {
    const int64_t rows = std::min(s.piece, a->vocab - v0);
    if ((rc = ce_operands(*a, s, v0, rows, &x, &w, st)) != P2P_OK) return rc;
    GemmArgs g{};
    add_pairs(&g, x, w, nullptr, a->dtype);
    g.lda = x.ld, g.ldb = w.ld;
    g.M = a->tokens, g.N = rows, g.K = a->hidden;
    g.ksplit = 1;
    const StatsEpi e{s.part, s.at_target, a->target, v0, a->dtype == P2P_DTYPE_F32};
    const bool big = gemm_plan(g.M, g.N, ksteps(g.K, g.nseg), false).big;
    if ((rc = gemm_launch<false, false, false>(g, a->dtype == P2P_DTYPE_F16, big, e, st)) != P2P_OK) return rc;
    const int tiles = static_cast<int>(ceil_div(rows, big ? Big::BN : Small::BN));
    const TileGrid grid = tile_grid(ceil_div(a->tokens, 64), 1024);
    ce_join_kernel<<<dim3(grid.gx, grid.gy), dim3(1024), 0, st>>>(s.part, tiles, s.state, v0 == 0, v0 + rows == a->vocab,
                                                                  a->vocab, s.at_target, a->lse, s.row_loss, ce_out(*a),
                                                                  grid.gx);
    if ((rc = launch_status()) != P2P_OK) return rc;
  }
  if (a->tokens <= 64) return P2P_OK;  // the join's one block has summed the losses
  ce_loss_kernel<<<dim3(1), dim3(1024), 0, st>>>(s.row_loss, ce_out(*a));
  return launch_status();
}

extern "C" int32_t p2p_linear_ce_bwd(const p2p_linear_ce_t* a, void* workspace, int64_t workspace_bytes,
                                     p2p_stream_t stream) {
  int32_t rc = ce_check(a);
  if (rc != P2P_OK || a->tokens == 0) return rc;
  const int size = dtype_bytes(a->dtype);
  if (!a->dx || !a->dw) return P2P_ERR_INVALID;
  if (!aligned_to(a->dx, size) || !aligned_to(a->dw, size) || !aligned_to(a->dloss, 4)) return P2P_ERR_ALIGN;
  CeSpace s;
  if (ce_carve(*a, true, workspace, &s) > workspace_bytes || !workspace) return P2P_ERR_INVALID;
  if (!aligned_to(workspace, 16)) return P2P_ERR_ALIGN;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (ce_direct(*a)) return ce_direct_bwd(*a, s, st);
  const bool f16_ = a->dtype == P2P_DTYPE_F16;
  const float alpha = f16_ ? 1.f / kHalfScale : 1.f;
  Mat x, w;
  for (int64_t v0 = 0; v0 < a->vocab; v0 += s.piece) {
    const int64_t rows = std::min(s.piece, a->vocab - v0), pitch = line_pitch(rows), plane = a->tokens * pitch;
    if ((rc = ce_operands(*a, s, v0, rows, &x, &w, st)) != P2P_OK) return rc;
    if (s.z) {
      if ((rc = ce_tile_logits(*a, s, x, w, st)) != P2P_OK) return rc;
      rc = a->dtype == P2P_DTYPE_F32 ? ce_tile_d<float>(*a, s, pitch, plane, st)
           : f16_                    ? ce_tile_d<f16>(*a, s, pitch, plane, st)
                                     : ce_tile_d<bf16>(*a, s, pitch, plane, st);
      if (rc != P2P_OK) return rc;
    } else {
      GemmArgs g{};
      add_pairs(&g, x, w, nullptr, a->dtype);
      g.lda = x.ld, g.ldb = w.ld;
      g.M = a->tokens, g.N = rows, g.K = a->hidden;
      g.ksplit = 1;
      const GradEpi e{s.d, pitch, plane, a->lse, a->target, v0, a->vocab, a->ignore_index, a->dtype};
      const bool big = gemm_plan(g.M, g.N, ksteps(g.K, g.nseg), false).big;
      if ((rc = gemm_launch<false, false, false>(g, f16_, big, e, st)) != P2P_OK) return rc;
    }
    const Mat d{{s.d, s.d + plane, s.d + 2 * plane}, pitch};
    {  // dx += d W
      GemmArgs g{};
      add_pairs(&g, d, w, nullptr, a->dtype);
      g.lda = pitch, g.ldb = w.ld;
      g.M = a->tokens, g.N = a->hidden, g.K = rows;
      g.ksplit = s.dx_plan.split;
      const StoreEpi e{{a->dx, nullptr}, 0, 0, a->hidden, a->dtype, {a->norm, a->dloss}, alpha, s.dx_parts, v0 > 0};
      if ((rc = gemm_launch<false, true, false>(g, f16_, s.dx_plan.big, e, st)) != P2P_OK) return rc;
    }
    {  // dW of the piece = d^T x
      GemmArgs g{};
      add_pairs(&g, d, x, nullptr, a->dtype);
      g.lda = pitch, g.ldb = x.ld;
      g.M = rows, g.N = a->hidden, g.K = a->tokens;
      const Plan plan = ce_dw_plan(*a, rows);
      g.ksplit = plan.split;
      void* out = static_cast<char*>(a->dw) + v0 * a->hidden * size;
      const StoreEpi e{{out, nullptr}, 0, 0, a->hidden, a->dtype, {a->norm, a->dloss}, alpha,
                       plan.split > 1 ? s.dw_parts : nullptr, 0};
      if ((rc = gemm_launch<true, true, false>(g, f16_, plan.big, e, st)) != P2P_OK) return rc;
      if (plan.split > 1 && (rc = join_parts(s.dw_parts, plan.split, g.M * g.N, g.M * g.N, 0, a->norm, a->dloss, alpha,
                                             out, nullptr, a->dtype, st)) != P2P_OK)
        return rc;
    }
  }
  if (s.dx_parts) {
    const int64_t n = a->tokens * a->hidden;
    return join_parts(s.dx_parts, s.dx_plan.split, n, n, 0, a->norm, a->dloss, alpha, a->dx, nullptr, a->dtype, st);
  }
  return P2P_OK;
}
