// K7 -- layer norm of a trainer's local step, forward and backward.
//
//   y  = (x - mean) * rstd * w + b,  rstd = 1 / sqrt(mean((x - mean)^2) + eps)
//   dx = rstd * (g - mean(g) - xh * mean(g * xh)),  g = dy * w, xh = (x - mean) * rstd
//   dw = sum over rows of dy * xh,  db = sum over rows of dy
//
// HBM-bound (about 20 operations for 8 bytes of a 16-bit element), so every
// element is moved once: a team of lanes holds a whole row in registers, 16
// bytes per lane and load, and takes the mean and then the squared
// deviations from what it holds (the two-pass variance, without a second
// read and without the cancellation of E[x^2] - mean^2).  The backward pass
// keeps dw and db of its columns in registers over all rows of a block and
// writes one partial row per block; a second kernel adds the partials in
// their order, so the gradients' bits do not depend on timing.
#include <algorithm>
#include <type_traits>

#include "train_common.h"

namespace p2p {

constexpr int kLnMaxCols = 16384;
constexpr int kLnFwdBlock = 256;
constexpr int kLnBwdBlock = 512;
constexpr int kLnAlone = 8;  // passes over its rows that one block makes alone
constexpr int kLnMaxParts = 512;  // partial rows of dw / db: two blocks of 512 lanes per CU

// How a row's 16-byte vectors fit it.  DENSE: its length is a multiple of them.
// SHIFTED: the last one is moved back to the row's end, over elements of the
// one before, which count once in the sums and are computed and stored
// twice, alike (a tail of single elements costs its wave a load and a store
// each: 4099 x 1001 float16 takes 23.3 us a pass with it, 21.1 us so).  SHORT: rows of less
// than one vector, element by element.
enum Fit { SHORT, DENSE, SHIFTED };
template <typename T, Fit FIT>
struct Span {
  int c, at;  // first element that counts, first element
  bool in;
  __device__ __forceinline__ Span(int vec, int cols) {
    constexpr int V = Vec16<T>::N;
    c = vec * V;
    in = c < cols;
    at = FIT == SHIFTED && c + V > cols ? cols - V : c;
  }
  __device__ __forceinline__ bool counts(int e, int cols) const {
    return FIT == DENSE ? in : FIT == SHIFTED ? in && at + e >= c : c + e < cols;
  }
};

// Sum over a team of TEAM lanes (one wave, or several through LDS: then every
// lane of the block must call it).
template <int TEAM, int BLOCK>
__device__ __forceinline__ float team_sum(float v, float* scratch) {
  v = wave_sum(v);
  if constexpr (TEAM > 64) {
    constexpr int W = TEAM / 64;
    const int wave = threadIdx.x / 64;
    __syncthreads();  // the scratch of the last sum has been read
    if ((threadIdx.x & 63) == 0) scratch[wave] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) v += scratch[(wave / W) * W + i];
  }
  return v;
}

template <typename T, int TEAM, int NV, Fit FIT>
__global__ __launch_bounds__(kLnFwdBlock < TEAM ? TEAM : kLnFwdBlock) void layernorm_fwd_kernel(
    const T* x, int64_t ldx, const T* w, const T* b, int64_t rows, int cols, float eps, T* y, float* mean_out,
    float* rstd_out, unsigned gx) {
  constexpr int BLOCK = kLnFwdBlock < TEAM ? TEAM : kLnFwdBlock;
  constexpr int V = Vec16<T>::N;
  __shared__ float scratch[BLOCK / 64];
  const int lane = threadIdx.x % TEAM;
  const int64_t row = tile_id(gx) * (BLOCK / TEAM) + threadIdx.x / TEAM;
  const int have = row < rows ? cols : 0;  // surplus teams of the last block hold an empty row
  const T* xr = x + row * ldx;
  float v[NV][V];
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const Span<T, FIT> p(i * TEAM + lane, have);
    const Raw r = p.in ? load_raw<T, FIT != SHORT>(xr, p.at, have) : Raw{{0u, 0u, 0u, 0u}};
#pragma unroll
    for (int e = 0; e < V; ++e) {
      v[i][e] = raw_at<T>(r, e);
      s += p.counts(e, have) ? v[i][e] : 0.f;
    }
  }
  const float mean = team_sum<TEAM, BLOCK>(s, scratch) / static_cast<float>(cols);
  s = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const Span<T, FIT> p(i * TEAM + lane, have);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      v[i][e] -= mean;
      s += p.counts(e, have) ? v[i][e] * v[i][e] : 0.f;
    }
  }
  const float rstd = 1.f / sqrtf(team_sum<TEAM, BLOCK>(s, scratch) / static_cast<float>(cols) + eps);
  if (row >= rows) return;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const Span<T, FIT> p(i * TEAM + lane, cols);
    if (!p.in) continue;
    float wv[V], bv[V], o[V];
#pragma unroll
    for (int e = 0; e < V; ++e) wv[e] = 1.f, bv[e] = 0.f;
    if (w) load_row<T, V>(w, p.at, cols, wv);
    if (b) load_row<T, V>(b, p.at, cols, bv);
#pragma unroll
    for (int e = 0; e < V; ++e) o[e] = v[i][e] * rstd * wv[e] + bv[e];
    store_row<T, V, FIT != SHORT>(y + row * cols, p.at, cols, o);
  }
  if (lane == 0) {
    mean_out[row] = mean;
    rstd_out[row] = rstd;
  }
}

// Block q takes the rows (it * gridDim.x + q) * teams + team; parts[q] is its
// row of 2 * cols sums: dw, then db.  The next row's x and dy are requested
// before this one is worked on (rows of up to 4096) and rows are held as they
// lie, two registers per four 16-bit elements, so that two blocks fit a CU:
// 16384 x 4096 bf16 in 143.6 us without either, 84 us (4.8 TB/s) with.
template <typename T, int TEAM, int NV, Fit FIT>
__global__ __launch_bounds__(kLnBwdBlock, NV * Vec16<T>::N <= 8 ? 4 : 2) void layernorm_bwd_kernel(
    const T* dy, int64_t lddy, const T* x, int64_t ldx, const T* w, const float* mean_in, const float* rstd_in, int64_t rows,
    int cols, T* dx, float* parts, T* dw, T* db) {
  constexpr int V = Vec16<T>::N;
  constexpr int TEAMS = kLnBwdBlock / TEAM, WAVES = TEAM / 64;
  __shared__ float2 sums[2][kLnBwdBlock / 64];
  __shared__ float joined[TEAMS > 1 ? kLnBwdBlock * V : 1];
  const int lane = threadIdx.x % TEAM, team = threadIdx.x / TEAM, wave = threadIdx.x / 64;
  float dwv[NV][V], dbv[NV][V];
  Raw wv[NV], xv[NV], gv[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
#pragma unroll
    for (int e = 0; e < V; ++e) dwv[i][e] = 0.f, dbv[i][e] = 0.f;
    const Span<T, FIT> p(i * TEAM + lane, cols);
    if (w && p.in) wv[i] = load_raw<T, FIT != SHORT>(w, p.at, cols);
    else wv[i] = Raw{{0u, 0u, 0u, 0u}};
  }
  const float inv = 1.f / static_cast<float>(cols);
  const int64_t step = static_cast<int64_t>(gridDim.x) * TEAMS;
  int64_t row = static_cast<int64_t>(blockIdx.x) * TEAMS + team;
  float mean = 0.f, rstd = 0.f;
  const auto request = [&](int64_t r) {
    const int have = r < rows ? cols : 0;
    mean = have ? ldg(mean_in + r) : 0.f;
    rstd = have ? ldg(rstd_in + r) : 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const Span<T, FIT> p(i * TEAM + lane, have);
      xv[i] = gv[i] = Raw{{0u, 0u, 0u, 0u}};
      if (p.in) {
        xv[i] = load_raw<T, FIT != SHORT>(x + r * ldx, p.at, have);
        gv[i] = load_raw<T, FIT != SHORT>(dy + r * lddy, p.at, have);
      }
    }
  };
  constexpr bool AHEAD = NV * V <= 8;
  if (AHEAD) request(row);
  int parity = 0;
  for (int64_t first = static_cast<int64_t>(blockIdx.x) * TEAMS; first < rows; first += step, row += step, parity ^= 1) {
    const int have = row < rows ? cols : 0;
    if (!AHEAD) request(row);
    const float mu = mean, rs = rstd;
    Raw xc[NV], gc[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) xc[i] = xv[i], gc[i] = gv[i];
    if (AHEAD) request(row + step);
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const Span<T, FIT> p(i * TEAM + lane, have);
      forget(wv[i]);
      // past the row x and dy are 0 and so is what they add to the sums, if h is: (0 - mean) * rstd may be an infinity
      const float mi = p.in ? mu : 0.f;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float h = (raw_at<T>(xc[i], e) - mi) * rs;
        if (FIT == SHORT) h = p.counts(e, have) ? h : 0.f;
        const float d = raw_at<T>(gc[i], e);
        float g = w ? d * raw_at<T>(wv[i], e) : d;
        dwv[i][e] += d * h;
        dbv[i][e] += d;
        if (FIT == SHIFTED) g = p.counts(e, have) ? g : 0.f;
        s1 += g;
        s2 += g * h;
      }
      forget(wv[i]);
      forget(xc[i]);
      forget(gc[i]);
    }
    s1 = wave_sum(s1);
    s2 = wave_sum(s2);
    if constexpr (WAVES > 1) {
      // one barrier per row: the sums of the row after next go to the same place, behind the next one's barrier
      if ((threadIdx.x & 63) == 0) sums[parity][wave] = make_float2(s1, s2);
      __syncthreads();
      s1 = s2 = 0.f;
#pragma unroll
      for (int i = 0; i < WAVES; ++i) {
        const float2 v = sums[parity][wave / WAVES * WAVES + i];
        s1 += v.x;
        s2 += v.y;
      }
    }
    s1 *= inv;
    s2 *= inv;
    if (have) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const Span<T, FIT> p(i * TEAM + lane, cols);
        float o[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float h = (raw_at<T>(xc[i], e) - mu) * rs;
          const float d = raw_at<T>(gc[i], e);
          o[e] = rs * ((w ? d * raw_at<T>(wv[i], e) : d) - s1 - h * s2);
        }
        if (p.in) store_row<T, V, FIT != SHORT>(dx + row * cols, p.at, cols, o);
      }
    }
  }
  if (!parts && !dw && !db) return;
  float* out = parts + static_cast<int64_t>(blockIdx.x) * 2 * cols;
  // the teams' sums of each column, added in team order by the first team
#pragma unroll
  for (int which = 0; which < 2; ++which)
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float (&v)[V] = which ? dbv[i] : dwv[i];
      if constexpr (TEAMS > 1) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < V; ++e) joined[e * kLnBwdBlock + threadIdx.x] = v[e];
        __syncthreads();
        if (team == 0)
#pragma unroll
          for (int e = 0; e < V; ++e)
#pragma unroll
            for (int t = 1; t < TEAMS; ++t) v[e] += joined[e * kLnBwdBlock + t * TEAM + lane];
      }
      const Span<T, FIT> p(i * TEAM + lane, cols);
      if (team == 0 && p.in) {
        T* const whole = which ? db : dw;  // a block alone has the whole sums
        if (parts) store_row<float, V, FIT != SHORT>(out + which * cols, p.at, cols, v);
        else if (whole) store_row<T, V, FIT != SHORT>(whole, p.at, cols, v);
      }
    }
}

// dw / db from the partial rows: 64 columns per block, 16 groups of rows.
template <typename T>
__global__ __launch_bounds__(1024) void layernorm_parts_kernel(const float* parts, int nparts, int cols, T* dw, T* db) {
  __shared__ float sums[16][64];
  const int lane = threadIdx.x & 63, group = threadIdx.x >> 6;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 64 + lane;
  float s = 0.f;
  if (c < 2 * static_cast<int64_t>(cols)) {
#pragma unroll 8
    for (int p = group; p < nparts; p += 16) s += ldg(parts + static_cast<int64_t>(p) * 2 * cols + c);
  }
  sums[group][lane] = s;
  __syncthreads();
  if (group || c >= 2 * static_cast<int64_t>(cols)) return;
#pragma unroll
  for (int q = 1; q < 16; ++q) s += sums[q][lane];
  if (c < cols) {
    if (dw) dw[c] = static_cast<T>(s);
  } else if (db) {
    db[c - cols] = static_cast<T>(s);
  }
}

// Team and vectors per lane of the backward pass by the row's 16-byte
// vectors: as few elements per lane as there are lanes for (8, so that the
// next row's fit beside them in 128 registers), teams of up to 512.
template <typename T, typename F>
static void ln_team(int cols, F&& go) {
  using std::integral_constant;
  const int vecs = static_cast<int>(ceil_div(cols, Vec16<T>::N));
  if constexpr (sizeof(T) == 4) {
    if (vecs <= 128) go(integral_constant<int, 64>(), integral_constant<int, 2>());
    else if (vecs <= 512) go(integral_constant<int, 256>(), integral_constant<int, 2>());
    else if (vecs <= 1024) go(integral_constant<int, 512>(), integral_constant<int, 2>());
    else if (vecs <= 2048) go(integral_constant<int, 512>(), integral_constant<int, 4>());
    else go(integral_constant<int, 512>(), integral_constant<int, 8>());
  } else {
    if (vecs <= 64) go(integral_constant<int, 64>(), integral_constant<int, 1>());
    else if (vecs <= 128) go(integral_constant<int, 128>(), integral_constant<int, 1>());
    else if (vecs <= 256) go(integral_constant<int, 256>(), integral_constant<int, 1>());
    else if (vecs <= 512) go(integral_constant<int, 512>(), integral_constant<int, 1>());
    else if (vecs <= 1024) go(integral_constant<int, 512>(), integral_constant<int, 2>());
    else go(integral_constant<int, 512>(), integral_constant<int, 4>());
  }
}

// Forward: teams of 256 from 128 vectors up (16384 x 4096 bf16: 56 us, 64 us
// with teams of 512, which wait for each other's sums).
template <typename T, typename F>
static void ln_fwd_team(int cols, F&& go) {
  using std::integral_constant;
  const int vecs = static_cast<int>(ceil_div(cols, Vec16<T>::N));
  if (vecs <= 64) go(integral_constant<int, 64>(), integral_constant<int, 1>());
  else if (vecs <= 128) go(integral_constant<int, 64>(), integral_constant<int, 2>());
  else if (vecs <= 256) go(integral_constant<int, 256>(), integral_constant<int, 1>());
  else if (vecs <= 512) go(integral_constant<int, 256>(), integral_constant<int, 2>());
  else if (vecs <= 1024) go(integral_constant<int, 512>(), integral_constant<int, 2>());
  else if (vecs <= 2048) go(integral_constant<int, 512>(), integral_constant<int, 4>());
  else if constexpr (sizeof(T) == 4) go(integral_constant<int, 512>(), integral_constant<int, 8>());
}

template <typename T>
static int ln_parts_of(int64_t rows, int cols) {
  int teams = 1;
  ln_team<T>(cols, [&](auto team, auto) { teams = kLnBwdBlock / decltype(team)::value; });
  // few rows: one block, which needs no second launch
  const int64_t blocks = ceil_div(rows, teams);
  return static_cast<int>(blocks <= kLnAlone ? 1 : std::min<int64_t>(blocks, kLnMaxParts));
}
static int ln_parts(int64_t rows, int cols, int32_t dtype) {
  return dtype == P2P_DTYPE_F32 ? ln_parts_of<float>(rows, cols) : ln_parts_of<f16>(rows, cols);
}

template <typename T>
static int32_t ln_fwd(const T* x, int64_t ldx, const T* w, const T* b, int64_t rows, int cols, float eps, T* y,
                      float* mean, float* rstd, hipStream_t st) {
  ln_fwd_team<T>(cols, [&](auto team, auto nv) {
    constexpr int TEAM = decltype(team)::value, BLOCK = kLnFwdBlock < TEAM ? TEAM : kLnFwdBlock;
    constexpr int NV = decltype(nv)::value, V = Vec16<T>::N;
    auto kernel = cols % V == 0 ? layernorm_fwd_kernel<T, TEAM, NV, DENSE> : layernorm_fwd_kernel<T, TEAM, NV, SHIFTED>;
    if constexpr (TEAM == 64)
      if (cols < V) kernel = layernorm_fwd_kernel<T, TEAM, NV, SHORT>;
    const TileGrid grid = tile_grid(ceil_div(rows, BLOCK / TEAM), BLOCK);
    kernel<<<dim3(grid.gx, grid.gy), dim3(BLOCK), 0, st>>>(x, ldx, w, b, rows, cols, eps, y, mean, rstd, grid.gx);
  });
  return launch_status();
}

template <typename T>
static int32_t ln_bwd(const T* dy, int64_t lddy, const T* x, int64_t ldx, const T* w, const float* mean,
                      const float* rstd, int64_t rows, int cols, T* dx, T* dw, T* db, float* parts, int32_t dtype,
                      hipStream_t st) {
  const int n = ln_parts(rows, cols, dtype);
  float* const to = (dw || db) && n > 1 ? parts : nullptr;
  ln_team<T>(cols, [&](auto team, auto nv) {
    constexpr int TEAM = decltype(team)::value, NV = decltype(nv)::value;
    constexpr int V = Vec16<T>::N;
    auto kernel = cols % V == 0 ? layernorm_bwd_kernel<T, TEAM, NV, DENSE> : layernorm_bwd_kernel<T, TEAM, NV, SHIFTED>;
    if constexpr (TEAM == 64)
      if (cols < V) kernel = layernorm_bwd_kernel<T, TEAM, NV, SHORT>;
    kernel<<<dim3(n), dim3(kLnBwdBlock), 0, st>>>(dy, lddy, x, ldx, w, mean, rstd, rows, cols, dx, to, dw, db);
  });
  const int32_t rc = launch_status();
  if (rc != P2P_OK || !to) return rc;
  layernorm_parts_kernel<T><<<dim3(static_cast<unsigned>(ceil_div(2 * static_cast<int64_t>(cols), 64))), dim3(1024), 0, st>>>(
      parts, n, cols, dw, db);
  return launch_status();
}

static int32_t ln_check(const void* x, int64_t ldx, int64_t rows, int64_t cols, int32_t dtype) {
  if (!known_dtype(dtype) || rows < 0 || cols < 1 || ldx < cols) return P2P_ERR_INVALID;
  if (cols > kLnMaxCols || rows > (int64_t(1) << 31) - 1) return P2P_ERR_UNSUPPORTED;
  if (rows > 0 && !x) return P2P_ERR_INVALID;
  if (!aligned_to(x, dtype_bytes(dtype))) return P2P_ERR_ALIGN;
  return P2P_OK;
}

}  // namespace p2p

using namespace p2p;

extern "C" int32_t p2p_layernorm_fwd(const void* x, int64_t ldx, const void* w, const void* b, int64_t rows,
                                     int64_t cols, float eps, void* y, float* mean, float* rstd, int32_t dtype,
                                     p2p_stream_t stream) {
  const int32_t rc = ln_check(x, ldx, rows, cols, dtype);
  if (rc != P2P_OK || rows == 0) return rc;
  if (!y || !mean || !rstd) return P2P_ERR_INVALID;
  if (!aligned_to(y, dtype_bytes(dtype)) || !aligned_to(w, dtype_bytes(dtype)) || !aligned_to(b, dtype_bytes(dtype)) ||
      !aligned_to(mean, 4) || !aligned_to(rstd, 4))
    return P2P_ERR_ALIGN;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const int c = static_cast<int>(cols);
  if (dtype == P2P_DTYPE_F32)
    return ln_fwd(static_cast<const float*>(x), ldx, static_cast<const float*>(w), static_cast<const float*>(b), rows, c,
                  eps, static_cast<float*>(y), mean, rstd, st);
  if (dtype == P2P_DTYPE_F16)
    return ln_fwd(static_cast<const f16*>(x), ldx, static_cast<const f16*>(w), static_cast<const f16*>(b), rows, c, eps,
                  static_cast<f16*>(y), mean, rstd, st);
  return ln_fwd(static_cast<const bf16*>(x), ldx, static_cast<const bf16*>(w), static_cast<const bf16*>(b), rows, c, eps,
                static_cast<bf16*>(y), mean, rstd, st);
}

extern "C" int64_t p2p_layernorm_bwd_workspace(int64_t rows, int64_t cols, int32_t dtype) {
  if (!known_dtype(dtype) || rows < 0 || cols < 1 || cols > kLnMaxCols) return P2P_ERR_INVALID;
  const int n = ln_parts(rows, static_cast<int>(cols), dtype);
  return n > 1 ? static_cast<int64_t>(n) * 2 * cols * 4 : 0;  // a block alone writes dw and db itself
}

extern "C" int32_t p2p_layernorm_bwd(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* w,
                                     const float* mean, const float* rstd, int64_t rows, int64_t cols, void* dx,
                                     void* dw, void* db, void* workspace, int64_t workspace_bytes, int32_t dtype,
                                     p2p_stream_t stream) {
  int32_t rc = ln_check(x, ldx, rows, cols, dtype);
  if (rc == P2P_OK) rc = ln_check(dy, lddy, rows, cols, dtype);
  if (rc != P2P_OK) return rc;
  // no rows: dw and db are empty sums, which the caller clears (nothing is launched)
  if (rows == 0) return P2P_OK;
  if (!mean || !rstd || !dx) return P2P_ERR_INVALID;
  if (dw || db) {
    const int64_t need = p2p_layernorm_bwd_workspace(rows, cols, dtype);
    if (workspace_bytes < need || (need && !workspace)) return P2P_ERR_INVALID;
    if (!aligned_to(workspace, 16)) return P2P_ERR_ALIGN;
  }
  const int s = dtype_bytes(dtype);
  if (!aligned_to(dx, s) || !aligned_to(w, s) || !aligned_to(dw, s) || !aligned_to(db, s) || !aligned_to(mean, 4) ||
      !aligned_to(rstd, 4))
    return P2P_ERR_ALIGN;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const int c = static_cast<int>(cols);
  float* parts = static_cast<float*>(workspace);
  if (dtype == P2P_DTYPE_F32)
    return ln_bwd(static_cast<const float*>(dy), lddy, static_cast<const float*>(x), ldx, static_cast<const float*>(w),
                  mean, rstd, rows, c, static_cast<float*>(dx), static_cast<float*>(dw), static_cast<float*>(db), parts,
                  dtype, st);
  if (dtype == P2P_DTYPE_F16)
    return ln_bwd(static_cast<const f16*>(dy), lddy, static_cast<const f16*>(x), ldx, static_cast<const f16*>(w), mean,
                  rstd, rows, c, static_cast<f16*>(dx), static_cast<f16*>(dw), static_cast<f16*>(db), parts, dtype, st);
  return ln_bwd(static_cast<const bf16*>(dy), lddy, static_cast<const bf16*>(x), ldx, static_cast<const bf16*>(w), mean,
                rstd, rows, c, static_cast<bf16*>(dx), static_cast<bf16*>(dw), static_cast<bf16*>(db), parts, dtype, st);
}
