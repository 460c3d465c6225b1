// K9 -- the gated linear layer of a feed-forward block, forward and backward.
//
//   g = x Wg^T, u = x Wu^T, h = act(g) * u            x [T, H], Wg / Wu [F, H]
//   dg = dh * u * act'(g), du = dh * act(g)
//   dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x
//
// Matrix-bound: 12 T H F operations over operands that are read once per
// 256 x 256 tile.  Forward: one kernel, both products (the tile's columns
// interleave 16 rows of Wg and 16 of Wu, so one lane ends up with g and u of
// the same unit), the activation and the product in its epilogue.
//
// Training keeps g and u in 32 bits (8 bytes a unit): rounded to 16 bits
// they would put their rounding on top of dg's and du's own and the
// gradients' error at twice that of one rounding, and computing them again
// would be two of then eight products (at H = 4096, 2 x 8192 operations per
// unit against 16 more bytes moved).  dg and du are rounded to the type of x
// once, as the operands of the matrix instructions (float32: not rounded,
// three planes), lie side by side in one [T, 2F] buffer, and feed dx as two
// segments of one sum and dWg, dWu as one product of 2F rows.  That rounding
// and the results' own make 1.4 times the RMS error of the latter alone (1023
// x 1001 x 2731 float16 2.9e-4, 8192 x 4096 x 16384 bfloat16 2.3e-3; with d in 32
// bits 2.1e-4, 1.7e-3); a second plane of d would double two of three products.
//
// float16 holds them times a power of two that brings the largest of the call
// to [2^14, 2^15), taken back from the 32-bit sums: without it gradients near
// 1e-6 lay among its subnormal numbers (off by 3% in dx and dW; 0 below
// 3e-8) and those past 65504 became infinities, which sums in 32 bits do not.
// What is below 2^-28 of the largest is off by up to 2^-39 of it.  The largest
// one takes a pass of its own over gate, up and dh (10 bytes a unit; backward, without /
// with it, us: 1023 x 1001 x 2731 70 / 80, 8192 x 4096 x 16384 3852 / 4097).
//
// Small layers take the product of direct.h instead, forward into
// sums of k-runs that a second kernel joins and activates (forward and
// backward of 32 x 512 x 512 float32 82 us on tiles, 21 so; 1 x 512 x 1000
// bfloat16 35, 22; direct.h has the sizes on both sides of the rule).
#include <type_traits>

#include "direct_tile.h"
#include "gemm_tile.h"

namespace p2p {

template <int ACT>
__device__ __forceinline__ void activation(float g, float* a, float* da) {
  if constexpr (ACT == P2P_ACT_SILU) {
    // exp(-g) with its argument rounded once: off by |g| 2^-23 of itself, so a by less than 2^-23 and, in the lower
    // tail, by |g| 2^-23 of itself (8192 x 4096 x 16384 bfloat16 forward 1905 us with the exact one, 1888 so)
    const float s = __builtin_amdgcn_rcpf(1.f + __expf(-g));
    *a = g * s;
    *da = s * (1.f + g * (1.f - s));
  } else if constexpr (ACT == P2P_ACT_GELU) {
    // phi(g) = erfc(-g / sqrt 2) / 2 out of the Gaussian that the derivative needs anyway: erfc(y) = t Q(t) exp(-y^2)
    // for y >= 0, t = 1 / (1 + 0.38 y), Q the polynomial of least relative error (2e-8, fitted to erfc exp(y^2) / t up to
    // y = 10.5): off by 4 * 2^-24 of 1, and in the lower tail by as much of phi itself as its exponential.
    const float y = fabsf(g) * 0.70710678118654752f, t = __builtin_amdgcn_rcpf(fmaf(0.38f, y, 1.f)), e = __expf(-0.5f * g * g);
    float q = 0.059016767889261246f;
    q = fmaf(q, t, -0.2625329792499542f);
    q = fmaf(q, t, 0.36440375447273254f);
    q = fmaf(q, t, -0.16210836172103882f);
    q = fmaf(q, t, 0.2304965704679489f);
    q = fmaf(q, t, 0.1384376883506775f);
    q = fmaf(q, t, 0.20396439731121063f);
    q = fmaf(q, t, 0.21391065418720245f);
    q = fmaf(q, t, 0.21441151201725006f);
    const float tail = 0.5f * q * t * e, phi = g < 0.f ? tail : 1.f - tail;
    *a = g * phi;
    *da = phi + g * e * 0.39894228040143268f;
  } else {
    *a = g < 0.f ? 0.f : g;  // a NaN stays one
    *da = g > 0.f ? 1.f : 0.f;
  }
}
// f(the activation as a type): chosen once for many elements; a choice for each would compute them all.
template <typename F>
__device__ __forceinline__ void with_activation(int act, const F& f) {
  if (act == P2P_ACT_SILU) f(std::integral_constant<int, P2P_ACT_SILU>());
  else if (act == P2P_ACT_GELU) f(std::integral_constant<int, P2P_ACT_GELU>());
  else f(std::integral_constant<int, P2P_ACT_RELU>());
}

struct GatedEpi {
  void* h;
  float *gate, *up;  // nullable
  int64_t units;
  int32_t dtype, act;

  template <class Cfg>
  __device__ __forceinline__ void finish(f4 (&acc)[Cfg::MI][Cfg::NJ], const Place& p, const GemmArgs& g, char* lds) const {
    with_activation(act, [&](auto kind) { tile<decltype(kind)::value, Cfg>(acc, p, g, lds); });
  }
  template <int ACT, class Cfg>
  __device__ __forceinline__ void tile(f4 (&acc)[Cfg::MI][Cfg::NJ], const Place& p, const GemmArgs& g, char* lds) const {
    const auto put = [&](int64_t m, int64_t n, f4 gv, f4 uv) {
      if (m >= g.M || n >= units) return;
      f4 hv;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float a, da;
        activation<ACT>(gv[e], &a, &da);
        hv[e] = a * uv[e];
      }
      store4_as(h, dtype, m, units, n, units, hv);
      if (gate) store4(gate + m * units, n, units, gv);
      if (up) store4(up + m * units, n, units, uv);
    };
    if constexpr (RowImage<Cfg>::USED) {
      constexpr int LANES = Cfg::BN / 8, PER = 64 / LANES, ROWS = RowImage<Cfg>::ROWS;
      const RowImage<Cfg> image{lds, p};
      const int k = p.lane % LANES, chunk = k / 4 * 8 + k % 4;  // four units: their g, and four chunks on their u
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        image.put(acc, half);
#pragma unroll 4
        for (int r = 0; r < ROWS; r += PER) {
          const int row = image.template row<PER>(p.wave, r + p.lane / LANES);
          put(static_cast<int64_t>(p.tm) * Cfg::BM + half * Cfg::HM + row, static_cast<int64_t>(p.tn) * (Cfg::BN / 2) + k * 4,
              image.get(row, chunk), image.get(row, chunk + 4));
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < Cfg::MI; ++i)
#pragma unroll
        for (int j = 0; j < Cfg::NJ; j += 2)
          put(p.m0 + Cfg::row(i) + (p.lane & 15), (p.n0 + Cfg::col(j)) / 2 + (p.lane >> 4) * 4, acc[i][j], acc[i][j + 1]);
    }
  }
};

// The k-runs' g and u instead, [runs][T, 2 units] (the tile's columns: 16 units' g, then their u).
struct GatedPartEpi {
  float* partial;
  int64_t units;

  template <class Cfg>
  __device__ __forceinline__ void finish(f4 (&acc)[Cfg::MI][Cfg::NJ], const Place& p, const GemmArgs& g, char* lds) const {
    by_rows<Cfg>(acc, p, lds, [&](int, int64_t m, int64_t n, f4 v) {
      const int64_t unit = n / 32 * 16 + n % 16;
      if (m < g.M && unit < units) store4(partial + ((p.part * g.M + m) * 2 + n / 16 % 2) * units, unit, units, v);
    });
  }
};

template <int ACT>
__device__ __forceinline__ void unit_grads(float g, float u, float dh, float* dg, float* du) {
  float a, da;
  activation<ACT>(g, &a, &da);
  *dg = dh * u * da;
  *du = dh * a;
}

// float16's power of two.  `largest`: the bits of the largest finite |dg|, |du|
// of each block (as unsigned numbers they order as the values do), joined by
// every block that scales; factor: what the sums are multiplied by.
struct GradScale {
  uint32_t* largest;
  float* factor;
  int blocks;
};
constexpr int kScaleBlocks = 4 * kBlock;  // four of them per lane

// The block's largest; every lane calls it.
__device__ __forceinline__ uint32_t block_max(uint32_t m) {
  __shared__ uint32_t waves[kBlock / 64];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = std::max<uint32_t>(m, __shfl_xor(m, o, 64));
  if ((threadIdx.x & 63) == 0) waves[threadIdx.x / 64] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kBlock / 64; ++w) m = std::max(m, waves[w]);
  return m;
}

template <int ACT>
__global__ __launch_bounds__(kBlock) void gated_largest_kernel(const f16* dh, int64_t lddh, const float* gate, const float* up,
                                                               int64_t rows, int64_t units, uint32_t* largest) {
  const int64_t per_row = (units + 7) / 8, all = rows * per_row;
  uint32_t m = 0;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x; i < all;
       i += static_cast<int64_t>(gridDim.x) * kBlock) {
    const int64_t r = i / per_row, c = (i - r * per_row) * 8;
    float g[8], u[8], dhv[8];
    load_row<float, 8>(gate + r * units, c, units, g);
    load_row<float, 8>(up + r * units, c, units, u);
    load_row<f16, 8>(dh + r * lddh, c, units, dhv);
#pragma unroll
    for (int e = 0; e < 8; ++e) {  // (0 past the units: their dh is)
      float dg, du;
      unit_grads<ACT>(g[e], u[e], dhv[e], &dg, &du);
      const uint32_t a = __float_as_uint(fabsf(dg)), b = __float_as_uint(fabsf(du));
      m = std::max(m, a < 0x7f800000u ? a : 0u);
      m = std::max(m, b < 0x7f800000u ? b : 0u);
    }
  }
  m = block_max(m);
  if (threadIdx.x == 0) stg(largest + blockIdx.x, m);
}

// What to multiply by; the factor that undoes it is left by the first block.
__device__ __forceinline__ float grad_scale(const GradScale& s) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < kScaleBlocks / kBlock; ++j) {
    const int i = j * kBlock + threadIdx.x;
    if (i < s.blocks) m = std::max(m, ldg(s.largest + i));
  }
  m = block_max(m);
  // 2^e of the largest in [2^14, 2^15); both 2^e and 2^-e among the normal numbers
  const int e = m == 0 ? 0 : std::min(14 - (static_cast<int>(m >> 23) - 127), 126);
  if (blockIdx.x == 0 && threadIdx.x == 0) stg(s.factor, __uint_as_float(static_cast<uint32_t>(127 - e) << 23));
  return __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
}

// dg and du of 8 units per lane, into d [T, 2 * pitch]: dg, then du, zeros
// in the columns past `units`; plane: elements from one plane to the next.
// DIRECT: as float, with no columns past `units` (pitch == units).
template <typename T, int ACT, bool DIRECT>
__global__ __launch_bounds__(kBlock) void gated_grad_kernel(const T* dh, int64_t lddh, const float* gate, const float* up,
                                                            int64_t rows, int64_t units, int64_t pitch, uint16_t* d,
                                                            int64_t plane, GradScale scale) {
  constexpr bool SCALED = std::is_same_v<T, f16> && !DIRECT;
  float by = 1.f;
  if constexpr (SCALED) by = grad_scale(scale);
  const int64_t per_row = (pitch + 7) / 8, all = rows * per_row;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x; i < all;
       i += static_cast<int64_t>(gridDim.x) * kBlock) {
    const int64_t r = i / per_row, c = (i - r * per_row) * 8;
    float g[8], u[8], dhv[8];
    load_row<float, 8>(gate + r * units, c, units, g);
    load_row<float, 8>(up + r * units, c, units, u);
    load_row<T, 8>(dh + r * lddh, c, units, dhv);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float dg, du;
      unit_grads<ACT>(g[e], u[e], dhv[e], &dg, &du);
      if (SCALED) dg *= by, du *= by;
      g[e] = c + e < units ? dg : 0.f;
      u[e] = c + e < units ? du : 0.f;
    }
    uint16_t* to = d + r * 2 * pitch + c;
    if constexpr (DIRECT) {
      float* row = reinterpret_cast<float*>(d) + r * 2 * pitch;
      store_row<float, 8>(row, c, units, g);
      store_row<float, 8>(row + pitch, c, units, u);
    } else if constexpr (sizeof(T) == 4) {
      Pack<uint16_t, 8> og[3], ou[3];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const Planes a = split3(g[e]), b = split3(u[e]);
#pragma unroll
        for (int q = 0; q < 3; ++q) og[q].v[e] = a.p[q], ou[q].v[e] = b.p[q];
      }
#pragma unroll
      for (int q = 0; q < 3; ++q) {
        store_pack<uint16_t, 8>(to + q * plane, og[q]);
        store_pack<uint16_t, 8>(to + q * plane + pitch, ou[q]);
      }
    } else {
      store_row<T, 8>(reinterpret_cast<T*>(to), 0, 8, g);
      store_row<T, 8>(reinterpret_cast<T*>(to) + pitch, 0, 8, u);
    }
  }
}

static int32_t gated_largest(const p2p_gated_linear_t& a, const GradScale& scale, hipStream_t st) {
  const auto kernel = a.activation == P2P_ACT_SILU   ? gated_largest_kernel<P2P_ACT_SILU>
                      : a.activation == P2P_ACT_GELU ? gated_largest_kernel<P2P_ACT_GELU>
                                                     : gated_largest_kernel<P2P_ACT_RELU>;
  kernel<<<dim3(scale.blocks), dim3(kBlock), 0, st>>>(static_cast<const f16*>(a.dh), a.lddh, a.gate, a.up, a.tokens, a.units,
                                                      scale.largest);
  return launch_status();
}

template <typename T, bool DIRECT>
static int32_t gated_grad(const p2p_gated_linear_t& a, int64_t pitch, uint16_t* d, const GradScale& scale, hipStream_t st) {
  if (std::is_same_v<T, f16> && !DIRECT) {
    const int32_t rc = gated_largest(a, scale, st);
    if (rc != P2P_OK) return rc;
  }
  const int64_t items = a.tokens * ceil_div(pitch, 8), blocks = ceil_div(items, kBlock);
  const dim3 grid(static_cast<unsigned>(blocks < 256 * 32 ? blocks : 256 * 32)), block(kBlock);
  const auto kernel = a.activation == P2P_ACT_SILU   ? gated_grad_kernel<T, P2P_ACT_SILU, DIRECT>
                      : a.activation == P2P_ACT_GELU ? gated_grad_kernel<T, P2P_ACT_GELU, DIRECT>
                                                     : gated_grad_kernel<T, P2P_ACT_RELU, DIRECT>;
  kernel<<<grid, block, 0, st>>>(static_cast<const T*>(a.dh), a.lddh, a.gate, a.up, a.tokens, a.units, pitch, d,
                                 a.tokens * 2 * pitch, scale);
  return launch_status();
}

// A product's runs [runs][T, 2 units] joined; gate, up and h.
__global__ __launch_bounds__(kBlock) void gated_join_kernel(const float* parts, int runs, int64_t rows, int64_t units, int act,
                                                            void* h, int32_t dtype, float* gate, float* up) {
  const int64_t per_row = (units + 3) / 4, all = rows * per_row;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x; i < all;
       i += static_cast<int64_t>(gridDim.x) * kBlock) {
    const int64_t r = i / per_row, c = (i - r * per_row) * 4;
    float g[4], u[4], o[4];
    const float* row = parts + r * 2 * units;
    sum_runs<4>(row, rows * 2 * units, runs, c, units, g);
    sum_runs<4>(row + units, rows * 2 * units, runs, c, units, u);
    with_activation(act, [&](auto kind) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float a, da;
        activation<decltype(kind)::value>(g[e], &a, &da);
        o[e] = a * u[e];
      }
    });
    if (dtype == P2P_DTYPE_F32) store_row<float, 4>(static_cast<float*>(h) + r * units, c, units, o);
    else if (dtype == P2P_DTYPE_F16) store_row<f16, 4>(static_cast<f16*>(h) + r * units, c, units, o);
    else store_row<bf16, 4>(static_cast<bf16*>(h) + r * units, c, units, o);
    if (gate) store_row<float, 4>(gate + r * units, c, units, g);
    if (up) store_row<float, 4>(up + r * units, c, units, u);
  }
}

static int32_t gated_check(const p2p_gated_linear_t* a) {
  if (!a || !known_dtype(a->dtype) || a->activation < 0 || a->activation > P2P_ACT_RELU) return P2P_ERR_INVALID;
  if (a->tokens < 0 || a->hidden < 1 || a->units < 1 || a->ldx < a->hidden || a->ldg < a->hidden || a->ldu < a->hidden)
    return P2P_ERR_INVALID;
  const int64_t most = (int64_t(1) << 31) - 256;
  if (a->hidden > kMaxPitch - 8 || a->units > kMaxPitch / 2 - 8 || a->tokens > most) return P2P_ERR_UNSUPPORTED;
  if (!a->w_gate || !a->w_up || (a->tokens > 0 && !a->x)) return P2P_ERR_INVALID;
  const int s = dtype_bytes(a->dtype);
  if (!aligned_to(a->x, s) || !aligned_to(a->w_gate, s) || !aligned_to(a->w_up, s)) return P2P_ERR_ALIGN;
  return P2P_OK;
}

// The forward product's tile and runs: few tiles over a long sum are cut along k (their sums at most half a gigabyte),
// joined and activated by the small product's kernel (whole / in runs, us: 64 x 4096 x 4096 bfloat16 47.4 / 24.1, 512 x
// 4096 x 1024 49.0 / 26.0, 256 x 2048 x 2048 28.6 / 22.6, 512 x 4096 x 2048 float32 285 / 133).
static Plan gated_fwd_plan(const p2p_gated_linear_t& a) {
  const int64_t steps = ksteps(a.hidden, a.dtype == P2P_DTYPE_F32 ? 6 : 1);
  const Plan p = gemm_plan(a.tokens, 2 * a.units, steps, true);
  return p.split * a.tokens * 2 * a.units * 4 <= int64_t(512) << 20 ? p : gemm_plan(a.tokens, 2 * a.units, steps, false);
}

// The workspace, in the order in which both passes carve it.
struct GatedSpace {
  uint16_t *x, *wg, *wu, *d;
  GradScale scale;  // float16 on tiles
  float* parts;
  float* dx_parts;  // of direct.h's product, whose gradients are made side by side
};
static int64_t gated_pitch(const p2p_gated_linear_t& a) { return line_pitch(a.units); }
static Plan gated_dx_plan(const p2p_gated_linear_t& a) {
  return gemm_plan(a.tokens, a.hidden, ksteps(a.units, a.dtype == P2P_DTYPE_F32 ? 12 : 2), true);
}
static Plan gated_dw_plan(const p2p_gated_linear_t& a) {
  return gemm_plan(2 * gated_pitch(a), a.hidden, ksteps(a.tokens, a.dtype == P2P_DTYPE_F32 ? 6 : 1), true);
}
static bool gated_direct(const p2p_gated_linear_t& a) {
  return direct_pays(a.tokens, 2 * a.units, a.hidden, a.dtype);
}
// Whether the direct gradients make d where they read it instead of reading
// it out of a buffer.  Backward, us, so / out of a buffer: 32 x 256 x 10 float32
// 7.1 / 11.1, 32 x 784 x 512 11.6 / 14.1, 256 x 256 x 256 16.0 / 17.2, 128 x 256 x
// 1000 23.0 / 23.2, 512 x 1024 x 1024 102 / 67.
static bool gated_made_in_place(const p2p_gated_linear_t& a) {
  return static_cast<double>(a.tokens) * static_cast<double>(2 * a.units) * static_cast<double>(a.hidden) <= 6.0e7;
}
static int64_t gated_carve(const p2p_gated_linear_t& a, bool backward, void* base, GatedSpace* s) {
  Carver c{static_cast<char*>(base)};
  if (gated_direct(a)) {
    const int64_t rows2 = 2 * a.units;
    *s = GatedSpace{};
    int64_t floats = 0;
    if (backward) {
      if (!gated_made_in_place(a)) s->d = static_cast<uint16_t*>(c.take(a.tokens * rows2 * 4));
      const int sx = direct_split(a.tokens, a.hidden, rows2, false), sw = direct_split(rows2, a.hidden, a.tokens, false);
      if (sx > 1) s->dx_parts = static_cast<float*>(c.take(sx * a.tokens * a.hidden * 4));
      if (sw > 1) floats = sw * rows2 * a.hidden;
    } else {
      floats = direct_split(a.tokens, 2 * a.units, a.hidden, true) * a.tokens * 2 * a.units;
    }
    if (floats) s->parts = static_cast<float*>(c.take(floats * 4));
    return c.used;
  }
  const auto operand = [&](const void* p, int64_t ld, int64_t rows) -> uint16_t* {
    return in_place(p, ld, a.hidden, a.dtype) ? nullptr : static_cast<uint16_t*>(c.take(packed_bytes(rows, a.hidden, a.dtype)));
  };
  s->x = operand(a.x, a.ldx, a.tokens);
  s->wg = operand(a.w_gate, a.ldg, a.units);
  // both weights share one pitch: packed together or not at all
  if (in_place(a.w_gate, a.ldg, a.hidden, a.dtype) && in_place(a.w_up, a.ldu, a.hidden, a.dtype) && a.ldg == a.ldu) {
    s->wu = nullptr;
  } else {
    if (!s->wg) s->wg = static_cast<uint16_t*>(c.take(packed_bytes(a.units, a.hidden, a.dtype)));
    s->wu = static_cast<uint16_t*>(c.take(packed_bytes(a.units, a.hidden, a.dtype)));
  }
  s->d = nullptr;
  s->scale = GradScale{};
  s->parts = s->dx_parts = nullptr;
  if (!backward) {
    const int64_t split = gated_fwd_plan(a).split;
    if (split > 1) s->parts = static_cast<float*>(c.take(split * a.tokens * 2 * a.units * 4));
  } else {
    const int64_t rows2 = 2 * gated_pitch(a);
    s->d = static_cast<uint16_t*>(c.take(a.tokens * rows2 * 2 * planes_of(a.dtype)));
    if (a.dtype == P2P_DTYPE_F16) {
      s->scale.blocks = static_cast<int>(std::min<int64_t>(ceil_div(a.tokens * ceil_div(a.units, 8), kBlock), kScaleBlocks));
      s->scale.largest = static_cast<uint32_t*>(c.take(kScaleBlocks * 4));
      s->scale.factor = static_cast<float*>(c.take(4));
    }
    const Plan px = gated_dx_plan(a), pw = gated_dw_plan(a);
    int64_t floats = 0;
    if (px.split > 1) floats = px.split * a.tokens * a.hidden;
    if (pw.split > 1) floats = std::max(floats, pw.split * rows2 * a.hidden);
    if (floats) s->parts = static_cast<float*>(c.take(floats * 4));
  }
  return c.used;
}

// x, w_gate and w_up as the products read them, copied (in one launch) where the workspace has a place for it.
static int32_t gated_operands(const p2p_gated_linear_t& a, const GatedSpace& s, Mat* x, Mat* wg, Mat* wu, hipStream_t st) {
  const PackJob jobs[3] = {{a.x, a.ldx, a.tokens, a.hidden, s.x, 0},
                           {a.w_gate, a.ldg, a.units, a.hidden, s.wg, 0},
                           {a.w_up, a.ldu, a.units, a.hidden, s.wu, 0}};
  *x = mat_of(jobs[0], a.dtype);
  *wg = mat_of(jobs[1], a.dtype);
  *wu = mat_of(jobs[2], a.dtype);
  return pack_matrices(jobs, 3, a.dtype, st);
}

static int32_t gated_join(const p2p_gated_linear_t& a, const GatedSpace& s, int split, hipStream_t st) {
  const int64_t blocks = ceil_div(a.tokens * ceil_div(a.units, 4), kBlock);
  gated_join_kernel<<<dim3(static_cast<unsigned>(std::min<int64_t>(blocks, 256 * 32))), dim3(kBlock), 0, st>>>(
      s.parts, split, a.tokens, a.units, a.activation, a.h, a.dtype, a.gate, a.up);
  return launch_status();
}

static int32_t gated_direct_fwd(const p2p_gated_linear_t& a, const GatedSpace& s, hipStream_t st) {
  const int split = direct_split(a.tokens, 2 * a.units, a.hidden, true);
  const DirectArgs g{a.x, a.w_gate, a.w_up, a.ldx, a.ldg, a.ldu, a.units, a.tokens, 2 * a.units, a.hidden, split,
                     {nullptr, nullptr}, INT64_MAX, {nullptr, nullptr}, s.parts};
  const int32_t rc = direct_product(g, a.dtype, st);
  return rc == P2P_OK ? gated_join(a, s, split, st) : rc;
}

// [dg du] of a token, made where the gradients' products read it (again for
// every 64 columns of x, against a launch and a buffer).
template <typename T>
struct GatedGrad {
  const T* dh;
  int64_t lddh;
  const float *gate, *up;
  int64_t units;
  int act;

  struct Raw4 {
    float g[4], u[4];
    uint32_t d[sizeof(T)];
    int first;  // how many of the four are dg's, the others du's
  };
  __device__ __forceinline__ Raw4 fetch(int64_t t, int64_t c, int64_t) const {
    const float *gr = gate + t * units, *ur = up + t * units;
    const T* dr = dh + t * lddh;
    Raw4 r;
    const int64_t n = c >= units ? c - units : c;
    if (n + 4 <= units) {
      const Pack<float, 4> g = load_pack<float, 4>(gr + n), u = load_pack<float, 4>(ur + n);
#pragma unroll
      for (int e = 0; e < 4; ++e) r.g[e] = g.v[e], r.u[e] = u.v[e];
      const Pack<T, 4> d = load_pack<T, 4>(dr + n);
      __builtin_memcpy(r.d, &d, sizeof(d));
      r.first = c >= units ? 0 : 4;
      return r;
    }
    // from dg into du, or past both: zeros, of which 0 is made
    Pack<T, 4> d;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int64_t m = c + e >= units ? c + e - units : c + e;
      const bool in = m < units;
      r.g[e] = in ? ldg(gr + m) : 0.f;
      r.u[e] = in ? ldg(ur + m) : 0.f;
      d.v[e] = in ? ldg(dr + m) : static_cast<T>(0.f);
    }
    __builtin_memcpy(r.d, &d, sizeof(d));
    r.first = c >= units ? 0 : static_cast<int>(units - c);
    return r;
  }
  __device__ __forceinline__ void of(const Raw4& r, float (&v)[4]) const {
    Pack<T, 4> d;
    __builtin_memcpy(&d, r.d, sizeof(d));
    with_activation(act, [&](auto kind) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = static_cast<float>(d.v[e]);
        float a, da;
        activation<decltype(kind)::value>(r.g[e], &a, &da);
        v[e] = e < r.first ? x * r.u[e] * da : x * a;
      }
    });
  }
};

template <typename T>
static int32_t gated_direct_bwd(const p2p_gated_linear_t& a, const GatedSpace& s, hipStream_t st) {
  const int64_t rows2 = 2 * a.units, nx = a.tokens * a.hidden, nw = a.units * a.hidden;
  const int sx = direct_split(a.tokens, a.hidden, rows2, false), sw = direct_split(rows2, a.hidden, a.tokens, false);
  // dx = [dg du] [Wg; Wu], [dWg; dWu] = [dg du]^T x
  const DirectArgs x{nullptr, a.w_gate, a.w_up, 0, a.ldg, a.ldu, a.units, a.tokens, a.hidden, rows2, sx,
                     {a.dx, nullptr}, INT64_MAX, {nullptr, nullptr}, sx > 1 ? s.dx_parts : nullptr};
  const DirectArgs w{nullptr, a.x, a.x, 0, a.ldx, a.ldx, INT64_MAX, rows2, a.hidden, a.tokens, sw,
                     {a.dw_gate, a.dw_up}, a.units, {nullptr, nullptr}, sw > 1 ? s.parts : nullptr};
  int32_t rc;
  if (s.d) {
    if ((rc = gated_grad<T, true>(a, a.units, s.d, s.scale, st)) != P2P_OK) return rc;
    const float* d = reinterpret_cast<const float*>(s.d);
    rc = direct_grads<DirectLines<float>, T>(x, w, {d, d, rows2, rows2, INT64_MAX}, st);
  } else {
    rc = direct_grads<GatedGrad<T>, T>(x, w, {static_cast<const T*>(a.dh), a.lddh, a.gate, a.up, a.units, a.activation}, st);
  }
  if (rc == P2P_OK && sx > 1) rc = join_parts(s.dx_parts, sx, nx, nx, 0, nullptr, nullptr, 1.f, a.dx, nullptr, a.dtype, st);
  if (rc == P2P_OK && sw > 1) rc = join_parts(s.parts, sw, 2 * nw, nw, nw, nullptr, nullptr, 1.f, a.dw_gate, a.dw_up, a.dtype, st);
  return rc;
}

}  // namespace p2p

using namespace p2p;

extern "C" int64_t p2p_gated_linear_workspace(const p2p_gated_linear_t* a, int32_t backward) {
  const int32_t rc = gated_check(a);
  if (rc != P2P_OK) return rc;
  GatedSpace s;
  return a->tokens ? gated_carve(*a, backward != 0, nullptr, &s) : 0;
}

extern "C" int32_t p2p_gated_linear_fwd(const p2p_gated_linear_t* a, void* workspace, int64_t workspace_bytes,
                                        p2p_stream_t stream) {
  int32_t rc = gated_check(a);
  if (rc != P2P_OK || a->tokens == 0) return rc;
  if (!a->h || !aligned_to(a->h, dtype_bytes(a->dtype)) || !aligned_to(a->gate, 4) || !aligned_to(a->up, 4))
    return a->h ? P2P_ERR_ALIGN : P2P_ERR_INVALID;
  GatedSpace s;
  const int64_t need = gated_carve(*a, false, workspace, &s);
  if (need > workspace_bytes || (need && !workspace)) return P2P_ERR_INVALID;
  if (!aligned_to(workspace, 16)) return P2P_ERR_ALIGN;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (gated_direct(*a)) return gated_direct_fwd(*a, s, st);
  Mat x, wg, wu;
  if ((rc = gated_operands(*a, s, &x, &wg, &wu, st)) != P2P_OK) return rc;
  GemmArgs g{};
  add_pairs(&g, x, wg, &wu, a->dtype);
  g.lda = x.ld, g.ldb = wg.ld;
  g.M = a->tokens, g.N = 2 * a->units, g.K = a->hidden;
  const Plan plan = gated_fwd_plan(*a);
  g.ksplit = plan.split;
  const bool f16_ = a->dtype == P2P_DTYPE_F16;
  if (plan.split == 1)
    return gemm_launch<false, false, true>(g, f16_, plan.big, GatedEpi{a->h, a->gate, a->up, a->units, a->dtype, a->activation}, st);
  rc = gemm_launch<false, false, true>(g, f16_, plan.big, GatedPartEpi{s.parts, a->units}, st);
  return rc == P2P_OK ? gated_join(*a, s, plan.split, st) : rc;
}

extern "C" int32_t p2p_gated_linear_bwd(const p2p_gated_linear_t* a, void* workspace, int64_t workspace_bytes,
                                        p2p_stream_t stream) {
  int32_t rc = gated_check(a);
  if (rc != P2P_OK || a->tokens == 0) return rc;
  if (!a->gate || !a->up || !a->dh || a->lddh < a->units || !a->dx || !a->dw_gate || !a->dw_up) return P2P_ERR_INVALID;
  const int size = dtype_bytes(a->dtype);
  if (!aligned_to(a->gate, 4) || !aligned_to(a->up, 4) || !aligned_to(a->dh, size) || !aligned_to(a->dx, size) ||
      !aligned_to(a->dw_gate, size) || !aligned_to(a->dw_up, size))
    return P2P_ERR_ALIGN;
  GatedSpace s;
  const int64_t need = gated_carve(*a, true, workspace, &s);
  if (need > workspace_bytes || (need && !workspace)) return P2P_ERR_INVALID;
  if (!aligned_to(workspace, 16)) return P2P_ERR_ALIGN;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const bool f16_ = a->dtype == P2P_DTYPE_F16;
  if (gated_direct(*a))
    return a->dtype == P2P_DTYPE_F32 ? gated_direct_bwd<float>(*a, s, st)
           : f16_                    ? gated_direct_bwd<f16>(*a, s, st)
                                     : gated_direct_bwd<bf16>(*a, s, st);
  Mat x, wg, wu;
  if ((rc = gated_operands(*a, s, &x, &wg, &wu, st)) != P2P_OK) return rc;
  const int64_t pitch = gated_pitch(*a), plane = a->tokens * 2 * pitch;
  rc = a->dtype == P2P_DTYPE_F32 ? gated_grad<float, false>(*a, pitch, s.d, s.scale, st)
       : f16_                    ? gated_grad<f16, false>(*a, pitch, s.d, s.scale, st)
                                 : gated_grad<bf16, false>(*a, pitch, s.d, s.scale, st);
  if (rc != P2P_OK) return rc;
  Mat dg{{s.d, s.d + plane, s.d + 2 * plane}, 2 * pitch};
  Mat du{{s.d + pitch, s.d + plane + pitch, s.d + 2 * plane + pitch}, 2 * pitch};

  {  // dx = dg Wg + du Wu
    GemmArgs g{};
    add_pairs(&g, dg, wg, nullptr, a->dtype);
    add_pairs(&g, du, wu, nullptr, a->dtype);
    g.lda = 2 * pitch, g.ldb = wg.ld;
    g.M = a->tokens, g.N = a->hidden, g.K = a->units;
    const Plan plan = gated_dx_plan(*a);
    g.ksplit = plan.split;
    StoreEpi e{{a->dx, nullptr}, 0, 0, a->hidden, a->dtype, {s.scale.factor, nullptr}, 1.f, plan.split > 1 ? s.parts : nullptr, 0};
    if ((rc = gemm_launch<false, true, false>(g, f16_, plan.big, e, st)) != P2P_OK) return rc;
    if (plan.split > 1 && (rc = join_parts(s.parts, plan.split, g.M * g.N, g.M * g.N, 0, s.scale.factor, nullptr, 1.f, a->dx,
                                           nullptr, a->dtype, st)) != P2P_OK)
      return rc;
  }
  {  // dWg = dg^T x, dWu = du^T x: one product of 2 pitch rows
    GemmArgs g{};
    add_pairs(&g, dg, x, nullptr, a->dtype);
    g.lda = 2 * pitch, g.ldb = x.ld;
    g.M = 2 * pitch, g.N = a->hidden, g.K = a->tokens;
    const Plan plan = gated_dw_plan(*a);
    g.ksplit = plan.split;
    StoreEpi e{{a->dw_gate, a->dw_up}, pitch, a->units, a->hidden, a->dtype, {s.scale.factor, nullptr}, 1.f,
               plan.split > 1 ? s.parts : nullptr, 0};
    if ((rc = gemm_launch<true, true, false>(g, f16_, plan.big, e, st)) != P2P_OK) return rc;
    if (plan.split > 1)
      return join_parts(s.parts, plan.split, g.M * g.N, a->units * a->hidden, pitch * a->hidden, s.scale.factor, nullptr, 1.f,
                        a->dw_gate, a->dw_up, a->dtype, st);
  }
  return P2P_OK;
}
