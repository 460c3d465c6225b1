// K8 -- dropout from a counter-based generator, its mask never stored.
//
//   y[i] = (keep(i) ? x[i] / (1 - p) : 0) (+ residual[i])
//   keep(i): word i % 4 of Philox4x32-10's block offset + i / 4 under the key
//   `seed` is at least floor(p * 2^32)
// (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3",
// SC 2011: ten rounds over the counter (block mod 2^32, block / 2^32, 0, 0)).
// The mask is a function of (seed, offset, i) alone: the backward pass is
// this kernel over dy, and another peer that has the seed recomputes the
// trainer's step bit for bit, whatever grid it runs on.
//
// A dropped element is selected away, not multiplied by 0: an infinity or a
// NaN there leaves 0.  One block of four words serves four elements; a lane
// moves 16 bytes per load, so a 16-bit lane runs two blocks side by side.
#include "train_common.h"

namespace p2p {

constexpr int kDropoutMaxGrid = 256 * 64;

struct Words {
  uint32_t w[4];
};

__device__ __forceinline__ Words philox(uint64_t block, uint32_t k0, uint32_t k1) {
  uint32_t c0 = static_cast<uint32_t>(block), c1 = static_cast<uint32_t>(block >> 32), c2 = 0, c3 = 0;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = static_cast<uint64_t>(c0) * 0xD2511F53u, b = static_cast<uint64_t>(c2) * 0xCD9E8D57u;
    c0 = static_cast<uint32_t>(b >> 32) ^ c1 ^ k0;
    c1 = static_cast<uint32_t>(b);
    c2 = static_cast<uint32_t>(a >> 32) ^ c3 ^ k1;
    c3 = static_cast<uint32_t>(a);
    k0 += 0x9E3779B9u;  // the keys are wave-uniform: scalar adds
    k1 += 0xBB67AE85u;
  }
  return Words{{c0, c1, c2, c3}};
}

template <typename T, bool RES>
__global__ __launch_bounds__(kBlock) void dropout_kernel(const T* x, const T* residual, int64_t n, uint32_t threshold,
                                                         float scale, uint32_t k0, uint32_t k1, uint64_t offset,
                                                         const uint64_t* offset_dev, T* y) {
  constexpr int V = Vec16<T>::N;
  if (offset_dev) offset += ldc(offset_dev);
  const int64_t step = static_cast<int64_t>(gridDim.x) * (kBlock * V);
  for (int64_t i = (static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x) * V; i < n; i += step) {
    float v[V], r[V];
    load_row<T, V>(x, i, n, v);
    if (RES) load_row<T, V>(residual, i, n, r);
#pragma unroll
    for (int q = 0; q < V / 4; ++q) {
      const Words u = philox(offset + static_cast<uint64_t>(i) / 4 + q, k0, k1);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float kept = u.w[e] >= threshold ? v[4 * q + e] * scale : 0.f;
        v[4 * q + e] = RES ? kept + r[4 * q + e] : kept;
      }
    }
    store_row<T, V>(y, i, n, v);
  }
}

// p = 1: nothing is kept.
template <typename T, bool RES>
__global__ __launch_bounds__(kBlock) void dropout_none_kernel(const T* residual, int64_t n, T* y) {
  const int64_t step = static_cast<int64_t>(gridDim.x) * kBlock;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x; i < n; i += step)
    stg(y + i, RES ? ldg(residual + i) : static_cast<T>(0.f));
}

template <typename T, bool RES>
static int32_t dropout_run(const T* x, const T* residual, int64_t n, double p, uint64_t seed, uint64_t offset,
                           const uint64_t* offset_dev, T* y, hipStream_t st) {
  const int64_t blocks = ceil_div(n, static_cast<int64_t>(kBlock) * Vec16<T>::N);
  const dim3 grid(static_cast<unsigned>(blocks < kDropoutMaxGrid ? blocks : kDropoutMaxGrid));
  if (p >= 1.0) {
    dropout_none_kernel<T, RES><<<grid, dim3(kBlock), 0, st>>>(residual, n, y);
  } else {
    dropout_kernel<T, RES><<<grid, dim3(kBlock), 0, st>>>(
        x, residual, n, static_cast<uint32_t>(p * 4294967296.0), static_cast<float>(1.0 / (1.0 - p)),
        static_cast<uint32_t>(seed), static_cast<uint32_t>(seed >> 32), offset, offset_dev, y);
  }
  return launch_status();
}

template <typename T>
static int32_t dropout_any(const void* x, const void* residual, int64_t n, double p, uint64_t seed, uint64_t offset,
                           const uint64_t* offset_dev, void* y, hipStream_t st) {
  const T *xt = static_cast<const T*>(x), *rt = static_cast<const T*>(residual);
  T* yt = static_cast<T*>(y);
  return rt ? dropout_run<T, true>(xt, rt, n, p, seed, offset, offset_dev, yt, st)
            : dropout_run<T, false>(xt, rt, n, p, seed, offset, offset_dev, yt, st);
}

}  // namespace p2p

using namespace p2p;

extern "C" int32_t p2p_dropout(const void* x, const void* residual, int64_t n, double p, uint64_t seed, uint64_t offset,
                               const uint64_t* offset_dev, void* y, int32_t dtype, p2p_stream_t stream) {
  if (!known_dtype(dtype) || n < 0 || !(p >= 0.0 && p <= 1.0)) return P2P_ERR_INVALID;
  if (n == 0) return P2P_OK;
  if (!x || !y) return P2P_ERR_INVALID;
  const int s = dtype_bytes(dtype);
  if (!aligned_to(x, s) || !aligned_to(y, s) || !aligned_to(residual, s) || !aligned_to(offset_dev, 8)) return P2P_ERR_ALIGN;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == P2P_DTYPE_F32) return dropout_any<float>(x, residual, n, p, seed, offset, offset_dev, y, st);
  if (dtype == P2P_DTYPE_F16) return dropout_any<f16>(x, residual, n, p, seed, offset, offset_dev, y, st);
  return dropout_any<bf16>(x, residual, n, p, seed, offset, offset_dev, y, st);
}
