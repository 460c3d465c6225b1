// What surrounds the products of gemm_tile.h: copies of operands that cannot
// be read in place, and the sum of a product's k-runs.
#include "gemm_tile.h"

namespace p2p {

// One lane per 8 elements of a packed row; grid.y: the matrix.
struct PackJobs {
  PackJob job[kMaxPack];
};
template <typename T>
__global__ __launch_bounds__(kBlock) void pack_kernel(PackJobs jobs) {
  const PackJob& job = jobs.job[blockIdx.y];
  const T* src = static_cast<const T*>(job.src);
  uint16_t* dst = job.dst;
  const int64_t ld = job.ld, cols = job.cols, pitch = job.pitch, plane = job.rows * pitch;
  const int64_t per_row = pitch / 8, all = job.rows * per_row;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x; i < all;
       i += static_cast<int64_t>(gridDim.x) * kBlock) {
    const int64_t r = i / per_row, c = (i - r * per_row) * 8;
    const T* s = src + r * ld;
    if constexpr (sizeof(T) == 4) {
      float v[8];
      load_row<T, 8>(s, c, cols, v);
      Pack<uint16_t, 8> o[3];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const Planes p = split3(v[e]);
#pragma unroll
        for (int q = 0; q < 3; ++q) o[q].v[e] = p.p[q];
      }
#pragma unroll
      for (int q = 0; q < 3; ++q) store_pack<uint16_t, 8>(dst + q * plane + r * pitch + c, o[q]);
    } else {
      Pack<uint16_t, 8> o;
      if (c + 8 <= cols) {
        o = load_pack<uint16_t, 8>(s + c);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) o.v[e] = c + e < cols ? ldg(s + c + e) : 0;
      }
      store_pack<uint16_t, 8>(dst + r * pitch + c, o);
    }
  }
}

static unsigned blocks_for(int64_t items) {
  const int64_t b = ceil_div(items, kBlock);
  return static_cast<unsigned>(b < 1 ? 1 : b > 256 * 32 ? 256 * 32 : b);
}

int32_t pack_matrices(const PackJob* jobs, int n, int32_t dtype, hipStream_t st) {
  PackJobs all{};
  int64_t most = 0;
  int used = 0;
  for (int i = 0; i < n; ++i) {
    if (!jobs[i].dst || jobs[i].rows == 0) continue;
    all.job[used] = jobs[i];
    all.job[used++].pitch = line_pitch(jobs[i].cols);
    most = std::max(most, jobs[i].rows * (line_pitch(jobs[i].cols) / 8));
  }
  if (!used) return P2P_OK;
  const dim3 grid(blocks_for(most), used);
  if (dtype == P2P_DTYPE_F32) pack_kernel<float><<<grid, dim3(kBlock), 0, st>>>(all);
  else pack_kernel<uint16_t><<<grid, dim3(kBlock), 0, st>>>(all);
  return launch_status();
}

template <typename T>
__global__ __launch_bounds__(kBlock) void join_kernel(const float* parts, int nparts, int64_t stride, int64_t n, int64_t second,
                                                      const float* scale0, const float* scale1, float alpha, T* out0, T* out1) {
  if (scale0) alpha *= ldc(scale0);
  if (scale1) alpha *= ldc(scale1);
  parts += blockIdx.y * second;
  T* out = blockIdx.y ? out1 : out0;
  for (int64_t i = (static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x) * 4; i < n;
       i += static_cast<int64_t>(gridDim.x) * kBlock * 4) {
    float s[4];
    sum_runs<4>(parts, stride, nparts, i, n, s);
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e] *= alpha;
    store_row<T, 4>(out, i, n, s);
  }
}

int32_t join_parts(const float* parts, int nparts, int64_t stride, int64_t n, int64_t second, const float* scale0,
                   const float* scale1, float alpha, void* out0, void* out1, int32_t dtype, hipStream_t st) {
  if (n == 0) return P2P_OK;
  const dim3 grid(blocks_for(ceil_div(n, 4)), out1 ? 2 : 1), block(kBlock);
  if (dtype == P2P_DTYPE_F32)
    join_kernel<float><<<grid, block, 0, st>>>(parts, nparts, stride, n, second, scale0, scale1, alpha,
                                               static_cast<float*>(out0), static_cast<float*>(out1));
  else if (dtype == P2P_DTYPE_F16)
    join_kernel<f16><<<grid, block, 0, st>>>(parts, nparts, stride, n, second, scale0, scale1, alpha, static_cast<f16*>(out0),
                                             static_cast<f16*>(out1));
  else
    join_kernel<bf16><<<grid, block, 0, st>>>(parts, nparts, stride, n, second, scale0, scale1, alpha,
                                              static_cast<bf16*>(out0), static_cast<bf16*>(out1));
  return launch_status();
}

}  // namespace p2p
