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

// GROUPS of a block's lanes each take a run of the parts; their sums are added in that order.  Many parts of a small
// result are a long chain of loads otherwise (1 x 108 x 6640 bfloat16, 32 runs: loss backward 24.9 us, 23.4 so).
template <typename T, int GROUPS>
__global__ __launch_bounds__(kBlock) void join_kernel(const float* parts, int nparts, int64_t stride, int64_t n, int64_t second,
                                                      const float* scale0, const float* scale1, float alpha, T* out0, T* out1) {
  constexpr int LANES = kBlock / GROUPS;
  __shared__ float sums[GROUPS > 1 ? GROUPS - 1 : 1][LANES * 4];
  if (scale0) alpha *= ldc(scale0);
  if (scale1) alpha *= ldc(scale1);
  T* out = blockIdx.y ? out1 : out0;
  const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
  const int from = nparts * group / GROUPS, to = nparts * (group + 1) / GROUPS;
  const float* mine = parts + blockIdx.y * second + from * stride;
  for (int64_t i0 = static_cast<int64_t>(blockIdx.x) * (LANES * 4); i0 < n; i0 += static_cast<int64_t>(gridDim.x) * (LANES * 4)) {
    const int64_t i = i0 + lane * 4;
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    if (i < n) sum_runs<4>(mine, stride, to - from, i, n, s);
    if constexpr (GROUPS > 1) {
      __syncthreads();  // the last ones have been read
      if (group)
#pragma unroll
        for (int e = 0; e < 4; ++e) sums[group - 1][e * LANES + lane] = s[e];
      __syncthreads();
      if (group) continue;
#pragma unroll
      for (int q = 0; q < GROUPS - 1; ++q)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[e] += sums[q][e * LANES + lane];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e] *= alpha;
    if (i < n) store_row<T, 4>(out, i, n, s);
  }
}

template <typename T>
static int32_t join_typed(const float* parts, int nparts, int64_t stride, int64_t n, int64_t second, const float* scale0,
                          const float* scale1, float alpha, void* out0, void* out1, hipStream_t st) {
  const bool groups = nparts > 8 && n <= int64_t(1) << 20;
  const dim3 grid(blocks_for(ceil_div(n, 4) * (groups ? 8 : 1)), out1 ? 2 : 1);
  const auto kernel = groups ? join_kernel<T, 8> : join_kernel<T, 1>;
  kernel<<<grid, dim3(kBlock), 0, st>>>(parts, nparts, stride, n, second, scale0, scale1, alpha, static_cast<T*>(out0),
                                        static_cast<T*>(out1));
  return launch_status();
}

int32_t join_parts(const float* parts, int nparts, int64_t stride, int64_t n, int64_t second, const float* scale0,
                   const float* scale1, float alpha, void* out0, void* out1, int32_t dtype, hipStream_t st) {
  if (n == 0) return P2P_OK;
  if (dtype == P2P_DTYPE_F32) return join_typed<float>(parts, nparts, stride, n, second, scale0, scale1, alpha, out0, out1, st);
  if (dtype == P2P_DTYPE_F16) return join_typed<f16>(parts, nparts, stride, n, second, scale0, scale1, alpha, out0, out1, st);
  return join_typed<bf16>(parts, nparts, stride, n, second, scale0, scale1, alpha, out0, out1, st);
}

}  // namespace p2p
