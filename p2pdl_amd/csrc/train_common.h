// What the kernels of a trainer's local step share (K7-K10): the element
// types, vector loads at any alignment, wave reductions.
#pragma once
#include "p2p_common.h"

namespace p2p {

using bf16 = __bf16;
using f16 = _Float16;

// Vectors that may start at any element: a row of an odd width, or a view
// into a larger tensor.  The target allows unaligned global accesses, so
// these stay 8- and 16-byte instructions.
using raw2 = uint32_t __attribute__((ext_vector_type(2), aligned(2), may_alias));
using raw4 = uint32_t __attribute__((ext_vector_type(4), aligned(2), may_alias));

template <typename T, int N>
struct Pack {
  T v[N];
};
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> load_pack(const T* p) {
  constexpr int BYTES = N * sizeof(T);
  static_assert(BYTES == 8 || BYTES % 16 == 0, "");
  if constexpr (BYTES == 8) {
    const uint2 r = __builtin_bit_cast(uint2, *(const P2P_GLOBAL raw2*)(p));
    return __builtin_bit_cast(Pack<T, N>, r);
  } else {
    struct {
      uint4 q[BYTES / 16];
    } r;
#pragma unroll
    for (int i = 0; i < BYTES / 16; ++i)
      r.q[i] = __builtin_bit_cast(uint4, *((const P2P_GLOBAL raw4*)(p + i * (16 / sizeof(T)))));
    return __builtin_bit_cast(Pack<T, N>, r);
  }
}
template <typename T, int N>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, N>& x) {
  constexpr int BYTES = N * sizeof(T);
  static_assert(BYTES == 8 || BYTES % 16 == 0, "");
  if constexpr (BYTES == 8) {
    *(P2P_GLOBAL raw2*)(p) = __builtin_bit_cast(raw2, x);
  } else {
    struct Quads {
      uint4 q[BYTES / 16];
    };
    const Quads r = __builtin_bit_cast(Quads, x);
#pragma unroll
    for (int i = 0; i < BYTES / 16; ++i) *((P2P_GLOBAL raw4*)(p + i * (16 / sizeof(T)))) = __builtin_bit_cast(raw4, r.q[i]);
  }
}

template <typename T>
struct Vec16 {
  static constexpr int N = 16 / sizeof(T);  // elements of a 16-byte vector
};

// A 16-byte vector x[c ..) as it lies, in four registers; elements at and past `cols` are 0.
struct Raw {
  uint32_t w[4];
};
// DENSE: the vector lies within the row, or past it whole.
template <typename T, bool DENSE>
__device__ __forceinline__ Raw load_raw(const T* row, int64_t c, int64_t cols) {
  constexpr int N = 16 / sizeof(T);
  if (c + N <= cols) return __builtin_bit_cast(Raw, *(const P2P_GLOBAL raw4*)(row + c));
  if (DENSE) return Raw{{0u, 0u, 0u, 0u}};
  Raw r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      r.w[i] = c + i < cols ? ldg(reinterpret_cast<const uint32_t*>(row) + c + i) : 0u;
    } else {
      const uint16_t* p = reinterpret_cast<const uint16_t*>(row) + c + 2 * i;
      const uint32_t lo = c + 2 * i < cols ? ldg(p) : 0u, hi = c + 2 * i + 1 < cols ? ldg(p + 1) : 0u;
      r.w[i] = lo | (hi << 16);
    }
  }
  return r;
}
// Keeps the compiler from holding values that it derived from r across this point (as floats
// they take twice the registers and are two instructions to make again).
__device__ __forceinline__ void forget(Raw& r) {
  asm volatile("" : "+v"(r.w[0]), "+v"(r.w[1]), "+v"(r.w[2]), "+v"(r.w[3]));
}
// Its element e as a float.
template <typename T>
__device__ __forceinline__ float raw_at(const Raw& r, int e) {
  if constexpr (sizeof(T) == 4) return __uint_as_float(r.w[e]);
  else return static_cast<float>(__builtin_bit_cast(T, static_cast<uint16_t>(r.w[e / 2] >> (e & 1) * 16)));
}
// x[c .. c + N) as floats; elements at and past `cols` read as 0.
template <typename T, int N>
__device__ __forceinline__ void load_row(const T* row, int64_t c, int64_t cols, float (&out)[N]) {
  if (c + N <= cols) {
    const Pack<T, N> p = load_pack<T, N>(row + c);
#pragma unroll
    for (int e = 0; e < N; ++e) out[e] = static_cast<float>(p.v[e]);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) out[e] = c + e < cols ? static_cast<float>(ldg(row + c + e)) : 0.f;
  }
}
template <typename T, int N, bool DENSE = false>
__device__ __forceinline__ void store_row(T* row, int64_t c, int64_t cols, const float (&x)[N]) {
  if (DENSE || c + N <= cols) {
    Pack<T, N> p;
#pragma unroll
    for (int e = 0; e < N; ++e) p.v[e] = static_cast<T>(x[e]);
    store_pack<T, N>(row + c, p);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (c + e < cols) stg(row + c + e, static_cast<T>(x[e]));
  }
}

// s[e] += p[c + e] + p[stride + c + e] + ... over `runs` <= W, all loads before the first sum, those past the last
// run again in its place (a loop over a remainder would wait for each).
template <int W, int N>
__device__ __forceinline__ void add_runs(const float* p, int64_t stride, int runs, int64_t c, int64_t cols, float (&s)[N]) {
  float v[W][N];
  if (c + N <= cols) {
#pragma unroll
    for (int u = 0; u < W; ++u) {
      const Pack<float, N> q = load_pack<float, N>(p + (u < runs ? u : runs - 1) * stride + c);
#pragma unroll
      for (int e = 0; e < N; ++e) v[u][e] = q.v[e];
    }
  } else {
#pragma unroll
    for (int u = 0; u < W; ++u)
#pragma unroll
      for (int e = 0; e < N; ++e) v[u][e] = ldg(p + (u < runs ? u : runs - 1) * stride + (c + e < cols ? c + e : cols - 1));
  }
#pragma unroll
  for (int u = 0; u < W; ++u)
#pragma unroll
    for (int e = 0; e < N; ++e) s[e] += u < runs && c + e < cols ? v[u][e] : 0.f;
}
// s[e] = p[c + e] + p[stride + c + e] + ... over `runs`, in that order, eight at a time; elements at and past `cols` are 0.
template <int N>
__device__ __forceinline__ void sum_runs(const float* p, int64_t stride, int runs, int64_t c, int64_t cols, float (&s)[N]) {
#pragma unroll
  for (int e = 0; e < N; ++e) s[e] = 0.f;
  for (int r = 0; r < runs; r += 8) add_runs<8, N>(p + r * stride, stride, runs - r < 8 ? runs - r : 8, c, cols, s);
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

__host__ inline bool known_dtype(int32_t d) {
  return d == P2P_DTYPE_F32 || d == P2P_DTYPE_F16 || d == P2P_DTYPE_BF16;
}
__host__ inline int dtype_bytes(int32_t d) { return d == P2P_DTYPE_F32 ? 4 : 2; }
__host__ inline bool aligned_to(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
__host__ inline int32_t launch_status() {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? P2P_OK : static_cast<int32_t>(e);
}

}  // namespace p2p
