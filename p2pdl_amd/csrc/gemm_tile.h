// The matrix product under the gated linear layer and the linear cross
// entropy: C[m, n] = sum over k of A(m, k) * B(n, k), 16-bit operands,
// accumulators in 32 bits, the epilogue in the caller's hands.
//
// Operands.  An operand is either k-contiguous (A[m][k], what x and a weight
// [out, in] are in the forward pass) or row-contiguous (A[k][m], what the same
// tensors are when the gradient sums over tokens or over units); neither is
// transposed in memory.  Requirements of both: 16-byte aligned base and
// pitch, contiguous extent a multiple of 8 (pack_kernel makes such a copy of
// what is not).  A product may be a sum over several (A, B) pairs of equal
// shape, its segments: the two halves of the gated layer's dx, and float32.
//
// float32.  x = hi + mid + lo exactly, three bf16 values of 8 bits each,
// rounded to nearest: |mid| <= 2^-8 |x|, |lo| <= 2^-16 |x| (below 2^-110 they
// meet bf16's smallest step, 2^-133: off by half of it).  Of the nine
// products the six of order 2^-16 and above are kept, the small ones first;
// what is left out is at most 2^-23 + 2^-32 of |a| |b|, the size of one
// rounding of a 32-bit sum.  Six bf16 products take 6/16 of the time of one on
// the 32-bit matrix instructions.  A value that is not finite is its own hi.
//
// Tile.  BM x BN x 64 per k-step, the operands of two steps in LDS (128 KiB
// for 256 x 256), filled by LDS-DMA: a wave's instruction writes 1 KiB in
// lane order, so the swizzles are made by choosing each lane's source
// address.  Lanes whose source lies outside the operand get an offset past
// the descriptor's range and write zeros.
//
// Schedule.  Each operand's tile has two halves (rows), a wave owns a part of
// every quadrant, and a k-step is four phases, one quadrant each:
//   phase   products   reads into registers   requests (LDS-DMA)
//     0     A0 B0      B1 of this step        B0 of the step after next
//     1     A0 B1      A1 of this step        B1 of the step after next
//     2     A1 B0      A0 of the next step    A1 of the step after next
//     3     A1 B1      B0 of the next step    A0 of the third step on
// A half is requested as soon as the last wave has read the one it replaces
// (one barrier per phase) and is read seven phases later, so a request has
// almost two k-steps to come back, and what is read in a phase is multiplied in
// the next: the matrix instructions wait for neither.  Six halves stay in
// flight over every wait.  Steps past the end request zeros, so that the
// counts hold throughout.
//
// LDS images.  k-contiguous: rows of 128 bytes, 16-byte chunk c at position
// c ^ (row / 2 % 8): the 16 lanes of one k-group, one row each, then hit the 64
// banks once.  Row-contiguous: one line per k, its 32-byte granule g at
// position g ^ f(k), f(k) = k % 4 + 4 * (k / 8 % 4), read with
// ds_read_b64_tr_b16 (a 4 x 16 block of 16-bit elements comes back transposed
// over 16 lanes); f spreads the 16 lines that one instruction reads.
#pragma once
#include <algorithm>

#include "train_common.h"

#define P2P_LDS __attribute__((address_space(3)))

namespace p2p {

constexpr int kGemmK = 64;
constexpr int kMaxSegs = 12;
constexpr int64_t kMaxPitch = int64_t(1) << 22;  // 256 rows of 16-bit elements stay below 2^31 bytes

using f4 = float __attribute__((ext_vector_type(4)));
using s4 = short __attribute__((ext_vector_type(4)));
using s8 = short __attribute__((ext_vector_type(8)));
using b8 = __bf16 __attribute__((ext_vector_type(8)));
using h8 = _Float16 __attribute__((ext_vector_type(8)));

struct GemmArgs {
  const uint16_t* a[kMaxSegs];
  const uint16_t* b[kMaxSegs];
  const uint16_t* b2[kMaxSegs];  // DUAL: the second weight
  int64_t lda, ldb;
  int64_t M, N, K;  // K of one segment
  int nseg;
  int ksplit;       // grid.y: the k-steps of all segments cut into this many runs
};

template <int BM_, int BN_, int WM_, int WN_>
struct GemmCfg {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_;
  static constexpr int WAVES = WM * WN, THREADS = 64 * WAVES;
  static constexpr int HM = BM / 2, HN = BN / 2;          // the tile's halves
  static constexpr int QM = HM / WM, QN = HN / WN;        // a wave's part of a half
  static constexpr int MI = 2 * QM / 16, NJ = 2 * QN / 16;
  static constexpr int A_HALF = HM * kGemmK * 2, B_HALF = HN * kGemmK * 2, STAGE = 2 * (A_HALF + B_HALF);
  static constexpr int BLOCKS_PER_CU = 2 * STAGE > 80 * 1024 ? 1 : 2;
  static __host__ __device__ constexpr int row(int i) { return i / (MI / 2) * HM + i % (MI / 2) * 16; }
  static __host__ __device__ constexpr int col(int j) { return j / (NJ / 2) * HN + j % (NJ / 2) * 16; }
};
using Big = GemmCfg<256, 256, 2, 4>;
using Small = GemmCfg<128, 128, 2, 2>;

constexpr uint32_t kOutside = 0x80000000u;
using i4 = int __attribute__((ext_vector_type(4)));
// Twice 16 bytes per lane, from base + v0 to dst + 16 * lane and from base + v1
// to dst + 1024 + 16 * lane (base, dst wave-uniform).  In assembly: for the
// builtin the compiler waits for all requests before any LDS read (970 against
// 1216 TFLOP/s at 8192 x 4096 x 32768).  The kernel counts and waits itself; no
// register is written.  (Idle cycles: the compiler does not look into the block
// for an address that a vector instruction has just made scalar, nor for the
// use of m0.)
__device__ __forceinline__ void lds_dma2(const void* base, uint32_t v0, uint32_t v1, char* dst) {
  const uint64_t b = uniform_u64(reinterpret_cast<uint64_t>(base));
  const i4 rs = {static_cast<int>(b), static_cast<int>(b >> 32), static_cast<int>(kOutside), 0x00020000};
  const uint32_t to = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(reinterpret_cast<uintptr_t>((P2P_LDS void*)(dst))));
  asm volatile(
      "s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %2, %4, 0 offen lds\n\t"
      "s_mov_b32 m0, %1\n\ts_nop 0\n\tbuffer_load_dwordx4 %3, %4, 0 offen lds" ::"s"(to),
      "s"(to + 1024), "v"(v0), "v"(v1), "s"(rs)
      : "memory");
}

template <int EXT>
__device__ __forceinline__ int line_swizzle(int k) {
  if constexpr (EXT >= 128) return ((k & 3) | (((k >> 3) & 3) << 2)) & (EXT / 16 - 1);
  else return ((k >> 3) + (k & 2)) & 3;
}

// One half of an operand's part of a stage.  EXT: its rows; two 1-KiB instructions per wave.
template <bool ROWMAJOR, int EXT>
struct TileLoader {
  uint32_t voff[2];
  int kpos[2];

  // Lane addresses relative to the half's origin; `rows` left from it.
  __device__ __forceinline__ void init(int wave, int lane, int64_t ld, int64_t rows) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int q = wave * 2 + j;
      if constexpr (!ROWMAJOR) {
        const int r = q * 8 + lane / 8;
        const int c = (lane & 7) ^ ((r >> 1) & 7);
        kpos[j] = c * 8;
        voff[j] = r < rows ? static_cast<uint32_t>(r * ld * 2 + c * 16) : kOutside;
      } else {
        constexpr int CPL = EXT / 8;  // 16-byte chunks of a line
        const int k = q * (64 / CPL) + lane / CPL;
        const int pos = lane % CPL;
        const int m = ((pos >> 1) ^ line_swizzle<EXT>(k)) * 16 + (pos & 1) * 8;
        kpos[j] = k;
        voff[j] = m < rows ? static_cast<uint32_t>(k * ld * 2 + m * 2) : kOutside;
      }
    }
  }

  // The k-step at `base` into the image at dst; `left`: k still in the segment.
  __device__ __forceinline__ void issue(const uint16_t* base, int left, char* dst, int wave) const {
    lds_dma2(base, kpos[0] < left ? voff[0] : kOutside, kpos[1] < left ? voff[1] : kOutside, dst + wave * 2048);
  }
};

template <bool F16>
__device__ __forceinline__ f4 mfma16(s8 a, s8 b, f4 c) {
  if constexpr (F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
}

// A 16-row fragment of 32 k out of an image: lane l gets row l % 16, k = 8 * (l / 16) ... + 7.
template <bool ROWMAJOR, int EXT>
struct FragReader {
  int base[2];  // k-contiguous: per half of the step
  int kline, f, part;

  __device__ __forceinline__ void init(int lane) {
    const int i = lane & 15, q = lane >> 4;
    if constexpr (!ROWMAJOR) {
      base[0] = i * 128 + ((q ^ (i >> 1)) & 7) * 16;
      base[1] = i * 128 + (((4 + q) ^ (i >> 1)) & 7) * 16;
    } else {
      kline = (8 * q + (i >> 2)) * EXT * 2;
      f = line_swizzle<EXT>(8 * q + (i >> 2));
      part = (i & 3) * 8;
    }
  }
  // row0: first row of the fragment in the tile, a multiple of 16
  __device__ __forceinline__ s8 read(const char* image, int row0, int half) const {
    if constexpr (!ROWMAJOR) {
      return *reinterpret_cast<const P2P_LDS s8*>((const P2P_LDS char*)(image) + base[half] + row0 * 128);
    } else {
      const P2P_LDS char* p = (const P2P_LDS char*)(image) + kline + half * 32 * EXT * 2 + (((row0 >> 4) ^ f) << 5) + part;
      const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P2P_LDS s4*)(p));
      const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P2P_LDS s4*)(p + 4 * EXT * 2));
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
};

// Blocks go to the eight XCDs in turn, each with an L2 of its own.  Large
// tiles: super-blocks of 16 x 16 tiles, as many as run at once, in which an
// XCD has 4 x 8: it reads 12 panels of the operands for 32 tiles, and the chip 32
// for 256.  What is left of the matrix at the right and below, and small tiles:
// a contiguous run of tiles per XCD, ordered in groups of 4 rows.  8192 x 4096
// x 32768, 32768 x 4096 x 8192 (A^T B): runs in groups of 8 rows 1786, 1951 us, of
// 4 rows 1776, 1875 us, super-blocks 1752, 1824 us.
__device__ __forceinline__ void tile_of_run(int pid, int total, int rows, int cols, int* m, int* n) {
  const int per = total / 8, extra = total % 8, xcd = pid % 8;
  const int t = xcd * per + (xcd < extra ? xcd : extra) + pid / 8;
  constexpr int G = 4;
  const int group = t / (G * cols), first = group * G;
  const int height = rows - first < G ? rows - first : G;
  const int in = t - first * cols;
  *n = in / height;
  *m = first + (in - *n * height);
}
template <bool SUPER>
__device__ __forceinline__ void tile_of_block(int tiles_m, int tiles_n, int* tm, int* tn) {
  const int pid = blockIdx.x;
  const int sm = SUPER ? tiles_m / 16 : 0, sn = sm ? tiles_n / 16 : 0, whole = sm * sn * 256;
  if (SUPER && pid < whole) {
    const int sup = pid / 256, xcd = pid % 8, slot = pid % 256 / 8;
    *tn = sup / sm * 16 + xcd % 2 * 8 + slot / 4;
    *tm = sup % sm * 16 + xcd / 2 * 4 + slot % 4;
    return;
  }
  // the columns past the super-blocks over all rows, then the rows below them
  const int right = tiles_n - sn * 16, below = whole + tiles_m * right;
  if (pid < below) {
    tile_of_run(pid - whole, below - whole, tiles_m, right, tm, tn);
    *tn += sn * 16;
  } else {
    tile_of_run(pid - below, tiles_m * tiles_n - below, tiles_m - sm * 16, sn * 16, tm, tn);
    *tm += sm * 16;
  }
}

// Where an accumulator element lies: acc[mi][nj][i] is C[m][n] of
// m = m0 + 16 mi + (lane % 16), n = n0 + 16 nj + 4 (lane / 16) + i
// (the second operand's rows come out as the register index, so a lane holds
// four neighbours of one output row).
struct Place {
  int64_t m0, n0;  // the wave's first row and column
  int lane, wave;
  int tm, tn;      // the tile
  int wm, wn;      // the wave in it
  int part;        // the k-run
};

// DUAL: B's tile interleaves 16 rows of b and 16 of b2; N counts both (the
// tile's columns [32 j, 32 j + 16) are b's rows [16 j, 16 j + 16)).
template <bool F16, bool AT, bool BT, bool DUAL, class Cfg, class Epi>
__global__ __launch_bounds__(Cfg::THREADS, Cfg::WAVES * Cfg::BLOCKS_PER_CU / 4) void gemm_kernel(GemmArgs g, Epi epi) {
  __shared__ __attribute__((aligned(1024))) char lds[2 * Cfg::STAGE];
  static_assert(Cfg::HM / 8 / Cfg::WAVES == 2 && Cfg::HN / 8 / Cfg::WAVES == 2, "the counts of the waits below");
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tiles_m = static_cast<int>(ceil_div(g.M, Cfg::BM)), tiles_n = static_cast<int>(ceil_div(g.N, Cfg::BN));
  int tm, tn;
  tile_of_block<Cfg::BLOCKS_PER_CU == 1>(tiles_m, tiles_n, &tm, &tn);
  const int64_t m0 = static_cast<int64_t>(tm) * Cfg::BM, n0 = static_cast<int64_t>(tn) * Cfg::BN;

  TileLoader<AT, Cfg::HM> la[2];
  TileLoader<BT, Cfg::HN> lb[2];
  int64_t a_org[2], b_org[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int64_t m = m0 + h * Cfg::HM, n = n0 + h * Cfg::HN;
    la[h].init(wave, lane, g.lda, g.M - m);
    a_org[h] = AT ? m : m * g.lda;
    if constexpr (DUAL) {
      static_assert(!BT, "two weights: k-contiguous");
      const int64_t units = g.N / 2 - n / 2;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int r = (wave * 2 + j) * 8 + lane / 8, u = (r >> 5) * 16 + (r & 15);
        const int c = (lane & 7) ^ ((r >> 1) & 7);
        lb[h].kpos[j] = c * 8;
        lb[h].voff[j] = u < units ? static_cast<uint32_t>(u * g.ldb * 2 + c * 16) : kOutside;
      }
      b_org[h] = n / 2 * g.ldb;
    } else {
      lb[h].init(wave, lane, g.ldb, g.N - n);
      b_org[h] = BT ? n : n * g.ldb;
    }
  }

  const int per_seg = static_cast<int>(ceil_div(g.K, kGemmK));
  const int all = per_seg * g.nseg;
  const int part = blockIdx.y;
  const int first = static_cast<int>(static_cast<int64_t>(all) * part / g.ksplit);
  const int last = static_cast<int>(static_cast<int64_t>(all) * (part + 1) / g.ksplit);
  int seg = first / per_seg, ks = first % per_seg, left_steps = last - first;

  int64_t k0 = 0;
  int left = 0;
  const uint16_t *pa = nullptr, *pb = nullptr, *pb2 = nullptr;
  const auto point = [&]() {
    k0 = static_cast<int64_t>(ks) * kGemmK;
    const bool in = left_steps > 0;
    const int sg = in ? seg : 0;
    left = in ? static_cast<int>(g.K - k0 < kGemmK ? g.K - k0 : kGemmK) : 0;
    if (!in) k0 = 0;
    pa = g.a[sg] + (AT ? k0 * g.lda : k0);
    pb = g.b[sg] + (BT ? k0 * g.ldb : k0);
    if constexpr (DUAL) pb2 = g.b2[sg] + k0;
  };
  const auto next = [&]() {
    --left_steps;
    if (++ks == per_seg) ks = 0, ++seg;
    point();
  };
  const auto issue_a = [&](int h, char* stage) { la[h].issue(pa + a_org[h], left, stage + h * Cfg::A_HALF, wave); };
  const auto issue_b = [&](int h, char* stage) {
    char* dst = stage + 2 * Cfg::A_HALF + h * Cfg::B_HALF;
    if constexpr (DUAL) {
      // a wave's two instructions are rows 16 wave .. + 15 of the half, all of one weight
      lb[h].issue((wave % 2 ? pb2 : pb) + b_org[h], left, dst, wave);
    } else {
      lb[h].issue(pb + b_org[h], left, dst, wave);
    }
  };

  FragReader<AT, Cfg::HM> ra;
  FragReader<BT, Cfg::HN> rb;
  ra.init(lane);
  rb.init(lane);
  const int wm = wave / Cfg::WN, wn = wave % Cfg::WN;
  constexpr int AI = Cfg::MI / 2, BJ = Cfg::NJ / 2;
  f4 acc[Cfg::MI][Cfg::NJ];
#pragma unroll
  for (int i = 0; i < Cfg::MI; ++i)
#pragma unroll
    for (int j = 0; j < Cfg::NJ; ++j) acc[i][j] = f4{0.f, 0.f, 0.f, 0.f};
  s8 fa[2][AI][2], fb[2][BJ][2];
  const auto read_a = [&](int h, const char* stage) {
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int i = 0; i < AI; ++i) fa[h][i][half] = ra.read(stage + h * Cfg::A_HALF, wm * Cfg::QM + i * 16, half);
  };
  const auto read_b = [&](int h, const char* stage) {
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int j = 0; j < BJ; ++j) fb[h][j][half] = rb.read(stage + 2 * Cfg::A_HALF + h * Cfg::B_HALF, wn * Cfg::QN + j * 16, half);
  };
  const auto mma = [&](int ha, int hb, int half) {
#pragma unroll
    for (int i = 0; i < AI; ++i)
#pragma unroll
      for (int t = 0; t < BJ; ++t) {
        const int j = i % 2 ? BJ - 1 - t : t;  // each instruction shares an operand with the last
        acc[ha * AI + i][hb * BJ + j] = mfma16<F16>(fb[hb][j][half], fa[ha][i][half], acc[ha * AI + i][hb * BJ + j]);
      }
  };
  // One phase's work.  A request holds its wave's issue for some hundred
  // cycles.  Where B is read transposed out of LDS the phase's reads go first
  // and the request between the products (KM 8192 x 4096 x 32768 1740 -> 1697
  // us, MM 32768 x 4096 x 8192 1800 -> 1769); where B's k is contiguous the
  // request goes first (KK 8192 x 32768 x 4096 1883 us, between them 1969).
  const auto work = [&](auto request, auto read, int ha, int hb) {
    if constexpr (BT) {
      read();
      __builtin_amdgcn_sched_barrier(0);
      mma(ha, hb, 0);
      __builtin_amdgcn_sched_barrier(0);
      request();
      __builtin_amdgcn_sched_barrier(0);
    } else {
      request();
      read();
      mma(ha, hb, 0);
    }
    mma(ha, hb, 1);
  };
  // this wave's reads are done, its oldest half has landed; then everyone's
  const auto phase = [&] {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt vmcnt(12) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };

  char* cur = lds;
  char* nxt = lds + Cfg::STAGE;
  point();
  issue_a(0, cur);
  issue_b(0, cur);
  issue_b(1, cur);
  issue_a(1, cur);
  next();
  issue_a(0, nxt);
  issue_b(0, nxt);
  issue_b(1, nxt);
  issue_a(1, nxt);
  phase();
  read_a(0, cur);
  read_b(0, cur);
  next();
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
  issue_a(0, cur);
  for (int s = first; s < last; ++s) {
    phase();
    work([&] { issue_b(0, cur); }, [&] { read_b(1, cur); }, 0, 0);
    phase();
    work([&] { issue_b(1, cur); }, [&] { read_a(1, cur); }, 0, 1);
    phase();
    work([&] { issue_a(1, cur); }, [&] { read_a(0, nxt); }, 1, 0);
    phase();
    next();
    work([&] { issue_a(0, nxt); }, [&] { read_b(0, nxt); }, 1, 1);
    char* const t = cur;
    cur = nxt;
    nxt = t;
  }
  // the last requests (zeros) land before the epilogue uses the images or the block ends
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __syncthreads();
  Place p;
  p.m0 = m0 + wm * Cfg::QM, p.n0 = n0 + wn * Cfg::QN;
  p.lane = lane, p.wave = wave, p.tm = tm, p.tn = tn, p.wm = wm, p.wn = wn, p.part = part;
  epi.template finish<Cfg>(acc, p, g, lds);
}

// ------------------------------------------------------------------ epilogues
// A large tile's halves (rows) laid out by rows in LDS, floats, 16-byte chunk c
// of row r at position c ^ r % 16: a wave then stores whole rows.  As the
// accumulators lie, 16 rows of 32 bytes an instruction, the 33 MB of bf16 of a
// round of tiles leave in 11 us, so in 8, the copy through LDS in it (1023 x 1001
// x 32003 float16: d 108 -> 101 us, dW 100 -> 94).  Small tiles, two blocks to
// a CU, are stored as they lie (1023 x 2731 x 1001: 27 us, by rows 29).
template <class Cfg>
struct RowImage {
  static constexpr bool USED = Cfg::BLOCKS_PER_CU == 1;
  static constexpr int PITCH = Cfg::BN * 4, ROWS = USED ? Cfg::HM / Cfg::WAVES : 0;  // a wave's rows of a half
  char* lds;
  const Place& p;

  // Half h, whole for every wave of the block when it returns.
  __device__ __forceinline__ void put(const f4 (&acc)[Cfg::MI][Cfg::NJ], int h) const {
    const int i16 = p.lane & 15;
    if (h) __syncthreads();  // the last half has been read
#pragma unroll
    for (int i = 0; i < Cfg::MI / 2; ++i)
#pragma unroll
      for (int j = 0; j < Cfg::NJ; ++j) {
        const int row = p.wm * Cfg::QM + i * 16 + i16, chunk = (p.wn * Cfg::QN + Cfg::col(j)) / 4 + (p.lane >> 4);
        *(P2P_LDS f4*)((P2P_LDS char*)(lds) + row * PITCH + ((chunk ^ i16) << 4)) = acc[h * (Cfg::MI / 2) + i][j];
      }
    __syncthreads();
  }
  __device__ __forceinline__ f4 get(int row, int chunk) const {
    return *(const P2P_LDS f4*)((const P2P_LDS char*)(lds) + row * PITCH + ((chunk ^ (row & 15)) << 4));
  }
  // Row r of a wave, PER of them an instruction: the waves' rows alternate, so that few rows are shared by all.
  template <int PER>
  static __device__ __forceinline__ int row(int wave, int r) {
    return (r / PER * Cfg::WAVES + wave) * PER + r % PER;
  }
};
// f(r, m, n, C[m][n .. n + 3]) over the wave's part of the tile, n in steps of 4; r: which of its rows m is.
template <class Cfg, typename F>
__device__ __forceinline__ void by_rows(const f4 (&acc)[Cfg::MI][Cfg::NJ], const Place& p, char* lds, const F& f) {
  if constexpr (RowImage<Cfg>::USED) {
    static_assert(Cfg::BN == 256, "a row per instruction");
    constexpr int ROWS = RowImage<Cfg>::ROWS;
    const RowImage<Cfg> image{lds, p};
    const int64_t n = static_cast<int64_t>(p.tn) * Cfg::BN + p.lane * 4;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      image.put(acc, h);
      const int64_t m0 = static_cast<int64_t>(p.tm) * Cfg::BM + h * Cfg::HM;
#pragma unroll 4
      for (int r = 0; r < ROWS; ++r) {
        const int row = image.template row<1>(p.wave, r);
        f(h * ROWS + r, m0 + row, n, image.get(row, p.lane));
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < Cfg::MI; ++i)
#pragma unroll
      for (int j = 0; j < Cfg::NJ; ++j)
        f(i * 16 + (p.lane & 15), p.m0 + Cfg::row(i) + (p.lane & 15), p.n0 + Cfg::col(j) + (p.lane >> 4) * 4, acc[i][j]);
  }
}
// The row m whose number r is the lane's own: the lane requests what the row needs from memory before the image is
// made, and the others take it from there.
template <class Cfg>
__device__ __forceinline__ int64_t row_of_lane(const Place& p) {
  if constexpr (RowImage<Cfg>::USED) {
    constexpr int ROWS = RowImage<Cfg>::ROWS;
    static_assert(2 * ROWS <= 64, "");
    const int r = p.lane & (2 * ROWS - 1);
    return static_cast<int64_t>(p.tm) * Cfg::BM + r / ROWS * Cfg::HM + RowImage<Cfg>::template row<1>(p.wave, r % ROWS);
  } else {
    static_assert(Cfg::MI == 4, "64 rows");
    return p.m0 + (p.lane / 32) * Cfg::HM + p.lane % 32;  // Cfg::row(lane / 16) + lane % 16
  }
}

// x of lane r, which in an image's rows is the wave's.
template <class Cfg, typename T>
__device__ __forceinline__ T from_lane(T x, int r) {
  if constexpr (RowImage<Cfg>::USED) return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), r));
  else return __shfl(x, r, 64);
}

// Four neighbours of one row, columns n .. n + 3 of `cols`, as T.
template <typename T>
__device__ __forceinline__ void store4(T* row, int64_t n, int64_t cols, f4 v) {
  if (n + 4 <= cols) {
    Pack<T, 4> p;
#pragma unroll
    for (int i = 0; i < 4; ++i) p.v[i] = static_cast<T>(v[i]);
    store_pack<T, 4>(row + n, p);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < cols) stg(row + n + i, static_cast<T>(v[i]));
  }
}
__device__ __forceinline__ void store4_as(void* base, int32_t dtype, int64_t row, int64_t pitch, int64_t n, int64_t cols,
                                          f4 v) {
  if (dtype == P2P_DTYPE_F32) store4(static_cast<float*>(base) + row * pitch, n, cols, v);
  else if (dtype == P2P_DTYPE_F16) store4(static_cast<f16*>(base) + row * pitch, n, cols, v);
  else store4(static_cast<bf16*>(base) + row * pitch, n, cols, v);
}

// A float as three bf16 (their bits): hi + mid + lo == x.
struct Planes {
  uint16_t p[3];
};
__device__ __forceinline__ uint16_t bf16_bits(float x) { return __builtin_bit_cast(uint16_t, static_cast<bf16>(x)); }
__device__ __forceinline__ Planes split3(float x) {
  Planes r;
  const uint32_t b = __float_as_uint(x);
  const bool finite = (b & 0x7f800000u) != 0x7f800000u;
  r.p[0] = bf16_bits(x);
  // the largest floats would round up to an infinity: cut them off instead
  if (finite && (r.p[0] & 0x7fff) == 0x7f80) r.p[0] = static_cast<uint16_t>(b >> 16);
  const float rest = finite ? x - __uint_as_float(static_cast<uint32_t>(r.p[0]) << 16) : 0.f;
  r.p[1] = bf16_bits(rest);
  r.p[2] = bf16_bits(rest - __uint_as_float(static_cast<uint32_t>(r.p[1]) << 16));
  return r;
}
// The six kept products, small ones first: (plane of A, plane of B).
constexpr int kSplitA[6] = {0, 2, 1, 0, 1, 0}, kSplitB[6] = {2, 0, 1, 1, 0, 0};

// C = alpha * acc as `dtype`, or the raw sums of one k-run into its own
// float plane (`partial`; add: on top of what is there).  With `half` > 0
// the rows from `half` on are a second result's (rows past `rows` of either
// are padding).
struct StoreEpi {
  void* out[2];
  int64_t half, rows;
  int64_t pitch;
  int32_t dtype;
  const float* scale[2];  // device factors (nullable)
  float alpha;
  float* partial;         // [ksplit][M][pitch]
  int add;

  template <class Cfg>
  __device__ __forceinline__ void finish(f4 (&acc)[Cfg::MI][Cfg::NJ], const Place& p, const GemmArgs& g, char* lds) const {
    float a = alpha;
    if (scale[0]) a *= ldc(scale[0]);
    if (scale[1]) a *= ldc(scale[1]);
    by_rows<Cfg>(acc, p, lds, [&](int, int64_t m, int64_t n, f4 v) {
      if (m >= g.M || n >= g.N) return;
      if (partial) {
        float* to = partial + (p.part * g.M + m) * pitch;
        if (add) {
          float o[4];
          load_row<float, 4>(to, n, g.N, o);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] += o[e];
        }
        store4(to, n, g.N, v);
        return;
      }
      const bool second = half > 0 && m >= half;
      const int64_t row = second ? m - half : m;
      if (half > 0 && row >= rows) return;
      store4_as(out[second], dtype, row, pitch, n, g.N, v * a);
    });
  }
};

// ------------------------------------------------------------------ host side
template <bool F16, bool AT, bool BT, bool DUAL, class Cfg, class Epi>
static int32_t gemm_launch_cfg(const GemmArgs& g, const Epi& epi, hipStream_t st) {
  const int64_t tiles = ceil_div(g.M, Cfg::BM) * ceil_div(g.N, Cfg::BN);
  if (tiles > (int64_t(1) << 31) / Cfg::THREADS) return P2P_ERR_UNSUPPORTED;
  gemm_kernel<F16, AT, BT, DUAL, Cfg, Epi>
      <<<dim3(static_cast<unsigned>(tiles), g.ksplit), dim3(Cfg::THREADS), 0, st>>>(g, epi);
  return launch_status();
}

template <bool AT, bool BT, bool DUAL, class Epi>
static int32_t gemm_launch(const GemmArgs& g, bool is_f16, bool big, const Epi& epi, hipStream_t st) {
  if (is_f16)
    return big ? gemm_launch_cfg<true, AT, BT, DUAL, Big>(g, epi, st)
               : gemm_launch_cfg<true, AT, BT, DUAL, Small>(g, epi, st);
  return big ? gemm_launch_cfg<false, AT, BT, DUAL, Big>(g, epi, st)
             : gemm_launch_cfg<false, AT, BT, DUAL, Small>(g, epi, st);
}

// Tile and k-runs of a product: what is least by the times of a k-step (us) of a
// round of blocks, 256 large or 512 small ones (256 alone on their CUs take
// less), and of writing and joining the runs' sums.  Kernel times, large / small
// (runs): M x N x K = 2048 x 4096 x 2048 64.3 / 43.8; 4096 x 2048 x 2048 57.1 (2) /
// 43.3 (1); 4096 x 512 x 4096 44.2 (8) / 33.0 (4); 1024 x 4096 x 8192 89.3 (4) /
// 82.7 (2); 1024 x 1000 x 64000 144.8 (16) / 173.9 (8); 8192 x 4096 x 1024 82.3 /
// 95.6; 1024 x 32000 x 1000 84.6 / 104.8.  Tiles of 256 x 128 were between the
// two or behind them everywhere.
constexpr int kMinRun = 8;
struct Plan {
  bool big;
  int split;
};
static inline double gemm_time(bool big, int64_t tiles, int64_t steps, int split, int64_t out) {
  const int64_t blocks = tiles * split, slots = big ? 256 : 512, rest = blocks % slots;
  const double round = big ? 1.8 : 1.05, last = rest == 0 ? 0.0 : !big && rest <= 256 ? 0.74 : round;
  const double product = (static_cast<double>(blocks / slots) * round + last) * static_cast<double>(ceil_div(steps, split));
  return split == 1 ? product : product + 5.0 + 8.0 * split * static_cast<double>(out) / 6.0e6;
}
static inline Plan gemm_plan(int64_t M, int64_t N, int64_t steps, bool may_split) {
  const int64_t tb = ceil_div(M, Big::BM) * ceil_div(N, Big::BN), ts = ceil_div(M, Small::BM) * ceil_div(N, Small::BN);
  const int64_t most = may_split ? std::max<int64_t>(1, steps / kMinRun) : 1;
  Plan best{true, 1};
  double least = gemm_time(true, tb, steps, 1, M * N);
  for (const int split : {1, 2, 3, 4, 6, 8, 12, 16})
    for (const bool big : {true, false}) {
      if (split > most) return best;
      const double t = gemm_time(big, big ? tb : ts, steps, split, M * N);
      if (t < least) least = t, best = Plan{big, split};
    }
  return best;
}
static inline int64_t ksteps(int64_t K, int nseg) { return ceil_div(K, kGemmK) * nseg; }

// An operand as the product reads it: 16-bit planes (one, or three of a float32 tensor).
struct Mat {
  const uint16_t* plane[3];
  int64_t ld;
};

// Whether a 16-bit tensor can be read where it is.
static inline bool in_place(const void* p, int64_t ld, int64_t cols, int32_t dtype) {
  return dtype != P2P_DTYPE_F32 && aligned_to(p, 16) && ld % 8 == 0 && cols % 8 == 0 && ld <= kMaxPitch;
}
static inline int64_t round_up(int64_t n, int64_t to) { return ceil_div(n, to) * to; }
// The pitch of a copy or of d: whole 128-byte lines, on which a tile's rows
// begin (1023 x 1001 x 32003 float16, forward and backward: 457 us with pitches
// of 16 bytes, 442 so).
static inline int64_t line_pitch(int64_t cols) { return round_up(cols, cols > 32 ? 64 : 8); }
static inline int planes_of(int32_t dtype) { return dtype == P2P_DTYPE_F32 ? 3 : 1; }
static inline int64_t packed_bytes(int64_t rows, int64_t cols, int32_t dtype) {
  return round_up(rows * line_pitch(cols) * 2 * planes_of(dtype), 256);
}

// src [rows, cols], pitch ld, as 16-bit planes of pitch line_pitch(cols) at dst, zeros in the
// added columns.  Up to kMaxPack of them in one launch; those without a dst are left out.
constexpr int kMaxPack = 3;
struct PackJob {
  const void* src;
  int64_t ld, rows, cols;
  uint16_t* dst;
  int64_t pitch;  // set by pack_matrices
};
P2P_INTERNAL int32_t pack_matrices(const PackJob* jobs, int n, int32_t dtype, hipStream_t st);

// What the product reads of a job: its copy, or src in place where it has none.
static inline Mat mat_of(const PackJob& j, int32_t dtype) {
  if (!j.dst) return Mat{{static_cast<const uint16_t*>(j.src), nullptr, nullptr}, j.ld};
  const int64_t pitch = line_pitch(j.cols), plane = j.rows * pitch;
  const bool three = planes_of(dtype) == 3;
  return Mat{{j.dst, three ? j.dst + plane : nullptr, three ? j.dst + 2 * plane : nullptr}, pitch};
}
// out0[i] = alpha * (parts[i] + parts[stride + i] + ...) in that order, i < n; out1 (nullable) the same from parts + second.
P2P_INTERNAL int32_t join_parts(const float* parts, int nparts, int64_t stride, int64_t n, int64_t second, const float* scale0,
                                const float* scale1, float alpha, void* out0, void* out1, int32_t dtype, hipStream_t st);

// The pairs of a product of two operands, appended to g (DUAL: b2 too).
static inline void add_pairs(GemmArgs* g, const Mat& a, const Mat& b, const Mat* b2, int32_t dtype) {
  const int n = dtype == P2P_DTYPE_F32 ? 6 : 1;
  for (int i = 0; i < n; ++i) {
    const int pa = n == 1 ? 0 : kSplitA[i], pb = n == 1 ? 0 : kSplitB[i];
    g->a[g->nseg] = a.plane[pa];
    g->b[g->nseg] = b.plane[pb];
    g->b2[g->nseg] = b2 ? b2->plane[pb] : nullptr;
    ++g->nseg;
  }
}

// Bytes handed out of a workspace; with base null it only counts them.
struct Carver {
  char* base;
  int64_t used = 0;
  void* take(int64_t bytes) {
    void* p = base ? base + used : nullptr;
    used += round_up(bytes, 256);
    return p;
  }
};

}  // namespace p2p
