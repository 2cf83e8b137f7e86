// SPDX-License-Identifier: MIT OR Apache-2.0
//
// What the templated CUDA-core kernels (hd_ffma.cu, cross_hd_ffma.cu) share: tile sizes, row loads,
// the score products and the dims of a thread.
#pragma once

#include "cfa_common.cuh"

namespace cfa {
namespace {

template <int D>
struct Hd;
// The forward's rows per thread: two candidates per head dim (query tiles of 8 RPT rows), the one
// that pads fewer rows at the sequence length taken (hd_fwd_rows; rows are independent, so the
// choice changes no bit), and blocks per SM.
template <>
struct Hd<32> {
  static constexpr int RPT_A = 8, RPT_B = 6;  // 64- or 48-query tiles
  static constexpr int FWD_MINB = 3;          // forward blocks per SM (registers)
};
template <>
struct Hd<128> {
  // 48-query tiles at every length: against 32-query tiles (4 rows per thread) they measured
  // faster at every shape tried (canvas-shaped 185 -> 158 us, s = 4096 causal 917 -> 820 us).
  static constexpr int RPT_A = 6, RPT_B = 6;
  static constexpr int FWD_MINB = 2;          // (shared memory: 107.3 KB per block)
};

template <int RPT>
__host__ __device__ constexpr int fwd_bm() {
  return 8 * RPT;  // 4 warps x 2 half-warps x RPT rows
}

// Row stride of the [rows][D] tiles: D + 4 floats, rows 16-byte aligned and 4 banks apart.
template <int D>
__host__ __device__ constexpr int ldh() {
  return D + 4;
}

template <int D, int RPT>
__host__ __device__ constexpr int hd_fwd_smem_floats() {
  return (fwd_bm<RPT>() + 2 * 64) * ldh<D>() + fwd_bm<RPT>() * LDP;
}

template <int D>
__host__ __device__ constexpr int hd_bwd_smem_floats() {
  return 4 * 64 * ldh<D>() + 2 * 64 * LDP + 2 * 64 + 4;
}

// ROWS rows of a strided [seq, D] slice starting at row0 into a [ROWS][D + 4] tile (zero past seq;
// the address given for such rows is row0's, which is < seq).
template <int ROWS, int NT, int D>
__device__ __forceinline__ void load_rows_async(float* dst, const float* __restrict__ src,
                                                int64_t s_stride, int row0, int seq) {
  constexpr int C = D / 4;
#pragma unroll
  for (int idx = threadIdx.x; idx < ROWS * C; idx += NT) {
    const int r = idx / C, c4 = idx % C;
    const int row = row0 + r;
    const bool ok = row < seq;
    const float* g = src + static_cast<int64_t>(ok ? row : row0) * s_stride + 4 * c4;
    cp_async16(dst + r * ldh<D>() + 4 * c4, g, ok ? 16 : 0);
  }
}

// S = A B^T for NR rows (rb + 2i) and the first JN of 4 key groups (keys tx + 16jj): an even-d
// chain plus an odd-d chain per score, as the head-dim-64 kernels do. Groups >= JN are left at 0.
template <int JN, int NR, int D>
__device__ __forceinline__ void scores(const float* As, const float* Bs, int rb, int tx,
                                       float (&s)[NR][4]) {
  uint64_t s2[NR][JN];
#pragma unroll
  for (int i = 0; i < NR; ++i)
#pragma unroll
    for (int jj = 0; jj < JN; ++jj) s2[i][jj] = 0ull;
#pragma unroll 2
  for (int c = 0; c < D; c += 4) {
    ulonglong2 bv[JN], av[NR];
#pragma unroll
    for (int jj = 0; jj < JN; ++jj) bv[jj] = ld2x2(Bs + (tx + 16 * jj) * ldh<D>() + c);
#pragma unroll
    for (int i = 0; i < NR; ++i) av[i] = ld2x2(As + (rb + 2 * i) * ldh<D>() + c);
#pragma unroll
    for (int i = 0; i < NR; ++i)
#pragma unroll
      for (int jj = 0; jj < JN; ++jj) s2[i][jj] = fma2(av[i].x, bv[jj].x, s2[i][jj]);
#pragma unroll
    for (int i = 0; i < NR; ++i)
#pragma unroll
      for (int jj = 0; jj < JN; ++jj) s2[i][jj] = fma2(av[i].y, bv[jj].y, s2[i][jj]);
  }
#pragma unroll
  for (int i = 0; i < NR; ++i)
#pragma unroll
    for (int jj = 0; jj < 4; ++jj) s[i][jj] = jj < JN ? sum2(s2[i][jj < JN ? jj : 0]) : 0.0f;
}

// This thread's D / 16 output dims of a row, as register pairs: D = 32 -> dims 2tx, 2tx + 1 (one
// pair); D = 128 -> dims 4tx .. 4tx + 3 and 64 + 4tx .. 64 + 4tx + 3 (four pairs).
template <int D>
struct Dims;
template <>
struct Dims<32> {
  static constexpr int NP = 1;
  __device__ __forceinline__ static void load(const float* row, int tx, uint64_t (&v)[1]) {
    v[0] = *reinterpret_cast<const uint64_t*>(row + 2 * tx);
  }
  __device__ __forceinline__ static void load_f(const float* row, int tx, float (&v)[2]) {
    const float2 x = *reinterpret_cast<const float2*>(row + 2 * tx);
    v[0] = x.x;
    v[1] = x.y;
  }
};
template <>
struct Dims<128> {
  static constexpr int NP = 4;
  __device__ __forceinline__ static void load(const float* row, int tx, uint64_t (&v)[4]) {
    const ulonglong2 a = ld2x2(row + 4 * tx), b = ld2x2(row + 64 + 4 * tx);
    v[0] = a.x;
    v[1] = a.y;
    v[2] = b.x;
    v[3] = b.y;
  }
  __device__ __forceinline__ static void load_f(const float* row, int tx, float (&v)[8]) {
    const float4 a = ld4(row + 4 * tx), b = ld4(row + 64 + 4 * tx);
    v[0] = a.x;
    v[1] = a.y;
    v[2] = a.z;
    v[3] = a.w;
    v[4] = b.x;
    v[5] = b.y;
    v[6] = b.z;
    v[7] = b.w;
  }
};

// Store this thread's D / 16 dims of a row (the layout of Dims<D>) into row `dst`.
template <int D>
__device__ __forceinline__ void store_dims(float* dst, int tx, const float (&v)[D / 16]) {
  if constexpr (D == 32) {
    *reinterpret_cast<float2*>(dst + 2 * tx) = make_float2(v[0], v[1]);
  } else {
    *reinterpret_cast<float4*>(dst + 4 * tx) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(dst + 64 + 4 * tx) = make_float4(v[4], v[5], v[6], v[7]);
  }
}

// The backward's thread layout.
template <int D>
struct Bwd;
template <>
struct Bwd<32> {
  static constexpr int NT = 256, WG = 4;   // threads; warps per group
  static constexpr int R1 = 8;             // phase 1 rows per thread (rows rb1 + 2i)
  static constexpr int K2 = 8;             // phase 2 keys per thread
  static constexpr int NP2 = 1;            // phase 2 dim pairs per key pair (dims 2tx, 2tx + 1)
};
template <>
struct Bwd<128> {
  static constexpr int NT = 512, WG = 8;
  static constexpr int R1 = 4;
  static constexpr int K2 = 4;
  static constexpr int NP2 = 4;            // dims 4tx .. + 3 and 64 + 4tx .. + 3
};

}  // namespace
}  // namespace cfa
