// SPDX-License-Identifier: MIT OR Apache-2.0
//
// What the tensor-core backwards (bwd_tc.cu, cross_bwd_tc.cu) share: the tile sizes, the shared
// memory and TMEM layouts, the row items and their splits, and the six-product windows.
#pragma once

#include <cuda_bf16.h>

#include "cfa_common.cuh"
#include "cfa_internal.h"
#include "cfa_split.cuh"
#include "cfa_tc.cuh"

namespace cfa {
using tc::kmaj_off;
using tc::split16;
using tc::split8;
using tc::store_parts;
using tc::tmem_ld8;
using tc::tmem_st8;
namespace {

constexpr int KB = 128;   // keys per block: MMA M of S^T, dP^T, dV, dK
constexpr int QT = 64;    // queries per tile: MMA N of S^T, dP^T; M of dQ
constexpr int NT = 512;   // compute threads (16 warps)
constexpr int NB = NT + 32;  // and the MMA warp
constexpr int PART_K = KB * 64 * 2;  // one bf16 part of a [128][64] operand
constexpr int PART_Q = QT * 64 * 2;  // one bf16 part of a [64][64] operand
constexpr int OFF_K = 0;                      // K parts [128 keys][64 d]
constexpr int OFF_Q = OFF_K + 3 * PART_K;     // Q parts [64 q][64 d], two tiles
constexpr int OFF_DO = OFF_Q + 6 * PART_Q;    // dO parts [64 q][64 d], two tiles
constexpr int OFF_DS = OFF_DO + 6 * PART_Q;   // dS^T parts [128 keys][64 q] (first: K staged)
constexpr int OFF_ST = OFF_DS + 3 * PART_K;   // staging: the next tile's Q, dO (fp32)
constexpr int OFF_LD = OFF_ST + 2 * QT * 64 * 4;  // L, D of two tiles: float [2][2][64]
constexpr int OFF_BAR = OFF_LD + 2 * 2 * QT * 4;  // eight mbarriers, the TMEM base, four ints
constexpr int SMEM = OFF_BAR + 96;
constexpr int SMEM_ALLOC = SMEM + 1024;
static_assert(SMEM_ALLOC <= 232448, "shared memory per block");
// TMEM columns (lane = key row). V's parts, the A operand of dP^T: part i, K-step ks (16 dims) in
// the 8 columns T_V + 32 i + 8 ks. S^T, dP^T of the current tile; P^T's parts (the A operand of
// dV: pt_col) over the S^T columns each thread has read and in T_X; dV, dK; dQ's two 64-key
// windows (M = 64).
constexpr uint32_t T_V = 0, T_S = 96, T_DP = 160, T_DV = 224, T_DK = 288, T_DQ0 = 352,
                   T_DQ1 = 416, T_X = 480;
constexpr uint32_t TMEM_COLS = 512;

// A split tail's window of one query tile (dV, dK sums of the tile as TMEM holds them, before the
// fold): WIN floats as float4 items [which: dV, dK][c4][column group][key row], so a warp's 32
// rows of one item are 512 contiguous bytes (coalesced stores, conflict-free shared-memory reads).
template <int HD>
struct TailWindow {
  static constexpr int WIN = 2 * KB * HD;
  static constexpr int CG = HD / 16;  // column groups of 16 floats
  __host__ __device__ static constexpr int item(int which, int c4, int cg, int row) {
    return ((which * 4 + c4) * CG + cg) * KB + row;
  }
};

// P^T part i of K-step ks (queries 16 ks .. 16 ks + 15: the columns of group ks): parts 0, 1 over
// that group's S^T columns, part 2 in T_X + 8 ks -- dP^T stays whole until dS^T is formed from
// it, while dV already runs.
__host__ __device__ constexpr uint32_t pt_col(int i, int ks) {
  return i < 2 ? T_S + 16 * ks + 8 * i : T_X + 8 * ks;
}
static_assert(T_X + 32 == TMEM_COLS, "TMEM budget");

// Row items (row r, elements 8 kc .. 8 kc + 7): item c takes row 8 (c / 64) + c % 8 and chunk
// (c / 8) % 8 (a quarter-warp writes 8 rows of one chunk: 8 bank groups). Every thread copies
// (cp.async) the fp32 chunks it splits into slots of its own: slot j of thread t at
// (j * NT + t) * 16 bytes.
__device__ __forceinline__ void row_item(int c, int& r, int& kc) {
  r = 8 * (c >> 6) + (c & 7);
  kc = (c >> 3) & 7;
}

// (Head dim 32: the row's chunks past the head dim are zero-filled, so the parts are those of a
// 64-wide row whose upper half is zero.)
template <int HD>
__device__ __forceinline__ void stage_row_item(unsigned char* st, int slot, int c, const float* src,
                                               int64_t stride, int r0, int seq) {
  int r, kc;
  row_item(c, r, kc);
  const bool ok = r0 + r < seq && 8 * kc < HD;
  const float* g = src + static_cast<int64_t>(ok ? r0 + r : 0) * stride + 8 * kc;
  cp_async16(st + 16 * ((2 * slot) * NT + threadIdx.x), g, ok ? 16 : 0);
  cp_async16(st + 16 * ((2 * slot + 1) * NT + threadIdx.x), g + 4, ok ? 16 : 0);
}

__device__ __forceinline__ void split_row_item(unsigned char* parts, int part_bytes,
                                               const unsigned char* st, int slot, int c) {
  int r, kc;
  row_item(c, r, kc);
  const float4 u = *reinterpret_cast<const float4*>(st + 16 * ((2 * slot) * NT + threadIdx.x));
  const float4 v = *reinterpret_cast<const float4*>(st + 16 * ((2 * slot + 1) * NT + threadIdx.x));
  const float x[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
  store_parts(parts, part_bytes, kmaj_off(r, kc), x);
}

// Row item c of a row-major staging area with rows of 68 floats (rows >= valid and columns >= HD
// read as zeros) into the K-major parts at part_bytes apart.
template <int HD>
__device__ __forceinline__ void split_staged_row(unsigned char* parts, int part_bytes,
                                                 const float* rows, int c, int valid) {
  int r, kc;
  row_item(c, r, kc);
  float x[8];
  if (r < valid && 8 * kc < HD) {
    const float4 u = reinterpret_cast<const float4*>(rows + r * 68 + 8 * kc)[0];
    const float4 v = reinterpret_cast<const float4*>(rows + r * 68 + 8 * kc)[1];
    x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w, x[4] = v.x, x[5] = v.y, x[6] = v.z, x[7] = v.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = 0.0f;
  }
  store_parts(parts, part_bytes, kmaj_off(r, kc), x);
}

// One window: six split products over STEPS K-steps into the fresh accumulator `d`; descriptors
// advance by A_STEP / B_STEP bytes per step and by A_PART / B_PART bytes per part. Part pairs
// (P0(p), P1(p)) -- the small (0, 1), (1, 0), (0, 2), (1, 1), (2, 0) of every step, then the
// (0, 0) of every step -- or, SWAP, (P1(p), P0(p)): the order in which the forward forms its
// products when A and B trade places. Called by the whole MMA warp (tc::mma_bf16_warp).
__host__ __device__ constexpr int P0(int p) { return p == 2 || p == 4 ? 1 : (p == 5 ? 2 : 0); }
__host__ __device__ constexpr int P1(int p) { return p == 1 || p == 4 ? 1 : (p == 3 ? 2 : 0); }
template <int STEPS, int A_PART, int B_PART, int A_STEP, int B_STEP, bool SWAP>
__device__ __forceinline__ void issue6(uint32_t d, tc::Desc ad, tc::Desc bd, uint32_t idesc) {
  const uint32_t alo = tc::opaque(ad.lo), blo = tc::opaque(bd.lo);
#pragma unroll
  for (int ks = 0; ks < STEPS; ++ks)
#pragma unroll
    for (int p = 1; p < 6; ++p) {
      const int pa = SWAP ? P1(p) : P0(p), pb = SWAP ? P0(p) : P1(p);
      tc::mma_bf16_warp(d, alo + ((pa * A_PART + A_STEP * ks) >> 4), ad.hi,
                        blo + ((pb * B_PART + B_STEP * ks) >> 4), bd.hi, idesc, ks > 0 || p > 1);
    }
#pragma unroll
  for (int ks = 0; ks < STEPS; ++ks)
    tc::mma_bf16_warp(d, alo + ((A_STEP * ks) >> 4), ad.hi, blo + ((B_STEP * ks) >> 4), bd.hi,
                      idesc, 1);
}

// The same window with the A operand in TMEM: part i of K-step ks at column acol(i, ks).
template <int B_PART, int B_STEP, typename ACol, int STEPS = 4>
__device__ __forceinline__ void issue6_tmem_a(uint32_t d, ACol acol, tc::Desc bd, uint32_t idesc) {
  const uint32_t blo = tc::opaque(bd.lo);
#pragma unroll
  for (int ks = 0; ks < STEPS; ++ks)
#pragma unroll
    for (int p = 1; p < 6; ++p)
      tc::mma_bf16_tmem_a_warp(d, acol(P0(p), ks), blo + ((P1(p) * B_PART + B_STEP * ks) >> 4),
                               bd.hi, idesc, ks > 0 || p > 1);
#pragma unroll
  for (int ks = 0; ks < STEPS; ++ks)
    tc::mma_bf16_tmem_a_warp(d, acol(0, ks), blo + ((B_STEP * ks) >> 4), bd.hi, idesc, 1);
}

constexpr float LOG2E = 1.4426950408889634f;  // log2(e), rounded to fp32

// Packed fp32 pairs (tc::pack2 / unpack2), one instruction a pair.
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t fma2v(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}

// Eight floats to global memory in one 32-byte store (address 32-byte aligned), cached in L2 only.
__device__ __forceinline__ void st_cg_v8(float* p, const float (&v)[8]) {
  asm volatile("st.global.cg.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(v[0]),
               "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
               : "memory");
}

// atomicAdd with acquire-release semantics at GPU scope.
__device__ __forceinline__ int atom_add_acq_rel(int* p, int v) {
  int old;
  asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], %2;" : "=r"(old) : "l"(p), "r"(v) : "memory");
  return old;
}

// Named barrier 1: the 16 compute warps (the MMA warp never takes part).
__device__ __forceinline__ void bar_sync(int id, int count) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(count) : "memory");
}

}  // namespace
}  // namespace cfa
