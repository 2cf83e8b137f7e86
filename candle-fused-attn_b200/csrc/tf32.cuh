// SPDX-License-Identifier: MIT OR Apache-2.0
//
// fp32 products on the tensor core by two tf32 parts an operand (split_attn.cu, cross_hd_tf32.cu).
#pragma once

#include <cstdint>

namespace cfa {
namespace {

// x in two parts of 11 bits each, x = hi + lo to 2^-22 |x|: hi rounded to the nearest, lo what is left (the
// tensor core drops its last bits).
__device__ __forceinline__ void split_tf32(const float4 x, uint32_t (&hi)[4], uint32_t (&lo)[4]) {
  const float v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    hi[e] = (__float_as_uint(v[e]) + 0x1000u) & 0xffffe000u;
    lo[e] = __float_as_uint(v[e] - __uint_as_float(hi[e]));
  }
}
__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The tensor core truncates a sum at its own magnitude, step by step: with one chain of all products over
// 128 dims or 64 keys, head dim 128's outputs were 8e-7 off in norm and gradients 1.2e-6. So the small
// products come first or in a sum of their own, and the large ones' sums are short (32 dims, 32 keys) and
// added in fp32: 1e-7 to 4e-7 and 2e-7 to 7e-7, for 2 % of the forward's time and 4 % of the backward's.
//
// A k-step of A (parts ah, al) times four columns of B (b0: k = t, b1: k = t + 4).
__device__ __forceinline__ void products(float (&small)[4][4], float (&large)[4][4], const uint32_t (&ah)[4],
                                         const uint32_t (&al)[4], const float4 b0, const float4 b1) {
  uint32_t xh[4], xl[4], yh[4], yl[4];
  split_tf32(b0, xh, xl);
  split_tf32(b1, yh, yl);
#pragma unroll
  for (int e = 0; e < 4; ++e) mma_tf32(small[e], al, xh[e], yh[e]);
#pragma unroll
  for (int e = 0; e < 4; ++e) mma_tf32(large[e], ah, xh[e], yh[e]);
#pragma unroll
  for (int e = 0; e < 4; ++e) mma_tf32(small[e], ah, xl[e], yl[e]);
}
// Two k-steps (dims 0, 1 and 2, 3 of b) of A times one column of a row-major B.
__device__ __forceinline__ void products(float (&c)[4], const uint32_t (&ah)[2][4], const uint32_t (&al)[2][4],
                                         const float4 b) {
  uint32_t h[4], l[4];
  split_tf32(b, h, l);
#pragma unroll
  for (int y = 0; y < 2; ++y) mma_tf32(c, al[y], h[2 * y], h[2 * y + 1]);
#pragma unroll
  for (int y = 0; y < 2; ++y) mma_tf32(c, ah[y], l[2 * y], l[2 * y + 1]);
#pragma unroll
  for (int y = 0; y < 2; ++y) mma_tf32(c, ah[y], h[2 * y], h[2 * y + 1]);
}
// The parts of rows g (x) and g + 8 (y) of A for two k-steps (dims 0, 1 and 2, 3).
__device__ __forceinline__ void split_rows(const float4 x, const float4 y, uint32_t (&ah)[2][4],
                                           uint32_t (&al)[2][4]) {
  split_tf32(make_float4(x.x, y.x, x.y, y.y), ah[0], al[0]);
  split_tf32(make_float4(x.z, y.z, x.w, y.w), ah[1], al[1]);
}
template <int N>
__device__ __forceinline__ void clear(float (&c)[N][4]) {
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int x = 0; x < 4; ++x) c[i][x] = 0.0f;
}
template <int N>
__device__ __forceinline__ void add(float (&s)[N][4], const float (&c)[N][4]) {
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int x = 0; x < 4; ++x) s[i][x] += c[i][x];
}

}  // namespace
}  // namespace cfa
