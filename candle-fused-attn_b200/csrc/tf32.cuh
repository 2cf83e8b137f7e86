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

}  // namespace
}  // namespace cfa
