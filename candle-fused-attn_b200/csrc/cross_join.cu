// SPDX-License-Identifier: MIT OR Apache-2.0
//
// The sums that cross attention's backwards leave to a kernel of their own: dQ = scale * (((p0 + p1) +
// p2) + ..) over the key blocks that take part, and, where the query tiles were cut into parts, dK and
// dV over the parts -- in these fixed orders, so reruns and batch splits give the same bits. Bound by
// memory: every partial is read once, four floats a thread.
#include "cfa_common.cuh"

namespace cfa {
namespace {

constexpr int JT = 256;

__device__ __forceinline__ float4 add4(float4 a, float4 b) {
  return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w);
}

__global__ void __launch_bounds__(JT) cross_join_kernel(const BwdArgs a, int D, int key_block,
                                                        int64_t n_dq, int64_t n_dkv) {
  griddep_wait();
  griddep_launch_dependents();
  const int C4 = D / 4;
  for (int64_t x = static_cast<int64_t>(blockIdx.x) * JT + threadIdx.x; x < n_dq + n_dkv;
       x += static_cast<int64_t>(gridDim.x) * JT) {
    if (x < n_dq) {  // (batch, head), query, column
      const int64_t row = x / C4, bh = row / a.S;
      const int c4 = static_cast<int>(x - row * C4), i = static_cast<int>(row - bh * a.S);
      const int b = static_cast<int>(bh / a.H), head = static_cast<int>(bh - static_cast<int64_t>(b) * a.H);
      const int keys = cross_keys(a, b), nkb = (keys + key_block - 1) / key_block;
      const float scale = grad_scale(a, keys);
      const float4* p = reinterpret_cast<const float4*>(a.dq_part) + (bh * a.n_kblocks * a.S + i) * C4 + c4;
      const int64_t step = static_cast<int64_t>(a.S) * C4;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (nkb > 0) v = __ldcs(p);
#pragma unroll 4
      for (int j = 1; j < nkb; ++j) v = add4(v, __ldcs(p + j * step));
      reinterpret_cast<float4*>(a.dq)[((static_cast<int64_t>(b) * a.S + i) * a.H + head) * C4 + c4] =
          make_float4(v.x * scale, v.y * scale, v.z * scale, v.w * scale);
    } else {
      const int64_t y = x - n_dq;
      const float4* p = reinterpret_cast<const float4*>(a.dkv) + y;
      float4 v = __ldcs(p);
#pragma unroll 4
      for (int j = 1; j < a.n_parts; ++j) v = add4(v, __ldcs(p + j * (a.part_stride / 4)));
      reinterpret_cast<float4*>(a.dkv_out)[y] = v;
    }
  }
}

}  // namespace

cudaError_t launch_cross_join(const BwdArgs& a, int head_dim, int key_block, cudaStream_t stream) {
  const int64_t n_dq = a.join_dq ? static_cast<int64_t>(a.B) * a.H * a.S * (head_dim / 4) : 0;
  const int64_t n_dkv =
      a.n_parts > 1 ? static_cast<int64_t>(a.B) * a.Sk * 2 * a.Hk * (head_dim / 4) : 0;
  if (n_dq + n_dkv == 0) return cudaSuccess;
  const int64_t blocks = (n_dq + n_dkv + JT - 1) / JT, most = 148 * 8;
  return launch_pdl(cross_join_kernel, dim3(static_cast<unsigned>(blocks < most ? blocks : most)), dim3(JT),
                    0, stream, a, head_dim, key_block, n_dq, n_dkv);
}

}  // namespace cfa
