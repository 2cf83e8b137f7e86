// SPDX-License-Identifier: MIT OR Apache-2.0
//
// Rotary positions (cfa_rotary) and the paged cache's append (cfa_paged_append).
//
// A pair (x1, x2) of frequency f_j (radians a position) at position p is turned by the angle p f_j:
//   y1 = x1 c - x2 s,  y2 = x2 c + x1 s,  c = A cos(p f_j),  s = A sin(p f_j),
// with pairs (j, j + r/2) or, interleaved, (2j, 2j + 1) of the first r dims; the other dims are
// copied. The inverse (the backward: the transpose of the rotation) negates s.
//
// Angles. p f_j is taken in 64 bits as t = p f_j / 2 pi, whose whole turns are dropped there: what
// is left, |t| <= 1/2, keeps an absolute error of 2^-53 |p f_j| when it is rounded to fp32, and
// sincospif(2 t) adds its own two ulp. In fp32 the product alone would be off by p f_j 2^-24 --
// 0.06 radians at position 10^6.
//
// Bound by memory: every element is read and written once, at 3 flops. A block takes `tokens`
// consecutive (batch, seq) positions and up to 1024 units of them -- a unit is two vectors of VEC
// elements, VEC pairs -- four a thread, all of whose loads are issued before the block computes its
// tokens' cosines and sines (one angle a thread and pass, shared by all heads, into shared memory).
//
// The append runs the same units over the heads of q, k and v: rotated q into its output, rotated
// k and plain v into the token's slot of the cache, rounded once from fp32 (or the 16-bit input).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "cfa_common.cuh"
#include "cfa_ops.h"

namespace cfa {
namespace {

constexpr int RT = 256;            // threads
constexpr int UPT = 4;             // units per thread
constexpr int MAX_UNITS = RT * UPT;
constexpr double INV_2PI = 0.15915494309189533577;

template <typename T>
__device__ __forceinline__ float to_f(T x);
template <>
__device__ __forceinline__ float to_f(float x) { return x; }
template <>
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f(float x) { return __float2bfloat16_rn(x); }

// VEC elements as one aligned access.
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Vec {
  T v[VEC];
};

// n / d for n d < 2^32 by one multiplication: m = ceil(2^32 / d) (d = 1: m = 0, n itself).
__device__ __forceinline__ uint32_t div_by(uint32_t n, uint32_t m) {
  return m ? __umulhi(n, m) : n;
}

// One unit's two vectors: element offsets a, b in the head's row (b < 0: the second is absent);
// pairs: the first pair's frequency, or -1 where the unit copies.
struct Unit {
  int a, b, pair;
};
template <int VEC>
__device__ __forceinline__ Unit unit_of(const RotaryArgs& p, int u, bool rotated) {
  const int r = rotated ? p.rot : 0;
  const int ru = r / (2 * VEC);
  if (u < ru)
    return p.interleaved ? Unit{2 * VEC * u, 2 * VEC * u + VEC, VEC * u}
                         : Unit{VEC * u, r / 2 + VEC * u, VEC * u};
  const int e = r + 2 * VEC * (u - ru);
  return {e, e + VEC < p.D ? e + VEC : -1, -1};
}

template <typename T, typename C, int VEC, bool APPEND>
__global__ void __launch_bounds__(RT) rotary_kernel(const RotaryArgs p) {
  extern __shared__ float cs[];  // [tokens][cos: rot / 2, sin: rot / 2]
  __shared__ int64_t slot_k[APPEND ? MAX_UNITS : 1], slot_v[APPEND ? MAX_UNITS : 1];
  griddep_wait();
  griddep_launch_dependents();
  const int tid = threadIdx.x;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * p.tokens;
  const int nt = static_cast<int>(min(static_cast<int64_t>(p.tokens), p.n_tokens - t0));
  const int h0 = static_cast<int>(blockIdx.y) * p.head_chunk;
  const int nh = min(p.head_chunk, p.H + (APPEND ? 2 * p.Hk : 0) - h0);
  const int n_units = nt * p.head_chunk * p.units;
  using V = Vec<T, VEC>;
  using W = Vec<C, VEC>;

  // The token of a unit, its (batch, seq), and whether it exists (append: a padded batch).
  auto position = [&](int64_t b, int64_t i, bool& valid) -> int64_t {
    if constexpr (APPEND) {
      int n = p.new_lengths ? p.new_lengths[b] : p.S;
      n = min(max(n, 0), p.S);
      const int64_t at = static_cast<int64_t>(p.lengths[b]) - n + i;
      valid = i < n && at >= 0;
      return at;
    } else {
      valid = true;
      if (!p.pos) return p.pos0 + i;
      const int64_t o = b * p.pos_sb + i * p.pos_ss;
      return p.pos64 ? static_cast<const int64_t*>(p.pos)[o]
                     : static_cast<int64_t>(static_cast<const int32_t*>(p.pos)[o]);
    }
  };

  // The loads of this thread's units.
  V xa[UPT], xb[UPT];
  int tok[UPT], head[UPT];
  Unit un[UPT];
#pragma unroll
  for (int j = 0; j < UPT; ++j) {
    const uint32_t i = tid + j * RT;
    tok[j] = -1;
    if (i >= static_cast<uint32_t>(n_units)) continue;
    const uint32_t th = div_by(i, p.div_units);
    const uint32_t t = div_by(th, p.div_heads);
    const int hh = static_cast<int>(th - t * p.head_chunk);
    const int u = static_cast<int>(i - th * p.units);
    if (hh >= nh) continue;
    const int h = h0 + hh;
    const bool rotated = APPEND ? h < p.H + p.Hk : h < p.rot_heads;
    un[j] = unit_of<VEC>(p, u, rotated);
    if (un[j].a >= p.D) continue;  // a copied head has fewer units than a rotated one at most
    const int64_t b = (t0 + t) / p.S, s = (t0 + t) - b * p.S;
    const T* src;
    if (!APPEND || h < p.H)
      src = static_cast<const T*>(p.x) + b * p.x_sb + h * p.x_sh + s * p.x_ss;
    else if (h < p.H + p.Hk)
      src = static_cast<const T*>(p.k) + b * p.k_sb + (h - p.H) * p.k_sh + s * p.k_ss;
    else
      src = static_cast<const T*>(p.v) + b * p.v_sb + (h - p.H - p.Hk) * p.v_sh + s * p.v_ss;
    tok[j] = static_cast<int>(t);
    head[j] = h;
    xa[j] = *reinterpret_cast<const V*>(src + un[j].a);
    if (un[j].b >= 0) xb[j] = *reinterpret_cast<const V*>(src + un[j].b);
  }

  // Meanwhile the tokens' angles, and (append) their slots.
  const int half = p.rot / 2;
  for (int i = tid; i < nt * half; i += RT) {
    const int t = i / half, f = i - t * half;
    const int64_t b = (t0 + t) / p.S, s = (t0 + t) - b * p.S;
    bool valid;
    const double turns = static_cast<double>(position(b, s, valid)) * (p.freqs[f] * INV_2PI);
    const float left = static_cast<float>(turns - rint(turns));
    float sn, c;
    sincospif(2.0f * left, &sn, &c);
    cs[t * p.rot + f] = c * p.amplitude;
    cs[t * p.rot + half + f] = (p.inverse ? -sn : sn) * p.amplitude;
  }
  if constexpr (APPEND) {
    for (int t = tid; t < nt; t += RT) {
      const int64_t b = (t0 + t) / p.S, s = (t0 + t) - b * p.S;
      bool valid;
      const int64_t at = position(b, s, valid);
      int64_t sk = -1, sv = -1;  // -1: no token; -2: a token without a page
      if (valid) {
        const int64_t lp = at / p.page;
        const int row = static_cast<int>(at - lp * p.page);
        const int pg = lp < p.table_width ? p.table[b * p.table_sb + lp] : -1;
        if (pg >= 0 && pg < p.n_pages) {
          sk = pg * p.kc_sp + row * p.kc_sr;
          sv = pg * p.vc_sp + row * p.vc_sr;
        } else {
          sk = -2;
          flag_error(p.sink, CFA_ERR_PAGE);
        }
      }
      slot_k[t] = sk;
      slot_v[t] = sv;
    }
  }
  __syncthreads();

#pragma unroll
  for (int j = 0; j < UPT; ++j) {
    if (tok[j] < 0) continue;
    const int t = tok[j], h = head[j];
    const Unit& u = un[j];
    float ya[VEC], yb[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      ya[e] = to_f(xa[j].v[e]);
      yb[e] = u.b >= 0 ? to_f(xb[j].v[e]) : 0.0f;
    }
    if (u.pair >= 0) {
      const float* c = cs + t * p.rot + u.pair;
      const float* s = c + half;
      if (p.interleaved) {
        // pairs (0, 1), (2, 3), .. of the unit's 2 VEC consecutive elements
        float z[2 * VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) z[e] = ya[e], z[VEC + e] = yb[e];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float lo = z[2 * e], hi = z[2 * e + 1];
          z[2 * e] = fmaf(lo, c[e], -hi * s[e]);
          z[2 * e + 1] = fmaf(hi, c[e], lo * s[e]);
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) ya[e] = z[e], yb[e] = z[VEC + e];
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float lo = ya[e], hi = yb[e];
          ya[e] = fmaf(lo, c[e], -hi * s[e]);
          yb[e] = fmaf(hi, c[e], lo * s[e]);
        }
      }
    }
    const int64_t b = (t0 + t) / p.S, s = (t0 + t) - b * p.S;
    if (!APPEND || h < p.H) {
      T* dst = static_cast<T*>(p.y) + b * p.y_sb + h * p.y_sh + s * p.y_ss;
      const bool live = !APPEND || slot_k[APPEND ? t : 0] != -1;  // a padded row's q comes back as zeros
      V oa, ob;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        oa.v[e] = from_f<T>(live ? ya[e] : 0.0f);
        ob.v[e] = from_f<T>(live ? yb[e] : 0.0f);
      }
      *reinterpret_cast<V*>(dst + u.a) = oa;
      if (u.b >= 0) *reinterpret_cast<V*>(dst + u.b) = ob;
    } else if constexpr (APPEND) {
      const bool is_k = h < p.H + p.Hk;
      if (slot_k[t] < 0) continue;
      C* dst = is_k ? static_cast<C*>(p.k_cache) + slot_k[t] + (h - p.H) * p.kc_sh
                    : static_cast<C*>(p.v_cache) + slot_v[t] + (h - p.H - p.Hk) * p.vc_sh;
      W oa, ob;
#pragma unroll
      for (int e = 0; e < VEC; ++e) oa.v[e] = from_f<C>(ya[e]), ob.v[e] = from_f<C>(yb[e]);
      *reinterpret_cast<W*>(dst + u.a) = oa;
      if (u.b >= 0) *reinterpret_cast<W*>(dst + u.b) = ob;
    }
  }
}

uint32_t magic(uint32_t d) {
  return d == 1 ? 0u : static_cast<uint32_t>(((uint64_t(1) << 32) + d - 1) / d);
}

template <typename T, typename C, int VEC, bool APPEND>
cudaError_t launch(RotaryArgs p, cudaStream_t stream) {
  const int heads = p.H + (APPEND ? 2 * p.Hk : 0);
  // Units of a rotated head and of a copied one (v, or rotary_qkv's v): the larger.
  const int tail = p.D - p.rot;
  p.units = p.rot / (2 * VEC) + (tail + 2 * VEC - 1) / (2 * VEC);
  const int copied = (p.D + 2 * VEC - 1) / (2 * VEC);
  if (copied > p.units) p.units = copied;
  p.head_chunk = heads;
  if (p.head_chunk > MAX_UNITS / p.units) p.head_chunk = MAX_UNITS / p.units;
  if (p.head_chunk < 1) return cudaErrorInvalidValue;  // units <= D / 2 + 1 <= 513
  // As many tokens as fill the block's units, their angles in at most 16 KB, but no fewer blocks
  // than four a SM where the tokens suffice.
  int64_t tokens = MAX_UNITS / (p.units * p.head_chunk);
  const int64_t by_smem = p.rot > 0 ? 4096 / p.rot : tokens;
  if (tokens > by_smem) tokens = by_smem;
  const int64_t spread = p.n_tokens / (4 * 148);
  if (tokens > spread) tokens = spread;
  if (tokens < 1) tokens = 1;
  p.tokens = static_cast<int>(tokens);
  p.div_units = magic(p.units);
  p.div_heads = magic(p.head_chunk);
  const int64_t gx = (p.n_tokens + tokens - 1) / tokens;
  const int64_t gy = (heads + p.head_chunk - 1) / p.head_chunk;
  if (gx > 0x7fffffff || gy > 65535) return cudaErrorInvalidConfiguration;
  const size_t smem = static_cast<size_t>(tokens) * p.rot * sizeof(float);
  return launch_pdl(rotary_kernel<T, C, VEC, APPEND>,
                    dim3(static_cast<unsigned>(gx), static_cast<unsigned>(gy)), dim3(RT), smem,
                    stream, p);
}

// The widest vector that the sizes, pointers and strides allow: 16 bytes of the input type, else
// (16-bit types) 4 bytes, else one element.
template <typename T, typename C, bool APPEND>
cudaError_t launch_vec(const RotaryArgs& p, cudaStream_t stream) {
  constexpr int E = sizeof(T);
  auto fits = [&](int vec) {
    if (p.rot % (2 * vec) != 0 || p.D % vec != 0) return false;
    auto ok = [&](const void* q, std::initializer_list<int64_t> st, int elt) {
      if (reinterpret_cast<uintptr_t>(q) % (vec * elt) != 0) return false;
      for (int64_t x : st)
        if (x % vec != 0) return false;
      return true;
    };
    if (p.H > 0 && (!ok(p.x, {p.x_sb, p.x_sh, p.x_ss}, E) || !ok(p.y, {p.y_sb, p.y_sh, p.y_ss}, E)))
      return false;
    if (!APPEND) return true;
    return ok(p.k, {p.k_sb, p.k_sh, p.k_ss}, E) && ok(p.v, {p.v_sb, p.v_sh, p.v_ss}, E) &&
           ok(p.k_cache, {p.kc_sp, p.kc_sr, p.kc_sh}, sizeof(C)) &&
           ok(p.v_cache, {p.vc_sp, p.vc_sr, p.vc_sh}, sizeof(C));
  };
  if (fits(16 / E)) return launch<T, C, 16 / E, APPEND>(p, stream);
  if constexpr (E == 2)
    if (fits(2)) return launch<T, C, 2, APPEND>(p, stream);
  return launch<T, C, 1, APPEND>(p, stream);
}

}  // namespace

cudaError_t launch_rotary(const RotaryArgs& p, int dtype, cudaStream_t stream) {
  if (dtype == CFA_F32) return launch_vec<float, float, false>(p, stream);
  if (dtype == CFA_F16) return launch_vec<__half, __half, false>(p, stream);
  return launch_vec<__nv_bfloat16, __nv_bfloat16, false>(p, stream);
}

cudaError_t launch_paged_append(const RotaryArgs& p, int dtype, int cache_dtype,
                                cudaStream_t stream) {
  if (dtype == CFA_F16) return launch_vec<__half, __half, true>(p, stream);
  if (dtype == CFA_BF16) return launch_vec<__nv_bfloat16, __nv_bfloat16, true>(p, stream);
  if (cache_dtype == CFA_F16) return launch_vec<float, __half, true>(p, stream);
  if (cache_dtype == CFA_BF16) return launch_vec<float, __nv_bfloat16, true>(p, stream);
  return launch_vec<float, float, true>(p, stream);
}

}  // namespace cfa
