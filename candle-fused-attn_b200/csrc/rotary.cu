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
// Bound by memory: every element is read and written once, at 3 flops: bf16 [4, 16, 8192, 128] 45 us, 6.0
// TB/s; fp32 [4, 32, 4096, 128] 80 us, 6.7 TB/s. A unit is two vectors of VEC
// elements (VEC pairs) of a head's row; a thread takes one unit of UPT heads of a token -- its index
// arithmetic, cosines and sines serve them all -- and issues their loads before the block computes its
// tokens' angles (one a thread and pass, shared by all heads through shared memory).
//
// The append runs the same units over the heads of q, k and v: rotated q into its output, rotated
// k and plain v into the token's slot of the cache, rounded once from fp32 (or the 16-bit input).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "cfa_common.cuh"
#include "cfa_ops.h"

namespace cfa {
namespace {

constexpr int RT = 256;            // most threads of a block
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

// Two adjacent vectors as one access of up to 32 bytes: a warp then moves whole sectors, where two
// accesses of every other 16 bytes would move each sector twice.
template <typename V>
__device__ __forceinline__ void load_pair(const void* p, V& a, V& b) {
  if constexpr (sizeof(V) == 16) {
    uint32_t* x = reinterpret_cast<uint32_t*>(&a);
    uint32_t* y = reinterpret_cast<uint32_t*>(&b);
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]), "=r"(y[0]), "=r"(y[1]), "=r"(y[2]),
                   "=r"(y[3])
                 : "l"(p));
  } else {
    struct alignas(2 * sizeof(V)) Two { V a, b; };
    const Two t = *static_cast<const Two*>(p);
    a = t.a, b = t.b;
  }
}
template <typename V>
__device__ __forceinline__ void store_pair(void* p, const V& a, const V& b) {
  if constexpr (sizeof(V) == 16) {
    const uint32_t* x = reinterpret_cast<const uint32_t*>(&a);
    const uint32_t* y = reinterpret_cast<const uint32_t*>(&b);
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(x[0]), "r"(x[1]),
                 "r"(x[2]), "r"(x[3]), "r"(y[0]), "r"(y[1]), "r"(y[2]), "r"(y[3])
                 : "memory");
  } else {
    struct alignas(2 * sizeof(V)) Two { V a, b; };
    *static_cast<Two*>(p) = Two{a, b};
  }
}

// The cache's type of an input element: itself, or an fp32 one rounded.
template <typename C, typename T>
__device__ __forceinline__ C cast(T x) {
  if constexpr (std::is_same_v<C, T>) return x;
  else return from_f<C>(to_f(x));
}

// VEC elements as one aligned access.
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Vec {
  T v[VEC];
};

// VEC floats of shared memory, 16 bytes at a time (a unit's pairs start at a multiple of VEC).
template <int VEC>
__device__ __forceinline__ void load_vec(float (&v)[VEC], const float* p) {
  if constexpr (VEC % 4 == 0) {
#pragma unroll
    for (int i = 0; i < VEC; i += 4) {
      const float4 x = ld4(p + i);
      v[i] = x.x, v[i + 1] = x.y, v[i + 2] = x.z, v[i + 3] = x.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = p[i];
  }
}

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

template <typename T, typename C, int VEC, int UPT, bool APPEND>
__global__ void __launch_bounds__(RT, UPT == 1 ? 4 : 3) rotary_kernel(const RotaryArgs p) {
  extern __shared__ __align__(16) float cs[];  // [tokens][cos: rot / 2, sin: rot / 2]
  __shared__ int64_t slot_k[APPEND ? RT : 1], slot_v[APPEND ? RT : 1];
  griddep_wait();
  griddep_launch_dependents();
  const int tid = threadIdx.x, threads = blockDim.x;
  const uint32_t t0 = blockIdx.x * p.tokens;  // (tokens fit 31 bits)
  const int nt = min(p.tokens, static_cast<int>(p.n_tokens - t0));
  const int heads = p.H + (APPEND ? 2 * p.Hk : 0), h0 = static_cast<int>(blockIdx.y) * p.head_step * UPT;
  const uint32_t n_items = nt * p.head_step * p.units;
  using V = Vec<T, VEC>;
  using W = Vec<C, VEC>;
  const int half = p.rot / 2;

  // A token's position, and whether it exists (append: a padded batch).
  auto position = [&](uint32_t b, uint32_t i, bool& valid) -> int64_t {
    if constexpr (APPEND) {
      int n = p.new_lengths ? p.new_lengths[b] : p.S;
      n = min(max(n, 0), p.S);
      const int64_t at = static_cast<int64_t>(p.lengths[b]) - n + i;
      valid = static_cast<int>(i) < n && at >= 0;
      return at;
    } else {
      valid = true;
      if (!p.pos) return p.pos0 + i;
      const int64_t o = b * p.pos_sb + i * p.pos_ss;  // (64-bit strides)
      return p.pos64 ? static_cast<const int64_t*>(p.pos)[o]
                     : static_cast<int64_t>(static_cast<const int32_t*>(p.pos)[o]);
    }
  };
  // The block's angles and (append) its tokens' slots.
  auto prepare = [&]() {
    for (int i = tid; i < nt * half; i += threads) {
      const int t = i / half, f = i - t * half;
      const uint32_t b = (t0 + t) / p.S, s = t0 + t - b * p.S;
      bool valid;
      const double turns = static_cast<double>(position(b, s, valid)) * (p.freqs[f] * INV_2PI);
      const float left = static_cast<float>(turns - rint(turns));
      float sn, c;
      sincospif(2.0f * left, &sn, &c);
      cs[t * p.rot + f] = c * p.amplitude;
      cs[t * p.rot + half + f] = (p.inverse ? -sn : sn) * p.amplitude;
    }
    if constexpr (APPEND) {
      for (int t = tid; t < nt; t += threads) {
        const uint32_t b = (t0 + t) / p.S, s = t0 + t - b * p.S;
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
  };

  // (One pass, unless a head alone has more units than the block threads.)
  for (uint32_t base = 0; base < n_items; base += threads) {
    // This thread's token, unit and heads h, h + head_step, ..: their loads first.
    const uint32_t item = base + tid;
    const uint32_t th = div_by(item, p.div_units);
    const uint32_t t = div_by(th, p.div_heads);
    const int hl = h0 + static_cast<int>(th - t * p.head_step);
    const int u = static_cast<int>(item - th * p.units);
    const uint32_t b = (t0 + t) / p.S, s = t0 + t - b * p.S;
    const Unit ur = unit_of<VEC>(p, u, true), uc = unit_of<VEC>(p, u, false);
    V xa[UPT], xb[UPT];
    // (a padded batch's rows behind its tokens are not read)
    const bool read = item < n_items &&
                      !(APPEND && p.new_lengths && static_cast<int>(s) >= p.new_lengths[b]);
#pragma unroll
    for (int j = 0; j < UPT; ++j) {
      const int h = hl + j * p.head_step;
      const Unit un = h < (APPEND ? p.H + p.Hk : p.rot_heads) ? ur : uc;
      if (!read || h >= heads || un.a >= p.D) continue;
      const T* src;
      if (!APPEND || h < p.H)
        src = static_cast<const T*>(p.x) + b * p.x_sb + h * p.x_sh + s * p.x_ss;
      else if (h < p.H + p.Hk)
        src = static_cast<const T*>(p.k) + b * p.k_sb + (h - p.H) * p.k_sh + s * p.k_ss;
      else
        src = static_cast<const T*>(p.v) + b * p.v_sb + (h - p.H - p.Hk) * p.v_sh + s * p.v_ss;
      if (p.pairs && un.b == un.a + VEC) {
        load_pair(src + un.a, xa[j], xb[j]);
      } else {
        xa[j] = *reinterpret_cast<const V*>(src + un.a);
        if (un.b >= 0) xb[j] = *reinterpret_cast<const V*>(src + un.b);
      }
    }
    if (base == 0) prepare();
    if (item >= n_items) continue;
    float c[VEC], sn[VEC];
    if (ur.pair >= 0) {
      load_vec<VEC>(c, cs + t * p.rot + ur.pair);
      load_vec<VEC>(sn, cs + t * p.rot + half + ur.pair);
    }
#pragma unroll
    for (int j = 0; j < UPT; ++j) {
      const int h = hl + j * p.head_step;
      const Unit un = h < (APPEND ? p.H + p.Hk : p.rot_heads) ? ur : uc;
      if (h >= heads || un.a >= p.D) continue;
      const bool to_cache = APPEND && h >= p.H;
      int64_t slot = 0;
      if constexpr (APPEND) {
        slot = h < p.H + p.Hk ? slot_k[t] : slot_v[t];
        if (to_cache && slot_k[t] < 0) continue;
        if (!to_cache && slot_k[t] == -1) {  // a padded row's q comes back as zeros
          xa[j] = V{};
          xb[j] = V{};
        }
      }
      if (un.pair >= 0) {
        float z[2 * VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) z[e] = to_f(xa[j].v[e]), z[VEC + e] = to_f(xb[j].v[e]);
        if (p.interleaved) {  // pairs (0, 1), (2, 3), .. of the unit's 2 VEC consecutive elements
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const float lo = z[2 * e], hi = z[2 * e + 1];
            z[2 * e] = fmaf(lo, c[e], -hi * sn[e]);
            z[2 * e + 1] = fmaf(hi, c[e], lo * sn[e]);
          }
        } else {
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const float lo = z[e], hi = z[VEC + e];
            z[e] = fmaf(lo, c[e], -hi * sn[e]);
            z[VEC + e] = fmaf(hi, c[e], lo * sn[e]);
          }
        }
        if (!to_cache) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) xa[j].v[e] = from_f<T>(z[e]), xb[j].v[e] = from_f<T>(z[VEC + e]);
        } else {
          W oa, ob;
#pragma unroll
          for (int e = 0; e < VEC; ++e) oa.v[e] = from_f<C>(z[e]), ob.v[e] = from_f<C>(z[VEC + e]);
          C* dst = static_cast<C*>(p.k_cache) + slot + (h - p.H) * p.kc_sh;
          if (p.pairs && un.b == un.a + VEC) {
            store_pair(dst + un.a, oa, ob);
          } else {
            *reinterpret_cast<W*>(dst + un.a) = oa;
            *reinterpret_cast<W*>(dst + un.b) = ob;
          }
          continue;
        }
      }
      if (!to_cache) {
        T* dst = static_cast<T*>(p.y) + b * p.y_sb + h * p.y_sh + s * p.y_ss;
        if (p.pairs && un.b == un.a + VEC) {
          store_pair(dst + un.a, xa[j], xb[j]);
        } else {
          *reinterpret_cast<V*>(dst + un.a) = xa[j];
          if (un.b >= 0) *reinterpret_cast<V*>(dst + un.b) = xb[j];
        }
      } else {  // copied dims of k, or v
        C* dst = h < p.H + p.Hk ? static_cast<C*>(p.k_cache) + slot + (h - p.H) * p.kc_sh
                                : static_cast<C*>(p.v_cache) + slot + (h - p.H - p.Hk) * p.vc_sh;
        W oa, ob;
#pragma unroll
        for (int e = 0; e < VEC; ++e) oa.v[e] = cast<C>(xa[j].v[e]);
#pragma unroll
        for (int e = 0; e < VEC; ++e) ob.v[e] = un.b >= 0 ? cast<C>(xb[j].v[e]) : C{};
        if (p.pairs && un.b == un.a + VEC) {
          store_pair(dst + un.a, oa, ob);
        } else {
          *reinterpret_cast<W*>(dst + un.a) = oa;
          if (un.b >= 0) *reinterpret_cast<W*>(dst + un.b) = ob;
        }
      }
    }
  }
}

uint32_t magic(uint32_t d) {
  return d == 1 ? 0u : static_cast<uint32_t>(((uint64_t(1) << 32) + d - 1) / d);
}

template <typename T, typename C, int VEC, int UPT, bool APPEND>
cudaError_t launch_upt(RotaryArgs p, int heads, cudaStream_t stream) {
  // A thread takes the unit of UPT heads head_step apart; a block as many tokens as its threads hold,
  // their angles in at most 16 KB, but no fewer blocks than four a SM where the tokens suffice.
  p.head_step = (heads + UPT - 1) / UPT;
  const int fit = RT / p.units > 0 ? RT / p.units : 1;
  if (p.head_step > fit) p.head_step = fit;
  int64_t tokens = RT / (p.units * p.head_step);
  const int64_t by_smem = p.rot > 0 ? 4096 / p.rot : tokens;
  if (tokens > by_smem) tokens = by_smem;
  const int64_t spread = p.n_tokens / (4 * 148);
  if (tokens > spread) tokens = spread;
  if (tokens < 1) tokens = 1;
  p.tokens = static_cast<int>(tokens);
  const int64_t items = tokens * p.units * p.head_step;
  const unsigned threads = items >= RT ? RT : static_cast<unsigned>((items + 31) / 32 * 32);
  p.div_units = magic(p.units);
  p.div_heads = magic(p.head_step);
  const int64_t gx = (p.n_tokens + tokens - 1) / tokens;
  const int64_t gy = (heads + p.head_step * UPT - 1) / (p.head_step * UPT);
  if (gx > 0x7fffffff || gy > 65535) return cudaErrorInvalidConfiguration;
  const size_t smem = static_cast<size_t>(tokens) * p.rot * sizeof(float);
  return launch_pdl(rotary_kernel<T, C, VEC, UPT, APPEND>,
                    dim3(static_cast<unsigned>(gx), static_cast<unsigned>(gy)), dim3(threads), smem,
                    stream, p);
}

// Four units a thread where they still fill the GPU (four blocks of 256 threads a SM): a thread then
// has 128 bytes in flight and shares its index arithmetic; else one, for the shortest path of a small
// call. On one B200, with four and with one: bf16 [4, 16, 8192, 128] 45 and 64 us, the append of 8
// ragged prompts of up to 1500 tokens (16 heads of 64, fp32 to bf16) 42 and 83 us; fp32 [64, 6, 1, 64] 2.9
// and 2.1 us, the append of 64 tokens (32 heads over 8 of 128) 4.9 and 3.1 us.
template <typename T, typename C, int VEC, bool APPEND>
cudaError_t launch(RotaryArgs p, cudaStream_t stream) {
  const int heads = p.H + (APPEND ? 2 * p.Hk : 0);
  // Units of a rotated head and of a copied one (v, or rotary_qkv's v): the larger.
  const int tail = p.D - p.rot;
  p.units = p.rot / (2 * VEC) + (tail + 2 * VEC - 1) / (2 * VEC);
  const int copied = (p.D + 2 * VEC - 1) / (2 * VEC);
  if (copied > p.units) p.units = copied;
  const int64_t all = p.n_tokens * heads * p.units;
  return all >= int64_t(4) * 148 * 4 * RT ? launch_upt<T, C, VEC, 4, APPEND>(p, heads, stream)
                                          : launch_upt<T, C, VEC, 1, APPEND>(p, heads, stream);
}

// The widest vector that the sizes, pointers and strides allow: 16 bytes of the input type, else
// (16-bit types) 4 bytes, else one element.
template <typename T, typename C, bool APPEND>
cudaError_t launch_vec(const RotaryArgs& args, cudaStream_t stream) {
  RotaryArgs p = args;
  constexpr int E = sizeof(T);
  auto aligned = [&](int vec) {
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
  auto fits = [&](int vec) {
    if (p.rot % (2 * vec) != 0 || p.D % vec != 0 || !aligned(vec)) return false;
    p.pairs = aligned(2 * vec);
    return true;
  };
  if (fits(16 / E)) return launch<T, C, 16 / E, APPEND>(p, stream);
  if constexpr (E == 2)
    if (fits(2)) return launch<T, C, 2, APPEND>(p, stream);
  p.pairs = 0;
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
