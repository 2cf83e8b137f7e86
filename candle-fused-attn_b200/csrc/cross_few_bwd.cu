// SPDX-License-Identifier: MIT OR Apache-2.0
//
// Cross attention's backward for few query rows (up to 32 a key head, of its whole group): key blocks of
// KB keys, a block each, four warps that run on their own, each over 16 keys at a time:
//   S^T = K Q^T, P^T = e^(S^T scale - L), dP^T = V dO^T, dS^T = P^T o (dP^T - D);
//   dV = P^T dO and dK = scale dS^T Q, whole, to memory; dQ += dS K in registers,
// the block's dQ partial summed over its warps in order, the key blocks' by cross_join_kernel. Products by
// mma.m16n8k8 on two-part tf32 operands (tf32.cuh; hi hi + hi lo + lo hi), the keys as the 16 rows, the
// queries as columns; a score's products and sums in the order of the forward that made L (split_attn.cu).
// P^T's and dS^T's fragments are those of the scores, dS's rows go through shared memory.
//
// K, V are read and dK, dV written once, at 20 rows D flops a key against 16 D bytes: 4.3 TB/s at 8 rows
// ([32, 8, 8, 64] over 1000 keys, 61 us), 3.3 at 16, 2.1 at 30, where the products' issue bounds it. The
// tcgen05 pair, whose tiles are 64 queries, spends a block's first loads, splits and last stores on 128 keys:
// [34, 24 over 8, 10, 64] over 1000 to 2000 keys 219 us here, 332 there; [32, 8, 32, 64] over 500 to 1000 108
// and 161.
#include "cfa_common.cuh"
#include "tf32.cuh"

namespace cfa {
namespace {

constexpr int WARPS = 4, NT = 32 * WARPS, TK = 16;
constexpr float LOG2E = 1.4426950408889634f;
constexpr int LS = TK + 4;  // row stride of dS

// Piece c of row r of an fp32 tile is piece c ^ swizzle(r): conflict-free 16-byte reads of two rows' four
// pieces and of every other row's two.
__device__ __forceinline__ int swizzle(int r) { return (4 * (r & 1)) ^ (2 * ((r >> 1) & 3)); }

template <int D>
constexpr int key_block() {
  return D == 128 ? 64 : 128;
}
template <int D, int NQ>
struct Few {
  static constexpr int KB = key_block<D>(), TILES = KB / (TK * WARPS);  // tiles of a warp, all in flight at once
  static constexpr int R = 8 * NQ;
  static constexpr int WARP_KV = TILES * 2 * TK * D;  // floats: its keys and values
  static constexpr int OFF_Q = WARPS * WARP_KV, OFF_DO = OFF_Q + R * D, OFF_DS = OFF_DO + R * D;
  static constexpr int OFF_L = OFF_DS + WARPS * R * LS, FLOATS = OFF_L + 2 * R;
  static_assert(WARPS * R * D <= OFF_Q, "the warps' dQ fit where their keys were");
};

template <int D, int NQ>
__global__ void __launch_bounds__(NT, 2) cross_few_bwd_kernel(const BwdArgs a) {
  using F = Few<D, NQ>;
  constexpr int KB = F::KB, TILES = F::TILES, R = F::R, C = D / 4, J = D / 16, JV = D / 32;
  constexpr int MQ = (NQ + 1) / 2;  // 16-row tiles of the queries
  extern __shared__ float4 smem4[];
  float* sm = reinterpret_cast<float*>(smem4);
  float* Qs = sm + F::OFF_Q;
  float* dOs = sm + F::OFF_DO;
  float* Ls = sm + F::OFF_L;  // [R]: L; [R]: D
  griddep_wait();  // the lengths, D: the previous kernels' writes
  griddep_launch_dependents();
  const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t4 = lane & 3;
  const int kb = static_cast<int>(blockIdx.x % a.n_kblocks);
  const int bh = static_cast<int>(blockIdx.x / a.n_kblocks);
  const int b = bh / a.Hk, hk = bh % a.Hk;
  const int group = a.H / a.Hk, rows = group * a.S, k0 = kb * KB;
  const int SK = cross_keys(a, b);
  float* dkv = a.dkv + (static_cast<int64_t>(b) * a.Sk + k0) * 2 * a.Hk * D + hk * D;
  const int64_t kv_row = 2 * static_cast<int64_t>(a.Hk) * D, dv_at = static_cast<int64_t>(a.Hk) * D;
  if (k0 >= SK) {  // no key of this block is attended: zeros, and no part in dQ's sums
    const int krows = min(KB, a.Sk - k0);
    for (int f = tid; f < 2 * krows * C; f += NT) {
      const int which = f / (krows * C), r = (f / C) % krows;
      reinterpret_cast<float4*>(dkv + r * kv_row + which * dv_at)[f % C] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    return;
  }
  auto query_of = [&](int r, int& head, int& i) {
    const int x = group == 1 ? 0 : r / a.S;
    head = hk * group + x;
    i = r - x * a.S;
  };
  // The warp's keys and values (rows past the length: zeros), tile by tile; the block's queries before them.
  float* kv = sm + w * F::WARP_KV;
  {
#pragma unroll
    for (int f = tid; f < R * C; f += NT) {
      const int r = f / C, c = f % C;
      const bool ok = r < rows;
      int head, i;
      query_of(ok ? r : 0, head, i);
      cp_async16(Qs + r * D + 4 * (c ^ swizzle(r)), a.q + b * a.q_sb + head * a.q_sh + i * a.q_ss + 4 * c,
                 ok ? 16 : 0);
      cp_async16(dOs + r * D + 4 * (c ^ swizzle(r)),
                 a.d_o + b * a.do_sb + head * a.do_sh + i * a.do_ss + 4 * c, ok ? 16 : 0);
    }
    if (tid < 2 * R) {
      const int r = tid < R ? tid : tid - R;
      const bool ok = r < rows;
      int head, i;
      query_of(ok ? r : 0, head, i);
      cp_async4(Ls + tid, (tid < R ? a.lse : a.dsum) + (static_cast<int64_t>(b) * a.H + head) * a.S + i, ok ? 4 : 0);
    }
    const float* kp = a.k + b * a.k_sb + hk * a.k_sh;
    const float* vp = a.v + b * a.v_sb + hk * a.v_sh;
#pragma unroll
    for (int n = 0; n < TILES; ++n) {
#pragma unroll
      for (int f = lane; f < TK * C; f += 32) {
        const int r = f / C, c = f % C, key = k0 + (WARPS * n + w) * TK + r;
        const bool ok = key < SK;
        float* dst = kv + n * 2 * TK * D + r * D + 4 * (c ^ swizzle(r));
        cp_async16(dst, kp + (ok ? key : 0) * a.k_ss + 4 * c, ok ? 16 : 0);
        cp_async16(dst + TK * D, vp + (ok ? key : 0) * a.v_ss + 4 * c, ok ? 16 : 0);
      }
      cp_async_commit();
    }
  }
  // A tile's 16 bytes as this lane reads them: dims 16 j + 4 t4 .. of row r8 + g; dims 32 j + 4 g .. of
  // rows 8 i + 2 t4 + y.
  const int by_row = g * D + 4 * (t4 ^ swizzle(g));
  auto at_row = [&](const float* x, int r8, int j) {
    return ld4(x + r8 * D + (by_row ^ (16 * (j & 1))) + 32 * (j >> 1));
  };
  const int by_col0 = 2 * t4 * D + 4 * (g ^ swizzle(2 * t4));
  const int by_col1 = (2 * t4 + 1) * D + 4 * (g ^ swizzle(2 * t4 + 1));
  auto at_col = [&](const float* x, int i, int y, int j) {
    return ld4(x + 8 * i * D + (y ? by_col1 : by_col0) + 32 * j);
  };

  float dq[MQ][JV][4][4];  // rows 16 m + g, + 8: dims 32 j + 8 t4 + e, + 4
#pragma unroll
  for (int m = 0; m < MQ; ++m)
#pragma unroll
    for (int j = 0; j < JV; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int x = 0; x < 4; ++x) dq[m][j][e][x] = 0.0f;
  float* ds_rows = sm + F::OFF_DS + w * R * LS;

  for (int n = 0; n < TILES; ++n) {
    // (the first pass waits for all but the tiles behind it; its barrier puts the queries in place)
    if (TILES == 2 && n == 0) asm volatile("cp.async.wait_group 1;\n" ::: "memory");
    else cp_async_wait_all();
    if (n == 0) __syncthreads();
    else __syncwarp();
    const int key0 = k0 + (WARPS * n + w) * TK;
    if (key0 >= a.Sk) break;  // (later tiles of the warp lie behind it)
    const float* K = kv + n * 2 * TK * D;
    const float* V = K + TK * D;
    // Scores' layout: keys g, g + 8 (x >> 1); queries 8 q + 2 t4, + 1 (x & 1).
    auto scores = [&](const float* A, const float* B, float (&s)[NQ][4]) {
      clear(s);
#pragma unroll
      for (int j = 0; j < J; ++j) {
        uint32_t ah[2][4], al[2][4];
        split_rows(at_row(A, 0, j), at_row(A, 8, j), ah, al);
        if constexpr (NQ == 1) {  // (the forward has the parts of up to 8 rows in sums of their own)
          uint32_t h[4], l[4];
          split_tf32(at_row(B, 0, j), h, l);
          float c[3][4];
          clear(c);
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            mma_tf32(c[0], al[y], h[2 * y], h[2 * y + 1]);
            mma_tf32(c[1], ah[y], l[2 * y], l[2 * y + 1]);
            mma_tf32(c[2], ah[y], h[2 * y], h[2 * y + 1]);
          }
#pragma unroll
          for (int x = 0; x < 4; ++x) s[0][x] += (c[1][x] + c[0][x]) + c[2][x];
        } else {
          float c[NQ][4];
          clear(c);
#pragma unroll
          for (int q = 0; q < NQ; ++q) products(c[q], ah, al, at_row(B, 8 * q, j));
          add(s, c);
        }
      }
    };
    // dst[keys][dims] = X^T Y for scores-shaped X (keys x queries) and Y [queries][dims], times f.
    auto rows_out = [&](const float (&x)[NQ][4], const float* Y, float* dst, float f) {
      uint32_t xh[NQ][4], xl[NQ][4];
#pragma unroll
      for (int q = 0; q < NQ; ++q) split_tf32(make_float4(x[q][0], x[q][2], x[q][1], x[q][3]), xh[q], xl[q]);
#pragma unroll
      for (int j = 0; j < JV; ++j) {
        float c[4][4], small[4][4];
        clear(c);
        clear(small);
#pragma unroll
        for (int q = 0; q < NQ; ++q) products(small, c, xh[q], xl[q], at_col(Y, q, 0, j), at_col(Y, q, 1, j));
        add(c, small);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (key0 + g + 8 * h >= a.Sk) continue;  // (rows past the length hold zeros)
          float* at = dst + (key0 - k0 + g + 8 * h) * kv_row + 32 * j + 8 * t4;
#pragma unroll
          for (int y = 0; y < 2; ++y)
            *reinterpret_cast<float4*>(at + 4 * y) =
                make_float4(c[0][2 * h + y] * f, c[1][2 * h + y] * f, c[2][2 * h + y] * f, c[3][2 * h + y] * f);
        }
      }
    };
    float p[NQ][4], ds[NQ][4];
    scores(K, Qs, p);
    scores(V, dOs, ds);
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      const float2 L = *reinterpret_cast<const float2*>(Ls + 8 * q + 2 * t4);
      const float2 d = *reinterpret_cast<const float2*>(Ls + R + 8 * q + 2 * t4);
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const bool live = key0 + g + 8 * (x >> 1) < SK && 8 * q + 2 * t4 + (x & 1) < rows;
        p[q][x] = live ? ex2(fmaf(p[q][x], a.scale, -(x & 1 ? L.y : L.x)) * LOG2E) : 0.0f;
        ds[q][x] = p[q][x] * (ds[q][x] - (x & 1 ? d.y : d.x));
        ds_rows[(8 * q + 2 * t4 + (x & 1)) * LS + g + 8 * (x >> 1)] = ds[q][x];
      }
    }
    rows_out(p, dOs, dkv + dv_at, 1.0f);
    rows_out(ds, Qs, dkv, grad_scale(a, SK));
    __syncwarp();  // dS's rows in place
#pragma unroll
    for (int m = 0; m < MQ; ++m) {
      uint32_t xh[2][4], xl[2][4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float* at = ds_rows + (16 * m + g) * LS + 8 * i + 2 * t4;
        const float2 x = *reinterpret_cast<const float2*>(at);
        float2 y = make_float2(0.f, 0.f);  // (8 rows: the product's other 8 are none)
        if constexpr (NQ > 1) y = *reinterpret_cast<const float2*>(at + 8 * LS);
        split_tf32(make_float4(x.x, y.x, x.y, y.y), xh[i], xl[i]);
      }
#pragma unroll
      for (int j = 0; j < JV; ++j) {
        float c[4][4], small[4][4];
        clear(c);
        clear(small);
#pragma unroll
        for (int i = 0; i < 2; ++i) products(small, c, xh[i], xl[i], at_col(K, i, 0, j), at_col(K, i, 1, j));
        add(c, small);
        add(dq[m][j], c);
      }
    }
    __syncwarp();  // dS's rows are read
  }
  cp_async_wait_all();  // (a warp that left at its first tile has the second one's copies in flight)
  __syncthreads();  // every warp's keys are read: their dQ take the place
#pragma unroll
  for (int m = 0; m < MQ; ++m)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (16 * m + 8 * h >= R) continue;
#pragma unroll
      for (int j = 0; j < JV; ++j)
#pragma unroll
        for (int y = 0; y < 2; ++y)
          *reinterpret_cast<float4*>(sm + (w * R + 16 * m + 8 * h + g) * D + 32 * j + 8 * t4 + 4 * y) =
              make_float4(dq[m][j][0][2 * h + y], dq[m][j][1][2 * h + y], dq[m][j][2][2 * h + y],
                          dq[m][j][3][2 * h + y]);
    }
  __syncthreads();
  for (int f = tid; f < min(R, rows) * C; f += NT) {
    const int r = f / C, c = f % C;
    float4 v = ld4(sm + r * D + 4 * c);
#pragma unroll
    for (int x = 1; x < WARPS; ++x) {
      const float4 y = ld4(sm + (x * R + r) * D + 4 * c);
      v = make_float4(v.x + y.x, v.y + y.y, v.z + y.z, v.w + y.w);
    }
    int head, i;
    query_of(r, head, i);
    reinterpret_cast<float4*>(
        a.dq_part + (((static_cast<int64_t>(b) * a.H + head) * a.n_kblocks + kb) * a.S + i) * D)[c] = v;
  }
}

template <int D, int NQ>
cudaError_t launch_nq(const BwdArgs& a, cudaStream_t stream) {
  const dim3 grid(static_cast<unsigned>(static_cast<int64_t>(a.n_kblocks) * a.B * a.Hk));
  const cudaError_t e = launch_pdl(cross_few_bwd_kernel<D, NQ>, grid, dim3(NT),
                                   static_cast<size_t>(Few<D, NQ>::FLOATS * 4), stream, a);
  return e == cudaSuccess ? launch_cross_join(a, D, key_block<D>(), stream) : e;
}
template <int D>
cudaError_t launch_d(const BwdArgs& args, cudaStream_t stream) {
  BwdArgs a = args;
  a.n_kblocks = (a.Sk + key_block<D>() - 1) / key_block<D>();
  const int rows = a.H / a.Hk * a.S;
  return rows <= 8 ? launch_nq<D, 1>(a, stream) : rows <= 16 ? launch_nq<D, 2>(a, stream) : launch_nq<D, 4>(a, stream);
}
template <int D>
cudaError_t set_attrs() {
  auto set = [](const void* fn, int floats) {
    return cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, floats * 4);
  };
  cudaError_t e = set(reinterpret_cast<const void*>(cross_few_bwd_kernel<D, 1>), Few<D, 1>::FLOATS);
  if (e == cudaSuccess) e = set(reinterpret_cast<const void*>(cross_few_bwd_kernel<D, 2>), Few<D, 2>::FLOATS);
  return e == cudaSuccess ? set(reinterpret_cast<const void*>(cross_few_bwd_kernel<D, 4>), Few<D, 4>::FLOATS) : e;
}

}  // namespace

cudaError_t setup_cross_few_bwd_attributes() {
  cudaError_t e = set_attrs<32>();
  if (e == cudaSuccess) e = set_attrs<64>();
  return e == cudaSuccess ? set_attrs<128>() : e;
}

cudaError_t launch_cross_few_bwd(const BwdArgs& a, int head_dim, cudaStream_t stream) {
  if (head_dim == 32) return launch_d<32>(a, stream);
  if (head_dim == 64) return launch_d<64>(a, stream);
  return launch_d<128>(a, stream);
}

}  // namespace cfa
