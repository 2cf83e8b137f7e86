// SPDX-License-Identifier: MIT OR Apache-2.0
//
// Cross attention at head dim 128: the forward O = softmax(Q K^T * scale) V and L, the log-sum-exp of its
// rows, over a.Sk key rows, of which batch element b attends the first cross_keys(a, b); and the backward
// (below). A block's query rows are those of a key head's whole group (row r: head r / S of it, query r %
// S). Forward: 64 of them, 16 a warp, over key tiles of 64, online softmax.
//
// Products by mma.m16n8k8 on tf32 operands in two parts (tf32.cuh): hi hi + hi lo + lo hi, what is left out
// below 2^-22 of the products' magnitudes, in short sums (32 dims, keys or queries) that are added in fp32.
// Dims and keys are numbered within a product so that a lane reads Q, K and V 16 bytes at a time (k = t, t + 4
// are adjacent dims, or keys 2 t, 2 t + 1) and P's fragment is S's. (Head dims 64 and 32 run on tcgen05, whose
// three-part operands do not fit at 128.)
//
// Bound by the issue of splits and products, two warps a scheduler: at the rate of these products (a third
// of tf32's: 96 TFLOP/s) the tensor core is busy for 0.5 to 0.6 of the time. [16, 8, 512 x 512, 128]:
// forward 303 us (57 TFLOP/s), backward 880 us (49); by fp32 FMAs, as hd_ffma.cu has the fused attention's,
// 442 and 1128 us. [2, 8, 2048 x 4096, 128]: 1.32 and 3.35 ms, for 1.70 and 4.33.
#include "cfa_common.cuh"
#include "tf32.cuh"

namespace cfa {
namespace {

constexpr int D = 128, C = D / 4;        // head dim, its 16-byte pieces
constexpr int NT = 128, BM = 64, BN = 64;
constexpr int LQ = D + 16, LV = D + 4;  // row strides: 16-byte reads of two rows, of every other row
constexpr int SMEM = (BM * LQ + BN * LQ + BN * LV) * 4;
constexpr float LOG2E = 1.4426950408889634f;

__global__ void __launch_bounds__(NT, 2) cross_hd_fwd_kernel(const FwdArgs a) {
  extern __shared__ float4 smem4[];
  float* Qs = reinterpret_cast<float*>(smem4);
  float* Ks = Qs + BM * LQ;
  float* Vs = Ks + BN * LQ;
  griddep_wait();  // q, k, v may come from the previous kernel on the stream
  griddep_launch_dependents();
  const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t4 = lane & 3;
  const int qt = static_cast<int>(blockIdx.x % a.n_qtiles);
  const int bh = static_cast<int>(blockIdx.x / a.n_qtiles);
  const int b = bh / a.Hk, hk = bh % a.Hk;
  const int group = a.H / a.Hk, rows = group * a.S, q0 = qt * BM;
  auto query_of = [&](int r, int& head, int& i) {
    const int x = group == 1 ? 0 : r / a.S;
    head = hk * group + x;
    i = r - x * a.S;
  };
  const int SK = cross_keys(a, b);
  if (SK == 0) {  // no key: O = 0, L = -inf
    for (int f = tid; f < min(BM, rows - q0) * (D / 4); f += NT) {
      int head, i;
      query_of(q0 + f / (D / 4), head, i);
      reinterpret_cast<float4*>(a.o + ((static_cast<int64_t>(b) * a.S + i) * a.H + head) * D)[f % (D / 4)] =
          make_float4(0.f, 0.f, 0.f, 0.f);
      if (f % (D / 4) == 0) a.lse[(static_cast<int64_t>(b) * a.H + head) * a.S + i] = -INFINITY;
    }
    return;
  }
  const float* kp = a.k + b * a.k_sb + hk * a.k_sh;
  const float* vp = a.v + b * a.v_sb + hk * a.v_sh;
#pragma unroll
  for (int f = tid; f < BM * C; f += NT) {
    const int r = f / C, c = f % C;
    const bool ok = q0 + r < rows;
    int head, i;
    query_of(ok ? q0 + r : q0, head, i);
    cp_async16(Qs + r * LQ + 4 * c, a.q + b * a.q_sb + head * a.q_sh + i * a.q_ss + 4 * c, ok ? 16 : 0);
  }
  auto load_keys = [&](float* dst, int stride, const float* src, int64_t ss, int k0) {
#pragma unroll
    for (int f = tid; f < BN * C; f += NT) {
      const int r = f / C, c = f % C;
      const bool ok = k0 + r < SK;
      cp_async16(dst + r * stride + 4 * c, src + (ok ? k0 + r : 0) * ss + 4 * c, ok ? 16 : 0);
    }
    cp_async_commit();
  };
  load_keys(Ks, LQ, kp, a.k_ss, 0);

  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
  float acc[D / 32][4][4];  // rows g, g + 8: dims 32 j + 8 t4 + e, + 4
#pragma unroll
  for (int j = 0; j < D / 32; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int x = 0; x < 4; ++x) acc[j][e][x] = 0.0f;
  const float* qa = Qs + (16 * w + g) * LQ + 4 * t4;
  const float* ka = Ks + g * LQ + 4 * t4;
  const float* va = Vs + 2 * t4 * LV + 4 * g;

  for (int k0 = 0; k0 < SK; k0 += BN) {
    cp_async_wait_all();
    __syncthreads();  // K in place; the last tile's V is read
    load_keys(Vs, LV, vp, a.v_ss, k0);
    float sc[BN / 8][4];  // rows g, g + 8; keys 8 i + 2 t4, + 1
    clear(sc);
#pragma unroll 1
    for (int j = 0; j < D / 16; j += 2) {
      float c[BN / 8][4];
      clear(c);
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        uint32_t ah[2][4], al[2][4];
        split_rows(ld4(qa + 16 * (j + y)), ld4(qa + 8 * LQ + 16 * (j + y)), ah, al);
#pragma unroll
        for (int i = 0; i < BN / 8; ++i) products(c[i], ah, al, ld4(ka + 8 * i * LQ + 16 * (j + y)));
      }
      add(sc, c);
    }
    const bool edge = k0 + BN > SK;
    uint32_t ph[BN / 8][4], pl[BN / 8][4];  // P as A fragments: k = t4 is key 8 i + 2 t4, t4 + 4 the next
    float alpha[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float s[BN / 8][2], top = m[h];
#pragma unroll
      for (int i = 0; i < BN / 8; ++i)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          s[i][x] = sc[i][2 * h + x] * a.scale;
          if (edge && k0 + 8 * i + 2 * t4 + x >= SK) s[i][x] = -INFINITY;
          top = fmaxf(top, s[i][x]);
        }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const float mu = top == -INFINITY ? 0.0f : top;
      alpha[h] = ex2((m[h] - mu) * LOG2E);
      m[h] = top;
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < BN / 8; ++i) {
        const float p0 = ex2((s[i][0] - mu) * LOG2E), p1 = ex2((s[i][1] - mu) * LOG2E);
        sum += p0 + p1;
        uint32_t hi[4], lo[4];
        split_tf32(make_float4(p0, p1, 0.f, 0.f), hi, lo);
        ph[i][h] = hi[0], ph[i][2 + h] = hi[1];
        pl[i][h] = lo[0], pl[i][2 + h] = lo[1];
      }
      l[h] = fmaf(l[h], alpha[h], sum);
    }
    cp_async_wait_all();
    __syncthreads();  // V in place; K is read
    if (k0 + BN < SK) load_keys(Ks, LQ, kp, a.k_ss, k0 + BN);
#pragma unroll
    for (int j = 0; j < D / 32; ++j) {
      float small[4][4], large[4][4];
      clear(small);
      clear(large);
#pragma unroll
      for (int i = 0; i < BN / 8; ++i) {
        const float* at = va + 8 * i * LV + 32 * j;
        products(small, large, ph[i], pl[i], ld4(at), ld4(at + LV));
        if (i == BN / 16 - 1) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int x = 0; x < 4; ++x) acc[j][e][x] = fmaf(acc[j][e][x], alpha[x >> 1], large[e][x]);
          clear(large);
        }
      }
      add(large, small);
      add(acc[j], large);
    }
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float sum = l[h] + __shfl_xor_sync(0xffffffffu, l[h], 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
    const int r = q0 + 16 * w + g + 8 * h;
    if (r >= rows) continue;
    int head, i;
    query_of(r, head, i);
    float* dst = a.o + ((static_cast<int64_t>(b) * a.S + i) * a.H + head) * D + 8 * t4;
    const float rl = 1.0f / sum;
#pragma unroll
    for (int j = 0; j < D / 32; ++j)
#pragma unroll
      for (int x = 0; x < 2; ++x)
        *reinterpret_cast<float4*>(dst + 32 * j + 4 * x) =
            make_float4(acc[j][0][2 * h + x] * rl, acc[j][1][2 * h + x] * rl, acc[j][2][2 * h + x] * rl,
                        acc[j][3][2 * h + x] * rl);
    if (t4 == 0) a.lse[(static_cast<int64_t>(b) * a.H + head) * a.S + i] = m[h] + logf(sum);
  }
}

// The backward, one pass over the query rows of a key head's group: key blocks of 64, query tiles of 64, 8
// warps. Per tile:
//   1. warps 0-3 S = Q K^T (the forward's order) and P = e^(S scale - L), warps 4-7 dP = dO V^T and, with P
//      out of shared memory, dS = P o (dP - D); both to shared memory, [query][key];
//   2. warps 0-3 dV += P^T dO, warps 4-7 dK += dS^T Q, 16 keys a warp, added in fp32;
//   3. all: the tile's dQ partial dS K, 16 queries and half the dims a warp.
// Key blocks, parts, dQ's order and the zeros of unattended keys are cross_bwd_tc.cu's, the dQ partials
// always cross_join_kernel's. The operands' tiles
// are read both by rows (products over the dims) and by columns: piece c of row r is piece c ^ swizzle(r),
// conflict-free for 16-byte reads of two rows' four pieces and of every other row's two.
constexpr int BT = 256, KB = 64, LP = KB + 4;
constexpr int BWD_SMEM = (4 * KB * D + 2 * 64 * LP + 128) * 4 + 16;
__device__ __forceinline__ int swizzle(int r) { return (4 * (r & 1)) ^ (2 * ((r >> 1) & 3)); }

__global__ void __launch_bounds__(BT, 1) cross_hd_bwd_kernel(const BwdArgs a) {
  extern __shared__ float4 smem4[];
  float* Ks = reinterpret_cast<float*>(smem4);
  float* Vs = Ks + KB * D;
  float* Qs = Vs + KB * D;
  float* dOs = Qs + 64 * D;
  float* Ps = dOs + 64 * D;  // [64][LP] query-major
  float* dSs = Ps + 64 * LP;
  float* Lt = dSs + 64 * LP;
  float* Dt = Lt + 64;
  int* s_int = reinterpret_cast<int*>(Dt + 64);

  griddep_launch_dependents();
  const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t4 = lane & 3;
  const int grp = w >> 2, wg = w & 3;  // grp 0: S, P, dV; grp 1: dP, dS, dK
  const int S = a.S;

  griddep_wait();  // the lengths, D, the cleared ticket and counters: the previous kernels' writes
  const bool no_wait = a.dq_part != nullptr;
  int ticket;
  if (no_wait) {
    ticket = static_cast<int>(blockIdx.x);
  } else {
    if (tid == 0) s_int[0] = atomicAdd(a.ticket, 1);
    __syncthreads();
    ticket = s_int[0];
  }
  const int BH = a.B * a.Hk;
  const int nparts = a.n_parts, part = ticket % nparts, unit = ticket / nparts;
  const int kb = no_wait ? unit % a.n_kblocks : unit / BH;
  const int bh = no_wait ? unit / a.n_kblocks : unit % BH;
  const int b = bh / a.Hk, hk = bh % a.Hk;
  const int k0 = kb * KB;
  const int group = a.H / a.Hk, rows = group * S, h0 = hk * group;
  auto query_of = [&](int r, int& head, int& i) {
    const int x = group == 1 ? 0 : r / S;
    head = h0 + x;
    i = r - x * S;
  };
  const int nqt = (rows + 63) / 64;
  const int SK = cross_keys(a, b);
  const int nkb = (SK + KB - 1) / KB;  // key blocks of this (batch, head) that take part
  const float dscale = grad_scale(a, SK);
  float* dkv = a.dkv + static_cast<int64_t>(part) * a.part_stride;  // (parts: in the workspace)
  if (kb >= nkb) {  // no key of this block is attended: zeros, and no part in dQ's sums
    const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
    const int krows = min(KB, a.Sk - k0);
    for (int f = tid; f < 2 * krows * C; f += BT) {
      const int which = f / (krows * C), r = (f / C) % krows;
      reinterpret_cast<float4*>(
          dkv + (((static_cast<int64_t>(b) * a.Sk + k0 + r) * 2 + which) * a.Hk + hk) * D)[f % C] = zero;
    }
    if (kb == 0 && part == 0)  // no key at all: dQ = 0
      for (int64_t f = tid; f < static_cast<int64_t>(rows) * C; f += BT)
        reinterpret_cast<float4*>(a.dq + ((static_cast<int64_t>(b) * S + f / (group * C)) * a.H + h0) *
                                             D)[f % (group * C)] = zero;
    return;
  }
  int* turn = a.turn + static_cast<int64_t>(bh) * nqt;       // turn chain: counters per tile

  {
    const float* kp = a.k + b * a.k_sb + hk * a.k_sh;
    const float* vp = a.v + b * a.v_sb + hk * a.v_sh;
#pragma unroll
    for (int f = tid; f < KB * C; f += BT) {
      const int r = f / C, c = f % C;
      const bool ok = k0 + r < SK;
      const int64_t row = ok ? k0 + r : 0;
      cp_async16(Ks + r * D + 4 * (c ^ swizzle(r)), kp + row * a.k_ss + 4 * c, ok ? 16 : 0);
      cp_async16(Vs + r * D + 4 * (c ^ swizzle(r)), vp + row * a.v_ss + 4 * c, ok ? 16 : 0);
    }
  }
  auto load_query_tile = [&](int t) {
#pragma unroll
    for (int f = tid; f < 64 * C; f += BT) {
      const int r = f / C, c = f % C;
      const bool ok = t * 64 + r < rows;
      int head, i;
      query_of(ok ? t * 64 + r : t * 64, head, i);
      cp_async16(Qs + r * D + 4 * (c ^ swizzle(r)), a.q + b * a.q_sb + head * a.q_sh + i * a.q_ss + 4 * c,
                 ok ? 16 : 0);
      cp_async16(dOs + r * D + 4 * (c ^ swizzle(r)),
                 a.d_o + b * a.do_sb + head * a.do_sh + i * a.do_ss + 4 * c, ok ? 16 : 0);
    }
    if (tid < 128) {
      const int r = tid & 63, x = t * 64 + r;
      const bool ok = x < rows;
      int head, i;
      query_of(ok ? x : t * 64, head, i);
      const float* src = (tid < 64 ? a.lse : a.dsum) + (static_cast<int64_t>(b) * a.H + head) * S + i;
      cp_async4((tid < 64 ? Lt : Dt) + r, src, ok ? 4 : 0);
    }
    cp_async_commit();
  };
  // A row-major tile's 16 bytes as this lane reads them: dims 16 j + 4 t4 .. of row r with r % 8 = g; and
  // dims 32 j + 4 g .. of rows 8 i + 2 t4 (y = 0) and + 1.
  const int by_row = g * D + 4 * (t4 ^ swizzle(g));
  auto at_row = [&](const float* x, int r8, int j) {
    return ld4(x + r8 * D + ((by_row + 0) ^ (16 * (j & 1))) + 32 * (j >> 1));
  };
  const int by_col0 = 2 * t4 * D + 4 * (g ^ swizzle(2 * t4)), by_col1 = (2 * t4 + 1) * D + 4 * (g ^ swizzle(2 * t4 + 1));
  auto at_col = [&](const float* x, int i, int y, int j) {
    return ld4(x + 8 * i * D + (y ? by_col1 : by_col0) + 32 * j);
  };

  float acc[D / 32][4][4];  // dV (dK): keys 16 wg + g, + 8; dims 32 j + 8 t4 + e, + 4
#pragma unroll
  for (int j = 0; j < D / 32; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int x = 0; x < 4; ++x) acc[j][e][x] = 0.0f;

  const int t_begin = static_cast<int>(static_cast<int64_t>(part) * nqt / nparts);
  const int t_end = static_cast<int>((static_cast<int64_t>(part) + 1) * nqt / nparts);
  load_query_tile(t_begin);
  for (int t = t_begin; t < t_end; ++t) {
    const int q0 = t * 64;
    cp_async_wait_all();
    __syncthreads();

    // 1. Queries 16 wg + g, + 8; keys 8 i + 2 t4, + 1.
    {
      const float* As = (grp ? dOs : Qs) + 16 * wg * D;
      const float* Bs = grp ? Vs : Ks;
      float sc[8][4];
      clear(sc);
#pragma unroll 1
      for (int j = 0; j < D / 16; j += 2) {  // (the forward's sums)
        float c[8][4];
        clear(c);
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          uint32_t ah[2][4], al[2][4];
          split_rows(at_row(As, 0, j + y), at_row(As, 8, j + y), ah, al);
#pragma unroll
          for (int i = 0; i < 8; ++i) products(c[i], ah, al, at_row(Bs, 8 * i, j + y));
        }
        add(sc, c);
      }
      const int r0 = 16 * wg + g;
      if (grp == 0) {
        const bool edge = (q0 + 64 > rows) || (k0 + KB > SK);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float L = Lt[r0 + 8 * h];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float p[2];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              p[x] = ex2(fmaf(sc[i][2 * h + x], a.scale, -L) * LOG2E);
              if (edge && !(q0 + r0 + 8 * h < rows && k0 + 8 * i + 2 * t4 + x < SK)) p[x] = 0.0f;
            }
            *reinterpret_cast<float2*>(Ps + (r0 + 8 * h) * LP + 8 * i + 2 * t4) = make_float2(p[0], p[1]);
          }
        }
      }
      __syncthreads();
      if (grp == 1) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float d = Dt[r0 + 8 * h];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int at = (r0 + 8 * h) * LP + 8 * i + 2 * t4;
            const float2 p = *reinterpret_cast<const float2*>(Ps + at);
            *reinterpret_cast<float2*>(dSs + at) = make_float2(p.x * (sc[i][2 * h] - d), p.y * (sc[i][2 * h + 1] - d));
          }
        }
        asm volatile("bar.sync 1, %0;" ::"n"(BT / 2) : "memory");  // dS in place for its warps; the others go on to dV
      }
    }

    // 2. Keys 16 wg + g, + 8 of the transposed [query][key] tile; queries 8 i + 2 t4, + 1.
    {
      const float* Xs = (grp ? dSs : Ps) + 16 * wg + g;
      const float* Ys = grp ? Qs : dOs;
      uint32_t xh[8][4], xl[8][4];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float* x = Xs + (8 * i + 2 * t4) * LP;
        split_tf32(make_float4(x[0], x[8], x[LP], x[LP + 8]), xh[i], xl[i]);
      }
#pragma unroll
      for (int j = 0; j < D / 32; ++j) {
        float small[4][4], large[4][4];
        clear(small);
        clear(large);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          products(small, large, xh[i], xl[i], at_col(Ys, i, 0, j), at_col(Ys, i, 1, j));
          if (i == 3) {
            add(acc[j], large);
            clear(large);
          }
        }
        add(large, small);
        add(acc[j], large);
      }
    }
    __syncthreads();
    if (t + 1 < t_end) load_query_tile(t + 1);

    // 3. Queries 16 wg + g, + 8; keys 8 i + 2 t4, + 1; dims 64 grp + 32 j + 8 t4 + e, + 4.
    float pq[2][4][4];
    {
      const float* Xs = dSs + (16 * wg + g) * LP + 2 * t4;
      uint32_t xh[8][4], xl[8][4];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float2 x = *reinterpret_cast<const float2*>(Xs + 8 * i);
        const float2 y = *reinterpret_cast<const float2*>(Xs + 8 * LP + 8 * i);
        split_tf32(make_float4(x.x, y.x, x.y, y.y), xh[i], xl[i]);
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float small[4][4], large[4][4];
        clear(pq[j]);
        clear(small);
        clear(large);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          products(small, large, xh[i], xl[i], at_col(Ks, i, 0, 2 * grp + j), at_col(Ks, i, 1, 2 * grp + j));
          if (i == 3) {
            add(pq[j], large);
            clear(large);
          }
        }
        add(large, small);
        add(pq[j], large);
      }
    }
    auto partial = [&](int j, int h, int x) {
      return make_float4(pq[j][0][2 * h + x], pq[j][1][2 * h + x], pq[j][2][2 * h + x], pq[j][3][2 * h + x]);
    };
    const int d0 = 64 * grp + 8 * t4;
    if (no_wait) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int x = q0 + 16 * wg + g + 8 * h;
        if (x >= rows) continue;
        int head, i;
        query_of(x, head, i);
        float* dst = a.dq_part +
                     (((static_cast<int64_t>(b) * a.H + head) * a.n_kblocks + kb) * S + i) * D + d0;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int y = 0; y < 2; ++y)
            __stcg(reinterpret_cast<float4*>(dst + 32 * j + 4 * y), partial(j, h, y));
      }
      continue;
    }
    // Turn chain: key blocks add into dQ in index order, each on its turn.
    const int last = nkb - 1;
    bool go = true;
    if (kb > 0) {
      if (tid == 0) {
        s_int[1] = wait_turn_bounded(turn + t, kb, a.err, a.timeout_ns, a.sink) ? 1 : 0;
        __threadfence();  // ORDER: with the barrier, extends thread 0's acquire to the block
      }
      __syncthreads();
      go = s_int[1] != 0;
    }
    if (go) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int x = q0 + 16 * wg + g + 8 * h;
        if (x >= rows) continue;
        int head, i;
        query_of(x, head, i);
        float* dst = a.dq + ((static_cast<int64_t>(b) * S + i) * a.H + head) * D + d0;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            float4* at = reinterpret_cast<float4*>(dst + 32 * j + 4 * y);
            float4 v = partial(j, h, y);
            if (kb > 0) {  // through L2: L1 is not coherent across SMs
              const float4 p = __ldcg(at);
              v = make_float4(p.x + v.x, p.y + v.y, p.z + v.z, p.w + v.w);
            }
            if (kb == last) v = make_float4(v.x * dscale, v.y * dscale, v.z * dscale, v.w * dscale);
            __stcg(at, v);
          }
      }
    }
    if (kb < last) {
      __threadfence();  // ORDER: this block's dQ stores are visible before the turn passes on
      __syncthreads();
      if (tid == 0) st_release_gpu(turn + t, kb + 1);
    }
  }

  // grp 0 stores dV, grp 1 stores dK * scale.
  // (dkv [b, Sk, 2, Hk, D], dK first; rows past the length hold zeros.)
  const float f = grp ? dscale : 1.0f;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = k0 + 16 * wg + g + 8 * h;
    if (r >= a.Sk) continue;
    float* dst = dkv + (((static_cast<int64_t>(b) * a.Sk + r) * 2 + (grp ? 0 : 1)) * a.Hk + hk) * D + 8 * t4;
#pragma unroll
    for (int j = 0; j < D / 32; ++j)
#pragma unroll
      for (int x = 0; x < 2; ++x)
        *reinterpret_cast<float4*>(dst + 32 * j + 4 * x) =
            make_float4(acc[j][0][2 * h + x] * f, acc[j][1][2 * h + x] * f, acc[j][2][2 * h + x] * f,
                        acc[j][3][2 * h + x] * f);
  }
}

}  // namespace

cudaError_t setup_cross_hd_attributes() {
  const cudaError_t e =
      cudaFuncSetAttribute(cross_hd_fwd_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
  return e != cudaSuccess ? e
                          : cudaFuncSetAttribute(cross_hd_bwd_kernel,
                                                 cudaFuncAttributeMaxDynamicSharedMemorySize, BWD_SMEM);
}

cudaError_t launch_cross_hd_fwd(const FwdArgs& args, cudaStream_t stream) {
  FwdArgs a = args;
  a.n_qtiles = static_cast<int>((static_cast<int64_t>(a.H / a.Hk) * a.S + BM - 1) / BM);
  const dim3 grid(static_cast<unsigned>(static_cast<int64_t>(a.n_qtiles) * a.B * a.Hk));
  return launch_pdl(cross_hd_fwd_kernel, grid, dim3(NT), static_cast<size_t>(SMEM), stream, a);
}

cudaError_t launch_cross_hd_bwd(const BwdArgs& args, cudaStream_t stream) {
  BwdArgs a = args;
  a.n_kblocks = (a.Sk + KB - 1) / KB;
  const dim3 grid(static_cast<unsigned>(static_cast<int64_t>(a.n_kblocks) * a.B * a.Hk * a.n_parts));
  const cudaError_t e =
      launch_pdl(cross_hd_bwd_kernel, grid, dim3(BT), static_cast<size_t>(BWD_SMEM), stream, a);
  return e == cudaSuccess ? launch_cross_join(a, D, KB, stream) : e;
}

}  // namespace cfa
