// SPDX-License-Identifier: MIT OR Apache-2.0
//
// Cross attention at head dim 128: the forward and the one-pass backward of hd_ffma.cu (whose header
// states the tiles, the thread layout and the orders of summation; hd_ffma.cuh holds what both
// share) with keys of another length and shared key heads, as the tensor-core pair has them at 64 and
// 32: a.Sk key rows, of which batch element b attends the first cross_keys(a, b); a block's query rows
// are those of a key head's whole group (row r: head r / S of it, query r % S), dK, dV of a shared
// head summed in that order; parts of the tiles and cross_join_kernel as in cross_bwd_tc.cu; dQ and
// dK, dV go to buffers of their own. Bound by fp32 FMA issue, as hd_ffma.cu
// is: [16, 8, 512 x 512, 128] forward 442 us, backward 1128 us, 39 and 38 TFLOP/s.
#include "hd_ffma.cuh"

namespace cfa {
namespace {

// The query rows of a key head's group: row r is query r % S of head h0 + r / S.
struct GroupRows {
  int h0, S, n, group;
  __device__ __forceinline__ GroupRows(int group_, int key_head, int S_)
      : h0(key_head * group_), S(S_), n(group_ * S_), group(group_) {}
  __device__ __forceinline__ void query_of(int r, int& head, int& i) const {
    const int g = group == 1 ? 0 : r / S;
    head = h0 + g;
    i = r - g * S;
  }
  // Rows row0 .. of a [heads, S, D] operand into a [ROWS][D + 4] tile (zeros past the last row).
  template <int ROWS, int NT, int D>
  __device__ __forceinline__ void load(float* dst, const float* src, int64_t h_stride, int64_t s_stride,
                                       int row0) const {
    constexpr int C = D / 4;
#pragma unroll
    for (int idx = threadIdx.x; idx < ROWS * C; idx += NT) {
      const int r = idx / C, c4 = idx % C;
      const bool ok = row0 + r < n;
      int head, i;
      query_of(ok ? row0 + r : row0, head, i);
      cp_async16(dst + r * ldh<D>() + 4 * c4, src + head * h_stride + i * s_stride + 4 * c4, ok ? 16 : 0);
    }
  }
};

template <int D, int RPT>
__global__ void __launch_bounds__(FWD_THREADS, Hd<D>::FWD_MINB) cross_hd_fwd_kernel(const FwdArgs a) {
  constexpr int BM = fwd_bm<RPT>(), L = ldh<D>(), NP = Dims<D>::NP;
  extern __shared__ float4 smem4[];
  float* Qs = reinterpret_cast<float*>(smem4);  // [BM][L]
  float* Ks = Qs + BM * L;                      // [64][L]
  float* Vs = Ks + 64 * L;                      // [64][L]
  float* Ps = Vs + 64 * L;                      // [BM][LDP]

  griddep_wait();  // q, k, v may come from the previous kernel on the stream
  griddep_launch_dependents();
  const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31;
  const int ty = lane >> 4, tx = lane & 15;
  const int qt = static_cast<int>(blockIdx.x % a.n_qtiles);
  const int bh = static_cast<int>(blockIdx.x / a.n_qtiles);
  const int b = bh / a.Hk, h = bh % a.Hk;  // the key head
  const int q0 = qt * BM;
  const int SK = cross_keys(a, b);
  const GroupRows rows(a.H / a.Hk, h, a.S);
  if (SK == 0) {  // no key: O = 0, L = -inf
    for (int f = tid; f < min(BM, rows.n - q0) * (D / 4); f += FWD_THREADS) {
      int head, i;
      rows.query_of(q0 + f / (D / 4), head, i);
      reinterpret_cast<float4*>(a.o + ((static_cast<int64_t>(b) * a.S + i) * a.H + head) * D)[f % (D / 4)] =
          make_float4(0.f, 0.f, 0.f, 0.f);
      if (f % (D / 4) == 0) a.lse[(static_cast<int64_t>(b) * a.H + head) * a.S + i] = -INFINITY;
    }
    return;
  }
  const float* kp = a.k + b * a.k_sb + h * a.k_sh;
  const float* vp = a.v + b * a.v_sb + h * a.v_sh;

  rows.load<BM, FWD_THREADS, D>(Qs, a.q + b * a.q_sb, a.q_sh, a.q_ss, q0);
  load_rows_async<64, FWD_THREADS, D>(Ks, kp, a.k_ss, 0, SK);
  cp_async_commit();

  const int rb = 2 * RPT * w + ty;  // rows rb + 2i
  float m[RPT], lpart[RPT];
  uint64_t acc2[RPT][NP];
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    m[i] = -INFINITY;
    lpart[i] = 0.0f;
#pragma unroll
    for (int p = 0; p < NP; ++p) acc2[i][p] = 0ull;
  }

  for (int k0 = 0; k0 < SK; k0 += 64) {
    cp_async_wait_all();
    __syncthreads();
    load_rows_async<64, FWD_THREADS, D>(Vs, vp, a.v_ss, k0, SK);
    cp_async_commit();

    const int jn = min(4, (SK - k0 + 15) / 16);
    float s[RPT][4];
    if (jn == 3)
      scores<3, RPT, D>(Qs, Ks, rb, tx, s);
    else
      scores<4, RPT, D>(Qs, Ks, rb, tx, s);

    const bool edge = k0 + 64 > SK;
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
      float x[4];
#pragma unroll
      for (int jj = 0; jj < 4; ++jj) x[jj] = s[i][jj] * a.scale;
      if (edge) {
#pragma unroll
        for (int jj = 0; jj < 4; ++jj)
          if (k0 + tx + 16 * jj >= SK) x[jj] = -INFINITY;
      }
      float tmax = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
      tmax = half_warp_max(tmax);
      const float m_new = fmaxf(m[i], tmax);
      const float mu = m_new == -INFINITY ? 0.0f : m_new;
      const float alpha = expf(m[i] - mu);
      float psum = 0.0f;
#pragma unroll
      for (int jj = 0; jj < 4; ++jj) {
        const float pr = expf(x[jj] - mu);
        Ps[(rb + 2 * i) * LDP + tx + 16 * jj] = pr;
        psum += pr;
      }
      lpart[i] = fmaf(lpart[i], alpha, psum);
      m[i] = m_new;
      const uint64_t al = dup2(alpha);
#pragma unroll
      for (int p = 0; p < NP; ++p) acc2[i][p] = mul2(acc2[i][p], al);
    }
    cp_async_wait_all();
    __syncthreads();
    if (k0 + 64 < SK) {
      load_rows_async<64, FWD_THREADS, D>(Ks, kp, a.k_ss, k0 + 64, SK);
      cp_async_commit();
    }

    // O += P V over the live key groups, keys in order (groups past the end hold P = 0).
    const int jlim = 16 * jn;
#pragma unroll 8
    for (int j = 0; j < jlim; j += 4) {
      uint64_t vv[4][NP];
      float4 pv[RPT];
#pragma unroll
      for (int t = 0; t < 4; ++t) Dims<D>::load(Vs + (j + t) * L, tx, vv[t]);
#pragma unroll
      for (int i = 0; i < RPT; ++i) pv[i] = ld4(Ps + (rb + 2 * i) * LDP + j);
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < RPT; ++i) {
          const uint64_t pr = dup2(f4c(pv[i], t));
#pragma unroll
          for (int p = 0; p < NP; ++p) acc2[i][p] = fma2(pr, vv[t][p], acc2[i][p]);
        }
    }
  }

#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    const float l = half_warp_sum(lpart[i]);
    const int r = q0 + rb + 2 * i;
    if (r >= rows.n) continue;
    int head, qi;
    rows.query_of(r, head, qi);
    float ov[D / 16];
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const float2 v = split2(acc2[i][p]);
      ov[2 * p] = __fdiv_rn(v.x, l);
      ov[2 * p + 1] = __fdiv_rn(v.y, l);
    }
    store_dims<D>(a.o + ((static_cast<int64_t>(b) * a.S + qi) * a.H + head) * D, tx, ov);
    if (tx == 0) a.lse[(static_cast<int64_t>(b) * a.H + head) * a.S + qi] = m[i] + logf(l);
  }
}

template <int D>
__global__ void __launch_bounds__(Bwd<D>::NT, 256 / (Bwd<D>::NT / 2)) cross_hd_bwd_kernel(const BwdArgs a) {
  constexpr int NT = Bwd<D>::NT, WG = Bwd<D>::WG, R1 = Bwd<D>::R1, K2 = Bwd<D>::K2;
  constexpr int NP2 = Bwd<D>::NP2, L = ldh<D>();
  constexpr int DPT = 2 * NP2;  // phase 2 dims per thread
  extern __shared__ float4 smem4[];
  float* Ks = reinterpret_cast<float*>(smem4);  // [64][L]
  float* Vs = Ks + 64 * L;
  float* Qs = Vs + 64 * L;
  float* dOs = Qs + 64 * L;
  float* Ps = dOs + 64 * L;   // [64][LDP] query-major
  float* dSs = Ps + 64 * LDP;
  float* Lt = dSs + 64 * LDP;
  float* Dt = Lt + 64;
  int* s_int = reinterpret_cast<int*>(Dt + 64);

  griddep_launch_dependents();
  const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31;
  const int ty = lane >> 4, tx = lane & 15;
  const int grp = w / WG, wg = w % WG;  // grp 0: S, P, dV; grp 1: dP, dS, dK
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
  const int b = bh / a.Hk, h = bh % a.Hk;  // the key head
  const int k0 = kb * 64;
  const int group = a.H / a.Hk;
  const GroupRows rows(group, h, S);  // the key block's query rows
  const int nqt = (rows.n + 63) / 64;
  const int SK = cross_keys(a, b);
  const int nkb = (SK + 63) / 64;  // key blocks of this (batch, head) that take part
  float* dkv = a.dkv + static_cast<int64_t>(part) * a.part_stride;  // (parts: in the workspace)
  if (kb >= nkb) {  // no key of this block is attended: zeros, and no part in dQ's sums
    constexpr int C4 = D / 4;
    const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
    const int krows = min(64, a.Sk - k0);
    for (int f = tid; f < 2 * krows * C4; f += NT) {
      const int which = f / (krows * C4), r = (f / C4) % krows;
      reinterpret_cast<float4*>(
          dkv + (((static_cast<int64_t>(b) * a.Sk + k0 + r) * 2 + which) * a.Hk + h) * D)[f % C4] = zero;
    }
    if (kb == 0 && part == 0)  // no key at all: dQ = 0
      for (int64_t f = tid; f < static_cast<int64_t>(rows.n) * C4; f += NT)
        reinterpret_cast<float4*>(a.dq + ((static_cast<int64_t>(b) * S + f / (group * C4)) * a.H + rows.h0) *
                                             D)[f % (group * C4)] = zero;
    return;
  }
  int* turn = a.turn + static_cast<int64_t>(bh) * nqt;  // turn chain: counters per tile
  const int64_t row_stride = static_cast<int64_t>(a.H) * D;  // dq floats per (b, s)

  load_rows_async<64, NT, D>(Ks, a.k + b * a.k_sb + h * a.k_sh, a.k_ss, k0, SK);
  load_rows_async<64, NT, D>(Vs, a.v + b * a.v_sb + h * a.v_sh, a.v_ss, k0, SK);

  // grp 0: dV, grp 1: dK (unscaled). acc2[rp][e]: keys kb2 + 2rp, kb2 + 2rp + 1 (a pair), dim e
  // of this thread's phase 2 dims.
  uint64_t acc2[K2 / 2][DPT];
#pragma unroll
  for (int i = 0; i < K2 / 2; ++i)
#pragma unroll
    for (int e = 0; e < DPT; ++e) acc2[i][e] = 0ull;

  const int rb1 = 2 * R1 * wg + ty;          // phase 1 rows: rb1 + 2i (warp: 2 R1 rows)
  const int kb2 = K2 * (2 * wg + ty);        // phase 2 keys: kb2 .. kb2 + K2 - 1
  // phase 3: rows rb3 + 2r (r < 4), dims d3 .. d3 + 3 (the two groups take the halves)
  const int rb3 = 8 * wg + ty;
  const int d3 = 64 * grp + 4 * tx;

  auto load_q_do = [&](int t) {
    rows.load<64, NT, D>(Qs, a.q + b * a.q_sb, a.q_sh, a.q_ss, t * 64);
    rows.load<64, NT, D>(dOs, a.d_o + b * a.do_sb, a.do_sh, a.do_ss, t * 64);
  };
  auto load_l_d = [&](int t) {
    if (tid < 128) {
      const int r = tid & 63, x = t * 64 + r;
      const bool ok = x < rows.n;
      int head, i;
      rows.query_of(ok ? x : t * 64, head, i);
      const float* src = (tid < 64 ? a.lse : a.dsum) + (static_cast<int64_t>(b) * a.H + head) * S + i;
      cp_async4((tid < 64 ? Lt : Dt) + r, src, ok ? 4 : 0);
    }
  };
  auto load_query_tile = [&](int t) {
    load_q_do(t);
    load_l_d(t);
  };

  const int t_begin = static_cast<int>(static_cast<int64_t>(part) * nqt / nparts);
  const int t_end = static_cast<int>((static_cast<int64_t>(part) + 1) * nqt / nparts);
  load_query_tile(t_begin);
  cp_async_commit();
  for (int t = t_begin; t < t_end; ++t) {
    const int q0 = t * 64;
    cp_async_wait_all();
    __syncthreads();

    const int jn = min(4, (SK - k0 + 15) / 16);
    const int iq = min(64, (rows.n - q0 + 15) / 16 * 16);

    // Phase 1. grp 0: s = Q K^T; grp 1: s = dO V^T (dP).
    {
      const float* As = grp ? dOs : Qs;
      const float* Bs = grp ? Vs : Ks;
      float s[R1][4];
      if (q0 + 2 * R1 * wg >= rows.n) {
#pragma unroll
        for (int i = 0; i < R1; ++i)
#pragma unroll
          for (int jj = 0; jj < 4; ++jj) s[i][jj] = 0.0f;
      } else if (jn == 4) {
        scores<4, R1, D>(As, Bs, rb1, tx, s);
      } else if (jn == 3) {
        scores<3, R1, D>(As, Bs, rb1, tx, s);
      } else if (jn == 2) {
        scores<2, R1, D>(As, Bs, rb1, tx, s);
      } else {
        scores<1, R1, D>(As, Bs, rb1, tx, s);
      }
      if (grp == 0) {
        const bool edge = (q0 + 64 > rows.n) || (k0 + 64 > SK);
#pragma unroll
        for (int i = 0; i < R1; ++i) {
          const int il = rb1 + 2 * i, qi = q0 + il;
          const float li = Lt[il];
#pragma unroll
          for (int jj = 0; jj < 4; ++jj) {
            const int jl = tx + 16 * jj, j = k0 + jl;
            float pr = expf(fmaf(s[i][jj], a.scale, -li));
            if (edge && !(qi < rows.n && j < SK)) pr = 0.0f;
            Ps[il * LDP + jl] = pr;
          }
        }
      }
      __syncthreads();
      if (grp == 1) {
#pragma unroll
        for (int i = 0; i < R1; ++i) {
          const int il = rb1 + 2 * i;
          const float di = Dt[il];
#pragma unroll
          for (int jj = 0; jj < 4; ++jj) {
            const int jl = tx + 16 * jj;
            dSs[il * LDP + jl] = Ps[il * LDP + jl] * (s[i][jj] - di);
          }
        }
      }
      __syncthreads();
    }

    // Phase 2. grp 0: dV[j] += sum_i P[i][j] dO[i]; grp 1: dK[j] += sum_i dS[i][j] Q[i]. Pairs
    // along keys, the dO / Q element broadcast; queries in index order.
    {
      const float* Xs = grp ? dSs : Ps;
      const float* Ys = grp ? Qs : dOs;
      const int iw = k0 + kb2 - K2 * ty >= SK ? 0 : iq;  // all this warp's keys past the end
#pragma unroll 8
      for (int i = 0; i < iw; ++i) {
        uint64_t xp[K2 / 2];
        if constexpr (K2 == 8) {
          const ulonglong2 xa = ld2x2(Xs + i * LDP + kb2), xb = ld2x2(Xs + i * LDP + kb2 + 4);
          xp[0] = xa.x;
          xp[1] = xa.y;
          xp[2] = xb.x;
          xp[3] = xb.y;
        } else {
          const ulonglong2 xa = ld2x2(Xs + i * LDP + kb2);
          xp[0] = xa.x;
          xp[1] = xa.y;
        }
        float y[DPT];
        Dims<D>::load_f(Ys + i * L, tx, y);
#pragma unroll
        for (int e = 0; e < DPT; ++e) {
          const uint64_t yb = dup2(y[e]);
#pragma unroll
          for (int rp = 0; rp < K2 / 2; ++rp) acc2[rp][e] = fma2(xp[rp], yb, acc2[rp][e]);
        }
      }
    }
    __syncthreads();
    if (t + 1 < t_end) {
      load_query_tile(t + 1);
      cp_async_commit();
    }

    // Phase 3: the dQ partial pq[r][e] = sum_j dS[rb3 + 2r][j] K[j][d3 + e], keys in order.
    constexpr int E3 = 4;
    uint64_t pq2[4][E3 / 2];
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int p = 0; p < E3 / 2; ++p) pq2[r][p] = 0ull;
    const int jlim = q0 + (rb3 - ty) >= rows.n ? 0 : 16 * jn;
#pragma unroll 2
    for (int j = 0; j < jlim; j += 4) {
      uint64_t k2[4][E3 / 2];
      float4 d4[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const ulonglong2 kv = ld2x2(Ks + (j + u) * L + d3);
        k2[u][0] = kv.x;
        k2[u][1] = kv.y;
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) d4[r] = ld4(dSs + (rb3 + 2 * r) * LDP + j);
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const uint64_t ds = dup2(f4c(d4[r], u));
#pragma unroll
          for (int p = 0; p < E3 / 2; ++p) pq2[r][p] = fma2(ds, k2[u][p], pq2[r][p]);
        }
    }
    float pq[4][E3];
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int p = 0; p < E3 / 2; ++p) {
        const float2 v = split2(pq2[r][p]);
        pq[r][2 * p] = v.x;
        pq[r][2 * p + 1] = v.y;
      }

    if (a.dq_part != nullptr) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int x = q0 + rb3 + 2 * r;
        if (x >= rows.n) continue;
        int head, qi;
        rows.query_of(x, head, qi);
        float* dst = a.dq_part +
                     (((static_cast<int64_t>(b) * a.H + head) * a.n_kblocks + kb) * S + qi) * D + d3;
        __stcg(reinterpret_cast<float4*>(dst), make_float4(pq[r][0], pq[r][1], pq[r][2], pq[r][3]));
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
      for (int r = 0; r < 4; ++r) {
        const int x = q0 + rb3 + 2 * r;
        if (x >= rows.n) continue;
        int head, qi;
        rows.query_of(x, head, qi);
        float* dst = a.dq + ((static_cast<int64_t>(b) * S + qi) * a.H + head) * D + d3;
#pragma unroll
        for (int e = 0; e < E3; ++e) {
          float v = pq[r][e];
          if (kb > 0) v = __ldcg(dst + e) + v;  // through L2: L1 is not coherent across SMs
          if (kb == last) v *= a.scale;
          __stcg(dst + e, v);
        }
      }
    }
    if (kb < last) {
      __threadfence();  // ORDER: this block's dQ stores are visible before the turn passes on
      __syncthreads();
      if (tid == 0) st_release_gpu(turn + t, kb + 1);
    }
  }

  if (a.dq_part != nullptr && !a.join_dq) {  // (without join_dq there is one part)
    // ORDER: partials visible GPU-wide before counting in; the last to count sums them all.
    __threadfence();
    __syncthreads();
    if (tid == 0) s_int[1] = atomicAdd(a.turn + bh, 1);
    __syncthreads();
    if (s_int[1] == nkb - 1) {
      __threadfence();
      constexpr int C = D / 4;  // float4 per row
      // DETERMINISM: (((p0 + p1) + p2) + ...) * scale over the contributing key blocks in order.
      for (int hq = rows.h0; hq < rows.h0 + group; ++hq) {
        const float* part = a.dq_part + (static_cast<int64_t>(b) * a.H + hq) * a.n_kblocks * S * D;
        float* dq_out = a.dq + static_cast<int64_t>(b) * S * row_stride + hq * D;
        for (int idx = tid; idx < S * C; idx += NT) {
          const int i = idx / C, c4 = idx % C;
          float4 v = __ldcg(reinterpret_cast<const float4*>(part + static_cast<int64_t>(i) * D + 4 * c4));
          for (int j = 1; j < nkb; ++j) {
            const float4 p = __ldcg(reinterpret_cast<const float4*>(
                part + (static_cast<int64_t>(j) * S + i) * D + 4 * c4));
            v = make_float4(v.x + p.x, v.y + p.y, v.z + p.z, v.w + p.w);
          }
          *reinterpret_cast<float4*>(dq_out + i * row_stride + 4 * c4) =
              make_float4(v.x * a.scale, v.y * a.scale, v.z * a.scale, v.w * a.scale);
        }
      }
    }
  }

  // grp 0 stores dV, grp 1 stores dK * scale.
  // (dkv [b, Sk, 2, Hk, D], dK first; rows past the length hold zeros.)
  const int64_t kv_stride = 2 * static_cast<int64_t>(a.Hk) * D;
  float* dst0 = dkv + static_cast<int64_t>(b) * a.Sk * kv_stride + (grp ? 0 : 1) * a.Hk * D + h * D;
  const float f = grp ? a.scale : 1.0f;
#pragma unroll
  for (int rp = 0; rp < K2 / 2; ++rp) {
    float lo[DPT], hi[DPT];
#pragma unroll
    for (int e = 0; e < DPT; ++e) {
      const float2 v = split2(acc2[rp][e]);
      lo[e] = v.x * f;
      hi[e] = v.y * f;
    }
    const int j = k0 + kb2 + 2 * rp;
    if (j < a.Sk) store_dims<D>(dst0 + j * kv_stride, tx, lo);
    if (j + 1 < a.Sk) store_dims<D>(dst0 + (j + 1) * kv_stride, tx, hi);
  }
}

}  // namespace

// Cross attention at head dim 128.
cudaError_t setup_cross_hd_attributes() {
  constexpr int A = Hd<128>::RPT_A;
  const cudaError_t e =
      cudaFuncSetAttribute(cross_hd_fwd_kernel<128, A>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           hd_fwd_smem_floats<128, A>() * 4);
  return e != cudaSuccess ? e
                          : cudaFuncSetAttribute(cross_hd_bwd_kernel<128>,
                                                 cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 hd_bwd_smem_floats<128>() * 4);
}

cudaError_t launch_cross_hd_fwd(const FwdArgs& args, cudaStream_t stream) {
  constexpr int A = Hd<128>::RPT_A, bm = fwd_bm<A>();
  FwdArgs a = args;
  a.n_qtiles = static_cast<int>((static_cast<int64_t>(a.H / a.Hk) * a.S + bm - 1) / bm);
  const dim3 grid(static_cast<unsigned>(static_cast<int64_t>(a.n_qtiles) * a.B * a.Hk));
  return launch_pdl(cross_hd_fwd_kernel<128, A>, grid, dim3(FWD_THREADS),
                    static_cast<size_t>(hd_fwd_smem_floats<128, A>() * 4), stream, a);
}

cudaError_t launch_cross_hd_bwd(const BwdArgs& args, cudaStream_t stream) {
  BwdArgs a = args;
  a.n_kblocks = (a.Sk + 63) / 64;
  const dim3 grid(static_cast<unsigned>(static_cast<int64_t>(a.n_kblocks) * a.B * a.Hk * a.n_parts));
  const cudaError_t e = launch_pdl(cross_hd_bwd_kernel<128>, grid, dim3(Bwd<128>::NT),
                                   static_cast<size_t>(hd_bwd_smem_floats<128>() * 4), stream, a);
  return e == cudaSuccess ? launch_cross_join(a, 128, 64, stream) : e;
}

}  // namespace cfa
