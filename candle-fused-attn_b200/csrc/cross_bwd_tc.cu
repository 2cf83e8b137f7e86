// SPDX-License-Identifier: MIT OR Apache-2.0
//
// Cross attention's backward on the tensor cores (head dims 64 and 32): dQ, dK, dV of O =
// softmax(Q K^T * scale) V where the keys have a length of their own and groups of query heads share
// a key head. The five products, their split fp32 operands and the schedule are bwd_tc.cu's (its
// header states them; bwd_tc.cuh holds what both share); what differs:
//  - a.Sk key rows, of which batch element b attends the first cross_keys(a, b). Key blocks past
//    them write zeros and take no part;
//  - a key block belongs to a key head and walks the query rows of its whole group, head after head
//    (row r: head r / S of the group, query r % S), in tiles of 64 rows, so dV and dK of a shared head
//    are summed in registers in that order and a group of short query sequences fills the tiles;
//  - with few key blocks a batch element (cross_layout's rule, by the shapes of one element alone) the
//    tiles are cut into parts of consecutive ones, a block each, whose dV, dK sums cross_join_kernel
//    adds in order. (bwd_tc.cu's split tail would have one block fold every tile of the others: at 16
//    heads over one, [2, 16, 1024, 64], that and one block's sum of all dQ partials took 1.2 of 1.5
//    ms.) Where the dQ partials of a (batch, key head) exceed 320 KB, or with parts, that kernel
//    sums them too, by all SMs; below, the key head's last block does, behind which the others run on
//    ([64, 6, 240, 64] over 100 to 600 keys: 272 us so, 279 by the join; kCrossJoinBytes has more);
//  - dQ [B, S, H, HD] and dK, dV [B, Sk, 2, Hk, HD] go to buffers of their own.
// It is a kernel of its own, because at 96 registers a thread the fused attention's backward keeps
// its registers only as it stands: as one template, that instance spilled or slowed by 0.2 to 3 %.
// Bound by the compute warps' work a tile, as bwd_tc.cu is: [4, 16 over 4, 2048 x 8192, 64] 4.4 to 4.7
// ms, 147 to 155 TFLOP/s of fp32 products (six bf16 ones each); the training step's ragged [64, 6, 240,
// 64] 272 us, 76 TFLOP/s: four tiles a block, whose first loads and last stores take 40 % of it.
#include <algorithm>

#include "bwd_tc.cuh"

namespace cfa {
namespace {

template <int HD>
__global__ void __launch_bounds__(NB, 1) cross_bwd_tc_kernel(const BwdArgs a) {
  static_assert(HD == 64 || HD == 32, "head dims of the tensor-core backward");
  constexpr int KSD = HD / 16;  // K-steps of the products that reduce over the head dim
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  const uint32_t raw = tc::smem_u32(smem_raw);
  unsigned char* sm = smem_raw + ((1024u - (raw & 1023u)) & 1023u);
  unsigned char* Kp = sm + OFF_K;
  unsigned char* Qp = sm + OFF_Q;
  unsigned char* dOp = sm + OFF_DO;
  unsigned char* dSp = sm + OFF_DS;
  unsigned char* st = sm + OFF_ST;
  float* ld = reinterpret_cast<float*>(sm + OFF_LD);  // [buf][0: L, 1: D][64]
  // Commits (each covers every earlier MMA of the block) and arrivals (one per compute warp).
  uint64_t* bar_s = reinterpret_cast<uint64_t*>(sm + OFF_BAR);  // S^T of a tile done
  uint64_t* bar_t2 = bar_s + 1;  // dK, dQ of a tile done: every MMA of the tile
  uint64_t* bar_c1 = bar_s + 2;  // dS^T of a tile in shared memory (arrivals)
  uint64_t* bar_q = bar_s + 3;   // Q, dO parts of the next tile in place (arrivals)
  uint64_t* bar_ld = bar_s + 4;  // bulk copies: the prologue's rows, then the heads' dQ partials
  uint64_t* bar_dp = bar_s + 5;  // dP^T of a tile done
  uint64_t* bar_p = bar_s + 6;   // P^T's parts of a tile in TMEM (arrivals)
  uint64_t* bar_dv = bar_s + 7;  // dV of a tile done
  uint32_t* tbase_p = reinterpret_cast<uint32_t*>(bar_s + 8);
  int* s_int = reinterpret_cast<int*>(bar_s + 9);

  const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31;
  const bool mma_warp = w == NT / 32;   // warp 16 issues every MMA
  const int row = 32 * (w & 3) + lane;  // key row: TMEM lane (compute warps)
  const int cg = (w >> 2) & 3;          // column group: 16 queries (S, dP) or dims (dV, dK, dQ)
  const int S = a.S;
  const int BH = a.B * a.Hk;
  griddep_wait();  // the lengths, the cleared counters: the previous kernels' writes
  // The work item. With the dQ partials (no block waits for another): the block index, (b, h)-major, so
  // a (b, h)'s key blocks run side by side and its last one finishes early. With the turn chain: a
  // ticket drawn after the prep kernel's wait, key-block-major -- a block waits only on key block
  // kb - 1 of its (b, h) and part, which holds a smaller ticket, so it is running or done.
  const bool chain = a.dq_part == nullptr;
  int ticket = static_cast<int>(blockIdx.x);
  if (chain) {
    if (tid == 0) s_int[1] = atomicAdd(a.ticket, 1);
    __syncthreads();
    ticket = s_int[1];
  }
  const int nparts = a.n_parts, part = ticket % nparts, unit = ticket / nparts;
  const int kb = chain ? unit / BH : unit % a.n_kblocks;
  const int bh = chain ? unit % BH : unit / a.n_kblocks;
  const int b = bh / a.Hk, h = bh % a.Hk;  // the key head
  const int k0 = kb * KB;
  const int group = a.H / a.Hk, h0 = h * group;  // the key block's query heads
  const int rows = group * S, nqt = (rows + QT - 1) / QT;  // and their rows, in tiles
  const int SK = cross_keys(a, b);
  const int nkb = (SK + KB - 1) / KB;  // key blocks of this (batch, head) that take part
  const float dscale = grad_scale(a, SK);
  float* dkv = a.dkv + static_cast<int64_t>(part) * a.part_stride;  // (parts: in the workspace)
  if (kb >= nkb) {  // no key of this block is attended: zeros, and no part in dQ's sums
    griddep_launch_dependents();
    constexpr int C4 = HD / 4;
    const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
    const int krows = min(KB, a.Sk - k0);
    for (int f = tid; f < 2 * krows * C4; f += NB) {
      const int which = f / (krows * C4), r = (f / C4) % krows;
      reinterpret_cast<float4*>(
          dkv + (((static_cast<int64_t>(b) * a.Sk + k0 + r) * 2 + which) * a.Hk + h) * HD)[f % C4] = zero;
    }
    if (kb == 0 && part == 0)  // no key at all: dQ = 0
      for (int64_t f = tid; f < static_cast<int64_t>(rows) * C4; f += NB)
        reinterpret_cast<float4*>(a.dq + ((static_cast<int64_t>(b) * S + f / (group * C4)) * a.H + h0) *
                                             HD)[f % (group * C4)] = zero;
    return;
  }
  const float* kp = a.k + b * a.k_sb + h * a.k_sh;
  const float* vp = a.v + b * a.v_sb + h * a.v_sh;
  // Row r of the group's rows as (query head, query).
  auto query_of = [&](int r, int& head, int& i) {
    const int g = group == 1 ? 0 : r / S;
    head = h0 + g;
    i = r - g * S;
  };
  const int n_lo = static_cast<int>(static_cast<int64_t>(part) * nqt / nparts);
  const int n_hi = static_cast<int>((static_cast<int64_t>(part) + 1) * nqt / nparts);
  const int t_begin = n_lo;  // this block's first query tile
  int* turn = a.turn + static_cast<int64_t>(bh) * nqt;  // turn chain: counters per tile
  const int N = n_hi - n_lo;  // this block's query tiles, >= 1 (n_parts <= nqt)
  bool err0 = false;

  if (tid == 0) {
    tc::mbar_init(bar_s, 1);
    tc::mbar_init(bar_t2, 1);
    tc::mbar_init(bar_c1, NT / 32);
    tc::mbar_init(bar_q, NT / 32);
    tc::mbar_init(bar_ld, 1);
    tc::mbar_init(bar_dp, 1);
    tc::mbar_init(bar_p, NT / 32);
    tc::mbar_init(bar_dv, 1);
    tc::fence_mbar_init();
    tc::mbar_arrive_expect_tx(bar_ld, 4u * HD * (2 * min(KB, SK - k0) + 2 * min(QT, rows - t_begin * QT)));
  }
  griddep_launch_dependents();

  // Q, dO of tile n into this thread's staging slots (Q: slots 0-1, dO: 2-3) and its L, D into
  // L / D buffer n % 2 (threads 0-127).
  auto stage_ld = [&](int n) {
    if (tid < 2 * QT) {
      const int r = tid & 63, x = (t_begin + n) * QT + r;
      const bool ok = x < rows;
      int head, i;
      query_of(ok ? x : 0, head, i);
      const float* src = (tid < QT ? a.lse : a.dsum) + (static_cast<int64_t>(b) * a.H + head) * S + i;
      cp_async4(ld + (n & 1) * 128 + (tid < QT ? 0 : QT) + r, src, ok ? 4 : 0);
    }
  };
  auto stage_tile = [&](int n) {
    int r, kc;
    row_item(tid, r, kc);
    const int x = (t_begin + n) * QT + r;
    const bool ok = x < rows && 8 * kc < HD;
    int head, i;
    query_of(ok ? x : 0, head, i);
    const float* q = a.q + b * a.q_sb + head * a.q_sh + i * a.q_ss + (ok ? 8 * kc : 0);
    const float* g = a.d_o + b * a.do_sb + head * a.do_sh + i * a.do_ss + (ok ? 8 * kc : 0);
    const int n16 = ok ? 16 : 0;  // (slots 0-1: Q, 2-3: dO, as split_row_item reads them)
    cp_async16(st + 16 * tid, q, n16);
    cp_async16(st + 16 * (NT + tid), q + 4, n16);
    cp_async16(st + 16 * (2 * NT + tid), g, n16);
    cp_async16(st + 16 * (3 * NT + tid), g + 4, n16);
    stage_ld(n);
  };
  // The block one wave later starts by reading its key block's K, V rows and its first query tile's
  // Q, dO rows: pull them into L2 while this one computes (one row a thread).
  auto prefetch_next_wave = [&]() {
    const int64_t nb = static_cast<int64_t>(ticket) + a.wave_ctas;
    if (a.wave_ctas <= 0 || nb >= gridDim.x || tid >= 2 * KB + 2 * QT) return;
    const int npart = static_cast<int>(nb % nparts), nu = static_cast<int>(nb / nparts);
    const int nk = chain ? nu / BH : nu % a.n_kblocks, nbh = chain ? nu % BH : nu / a.n_kblocks;
    const int nb_b = nbh / a.Hk, nb_h = nbh % a.Hk;
    const float* src;
    if (tid < 2 * KB) {
      const int r = nk * KB + (tid & (KB - 1));
      if (r >= cross_keys(a, nb_b)) return;
      src = tid < KB ? a.k + nb_b * a.k_sb + nb_h * a.k_sh + r * a.k_ss
                     : a.v + nb_b * a.v_sb + nb_h * a.v_sh + r * a.v_ss;
    } else {
      const int r = static_cast<int>(static_cast<int64_t>(npart) * nqt / nparts) * QT + (tid & (QT - 1));
      if (r >= rows) return;
      const int g = group == 1 ? 0 : r / S;
      src = tid < 2 * KB + QT ? a.q + nb_b * a.q_sb + (nb_h * group + g) * a.q_sh + (r - g * S) * a.q_ss
                              : a.d_o + nb_b * a.do_sb + (nb_h * group + g) * a.do_sh + (r - g * S) * a.do_ss;
    }
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(src), "n"(4 * HD) : "memory");
  };
  auto split_tile = [&](int n) {
    split_row_item(Qp + (n & 1) * 3 * PART_Q, PART_Q, st, 0, tid);
    split_row_item(dOp + (n & 1) * 3 * PART_Q, PART_Q, st, 1, tid);
  };

  // Prologue: K's parts into shared memory, V's into TMEM (this thread's key row and 16 dims:
  // K-step cg of the A operand of dP^T), tile 0's Q and dO parts. The rows of K, V, Q, dO travel
  // as one bulk copy each (threads 0-383, one row apiece) into row-major staging with rows of
  // LDP = 68 floats (the dS^T and staging buffers: K, V; the second Q and dO part buffers: Q, dO
  // of tile 0); rows past the sequence are not copied and read as zeros. L, D and the cleared
  // counters come after the prep kernel's wait.
  constexpr int LDP = 68;
  float* k_rows = reinterpret_cast<float*>(dSp);
  float* v_rows = k_rows + KB * LDP;
  float* q_st = reinterpret_cast<float*>(Qp + 3 * PART_Q);
  float* o_st = reinterpret_cast<float*>(dOp + 3 * PART_Q);
  static_assert(2 * KB * LDP * 4 <= 3 * PART_K + 2 * QT * 64 * 4 && QT * LDP * 4 <= 3 * PART_Q,
                "prologue staging");
  const int nk = min(KB, SK - k0), nq = min(QT, rows - t_begin * QT);
  __syncthreads();  // the mbarriers' initialisation
  if (mma_warp) {  // TMEM, by the warp that is idle while the rows travel (it also frees it)
    tc::tmem_alloc(tbase_p, TMEM_COLS);
    tc::tmem_relinquish();
  }
  float vx[16];
  if (!mma_warp) {
    if (tid < 2 * KB + 2 * QT) {
      const int r = tid < 2 * KB ? (tid & (KB - 1)) : (tid & (QT - 1));
      if (tid < KB) {
        if (r < nk) tc::bulk_load(k_rows + r * LDP, kp + static_cast<int64_t>(k0 + r) * a.k_ss, 4 * HD, bar_ld);
      } else if (tid < 2 * KB) {
        if (r < nk) tc::bulk_load(v_rows + r * LDP, vp + static_cast<int64_t>(k0 + r) * a.v_ss, 4 * HD, bar_ld);
      } else if (r < nq) {
        int head, i;
        query_of(t_begin * QT + r, head, i);
        if (tid < 2 * KB + QT)
          tc::bulk_load(q_st + r * LDP, a.q + b * a.q_sb + head * a.q_sh + i * a.q_ss, 4 * HD, bar_ld);
        else
          tc::bulk_load(o_st + r * LDP, a.d_o + b * a.do_sb + head * a.do_sh + i * a.do_ss, 4 * HD, bar_ld);
      }
    }
    stage_ld(0);
    cp_async_commit();
    prefetch_next_wave();
    err0 = !tc::mbar_wait(bar_ld, 0, WAIT_TIMEOUT_NS);
    cp_async_wait_all();
    split_staged_row<HD>(Kp, PART_K, k_rows, tid, nk);
    split_staged_row<HD>(Kp, PART_K, k_rows, tid + NT, nk);
    split_staged_row<HD>(Qp, PART_Q, q_st, tid, nq);
    split_staged_row<HD>(dOp, PART_Q, o_st, tid, nq);
#pragma unroll
    for (int c4 = 0; c4 < 4; ++c4) {
      const float4 u = row < nk && 16 * cg < HD
                           ? reinterpret_cast<const float4*>(v_rows + row * LDP + 16 * cg)[c4]
                           : make_float4(0.f, 0.f, 0.f, 0.f);
      vx[4 * c4] = u.x;
      vx[4 * c4 + 1] = u.y;
      vx[4 * c4 + 2] = u.z;
      vx[4 * c4 + 3] = u.w;
    }
    tc::fence_async_smem();
  }
  tc::fence_before_sync();
  __syncthreads();  // the TMEM base; L, D of tile 0 (threads 0-127); the K staging read
  tc::fence_after_sync();
  const uint32_t tbase = *tbase_p;
  const uint32_t lane_sel = static_cast<uint32_t>(32 * (w & 3)) << 16;
  if (!mma_warp) {
    uint32_t vparts[3][8];
    split16(vx, vparts);
#pragma unroll
    for (int i = 0; i < 3; ++i) tmem_st8(tbase + lane_sel + T_V + 32 * i + 8 * cg, vparts[i]);
    tc::tmem_wait_st();
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();

  bool err = err0;
  uint32_t ld_phase = 1;  // bar_ld's next phase: the prologue's copies completed phase 0
  const int key = k0 + row;
  const uint64_t nsc2 = tc::pack2(-a.scale, -a.scale);     // L - s scale = fma(s, -scale, L)
  const uint64_t nl2e2 = tc::pack2(-LOG2E, -LOG2E);        // e^-y = 2^(-y log2 e)
  float dv[16], dk[16];  // compute threads: dV, dK of the key row, this thread's 16 dims
#pragma unroll
  for (int c = 0; c < 16; ++c) dv[c] = dk[c] = 0.0f;
  if (mma_warp) {
    {  // every lane runs the loop (warp-uniform); one elected lane issues each MMA and commit
      const uint32_t id128 = tc::idesc_f32acc(1, KB, QT);           // S^T, dP^T: M 128, N 64
      const uint32_t id_mn = tc::idesc_f32acc(1, KB, HD) | (1u << 16);  // dV, dK: N = d, B MN
      const uint32_t id_dq = tc::idesc_f32acc(1, QT, HD) | (1u << 15) | (1u << 16);  // M 64
      const uint32_t sK = tc::smem_u32(Kp), sS = tc::smem_u32(dSp);
      // S^T (the forward's product order) and dP^T (A: V's parts in TMEM) of tile n, committed
      // one by one: the compute warps form P^T while dP^T runs.
      auto issue_t1 = [&](int n) {
        const uint32_t sQ = tc::smem_u32(Qp + (n & 1) * 3 * PART_Q);
        const uint32_t sO = tc::smem_u32(dOp + (n & 1) * 3 * PART_Q);
        issue6<KSD, PART_K, PART_Q, 256, 256, true>(tbase + T_S,
                                                  tc::split_desc(tc::desc_kmajor(sK, 128, 1024)),
                                                  tc::split_desc(tc::desc_kmajor(sQ, 128, 1024)), id128);
        tc::commit_warp(bar_s);
        auto vcol = [&](int i, int ks) { return tbase + T_V + 32 * i + 8 * ks; };
        issue6_tmem_a<PART_Q, 256, decltype(vcol), KSD>(
            tbase + T_DP, vcol, tc::split_desc(tc::desc_kmajor(sO, 128, 1024)), id128);
        tc::commit_warp(bar_dp);
      };
      // dV (A: P^T's parts in TMEM) of tile n: it runs while the compute warps form dS^T.
      auto issue_dv = [&](int n) {
        const uint32_t sO = tc::smem_u32(dOp + (n & 1) * 3 * PART_Q);
        issue6_tmem_a<PART_Q, 2048>(tbase + T_DV, [&](int i, int ks) { return tbase + pt_col(i, ks); },
                                    tc::split_desc(tc::desc_kmajor(sO, 1024, 128)), id_mn);
        tc::commit_warp(bar_dv);
      };
      // dK, dQ (two windows of 64 keys) of tile n.
      auto issue_t2 = [&](int n) {
        const uint32_t sQ = tc::smem_u32(Qp + (n & 1) * 3 * PART_Q);
        issue6<4, PART_K, PART_Q, 256, 2048, false>(tbase + T_DK,
                                                    tc::split_desc(tc::desc_kmajor(sS, 128, 1024)),
                                                    tc::split_desc(tc::desc_kmajor(sQ, 1024, 128)), id_mn);
        const tc::Desc as_mn = tc::split_desc(tc::desc_kmajor(sS, 1024, 128));
        const tc::Desc bk_mn = tc::split_desc(tc::desc_kmajor(sK, 1024, 128));
        issue6<4, PART_K, PART_K, 2048, 2048, false>(tbase + T_DQ0, as_mn, bk_mn, id_dq);
        issue6<4, PART_K, PART_K, 2048, 2048, false>(
            tbase + T_DQ1, {as_mn.lo + (8192 >> 4), as_mn.hi}, {bk_mn.lo + (8192 >> 4), bk_mn.hi},
            id_dq);
        tc::commit_warp(bar_t2);
      };
      // The tensor core's order: S^T(n), dP^T(n), dV(n) once P^T(n) is in TMEM, dK(n), dQ(n)
      // once dS^T(n) is in shared memory, then S^T(n + 1) -- over P^T(n)'s columns, once dV(n) has
      // completed -- and dP^T(n + 1), queued behind dK(n), dQ(n).
      issue_t1(0);
      for (int n = 0; n < N; ++n) {
        err |= !tc::mbar_wait(bar_p, n & 1, WAIT_TIMEOUT_NS);
        tc::fence_after_sync();
        issue_dv(n);
        err |= !tc::mbar_wait(bar_c1, n & 1, WAIT_TIMEOUT_NS);  // dP^T(n) read, dS^T(n) stored
        tc::fence_after_sync();
        issue_t2(n);
        if (n + 1 < N) {
          err |= !tc::mbar_wait(bar_q, n & 1, WAIT_TIMEOUT_NS);
          err |= !tc::mbar_wait(bar_dv, n & 1, WAIT_TIMEOUT_NS);  // dV(n) has read P^T(n)
          tc::fence_after_sync();
          issue_t1(n + 1);
        }
      }
    }
  } else {
    if (N > 1) stage_tile(1);  // while the MMA warp issues T1(0)
    cp_async_commit();
    for (int n = 0; n < N; ++n) {
      const int q0 = (t_begin + n) * QT;
      // (C1a) P^T for this thread's 16 queries, its parts into TMEM (pt_col) for dV -- while the
      // tensor core computes dP^T.
      err |= !tc::mbar_wait(bar_s, n & 1, WAIT_TIMEOUT_NS);
      tc::fence_after_sync();
      const float* Lt = ld + (n & 1) * 128;
      const float* Dt = Lt + QT;
      const bool edge = (q0 + QT > rows) || (k0 + KB > SK);
      float pr[16];
      tc::tmem_ld16(tbase + lane_sel + T_S + 16 * cg, pr);
      tc::tmem_wait_ld();
      // Two halves of 8 queries, each half's parts stored (columns 4 h .. 4 h + 3 of its K-step)
      // while the next half is formed: the stores' latency no longer trails the arithmetic.
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
#pragma unroll
        for (int u = 8 * hh; u < 8 * hh + 8; u += 2) {
          const int ql = 16 * cg + u;
          // P = e^(s * scale - L): the argument with one rounding (L - s scale by one fma, so the
          // cancellation is exact), then 2^(arg log2 e) on the SFU (ex2.approx, max relative
          // error about 2^-22). Pairs of queries in packed fp32.
          const uint64_t l2 = *reinterpret_cast<const uint64_t*>(Lt + ql);
          float x0, x1;
          tc::unpack2(mul2(fma2v(tc::pack2(pr[u], pr[u + 1]), nsc2, l2), nl2e2), x0, x1);
          float p0 = ex2(x0), p1 = ex2(x1);
          if (edge) {
            if (!(q0 + ql < rows && key < SK)) p0 = 0.0f;
            if (!(q0 + ql + 1 < rows && key < SK)) p1 = 0.0f;
          }
          pr[u] = p0;
          pr[u + 1] = p1;
        }
        const float xh[8] = {pr[8 * hh], pr[8 * hh + 1], pr[8 * hh + 2], pr[8 * hh + 3],
                             pr[8 * hh + 4], pr[8 * hh + 5], pr[8 * hh + 6], pr[8 * hh + 7]};
        uint4 h0, h1, h2;
        split8(xh, h0, h1, h2);
        tc::tmem_st4(tbase + lane_sel + pt_col(0, cg) + 4 * hh, h0);
        tc::tmem_st4(tbase + lane_sel + pt_col(1, cg) + 4 * hh, h1);
        tc::tmem_st4(tbase + lane_sel + pt_col(2, cg) + 4 * hh, h2);
      }
      tc::tmem_wait_st();
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(bar_p);
      // (C1b) dS^T = P^T o (dP^T - D), its parts into shared memory for dK, dQ -- while the tensor
      // core computes dV.
      err |= !tc::mbar_wait(bar_dp, n & 1, WAIT_TIMEOUT_NS);
      tc::fence_after_sync();
#pragma unroll
      for (int h8 = 0; h8 < 2; ++h8) {
        const uint32_t col = 16 * cg + 8 * h8;
        float gb[8];
        tmem_ld8(tbase + lane_sel + T_DP + col, gb);
        tc::tmem_wait_ld();
        float ds[8];
#pragma unroll
        for (int u = 0; u < 8; u += 2) {
          const uint64_t d2 = *reinterpret_cast<const uint64_t*>(Dt + col + u);
          tc::unpack2(mul2(tc::pack2(pr[8 * h8 + u], pr[8 * h8 + u + 1]),
                           tc::sub2(tc::pack2(gb[u], gb[u + 1]), d2)),
                      ds[u], ds[u + 1]);
        }
        store_parts(dSp, PART_K, kmaj_off(row, 2 * cg + h8), ds);
      }
      tc::fence_async_smem();
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(bar_c1);
      // (C3) The next tile's Q, dO into their parts (its buffer was last read by T2(n - 1)), while
      // the tensor core computes dV, dK, dQ; the tile after it travels.
      if (n + 1 < N) {
        cp_async_wait_all();
        bar_sync(1, NT);  // L, D of tile n + 1 in place; every thread is past C1(n)
        split_tile(n + 1);
        tc::fence_async_smem();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(bar_q);
        if (n + 2 < N) stage_tile(n + 2);
        cp_async_commit();
      }
      // (C2) Fold dV, dK; write the dQ partial.
      err |= !tc::mbar_wait(bar_t2, n & 1, WAIT_TIMEOUT_NS);
      tc::fence_after_sync();
      float xb[16], xs[16];
      tc::tmem_ld16(tbase + lane_sel + T_DV + 16 * cg, xb);
      tc::tmem_ld16(tbase + lane_sel + T_DK + 16 * cg, xs);
      tc::tmem_wait_ld();
      if (16 * cg < HD) {  // dV, dK have HD columns
#pragma unroll
        for (int c = 0; c < 16; ++c) {
          dv[c] += xb[c];
          dk[c] += xs[c];
        }
      }
      // dQ (M = 64): query row 16 (w % 4) + lane in lanes 0-15 of each quarter; the two windows.
      tc::tmem_ld16(tbase + lane_sel + T_DQ0 + 16 * cg, xb);
      tc::tmem_ld16(tbase + lane_sel + T_DQ1 + 16 * cg, xs);
      tc::tmem_wait_ld();
      const int x = q0 + 16 * (w & 3) + lane;
      const bool mine = lane < 16 && x < rows && 16 * cg < HD;
      int head, qi;
      query_of(mine ? x : 0, head, qi);
      if (!chain) {
        if (mine && !err) {
          // Two 32-byte stores: whole L2 sectors (16-byte stores 256 bytes apart across the warp
          // each wrote half of 16 sectors).
          float* dst = a.dq_part +
                       (((static_cast<int64_t>(b) * a.H + head) * a.n_kblocks + kb) * S + qi) * HD + 16 * cg;
#pragma unroll
          for (int c8 = 0; c8 < 2; ++c8) {
            float v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = xb[8 * c8 + u] + xs[8 * c8 + u];
            st_cg_v8(dst + 8 * c8, v);
          }
        }
      } else {
        // Turn chain: key blocks 0 .. last each add their partial into dQ on their turn, through L2
        // (__ldcg / __stcg), and the last multiplies by `scale`: dQ = ((p0 + p1) + ...) * scale, the
        // partials' sums bit for bit.
        const int t = t_begin + n;
        const int last = nkb - 1;
        bool go = true;
        if (kb > 0) {
          if (tid == 0) {
            // (slot by tile parity: a thread may still read the last tile's flag)
            s_int[2 + (n & 1)] = wait_turn_bounded(turn + t, kb, a.err, a.timeout_ns, a.sink) ? 1 : 0;
            // ORDER: with the barrier below, extends thread 0's acquire to the compute warps.
            __threadfence();
          }
          bar_sync(1, NT);
          go = s_int[2 + (n & 1)] != 0;
        }
        if (go && mine) {
          float4* dst = reinterpret_cast<float4*>(
              a.dq + ((static_cast<int64_t>(b) * S + qi) * a.H + head) * HD + 16 * cg);
#pragma unroll
          for (int c4 = 0; c4 < 4; ++c4) {
            float4 v = make_float4(xb[4 * c4] + xs[4 * c4], xb[4 * c4 + 1] + xs[4 * c4 + 1],
                                   xb[4 * c4 + 2] + xs[4 * c4 + 2], xb[4 * c4 + 3] + xs[4 * c4 + 3]);
            if (kb > 0) {
              const float4 prev = __ldcg(dst + c4);
              v = make_float4(prev.x + v.x, prev.y + v.y, prev.z + v.z, prev.w + v.w);
            }
            if (kb == last) v = make_float4(v.x * dscale, v.y * dscale, v.z * dscale, v.w * dscale);
            __stcg(dst + c4, v);
          }
        }
        err |= !go;
        if (kb < last) {
          // ORDER: every thread's dQ stores are visible GPU-wide before thread 0 hands the tile to
          // key block kb + 1 (its acquire in wait_turn_bounded).
          __threadfence();
          bar_sync(1, NT);
          if (tid == 0) st_release_gpu(turn + t, kb + 1);
        }
      }
    }
  }
  cp_async_wait_all();
  err = __syncthreads_or(err);  // any expired wait in the block: nothing is written
  if (err) {
    if (tid == 0) flag_timeout(a.err, a.sink);
    tc::mbar_wait(bar_t2, (N - 1) & 1, WAIT_TIMEOUT_NS);  // no MMA left in flight
  } else {
    // The dQ partials' hand-off: after the barrier above, thread 0's acquire-release count
    // publishes every thread's partial stores (the barrier orders them before it) and, for the
    // last of the (b, h)'s key blocks, makes the other blocks' visible; that block sums them in
    // key-block order (the loads bypass L1).
    // dV and dK * scale go through shared memory (the dS^T and staging buffers, free since the last
    // T2): rows of 68 floats (a 16-byte rotation per
    // row keeps both passes conflict-free), stored as whole rows at the end.
    constexpr int LDS = 68;
    float* sv = reinterpret_cast<float*>(dSp);
    float* sk = sv + KB * LDS;
    static_assert(2 * KB * LDS * 4 <= 3 * PART_K + 2 * QT * 64 * 4, "dV, dK rows fit");
    if (!mma_warp) {
#pragma unroll
      for (int c4 = 0; c4 < 4; ++c4) {
        reinterpret_cast<float4*>(sv + row * LDS + 16 * cg)[c4] =
            make_float4(dv[4 * c4], dv[4 * c4 + 1], dv[4 * c4 + 2], dv[4 * c4 + 3]);
        reinterpret_cast<float4*>(sk + row * LDS + 16 * cg)[c4] =
            make_float4(dk[4 * c4] * dscale, dk[4 * c4 + 1] * dscale, dk[4 * c4 + 2] * dscale,
                        dk[4 * c4 + 3] * dscale);
      }
    }
    __syncthreads();  // the dV, dK rows in place
    constexpr int C4 = HD / 4;  // float4 columns of a dQ, dK or dV row
    // Thread 0's count -- an acquire-release round trip through L2 -- travels while the block
    // stores the dV, dK rows.
    int count = -1;
    if (tid == 0 && !chain && !a.join_dq) count = atom_add_acq_rel(a.turn + bh, 1);
    // dV, dK rows out of shared memory: every 16 threads store one whole row.
    {
      for (int f = tid; f < 2 * KB * C4; f += NB) {
        const int which = f / (KB * C4), r = (f / C4) % KB, c4 = f % C4;
        if (k0 + r < a.Sk) {  // (rows past the length hold zeros)
          float* dst = dkv + (static_cast<int64_t>(b) * a.Sk + k0 + r) * 2 * a.Hk * HD +
                       (1 - which) * a.Hk * HD + h * HD;
          reinterpret_cast<float4*>(dst)[c4] =
              reinterpret_cast<const float4*>((which ? sk : sv) + r * LDS)[c4];
        }
      }
    }
    if (tid == 0) s_int[0] = count;
    __syncthreads();
    const int64_t part_bytes = static_cast<int64_t>(nkb) * S * HD * 4;
    const int64_t row_stride = static_cast<int64_t>(a.H) * HD;  // dq floats per (b, s)
    auto sum_partials = [&](const float* part, float* dq_out) {
      if (part_bytes <= OFF_DS) {
        // The (b, h)'s partials, contiguous [nkb][S][64], as one bulk copy into shared memory (the
        // part buffers, free since the last T2; the dS^T buffer holds dV, dK), then summed there.
        const float* sp = reinterpret_cast<const float*>(sm);
        if (tid == 0) {
          tc::fence_async_global();  // the partials the count made visible, for the copy engine
          tc::mbar_arrive_expect_tx(bar_ld, static_cast<uint32_t>(part_bytes));
          tc::bulk_load(sm, part, static_cast<uint32_t>(part_bytes), bar_ld);
        }
        const bool ok = tc::mbar_wait(bar_ld, ld_phase & 1, WAIT_TIMEOUT_NS);
        // DETERMINISM: dQ = (((p0 + p1) + p2) + ...) * scale, as below.
        for (int idx = tid; idx < S * C4 && ok; idx += NB) {
          const int i = idx / C4, c4 = idx % C4;
          const int last = nkb - 1;
          float4 v = reinterpret_cast<const float4*>(sp + i * HD)[c4];
          for (int j = 1; j <= last; ++j) {
            const float4 q = reinterpret_cast<const float4*>(sp + (j * S + i) * HD)[c4];
            v = make_float4(v.x + q.x, v.y + q.y, v.z + q.z, v.w + q.w);
          }
          reinterpret_cast<float4*>(dq_out + i * row_stride)[c4] =
              make_float4(v.x * dscale, v.y * dscale, v.z * dscale, v.w * dscale);
        }
        if (!ok && tid == 0) flag_timeout(a.err, a.sink);
        return;
      }
      // DETERMINISM: dQ = (((p0 + p1) + p2) + ...) * scale over the key blocks. Eight float4 items per thread at a time, each key
      // block's loads for the eight issued together.
      constexpr int U = 8;
      const int items = S * C4;
      for (int base = tid; base < items; base += U * NB) {
        float4 v[U];
        int last[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int idx = base + u * NB;
          const int i = idx / C4;
          last[u] = idx < items ? nkb - 1 : -1;
          v[u] = last[u] >= 0
                     ? __ldcg(reinterpret_cast<const float4*>(part + static_cast<int64_t>(i) * HD) +
                              (idx % C4))
                     : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        for (int j = 1; j < nkb; ++j) {
          float4 p[U];
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int idx = base + u * NB;
            p[u] = j <= last[u] ? __ldcg(reinterpret_cast<const float4*>(
                                             part + (static_cast<int64_t>(j) * S + idx / C4) * HD) +
                                         (idx % C4))
                                : make_float4(0.f, 0.f, 0.f, 0.f);
          }
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (j <= last[u]) v[u] = make_float4(v[u].x + p[u].x, v[u].y + p[u].y, v[u].z + p[u].z,
                                                 v[u].w + p[u].w);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int idx = base + u * NB;
          if (last[u] >= 0)
            reinterpret_cast<float4*>(dq_out + (idx / C4) * row_stride)[idx % C4] =
                make_float4(v[u].x * dscale, v[u].y * dscale, v[u].z * dscale, v[u].w * dscale);
        }
      }
    };
    if (s_int[0] == nkb - 1) {  // (without join_dq there is one part)
      // Head by head of the group, the partials of a head a.n_kblocks apart.
      for (int hq = h0; hq < h0 + group; ++hq) {
        sum_partials(a.dq_part + (static_cast<int64_t>(b) * a.H + hq) * a.n_kblocks * S * HD, a.dq + static_cast<int64_t>(b) * S * row_stride + hq * HD);
        ++ld_phase;
        __syncthreads();  // this head's sums are read: the next one's partials may land
      }
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  if (mma_warp) tc::tmem_dealloc(tbase, TMEM_COLS);
}

}  // namespace

cudaError_t setup_cross_bwd_tc_attributes() {
  const cudaError_t e = cudaFuncSetAttribute(cross_bwd_tc_kernel<64>,
                                             cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_ALLOC);
  return e != cudaSuccess ? e
                          : cudaFuncSetAttribute(cross_bwd_tc_kernel<32>,
                                                 cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_ALLOC);
}

cudaError_t launch_cross_bwd_tc(const BwdArgs& args, int head_dim, cudaStream_t stream) {
  BwdArgs a = args;
  a.n_kblocks = (a.Sk + KB - 1) / KB;
  int dev = 0, sms = 0;  // one block per SM: a wave is the SM count
  a.wave_ctas = cudaGetDevice(&dev) == cudaSuccess &&
                        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess
                    ? sms
                    : 0;
  const int64_t blocks = static_cast<int64_t>(a.n_kblocks) * a.B * a.Hk * a.n_parts;
  const dim3 grid(static_cast<unsigned>(blocks));
  const cudaError_t e =
      head_dim == 32 ? launch_pdl(cross_bwd_tc_kernel<32>, grid, dim3(NB), SMEM_ALLOC, stream, a)
                     : launch_pdl(cross_bwd_tc_kernel<64>, grid, dim3(NB), SMEM_ALLOC, stream, a);
  return e == cudaSuccess ? launch_cross_join(a, head_dim, KB, stream) : e;
}

}  // namespace cfa
