// SPDX-License-Identifier: MIT OR Apache-2.0
//
// Attention of few query rows over many keys, split over the keys and joined: paged_attention (one
// or a few new tokens over a paged cache) and cross_attention's few-row form (a dense operand).
//
//   o = sum_j e^(y_j - m) v_j / sum_j e^(y_j - m),  y_j = scale q k_j,  m = max_j y_j
//
// over the keys a row sees. A sequence's keys are cut into chunks (split_chunk: by its own length
// alone); a block forms one chunk's (m_c, l_c, o_c) for the rows that share a key head, and a second
// kernel joins the chunks in order: m = max m_c, l = sum e^(m_c - m) l_c, o = sum e^(m_c - m) o_c / l.
// A sequence of one chunk is written by the first kernel.
//
// Bound by memory: every key and value is read once for all the query rows of its head (up to 8 or 16
// a block), at 4 rows D flops a key against 2 D elements. Each warp runs on its own: it takes every
// fourth 8 KB tile of the chunk through a ring of its own (cp.async, 16 bytes a lane, rows padded by
// 16 bytes or their pieces exchanged, so that every later read is free of bank conflicts), and the four
// warps' sums are joined through shared memory once a chunk. The ring runs on through a block's chunks: a ring that drained
// at the end of each took 204 us where this takes 199.
//   16-bit caches, up to 8 query rows: S^T = K Q^T and O^T += V^T P^T by mma.m16n8k16, the keys (dims)
//     as the 16 rows and the query rows as the 8 columns: a column's softmax state then lives in the lanes
//     that hold the column's output. fp32 queries enter in parts that keep their 24 bits (three
//     bf16, or two fp16 under a power of two a row: 22 bits), p as three parts over bf16 (24 bits) or
//     two over fp16 (22; P_UP_F16), every tile's product a fresh accumulator
//     folded by an fp32 FMA -- the tensor core's truncating sums never run longer than a tile. (p in two
//     bf16 parts for bf16 outputs: 192.4 us where three take 195.8, but 0.19 % of the outputs are then not
//     the bf16 number nearest the exact one, with three 0.016 %.)
//     tcgen05 has no shape below 64 rows, and at a few rows the product is a small share of the
//     tile's load time. Three stages of two blocks a SM (two of three blocks: 245 us for 204).
//   16-bit caches, more rows: S = Q K^T and O += P V, 16 query rows as the 16 rows; the same parts, but p in
//     two (16 bits) for bf16 outputs, whose own rounding is 2^-9: bound by the products' issue, a third part
//     takes 16 rows bf16 from 56 to 65 us (d 64) and from 81 to 94 (d 128), for 0.21 % and 0.024 % of outputs
//     that are not the nearest. In blocks of 8 and of 16, 32 sequences of 100 to 8000 keys, four key heads,
//     in us: 16 rows bf16 69 and 56 (d 64), 113 and 81 (d 128), fp32 over bf16 75 and 68, 131 and 98; 40 rows
//     bf16 d 128 270 and 209. Bound by the issue of the products and the softmax, two warps a scheduler.
//   fp32 caches, three query rows and more: S = Q K^T and O += P V by mma.m16n8k8 on tf32 operands, 8 or
//     16 query rows as the 16 rows. Every operand enters in two parts of 11 bits (x = hi + lo to 2^-22
//     |x|; three or all four of the products of the parts), and dims and keys are numbered within a
//     product so that a lane reads K and V 16 bytes at a time and P's fragment is S's. Three stages of
//     two blocks a SM; bound by the issue of the splits and products at 16 rows.
//   fp32 caches, one or two rows (where no log-sum-exp is asked for): 32 D / 1024 lanes a key for the scores,
//     four dims a lane for the output, p through shared memory; packed FMAs. Two stages of three blocks a SM.
//     By FMAs and by products, 32 sequences of 100 to 8000 keys, four key heads, in us: one row 61 and
//     64 (d 64), 107 and 120 (d 128), two rows 63 and 65, 115 and 121, four rows 79 and 66, 148 and 125,
//     eight rows 121 and 67, 241 and 129; 16 rows, in blocks of 8 and of 16: 222 and 92, 461 and 171; one
//     row of 64 sequences over 240 keys 11.7 and 16. (Training takes the products: the backward's scores.)
// On one B200, with the join: 64 sequences of up to 8192 keys, 32 heads over 8, [page 16] bf16, d = 128
// 196 us (5.7 TB/s); 2 of 131071 keys, fp32 over bf16, d = 64 55 us; 16 of 1000 to 6000 keys, 16 heads,
// fp32, d = 64 79 us (5.9 TB/s). One sequence of 240 keys: 6.9 us.
//
// Order of summation: fixed by the sequence's length, the number of rows and the row alone (not by the
// batch, the grid or the SM count): results are bit-identical across reruns and batches.
//
// Masked keys are excluded rather than weighted by zero, so what lies behind a sequence's end or a
// row's last key -- infinities and NaN among it -- never reaches a result. A page id outside the
// pool is reported through the page sink and its keys are left out.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>
#include <type_traits>

#include "cfa_common.cuh"
#include "cfa_ops.h"
#include "cfa_split.cuh"
#include "cfa_tc.cuh"
#include "tf32.cuh"

namespace cfa {
namespace {

constexpr int WARPS = 4;
constexpr int NT = 32 * WARPS;
constexpr int MAXR = 16;   // most query rows per block
constexpr float LOG2E = 1.4426950408889634f;
// fp16 caches: p, and with it the sums l and o, carries this factor, which o / l drops (no log-sum-exp is
// written there). p's two fp16 parts then keep 22 bits from p = 2^-17 on and miss at most 2^-39 below; without
// it the small part is subnormal below p = 2^-3 and the large one below 2^-14, both miss 2^-25, and a tail of
// weights near 1e-7 beside one large weight counts in l but not in o.
constexpr float P_UP_F16 = 16384.0f;

// Keys per chunk, as a power of two, of a sequence of `len` keys in tiles of 2^tile_log keys: 16 tiles
// (four a warp, 128 KB of keys and values) up to 16 chunks, then 32 tiles up to 256 chunks, then as many
// as keep them 256. (64 sequences of up to 8192 keys, at 204 us so: 279 and 256 us with chunks of 64 and
// 128 keys throughout, 225 with the step at 32, 64 or 256 chunks.)
constexpr int FEW_CHUNKS_LOG = 4, MOST_CHUNKS_LOG = 8, MOST_CHUNKS = 1 << MOST_CHUNKS_LOG;
__host__ __device__ __forceinline__ int bits_of(uint32_t x) {  // x < 2^bits
#ifdef __CUDA_ARCH__
  return 32 - __clz(x);
#else
  return x ? 32 - __builtin_clz(x) : 0;
#endif
}
__host__ __device__ __forceinline__ int chunk_log(int len, int tile_log) {
  const int few = tile_log + 4;
  if (len <= 1 << (few + FEW_CHUNKS_LOG)) return few;
  const int need = bits_of(static_cast<uint32_t>(len - 1)) - MOST_CHUNKS_LOG;
  return need > few + 1 ? need : few + 1;
}
__host__ __device__ __forceinline__ int chunks_of(int len, int tile_log) {
  if (len <= 0) return 1;  // one empty chunk: its block writes the zeros
  const int c = chunk_log(len, tile_log);
  return static_cast<int>((static_cast<uint32_t>(len) + (1u << c) - 1) >> c);
}

template <typename T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f(float x) { return __float2bfloat16_rn(x); }

__device__ __forceinline__ int seq_len(const SplitArgs& a, int b) {
  return a.lengths ? min(max(a.lengths[b], 0), a.max_len) : a.max_len;
}
__device__ __forceinline__ int seq_new(const SplitArgs& a, int b) {
  return a.new_lengths ? min(max(a.new_lengths[b], 0), a.S) : a.S;
}

// The chunks of the batch in order: each lane holds its share of the sequences (a contiguous range)
// and the chunks before and in it.
struct ChunkIndex {
  int first, per, before, count, total;
  __device__ __forceinline__ void init(const SplitArgs& a, int lane) {
    per = (a.B + 31) / 32;
    first = lane * per;
    count = 0;
    for (int i = first; i < min(first + per, a.B); ++i) {
      count += chunks_of(seq_len(a, i), a.tile_log);
      if (a.table && blockIdx.x == 0 && a.lengths[i] > a.max_len) flag_error(a.sink, CFA_ERR_PAGE);
    }
    int incl = count;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += x;
    }
    before = incl - count;
    total = __shfl_sync(0xffffffffu, incl, 31);
  }
  // Chunk g of the batch (g < total): its sequence, chunk in the sequence, chunks of it.
  __device__ __forceinline__ void find(const SplitArgs& a, int g, int& b, int& c, int& nc) const {
    const unsigned in = __ballot_sync(0xffffffffu, g >= before && g < before + count);
    const int owner = __ffs(in) - 1;
    b = __shfl_sync(0xffffffffu, first, owner);
    c = g - __shfl_sync(0xffffffffu, before, owner);
    nc = chunks_of(seq_len(a, b), a.tile_log);
    while (c >= nc) {
      c -= nc;
      nc = chunks_of(seq_len(a, ++b), a.tile_log);
    }
  }
};

// What a block knows of its unit.
struct UnitInfo {
  int b, hk, r0, chunk, nc, len, n_new, lo, hi;  // rows r0 .., keys lo .. hi - 1
};
__device__ __forceinline__ UnitInfo unit_info(const SplitArgs& a, const ChunkIndex& ix, uint32_t u) {
  UnitInfo n;
  const uint32_t per = a.Hk * a.row_chunks;
  const int g = static_cast<int>(u / per), rest = static_cast<int>(u - g * per);
  n.hk = rest / a.row_chunks;
  n.r0 = (rest - n.hk * a.row_chunks) * a.block_rows;
  ix.find(a, g, n.b, n.chunk, n.nc);
  n.len = seq_len(a, n.b);
  n.n_new = seq_new(a, n.b);
  const int c = chunk_log(n.len, a.tile_log);
  n.lo = n.chunk << c;
  n.hi = n.len - n.lo > 1 << c ? n.lo + (1 << c) : n.len;
  return n;
}
// A 16-byte asynchronous copy past L1 (the rows are read once).
__device__ __forceinline__ void cp_async16_full(void* smem, const void* gmem) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(tc::smem_u32(smem)), "l"(gmem)
               : "memory");
}

// One warp's ring of tiles: TK rows of K, then of V, RB bytes apart, a stage a tile. Each lane copies
// the 16-byte piece `lane % CPR` of every RPI-th row. The ring runs through the block's units (u, u +
// grid, ..) and, in each, the warp's tiles (w, w + 4, ..) without a pause: ST - 1 tiles are in flight
// while one is in use, those of the next unit behind the last of this one, and a unit's index and
// first page are looked up an iteration before they are needed.
template <int D, int ES, int TK_, int ST_, bool SWIZZLE>
struct Ring {
  static constexpr int ST = ST_;   // stages
  static constexpr int TK = TK_;   // keys per tile
  static constexpr int RB = D * ES + (SWIZZLE ? 0 : 16);
  static constexpr int KV = TK * RB;          // bytes of a tile's K (or V)
  static constexpr int STAGE = 2 * KV;
  static constexpr int CPR = D * ES / 16;     // 16-byte pieces of a row
  static constexpr int RPI = 32 / CPR;        // rows that the warp copies at once
  static constexpr int BYTES = ST * STAGE;
  static constexpr unsigned ALL = 0xffffffffu >> (32 - TK);

  // SWIZZLE: the piece c of row r of K, V is piece c ^ this of its row, by which the eight lanes of a
  // 16-byte read meet eight banks of 16 bytes (fp32: two rows of K, four pieces; every other row of eight
  // of V, two pieces; 16-bit: one piece of eight rows). Else rows are padded by 16 bytes.
  static __device__ __forceinline__ int k_swizzle(int r) {
    return !SWIZZLE ? 0 : ES == 4 ? 4 * (r & 1) : CPR == 4 ? (r >> 1) & 3 : r & 7;
  }
  static __device__ __forceinline__ int v_swizzle(int r) {
    return SWIZZLE && ES == 4 ? 2 * ((r >> 1) & 3) : k_swizzle(r);
  }

  const SplitArgs& a;
  const ChunkIndex& ix;
  unsigned char* base;
  int lane, w;
  uint32_t units, unit;    // all of them; the one being loaded
  UnitInfo info;           // (of unit)
  int64_t k_lane, v_lane;  // this lane's first row and piece within a tile, in bytes
  const char* kp;          // this (batch, key head)'s keys and values
  const char* vp;
  const int* table;
  int tiles, next, pg;  // of the unit: its tiles; the next one, its page
  unsigned live[ST];    // the live keys of the tiles in flight, oldest first
  bool bad = false;

  __device__ __forceinline__ Ring(const SplitArgs& a_, const ChunkIndex& ix_, uint32_t units_,
                                  unsigned char* base_, int lane_, int w_)
      : a(a_), ix(ix_), base(base_), lane(lane_), w(w_), units(units_), unit(blockIdx.x) {
    k_lane = (lane / CPR) * a.k_sr * ES + 16 * (lane % CPR);
    v_lane = (lane / CPR) * a.v_sr * ES + 16 * (lane % CPR);
    open();
#pragma unroll
    for (int s = 0; s < ST - 1; ++s) live[s] = issue(s);
  }
  // Looks up `unit`, or the first after it that has a tile for this warp.
  __device__ __forceinline__ void open() {
    for (; unit < units; unit += gridDim.x) {
      info = unit_info(a, ix, unit);
      tiles = (info.hi - info.lo + TK - 1) / TK;
      next = w;
      if (next < tiles) break;
    }
    if (unit >= units) return;
    kp = static_cast<const char*>(a.k) + ES * (info.hk * a.k_sh + (a.table ? 0 : info.b * a.k_sp));
    vp = static_cast<const char*>(a.v) + ES * (info.hk * a.v_sh + (a.table ? 0 : info.b * a.v_sp));
    table = a.table ? a.table + info.b * a.table_sb : nullptr;
    pg = page_of(next);
  }
  __device__ __forceinline__ int page_at(int key) const {  // key / a.page (key < 2^31)
    return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(key)) * a.page_mul) >> a.page_shift);
  }
  // The page of the next tile: of its first key, or (pages that end inside a tile) of this lane's
  // row. 0 where dense, -1 where there is none.
  __device__ __forceinline__ int page_of(int t) const {
    const int key = info.lo + TK * t + (a.one_page ? 0 : (lane & (TK - 1)));
    if (key >= info.hi) return -1;
    return table ? __ldg(table + page_at(key)) : 0;
  }
  // The oldest tile's live keys as bits; the tile after those in flight goes into `stage`.
  __device__ __forceinline__ unsigned advance(int stage) {
    const unsigned now = live[0];
#pragma unroll
    for (int s = 0; s + 1 < ST - 1; ++s) live[s] = live[s + 1];
    live[ST - 2] = issue(stage);
    return now;
  }
  __device__ __forceinline__ unsigned issue(int stage) {
    unsigned x = 0;
    if (unit < units) {
      const int k0 = info.lo + TK * next;
      x = a.one_page ? load_page(k0, stage, pg) : load_rows(k0, stage, pg);
      next += WARPS;
      if (next < tiles) {
        pg = page_of(next);
      } else {
        unit += gridDim.x;
        open();
      }
    }
    cp_async_commit();
    return x;
  }
  // A tile whose rows lie on one page (page sizes that are multiples of TK; a dense operand).
  __device__ __forceinline__ unsigned load_page(int k0, int stage, int p) {
    int rows = min(TK, info.hi - k0);
    int64_t ko = 0, vo = 0;
    if (!table) {
      ko = k0 * a.k_sr;
      vo = k0 * a.v_sr;
    } else if (p < 0 || p >= a.n_pages) {
      bad = true;
      rows = 0;
    } else {
      const int row = k0 - page_at(k0) * a.page;
      ko = p * a.k_sp + row * a.k_sr;
      vo = p * a.v_sp + row * a.v_sr;
    }
    const char* kg = kp + ES * ko + k_lane;
    const char* vg = vp + ES * vo + v_lane;
    unsigned char* st = base + stage * STAGE + (lane / CPR) * RB;
    const int ck = (lane % CPR) ^ k_swizzle(lane / CPR), cv = (lane % CPR) ^ v_swizzle(lane / CPR);
    const int64_t kj = RPI * ES * a.k_sr, vj = RPI * ES * a.v_sr;
    if (rows == TK) {
#pragma unroll
      for (int j = 0; j < TK / RPI; ++j) {
        cp_async16_full(st + j * RPI * RB + 16 * (ck ^ k_swizzle(j * RPI)), kg + j * kj);
        cp_async16_full(st + KV + j * RPI * RB + 16 * (cv ^ v_swizzle(j * RPI)), vg + j * vj);
      }
      return ALL;
    }
#pragma unroll
    for (int j = 0; j < TK / RPI; ++j) {  // rows past the end: zeros (from an address that exists)
      const bool ok = j * RPI + lane / CPR < rows;
      cp_async16(st + j * RPI * RB + 16 * (ck ^ k_swizzle(j * RPI)), ok ? kg + j * kj : kp, ok ? 16 : 0);
      cp_async16(st + KV + j * RPI * RB + 16 * (cv ^ v_swizzle(j * RPI)), ok ? vg + j * vj : vp, ok ? 16 : 0);
    }
    return (1u << rows) - 1;
  }
  // Any page size: lane r % TK finds row r's address, the copying lanes ask it for theirs.
  __device__ __forceinline__ unsigned load_rows(int k0, int stage, int p) {
    const int key = k0 + (lane & (TK - 1));
    bool ok = key < info.hi;
    int64_t ko = 0, vo = 0;
    if (ok && (p < 0 || p >= a.n_pages)) {
      ok = false;
      bad = true;
    }
    if (ok) {
      const int row = key - page_at(key) * a.page;
      ko = p * a.k_sp + row * a.k_sr;
      vo = p * a.v_sp + row * a.v_sr;
    }
    const unsigned alive = __ballot_sync(0xffffffffu, ok) & ALL;
    unsigned char* st = base + stage * STAGE;
    const int c = lane % CPR;
#pragma unroll
    for (int j = 0; j < TK / RPI; ++j) {
      const int r = j * RPI + lane / CPR;
      const int64_t kr = __shfl_sync(0xffffffffu, ko, r), vr = __shfl_sync(0xffffffffu, vo, r);
      const int n = (alive >> r) & 1u ? 16 : 0;
      cp_async16(st + r * RB + 16 * (c ^ k_swizzle(r)), kp + ES * kr + 16 * c, n);
      cp_async16(st + KV + r * RB + 16 * (c ^ v_swizzle(r)), vp + ES * vr + 16 * c, n);
    }
    return alive;
  }
};

template <int N>
__device__ __forceinline__ void cp_async_wait_group() {
  asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory");
}

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(tc::smem_u32(p))
               : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(tc::smem_u32(p))
               : "memory");
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
template <typename T>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same_v<T, __half>)
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// A pair of floats as the 16-bit type, the first low; and the pair it stands for.
template <typename T>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  if constexpr (std::is_same_v<T, __half>) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
template <typename T>
__device__ __forceinline__ float2 unpack16(uint32_t x) {
  if constexpr (std::is_same_v<T, __half>) return __half22float2(*reinterpret_cast<__half2*>(&x));
  else return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
}

// Row r of a key head's rows: query head r / S of the group, new token r % S.
__device__ __forceinline__ void row_of(const SplitArgs& a, int r, int& head, int& i) {
  head = a.S == 1 ? r : r / a.S;
  i = a.S == 1 ? 0 : r - head * a.S;
}
// The keys it sees (a row that is not there sees them all: its result is never written).
__device__ __forceinline__ int row_limit(const SplitArgs& a, const UnitInfo& n, int r) {
  int head, i;
  row_of(a, r, head, i);
  if (!a.causal || r >= a.rows || i >= n.n_new) return n.len;
  return min(max(n.len - n.n_new + i + 1, 0), n.len);
}

// Joins the four warps' sums of the block's first nr rows (warp w's: [row][D] at red + red_at[w]; ml:
// [warp][row]) and writes the chunk's partial result, or, the sequence's only chunk,
// the output.
template <typename QT, int D>
__device__ __forceinline__ void write_chunk(const SplitArgs& a, const UnitInfo& n,
                                            const unsigned char* red, const int* red_at,
                                            const float2* ml,
                                            int nr) {
  for (int idx = threadIdx.x; idx < nr * (D / 4); idx += NT) {
    const int r = idx / (D / 4), c4 = idx % (D / 4);
    const int row = n.r0 + r;
    if (row >= a.rows) continue;
    int head, i;
    row_of(a, row, head, i);
    head += n.hk * a.group;
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) m = fmaxf(m, ml[w * MAXR + r].x);
    float l = 0.0f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    const float mu = m == -INFINITY ? 0.0f : m;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float2 x = ml[w * MAXR + r];
      const float f = ex2((x.x - mu) * LOG2E);
      const float4 v = *reinterpret_cast<const float4*>(red + red_at[w] + (r * D + 4 * c4) * 4);
      l = fmaf(x.y, f, l);
      o.x = fmaf(v.x, f, o.x);
      o.y = fmaf(v.y, f, o.y);
      o.z = fmaf(v.z, f, o.z);
      o.w = fmaf(v.w, f, o.w);
    }
    if (n.nc == 1) {
      const bool live = i < n.n_new && l != 0.0f;  // no keys, or no such token: zeros
      QT* dst = static_cast<QT*>(a.o) + ((static_cast<int64_t>(n.b) * a.S + i) * a.H + head) * D + 4 * c4;
      dst[0] = from_f<QT>(live ? o.x / l : 0.0f);
      dst[1] = from_f<QT>(live ? o.y / l : 0.0f);
      dst[2] = from_f<QT>(live ? o.z / l : 0.0f);
      dst[3] = from_f<QT>(live ? o.w / l : 0.0f);
      if (a.lse && c4 == 0) a.lse[(static_cast<int64_t>(n.b) * a.H + head) * a.S + i] = m + logf(l);
    } else if (i < n.n_new) {
      const int64_t at = ((static_cast<int64_t>(n.b) * a.H + head) * a.S + i) * a.max_chunks + n.chunk;
      *reinterpret_cast<float4*>(a.part_o + at * D + 4 * c4) = o;
      if (c4 == 0) a.part_ml[at] = make_float2(m, l);
    }
  }
}

// Keys per tile (8 KB of keys and values for 16-bit caches at D = 64, 128 and for fp32) and the ring of
// a kernel.
template <int D, int ES>
__host__ __device__ constexpr int tile_keys() {
  return ES == 2 ? (D == 128 ? 16 : 32) : 1024 / D;  // (tile_log_of says the same to the host)
}
// ROWS: query rows of a block, 8 or 16 (fp32 caches: one or two by FMAs).
template <int D, int ES, int ROWS>
using RingOf = Ring<D, ES, tile_keys<D, ES>(), (ROWS <= 2 ? 2 : 3), (ES == 4 ? ROWS > 2 : ROWS == 16)>;
// Shared memory: the rings -- whose free stage also takes a warp's sums when a unit ends -- the (m, l)
// of the warps' rows and where their sums are, and two sets of query rows and p (FMAs) or the fragments
// of 16 rows (two parts of fp32, up to three of 16 bits).
template <int D, int ES, int ROWS>
__host__ __device__ constexpr int off_ml() {
  static_assert(RingOf<D, ES, ROWS>::STAGE >= ROWS * D * 4, "a stage holds a warp's sums");
  return WARPS * RingOf<D, ES, ROWS>::BYTES;
}
template <int D, int ES, int ROWS>
__host__ __device__ constexpr int off_q() {
  return off_ml<D, ES, ROWS>() + WARPS * MAXR * 8 + WARPS * 4;
}
template <int D, int ES, int ROWS>
__host__ __device__ constexpr int split_smem() {
  return off_q<D, ES, ROWS>() +
         (ROWS <= 2 ? ROWS * (2 * D * 4 + WARPS * tile_keys<D, ES>() * 8) : ROWS == 16 ? 16 * D * (ES == 4 ? 8 : 6) : 0);
}

// 16-bit caches.
template <typename QT, typename T, int D>
__global__ void __launch_bounds__(NT, 2)
    split_mma_kernel(const SplitArgs a) {
  using R = RingOf<D, 2, 8>;
  constexpr int ST = R::ST, TK = R::TK, MT = TK / 16;
  constexpr bool F32 = std::is_same_v<QT, float>;
  constexpr bool HALF = std::is_same_v<T, __half>;
  constexpr int QP = F32 ? (HALF ? 2 : 3) : 1;  // parts of q
  constexpr int PP = HALF ? 2 : 3;              // parts of p
  constexpr float P_UP = HALF ? P_UP_F16 : 1.0f;
  constexpr int KS = D / 16;
  using QPair = std::conditional_t<F32, float2, uint32_t>;
  extern __shared__ __align__(128) unsigned char smem[];
  const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31;
  const int qr = lane >> 2, qc = lane & 3;  // a fragment's row (key, dim; B: column) and pair
  float2* ml = reinterpret_cast<float2*>(smem + off_ml<D, 2, 8>());
  int* red_at = reinterpret_cast<int*>(ml + WARPS * MAXR);
  griddep_wait();
  griddep_launch_dependents();
  ChunkIndex ix;
  ix.init(a, lane);
  const uint32_t units = static_cast<uint32_t>(ix.total) * a.Hk * a.row_chunks;
  R ring(a, ix, units, smem + w * R::BYTES, lane, w);

  // Q^T's pairs of column qr: dims 16 ks + 2 qc, + 1 and + 8, + 9 (zeros where there is no row).
  QPair qx[KS][2];
  auto load_q = [&](const UnitInfo& n) {
    const int row = n.r0 + qr;
    int head, i;
    row_of(a, row, head, i);
    const bool ok = row < a.rows && i < n.n_new;
    const QT* q = static_cast<const QT*>(a.q) + n.b * a.q_sb +
                  (n.hk * a.group + (ok ? head : 0)) * a.q_sh + (ok ? i : 0) * a.q_ss;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        qx[ks][h] = ok ? *reinterpret_cast<const QPair*>(q + 16 * ks + 8 * h + 2 * qc) : QPair{};
  };
  UnitInfo n;
  if (blockIdx.x < units) {
    n = unit_info(a, ix, blockIdx.x);
    load_q(n);
  }
  int stage = 0;  // of the next tile; the stage before it is free
  for (uint32_t u = blockIdx.x; u < units; u += gridDim.x) {
    const int tiles = (n.hi - n.lo + TK - 1) / TK;
    // Q^T as B fragments.
    uint32_t qb[QP][KS][2];
    float qscale0 = a.scale, qscale1 = a.scale;  // of columns 2 qc, 2 qc + 1
    if constexpr (!F32) {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) qb[0][ks][0] = qx[ks][0], qb[0][ks][1] = qx[ks][1];
    } else if constexpr (HALF) {
      // q = 2^e (h0 + 2^-11 h1), |h0| <= 2: what the two parts miss is below 2^-24 of q, or
      // 2^-36 of the row's largest.
      float top = 0.0f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int h = 0; h < 2; ++h) top = fmaxf(top, fmaxf(fabsf(qx[ks][h].x), fabsf(qx[ks][h].y)));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      int e = top > 0.0f && top < INFINITY ? ilogbf(top) : 0;
      e = max(-120, min(120, e));
      const float down = ldexpf(1.0f, -e), up = ldexpf(1.0f, e);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float lo = qx[ks][h].x * down, hi = qx[ks][h].y * down;
          qb[0][ks][h] = pack16<T>(lo, hi);
          const float2 z = unpack16<T>(qb[0][ks][h]);
          qb[QP - 1][ks][h] = pack16<T>((lo - z.x) * 2048.0f, (hi - z.y) * 2048.0f);
        }
      qscale0 *= __shfl_sync(0xffffffffu, up, 8 * qc);
      qscale1 *= __shfl_sync(0xffffffffu, up, 8 * qc + 4);
    } else {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float2 y = qx[ks][h];
#pragma unroll
          for (int p = 0; p < QP; ++p) {
            qb[p][ks][h] = pack16<T>(y.x, y.y);
            const float2 z = unpack16<T>(qb[p][ks][h]);
            y = make_float2(y.x - z.x, y.y - z.y);
          }
        }
    }
    const int lim0 = row_limit(a, n, n.r0 + 2 * qc), lim1 = row_limit(a, n, n.r0 + 2 * qc + 1);
    // What the sequence's first new token sees, the fewest of all: a tile that ends behind it masks row by
    // row, in every block (a prompt's every tile: its value products are then issued once a row).
    const int lim_min = a.causal ? max(n.len - n.n_new + 1, 0) : n.len;

    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;
    float acc[KS][4];  // O^T: dims 16 mt + qr (+ 8), columns 2 qc, + 1
#pragma unroll
    for (int i = 0; i < KS; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = 0.0f;

    for (int t = w; t < tiles; t += WARPS) {
      cp_async_wait_group<ST - 2>();
      __syncwarp();  // the tile is in place for every lane, and the stage before it is free
      const unsigned char* kt = ring.base + stage * R::STAGE;
      const unsigned char* vt = kt + R::KV;
      const int k0 = n.lo + TK * t;

      // Scores: s[i][0], [1]: key 16 i + qr, columns 2 qc, + 1; s[i][2], [3]: key 16 i + qr + 8.
      float s[MT][4];
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const unsigned char* ka_at = kt + (16 * i + (lane & 15)) * R::RB + 16 * (lane >> 4);
        float c[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
        if constexpr (F32) {  // the small parts in a chain of their own, truncated at their magnitude
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) {
            uint32_t ka[4];
            ldsm4(ka, ka_at + 32 * ks);
#pragma unroll
            for (int p = QP - 1; p > 0; --p) mma<T>(c[1], ka, qb[p][ks][0], qb[p][ks][1]);
            mma<T>(c[0], ka, qb[0][ks][0], qb[0][ks][1]);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j)
            s[i][j] = (HALF ? fmaf(c[1][j], 1.0f / 2048.0f, c[0][j]) : c[1][j] + c[0][j]) *
                      (j & 1 ? qscale1 : qscale0);
        } else {  // two chains, half as long
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) {
            uint32_t ka[4];
            ldsm4(ka, ka_at + 32 * ks);
            mma<T>(c[ks & 1], ka, qb[0][ks][0], qb[0][ks][1]);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) s[i][j] = (c[0][j] + c[1][j]) * (j & 1 ? qscale1 : qscale0);
        }
      }
      // (behind the products: their latency hides the next loads' issue)
      const unsigned now = ring.advance(stage == 0 ? ST - 1 : stage - 1);
      const bool edge = lim_min < min(k0 + TK, n.hi);
      if (now != R::ALL || edge) {
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          const int ka = 16 * i + qr, kb = ka + 8;
          const bool la = (now >> ka) & 1u, lb = (now >> kb) & 1u;
          if (!la || k0 + ka >= lim0) s[i][0] = -INFINITY;
          if (!la || k0 + ka >= lim1) s[i][1] = -INFINITY;
          if (!lb || k0 + kb >= lim0) s[i][2] = -INFINITY;
          if (!lb || k0 + kb >= lim1) s[i][3] = -INFINITY;
        }
      }
      float t0 = fmaxf(s[0][0], s[0][2]), t1 = fmaxf(s[0][1], s[0][3]);
#pragma unroll
      for (int i = 1; i < MT; ++i) {
        t0 = fmaxf(t0, fmaxf(s[i][0], s[i][2]));
        t1 = fmaxf(t1, fmaxf(s[i][1], s[i][3]));
      }
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, o));
        t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, o));
      }
      t0 = fmaxf(t0, m0);
      t1 = fmaxf(t1, m1);
      const float u0 = t0 == -INFINITY ? 0.0f : t0, u1 = t1 == -INFINITY ? 0.0f : t1;
      const float a0 = ex2((m0 - u0) * LOG2E), a1 = ex2((m1 - u1) * LOG2E);
      m0 = t0;
      m1 = t1;
      // P^T as B fragments (transposed 8 x 8 blocks), in parts.
      uint32_t pb[MT][PP][2];
      float ps0 = 0.0f, ps1 = 0.0f;
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        float2 x = make_float2(ex2((s[i][0] - u0) * LOG2E) * P_UP, ex2((s[i][1] - u1) * LOG2E) * P_UP);
        float2 y = make_float2(ex2((s[i][2] - u0) * LOG2E) * P_UP, ex2((s[i][3] - u1) * LOG2E) * P_UP);
        ps0 += x.x + y.x;
        ps1 += x.y + y.y;
#pragma unroll
        for (int p = 0; p < PP; ++p) {
          const uint32_t hx = pack16<T>(x.x, x.y), hy = pack16<T>(y.x, y.y);
          if (p + 1 < PP) {
            const float2 zx = unpack16<T>(hx), zy = unpack16<T>(hy);
            x = make_float2(x.x - zx.x, x.y - zx.y);
            y = make_float2(y.x - zy.x, y.y - zy.y);
          }
          pb[i][p][0] = transpose8(hx);
          pb[i][p][1] = transpose8(hy);
        }
      }
      l0 = fmaf(l0, a0, ps0);
      l1 = fmaf(l1, a1, ps1);
      // The V^T block of dims 16 mt ..: rows (keys) (lane % 8) + 8 (lane / 16), dims + 8 (lane / 8 % 2).
      const unsigned char* va_at = vt + ((lane & 7) + 8 * (lane >> 4)) * R::RB + 16 * ((lane >> 3) & 1);
      if (!edge) {
#pragma unroll
        for (int mt = 0; mt < KS; ++mt) {
          float c[4] = {0.f, 0.f, 0.f, 0.f};
          uint32_t va[MT][4];
#pragma unroll
          for (int i = 0; i < MT; ++i) ldsm4t(va[i], va_at + 16 * i * R::RB + 32 * mt);
#pragma unroll
          for (int p = PP - 1; p >= 0; --p)
#pragma unroll
            for (int i = 0; i < MT; ++i) mma<T>(c, va[i], pb[i][p][0], pb[i][p][1]);
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[mt][j] = fmaf(acc[mt][j], j & 1 ? a1 : a0, c[j]);
        }
      } else {
        // Keys that only some of the rows see: one row at a time, the values it does not see as
        // zeros (0 times what they hold could be NaN).
#pragma unroll
        for (int mt = 0; mt < KS; ++mt)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[mt][j] *= j & 1 ? a1 : a0;
        for (int r = 0; r < min(8, a.rows - n.r0); ++r) {
          const int lim = row_limit(a, n, n.r0 + r);
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            const int k = k0 + 16 * i + 2 * qc;  // this lane's keys of an A fragment: k, + 1, + 8, + 9
            const uint32_t mlo = (k < lim ? 0xffffu : 0u) | (k + 1 < lim ? 0xffff0000u : 0u);
            const uint32_t mhi = (k + 8 < lim ? 0xffffu : 0u) | (k + 9 < lim ? 0xffff0000u : 0u);
#pragma unroll
            for (int mt = 0; mt < KS; ++mt) {
              uint32_t va[4];
              ldsm4t(va, va_at + 16 * i * R::RB + 32 * mt);
              va[0] &= mlo;
              va[1] &= mlo;
              va[2] &= mhi;
              va[3] &= mhi;
              float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
              for (int p = PP - 1; p >= 0; --p)
                mma<T>(c, va, qr == r ? pb[i][p][0] : 0u, qr == r ? pb[i][p][1] : 0u);
#pragma unroll
              for (int j = 0; j < 4; ++j)
                if (2 * qc + (j & 1) == r) acc[mt][j] += c[j];
            }
          }
        }
      }
      stage = stage + 1 == ST ? 0 : stage + 1;
    }
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) {
      l0 += __shfl_xor_sync(0xffffffffu, l0, o);
      l1 += __shfl_xor_sync(0xffffffffu, l1, o);
    }
    // The next unit's queries travel while this one's sums are joined.
    const UnitInfo done = n;
    const int free_at = w * R::BYTES + (stage == 0 ? ST - 1 : stage - 1) * R::STAGE;
    __syncwarp();  // every lane has read its last tile
    if (u + gridDim.x < units) {
      n = ring.unit == u + gridDim.x ? ring.info : unit_info(a, ix, u + gridDim.x);
      load_q(n);
    }
    if (lane == 0) red_at[w] = free_at;
    if (qr == 0) {
      ml[w * MAXR + 2 * qc] = make_float2(m0, l0);
      ml[w * MAXR + 2 * qc + 1] = make_float2(m1, l1);
    }
    float* sums = reinterpret_cast<float*>(smem + free_at);
#pragma unroll
    for (int mt = 0; mt < KS; ++mt)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        sums[(2 * qc + (j & 1)) * D + 16 * mt + qr + 8 * (j >> 1)] = acc[mt][j];
    __syncthreads();
    write_chunk<QT, D>(a, done, smem, red_at, ml, min(8, a.rows - done.r0));
    __syncthreads();  // the sums are read: their stages take tiles again
  }
  if (ring.bad) flag_error(a.sink, CFA_ERR_PAGE);
}

// 16-bit caches, up to 16 query rows a block as the 16 rows of the products: S = Q K^T, O += P V, the
// queries' fragments in shared memory, P's those of S.
template <typename QT, typename T, int D>
__global__ void __launch_bounds__(NT, 2) split_rows_kernel(const SplitArgs a) {
  using R = RingOf<D, 2, 16>;
  constexpr int ST = R::ST, TK = R::TK, MT = TK / 16, KS = D / 16;
  constexpr bool F32 = std::is_same_v<QT, float>;
  constexpr bool HALF = std::is_same_v<T, __half>;
  constexpr int QP = F32 ? (HALF ? 2 : 3) : 1;  // parts of q
  constexpr int PP = F32 && !HALF ? 3 : 2;      // parts of p
  constexpr float P_UP = HALF ? P_UP_F16 : 1.0f;
  constexpr int JQ = (KS + WARPS - 1) / WARPS;  // this warp's share of q's columns
  using QPair = std::conditional_t<F32, float2, uint32_t>;
  extern __shared__ __align__(128) unsigned char smem[];
  const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t4 = lane & 3;  // a fragment's row (B: column) and pair
  float2* ml = reinterpret_cast<float2*>(smem + off_ml<D, 2, 16>());
  int* red_at = reinterpret_cast<int*>(ml + WARPS * MAXR);
  uint4* qs = reinterpret_cast<uint4*>(smem + off_q<D, 2, 16>());  // [KS][part][lane]
  griddep_wait();
  griddep_launch_dependents();
  ChunkIndex ix;
  ix.init(a, lane);
  const uint32_t units = static_cast<uint32_t>(ix.total) * a.Hk * a.row_chunks;
  R ring(a, ix, units, smem + w * R::BYTES, lane, w);

  // Dims 16 ks + 2 t4, + 1 and + 8, + 9 of rows g and g + 8 (zeros where there is no row).
  QPair qx[JQ][2][2];
  float up[2];  // fp32 queries over fp16: a row's power of two
  auto load_q = [&](const UnitInfo& n) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = n.r0 + g + 8 * h;
      int head, i;
      row_of(a, row, head, i);
      const bool ok = row < a.rows && i < n.n_new;
      const QT* q = static_cast<const QT*>(a.q) + n.b * a.q_sb +
                    (n.hk * a.group + (ok ? head : 0)) * a.q_sh + (ok ? i : 0) * a.q_ss + 2 * t4;
#pragma unroll
      for (int x = 0; x < JQ; ++x)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const int ks = w + WARPS * x;
          qx[x][h][y] = ok && ks < KS ? *reinterpret_cast<const QPair*>(q + 16 * ks + 8 * y) : QPair{};
        }
      up[h] = 1.0f;
      if constexpr (F32 && HALF) {  // (as split_mma_kernel: q = 2^e (h0 + 2^-11 h1), |h0| <= 2)
        float top = 0.0f;
        if (ok) {
#pragma unroll
          for (int x = 0; x < D / 8; ++x) {
            const float2 z = *reinterpret_cast<const float2*>(q + 8 * x);
            top = fmaxf(top, fmaxf(fabsf(z.x), fabsf(z.y)));
          }
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int e = top > 0.0f && top < INFINITY ? ilogbf(top) : 0;
        up[h] = ldexpf(1.0f, max(-120, min(120, e)));
      }
    }
  };
  auto store_q = [&]() {
#pragma unroll
    for (int x = 0; x < JQ; ++x) {
      const int ks = w + WARPS * x;
      uint32_t parts[QP][4];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          if constexpr (!F32) {
            parts[0][h + 2 * y] = qx[x][h][y];
          } else if constexpr (HALF) {
            const float down = 1.0f / up[h], lo = qx[x][h][y].x * down, hi = qx[x][h][y].y * down;
            parts[0][h + 2 * y] = pack16<T>(lo, hi);
            const float2 z = unpack16<T>(parts[0][h + 2 * y]);
            parts[QP - 1][h + 2 * y] = pack16<T>((lo - z.x) * 2048.0f, (hi - z.y) * 2048.0f);
          } else {
            float2 v = qx[x][h][y];
#pragma unroll
            for (int p = 0; p < QP; ++p) {
              parts[p][h + 2 * y] = pack16<T>(v.x, v.y);
              const float2 z = unpack16<T>(parts[p][h + 2 * y]);
              v = make_float2(v.x - z.x, v.y - z.y);
            }
          }
        }
      if (ks < KS) {
#pragma unroll
        for (int p = 0; p < QP; ++p)
          qs[(ks * QP + p) * 32 + lane] = make_uint4(parts[p][0], parts[p][1], parts[p][2], parts[p][3]);
      }
    }
  };
  UnitInfo n;
  if (blockIdx.x < units) {
    n = unit_info(a, ix, blockIdx.x);
    load_q(n);
    store_q();
    __syncthreads();  // q in place
  }
  // Addresses within a tile: K's rows (lane % 8) + 8 (lane / 16), pieces 2 ks + lane / 8 % 2; V's rows
  // (lane % 8) + 8 (lane / 8 % 2), pieces 2 mt + lane / 16.
  const int k_row = (lane & 7) + 8 * (lane >> 4), k_piece = (lane >> 3) & 1;
  const int v_row = (lane & 7) + 8 * ((lane >> 3) & 1), v_piece = lane >> 4;
  int stage = 0;  // of the next tile; the stage before it is free
  for (uint32_t u = blockIdx.x; u < units; u += gridDim.x) {
    const int tiles = (n.hi - n.lo + TK - 1) / TK;
    const float qscale[2] = {a.scale * up[0], a.scale * up[1]};
    const int lim[2] = {row_limit(a, n, n.r0 + g), row_limit(a, n, n.r0 + g + 8)};
    // What the sequence's first new token sees, the fewest of all: a tile that ends behind it masks row by
    // row, in every block (a prompt's every tile: its value products are then issued once a row).
    const int lim_min = a.causal ? max(n.len - n.n_new + 1, 0) : n.len;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
    float acc[KS][2][4];  // rows g, g + 8: dims 16 mt + 8 y + 2 t4, + 1
#pragma unroll
    for (int mt = 0; mt < KS; ++mt)
#pragma unroll
      for (int y = 0; y < 2; ++y)
#pragma unroll
        for (int x = 0; x < 4; ++x) acc[mt][y][x] = 0.0f;

    for (int t = w; t < tiles; t += WARPS) {
      cp_async_wait_group<ST - 2>();
      __syncwarp();  // the tile is in place for every lane, and the stage before it is free
      const unsigned char* kt = ring.base + stage * R::STAGE;
      const unsigned char* vt = kt + R::KV;
      const int k0 = n.lo + TK * t;

      // Scores of rows g, g + 8 and keys 16 i + 8 y + 2 t4, + 1. fp32: the small parts in a chain of
      // their own, truncated at their magnitude; else two chains, half as long.
      float c[MT][2][2][4];
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
          for (int x = 0; x < 4; ++x) c[i][y][0][x] = c[i][y][1][x] = 0.0f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        uint32_t qa[QP][4];
#pragma unroll
        for (int p = 0; p < QP; ++p) {
          const uint4 z = qs[(ks * QP + p) * 32 + lane];
          qa[p][0] = z.x, qa[p][1] = z.y, qa[p][2] = z.z, qa[p][3] = z.w;
        }
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          uint32_t kf[4];
          ldsm4(kf, kt + (16 * i + k_row) * R::RB + 16 * ((2 * ks + k_piece) ^ R::k_swizzle(k_row)));
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            if constexpr (F32) {
#pragma unroll
              for (int p = QP - 1; p > 0; --p) mma<T>(c[i][y][1], qa[p], kf[2 * y], kf[2 * y + 1]);
              mma<T>(c[i][y][0], qa[0], kf[2 * y], kf[2 * y + 1]);
            } else {
              mma<T>(c[i][y][ks & 1], qa[0], kf[2 * y], kf[2 * y + 1]);
            }
          }
        }
      }
      float s[MT][2][4];
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
          for (int x = 0; x < 4; ++x)
            s[i][y][x] = (F32 && HALF ? fmaf(c[i][y][1][x], 1.0f / 2048.0f, c[i][y][0][x])
                                      : c[i][y][1][x] + c[i][y][0][x]) * qscale[x >> 1];
      // (behind the products: their latency hides the next loads' issue)
      const unsigned now = ring.advance(stage == 0 ? ST - 1 : stage - 1);
      const bool edge = lim_min < min(k0 + TK, n.hi);
      if (now != R::ALL || edge) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const int k = 16 * i + 8 * y + 2 * t4 + (x & 1);
              if (!((now >> k) & 1u) || k0 + k >= lim[x >> 1]) s[i][y][x] = -INFINITY;
            }
      }
      uint32_t pa[MT][PP][4];  // P as A fragments, in parts
      float alpha[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float top = m[h];
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int y = 0; y < 2; ++y) top = fmaxf(top, fmaxf(s[i][y][2 * h], s[i][y][2 * h + 1]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const float mu = top == -INFINITY ? 0.0f : top;
        alpha[h] = ex2((m[h] - mu) * LOG2E);
        m[h] = top;
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            float2 v = make_float2(ex2((s[i][y][2 * h] - mu) * LOG2E) * P_UP,
                                   ex2((s[i][y][2 * h + 1] - mu) * LOG2E) * P_UP);
            sum += v.x + v.y;
#pragma unroll
            for (int p = 0; p < PP; ++p) {
              pa[i][p][h + 2 * y] = pack16<T>(v.x, v.y);
              const float2 z = unpack16<T>(pa[i][p][h + 2 * y]);
              v = make_float2(v.x - z.x, v.y - z.y);
            }
          }
        l[h] = fmaf(l[h], alpha[h], sum);
      }
      auto v_at = [&](int i, int mt) {
        return vt + (16 * i + v_row) * R::RB + 16 * ((2 * mt + v_piece) ^ R::v_swizzle(v_row));
      };
      if (!edge) {
#pragma unroll
        for (int mt = 0; mt < KS; ++mt) {
          float o[2][4] = {};
          uint32_t vf[MT][4];
#pragma unroll
          for (int i = 0; i < MT; ++i) ldsm4t(vf[i], v_at(i, mt));
#pragma unroll
          for (int p = PP - 1; p >= 0; --p)
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
              for (int y = 0; y < 2; ++y) mma<T>(o[y], pa[i][p], vf[i][2 * y], vf[i][2 * y + 1]);
#pragma unroll
          for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int x = 0; x < 4; ++x) acc[mt][y][x] = fmaf(acc[mt][y][x], alpha[x >> 1], o[y][x]);
        }
      } else {
        // Keys that only some of the rows see: one row at a time, the values it does not see as
        // zeros (0 times what they hold could be NaN).
#pragma unroll
        for (int mt = 0; mt < KS; ++mt)
#pragma unroll
          for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int x = 0; x < 4; ++x) acc[mt][y][x] *= alpha[x >> 1];
        for (int r = 0; r < min(16, a.rows - n.r0); ++r) {
          const int end = row_limit(a, n, n.r0 + r);
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            const int k = k0 + 16 * i + 2 * t4;  // this lane's keys of a B fragment: k, + 1, + 8, + 9
            const uint32_t mlo = (k < end ? 0xffffu : 0u) | (k + 1 < end ? 0xffff0000u : 0u);
            const uint32_t mhi = (k + 8 < end ? 0xffffu : 0u) | (k + 9 < end ? 0xffff0000u : 0u);
            uint32_t mine[PP][4];
#pragma unroll
            for (int p = 0; p < PP; ++p)
#pragma unroll
              for (int x = 0; x < 4; ++x) mine[p][x] = g + 8 * (x & 1) == r ? pa[i][p][x] : 0u;
#pragma unroll
            for (int mt = 0; mt < KS; ++mt) {
              uint32_t vf[4];
              ldsm4t(vf, v_at(i, mt));
#pragma unroll
              for (int y = 0; y < 2; ++y) {
                float o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int p = PP - 1; p >= 0; --p) mma<T>(o, mine[p], vf[2 * y] & mlo, vf[2 * y + 1] & mhi);
#pragma unroll
                for (int x = 0; x < 4; ++x)
                  if (g + 8 * (x >> 1) == r) acc[mt][y][x] += o[x];
              }
            }
          }
        }
      }
      stage = stage + 1 == ST ? 0 : stage + 1;
    }
    const UnitInfo done = n;
    const int free_at = w * R::BYTES + (stage == 0 ? ST - 1 : stage - 1) * R::STAGE;
    __syncwarp();  // every lane has read its last tile
    if (lane == 0) red_at[w] = free_at;
    float* sums = reinterpret_cast<float*>(smem + free_at);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
      if (t4 == 0) ml[w * MAXR + g + 8 * h] = make_float2(m[h], l[h]);
#pragma unroll
      for (int mt = 0; mt < KS; ++mt)
#pragma unroll
        for (int y = 0; y < 2; ++y)
          *reinterpret_cast<float2*>(sums + (g + 8 * h) * D + 16 * mt + 8 * y + 2 * t4) =
              make_float2(acc[mt][y][2 * h], acc[mt][y][2 * h + 1]);
    }
    // The next unit's queries travel while this one's sums are joined.
    const bool more = u + gridDim.x < units;
    if (more) {
      n = ring.unit == u + gridDim.x ? ring.info : unit_info(a, ix, u + gridDim.x);
      load_q(n);
    }
    __syncthreads();
    write_chunk<QT, D>(a, done, smem, red_at, ml, min(16, a.rows - done.r0));
    if (more) store_q();
    __syncthreads();  // the sums are read: their stages take tiles again, and q is in place
  }
  if (ring.bad) flag_error(a.sink, CFA_ERR_PAGE);
}

// fp32 caches, one or two query rows (NR): FMAs.
template <int D, int NR>
__global__ void __launch_bounds__(NT, 3) split_fma_kernel(const SplitArgs a) {
  using R = RingOf<D, 4, NR>;
  constexpr int ST = R::ST, TK = R::TK;
  constexpr int LPK = 32 / TK, DL = D / LPK;  // lanes of a key's score, dims of each
  constexpr int LPR = D / 4, KPI = 32 / LPR;  // lanes of a V row; keys at a time
  extern __shared__ __align__(128) unsigned char smem[];
  const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31;
  float2* ml = reinterpret_cast<float2*>(smem + off_ml<D, 4, NR>());
  int* red_at = reinterpret_cast<int*>(ml + WARPS * MAXR);
  float* q_sets = reinterpret_cast<float*>(smem + off_q<D, 4, NR>());  // two sets of [NR][D]
  uint64_t* ps = reinterpret_cast<uint64_t*>(q_sets + 2 * NR * D) + w * TK * NR;  // p twice: [key][NR]
  griddep_wait();
  griddep_launch_dependents();
  ChunkIndex ix;
  ix.init(a, lane);
  const uint32_t units = static_cast<uint32_t>(ix.total) * a.Hk * a.row_chunks;
  R ring(a, ix, units, smem + w * R::BYTES, lane, w);

  auto load_q = [&](const UnitInfo& n, float* qs) {
    for (int i = tid; i < NR * LPR; i += NT) {
      const int row = n.r0 + i / LPR, c = i % LPR;
      int head, t;
      row_of(a, row, head, t);
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      if (row < a.rows && t < n.n_new)
        x = *reinterpret_cast<const float4*>(static_cast<const float*>(a.q) + n.b * a.q_sb +
                                             (n.hk * a.group + head) * a.q_sh + t * a.q_ss + 4 * c);
      reinterpret_cast<float4*>(qs)[i] = x;
    }
  };
  UnitInfo n;
  if (blockIdx.x < units) {
    n = unit_info(a, ix, blockIdx.x);
    load_q(n, q_sets);
    __syncthreads();  // q in place
  }
  int stage = 0;  // of the next tile; the stage before it is free
  int set = 0;
  for (uint32_t u = blockIdx.x; u < units; u += gridDim.x, set ^= 1) {
    const float* qs = q_sets + set * (NR * D);
    const int tiles = (n.hi - n.lo + TK - 1) / TK;
    const int lim_min = a.causal ? max(n.len - n.n_new + 1, 0) : n.len;
    float m[NR], l[NR];
    uint64_t acc[NR][2];  // this lane's four dims, packed
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      m[r] = -INFINITY;
      l[r] = 0.0f;
      acc[r][0] = acc[r][1] = 0ull;
    }
    for (int t = w; t < tiles; t += WARPS) {
      cp_async_wait_group<ST - 2>();
      __syncwarp();
      const unsigned now = ring.advance(stage == 0 ? ST - 1 : stage - 1);
      const unsigned char* kt = ring.base + stage * R::STAGE;
      const unsigned char* vt = kt + R::KV;
      const int k0 = n.lo + TK * t;
      const bool edge = lim_min < min(k0 + TK, n.hi);
      // Scores: lane x takes dims DL (x / TK) .. of key x % TK.
      // (packed fp32: dims 4 c, 4 c + 2, .. and the odd ones in two chains, added at the end)
      uint64_t s2[NR];
#pragma unroll
      for (int r = 0; r < NR; ++r) s2[r] = 0ull;
      const float* kr = reinterpret_cast<const float*>(kt + (lane % TK) * R::RB) + lane / TK * DL;
      const float* qh = qs + lane / TK * DL;
#pragma unroll
      for (int c = 0; c < DL / 4; ++c) {
        const ulonglong2 x = ld2x2(kr + 4 * c);
#pragma unroll
        for (int r = 0; r < NR; ++r) {
          const ulonglong2 y = ld2x2(qh + r * D + 4 * c);
          s2[r] = fma2(x.y, y.y, fma2(x.x, y.x, s2[r]));
        }
      }
      float p[NR];
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        float y = sum2(s2[r]);
#pragma unroll
        for (int o = TK; o < 32; o <<= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
        y *= a.scale;
        const int key = lane % TK;
        if (!((now >> key) & 1u) || (edge && k0 + key >= row_limit(a, n, n.r0 + r))) y = -INFINITY;
        float top = y;
#pragma unroll
        for (int o = 1; o < TK; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        top = fmaxf(top, m[r]);
        const float mu = top == -INFINITY ? 0.0f : top;
        const float al = ex2((m[r] - mu) * LOG2E);
        m[r] = top;
        p[r] = ex2((y - mu) * LOG2E);
        l[r] = fmaf(l[r], al, p[r]);  // this lane's keys (the lanes of a key hold the same)
        const uint64_t al2 = dup2(al);
        acc[r][0] = mul2(acc[r][0], al2);
        acc[r][1] = mul2(acc[r][1], al2);
        if (lane < TK) ps[lane * NR + r] = dup2(p[r]);
      }
      __syncwarp();  // every key's p in place
      auto fold_keys = [&](auto masked) {
#pragma unroll
        for (int j = 0; j < TK / KPI; ++j) {
          const int k = KPI * j + lane / LPR;
          const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(vt + k * R::RB + 16 * (lane % LPR));
          uint64_t pk[NR];
          if constexpr (NR == 1) {
            pk[0] = ps[k];
          } else {
#pragma unroll
            for (int r = 0; r < NR; r += 2) {
              const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(ps + k * NR + r);
              pk[r] = x.x;
              pk[r + 1] = x.y;
            }
          }
#pragma unroll
          for (int r = 0; r < NR; ++r) {
            if (!decltype(masked)::value || pk[r] != 0ull) {
              acc[r][0] = fma2(pk[r], v.x, acc[r][0]);
              acc[r][1] = fma2(pk[r], v.y, acc[r][1]);
            }
          }
        }
      };
      if (!edge) fold_keys(std::false_type{});
      else fold_keys(std::true_type{});  // an unseen key's value may be NaN
      __syncwarp();  // read: the next tile's p may land
      stage = stage + 1 == ST ? 0 : stage + 1;
    }
    float4 o4[NR];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
#pragma unroll
      for (int o = 1; o < TK; o <<= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], o);
      const float2 lo = split2(acc[r][0]), hi = split2(acc[r][1]);
      o4[r] = make_float4(lo.x, lo.y, hi.x, hi.y);
#pragma unroll
      for (int o = LPR; o < 32; o <<= 1) {
        o4[r].x += __shfl_xor_sync(0xffffffffu, o4[r].x, o);
        o4[r].y += __shfl_xor_sync(0xffffffffu, o4[r].y, o);
        o4[r].z += __shfl_xor_sync(0xffffffffu, o4[r].z, o);
        o4[r].w += __shfl_xor_sync(0xffffffffu, o4[r].w, o);
      }
    }
    // The next unit's queries travel while this one's sums are joined.
    const UnitInfo done = n;
    const int free_at = w * R::BYTES + (stage == 0 ? ST - 1 : stage - 1) * R::STAGE;
    __syncwarp();  // every lane has read its last tile
    if (u + gridDim.x < units) {
      n = ring.unit == u + gridDim.x ? ring.info : unit_info(a, ix, u + gridDim.x);
      load_q(n, q_sets + (set ^ 1) * (NR * D));
    }
    if (lane == 0) red_at[w] = free_at;
    float* sums = reinterpret_cast<float*>(smem + free_at);
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      if (lane == 0) ml[w * MAXR + r] = make_float2(m[r], l[r]);
      if (lane < LPR)
        *reinterpret_cast<float4*>(sums + r * D + 4 * lane) = o4[r];
    }
    __syncthreads();  // (the next unit's queries are in place too)
    write_chunk<float, D>(a, done, smem, red_at, ml, min(NR, a.rows - done.r0));
    __syncthreads();  // the sums are read: their stages take tiles again
  }
  if (ring.bad) flag_error(a.sink, CFA_ERR_PAGE);
}

// fp32 caches: up to 8 HALVES query rows a block. One half: rows g of m16n8k8 are a query row's large
// part, rows g + 8 its small one, so two products take all four parts of it and a key; two halves: the
// parts are products of their own, and the one of both small parts is left out.
template <int D, int HALVES>
__global__ void __launch_bounds__(NT, 2) split_f32_kernel(const SplitArgs a) {
  using R = RingOf<D, 4, 8 * HALVES>;
  constexpr int ST = R::ST, TK = R::TK;
  constexpr int NK = TK / 8, J = D / 16, JV = D / 32;
  constexpr int JQ = HALVES == 1 ? J : (J + WARPS - 1) / WARPS;  // this warp's share of q's columns
  extern __shared__ __align__(128) unsigned char smem[];
  const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t4 = lane & 3;  // a fragment's row (B: column), and k
  float2* ml = reinterpret_cast<float2*>(smem + off_ml<D, 4, 8 * HALVES>());
  int* red_at = reinterpret_cast<int*>(ml + WARPS * MAXR);
  uint4* qs = reinterpret_cast<uint4*>(smem + off_q<D, 4, 8 * HALVES>());  // [J][k-step][hi, lo][lane]
  griddep_wait();
  griddep_launch_dependents();
  ChunkIndex ix;
  ix.init(a, lane);
  const uint32_t units = static_cast<uint32_t>(ix.total) * a.Hk * a.row_chunks;
  R ring(a, ix, units, smem + w * R::BYTES, lane, w);

  // Dims 16 j + 4 t4 .. + 3 of rows g (and g + 8): k-steps 2 j, 2 j + 1 with k = t4, t4 + 4 for each
  // adjacent pair of dims.
  float4 qx[JQ][HALVES];
  auto load_q = [&](const UnitInfo& n) {
#pragma unroll
    for (int h = 0; h < HALVES; ++h) {
      const int row = n.r0 + g + 8 * h;
      int head, i;
      row_of(a, row, head, i);
      const bool ok = row < a.rows && i < n.n_new;
      const float* q = static_cast<const float*>(a.q) + n.b * a.q_sb +
                       (n.hk * a.group + (ok ? head : 0)) * a.q_sh + (ok ? i : 0) * a.q_ss;
#pragma unroll
      for (int x = 0; x < JQ; ++x) {
        const int j = HALVES == 1 ? x : w + WARPS * x;
        qx[x][h] = ok && j < J ? ld4(q + 16 * j + 4 * t4) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
    }
  };
  // (two halves: the fragments in shared memory, shared by the warps)
  auto store_q = [&]() {
    if constexpr (HALVES == 2) {
#pragma unroll
      for (int x = 0; x < JQ; ++x) {
        const int j = w + WARPS * x;
        uint32_t hi[2][4], lo[2][4];
        split_tf32(qx[x][0], hi[0], lo[0]);
        split_tf32(qx[x][1], hi[1], lo[1]);
        if (j < J) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            qs[(j * 4 + 2 * k) * 32 + lane] = make_uint4(hi[0][2 * k], hi[1][2 * k], hi[0][2 * k + 1], hi[1][2 * k + 1]);
            qs[(j * 4 + 2 * k + 1) * 32 + lane] = make_uint4(lo[0][2 * k], lo[1][2 * k], lo[0][2 * k + 1], lo[1][2 * k + 1]);
          }
        }
      }
    }
  };
  UnitInfo n;
  if (blockIdx.x < units) {
    n = unit_info(a, ix, blockIdx.x);
    load_q(n);
    if constexpr (HALVES == 2) {
      store_q();
      __syncthreads();  // q in place
    }
  }
  int stage = 0;  // of the next tile; the stage before it is free
  for (uint32_t u = blockIdx.x; u < units; u += gridDim.x) {
    const int tiles = (n.hi - n.lo + TK - 1) / TK;
    uint32_t qa[HALVES == 1 ? J : 1][2][4];
    if constexpr (HALVES == 1) {
#pragma unroll
      for (int j = 0; j < J; ++j) {
        uint32_t hi[4], lo[4];
        split_tf32(qx[j][0], hi, lo);
#pragma unroll
        for (int x = 0; x < 4; ++x) qa[j][x >> 1][2 * (x & 1)] = hi[x], qa[j][x >> 1][2 * (x & 1) + 1] = lo[x];
      }
    }
    int lim[HALVES];
#pragma unroll
    for (int h = 0; h < HALVES; ++h) lim[h] = row_limit(a, n, n.r0 + g + 8 * h);
    // What the sequence's first new token sees, the fewest of all: a tile that ends behind it masks row by
    // row, in every block (a prompt's every tile: its value products are then issued once a row).
    const int lim_min = a.causal ? max(n.len - n.n_new + 1, 0) : n.len;
    float m[HALVES], l[HALVES];
    float acc[JV][4][2 * HALVES];  // rows g (, g + 8): dims 32 j + 8 t4 + e (, + 4)
#pragma unroll
    for (int h = 0; h < HALVES; ++h) m[h] = -INFINITY, l[h] = 0.0f;
#pragma unroll
    for (int j = 0; j < JV; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int x = 0; x < 2 * HALVES; ++x) acc[j][e][x] = 0.0f;

    for (int t = w; t < tiles; t += WARPS) {
      cp_async_wait_group<ST - 2>();
      __syncwarp();  // the tile is in place for every lane, and the stage before it is free
      const unsigned char* kt = ring.base + stage * R::STAGE;
      const unsigned char* vt = kt + R::KV;
      const int k0 = n.lo + TK * t;

      // Scores: rows g, g + 8; keys 8 i + 2 t4, + 1, in sums of 16 dims, their products and additions in
      // cross_few_bwd.cu's order: its e^(s - L) is then what L was made of. (With the dims in one chain of
      // products, truncated at its own magnitude, and one or two rows by FMAs in training too, dV at scores of
      // a hundred was 1e-5 off where it is 2e-6 now; 8 rows 126 us for 129 at d 128, 66.1 for 66.6 at 64.)
      float s[NK][2 * HALVES];
#pragma unroll
      for (int i = 0; i < NK; ++i)
#pragma unroll
        for (int x = 0; x < 2 * HALVES; ++x) s[i][x] = 0.0f;
      const unsigned char* ka = kt + g * R::RB + 16 * (t4 ^ (4 * (g & 1)));
      const unsigned char* kb = kt + g * R::RB + 16 * (t4 ^ (4 * (~g & 1)));
#pragma unroll
      for (int j = 0; j < J; ++j) {
        uint32_t ah[2][4], al[2][4];  // (one half: both parts in ah)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          if constexpr (HALVES == 1) {
#pragma unroll
            for (int e = 0; e < 4; ++e) ah[x][e] = qa[j][x][e];
          } else {
            const uint4 h = qs[(j * 4 + 2 * x) * 32 + lane], y = qs[(j * 4 + 2 * x + 1) * 32 + lane];
            ah[x][0] = h.x, ah[x][1] = h.y, ah[x][2] = h.z, ah[x][3] = h.w;
            al[x][0] = y.x, al[x][1] = y.y, al[x][2] = y.z, al[x][3] = y.w;
          }
        }
#pragma unroll
        for (int i = 0; i < NK; ++i) {
          const float4 key = *reinterpret_cast<const float4*>((j & 1 ? kb : ka) + 8 * i * R::RB + 128 * (j >> 1));
          float c[4] = {0.f, 0.f, 0.f, 0.f};
          if constexpr (HALVES == 2) {
            products(c, ah, al, key);
#pragma unroll
            for (int x = 0; x < 4; ++x) s[i][x] += c[x];
          } else {
            uint32_t kh[4], kl[4];
            float cl[4] = {0.f, 0.f, 0.f, 0.f};
            split_tf32(key, kh, kl);
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              mma_tf32(cl, ah[x], kl[2 * x], kl[2 * x + 1]);
              mma_tf32(c, ah[x], kh[2 * x], kh[2 * x + 1]);
            }
#pragma unroll
            for (int x = 0; x < 2; ++x) s[i][x] += (c[2 + x] + cl[x]) + c[x];  // (not both small parts: cl[2 + x])
          }
        }
      }
#pragma unroll
      for (int i = 0; i < NK; ++i)
#pragma unroll
        for (int x = 0; x < 2 * HALVES; ++x) s[i][x] *= a.scale;
      // (behind the products: their latency hides the next loads' issue)
      const unsigned now = ring.advance(stage == 0 ? ST - 1 : stage - 1);
      const bool edge = lim_min < min(k0 + TK, n.hi);
      if (now != R::ALL || edge) {
#pragma unroll
        for (int i = 0; i < NK; ++i)
#pragma unroll
          for (int x = 0; x < 2 * HALVES; ++x) {
            const int k = 8 * i + 2 * t4 + (x & 1);
            if (!((now >> k) & 1u) || k0 + k >= lim[x >> 1]) s[i][x] = -INFINITY;
          }
      }
      // P as A fragments: k = t4 is key 8 i + 2 t4, t4 + 4 the one after (one half: both parts in ph).
      uint32_t ph[NK][4], pl[NK][4];
      float alpha[HALVES];
#pragma unroll
      for (int h = 0; h < HALVES; ++h) {
        float top = fmaxf(s[0][2 * h], s[0][2 * h + 1]);
#pragma unroll
        for (int i = 1; i < NK; ++i) top = fmaxf(top, fmaxf(s[i][2 * h], s[i][2 * h + 1]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        top = fmaxf(top, m[h]);
        const float mu = top == -INFINITY ? 0.0f : top;
        alpha[h] = ex2((m[h] - mu) * LOG2E);
        m[h] = top;
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < NK; ++i) {
          const float p0 = ex2((s[i][2 * h] - mu) * LOG2E), p1 = ex2((s[i][2 * h + 1] - mu) * LOG2E);
          sum += p0 + p1;
          uint32_t hi[4], lo[4];
          split_tf32(make_float4(p0, p1, 0.f, 0.f), hi, lo);
          ph[i][h] = hi[0], ph[i][2 + h] = hi[1];
          if constexpr (HALVES == 1) ph[i][1] = lo[0], ph[i][3] = lo[1];
          else pl[i][h] = lo[0], pl[i][2 + h] = lo[1];
        }
        l[h] = fmaf(l[h], alpha[h], sum);
      }
      // Values of keys 8 i + 2 t4, + 1; columns g of the four products e: dims 32 j + 4 g + e.
      const unsigned char* va = vt + 2 * t4 * R::RB + 16 * (g ^ (2 * t4));
      if (!edge) {
#pragma unroll
        for (int j = 0; j < JV; ++j) {
          float c[4][4] = {};
#pragma unroll
          for (int i = 0; i < NK; ++i) {
            uint32_t xh[4], xl[4], yh[4], yl[4];
            const unsigned char* at = va + 8 * i * R::RB + 128 * j;
            split_tf32(*reinterpret_cast<const float4*>(at), xh, xl);
            split_tf32(*reinterpret_cast<const float4*>(at + R::RB), yh, yl);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if constexpr (HALVES == 2) mma_tf32(c[e], pl[i], xh[e], yh[e]);
#pragma unroll
            for (int e = 0; e < 4; ++e) mma_tf32(c[e], ph[i], xl[e], yl[e]);
#pragma unroll
            for (int e = 0; e < 4; ++e) mma_tf32(c[e], ph[i], xh[e], yh[e]);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int x = 0; x < 2 * HALVES; ++x)
              acc[j][e][x] = fmaf(acc[j][e][x], alpha[x >> 1], HALVES == 1 ? c[e][x] + c[e][2 + x] : c[e][x]);
        }
      } else {
        // Keys that only some of the rows see: one row at a time, the values it does not see as
        // zeros (0 times what they hold could be NaN).
#pragma unroll
        for (int j = 0; j < JV; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int x = 0; x < 2 * HALVES; ++x) acc[j][e][x] *= alpha[x >> 1];
        for (int r = 0; r < min(8 * HALVES, a.rows - n.r0); ++r) {
          const int end = row_limit(a, n, n.r0 + r);
#pragma unroll
          for (int i = 0; i < NK; ++i) {
            const int k = k0 + 8 * i + 2 * t4;
            uint32_t rh[4], rl[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const bool mine = g + (HALVES == 1 ? 0 : 8 * (x & 1)) == r;
              rh[x] = mine ? ph[i][x] : 0u;
              if constexpr (HALVES == 2) rl[x] = mine ? pl[i][x] : 0u;
            }
#pragma unroll
            for (int j = 0; j < JV; ++j) {
              const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
              const unsigned char* at = va + 8 * i * R::RB + 128 * j;
              uint32_t xh[4], xl[4], yh[4], yl[4];
              split_tf32(k < end ? *reinterpret_cast<const float4*>(at) : zero, xh, xl);
              split_tf32(k + 1 < end ? *reinterpret_cast<const float4*>(at + R::RB) : zero, yh, yl);
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                float c[4] = {0.f, 0.f, 0.f, 0.f};
                if constexpr (HALVES == 2) mma_tf32(c, rl, xh[e], yh[e]);
                mma_tf32(c, rh, xl[e], yl[e]);
                mma_tf32(c, rh, xh[e], yh[e]);
#pragma unroll
                for (int x = 0; x < 2 * HALVES; ++x)
                  if (g + 8 * (x >> 1) == r) acc[j][e][x] += HALVES == 1 ? c[x] + c[2 + x] : c[x];
              }
            }
          }
        }
      }
      stage = stage + 1 == ST ? 0 : stage + 1;
    }
    const UnitInfo done = n;
    const int free_at = w * R::BYTES + (stage == 0 ? ST - 1 : stage - 1) * R::STAGE;
    __syncwarp();  // every lane has read its last tile
    if (lane == 0) red_at[w] = free_at;
    float* sums = reinterpret_cast<float*>(smem + free_at);
#pragma unroll
    for (int h = 0; h < HALVES; ++h) {
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
      if (t4 == 0) ml[w * MAXR + g + 8 * h] = make_float2(m[h], l[h]);
#pragma unroll
      for (int j = 0; j < JV; ++j)
#pragma unroll
        for (int x = 0; x < 2; ++x)
          *reinterpret_cast<float4*>(sums + (g + 8 * h) * D + 32 * j + 8 * t4 + 4 * x) =
              make_float4(acc[j][0][2 * h + x], acc[j][1][2 * h + x], acc[j][2][2 * h + x],
                          acc[j][3][2 * h + x]);
    }
    // The next unit's queries travel while this one's sums are joined.
    const bool more = u + gridDim.x < units;
    if (more) {
      n = ring.unit == u + gridDim.x ? ring.info : unit_info(a, ix, u + gridDim.x);
      load_q(n);
    }
    __syncthreads();
    write_chunk<float, D>(a, done, smem, red_at, ml, min(8 * HALVES, a.rows - done.r0));
    if constexpr (HALVES == 2) {
      if (more) store_q();
    }
    __syncthreads();  // the sums are read: their stages take tiles again (and q is in place)
  }
  if (ring.bad) flag_error(a.sink, CFA_ERR_PAGE);
}

// The chunks' join, chunk c of a row in group c % G (G = 128 / (D / 4)): the groups' sums in chunk order,
// then over the groups in order. Everything that does not come from the chunks' kernel is read before
// waiting for it: that kernel has waited for its own predecessors when it lets this one start.
template <int D>
struct JoinRow {
  static constexpr int C4 = D / 4, G = NT / C4;
  int64_t row;  // (b H + head) S + i
  int b, head, i, nc;
  bool live;
  __device__ __forceinline__ JoinRow(const SplitArgs& a, int64_t row_) : row(row_) {
    i = a.S == 1 ? 0 : static_cast<int>(row % a.S);
    const int64_t bh = a.S == 1 ? row : row / a.S;
    b = static_cast<int>(bh / a.H);
    head = static_cast<int>(bh - static_cast<int64_t>(b) * a.H);
    nc = chunks_of(seq_len(a, b), a.tile_log);
    live = i < seq_new(a, b);
  }
  template <typename QT>
  __device__ __forceinline__ void store(const SplitArgs& a, int c4, float4 o, float l) const {
    const bool some = live && l != 0.0f;
    QT* dst = static_cast<QT*>(a.o) + ((static_cast<int64_t>(b) * a.S + i) * a.H + head) * D + 4 * c4;
    dst[0] = from_f<QT>(some ? o.x / l : 0.0f);
    dst[1] = from_f<QT>(some ? o.y / l : 0.0f);
    dst[2] = from_f<QT>(some ? o.z / l : 0.0f);
    dst[3] = from_f<QT>(some ? o.w / l : 0.0f);
  }
};
__device__ __forceinline__ void fold(float4& o, float4 v, float f) {
  o.x = fmaf(v.x, f, o.x);
  o.y = fmaf(v.y, f, o.y);
  o.z = fmaf(v.z, f, o.z);
  o.w = fmaf(v.w, f, o.w);
}
__device__ __forceinline__ float4 plus(float4 o, float4 v) {
  return make_float4(o.x + v.x, o.y + v.y, o.z + v.z, o.w + v.w);
}

// A block a row; its threads take the row's columns and, side by side, the groups. The first chunks of
// each group travel while the weights are found.
template <typename QT, int D>
__global__ void __launch_bounds__(NT) split_join_kernel(const SplitArgs a) {
  using J = JoinRow<D>;
  __shared__ float wt[MOST_CHUNKS];
  __shared__ float4 sums[J::G][J::C4];
  __shared__ float red[2][WARPS];
  const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31;
  const J r(a, blockIdx.x);
  griddep_wait();
  griddep_launch_dependents();
  if (r.nc == 1) return;  // written by the first kernel
  const float2* ml = a.part_ml + r.row * a.max_chunks;
  const int c4 = tid % J::C4, g = tid / J::C4;
  const float4* po = reinterpret_cast<const float4*>(a.part_o + r.row * a.max_chunks * D) + c4;
  constexpr int EARLY = 4;
  float4 early[EARLY];
#pragma unroll
  for (int j = 0; j < EARLY; ++j) {
    const int c = g + J::G * j;
    early[j] = r.live && c < r.nc ? po[static_cast<int64_t>(c) * J::C4] : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  float m = -INFINITY;
  float2 x[MOST_CHUNKS / NT];
#pragma unroll
  for (int j = 0; j < MOST_CHUNKS / NT; ++j) {
    const int c = tid + j * NT;
    x[j] = r.live && c < r.nc ? ml[c] : make_float2(-INFINITY, 0.0f);
    m = fmaxf(m, x[j].x);
  }
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane == 0) red[0][w] = m;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < WARPS; ++j) m = fmaxf(m, red[0][j]);
  const float mu = m == -INFINITY ? 0.0f : m;
  float l = 0.0f;
#pragma unroll
  for (int j = 0; j < MOST_CHUNKS / NT; ++j) {
    const int c = tid + j * NT;
    const float f = ex2((x[j].x - mu) * LOG2E);
    if (c < r.nc) wt[c] = f;
    l = j == 0 ? x[j].y * f : fmaf(x[j].y, f, l);
  }
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
  if (lane == 0) red[1][w] = l;
  __syncthreads();
  l = ((red[1][0] + red[1][1]) + red[1][2]) + red[1][3];
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  if (r.live) {
#pragma unroll
    for (int j = 0; j < EARLY; ++j)
      if (g + J::G * j < r.nc) fold(o, early[j], wt[g + J::G * j]);
#pragma unroll 8
    for (int c = g + J::G * EARLY; c < r.nc; c += J::G) fold(o, po[static_cast<int64_t>(c) * J::C4], wt[c]);
  }
  sums[g][c4] = o;
  __syncthreads();
  if (g == 0) {
#pragma unroll
    for (int j = 1; j < J::G; ++j) o = plus(o, sums[j][c4]);
    r.template store<QT>(a, c4, o, l);
    if (a.lse && c4 == 0) a.lse[r.row] = m + logf(l);  // (no key: -inf)
  }
}

// A persistent grid: as many blocks as fit at once, or as there are units at most. The occupancy of a
// kernel is asked for once (every device here is an sm_100a).
template <auto Kernel>
cudaError_t launch_split(int smem, const SplitArgs& a, cudaStream_t stream) {
  static std::atomic<int> kept{0};
  int dev = 0, sms = 0, per = kept.load(std::memory_order_relaxed);
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e == cudaSuccess && per == 0) {
    e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, Kernel, NT, smem);
    if (e == cudaSuccess && per == 0) e = cudaErrorInvalidConfiguration;
    kept.store(per, std::memory_order_relaxed);
  }
  if (e != cudaSuccess) return e;
  const int64_t units = static_cast<int64_t>(a.B) * a.max_chunks * a.Hk * a.row_chunks;
  const int64_t fit = static_cast<int64_t>(sms) * per;
  return launch_pdl(Kernel, dim3(static_cast<unsigned>(units < fit ? units : fit)), dim3(NT), smem,
                    stream, a);
}

template <typename QT, int D>
cudaError_t launch_join(const SplitArgs& a, cudaStream_t stream) {
  if (a.max_chunks == 1) return cudaSuccess;
  const int64_t rows = static_cast<int64_t>(a.B) * a.H * a.S;
  return launch_pdl(split_join_kernel<QT, D>, dim3(static_cast<unsigned>(rows)), dim3(NT), 0, stream, a);
}

// A 16-bit cache.
template <typename QT, typename T, int D>
cudaError_t launch_16(const SplitArgs& a, cudaStream_t stream) {
  return a.block_rows == 8 ? launch_split<split_mma_kernel<QT, T, D>>(split_smem<D, 2, 8>(), a, stream)
                           : launch_split<split_rows_kernel<QT, T, D>>(split_smem<D, 2, 16>(), a, stream);
}

template <int D>
cudaError_t launch_d(const SplitArgs& a, int qd, int kd, cudaStream_t stream) {
  cudaError_t e;
  if (qd == CFA_F32) {
    if (kd == CFA_F32) {
      e = a.rows == 1 && !a.lse   ? launch_split<split_fma_kernel<D, 1>>(split_smem<D, 4, 1>(), a, stream)
          : a.rows == 2 && !a.lse ? launch_split<split_fma_kernel<D, 2>>(split_smem<D, 4, 2>(), a, stream)
          : a.block_rows == 8 ? launch_split<split_f32_kernel<D, 1>>(split_smem<D, 4, 8>(), a, stream)
                              : launch_split<split_f32_kernel<D, 2>>(split_smem<D, 4, 16>(), a, stream);
    } else if (kd == CFA_F16) {
      e = launch_16<float, __half, D>(a, stream);
    } else {
      e = launch_16<float, __nv_bfloat16, D>(a, stream);
    }
    return e == cudaSuccess ? launch_join<float, D>(a, stream) : e;
  }
  if (qd == CFA_F16) {
    e = launch_16<__half, __half, D>(a, stream);
    return e == cudaSuccess ? launch_join<__half, D>(a, stream) : e;
  }
  e = launch_16<__nv_bfloat16, __nv_bfloat16, D>(a, stream);
  return e == cudaSuccess ? launch_join<__nv_bfloat16, D>(a, stream) : e;
}

template <int D>
cudaError_t set_attrs() {
  cudaError_t e = cudaSuccess;
  auto set = [&](const void* fn, int bytes) {
    if (e == cudaSuccess) e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  };
  constexpr int S2 = split_smem<D, 2, 8>();
  static_assert(S2 <= 232448 && split_smem<D, 4, 16>() <= 232448, "shared memory per block");
  set(reinterpret_cast<const void*>(split_fma_kernel<D, 1>), split_smem<D, 4, 1>());
  set(reinterpret_cast<const void*>(split_fma_kernel<D, 2>), split_smem<D, 4, 2>());
  set(reinterpret_cast<const void*>(split_f32_kernel<D, 1>), split_smem<D, 4, 8>());
  set(reinterpret_cast<const void*>(split_f32_kernel<D, 2>), split_smem<D, 4, 16>());
  set(reinterpret_cast<const void*>(split_mma_kernel<float, __half, D>), S2);
  set(reinterpret_cast<const void*>(split_mma_kernel<float, __nv_bfloat16, D>), S2);
  set(reinterpret_cast<const void*>(split_mma_kernel<__half, __half, D>), S2);
  set(reinterpret_cast<const void*>(split_mma_kernel<__nv_bfloat16, __nv_bfloat16, D>), S2);
  constexpr int S16 = split_smem<D, 2, 16>();
  static_assert(S16 <= 232448, "shared memory per block");
  set(reinterpret_cast<const void*>(split_rows_kernel<float, __half, D>), S16);
  set(reinterpret_cast<const void*>(split_rows_kernel<float, __nv_bfloat16, D>), S16);
  set(reinterpret_cast<const void*>(split_rows_kernel<__half, __half, D>), S16);
  set(reinterpret_cast<const void*>(split_rows_kernel<__nv_bfloat16, __nv_bfloat16, D>), S16);
  return e;
}

}  // namespace

cudaError_t setup_split_attributes() {
  cudaError_t e = set_attrs<32>();
  if (e == cudaSuccess) e = set_attrs<64>();
  return e == cudaSuccess ? set_attrs<128>() : e;
}

// log2 of tile_keys.
static int tile_log_of(int64_t head_dim, int kv_dtype) {
  if (kv_dtype == CFA_F32) return head_dim == 32 ? 5 : head_dim == 64 ? 4 : 3;
  return head_dim == 128 ? 4 : 5;
}

// Most chunks of a sequence of at most max_len keys: its own, or 16 of a shorter one whose chunks are
// half as long.
int split_max_chunks(int64_t max_len, int64_t head_dim, int kv_dtype) {
  const int t = tile_log_of(head_dim, kv_dtype), len = static_cast<int>(max_len);
  const int own = chunks_of(len, t), few = 1 << (t + 4 + FEW_CHUNKS_LOG);
  const int most = len > few && own < (1 << FEW_CHUNKS_LOG) ? 1 << FEW_CHUNKS_LOG : own;
  // (past 256 chunks the count falls back to 129 at the next power of two)
  return bits_of(static_cast<uint32_t>(len > 0 ? len - 1 : 0)) - MOST_CHUNKS_LOG > t + 5 ? MOST_CHUNKS : most;
}

size_t split_workspace_bytes(int64_t rows, int64_t max_len, int64_t head_dim, int kv_dtype) {
  const int64_t n = split_max_chunks(max_len, head_dim, kv_dtype);
  if (n == 1) return 0;
  return static_cast<size_t>(rows * n) * (head_dim + 2) * sizeof(float);
}

cudaError_t launch_split_attention(const SplitArgs& args, int q_dtype, int kv_dtype, void* workspace,
                                   cudaStream_t stream) {
  SplitArgs a = args;
  a.group = a.H / a.Hk;
  a.rows = a.group * a.S;
  a.block_rows = a.rows > 8 ? 16 : 8;
  a.row_chunks = (a.rows + a.block_rows - 1) / a.block_rows;
  a.max_chunks = split_max_chunks(a.max_len, a.D, kv_dtype);
  a.tile_log = tile_log_of(a.D, kv_dtype);
  // key / page for key < 2^31: key mul >> shift, mul = ceil(2^shift / page), 2^shift >= 2^31 page.
  if (!a.table) a.page = 1;
  a.page_shift = 31;
  while ((int64_t(1) << (a.page_shift - 31)) < a.page) ++a.page_shift;
  a.page_mul = static_cast<uint32_t>(((uint64_t(1) << a.page_shift) + a.page - 1) / a.page);
  a.one_page = !a.table || a.page % (1 << a.tile_log) == 0;
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = a.max_chunks == 1
                  ? nullptr
                  : reinterpret_cast<float2*>(a.part_o + static_cast<int64_t>(a.B) * a.H * a.S *
                                                             a.max_chunks * a.D);
  if (a.D == 32) return launch_d<32>(a, q_dtype, kv_dtype, stream);
  if (a.D == 64) return launch_d<64>(a, q_dtype, kv_dtype, stream);
  return launch_d<128>(a, q_dtype, kv_dtype, stream);
}

}  // namespace cfa
