// SPDX-License-Identifier: MIT OR Apache-2.0
//
// Internal launch interface of the operators beside the fused attention: rotary positions, the
// paged cache's append and the split attention of few query rows. Host-only types.
#pragma once

#include <cstddef>
#include <cstdint>
#include <cuda_runtime.h>

#include "cfa.h"

namespace cfa {

// Strides in elements. Rotary: x -> y over [B, H, S, D]. Append: q (x -> y, H = 0: none), k and v
// [B, Hk, S, D] into the caches.
struct RotaryArgs {
  const void* x;
  void* y;
  int64_t x_sb, x_sh, x_ss, y_sb, y_sh, y_ss;
  const double* freqs;  // [rot / 2] radians a position
  float amplitude;
  int inverse, interleaved;
  int B, H, rot_heads, S, D, rot;
  const void* pos;  // rotary: positions (pos64: int64, else int32), or nullptr: pos0 + index
  int pos64;
  int64_t pos_sb, pos_ss, pos0;
  // append
  const void* k;
  const void* v;
  int64_t k_sb, k_sh, k_ss, v_sb, v_sh, v_ss;
  int Hk;
  void* k_cache;
  void* v_cache;
  int64_t kc_sp, kc_sr, kc_sh, vc_sp, vc_sr, vc_sh;  // page, row in the page, head
  const int* table;                                  // [B][table_width]
  int64_t table_sb;
  int table_width, n_pages, page;
  const int* lengths;
  const int* new_lengths;  // or nullptr: S each
  int* sink;
  // set by the launcher
  int64_t n_tokens;  // (set by the caller: B S)
  int tokens, units, head_step;
  int pairs;  // rows aligned to two vectors: adjacent ones move as one access
  uint32_t div_units, div_heads;
};
cudaError_t launch_rotary(const RotaryArgs& p, int dtype, cudaStream_t stream);
cudaError_t launch_paged_append(const RotaryArgs& p, int dtype, int cache_dtype,
                                cudaStream_t stream);

// Attention of few query rows a key head over many keys, split over the keys and joined.
struct SplitArgs {
  const void* q;
  int64_t q_sb, q_sh, q_ss;
  const void* k;
  const void* v;
  // Paged (table set): strides of page, row in the page, head. Dense: batch, row, head.
  int64_t k_sp, k_sr, k_sh, v_sp, v_sr, v_sh;
  const int* table;
  int64_t table_sb;
  int table_width, n_pages, page;
  const int* lengths;      // [B] keys of each sequence, or nullptr: max_len
  const int* new_lengths;  // [B] query rows in use, or nullptr: S
  int causal;              // query i of n sees lengths - n + i + 1 keys, else all of them
  int max_len;             // most keys of a sequence (lengths beyond are cut)
  void* o;                 // [B, S, H, D] dense
  float* lse;              // [B, H, S] or nullptr: the rows' log-sum-exp
  int B, H, Hk, S, D;
  float scale;
  int* sink;
  // set by the launcher
  int group, rows, block_rows, row_chunks, max_chunks;  // rows of a key head, of a block; blocks of them
  uint32_t page_mul;  // key / page = key page_mul >> page_shift
  int page_shift;
  int one_page;       // every tile of keys lies on one page
  int tile_log;       // log2 of the keys of a tile
  float* part_o;   // [B H S][max_chunks][D] unnormalised partial outputs
  float2* part_ml; // [B H S][max_chunks] running maximum and sum
};
int split_max_chunks(int64_t max_len, int64_t head_dim, int kv_dtype);
size_t split_workspace_bytes(int64_t rows, int64_t max_len, int64_t head_dim, int kv_dtype);
cudaError_t setup_split_attributes();
cudaError_t launch_split_attention(const SplitArgs& a, int q_dtype, int kv_dtype, void* workspace,
                                   cudaStream_t stream);

}  // namespace cfa
