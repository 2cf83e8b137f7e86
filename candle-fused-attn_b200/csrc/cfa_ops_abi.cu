// SPDX-License-Identifier: MIT OR Apache-2.0
//
// The C ABI of the operators beside the fused attention (include/cfa.h): cross attention, rotary
// positions, the paged cache's append and its attention. Argument checks and launches, as
// cfa_abi.cu does for the fused attention; everything on the caller's stream, no synchronisation.
#include <algorithm>
#include <mutex>

#include "cfa_internal.h"
#include "cfa_ops.h"

namespace {

constexpr int kMaxDevices = 64;
struct DeviceOnce {
  std::once_flag flag;
  cudaError_t result = cudaSuccess;
};
DeviceOnce g_cross_once[kMaxDevices], g_split_once[kMaxDevices];

int setup(DeviceOnce* table, cudaError_t (*fn)()) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return CFA_ERR_CUDA;
  DeviceOnce& d = table[dev];
  std::call_once(d.flag, [&] { d.result = fn(); });
  return d.result == cudaSuccess ? CFA_OK : CFA_ERR_LAUNCH;
}

cudaError_t setup_cross() {
  cudaError_t e = cfa::setup_cross_tc_attributes();
  if (e == cudaSuccess) e = cfa::setup_cross_bwd_tc_attributes();
  if (e == cudaSuccess) e = cfa::setup_cross_hd_attributes();
  return e == cudaSuccess ? cfa::setup_cross_few_bwd_attributes() : e;
}

constexpr int64_t kLim = (int64_t(1) << 31) - 1;

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool strides_ok(const int64_t* s, int64_t unit) {
  return s[0] % unit == 0 && s[1] % unit == 0 && s[2] % unit == 0;
}
bool type_ok(int t) { return t == CFA_F32 || t == CFA_F16 || t == CFA_BF16; }
// Input and cache types: the same, or an fp32 input over any cache.
bool types_ok(int t, int cache) { return type_ok(t) && type_ok(cache) && (t == cache || t == CFA_F32); }
int64_t type_size(int t) { return t == CFA_F32 ? 4 : 2; }
bool head_dim_ok(int64_t d) { return d == 32 || d == 64 || d == 128; }
int status(cudaError_t e) {
  if (e == cudaSuccess) return CFA_OK;
  return e == cudaErrorInvalidConfiguration ? CFA_ERR_OVERFLOW : CFA_ERR_LAUNCH;
}

// The split attention's units (chunks x key heads x rows of 8) fit 31 bits.
bool split_units_ok(int64_t B, int64_t H, int64_t Hk, int64_t S, int64_t max_len, int64_t D, int kv) {
  const int64_t chunks = B * cfa::split_max_chunks(max_len, D, kv);
  const int64_t per = Hk * ((H / Hk * S + 7) / 8);
  return chunks <= kLim && per <= kLim && chunks <= kLim / per;
}

// B, H, Hk, Sq, Sk of a cross attention.
int check_cross(int64_t B, int64_t H, int64_t Hk, int64_t Sq, int64_t Sk, int64_t D) {
  if (B < 0 || H < 0 || Hk < 0 || Sq < 0 || Sk < 0 || D < 0) return CFA_ERR_SHAPE;
  if (!head_dim_ok(D)) return CFA_ERR_HEAD_DIM;
  if (Hk == 0 ? H != 0 : H % Hk != 0) return CFA_ERR_HEADS;
  if (B > kLim || H > kLim || Hk > kLim || Sq > kLim - 1024 || Sk > kLim - 1024) return CFA_ERR_OVERFLOW;
  if (B == 0 || Hk == 0) return CFA_OK;
  if (B * Hk > kLim / ((Sk + 31) / 32 + 1)) return CFA_ERR_OVERFLOW;
  if (B * H > kLim / ((std::max(Sq, Sk) + 31) / 32 + 1)) return CFA_ERR_OVERFLOW;
  if (B * H * Sq > kLim || B * Hk * Sk > kLim) return CFA_ERR_OVERFLOW;
  if (B * Hk * ((Sk + 63) / 64) > kLim / cfa::LIN_SMS) return CFA_ERR_OVERFLOW;  // key blocks x parts
  return CFA_OK;
}

// The cross backward's workspace: ticket and error flag, turn counters, the slices' tickets (one cleared
// range), D, where the query tiles are cut into parts a slice's dK, dV, and, in a workspace of `total_fast`, the dQ partials. The
// parts follow from the shapes of one batch element: no sum depends on the batch.
// dQ by partials (up to 4 GB of them) or by the turn chain, whose blocks wait for one another: the same
// sums in the same order, but at [4, 16 over 4, 2048 x 8192, 64] 4.53 ms against 6.61, at 470 rows over
// 6990 keys 157 us against 311.
constexpr int64_t kCrossPartialBytes = int64_t(4) << 30;
// Most dQ partials of a (batch, key head) that its last block sums; more are summed by the join kernel. Last
// block and join, in us, backward alone, at 64 dims: 256 KB [16, 8, 512 x 256] 107 and 106, 300 KB [64, 6, 240 x
// 600] 378 and 374, the same over 100 to 600 keys 272 and 279, 375 KB [64, 6, 300 x 640] 444 and 437, 384 KB
// [8, 8, 384 x 512] 83 and 79, 512 KB [8, 8, 512 x 512] 103 and 97, [8, 8 over 2, 128 x 512] 54 and 57, 1 MB
// [4, 8, 512 x 1024] 113 and 96. At 128 dims always the join: 400 KB [32, 8, 200 x 256] 517 and 457, 480 KB [64,
// 6, 240 x 240] 761 and 719, 512 KB [32, 8, 128 x 512] 540 and 491, 2 MB [16, 8, 512 x 512] 1027 and 880.
constexpr int64_t kCrossJoinBytes = 320 << 10;
// Fewest query tiles of a part: each reads its keys again. With 4, 8, 16 and without parts: [1, 8 over 2,
// 700 x 300, 64] 32, 51, 103 and 192 us; [8, 8, 512 x 512, 64] 122, 106, 106, 106; [2, 16 over 1, 1024 x
// 1024, 64] 215, 215, 176, 1023.
constexpr int kCrossPartTiles = 8;
// Most bytes of the parts' dK and dV: with more (one part of 19 a batch element of [64, 16 over 1, 1024 x
// 1024, 64] takes 0.5 MB, the batch 638), the batch goes in slices that use the same memory one after another,
// the same bits as each element's are its own. A slice of that size is still many times what the SMs take at once.
constexpr int64_t kCrossPartsBytes = int64_t(512) << 20;
struct CrossLayout {
  int64_t n_zero;  // ints cleared before the backward
  size_t turn_off, dsum_off, kv_off, part_off, total, total_fast;
  bool join_dq;    // (with the partials)
  int n_parts;
  int64_t slice, tickets;  // batch elements of a launch; where the slices' tickets are, in ints
  bool few;
};
CrossLayout cross_layout(int64_t B, int64_t H, int64_t Hk, int64_t Sq, int64_t Sk, int64_t D) {
  CrossLayout w{};
  const int64_t kb = D == 128 ? 64 : 128, nkb = (Sk + kb - 1) / kb;
  const int64_t group = H / Hk, tiles = (group * Sq + 63) / 64;
  // A batch element with fewer key blocks than the GPU has SMs: parts of at least 8 tiles that give
  // it as many blocks.
  const int64_t want = (cfa::LIN_SMS + nkb * Hk - 1) / (nkb * Hk);
  w.n_parts = static_cast<int>(std::max<int64_t>(1, std::min(want, tiles / kCrossPartTiles)));
  const int64_t row_bytes = nkb * D * 4;  // of one query's dQ partials (below 2^34)
  w.join_dq = w.n_parts > 1 || D == 128 || group * Sq > kCrossJoinBytes / row_bytes;
  w.turn_off = 256;
  const int64_t turns = B * Hk * tiles;
  const int64_t parts = w.n_parts > 1 ? w.n_parts * Sk * 2 * Hk * D * 4 : 0;  // bytes of an element's (< 2^50)
  w.slice = parts == 0 ? B : std::max<int64_t>(1, std::min(B, kCrossPartsBytes / parts));
  const int64_t slices = (B + w.slice - 1) / w.slice;
  w.tickets = slices == 1 ? 0 : 64 + turns;
  const int64_t counters = turns + (slices == 1 ? 0 : slices);
  w.n_zero = 64 + counters;
  w.dsum_off = w.turn_off + cfa::align256(static_cast<size_t>(counters) * 4);
  w.kv_off = w.dsum_off + cfa::align256(static_cast<size_t>(B * H * Sq) * 4);
  w.total = w.kv_off + static_cast<size_t>(w.slice * parts);
  w.part_off = w.total;
  const int64_t queries = B * H * Sq;
  w.total_fast = w.total + (queries <= kCrossPartialBytes / row_bytes ? static_cast<size_t>(queries * row_bytes) : 0);
  // Few query rows: by partials alone (at most a quarter of what the key blocks' keys and values take).
  w.few = group * Sq <= cfa::CROSS_FEW_ROWS;
  if (w.few) w.total = w.total_fast = w.part_off + static_cast<size_t>(queries * row_bytes);
  return w;
}

}  // namespace

extern "C" {

int cfa_cross_fwd_f32(const float* q, const int64_t q_strides[3], const float* k,
                      const int64_t k_strides[3], const float* v, const int64_t v_strides[3],
                      const int32_t* key_lengths, float* o, float* lse, int64_t batch, int64_t heads,
                      int64_t key_heads, int64_t seq, int64_t key_seq, int64_t head_dim, float scale,
                      void* stream) {
  int st = check_cross(batch, heads, key_heads, seq, key_seq, head_dim);
  if (st != CFA_OK || batch == 0 || heads == 0 || seq == 0) return st;
  if (!q || !o || !lse || !q_strides || !k_strides || !v_strides || (key_seq > 0 && (!k || !v)))
    return CFA_ERR_NULL;
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(o) || !strides_ok(q_strides, 4) ||
      !strides_ok(k_strides, 4) || !strides_ok(v_strides, 4))
    return CFA_ERR_ALIGNMENT;
  st = setup(g_cross_once, setup_cross);
  if (st != CFA_OK) return st;
  cfa::FwdArgs a{};
  a.q = q, a.k = k, a.v = v, a.o = o, a.lse = lse;
  a.q_sb = q_strides[0], a.q_sh = q_strides[1], a.q_ss = q_strides[2];
  a.k_sb = k_strides[0], a.k_sh = k_strides[1], a.k_ss = k_strides[2];
  a.v_sb = v_strides[0], a.v_sh = v_strides[1], a.v_ss = v_strides[2];
  a.B = static_cast<int>(batch), a.H = static_cast<int>(heads), a.S = static_cast<int>(seq);
  a.Hk = static_cast<int>(key_heads), a.Sk = static_cast<int>(key_seq);
  a.key_lengths = key_lengths;
  a.scale = scale;
  a.sink = cfa::error_sink();
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  return status(head_dim == 128 ? cfa::launch_cross_hd_fwd(a, s)
                                : cfa::launch_cross_fwd_tc(a, static_cast<int>(head_dim), s));
}

size_t cfa_cross_bwd_workspace_bytes(int64_t batch, int64_t heads, int64_t key_heads, int64_t seq,
                                     int64_t key_seq, int64_t head_dim) {
  if (check_cross(batch, heads, key_heads, seq, key_seq, head_dim) != CFA_OK || batch == 0 ||
      heads == 0 || seq == 0 || key_seq == 0)
    return 256;
  return cross_layout(batch, heads, key_heads, seq, key_seq, head_dim).total;
}

size_t cfa_cross_bwd_workspace_bytes_fast(int64_t batch, int64_t heads, int64_t key_heads, int64_t seq,
                                          int64_t key_seq, int64_t head_dim) {
  if (check_cross(batch, heads, key_heads, seq, key_seq, head_dim) != CFA_OK || batch == 0 ||
      heads == 0 || seq == 0 || key_seq == 0)
    return 256;
  return cross_layout(batch, heads, key_heads, seq, key_seq, head_dim).total_fast;
}

int cfa_cross_bwd_f32(const float* q, const int64_t q_strides[3], const float* k,
                      const int64_t k_strides[3], const float* v, const int64_t v_strides[3],
                      const int32_t* key_lengths, const float* o, const float* lse, const float* d_o,
                      const int64_t do_strides[3], float* dq, float* dkv, void* workspace,
                      size_t workspace_bytes, int64_t batch, int64_t heads, int64_t key_heads,
                      int64_t seq, int64_t key_seq, int64_t head_dim, float scale, void* stream) {
  int st = check_cross(batch, heads, key_heads, seq, key_seq, head_dim);
  if (st != CFA_OK) return st;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int64_t queries = heads * seq, keys = key_heads * key_seq;
  if (batch == 0 || queries == 0 || keys == 0) {  // no score at all: the gradients that exist are zero
    if (batch == 0 || queries == keys) return CFA_OK;
    float* g = queries == 0 ? dkv : dq;
    const int64_t n = batch * (queries == 0 ? 2 * keys : queries);
    if (!g) return CFA_ERR_NULL;
    return status(cudaMemsetAsync(g, 0, static_cast<size_t>(n * head_dim) * 4, s));
  }
  if (!q || !k || !v || !o || !lse || !d_o || !dq || !dkv || !workspace || !q_strides || !k_strides ||
      !v_strides || !do_strides)
    return CFA_ERR_NULL;
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(o) || !aligned16(d_o) ||
      !aligned16(dq) || !aligned16(dkv) || !strides_ok(q_strides, 4) || !strides_ok(k_strides, 4) ||
      !strides_ok(v_strides, 4) || !strides_ok(do_strides, 4))
    return CFA_ERR_ALIGNMENT;
  const CrossLayout lay = cross_layout(batch, heads, key_heads, seq, key_seq, head_dim);
  if (workspace_bytes < lay.total || (reinterpret_cast<uintptr_t>(workspace) & 255u) != 0)
    return CFA_ERR_WORKSPACE;
  st = setup(g_cross_once, setup_cross);
  if (st != CFA_OK) return st;
  char* ws = static_cast<char*>(workspace);
  int* ticket = reinterpret_cast<int*>(ws);

  cfa::PrepArgs p{};
  p.o = o, p.d_o = d_o;
  p.dsum = reinterpret_cast<float*>(ws + lay.dsum_off);
  p.zero = ticket;
  p.n_zero = lay.n_zero;
  p.do_sb = do_strides[0], p.do_sh = do_strides[1], p.do_ss = do_strides[2];
  p.B = static_cast<int>(batch), p.H = static_cast<int>(heads), p.S = static_cast<int>(seq);
  cudaError_t e = head_dim == 64 ? cfa::launch_bwd_prep(p, s)
                                 : cfa::launch_hd_bwd_prep(p, static_cast<int>(head_dim), s);
  if (e != cudaSuccess) return status(e);

  // The dQ partials when the workspace holds them (the same results, bit for bit).
  const bool partials = lay.few || (lay.total_fast > lay.total && workspace_bytes >= lay.total_fast);
  const int64_t kb = head_dim == 128 ? 64 : 128, nkb = (key_seq + kb - 1) / kb;
  const int64_t tiles = (heads / key_heads * seq + 63) / 64;
  const int64_t dkv_size = key_seq * 2 * key_heads * head_dim;  // floats of a batch element's
  for (int64_t b0 = 0, i = 0; b0 < batch; b0 += lay.slice, ++i) {
    cfa::BwdArgs a{};
    a.q = q + b0 * q_strides[0], a.k = k + b0 * k_strides[0], a.v = v + b0 * v_strides[0];
    a.d_o = d_o + b0 * do_strides[0];
    a.lse = lse + b0 * queries, a.dsum = p.dsum + b0 * queries;
    a.dq = dq + b0 * queries * head_dim;
    a.dkv = a.dkv_out = dkv + b0 * dkv_size;
    a.ticket = ticket + lay.tickets + (lay.tickets ? i : 0);
    a.err = ticket + 1;
    a.turn = reinterpret_cast<int*>(ws + lay.turn_off) + b0 * key_heads * tiles;
    a.q_sb = q_strides[0], a.q_sh = q_strides[1], a.q_ss = q_strides[2];
    a.k_sb = k_strides[0], a.k_sh = k_strides[1], a.k_ss = k_strides[2];
    a.v_sb = v_strides[0], a.v_sh = v_strides[1], a.v_ss = v_strides[2];
    a.do_sb = do_strides[0], a.do_sh = do_strides[1], a.do_ss = do_strides[2];
    const int64_t n = std::min(lay.slice, batch - b0);
    a.B = static_cast<int>(n), a.H = static_cast<int>(heads), a.S = static_cast<int>(seq);
    a.Hk = static_cast<int>(key_heads), a.Sk = static_cast<int>(key_seq);
    a.key_lengths = key_lengths ? key_lengths + b0 : nullptr;
    a.scale = scale;
    a.n_qtiles = static_cast<int>((seq + 63) / 64);
    a.timeout_ns = cfa::WAIT_TIMEOUT_NS;
    a.sink = cfa::error_sink();
    a.dq_part = partials ? reinterpret_cast<float*>(ws + lay.part_off) + b0 * queries * nkb * head_dim : nullptr;
    a.n_parts = lay.n_parts;
    a.join_dq = lay.few || (partials && lay.join_dq);
    if (lay.n_parts > 1) {
      a.dkv = reinterpret_cast<float*>(ws + lay.kv_off);
      a.part_stride = n * dkv_size;
    }
    e = lay.few            ? cfa::launch_cross_few_bwd(a, static_cast<int>(head_dim), s)
        : head_dim == 128  ? cfa::launch_cross_hd_bwd(a, s)
                           : cfa::launch_cross_bwd_tc(a, static_cast<int>(head_dim), s);
    if (e != cudaSuccess) return status(e);
  }
  return CFA_OK;
}

size_t cfa_cross_few_workspace_bytes(int64_t batch, int64_t heads, int64_t seq, int64_t key_seq,
                                     int64_t head_dim) {
  if (batch <= 0 || heads <= 0 || seq <= 0 || key_seq <= 0 || !head_dim_ok(head_dim) ||
      batch > kLim || heads > kLim || seq > kLim || key_seq > kLim - 1024 || batch * heads > kLim / seq)
    return 0;
  return cfa::split_workspace_bytes(batch * heads * seq, key_seq, head_dim, CFA_F32);
}

int cfa_cross_few_f32(const float* q, const int64_t q_strides[3], const float* k,
                      const int64_t k_strides[3], const float* v, const int64_t v_strides[3],
                      const int32_t* key_lengths, float* o, float* lse, void* workspace,
                      size_t workspace_bytes, int64_t batch, int64_t heads, int64_t key_heads, int64_t seq,
                      int64_t key_seq, int64_t head_dim, float scale, void* stream) {
  int st = check_cross(batch, heads, key_heads, seq, key_seq, head_dim);
  if (st != CFA_OK || batch == 0 || heads == 0 || seq == 0) return st;
  const size_t need = cfa_cross_few_workspace_bytes(batch, heads, seq, key_seq, head_dim);
  if (!q || !o || !q_strides || !k_strides || !v_strides || (key_seq > 0 && (!k || !v)) ||
      (need > 0 && !workspace))
    return CFA_ERR_NULL;
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !strides_ok(q_strides, 4) ||
      !strides_ok(k_strides, 4) || !strides_ok(v_strides, 4))
    return CFA_ERR_ALIGNMENT;
  if (workspace_bytes < need || (need && (reinterpret_cast<uintptr_t>(workspace) & 255u) != 0))
    return CFA_ERR_WORKSPACE;
  if (!split_units_ok(batch, heads, key_heads, seq, key_seq, head_dim, CFA_F32)) return CFA_ERR_OVERFLOW;
  st = setup(g_split_once, cfa::setup_split_attributes);
  if (st != CFA_OK) return st;
  cfa::SplitArgs a{};
  a.q = q, a.k = k, a.v = v, a.o = o, a.lse = lse;
  a.q_sb = q_strides[0], a.q_sh = q_strides[1], a.q_ss = q_strides[2];
  a.k_sp = k_strides[0], a.k_sh = k_strides[1], a.k_sr = k_strides[2];
  a.v_sp = v_strides[0], a.v_sh = v_strides[1], a.v_sr = v_strides[2];
  a.lengths = key_lengths;
  a.max_len = static_cast<int>(key_seq);
  a.B = static_cast<int>(batch), a.H = static_cast<int>(heads), a.Hk = static_cast<int>(key_heads);
  a.S = static_cast<int>(seq), a.D = static_cast<int>(head_dim);
  a.scale = scale;
  return status(cfa::launch_split_attention(a, CFA_F32, CFA_F32, workspace,
                                            static_cast<cudaStream_t>(stream)));
}

int cfa_rotary(const void* x, const int64_t x_strides[3], void* y, const int64_t y_strides[3],
               int dtype, const void* positions, int position_bytes, const int64_t position_strides[2],
               int64_t first_position, const double* freqs, float amplitude, int64_t batch,
               int64_t heads, int64_t rotated_heads, int64_t seq, int64_t head_dim,
               int64_t rotary_dim, int interleaved, int inverse, void* stream) {
  if (batch < 0 || heads < 0 || seq < 0 || head_dim < 0 || rotated_heads < 0 || rotated_heads > heads)
    return CFA_ERR_SHAPE;
  if (rotary_dim < 0 || rotary_dim % 2 != 0 || rotary_dim > head_dim) return CFA_ERR_ROTARY;
  if (head_dim > 1024) return CFA_ERR_HEAD_DIM;
  if (!type_ok(dtype) || (positions && position_bytes != 4 && position_bytes != 8)) return CFA_ERR_TYPE;
  if (batch == 0 || heads == 0 || seq == 0 || head_dim == 0) return CFA_OK;
  if (batch > kLim || heads > kLim || seq > kLim || batch > kLim / seq) return CFA_ERR_OVERFLOW;
  if (!x || !y || !x_strides || !y_strides || (positions && !position_strides) ||
      (rotary_dim > 0 && !freqs))
    return CFA_ERR_NULL;
  cfa::RotaryArgs a{};
  a.x = x, a.y = y;
  a.x_sb = x_strides[0], a.x_sh = x_strides[1], a.x_ss = x_strides[2];
  a.y_sb = y_strides[0], a.y_sh = y_strides[1], a.y_ss = y_strides[2];
  a.freqs = freqs;
  a.amplitude = amplitude;
  a.interleaved = interleaved != 0, a.inverse = inverse != 0;
  a.B = static_cast<int>(batch), a.H = static_cast<int>(heads), a.S = static_cast<int>(seq);
  a.rot_heads = static_cast<int>(rotated_heads);
  a.D = static_cast<int>(head_dim), a.rot = static_cast<int>(rotary_dim);
  a.pos = positions;
  a.pos64 = position_bytes == 8;
  if (positions) a.pos_sb = position_strides[0], a.pos_ss = position_strides[1];
  a.pos0 = first_position;
  a.n_tokens = batch * seq;
  return status(cfa::launch_rotary(a, dtype, static_cast<cudaStream_t>(stream)));
}

int cfa_paged_append(const void* q, const int64_t q_strides[3], void* q_out,
                     const int64_t q_out_strides[3], const void* k, const int64_t k_strides[3],
                     const void* v, const int64_t v_strides[3], int dtype, void* k_cache,
                     const int64_t k_cache_strides[3], void* v_cache,
                     const int64_t v_cache_strides[3], int cache_dtype, int64_t pages,
                     int64_t page_size, const int32_t* page_table, int64_t table_stride,
                     int64_t table_width, const int32_t* lengths, const int32_t* new_lengths,
                     const double* freqs, float amplitude, int64_t batch, int64_t heads,
                     int64_t key_heads, int64_t seq, int64_t head_dim, int64_t rotary_dim,
                     int interleaved, void* stream) {
  if (batch < 0 || heads < 0 || key_heads < 0 || seq < 0 || head_dim < 0 || pages < 0 ||
      table_width < 0 || page_size < 1)
    return CFA_ERR_SHAPE;
  if (rotary_dim < 0 || rotary_dim % 2 != 0 || rotary_dim > head_dim) return CFA_ERR_ROTARY;
  if (head_dim > 1024) return CFA_ERR_HEAD_DIM;
  if (!types_ok(dtype, cache_dtype)) return CFA_ERR_TYPE;
  if (!q) heads = 0;
  if (batch == 0 || seq == 0 || head_dim == 0 || (heads == 0 && key_heads == 0)) return CFA_OK;
  if (batch > kLim || seq > kLim || batch > kLim / seq || heads + 2 * key_heads > kLim ||
      pages > kLim || page_size > kLim || table_width > kLim)
    return CFA_ERR_OVERFLOW;
  if ((q && (!q_out || !q_strides || !q_out_strides)) || !k || !v || !k_strides || !v_strides ||
      !k_cache || !v_cache || !k_cache_strides || !v_cache_strides ||
      (table_width > 0 && !page_table) || !lengths || (rotary_dim > 0 && !freqs))
    return CFA_ERR_NULL;
  cfa::RotaryArgs a{};
  if (q) {
    a.x = q, a.y = q_out;
    a.x_sb = q_strides[0], a.x_sh = q_strides[1], a.x_ss = q_strides[2];
    a.y_sb = q_out_strides[0], a.y_sh = q_out_strides[1], a.y_ss = q_out_strides[2];
  }
  a.k = k, a.v = v;
  a.k_sb = k_strides[0], a.k_sh = k_strides[1], a.k_ss = k_strides[2];
  a.v_sb = v_strides[0], a.v_sh = v_strides[1], a.v_ss = v_strides[2];
  a.k_cache = k_cache, a.v_cache = v_cache;
  a.kc_sp = k_cache_strides[0], a.kc_sr = k_cache_strides[1], a.kc_sh = k_cache_strides[2];
  a.vc_sp = v_cache_strides[0], a.vc_sr = v_cache_strides[1], a.vc_sh = v_cache_strides[2];
  a.table = page_table;
  a.table_sb = table_stride;
  a.table_width = static_cast<int>(table_width), a.n_pages = static_cast<int>(pages);
  a.page = static_cast<int>(page_size);
  a.lengths = lengths, a.new_lengths = new_lengths;
  a.freqs = freqs;
  a.amplitude = amplitude;
  a.interleaved = interleaved != 0;
  a.B = static_cast<int>(batch), a.H = static_cast<int>(heads), a.Hk = static_cast<int>(key_heads);
  a.rot_heads = a.H;
  a.S = static_cast<int>(seq), a.D = static_cast<int>(head_dim), a.rot = static_cast<int>(rotary_dim);
  a.n_tokens = batch * seq;
  a.sink = cfa::page_sink();
  return status(cfa::launch_paged_append(a, dtype, cache_dtype, static_cast<cudaStream_t>(stream)));
}

size_t cfa_paged_attention_workspace_bytes(int64_t batch, int64_t heads, int64_t seq,
                                           int64_t max_keys, int64_t head_dim, int cache_dtype) {
  if (batch <= 0 || heads <= 0 || seq <= 0 || max_keys <= 0 || !head_dim_ok(head_dim) ||
      !type_ok(cache_dtype) || batch > kLim || heads > kLim || seq > kLim || max_keys > kLim - 1024 ||
      batch * heads > kLim / seq)
    return 0;
  return cfa::split_workspace_bytes(batch * heads * seq, max_keys, head_dim, cache_dtype);
}

int cfa_paged_attention(const void* q, const int64_t q_strides[3], int dtype, const void* k_cache,
                        const int64_t k_cache_strides[3], const void* v_cache,
                        const int64_t v_cache_strides[3], int cache_dtype, int64_t pages,
                        int64_t page_size, const int32_t* page_table, int64_t table_stride,
                        int64_t table_width, const int32_t* lengths, const int32_t* new_lengths,
                        void* o, void* workspace, size_t workspace_bytes, int64_t batch,
                        int64_t heads, int64_t key_heads, int64_t seq, int64_t head_dim,
                        float scale, void* stream) {
  if (batch < 0 || heads < 0 || key_heads < 0 || seq < 0 || head_dim < 0 || pages < 0 ||
      table_width < 0 || page_size < 1)
    return CFA_ERR_SHAPE;
  if (!head_dim_ok(head_dim)) return CFA_ERR_HEAD_DIM;
  if (key_heads == 0 ? heads != 0 : heads % key_heads != 0) return CFA_ERR_HEADS;
  if (!types_ok(dtype, cache_dtype)) return CFA_ERR_TYPE;
  if (batch == 0 || heads == 0 || seq == 0) return CFA_OK;
  if (batch > kLim || heads > kLim || seq > kLim || batch * heads > kLim / seq || pages > kLim ||
      page_size > kLim || table_width > kLim || table_width * page_size > kLim - 1024)
    return CFA_ERR_OVERFLOW;
  const int64_t max_keys = table_width * page_size;
  const size_t need = cfa_paged_attention_workspace_bytes(batch, heads, seq, max_keys, head_dim, cache_dtype);
  if (!q || !o || !q_strides || !k_cache_strides || !v_cache_strides || !lengths ||
      (max_keys > 0 && (!k_cache || !v_cache || !page_table)) || (need > 0 && !workspace))
    return CFA_ERR_NULL;
  const int64_t unit = 16 / type_size(cache_dtype);
  if (!aligned16(q) || !aligned16(k_cache) || !aligned16(v_cache) ||
      !strides_ok(q_strides, 16 / type_size(dtype)) || !strides_ok(k_cache_strides, unit) ||
      !strides_ok(v_cache_strides, unit))
    return CFA_ERR_ALIGNMENT;
  if (workspace_bytes < need || (need && (reinterpret_cast<uintptr_t>(workspace) & 255u) != 0))
    return CFA_ERR_WORKSPACE;
  if (!split_units_ok(batch, heads, key_heads, seq, max_keys, head_dim, cache_dtype))
    return CFA_ERR_OVERFLOW;
  const int st = setup(g_split_once, cfa::setup_split_attributes);
  if (st != CFA_OK) return st;
  cfa::SplitArgs a{};
  a.q = q, a.k = k_cache, a.v = v_cache, a.o = o;
  a.q_sb = q_strides[0], a.q_sh = q_strides[1], a.q_ss = q_strides[2];
  a.k_sp = k_cache_strides[0], a.k_sr = k_cache_strides[1], a.k_sh = k_cache_strides[2];
  a.v_sp = v_cache_strides[0], a.v_sr = v_cache_strides[1], a.v_sh = v_cache_strides[2];
  a.table = page_table;
  a.table_sb = table_stride;
  a.table_width = static_cast<int>(table_width), a.n_pages = static_cast<int>(pages);
  a.page = static_cast<int>(page_size);
  a.lengths = lengths, a.new_lengths = new_lengths;
  a.causal = 1;
  a.max_len = static_cast<int>(max_keys);
  a.B = static_cast<int>(batch), a.H = static_cast<int>(heads), a.Hk = static_cast<int>(key_heads);
  a.S = static_cast<int>(seq), a.D = static_cast<int>(head_dim);
  a.scale = scale;
  a.sink = cfa::page_sink();
  return status(cfa::launch_split_attention(a, dtype, cache_dtype, workspace,
                                            static_cast<cudaStream_t>(stream)));
}

}  // extern "C"
