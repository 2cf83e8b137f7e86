// SPDX-License-Identifier: MIT OR Apache-2.0
//
// _ops.so: the operators beside the fused attention (cross attention, rotary positions, the paged cache)
// as a Python extension over torch tensors: argument checks, outputs, workspaces, autograd nodes, and the
// calls of the C ABI (include/cfa.h). What the functions do is documented where Python shows them
// (cross.py, positions.py, paged.py).
//
// It is C++ because a decoding step's calls last as long as their host side: through Python and ctypes
// [64, 6, 1, 64] rotary took 15 us for 2 us on the GPU, a rotary forward and backward 102 us, most of it
// in the Python node's forward, backward and changes of thread.
//
// Errors are Python exceptions (FusedAttentionError), in a backward too; none leaves through a C entry.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>

#include <array>
#include <initializer_list>
#include <string>

#include "cfa.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// The library's entry points (of the one library that _abi.py loaded), the error class, and Python's
// side of failure detection: where its flag is, and what raises for it.
struct Abi {
  decltype(&cfa_cross_fwd_f32) cross_fwd;
  decltype(&cfa_cross_bwd_workspace_bytes) cross_bwd_least;
  decltype(&cfa_cross_bwd_workspace_bytes_fast) cross_bwd_workspace;
  decltype(&cfa_cross_bwd_f32) cross_bwd;
  decltype(&cfa_cross_few_workspace_bytes) cross_few_workspace;
  decltype(&cfa_cross_few_f32) cross_few;
  decltype(&cfa_rotary) rotary;
  decltype(&cfa_paged_append) paged_append;
  decltype(&cfa_paged_attention_workspace_bytes) paged_attention_workspace;
  decltype(&cfa_paged_attention) paged_attention;
  decltype(&cfa_strerror) strerror;
} abi;
PyObject *error_class, *flag_address, *raise_flag;
volatile int32_t* flag = nullptr;

struct Gil {
  PyGILState_STATE state = PyGILState_Ensure();
  ~Gil() { PyGILState_Release(state); }
};

[[noreturn]] void throw_python() {
  python_error e;
  e.persist();
  throw e;
}
[[noreturn]] void fail(const std::string& message) {
  Gil gil;
  PyErr_SetString(error_class, message.c_str());
  throw_python();
}
// Pieces of a message.
std::string text(const char* s) { return s; }
std::string text(int64_t n) { return std::to_string(n); }
std::string text(at::IntArrayRef sizes) {
  std::string s = "[";
  for (size_t i = 0; i < sizes.size(); ++i) s += (i ? ", " : "") + std::to_string(sizes[i]);
  return s + "]";
}
template <typename... A>
[[noreturn]] void fail_with(const A&... parts) {
  fail((text(parts) + ...));
}
#define REQUIRE(ok, ...) \
  do {                   \
    if (C10_UNLIKELY(!(ok))) fail_with(__VA_ARGS__); \
  } while (0)

// Before every launch, as the fused attention does: raises for a bad page or an expired wait of an
// earlier kernel. The flag is read as it stands.
void raise_if_expired() {
  if (C10_UNLIKELY(flag == nullptr)) {
    Gil gil;
    PyObject* address = PyObject_CallNoArgs(flag_address);
    if (!address) throw_python();
    flag = reinterpret_cast<volatile int32_t*>(PyLong_AsSize_t(address));
    Py_DECREF(address);
  }
  if (C10_UNLIKELY(*flag != 0)) {
    Gil gil;
    PyObject* none = PyObject_CallNoArgs(raise_flag);
    if (!none) throw_python();
    Py_DECREF(none);
  }
}
void check_status(int status, const char* who) {
  REQUIRE(status == CFA_OK, who, ": ", abi.strerror(status));
}

// --- checks ---------------------------------------------------------------------------------------

const char* type_name(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return "torch.float32";
    case at::kHalf: return "torch.float16";
    case at::kBFloat16: return "torch.bfloat16";
    case at::kDouble: return "torch.float64";
    case at::kInt: return "torch.int32";
    case at::kLong: return "torch.int64";
    default: return at::toString(t.scalar_type());
  }
}
// The ABI's number of a type, or -1.
int dtype_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return CFA_F32;
    case at::kHalf: return CFA_F16;
    case at::kBFloat16: return CFA_BF16;
    default: return -1;
  }
}
using Tensors = std::initializer_list<const Tensor*>;
void one_device(const char* who, Tensors ts) {
  const auto index = (*ts.begin())->get_device();
  bool same = index >= 0, cuda = true;
  for (const Tensor* t : ts)
    if (t->defined()) same &= t->get_device() == index, cuda &= t->is_cuda();
  REQUIRE(same, who, cuda ? ": tensors on different devices" : ": CUDA tensors required");
}
// A forward-mode tangent (torch.autograd.forward_ad) rides on a tensor without requires_grad: no result
// here would carry it on, which reads as a derivative of zero.
void no_tangent(const char* who, const char* what, Tensors ts) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const Tensor* t : ts)
    REQUIRE(!t->defined() || !t->_fw_grad(/*level=*/0).defined(), who, what,
            ": has no forward-mode derivative");
}
void no_gradient(const char* who, const char* what, Tensors ts) {
  no_tangent(who, what, ts);
  if (!at::GradMode::is_enabled()) return;
  for (const Tensor* t : ts)
    REQUIRE(!t->defined() || !t->requires_grad(), who, what,
            ": has no backward (call it under torch.no_grad())");
}
void int32_vector(const char* who, const char* name, const Tensor& t, int64_t n) {
  if (!t.defined()) return;
  REQUIRE(t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == n && (n <= 1 || t.stride(0) == 1),
          who, ": ", name, " must be a dense int32 tensor [", n, "], got ", type_name(t), " ", t.sizes());
}
void check_freqs(const char* who, const Tensor& f, int64_t d) {
  no_gradient(who, ": freqs", {&f});
  REQUIRE(f.scalar_type() == at::kDouble && f.dim() == 1 && (f.numel() <= 1 || f.stride(0) == 1), who,
          ": freqs must be a dense float64 vector, got ", type_name(f), " ", f.sizes());
  REQUIRE(2 * f.numel() <= d, who, ": ", f.numel(), " frequencies turn ", 2 * f.numel(),
          " dims, the head has ", d);
}
void check_head_dim(int64_t d) {
  REQUIRE(d == 32 || d == 64 || d == 128,
          "fused_attention: the CUDA kernels take head_dim 64 (and 32 or 128), got ", d);
}
// [b, h, s, d] operands of 16-byte rows.
bool aligned(const Tensor& t) {
  const int64_t unit = 16 / t.element_size();
  return t.stride(3) == 1 && reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0 &&
         t.stride(0) % unit == 0 && t.stride(1) % unit == 0 && t.stride(2) % unit == 0;
}
Tensor aligned_rows(const Tensor& t) {
  return aligned(t) ? t : t.clone(at::MemoryFormat::Contiguous);
}
// [b, h, s, d] with its last dim contiguous.
Tensor dense_rows(const Tensor& t) {
  return t.stride(3) == 1 || t.size(3) <= 1 ? t : t.contiguous();
}

// --- outputs and arguments of the ABI -------------------------------------------------------------

struct Strides3 {
  int64_t s[3];
  explicit Strides3(const Tensor& t) : s{t.stride(0), t.stride(1), t.stride(2)} {}
  Strides3(int64_t a, int64_t b, int64_t c) : s{a, b, c} {}
  operator const int64_t*() const { return s; }
};
template <typename T>
const T* ptr(const Tensor& t) {
  return t.defined() ? static_cast<const T*>(t.const_data_ptr()) : nullptr;
}
Tensor empty(at::IntArrayRef sizes, at::IntArrayRef strides, const Tensor& like, at::ScalarType type) {
  return at::detail::empty_strided_cuda(sizes, strides, type, like.device());
}
// [b, h, s, d] laid out as a dense [b, s, h, d] (merge-heads ready), of like's type.
Tensor merged_heads(int64_t b, int64_t h, int64_t s, int64_t d, const Tensor& like) {
  return empty({b, h, s, d}, {s * h * d, d, h * d, 1}, like, like.scalar_type());
}
Tensor workspace(size_t bytes, const Tensor& like) {
  return bytes ? empty({static_cast<int64_t>(bytes)}, {1}, like, at::kByte) : Tensor();
}
// The device of the operands as the current one, and its current stream.
struct Launch {
  c10::cuda::CUDAGuard guard;
  void* stream;
  explicit Launch(const Tensor& t)
      : guard(t.device()), stream(c10::cuda::getCurrentCUDAStream(t.device().index()).stream()) {
    raise_if_expired();
  }
};

// The gradients of a backward: where a graph of them is made (create_graph), one that says so when it is
// differentiated in its turn -- the kernels record nothing. `sources`: what the gradients depend on.
variable_list first_order(Tensors sources, variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  bool differentiable = false;
  for (const Tensor* t : sources) differentiable |= t->requires_grad();
  if (!differentiable) return grads;
  variable_list leaves;
  for (const Tensor& g : grads)
    if (g.defined()) leaves.push_back(g.detach().set_requires_grad(true));
  auto node = std::make_shared<torch::autograd::DelayedError>(
      "fused_attention: a gradient of this operator cannot be differentiated again", leaves.size());
  leaves = (*node)(std::move(leaves));
  size_t next = 0;
  for (Tensor& g : grads)
    if (g.defined()) g = leaves[next++];
  return grads;
}

// --- rotary positions -----------------------------------------------------------------------------

struct Turn {
  const char* who;
  Tensor positions;  // [b, s], or undefined: consecutive from `first`
  int64_t first;
  Tensor freqs;
  double amplitude;
  bool interleaved;
  int64_t heads;  // of a fused projection [b, s, 3 heads d]; 0: [b, h, s, d]
};
Tensor turn(const Tensor& x_, const Turn& t, bool inverse) {
  const Launch on(x_);
  const int64_t pos_strides[2] = {t.positions.defined() ? t.positions.stride(0) : 0,
                                  t.positions.defined() ? t.positions.stride(1) : 0};
  const int pos_bytes = t.positions.defined() ? static_cast<int>(t.positions.element_size()) : 0;
  auto run = [&](const Tensor& x, const int64_t* xs, const Tensor& y, const int64_t* ys, int64_t b, int64_t h,
                 int64_t rotated, int64_t s, int64_t d) {
    check_status(abi.rotary(x.const_data_ptr(), xs, y.mutable_data_ptr(), ys, dtype_of(x),
                            ptr<void>(t.positions), pos_bytes, pos_strides, t.first, ptr<double>(t.freqs),
                            static_cast<float>(t.amplitude), b, h, rotated, s, d, 2 * t.freqs.numel(),
                            t.interleaved, inverse, on.stream),
                 t.who);
  };
  if (t.heads == 0) {
    const Tensor x = dense_rows(x_);
    const int64_t b = x.size(0), h = x.size(1), s = x.size(2), d = x.size(3);
    const Tensor y = merged_heads(b, h, s, d, x);
    run(x, Strides3(x), y, Strides3(s * h * d, d, h * d), b, h, h, s, d);
    return y;
  }
  const Tensor x = x_.stride(2) == 1 ? x_ : x_.contiguous();
  const int64_t b = x.size(0), s = x.size(1), h = t.heads, d = x.size(2) / (3 * h), row = 3 * h * d;
  const Tensor y = empty(x.sizes(), {s * row, row, 1}, x, x.scalar_type());
  run(x, Strides3(x.stride(0), d, x.stride(1)), y, Strides3(s * row, d, row), b, 3 * h, 2 * h, s, d);
  return y;
}

// y = R x; dx = R^T dy, the inverse rotation with the same amplitude.
struct Rotary : torch::autograd::Function<Rotary> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Turn& t) {
    ctx->save_for_backward({t.freqs, t.positions});
    ctx->saved_data["first"] = t.first;
    ctx->saved_data["amplitude"] = t.amplitude;
    ctx->saved_data["layout"] = 2 * t.heads + t.interleaved;
    return turn(x, t, false);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const int64_t layout = ctx->saved_data["layout"].toInt();
    const Turn t{layout > 1 ? "rotary_qkv" : "rotary", saved[1], ctx->saved_data["first"].toInt(), saved[0],
                 ctx->saved_data["amplitude"].toDouble(), (layout & 1) != 0, layout / 2};
    return first_order({&grads[0]}, {turn(grads[0], t, true), Tensor()});  // (linear: no part of x in it)
  }
};
Tensor rotate(const Tensor& x, const Turn& t) {
  return at::GradMode::is_enabled() && x.requires_grad() ? Rotary::apply(x, t) : turn(x, t, false);
}

// --- cross attention ------------------------------------------------------------------------------

struct Dims {
  int64_t b, h, hk, sq, sk, d;
};
// Up to as many query rows a key head (query heads of a group x queries) the forward runs split over the
// keys, one block a chunk of keys and up to 16 rows; above, kernels that take 256 rows a block (64 at head
// dim 128). The batch plays no part: the choice changes bits. Split and whole, in us, [b, 6, rows, 64] over
// 1500 keys: 16 rows 11 and 55 (b 1), 23 and 58 (16), 82 and 169 (64); 32 rows 11 and 55, 42 and 58, 156 and
// 169; 48 rows 11 and 55, 60 and 58, 226 and 170.
constexpr int64_t kFewRows = 32;

Tensor cross_forward(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lengths, float scale,
                     const Dims& m, bool gradients, Tensor& lse) {
  const Launch on(q);
  const Tensor o = merged_heads(m.b, m.h, m.sq, m.d, q);
  const bool few = m.hk && m.h / m.hk * m.sq <= kFewRows;
  if (gradients || !few) lse = empty({m.b, m.h, m.sq}, {m.h * m.sq, m.sq, 1}, q, at::kFloat);
  float *const op = o.mutable_data_ptr<float>(), *const lp = lse.defined() ? lse.mutable_data_ptr<float>() : nullptr;
  if (few) {
    const size_t n = abi.cross_few_workspace(m.b, m.h, m.sq, m.sk, m.d);
    const Tensor ws = workspace(n, q);
    check_status(abi.cross_few(ptr<float>(q), Strides3(q), ptr<float>(k), Strides3(k), ptr<float>(v),
                               Strides3(v), ptr<int32_t>(lengths), op, lp, n ? ws.mutable_data_ptr() : nullptr,
                               n, m.b, m.h, m.hk, m.sq, m.sk, m.d, scale, on.stream),
                 "cross_attention");
    return o;
  }
  check_status(abi.cross_fwd(ptr<float>(q), Strides3(q), ptr<float>(k), Strides3(k), ptr<float>(v),
                             Strides3(v), ptr<int32_t>(lengths), op, lp, m.b, m.h, m.hk, m.sq, m.sk, m.d, scale,
                             on.stream),
               "cross_attention");
  return o;
}
struct Keys {  // (in one argument: an undefined tensor is none that a node's inputs may hold)
  Tensor lengths;
};
struct Cross : torch::autograd::Function<Cross> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v,
                        const Keys& keys, double scale, const Dims& m) {
    Tensor lse;
    const Tensor o = cross_forward(q, k, v, keys.lengths, static_cast<float>(scale), m, true, lse);
    ctx->save_for_backward({q, k, v, keys.lengths, o, lse});
    ctx->saved_data["scale"] = scale;
    return o;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &q = saved[0], &k = saved[1], &v = saved[2], &lengths = saved[3], &o = saved[4], &lse = saved[5];
    const Dims m{q.size(0), q.size(1), k.size(1), q.size(2), k.size(2), q.size(3)};
    const Launch on(q);
    const Tensor g = aligned_rows(grads[0].detach());
    const Tensor dq = merged_heads(m.b, m.h, m.sq, m.d, q);
    const int64_t row = 2 * m.hk * m.d;
    const Tensor dkv = empty({m.b, m.sk, 2, m.hk, m.d}, {m.sk * row, row, m.hk * m.d, m.d, 1}, q, at::kFloat);
    // With the dQ partials (up to 4 GB) or, where there is no room for them, without: the same bits.
    size_t n = abi.cross_bwd_workspace(m.b, m.h, m.hk, m.sq, m.sk, m.d);
    Tensor ws;
    try {
      ws = workspace(n, q);
    } catch (const c10::OutOfMemoryError&) {
      const size_t least = abi.cross_bwd_least(m.b, m.h, m.hk, m.sq, m.sk, m.d);
      if (least == n) throw;
      ws = workspace(n = least, q);
    }
    check_status(abi.cross_bwd(ptr<float>(q), Strides3(q), ptr<float>(k), Strides3(k), ptr<float>(v),
                               Strides3(v), ptr<int32_t>(lengths), ptr<float>(o), ptr<float>(lse),
                               ptr<float>(g), Strides3(g), dq.mutable_data_ptr<float>(),
                               dkv.mutable_data_ptr<float>(), ws.mutable_data_ptr(), n, m.b, m.h, m.hk, m.sq,
                               m.sk, m.d, static_cast<float>(ctx->saved_data["scale"].toDouble()), on.stream),
                 "cross_attention");
    const std::array<int64_t, 4> size{m.b, m.hk, m.sk, m.d}, stride{m.sk * row, m.d, row, 1};
    return first_order({&grads[0], &q, &k, &v},
                       {dq, dkv.as_strided(size, stride), dkv.as_strided(size, stride, m.hk * m.d), Tensor(),
                        Tensor(), Tensor()});
  }
};

// --- Python ---------------------------------------------------------------------------------------

Tensor tensor_of(PyObject* o, const char* who, const char* name) {
  REQUIRE(THPVariable_Check(o), who, ": ", name, " must be a tensor");
  return THPVariable_Unpack(o);
}
Tensor optional_of(PyObject* o, const char* who, const char* name) {
  return o == Py_None ? Tensor() : tensor_of(o, who, name);
}
double double_of(PyObject* o) {
  const double x = PyFloat_AsDouble(o);
  if (x == -1.0 && PyErr_Occurred()) throw_python();
  return x;
}
int64_t int_of(PyObject* o) {
  const int64_t x = PyLong_AsLongLong(o);
  if (x == -1 && PyErr_Occurred()) throw_python();
  return x;
}
bool bool_of(PyObject* o) {
  const int x = PyObject_IsTrue(o);
  if (x < 0) throw_python();
  return x != 0;
}
void count(Py_ssize_t got, Py_ssize_t want) { REQUIRE(got == want, "_ops: ", want, " arguments expected"); }

// x, positions, freqs, amplitude, interleaved as a Turn of x's [b, s] tokens.
Turn turn_of(const char* who, const Tensor& x, PyObject* const* a, int64_t b, int64_t s, int64_t d,
             int64_t heads) {
  REQUIRE(dtype_of(x) >= 0, who, ": f32, f16 or bf16 expected, got ", type_name(x));
  no_tangent(who, "", {&x});
  Turn t{who, Tensor(), 0, tensor_of(a[1], who, "freqs"), double_of(a[2]), bool_of(a[3]), heads};
  check_freqs(who, t.freqs, d);
  if (!THPVariable_Check(a[0])) {
    t.first = int_of(a[0]);
    one_device(who, {&x, &t.freqs});
    return t;
  }
  Tensor p = THPVariable_Unpack(a[0]);
  REQUIRE(p.scalar_type() == at::kInt || p.scalar_type() == at::kLong, who,
          ": int32 or int64 positions expected");
  const int64_t n = p.dim();
  REQUIRE((n == 1 && p.size(0) == s) ||
              (n == 2 && (p.size(0) == b || p.size(0) == 1) && (p.size(1) == s || (p.size(1) == 1 && p.size(0) == b))),
          who, ": positions [", s, "], [", b, ", ", s, "] or [", b, ", 1] expected, got ", p.sizes());
  one_device(who, {&x, &t.freqs, &p});
  t.positions = n == 2 && p.size(0) == b && p.size(1) == s ? p : p.expand({b, s});
  return t;
}

PyObject* rotary(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 5);
  const Tensor x = tensor_of(a[0], "rotary", "x");
  REQUIRE(x.dim() == 4, "rotary: [b, h, s, d] expected, shape ", x.sizes());
  return THPVariable_Wrap(rotate(x, turn_of("rotary", x, a + 1, x.size(0), x.size(2), x.size(3), 0)));
  END_HANDLE_TH_ERRORS
}

PyObject* rotary_qkv(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 6);
  const Tensor x = tensor_of(a[0], "rotary_qkv", "qkv");
  const int64_t heads = int_of(a[1]);
  REQUIRE(x.dim() == 3, "fused_attention_qkv: rank-3 qkv expected, shape ", x.sizes());
  REQUIRE(heads > 0 && x.size(2) % (3 * heads) == 0, "fused_attention_qkv: last dimension ", x.size(2),
          " is not 3 x ", heads, " heads x head_dim");
  const Turn t = turn_of("rotary_qkv", x, a + 2, x.size(0), x.size(1), x.size(2) / (3 * heads), heads);
  return THPVariable_Wrap(rotate(x, t));
  END_HANDLE_TH_ERRORS
}

PyObject* cross_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const char* who = "cross_attention";
  count(n, 5);
  Tensor q = tensor_of(a[0], who, "q"), k = tensor_of(a[1], who, "k"), v = tensor_of(a[2], who, "v");
  const double scale = double_of(a[3]);
  const Tensor lengths = optional_of(a[4], who, "key_lengths");
  for (const Tensor* t : {&q, &k, &v}) REQUIRE(t->scalar_type() == at::kFloat, who, ": f32 only");
  REQUIRE(q.dim() == 4 && k.dim() == 4 && v.sizes() == k.sizes() && k.size(0) == q.size(0) &&
              k.size(3) == q.size(3),
          who, ": q [b, h, sq, d], k and v [b, hk, sk, d] expected, got ", q.sizes(), " ", k.sizes(), " ",
          v.sizes());
  const Dims m{q.size(0), q.size(1), k.size(1), q.size(2), k.size(2), q.size(3)};
  REQUIRE((m.hk ? m.h % m.hk : m.h) == 0, who, ": ", m.h, " query heads are no multiple of ", m.hk,
          " key heads");
  check_head_dim(m.d);
  no_tangent(who, "", {&q, &k, &v});
  one_device(who, {&q, &k, &v, &lengths});
  int32_vector(who, "key_lengths", lengths, m.b);
  q = aligned_rows(q), k = aligned_rows(k), v = aligned_rows(v);
  if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad()))
    return THPVariable_Wrap(Cross::apply(q, k, v, Keys{lengths}, scale, m));
  Tensor lse;
  return THPVariable_Wrap(cross_forward(q, k, v, lengths, static_cast<float>(scale), m, false, lse));
  END_HANDLE_TH_ERRORS
}

void check_cache(const char* who, const Tensor& x, const Tensor& kc, const Tensor& vc, const Tensor& table,
                 const Tensor& lengths, const Tensor& new_lengths, int64_t b, int64_t hk, int64_t d) {
  REQUIRE(kc.dim() == 4 && vc.sizes() == kc.sizes() && kc.size(2) == hk && kc.size(3) == d, who,
          ": caches [pages, page_size, ", hk, ", ", d, "] expected, got ", kc.sizes(), " ", vc.sizes());
  REQUIRE(kc.size(1) >= 1, who, ": a page needs at least one row");
  const int type = dtype_of(x), cache = dtype_of(kc);
  REQUIRE(type >= 0 && cache >= 0 && dtype_of(vc) == cache && (type == cache || type == CFA_F32), who,
          ": f32, f16 or bf16 inputs over a cache of their type, or f32 over any, expected; got ",
          type_name(x), " over ", type_name(kc), " ", type_name(vc));
  REQUIRE(kc.stride(3) == 1 && vc.stride(3) == 1, who, ": the caches' last dimension must be contiguous");
  REQUIRE(table.scalar_type() == at::kInt && table.dim() == 2 && table.size(0) == b &&
              (table.size(1) <= 1 || table.stride(1) == 1),
          who, ": page_table int32 [", b, ", width] with dense rows expected, got ", type_name(table), " ",
          table.sizes());
  int32_vector(who, "lengths", lengths, b);
  int32_vector(who, "new_lengths", new_lengths, b);
}

PyObject* paged_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const char* who = "paged_append";
  count(n, 11);
  Tensor k = tensor_of(a[0], who, "k"), v = tensor_of(a[1], who, "v");
  const Tensor kc = tensor_of(a[2], who, "k_cache"), vc = tensor_of(a[3], who, "v_cache");
  const Tensor table = tensor_of(a[4], who, "page_table"), lengths = tensor_of(a[5], who, "lengths");
  Tensor q = optional_of(a[6], who, "q");
  const Tensor freqs = optional_of(a[7], who, "freqs");
  const double amplitude = double_of(a[8]);
  const bool interleaved = bool_of(a[9]);
  const Tensor fresh = optional_of(a[10], who, "new_lengths");
  REQUIRE(k.dim() == 4 && v.sizes() == k.sizes(), who, ": k and v [b, hk, s, d] expected, got ", k.sizes(),
          " ", v.sizes());
  const int64_t b = k.size(0), hk = k.size(1), s = k.size(2), d = k.size(3);
  REQUIRE(v.scalar_type() == k.scalar_type(), who, ": k and v must have one type");
  REQUIRE(!q.defined() || (q.dim() == 4 && q.size(0) == b && q.size(2) == s && q.size(3) == d &&
                           q.scalar_type() == k.scalar_type()),
          who, ": q [", b, ", h, ", s, ", ", d, "] of k's type expected, got ", type_name(q), " ", q.sizes());
  check_cache(who, k, kc, vc, table, lengths, fresh, b, hk, d);
  no_gradient(who, "", {&q, &k, &v, &kc, &vc});
  if (freqs.defined()) check_freqs(who, freqs, d);
  one_device(who, {&k, &v, &kc, &vc, &table, &lengths, &fresh, &q, &freqs});
  const Launch on(k);
  k = dense_rows(k), v = dense_rows(v);
  Tensor out;
  int64_t h = 0;
  if (q.defined()) {
    q = dense_rows(q);
    h = q.size(1);
    out = merged_heads(b, h, s, d, q);
  }
  const Strides3 none(0, 0, 0);
  check_status(abi.paged_append(ptr<void>(q), q.defined() ? Strides3(q) : none,
                                q.defined() ? out.mutable_data_ptr() : nullptr,
                                Strides3(s * h * d, d, h * d), ptr<void>(k), Strides3(k), ptr<void>(v),
                                Strides3(v), dtype_of(k), kc.mutable_data_ptr(), Strides3(kc),
                                vc.mutable_data_ptr(), Strides3(vc), dtype_of(kc), kc.size(0), kc.size(1),
                                ptr<int32_t>(table), table.stride(0), table.size(1), ptr<int32_t>(lengths),
                                ptr<int32_t>(fresh), ptr<double>(freqs), static_cast<float>(amplitude), b, h,
                                hk, s, d, freqs.defined() ? 2 * freqs.numel() : 0, interleaved, on.stream),
               who);
  // As every in-place operation: a backward that saved the cache before is told.
  for (const Tensor* t : {&kc, &vc})
    if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
  if (!q.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

PyObject* paged_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const char* who = "paged_attention";
  count(n, 7);
  Tensor q = tensor_of(a[0], who, "q");
  const Tensor kc = tensor_of(a[1], who, "k_cache"), vc = tensor_of(a[2], who, "v_cache");
  const Tensor table = tensor_of(a[3], who, "page_table"), lengths = tensor_of(a[4], who, "lengths");
  const double scale = double_of(a[5]);
  const Tensor fresh = optional_of(a[6], who, "new_lengths");
  REQUIRE(q.dim() == 4, who, ": [b, h, s, d] expected, shape ", q.sizes());
  const int64_t b = q.size(0), h = q.size(1), s = q.size(2), d = q.size(3);
  check_head_dim(d);
  const int64_t hk = kc.dim() == 4 ? kc.size(2) : 0;
  check_cache(who, q, kc, vc, table, lengths, fresh, b, hk, d);
  REQUIRE((hk ? h % hk : h) == 0, who, ": ", h, " query heads are no multiple of ", hk, " key heads");
  no_gradient(who, "", {&q, &kc, &vc});
  one_device(who, {&q, &kc, &vc, &table, &lengths, &fresh});
  REQUIRE(kc.numel() == 0 || aligned(kc), who, ": k_cache: rows must be 16-byte aligned");
  REQUIRE(vc.numel() == 0 || aligned(vc), who, ": v_cache: rows must be 16-byte aligned");
  const Launch on(q);
  q = aligned_rows(q);
  const Tensor o = merged_heads(b, h, s, d, q);
  const int64_t width = table.size(1), page = kc.size(1);
  const size_t bytes = abi.paged_attention_workspace(b, h, s, width * page, d, dtype_of(kc));
  const Tensor ws = workspace(bytes, q);
  check_status(abi.paged_attention(ptr<void>(q), Strides3(q), dtype_of(q), ptr<void>(kc), Strides3(kc),
                                   ptr<void>(vc), Strides3(vc), dtype_of(kc), kc.size(0), page,
                                   ptr<int32_t>(table), table.stride(0), width, ptr<int32_t>(lengths),
                                   ptr<int32_t>(fresh), o.mutable_data_ptr(),
                                   bytes ? ws.mutable_data_ptr() : nullptr, bytes, b, h, hk, s, d,
                                   static_cast<float>(scale), on.stream),
               who);
  return THPVariable_Wrap(o);
  END_HANDLE_TH_ERRORS
}

// bind(addresses, error_class, flag_address, raise_flag): the ABI's functions in Abi's order.
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  constexpr Py_ssize_t entries = sizeof(Abi) / sizeof(void*);
  if (n != 4 || !PyTuple_Check(a[0]) || PyTuple_GET_SIZE(a[0]) != entries) {
    PyErr_SetString(PyExc_TypeError, "bind: eleven addresses, a class and two functions expected");
    return nullptr;
  }
  void* at[entries];
  for (Py_ssize_t i = 0; i < entries; ++i)
    if (!(at[i] = PyLong_AsVoidPtr(PyTuple_GET_ITEM(a[0], i)))) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "bind: a null address");
      return nullptr;
    }
  std::memcpy(&abi, at, sizeof abi);
  error_class = Py_NewRef(a[1]);
  flag_address = Py_NewRef(a[2]);
  raise_flag = Py_NewRef(a[3]);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyMethodDef method(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F)), METH_FASTCALL, nullptr};
}
PyMethodDef methods[] = {method<bind>("bind"),
                         method<rotary>("rotary"),
                         method<rotary_qkv>("rotary_qkv"),
                         method<cross_attention>("cross_attention"),
                         method<paged_append>("paged_append"),
                         method<paged_attention>("paged_attention"),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_ops", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__ops() { return PyModule_Create(&module); }
