// fa4d_torch.cpp — host binding of the operators around the attention (_fa4d_host.so): argument
// checks, output and workspace allocation, the current stream, and the calls into libfa4d.so.
// A decode step's kernels take a few microseconds each, so the path from Python to the launch
// is native: bound through ctypes the same checks took 25 to 35 us a call.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/python_headers.h>
#include <ATen/ATen.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <string>

#include "fa4d.h"

namespace {

using at::Tensor;

// An argument the operators refuse: ValueError, or RuntimeError where the device is wrong.
struct Refused {
  PyObject* type;
  std::string text;
};
[[noreturn]] void refuse(std::string text) { throw Refused{PyExc_ValueError, std::move(text)}; }

template <typename... Args>
std::string cat(const Args&... args) {
  return c10::str(args...);
}

std::string name_of(at::ScalarType t) {
  return cat("torch.", t == at::kBFloat16 ? "bfloat16" : t == at::kHalf ? "float16" : t == at::kFloat ? "float32"
             : t == at::kDouble ? "float64" : t == at::kInt ? "int32" : t == at::kLong ? "int64" : at::toString(t));
}

void check(int rc, const char* what) {
  if (rc == FA4D_OK) return;
  const std::string text = cat(what, ": ", fa4d_last_error(), " (code ", rc, ")");
  const bool value = rc == FA4D_ERR_INVALID || rc == FA4D_ERR_UNSUPPORTED || rc == FA4D_ERR_WORKSPACE || rc == FA4D_ERR_LAYOUT;
  throw Refused{value ? PyExc_ValueError : PyExc_RuntimeError, text};
}

bool half_type(const Tensor& x) { return x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf; }
int dtype_code(const Tensor& x) { return x.scalar_type() == at::kBFloat16 ? FA4D_BF16 : FA4D_F16; }

// Dimension of the sequence (or slots) in a rank-4 tensor; heads are the other of 1 and 2.
struct Layout {
  bool bhsd;
  int seq() const { return bhsd ? 2 : 1; }
  int head() const { return bhsd ? 1 : 2; }
};

// Whether two elements share memory through a stride of 0, which a tensor that is written may not.
bool repeats(const Tensor& x) {
  for (int i = 0; i < x.dim(); ++i)
    if (x.size(i) > 1 && x.stride(i) == 0) return true;
  return false;
}

void set3(int64_t (&out)[3], const Tensor& x, Layout l) {
  out[0] = x.stride(0);
  out[1] = x.stride(l.seq());
  out[2] = x.stride(l.head());
}

// A tangent (torch.autograd.forward_ad) is not carried through, so a tensor with one is refused, as
// the attention's autograd function does.  Such a tensor need not require a gradient.
void no_tangent(const char* name, std::initializer_list<const Tensor*> tensors) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const Tensor* x : tensors)
    if (x->defined() && x->_fw_grad(0).defined())
      throw Refused{PyExc_NotImplementedError, cat(name, " has no forward-mode derivative")};
}

void no_gradient(const char* name, std::initializer_list<const Tensor*> tensors) {
  no_tangent(name, tensors);
  if (!at::GradMode::is_enabled()) return;
  for (const Tensor* x : tensors)
    if (x->defined() && x->requires_grad()) refuse(cat(name, " has no gradient: call it under torch.no_grad()"));
}

// Tells autograd that tensors have been written (an inference tensor has no version to tell).
void written(std::initializer_list<const Tensor*> tensors) {
  for (const Tensor* x : tensors)
    if (x->defined() && !x->is_inference()) x->unsafeGetTensorImpl()->bump_version();
}

void need_cuda(const char* name, const Tensor& x) {
  if (!x.is_cuda()) throw Refused{PyExc_RuntimeError, cat(name, " runs on CUDA (sm_100a) tensors only")};
}

Tensor unit_rows(const Tensor& x) { return x.stride(3) == 1 ? x : x.contiguous(); }

// A new tensor in x's order of strides, with whole rows: where the rows of x overlap (windows of
// one another, which have no order), a contiguous one.
Tensor new_rows(const Tensor& x) {
  Tensor out = at::empty_like(x);
  return out.stride(3) == 1 ? out : at::empty_like(x, at::MemoryFormat::Contiguous);
}

// x with rows that 16-byte accesses can reach: itself, or a copy.  `walked`: no dimension may
// have stride 0 either.
Tensor rows16(const Tensor& x, bool walked = false) {
  const int n = static_cast<int>(x.dim());
  bool ok = x.stride(n - 1) == 1 && reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0;
  for (int i = 0; i + 1 < n; ++i) ok = ok && x.stride(i) % 8 == 0 && (!walked || x.stride(i) > 0 || x.size(i) == 1);
  return ok ? x : x.clone(at::MemoryFormat::Contiguous);
}

void* stream_of(const Tensor& x) { return c10::cuda::getCurrentCUDAStream(x.get_device()).stream(); }

// ------------------------------------------------------------------ arguments

Tensor tensor_arg(PyObject* o, const char* name, int dim) {
  if (!THPVariable_Check(o)) refuse(cat(name, " must be a rank-", dim, " tensor"));
  const Tensor& x = THPVariable_Unpack(o);
  if (x.dim() != dim) refuse(cat(name, " must be a rank-", dim, " tensor"));
  return x;
}
Tensor any_tensor(PyObject* o, const char* otherwise) {
  if (!THPVariable_Check(o)) refuse(otherwise);
  return THPVariable_Unpack(o);
}
Tensor optional_arg(PyObject* o, const char* otherwise) { return o == Py_None ? Tensor() : any_tensor(o, otherwise); }

Layout layout_arg(PyObject* o) {
  const char* s = PyUnicode_Check(o) ? PyUnicode_AsUTF8(o) : "";
  if (s && !strcmp(s, "bhsd")) return {true};
  if (s && !strcmp(s, "bshd")) return {false};
  refuse(cat("unsupported layout: ", s ? s : ""));
}
int64_t int_arg(PyObject* o, const char* name) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    refuse(cat(name, " must be an integer"));
  }
  return v;
}
int small(int64_t v, const char* name) {
  if (v < INT32_MIN || v > INT32_MAX) refuse(cat(name, " is too large"));
  return static_cast<int>(v);
}

// ------------------------------------------------------------------ rotary

struct Table : torch::CustomClassHolder {
  fa4d_rotary_table t;
};
constexpr const char* kTableName = "fa4d_rotary_table";

Table* table_arg(PyObject* o) {
  auto* p = static_cast<Table*>(PyCapsule_GetPointer(o, kTableName));
  if (!p) {
    PyErr_Clear();
    refuse("not a rotary table");
  }
  return p;
}

// New tokens: query and key (and value, with the key's heads).
void check_tokens(const Tensor& q, const Tensor& k, const Tensor& v, Layout l, int head_dim) {
  const std::pair<const char*, const Tensor*> all[] = {{"query", &q}, {"key", &k}, {"value", &v}};
  for (const auto& [name, x] : all) {
    if (!x->defined()) continue;
    if (!half_type(*x)) refuse(cat(name, " must be fp16 or bf16, got ", name_of(x->scalar_type())));
    if (x->scalar_type() != q.scalar_type() || x->device() != q.device())
      refuse(cat(name, " must have the dtype and device of query"));
    if (x->size(0) != q.size(0) || x->size(l.seq()) != q.size(l.seq()))
      refuse(cat(name, " must have the batch size and sequence length of query"));
    if (x->size(3) != head_dim) refuse(cat(name, " has head dimension ", x->size(3), ", expected ", head_dim));
  }
  if (v.defined() && v.size(l.head()) != k.size(l.head())) refuse("value must have the heads of key");
}

// Integer positions [axes, B or 1, T], as int32 or int64.
Tensor check_positions(PyObject* o, const Table& table, int64_t B, int64_t T, const Tensor& like) {
  Tensor p = any_tensor(o, "positions must be an integer tensor");
  if (p.dim() != 3 || p.size(0) != table.t.axes || (p.size(1) != 1 && p.size(1) != B) || p.size(2) != T)
    refuse(cat("positions must be an integer tensor of shape [", table.t.axes, ", ", B, " or 1, ", T, "]"));
  if (!at::isIntegralType(p.scalar_type(), false)) refuse("positions must be an integer tensor");
  if (p.device() != like.device()) refuse(cat("positions must be on ", like.device(), ", got ", p.device()));
  return p.scalar_type() == at::kInt || p.scalar_type() == at::kLong ? p : p.to(at::kLong);
}
template <typename Args>
void set_positions(Args& a, const Tensor& p) {
  a.positions = p.data_ptr();
  a.positions_stride[0] = p.stride(0);
  a.positions_stride[1] = p.size(1) == 1 ? 0 : p.stride(1);
  a.positions_stride[2] = p.stride(2);
  a.positions_bits = p.scalar_type() == at::kLong ? 64 : 32;
}

std::pair<Tensor, Tensor> rotate(Tensor q, Tensor k, const Tensor& positions, const Table& table, Layout l, bool inverse) {
  q = unit_rows(q);
  k = unit_rows(k);
  Tensor qo = new_rows(q), ko = new_rows(k);
  if (q.numel() == 0 || k.numel() == 0) {
    if (q.numel() || k.numel()) refuse("query and key need at least one head");
    return {qo, ko};
  }
  const c10::cuda::OptionalCUDAGuard guard(q.device());
  fa4d_rotary_args a;
  a.table = table.t;
  a.q = q.data_ptr();
  a.k = k.data_ptr();
  a.q_out = qo.data_ptr();
  a.k_out = ko.data_ptr();
  set3(a.q_stride, q, l);
  set3(a.k_stride, k, l);
  set3(a.q_out_stride, qo, l);
  set3(a.k_out_stride, ko, l);
  set_positions(a, positions);
  a.B = small(q.size(0), "batch");
  a.T = small(q.size(l.seq()), "sequence");
  a.Hq = small(q.size(l.head()), "heads");
  a.Hk = small(k.size(l.head()), "heads");
  a.dtype = dtype_code(q);
  a.inverse = inverse;
  check(fa4d_rotary(&a, stream_of(q)), "fa4d_rotary");
  return {qo, ko};
}

// A turn by phi; its gradient is the turn by -phi, itself differentiable.
struct Rotate : torch::autograd::Function<Rotate> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& q, const Tensor& k,
                                                const Tensor& positions, c10::intrusive_ptr<torch::CustomClassHolder> table,
                                                bool bhsd, bool inverse) {
    ctx->save_for_backward({positions});
    ctx->saved_data["table"] = c10::IValue::make_capsule(table);
    ctx->saved_data["bhsd"] = bhsd;
    ctx->saved_data["inverse"] = inverse;
    auto out = rotate(q, k, positions, static_cast<const Table&>(*table), Layout{bhsd}, inverse);
    return {out.first, out.second};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list g) {
    const Tensor positions = ctx->get_saved_variables()[0];
    auto table = ctx->saved_data["table"].toCapsule();
    try {
      auto out = apply(g[0], g[1], positions, table, ctx->saved_data["bhsd"].toBool(), !ctx->saved_data["inverse"].toBool());
      return {out[0], out[1], Tensor(), Tensor(), Tensor(), Tensor()};
    } catch (const Refused& e) {  // the engine's thread only knows torch's errors
      TORCH_CHECK(false, e.text);
    }
  }
};

PyObject* pair_of(const Tensor& a, const Tensor& b) {
  PyObject* out = PyTuple_New(2);
  if (!out) return nullptr;
  PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(a));
  PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(b));
  return out;
}

// ------------------------------------------------------------------ caches

// A batch's cache; returns its slots.
int64_t check_cache(const Tensor& k, const Tensor& v, const Tensor& lengths, const Tensor& weights, Layout l, int64_t B,
                    int64_t Hk, int64_t D, const Tensor& like) {
  const std::pair<const char*, const Tensor*> all[] = {{"key cache", &k}, {"value cache", &v}};
  for (const auto& [name, x] : all) {
    if (x->scalar_type() != like.scalar_type() || x->device() != like.device())
      refuse(cat(name, " must be ", name_of(like.scalar_type()), " on ", like.device()));
    if (x->size(0) != B || x->size(l.head()) != Hk || x->size(3) != D || x->size(l.seq()) != k.size(l.seq()))
      refuse(cat(name, " has shape ", x->sizes(), ", expected batch ", B, ", ", Hk, " heads of ", D,
                 " and the same slots for keys and values"));
  }
  const int64_t C = k.size(l.seq());
  if (C < 1) refuse("the cache has no slots");
  if (lengths.scalar_type() != at::kInt || lengths.dim() != 1 || lengths.size(0) != B || lengths.device() != like.device() ||
      !lengths.is_contiguous())
    refuse(cat("lengths must be a contiguous int32 tensor of shape [", B, "] on ", like.device()));
  if (weights.defined() &&
      (weights.scalar_type() != at::kFloat || weights.dim() != 3 || weights.size(0) != B || weights.size(1) != Hk ||
       weights.size(2) != C || weights.device() != like.device() || weights.stride(2) != 1))
    refuse(cat("weights must be an fp32 tensor of shape [", B, ", ", Hk, ", ", C, "] with unit slot stride on ", like.device()));
  return C;
}

void set_weights(int64_t (&out)[2], const Tensor& w) {
  out[0] = w.defined() ? w.stride(0) : 0;
  out[1] = w.defined() ? w.stride(1) : 0;
}

const char* kWeights = "weights must be an fp32 tensor";
const char* kLengths = "lengths must be a contiguous int32 tensor";

// ------------------------------------------------------------------ entry points

// make_table(base, sections, head_dim, rotary_dim, pairing) -> capsule.  Pair i turns by
// base^(-2 i / rotary_dim) radians a position: as turns, modulo one, to the nearest 2^-64 (at
// most 1.12 of these off, for a base of 1 or more).
PyObject* make_table(PyObject* const* args) {
  auto table = c10::make_intrusive<Table>();
  fa4d_rotary_table& t = table->t;
  memset(&t, 0, sizeof(t));
  const double base = PyFloat_AsDouble(args[0]);
  t.D = small(int_arg(args[2], "head_dim"), "head_dim");
  t.rotary_dim = small(int_arg(args[3], "rotary_dim"), "rotary_dim");
  t.pairing = small(int_arg(args[4], "pairing"), "pairing");
  t.axes = small(PyTuple_Size(args[1]), "sections");
  int i = 0;
  for (int a = 0; a < t.axes; ++a) {
    const int64_t n = int_arg(PyTuple_GET_ITEM(args[1], a), "sections");
    for (int64_t j = 0; j < n && i < FA4D_ROTARY_MAX_PAIRS; ++j, ++i) {
      const long double turns = std::pow(static_cast<long double>(base), -2.0L * i / t.rotary_dim) / 6.283185307179586476925287L;
      const long double units = std::rint(std::ldexp(turns - std::floor(turns), 64));
      t.turn[i] = units < 18446744073709551616.0L ? static_cast<uint64_t>(units) : 0;  // a whole turn
      t.axis[i] = static_cast<uint8_t>(a);
    }
  }
  return PyCapsule_New(table.release(), kTableName, [](PyObject* o) {
    c10::intrusive_ptr<Table>::reclaim(static_cast<Table*>(PyCapsule_GetPointer(o, kTableName)));
  });
}

// table_turns(table) -> (turns per position of each pair in 2^-64 turns, axis of each pair)
PyObject* table_turns(PyObject* const* args) {
  const fa4d_rotary_table& t = table_arg(args[0])->t;
  const int n = t.rotary_dim / 2;
  PyObject* turns = PyTuple_New(n);
  PyObject* axes = PyTuple_New(n);
  for (int i = 0; i < n; ++i) {
    PyTuple_SET_ITEM(turns, i, PyLong_FromUnsignedLongLong(t.turn[i]));
    PyTuple_SET_ITEM(axes, i, PyLong_FromLong(t.axis[i]));
  }
  PyObject* out = PyTuple_Pack(2, turns, axes);
  Py_DECREF(turns);
  Py_DECREF(axes);
  return out;
}

// rotary(table, query, key, positions, layout) -> (query, key)
PyObject* rotary(PyObject* const* args) {
  Table* table = table_arg(args[0]);
  const Layout l = layout_arg(args[4]);
  const Tensor q = tensor_arg(args[1], "query", 4), k = tensor_arg(args[2], "key", 4);
  check_tokens(q, k, Tensor(), l, table->t.D);
  const Tensor positions = check_positions(args[3], *table, q.size(0), q.size(l.seq()), q);
  no_tangent("MultiAxisRotary", {&q, &k});
  need_cuda("MultiAxisRotary", q);
  if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad())) {
    auto holder = c10::intrusive_ptr<torch::CustomClassHolder>(c10::intrusive_ptr<Table>::unsafe_reclaim_from_nonowning(table));
    auto out = Rotate::apply(q, k, positions, holder, l.bhsd, false);
    return pair_of(out[0], out[1]);
  }
  auto out = rotate(q, k, positions, *table, l, false);
  return pair_of(out.first, out.second);
}

// rotary_append(table, query, key, value, positions, key_cache, value_cache, lengths, weights,
// layout) -> (query, lengths)
PyObject* rotary_append(PyObject* const* args) {
  Table* table = table_arg(args[0]);
  const Layout l = layout_arg(args[9]);
  Tensor q = tensor_arg(args[1], "query", 4), k = tensor_arg(args[2], "key", 4), v = tensor_arg(args[3], "value", 4);
  check_tokens(q, k, v, l, table->t.D);
  const int64_t B = q.size(0), T = q.size(l.seq()), Hq = q.size(l.head()), Hk = k.size(l.head());
  const Tensor positions = check_positions(args[4], *table, B, T, q);
  const Tensor kc = tensor_arg(args[5], "key cache", 4), vc = tensor_arg(args[6], "value cache", 4);
  const Tensor lengths = any_tensor(args[7], kLengths), weights = optional_arg(args[8], kWeights);
  const int64_t C = check_cache(kc, vc, lengths, weights, l, B, Hk, table->t.D, q);
  no_gradient("append", {&q, &k, &v, &kc, &vc, &weights});
  if (kc.stride(3) != 1 || vc.stride(3) != 1) refuse("the caches are written in place and need unit head-dim stride");
  if (repeats(kc) || repeats(vc) || (weights.defined() && repeats(weights)))
    refuse("the caches and weights are written in place and may not repeat memory");
  need_cuda("MultiAxisRotary", q);
  q = unit_rows(q);
  k = unit_rows(k);
  v = unit_rows(v);
  Tensor qo = new_rows(q);
  if (B == 0 || T == 0) return pair_of(qo, lengths.clone());
  Tensor lengths_out = at::empty_like(lengths);
  const c10::cuda::OptionalCUDAGuard guard(q.device());
  fa4d_rotary_append_args a;
  a.table = table->t;
  a.q = q.data_ptr();
  a.k = k.data_ptr();
  a.v = v.data_ptr();
  a.q_out = qo.data_ptr();
  a.k_cache = kc.data_ptr();
  a.v_cache = vc.data_ptr();
  a.weights = weights.defined() ? weights.data_ptr<float>() : nullptr;
  a.lengths = lengths.data_ptr<int32_t>();
  a.lengths_out = lengths_out.data_ptr<int32_t>();
  set3(a.q_stride, q, l);
  set3(a.k_stride, k, l);
  set3(a.v_stride, v, l);
  set3(a.q_out_stride, qo, l);
  set3(a.k_cache_stride, kc, l);
  set3(a.v_cache_stride, vc, l);
  set_weights(a.weights_stride, weights);
  set_positions(a, positions);
  a.B = small(B, "batch");
  a.T = small(T, "sequence");
  a.Hq = small(Hq, "heads");
  a.Hk = small(Hk, "heads");
  a.C = small(C, "cache");
  a.dtype = dtype_code(q);
  check(fa4d_rotary_append(&a, stream_of(q)), "fa4d_rotary_append");
  written({&kc, &vc, &weights});
  return pair_of(qo, lengths_out);
}

// shared_prefix_attention(query, prefix_key, prefix_value, key, value, lengths, mask, weights,
// scale, is_causal, layout) -> out
PyObject* shared_prefix_attention(PyObject* const* args) {
  const Layout l = layout_arg(args[10]);
  Tensor q = tensor_arg(args[0], "query", 4);
  if (!half_type(q)) refuse(cat("query must be fp16 or bf16, got ", name_of(q.scalar_type())));
  Tensor k = tensor_arg(args[3], "key cache", 4), v = tensor_arg(args[4], "value cache", 4);
  const int64_t B = q.size(0), T = q.size(l.seq()), Hq = q.size(l.head()), D = q.size(3), Hk = k.size(l.head());
  if (Hk == 0 || Hq % Hk != 0) refuse(cat("query heads (", Hq, ") must be divisible by key/value heads (", Hk, ")"));
  if (D != 64 && D != 96 && D != 128 && D != 256) refuse(cat("head dim ", D, " is not built (64, 96, 128, 256)"));
  const Tensor lengths = any_tensor(args[5], kLengths), weights = optional_arg(args[7], kWeights);
  const int64_t C = check_cache(k, v, lengths, weights, l, B, Hk, D, q);
  if (weights.defined() && repeats(weights)) refuse("weights are written in place and may not repeat memory");
  if ((args[1] == Py_None) != (args[2] == Py_None)) refuse("prefix_key and prefix_value go together");
  Tensor pk, pv;
  int64_t P = 0;
  const int seq = l.bhsd ? 1 : 0;
  if (args[1] != Py_None) {
    auto one = [&](PyObject* o, const char* name) {
      const Tensor x = tensor_arg(o, name, 3);
      if (x.size(1 - seq) != Hk || x.size(2) != D || (pk.defined() && x.size(seq) != pk.size(seq)))
        refuse(cat(name, " must have shape ", l.bhsd ? cat("[", Hk, ", P, ", D, "]") : cat("[P, ", Hk, ", ", D, "]")));
      if (x.scalar_type() != q.scalar_type() || x.device() != q.device())
        refuse(cat(name, " must be ", name_of(q.scalar_type()), " on ", q.device()));
      return x;
    };
    pk = one(args[1], "prefix_key");
    pv = one(args[2], "prefix_value");
    P = pk.size(seq);
  }
  Tensor mask;
  if (args[6] != Py_None) {
    mask = any_tensor(args[6], "mask must be a bool tensor");
    if (mask.dim() != 4 || mask.scalar_type() != at::kBool || (mask.size(0) != 1 && mask.size(0) != B) ||
        (mask.size(1) != 1 && mask.size(1) != Hq) || mask.size(2) != T || mask.size(3) != C)
      refuse(cat("mask must be a bool tensor of shape [", B, " or 1, ", Hq, " or 1, ", T, ", ", C, "]"));
    if (mask.device() != q.device()) refuse(cat("mask must be on ", q.device(), ", got ", mask.device()));
  }
  double scale = 1.0 / std::sqrt(static_cast<double>(D));
  if (args[8] != Py_None) {
    scale = PyFloat_AsDouble(args[8]);
    if (PyErr_Occurred()) {
      PyErr_Clear();
      refuse("scale must be a number");
    }
  }
  if (!std::isfinite(scale)) refuse("scale must be finite");
  const int causal = PyObject_IsTrue(args[9]);
  no_gradient("shared_prefix_attention", {&q, &pk, &pv, &k, &v, &weights});
  need_cuda("shared_prefix_attention", q);

  const c10::cuda::OptionalCUDAGuard guard(q.device());
  q = rows16(q);
  Tensor out = new_rows(q);
  if (out.numel() == 0) return THPVariable_Wrap(out);
  k = rows16(k, true);  // keys and values go through tensor maps
  v = rows16(v, true);
  fa4d_prefix_attention_args a;
  memset(&a, 0, sizeof(a));
  if (P) {
    pk = rows16(pk, true);
    pv = rows16(pv, true);
    a.prefix_k = pk.data_ptr();
    a.prefix_v = pv.data_ptr();
    a.prefix_k_stride[0] = pk.stride(seq);
    a.prefix_k_stride[1] = pk.stride(1 - seq);
    a.prefix_v_stride[0] = pv.stride(seq);
    a.prefix_v_stride[1] = pv.stride(1 - seq);
  }
  if (mask.defined()) {
    if (mask.stride(3) != 1) mask = mask.contiguous();
    a.mask = static_cast<const uint8_t*>(mask.data_ptr());
    a.mask_stride[0] = mask.size(0) == 1 ? 0 : mask.stride(0);
    a.mask_stride[1] = mask.size(1) == 1 ? 0 : mask.stride(1);
    a.mask_stride[2] = mask.stride(2);
  }
  a.q = q.data_ptr();
  a.k = k.data_ptr();
  a.v = v.data_ptr();
  a.o = out.data_ptr();
  a.lengths = lengths.data_ptr<int32_t>();
  a.weights = weights.defined() ? weights.data_ptr<float>() : nullptr;
  set3(a.q_stride, q, l);
  set3(a.k_stride, k, l);
  set3(a.v_stride, v, l);
  set3(a.o_stride, out, l);
  set_weights(a.weights_stride, weights);
  a.B = small(B, "batch");
  a.T = small(T, "sequence");
  a.Hq = small(Hq, "heads");
  a.Hk = small(Hk, "heads");
  a.D = small(D, "head dim");
  a.P = small(P, "prefix");
  a.C = small(C, "cache");
  a.dtype = dtype_code(q);
  a.causal = causal;
  a.scale = static_cast<float>(scale);
  a.workspace_bytes = fa4d_prefix_attention_workspace(a.B, a.T, a.Hq, a.Hk, a.D, a.P, a.C, weights.defined());
  if (!a.workspace_bytes) check(FA4D_ERR_INVALID, "fa4d_prefix_attention");
  const Tensor workspace = at::empty({static_cast<int64_t>(a.workspace_bytes)}, q.options().dtype(at::kByte));
  a.workspace = workspace.data_ptr();
  check(fa4d_prefix_attention(&a, stream_of(q)), "fa4d_prefix_attention");
  written({&weights});
  return THPVariable_Wrap(out);
}

// Whether two tensors share a byte.  A byte of x lies at its base + the sum of index * stride +
// the byte within its element, so they do where whole numbers c, each within the range that the
// indices leave it, solve  sum c * stride = base of y - base of x  (c of x's dimensions from 0
// up, of y's from 0 down).
class Meeting {
 public:
  static bool of(const Tensor& x, const Tensor& y) {
    if (x.numel() == 0 || y.numel() == 0) return false;
    Meeting m;
    m.add(x, 1);
    m.add(y, -1);
    m.terms.push_back({1, 1 - static_cast<int64_t>(y.element_size()), static_cast<int64_t>(x.element_size()) - 1});
    return m.solve(static_cast<const char*>(y.data_ptr()) - static_cast<const char*>(x.data_ptr()));
  }

 private:
  struct Term {
    int64_t stride, lo, hi;  // of the number that multiplies the stride
    // Of the sums of this term and the shorter strides' behind it: the least and the largest, and
    // whether every number between them is one.
    int64_t least = 0, most = 0;
    bool dense = false;
  };
  c10::SmallVector<Term, 16> terms;
  int steps = 0;

  void add(const Tensor& x, int sign) {
    for (int i = 0; i < x.dim(); ++i) {
      if (x.size(i) == 1 || x.stride(i) == 0) continue;
      const int64_t stride = x.stride(i) * static_cast<int64_t>(x.element_size()), last = x.size(i) - 1;
      terms.push_back({stride, sign > 0 ? 0 : -last, sign > 0 ? last : 0});
    }
  }

  bool solve(int64_t sum) {
    std::sort(terms.begin(), terms.end(), [](const Term& a, const Term& b) { return a.stride > b.stride; });
    size_t n = 0;  // equal strides make one term
    for (size_t i = 1; i < terms.size(); ++i) {
      if (terms[i].stride == terms[n].stride) {
        terms[n].lo += terms[i].lo;
        terms[n].hi += terms[i].hi;
      } else {
        terms[++n] = terms[i];
      }
    }
    terms.resize(n + 1);
    int64_t least = 0, most = 0;
    bool dense = true;
    for (size_t i = terms.size(); i-- > 0;) {
      Term& t = terms[i];
      dense = dense && (t.lo == t.hi || t.stride <= most - least + 1);
      t.least = least += t.lo * t.stride;
      t.most = most += t.hi * t.stride;
      t.dense = dense;
    }
    return search(0, sum);
  }

  // From the longest stride down.  Where strides are nested few numbers fit at each; what is not
  // decided within the steps counts as shared.
  bool search(size_t i, int64_t sum) {
    if (i == terms.size()) return sum == 0;
    const Term& t = terms[i];
    if (sum < t.least || sum > t.most) return false;
    if (t.dense || ++steps > 10000) return true;
    const int64_t rest_least = t.least - t.lo * t.stride, rest_most = t.most - t.hi * t.stride;
    auto down = [&](int64_t v) { return v / t.stride - (v % t.stride < 0); };
    const int64_t from = std::max(t.lo, -down(rest_most - sum)), to = std::min(t.hi, down(sum - rest_least));
    for (int64_t c = from; c <= to; ++c)
      if (search(i + 1, sum - c * t.stride)) return true;
    return false;
  }
};
bool meet(const Tensor& x, const Tensor& y) { return Meeting::of(x, y); }

// evict_by_weight(key, value, weights, lengths, keep, sinks, recent, out, layout) -> (key,
// value, weights, lengths, index)
PyObject* evict_by_weight(PyObject* const* args) {
  const Layout l = layout_arg(args[8]);
  Tensor k = tensor_arg(args[0], "key cache", 4), v = tensor_arg(args[1], "value cache", 4);
  if (!half_type(k)) refuse(cat("key cache must be fp16 or bf16, got ", name_of(k.scalar_type())));
  const Tensor weights = any_tensor(args[2], "weights are required"), lengths = any_tensor(args[3], kLengths);
  const int64_t B = k.size(0), D = k.size(3), Hk = k.size(l.head());
  if (Hk == 0 || D == 0) refuse("the caches need at least one head of at least one element");
  const int64_t C = check_cache(k, v, lengths, weights, l, B, Hk, D, k);
  const int64_t keep = int_arg(args[4], "keep"), sinks = int_arg(args[5], "sinks"), recent = int_arg(args[6], "recent");
  if (keep < 1 || sinks < 0 || recent < 0 || sinks > keep || recent > keep - sinks)
    refuse(cat("sinks (", sinks, ") and recent (", recent, ") must fit in keep (", keep, ")"));
  no_gradient("evict_by_weight", {&k, &v, &weights});
  Tensor ko, vo, wo;
  if (args[7] != Py_None) {
    const char* what = "out must be (key, value, weights)";
    if (!PyTuple_Check(args[7]) || PyTuple_GET_SIZE(args[7]) != 3) refuse(what);
    ko = tensor_arg(PyTuple_GET_ITEM(args[7], 0), "key cache", 4);
    vo = tensor_arg(PyTuple_GET_ITEM(args[7], 1), "value cache", 4);
    wo = any_tensor(PyTuple_GET_ITEM(args[7], 2), what);
    if (check_cache(ko, vo, lengths, wo, l, B, Hk, D, k) < keep) refuse(cat(what, " with at least keep = ", keep, " slots"));
    if (ko.stride(3) != 1 || vo.stride(3) != 1) refuse("out is written in place and needs unit head-dim stride");
    if (repeats(ko) || repeats(vo) || repeats(wo)) refuse("out is written in place and may not repeat memory");
    for (const Tensor* x : std::initializer_list<const Tensor*>{&ko, &vo, &wo})
      for (const Tensor* y : std::initializer_list<const Tensor*>{&k, &v, &weights, &lengths})
        if (meet(*x, *y)) refuse("out may not share memory with the inputs");
    if (meet(ko, vo) || meet(ko, wo) || meet(vo, wo)) refuse("out's tensors may not share memory with each other");
    no_gradient("evict_by_weight", {&ko, &vo, &wo});
  }
  need_cuda("evict_by_weight", k);
  const c10::cuda::OptionalCUDAGuard guard(k.device());
  k = unit_rows(k);
  v = unit_rows(v);
  if (!ko.defined()) {
    ko = l.bhsd ? at::empty({B, Hk, keep, D}, k.options()) : at::empty({B, keep, Hk, D}, k.options());
    vo = at::empty_like(ko);
    wo = at::empty({B, Hk, keep}, weights.options());
  }
  Tensor lengths_out = at::empty_like(lengths), index = at::empty({B, Hk, keep}, lengths.options());
  if (B) {
    fa4d_evict_args a;
    a.k = k.data_ptr();
    a.v = v.data_ptr();
    a.weights = weights.data_ptr<float>();
    a.lengths = lengths.data_ptr<int32_t>();
    a.k_out = ko.data_ptr();
    a.v_out = vo.data_ptr();
    a.weights_out = wo.data_ptr<float>();
    a.lengths_out = lengths_out.data_ptr<int32_t>();
    a.index_out = index.data_ptr<int32_t>();
    set3(a.k_stride, k, l);
    set3(a.v_stride, v, l);
    set3(a.k_out_stride, ko, l);
    set3(a.v_out_stride, vo, l);
    set_weights(a.weights_stride, weights);
    set_weights(a.weights_out_stride, wo);
    a.B = small(B, "batch");
    a.C = small(C, "cache");
    a.Hk = small(Hk, "heads");
    a.D = small(D, "head dim");
    a.keep = small(keep, "keep");
    a.sinks = small(sinks, "sinks");
    a.recent = small(recent, "recent");
    check(fa4d_evict(&a, stream_of(k)), "fa4d_evict");
    written({&ko, &vo, &wo});
  }
  PyObject* out = PyTuple_New(5);
  if (!out) return nullptr;
  const Tensor* all[] = {&ko, &vo, &wo, &lengths_out, &index};
  for (int i = 0; i < 5; ++i) {
    // The caller's own objects where it gave `out`.
    PyObject* x = i < 3 && args[7] != Py_None ? Py_NewRef(PyTuple_GET_ITEM(args[7], i)) : THPVariable_Wrap(*all[i]);
    PyTuple_SET_ITEM(out, i, x);
  }
  return out;
}

// No exception leaves an entry point: refusals and torch's errors become Python ones.
template <PyObject* (*kBody)(PyObject* const*), int kArgs>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != kArgs) {
    PyErr_Format(PyExc_TypeError, "expected %d arguments, got %zd", kArgs, n);
    return nullptr;
  }
  try {
    return kBody(args);
  } catch (const Refused& e) {
    PyErr_SetString(e.type, e.text.c_str());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

#define FA4D_ENTRY(name, n) \
  { #name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(entry<name, n>)), METH_FASTCALL, nullptr }
PyMethodDef kMethods[] = {FA4D_ENTRY(make_table, 5),      FA4D_ENTRY(table_turns, 1),
                          FA4D_ENTRY(rotary, 5),
                          FA4D_ENTRY(rotary_append, 10),  FA4D_ENTRY(shared_prefix_attention, 11),
                          FA4D_ENTRY(evict_by_weight, 9), {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_fa4d_host", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fa4d_host() { return PyModule_Create(&kModule); }
