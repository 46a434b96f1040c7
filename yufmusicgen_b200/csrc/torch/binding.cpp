// Python module `_yuf_torch`: the gated recurrence and dropout as calls on torch
// tensors, with their autograd nodes.  It checks arguments, allocates outputs and
// hands plain pointers to the C ABI (include/yufb200.h) on the tensors' device and
// its current stream.  In C++ because the smallest calls are bound by the host: a
// training call through a Python autograd function took 160 us, 100 of it Python.
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <array>
#include <optional>
#include <sstream>
#include <string>

#include "yufb200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// An error for Python, of a given type.
struct Refused {
  PyObject* type;
  std::string message;
};
template <typename... Args>
[[noreturn]] void refuse(PyObject* type, const Args&... args) {
  std::ostringstream s;
  (s << ... << args);
  throw Refused{type, s.str()};
}
#define NEED(cond, type, ...) \
  do {                        \
    if (!(cond)) refuse(PyExc_##type, __VA_ARGS__); \
  } while (0)

int dtype_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return YUF_DTYPE_F32;
    case at::kBFloat16: return YUF_DTYPE_BF16;
    case at::kHalf: return YUF_DTYPE_F16;
    default: return -1;
  }
}
// Whether t has memory behind it.  Fake tensors, wrappers of other tensors and tensors of
// zeros that torch does not store have none, and data_ptr() of a slice of one is an offset
// from address 0.
bool has_memory(const Tensor& t) { return t.has_storage() && t.unsafeGetTensorImpl()->storage_initialized(); }
// for the library: every pointer it gets comes from here
template <typename T>
T* ptr(const Tensor& t) {
  if (!t.defined()) return nullptr;
  TORCH_CHECK(has_memory(t), "a tensor without memory of its own cannot go to a kernel");
  return static_cast<T*>(t.data_ptr());
}
// the values as they lie in memory: a copy where torch negates them only when it reads
// them, or does not store them because they are all zero
Tensor as_stored(const Tensor& t) {
  if (!t.defined() || !(t.is_neg() || t._is_zerotensor())) return t;
  return t._is_zerotensor() ? at::zeros(t.sizes(), t.options()) : t.resolve_neg();
}
// a unit stride along the last axis (a copy where it has none)
Tensor unit_rows(const Tensor& t) {
  return !t.defined() || t.size(-1) == 1 || t.stride(-1) == 1 ? as_stored(t) : as_stored(t).contiguous();
}
Tensor dense(const Tensor& t) { return t.defined() ? as_stored(t).contiguous() : t; }
// Arguments of an autograd node that may be absent.
using Maybe = std::optional<Tensor>;
Maybe maybe(const Tensor& t) { return t.defined() ? Maybe(t) : std::nullopt; }
Tensor defined_or_not(const Maybe& t) { return t.has_value() ? *t : Tensor(); }
bool wants_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}
// Derivatives in forward mode are not there: a tangent must not get lost in silence.  Where
// forward mode is off _fw_grad gives none.
void no_tangents(const char* name, std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    NEED(!t->defined() || !t->_fw_grad(/*level=*/0).defined(), NotImplementedError, name,
         " has no forward-mode derivatives (an input has a tangent)");
}
void no_tangents(const char* name, const variable_list& grads) {  // of a backward
  for (const Tensor& t : grads)
    TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(/*level=*/0).defined(), name,
                                " has no forward-mode derivatives (a gradient has a tangent)");
}
// A failing library call (the message of its thread).
void check(const char* name, yuf_status_t st) {
  TORCH_CHECK(st == YUF_OK, name, " failed with ", yuf_status_string(st), ": ", yuf_last_error());
}
// Gradients made while a graph of the backward is recorded (create_graph): they may be
// used, but an attempt to differentiate through them is an error.
variable_list once(const char* name, bool recorded, variable_list grads) {
  if (!recorded) return grads;
  for (Tensor& t : grads)
    if (t.defined())
      t = torch::autograd::DelayedError(std::string(name) + ": the gradients are not differentiable themselves", 1)
              .apply({t.detach().set_requires_grad(true)})[0];
  return grads;
}
// The tensors' device for as long as a call lasts, and its current stream.
struct On {
  c10::cuda::CUDAGuard guard;
  void* stream;
  explicit On(const Tensor& t)
      : guard(t.device()), stream(c10::cuda::getCurrentCUDAStream(t.device().index()).stream()) {}
};

// ---- gated recurrence -------------------------------------------------------

struct Inputs {
  Tensor x, f, g, lower, state, cu;  // g, lower, state and cu may be undefined
  int dtype;
  int64_t rows;                      // states
  int B() const { return (int)x.size(0); }
  int T() const { return (int)x.size(1); }
  int D() const { return (int)x.size(2); }
  int n_seqs() const { return cu.defined() ? (int)rows : 0; }
};

void check_tokens(const Tensor& x, const Tensor& f, const Tensor& g, const Tensor& lower, int64_t ndim) {
  NEED(x.defined() && f.defined(), TypeError, "gated scan: x and forget must be tensors");
  NEED(x.dim() == ndim, ValueError, "gated scan: x must have shape ", ndim == 3 ? "[B, T, D]" : "[B, D]", ", got ",
       x.sizes());
  NEED(dtype_of(x) >= 0, TypeError, "gated scan: x must be float32, bfloat16 or float16, got ", x.scalar_type());
  for (const Tensor* t : {&f, &g})
    NEED(!t->defined() || (t->sizes() == x.sizes() && t->scalar_type() == x.scalar_type() && t->device() == x.device()),
         ValueError, "gated scan: ", t == &f ? "forget" : "gate", " must have x's shape, type and device");
  NEED(x.size(-1) >= 1, ValueError, "gated scan: D must be at least 1");
  // the library's own limits, before anything is allocated
  bool fits = true;
  for (int64_t n : x.sizes()) fits = fits && n <= INT32_MAX;
  const int64_t B = x.size(0), D = x.size(-1);
  if (ndim == 3) fits = fits && x.size(1) <= (int64_t{1} << 30) && B * ((D + 31) / 32) <= (int64_t{1} << 26);
  else fits = fits && B * D <= (int64_t{1} << 38);
  NEED(fits, ValueError, "gated scan: x is too large: ", x.sizes());
  if (lower.defined()) {
    NEED(lower.scalar_type() == at::kFloat, TypeError, "gated scan: lower must be float32");
    NEED(lower.dim() == 1 && lower.size(0) == x.size(-1) && lower.device() == x.device(), ValueError,
         "gated scan: lower must be a [D] tensor on x's device");
  }
}
void check_cuda(const Tensor& x) { NEED(x.is_cuda(), ValueError, "gated scan inputs must be on CUDA"); }

int64_t check_states(const Tensor& x, const Tensor& state, const Tensor& cu) {
  int64_t rows = x.size(0);
  if (cu.defined()) {
    NEED(rows == 1, ValueError, "gated scan: packed sequences need x of shape [1, total, D]");
    NEED(cu.scalar_type() == at::kInt && cu.dim() == 1 && cu.numel() >= 1 && cu.numel() <= INT32_MAX, ValueError,
         "gated scan: cu_seqlens must be an int32 [n_sequences + 1] tensor");
    NEED(cu.device() == x.device() && cu.is_contiguous(), ValueError,
         "gated scan: cu_seqlens must be contiguous and on x's device");
    rows = cu.numel() - 1;
  }
  if (state.defined()) {
    NEED(state.scalar_type() == at::kFloat, TypeError, "gated scan: state must be float32");
    NEED(state.dim() == 2 && state.size(0) == rows && state.size(1) == x.size(2) && state.device() == x.device(),
         ValueError, "gated scan: state must be a [", rows, ", ", x.size(2), "] tensor on x's device");
  }
  return rows;
}

// Whether an input shares memory with the state that a step updates in place: `ns` state
// rows of `ws` bytes, `ss` bytes apart, and `nt` of the input's, its first byte `d` bytes
// behind the state's first.
bool rows_clash(int64_t ns, int64_t ws, int64_t ss, int64_t nt, int64_t wt, int64_t ts, int64_t d) {
  if (ts == 0) nt = 1;  // a shared row is one row
  for (int64_t i = 0; i < ns; ++i) {
    const int64_t at = i * ss - d, end = at - wt;  // state row i from the input's first byte on; rows that end before it
    const int64_t j = ts == 0 || end < 0 ? 0 : end / ts + 1;
    if (j < nt && j * ts < at + ws && j * ts + wt > at) return true;
  }
  return false;
}
void check_apart(const Tensor& state, const Tensor* gate, std::initializer_list<const Tensor*> inputs) {
  const int64_t ns = state.size(0), ws = state.size(1) * 4, ss = state.stride(0) * 4;
  if (ns == 0) return;
  const char* const from = static_cast<const char*>(state.const_data_ptr());
  const char* const to = from + (ns - 1) * ss + ws;
  for (const Tensor* t : inputs) {
    if (!t->defined() || t->_is_zerotensor()) continue;
    const char* const at = static_cast<const char*>(t->const_data_ptr());
    if (at >= to) continue;
    // all but the gate may be the state element by element: it is written from their values
    const int64_t e = (int64_t)t->itemsize(), wt = t->size(-1) * e, nt = t->dim() == 2 ? t->size(0) : 1,
                  ts = nt > 1 ? t->stride(0) * e : 0;
    if (at == from && wt == ws && nt == ns && (ns == 1 || ts == ss) && t != gate) continue;
    if (at + (nt - 1) * ts + wt <= from || (t->size(-1) > 1 && t->stride(-1) != 1)) continue;  // apart, or copied first
    NEED(!rows_clash(ns, ws, ss, nt, wt, ts, at - from), ValueError,
         "gated scan: state must not share memory with an input, other than x or forget element by element");
  }
}

Tensor workspace(const Inputs& in, bool backward) {
  const size_t n = yuf_gated_scan_workspace_bytes(in.B(), in.T(), in.D(), in.dtype, backward);
  return n ? at::empty({(int64_t)n}, in.x.options().dtype(at::kByte)) : Tensor();
}

// y, final state and, where `save`, the backward's checkpoints
std::array<Tensor, 3> scan_forward(const Inputs& in, bool save) {
  const Tensor &x = in.x, &f = in.f, &g = in.g;
  const auto f32 = x.options().dtype(at::kFloat);
  On on(x);
  Tensor y = at::empty({x.size(0), x.size(1), x.size(2)}, x.options());
  Tensor last = at::empty({in.rows, x.size(2)}, f32), ckpt;
  if (save) {
    const int block = yuf_gated_scan_block(in.dtype);
    ckpt = at::empty({x.size(0), (x.size(1) + block - 1) / block, x.size(2)}, f32);
  }
  const Tensor work = workspace(in, false);
  const int64_t strides[6] = {x.stride(0), x.stride(1), f.stride(0), f.stride(1),
                              g.defined() ? g.stride(0) : 0, g.defined() ? g.stride(1) : 0};
  check("yuf_gated_scan_forward",
        yuf_gated_scan_forward(ptr<void>(x), ptr<void>(f), ptr<void>(g), strides, ptr<float>(in.lower),
                               ptr<float>(in.state), ptr<int32_t>(in.cu), in.n_seqs(), ptr<void>(y), ptr<float>(last),
                               ptr<float>(ckpt), ptr<void>(work), in.dtype, in.B(), in.T(), in.D(), on.stream));
  return {y, last, ckpt};
}

struct GatedScan : torch::autograd::Function<GatedScan> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& f, const Maybe& g,
                               const Maybe& lower, const Maybe& state, const Maybe& cu, int64_t rows) {
    const Inputs in{x, f, defined_or_not(g), defined_or_not(lower), defined_or_not(state), defined_or_not(cu),
                    dtype_of(x), rows};
    auto out = scan_forward(in, true);
    ctx->save_for_backward({x, f, in.g, in.lower, in.state, in.cu, out[2]});
    ctx->saved_data["rows"] = rows;
    ctx->saved_data["wants"] = (int64_t)((in.lower.defined() && in.lower.requires_grad()) |
                                         (in.state.defined() && in.state.requires_grad()) << 1);
    ctx->set_materialize_grads(false);
    return {out[0], out[1]};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const bool recorded = at::GradMode::is_enabled();
    const at::NoGradGuard no_grad;
    no_tangents("gated_scan", grads);
    const auto saved = ctx->get_saved_variables();
    const Inputs in{saved[0], saved[1], saved[2], saved[3], saved[4], saved[5], dtype_of(saved[0]),
                    ctx->saved_data["rows"].toInt()};
    const Tensor &x = in.x, &f = in.f, &g = in.g;
    On on(x);
    const std::array<int64_t, 3> shape{x.size(0), x.size(1), x.size(2)};
    const Tensor dy = grads[0].defined() ? unit_rows(grads[0]) : at::zeros(shape, x.options());
    const Tensor dlast = dense(grads[1]);
    const auto like = [&](const Tensor& t) { return t.defined() ? at::empty(shape, x.options()) : Tensor(); };
    const Tensor dx = like(x), df = like(f), dg = like(g), work = workspace(in, true);
    Tensor dlower, dstate;
    const int64_t wants = ctx->saved_data["wants"].toInt();
    if (wants & 1) dlower = at::empty_like(in.lower);
    if (wants & 2) dstate = at::empty_like(in.state);
    const int64_t strides[8] = {x.stride(0), x.stride(1), f.stride(0), f.stride(1), g.defined() ? g.stride(0) : 0,
                                g.defined() ? g.stride(1) : 0, dy.stride(0), dy.stride(1)};
    check("yuf_gated_scan_backward",
          yuf_gated_scan_backward(ptr<void>(x), ptr<void>(f), ptr<void>(g), ptr<void>(dy), strides,
                                  ptr<float>(in.lower), ptr<float>(in.state), ptr<int32_t>(in.cu), in.n_seqs(),
                                  ptr<float>(saved[6]), ptr<float>(dlast), ptr<void>(dx), ptr<void>(df), ptr<void>(dg),
                                  ptr<float>(dlower), ptr<float>(dstate), ptr<void>(work), in.dtype, in.B(), in.T(),
                                  in.D(), on.stream));
    return once("gated_scan", recorded, {dx, df, dg, dlower, dstate, Tensor(), Tensor()});
  }
};

// ---- dropout ------------------------------------------------------------------

// Stride between the rows (last axis) of t, -1 where they have none.
int64_t row_stride(const Tensor& t) {
  const int64_t n = t.dim();
  if (t.size(n - 1) != 1 && t.stride(n - 1) != 1) return -1;
  int64_t row = -1, expect = 0;
  for (int64_t d = n - 2; d >= 0; --d) {
    if (t.size(d) == 1) continue;
    if (row < 0) row = t.stride(d);
    else if (t.stride(d) != expect) return -1;
    expect = t.stride(d) * t.size(d);
  }
  return row < 0 ? t.size(n - 1) : row;
}

struct Draw {
  double p;
  uint64_t seed, step;
};
// step_t, where defined, holds the step on the device
Tensor drop(Tensor x, Tensor r, const Draw& d, const Tensor& step_t, at::ScalarType out_type) {
  On on(x);
  x = as_stored(x);
  r = as_stored(r);
  const Tensor out = at::empty(x.sizes(), x.options().dtype(out_type).memory_format(at::MemoryFormat::Contiguous));
  int64_t rows = 1, cols = x.numel(), xs = cols, rs = cols;
  if (x.dim() > 0 && x.numel() > 0 && !(x.is_contiguous() && (!r.defined() || r.is_contiguous()))) {
    cols = x.size(-1);
    rows = x.numel() / cols;
    xs = row_stride(x);
    if (xs < 0) x = x.contiguous(), xs = cols;
    rs = r.defined() ? row_stride(r) : cols;
    if (rs < 0) r = r.contiguous(), rs = cols;
  }
  check("yuf_dropout", yuf_dropout(ptr<void>(x), xs, dtype_of(x), ptr<void>(r), rs, ptr<void>(out), dtype_of(out), rows,
                                   cols, d.p, d.seed, d.step, ptr<uint64_t>(step_t), on.stream));
  return out;
}

struct Dropout : torch::autograd::Function<Dropout> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Maybe& residual, const Maybe& step_on_device,
                        double p, int64_t seed, int64_t step) {
    const Tensor r = defined_or_not(residual), step_t = defined_or_not(step_on_device);
    ctx->saved_data["draw"] = c10::IValue(std::vector<int64_t>{seed, step, (int64_t)x.scalar_type()});
    ctx->saved_data["p"] = p;
    ctx->saved_data["residual"] = r.defined() && r.requires_grad();
    if (step_t.defined()) ctx->save_for_backward({step_t});  // a step changed before the backward is an error
    ctx->set_materialize_grads(false);
    return drop(x, r, Draw{p, (uint64_t)seed, (uint64_t)step}, step_t, r.defined() ? r.scalar_type() : x.scalar_type());
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const bool recorded = at::GradMode::is_enabled();
    const at::NoGradGuard no_grad;
    no_tangents("dropout", grads);
    const auto draw = ctx->saved_data["draw"].toIntVector();
    const auto saved = ctx->get_saved_variables();
    const Tensor& dy = grads[0];
    Tensor dx;
    if (dy.defined() && ctx->needs_input_grad(0))
      dx = drop(dy, Tensor(), Draw{ctx->saved_data["p"].toDouble(), (uint64_t)draw[0], (uint64_t)draw[1]},
                saved.empty() ? Tensor() : saved[0], (at::ScalarType)draw[2]);
    const Tensor dr = ctx->saved_data["residual"].toBool() ? dy : Tensor();
    dx = once("dropout", recorded, {dx})[0];  // dr is dy, with its own history
    return {dx, dr, Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

// ---- Python ---------------------------------------------------------------------

Tensor tensor_of(PyObject* o, const char* what) {
  if (o == Py_None) return Tensor();
  NEED(THPVariable_Check(o), TypeError, what, " must be a tensor, got ", Py_TYPE(o)->tp_name);
  const Tensor& t = THPVariable_Unpack(o);
  NEED(t._is_zerotensor() || has_memory(t), TypeError, what,
       " must be a plain tensor with memory of its own (not fake, batched, sparse or a wrapper)");
  return t;
}
// a Python integer modulo 2^64
uint64_t word_of(PyObject* o) {
  PyObject* const n = PyNumber_Index(o);
  if (!n) throw Refused{nullptr, ""};
  const uint64_t v = PyLong_AsUnsignedLongLongMask(n);
  Py_DECREF(n);
  if (PyErr_Occurred()) throw Refused{nullptr, ""};
  return v;
}
template <typename F>
PyObject* guarded(const F& body) {
  try {
    return body();
  } catch (const Refused& e) {
    if (e.type) PyErr_SetString(e.type, e.message.c_str());
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}
bool arity(Py_ssize_t n, Py_ssize_t want, const char* name) {
  if (n == want) return true;
  PyErr_Format(PyExc_TypeError, "%s takes %zd arguments (%zd given)", name, want, n);
  return false;
}

// gated_scan(x, forget, gate, lower, state, cu_seqlens) -> (y, final_state)
PyObject* py_gated_scan(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arity(n, 6, "gated_scan")) return nullptr;
  return guarded([&]() -> PyObject* {
    const char* names[] = {"x", "forget", "gate", "lower", "state", "cu_seqlens"};
    Tensor t[6];
    for (int i = 0; i < 6; ++i) t[i] = tensor_of(a[i], names[i]);
    no_tangents("gated_scan", {&t[0], &t[1], &t[2], &t[3], &t[4]});
    check_tokens(t[0], t[1], t[2], t[3], 3);
    const int64_t rows = check_states(t[0], t[4], t[5]);
    check_cuda(t[0]);
    for (int i = 0; i < 3; ++i) t[i] = unit_rows(t[i]);
    t[5] = as_stored(t[5]);
    t[3] = dense(t[3]);
    t[4] = dense(t[4]);
    Tensor y, last;
    if (wants_grad({&t[0], &t[1], &t[2], &t[3], &t[4]})) {
      auto out = GatedScan::apply(t[0], t[1], maybe(t[2]), maybe(t[3]), maybe(t[4]), maybe(t[5]), rows);
      y = out[0];
      last = out[1];
    } else {
      auto out = scan_forward(Inputs{t[0], t[1], t[2], t[3], t[4], t[5], dtype_of(t[0]), rows}, false);
      y = out[0];
      last = out[1];
    }
    PyObject* const r = PyTuple_New(2);
    if (!r) return nullptr;
    PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(std::move(y)));
    PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(std::move(last)));
    return r;
  });
}

// gated_scan_step(x, forget, state, gate, lower) -> y; state in place
PyObject* py_gated_scan_step(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arity(n, 5, "gated_scan_step")) return nullptr;
  return guarded([&]() -> PyObject* {
    Tensor x = tensor_of(a[0], "x"), f = tensor_of(a[1], "forget"), state = tensor_of(a[2], "state"),
           g = tensor_of(a[3], "gate"), lower = tensor_of(a[4], "lower");
    no_tangents("gated_scan_step", {&x, &f, &state, &g, &lower});
    check_tokens(x, f, g, lower, 2);
    NEED(state.defined() && state.scalar_type() == at::kFloat, TypeError, "gated scan: state must be float32");
    NEED(state.sizes() == x.sizes() && state.device() == x.device(), ValueError,
         "gated scan: state must be a [B, D] tensor on x's device");
    const int64_t B = x.size(0), D = x.size(1);
    NEED((D == 1 || state.stride(1) == 1) && (B <= 1 || state.stride(0) >= D), ValueError,
         "gated scan: state rows must be contiguous and must not overlap");
    NEED(!state.is_neg() && !state._is_zerotensor(), ValueError,
         "gated scan: state must not be a lazily negated view or a tensor of zeros without memory");
    NEED(!wants_grad({&x, &f, &g, &lower, &state}), NotImplementedError,
         "gated_scan_step has no gradients: use gated_scan, or torch.no_grad()");
    check_apart(state, &g, {&x, &f, &g, &lower});
    check_cuda(x);
    x = unit_rows(x);
    f = unit_rows(f);
    g = unit_rows(g);
    lower = dense(lower);
    On on(x);
    Tensor y = at::empty({B, D}, x.options());
    const int64_t strides[3] = {x.stride(0), f.stride(0), g.defined() ? g.stride(0) : 0};
    check("yuf_gated_scan_step",
          yuf_gated_scan_step(ptr<void>(x), ptr<void>(f), ptr<void>(g), strides, ptr<float>(lower), ptr<float>(state),
                              state.stride(0), ptr<void>(y), dtype_of(x), (int)B, (int)D, on.stream));
    if (!state.is_inference()) state.unsafeGetTensorImpl()->bump_version();
    return THPVariable_Wrap(std::move(y));
  });
}

// dropout(x, p, seed, step, residual) -> y
PyObject* py_dropout(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arity(n, 5, "dropout")) return nullptr;
  return guarded([&]() -> PyObject* {
    const Tensor x = tensor_of(a[0], "dropout: x"), r = tensor_of(a[4], "dropout: residual");
    no_tangents("dropout", {&x, &r});
    NEED(x.defined(), TypeError, "dropout: x must be a tensor, got None");
    NEED(dtype_of(x) >= 0, TypeError, "dropout: x must be float32, bfloat16 or float16, got ", x.scalar_type());
    const double p = PyFloat_AsDouble(a[1]);
    if (p == -1.0 && PyErr_Occurred()) throw Refused{nullptr, ""};
    NEED(p >= 0.0 && p <= 1.0, ValueError, "dropout: p must lie in [0, 1], got ", p);
    if (r.defined()) {
      NEED(r.sizes() == x.sizes() && r.device() == x.device(), ValueError,
           "dropout: residual must have x's shape and device");
      NEED(r.scalar_type() == x.scalar_type() || r.scalar_type() == at::kFloat, TypeError,
           "dropout: residual must have x's type or be float32");
    }
    NEED(x.numel() <= (int64_t{1} << 40), ValueError, "dropout: x is too large: ", x.sizes());
    Draw d{p, word_of(a[2]), 0};
    Tensor step_t;
    if (THPVariable_Check(a[3])) {
      step_t = as_stored(tensor_of(a[3], "dropout: step"));
      NEED(step_t.scalar_type() == at::kLong && step_t.numel() == 1 && step_t.device() == x.device(), ValueError,
           "dropout: a step tensor must hold one int64 on x's device");
    } else {
      d.step = word_of(a[3]);
    }
    NEED(x.is_cuda(), ValueError, "dropout: x must be on CUDA");
    return THPVariable_Wrap(wants_grad({&x, &r})
                                ? Dropout::apply(x, maybe(r), maybe(step_t), d.p, (int64_t)d.seed, (int64_t)d.step)
                                : drop(x, r, d, step_t, r.defined() ? r.scalar_type() : x.scalar_type()));
  });
}

// row_stride(t): what dropout takes as the stride of t's rows, or None
PyObject* py_row_stride(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arity(n, 1, "row_stride")) return nullptr;
  return guarded([&]() -> PyObject* {
    const int64_t s = row_stride(tensor_of(a[0], "t"));
    if (s < 0) Py_RETURN_NONE;
    return PyLong_FromLongLong(s);
  });
}

PyMethodDef methods[] = {
    {"gated_scan", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_gated_scan)), METH_FASTCALL, nullptr},
    {"gated_scan_step", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_gated_scan_step)), METH_FASTCALL,
     nullptr},
    {"dropout", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_dropout)), METH_FASTCALL, nullptr},
    {"row_stride", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_row_stride)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_yuf_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__yuf_torch(void) { return PyModule_Create(&module); }
