// PyTorch side of the language-model operators (layer norm, gated scan, the
// layer's scan, logit shaping): allocation, streams and autograd nodes around
// the C ABI, in C++ because a small call is bound by the host.  A call through
// ctypes and a Python autograd Function took 10.8 us forward and, trained,
// 104 us, of which the hand-over to the engine's thread and back is 45; here a
// call takes 7 and a small training step 65 to 80.
// Arguments arrive checked (norm.py, scan.py, cuda/ops.py, sampling.py); the
// entry points of the C ABI are handed over by bind(), so that one library is
// loaded whoever calls.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>

#include <climits>
#include <optional>
#include <stdexcept>
#include <string>

#include "../../include/gfn_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// Entry points in the order of _lib.TORCH_ENTRIES.
#define GFN_ENTRIES(X)                                                                            \
  X(gfn_status_string) X(gfn_last_error_message) X(gfn_layer_norm_forward)                        \
  X(gfn_layer_norm_backward_workspace_floats) X(gfn_layer_norm_backward)                          \
  X(gfn_gated_scan_states_floats) X(gfn_gated_scan_workspace_bytes) X(gfn_gated_scan_forward)     \
  X(gfn_gated_scan_backward) X(gfn_layer_scan_forward) X(gfn_layer_scan_backward) X(gfn_process_logits)
struct Api {
#define X(name) decltype(&::name) name;
  GFN_ENTRIES(X)
#undef X
};
Api api = {};
PyObject* gfn_error = nullptr;

struct Failure : std::runtime_error {
  using std::runtime_error::runtime_error;
};

void check(int status, const char* what) {
  if (status)
    throw Failure(std::string(what) + ": " + api.gfn_status_string(status) + " (" + std::to_string(status) +
                  "): " + api.gfn_last_error_message());
}

// Runs `f`, the body of a node's backward.  It runs on a thread of the engine,
// which hands the caller's thread a Python error as it is and makes a RuntimeError
// of any other.
template <class F>
variable_list backward_body(F f) {
  try {
    return f();
  } catch (const Failure& e) {
    const PyGILState_STATE held = PyGILState_Ensure();
    PyErr_SetString(gfn_error, e.what());
    python_error error;
    error.persist();
    PyGILState_Release(held);
    throw error;
  }
}

int extent(int64_t n, const char* what) {
  if (n > INT_MAX) throw Failure(std::string(what) + ": extent " + std::to_string(n) + " above 2^31 - 1");
  return (int)n;
}

int code_of(const Tensor& t) {
  return t.scalar_type() == at::kFloat ? GFN_F32 : t.scalar_type() == at::kBFloat16 ? GFN_BF16 : GFN_F16;
}
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
float* fptr(const Tensor& t) { return static_cast<float*>(ptr(t)); }

// The tensor's device made current, and its current stream.
struct Launch {
  c10::cuda::CUDAGuard guard;
  gfn_stream_t stream;
  explicit Launch(const Tensor& t)
      : guard(t.device()), stream(c10::cuda::getCurrentCUDAStream(t.get_device()).stream()) {}
};

Tensor fresh(const Tensor& like, at::IntArrayRef sizes, at::ScalarType type) {
  return at::empty(sizes, like.options().dtype(type));
}
Tensor fresh(const Tensor& like) { return at::empty(like.sizes(), like.options()); }
using Maybe = std::optional<Tensor>;  // an operand that may be absent, as a node's argument
Maybe maybe(const Tensor& t) { return t.defined() ? Maybe(t) : Maybe(); }
Tensor whole(const Tensor& t) { return t.defined() && !t.is_contiguous() ? t.contiguous() : t; }

// Gradients of a backward whose result is not differentiable: where a graph of
// them is being recorded, using that graph raises.
variable_list first_order(variable_list out, const variable_list& grads, bool recording) {
  bool wanted = false;
  for (const Tensor& g : grads) wanted = wanted || (g.defined() && g.requires_grad());
  if (!recording || !wanted) return out;
  variable_list in;
  for (const Tensor& t : out)
    if (t.defined()) in.push_back(t.detach().set_requires_grad(true));
  const int64_t n = (int64_t)in.size();
  auto error = std::make_shared<torch::autograd::DelayedError>(
      "this operator's gradients cannot be differentiated again", n);
  variable_list marked = (*error)(std::move(in));
  size_t k = 0;
  for (Tensor& t : out)
    if (t.defined()) t = marked[k++];
  return out;
}

// ---------------------------------------------------------------------- norm
struct Rows {
  Tensor t;
  long long n, stride;
};

// Rows of `dim` elements with inner stride 1, in place where t has them.
Rows rows_of(const Tensor& t, int64_t dim) {
  if (t.is_contiguous()) return {t, t.numel() / dim, dim};
  Tensor r = t.reshape({-1, dim});
  if ((dim > 1 && r.stride(1) != 1) || (r.size(0) > 1 && r.stride(0) < dim)) r = r.contiguous();  // expanded rows overlap
  return {r, r.size(0), r.size(0) > 1 ? r.stride(0) : dim};
}

Tensor norm_run(const Tensor& x, const Tensor& w, const Tensor& b, double eps, Tensor* stats) {
  at::AutoDispatchBelowADInplaceOrView plain;
  const Launch on(x);
  const int dim = extent(x.size(-1), "layer_norm");
  const Rows r = rows_of(x, dim);
  Tensor y = fresh(x);
  if (stats) *stats = fresh(x, {r.n, 2}, at::kFloat);
  const Tensor& wt = w.defined() ? w : b.defined() ? b : x;
  check(api.gfn_layer_norm_forward(r.t.data_ptr(), r.stride, ptr(w), ptr(b), code_of(x), code_of(wt), r.n, dim,
                                   (float)eps, y.data_ptr(), stats ? fptr(*stats) : nullptr, on.stream),
        "gfn_layer_norm_forward");
  return y;
}

struct NormNode : torch::autograd::Function<NormNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Maybe& weight, const Maybe& bias, double eps) {
    const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor());
    Tensor stats;
    Tensor y = norm_run(x, w, b, eps, &stats);
    // the caller's own tensors, so that a later in-place change of one is noticed
    ctx->save_for_backward({x, w, stats});
    ctx->saved_data["weights"] = (int64_t)(w.defined() ? w : b.defined() ? b : x).scalar_type();
    ctx->saved_data["bias"] = b.defined();
    return y;
  }

  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    return backward_body([&] { return gradients(ctx, grads); });
  }

  static variable_list gradients(AutogradContext* ctx, const variable_list& grads) {
    const bool recording = at::GradMode::is_enabled();
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &stats = saved[2];
    Tensor dx, dw, db, ws;
    {
      at::AutoDispatchBelowADInplaceOrView plain;
      const Launch on(x);
      const auto wt = (at::ScalarType)ctx->saved_data["weights"].toInt();
      const int dim = (int)x.size(-1);
      const Rows r = rows_of(x, dim), g = rows_of(grads[0], dim);
      if (ctx->needs_input_grad(0)) dx = fresh(x);
      // inputs are numbered without the absent ones
      if (w.defined() && ctx->needs_input_grad(1)) dw = fresh(x, {dim}, wt);
      if (ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(w.defined() ? 2 : 1)) db = fresh(x, {dim}, wt);
      long long n = 0;
      if (dw.defined() || db.defined()) {
        n = api.gfn_layer_norm_backward_workspace_floats(r.n, dim);
        ws = fresh(x, {n}, at::kFloat);
      }
      const int wcode = wt == at::kFloat ? GFN_F32 : wt == at::kBFloat16 ? GFN_BF16 : GFN_F16;
      check(api.gfn_layer_norm_backward(r.t.data_ptr(), r.stride, g.t.data_ptr(), g.stride, ptr(w), fptr(stats),
                                        code_of(x), wcode, r.n, dim, ptr(dx), ptr(dw), ptr(db), fptr(ws), n,
                                        on.stream),
            "gfn_layer_norm_backward");
    }
    return first_order({dx, dw, db, Tensor()}, grads, recording);
  }
};

// --------------------------------------------------------------------- scans
// t [B, L, D] with inner stride 1 (itself where it has one: strided and
// broadcast batches and steps are read in place).
Tensor operand(const Tensor& t) {
  return !t.defined() || t.is_contiguous() || t.stride(2) == 1 || t.size(2) == 1 ? t : t.contiguous();
}

struct Operand {
  Tensor t;
  void* p = nullptr;
  long long sb = 0, st = 0;
  explicit Operand(const Tensor& u) : t(operand(u)) {
    if (!t.defined()) return;
    p = t.data_ptr();
    sb = t.stride(0);
    st = t.stride(1);
  }
};

struct Shape {
  int B, L, D;
  Shape(const Tensor& x, int parts, const char* what)
      : B(extent(x.size(0), what)), L(extent(x.size(1), what)), D(extent(x.size(2) / parts, what)) {}
  Tensor states(const Tensor& x) const { return fresh(x, {api.gfn_gated_scan_states_floats(B, L, D)}, at::kFloat); }
  Tensor row(const Tensor& x) const { return fresh(x, {B, D}, at::kFloat); }
  long long bytes() const { return L > 1 ? api.gfn_gated_scan_workspace_bytes(B, L, D) : 0; }
  Tensor workspace(const Tensor& x, long long n) const { return n ? fresh(x, {n}, at::kByte) : Tensor(); }
};

Tensor gated_run(const Tensor& a, const Tensor& x, const Tensor& h0, Tensor* last, Tensor* states) {
  at::AutoDispatchBelowADInplaceOrView plain;
  const Launch on(x);
  const Shape s(x, 1, "gated_scan");
  const Operand oa(a), ox(x);
  const Tensor start = whole(h0);
  Tensor h = fresh(x);
  if (last) *last = s.row(x);
  if (states) *states = s.states(x);
  const long long n = s.bytes();
  const Tensor ws = s.workspace(x, n);
  check(api.gfn_gated_scan_forward(oa.p, oa.sb, oa.st, ox.p, ox.sb, ox.st, fptr(start), code_of(x), s.B, s.L, s.D,
                                   h.data_ptr(), last ? fptr(*last) : nullptr, states ? fptr(*states) : nullptr,
                                   ptr(ws), n, on.stream),
        "gfn_gated_scan_forward");
  return h;
}

struct GatedNode : torch::autograd::Function<GatedNode> {
  static variable_list forward(AutogradContext* ctx, const Maybe& gate, const Tensor& x, const Maybe& start,
                               bool want_last) {
    const Tensor a = gate.value_or(Tensor()), h0 = start.value_or(Tensor());
    Tensor last, states;
    Tensor h = gated_run(a, x, h0, want_last ? &last : nullptr, &states);
    ctx->save_for_backward({a, x, states});
    ctx->saved_data["h0"] = h0.defined();
    ctx->set_materialize_grads(false);
    return want_last ? variable_list{h, last} : variable_list{h};
  }

  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    return backward_body([&] { return gradients(ctx, grads); });
  }

  static variable_list gradients(AutogradContext* ctx, const variable_list& grads) {
    const bool recording = at::GradMode::is_enabled();
    const Tensor dlast = grads.size() > 1 ? grads[1] : Tensor();
    if (!grads[0].defined() && !dlast.defined()) return variable_list(4);
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &a = saved[0], &x = saved[1], &states = saved[2];
    Tensor da, dx, dh0;
    {
      at::AutoDispatchBelowADInplaceOrView plain;
      const Launch on(x);
      const Shape s(x, 1, "gated_scan");
      const Operand oa(a), ox(x), og(grads[0]);
      const Tensor gl = whole(dlast);
      const size_t at = a.defined();  // inputs are numbered without the absent ones
      if (at && ctx->needs_input_grad(0)) da = fresh(x);
      if (ctx->needs_input_grad(at)) dx = fresh(x);
      if (ctx->saved_data["h0"].toBool() && ctx->needs_input_grad(at + 1)) dh0 = s.row(x);
      const long long n = s.bytes();
      const Tensor ws = s.workspace(x, n);
      check(api.gfn_gated_scan_backward(oa.p, oa.sb, oa.st, ox.p, ox.sb, ox.st, fptr(states), og.p, og.sb, og.st,
                                        fptr(gl), code_of(x), s.B, s.L, s.D, ptr(da), ptr(dx), fptr(dh0), ptr(ws), n,
                                        on.stream),
            "gfn_gated_scan_backward");
    }
    return first_order({da, dx, dh0, Tensor()}, grads, recording);
  }
};

// (x_seq, v_seq) and, where asked for, (v_last, x_last)
variable_list layer_run(const Tensor& z, const Tensor& v0, const Tensor& x0, int64_t heads, double base_dt,
                        bool want_last, Tensor* states) {
  at::AutoDispatchBelowADInplaceOrView plain;
  const Launch on(z);
  const Shape s(z, 3, "parallel_layer_scan");
  const Tensor zc = whole(z), v = whole(v0), x = whole(x0);
  Tensor xs = fresh(z, {s.B, s.L, s.D}, at::kFloat), vs = fresh(xs), vl, xl;
  if (want_last) {
    vl = s.row(z);
    xl = s.row(z);
  }
  if (states) *states = s.states(z);
  const long long n = s.bytes();
  const Tensor ws = s.workspace(z, n);
  check(api.gfn_layer_scan_forward(fptr(zc), fptr(v), fptr(x), s.B, s.L, s.D, extent(heads, "parallel_layer_scan"),
                                   (float)base_dt, fptr(xs), fptr(vs), fptr(xl), fptr(vl),
                                   states ? fptr(*states) : nullptr, ptr(ws), n, on.stream),
        "gfn_layer_scan_forward");
  return want_last ? variable_list{xs, vs, vl, xl} : variable_list{xs, vs};
}

struct LayerNode : torch::autograd::Function<LayerNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& z, const Maybe& v, const Maybe& x, int64_t heads,
                               double base_dt, bool want_last) {
    const Tensor v0 = v.value_or(Tensor()), x0 = x.value_or(Tensor());
    Tensor states;
    variable_list out = layer_run(z, v0, x0, heads, base_dt, want_last, &states);
    ctx->save_for_backward({z, states});
    ctx->saved_data["heads"] = heads;
    ctx->saved_data["base_dt"] = base_dt;
    ctx->saved_data["v0"] = v0.defined();
    ctx->saved_data["x0"] = x0.defined();
    ctx->set_materialize_grads(false);
    return out;
  }

  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    return backward_body([&] { return gradients(ctx, grads); });
  }

  static variable_list gradients(AutogradContext* ctx, const variable_list& grads) {
    const bool recording = at::GradMode::is_enabled();
    Tensor g[4];  // of x_seq, v_seq, v_last, x_last
    bool any = false;
    for (size_t i = 0; i < grads.size(); ++i) any = any || grads[i].defined();
    if (!any) return variable_list(6);
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &z = saved[0], &states = saved[1];
    Tensor dz, dv0, dx0;
    {
      at::AutoDispatchBelowADInplaceOrView plain;
      const Launch on(z);
      const Shape s(z, 3, "parallel_layer_scan");
      for (size_t i = 0; i < grads.size(); ++i) g[i] = whole(grads[i]);
      const Tensor zc = whole(z);
      dz = fresh(z);
      const bool has_v = ctx->saved_data["v0"].toBool(), has_x = ctx->saved_data["x0"].toBool();
      if (has_v && ctx->needs_input_grad(1)) dv0 = s.row(z);
      if (has_x && ctx->needs_input_grad(has_v ? 2 : 1)) dx0 = s.row(z);  // numbered without the absent ones
      const long long n = s.bytes();
      const Tensor ws = s.workspace(z, n);
      check(api.gfn_layer_scan_backward(fptr(zc), fptr(states), fptr(g[0]), fptr(g[1]), fptr(g[3]), fptr(g[2]), s.B,
                                        s.L, s.D, (int)ctx->saved_data["heads"].toInt(),
                                        (float)ctx->saved_data["base_dt"].toDouble(), fptr(dz), fptr(dx0), fptr(dv0),
                                        ptr(ws), n, on.stream),
            "gfn_layer_scan_backward");
    }
    return first_order({dz, dv0, dx0, Tensor(), Tensor(), Tensor()}, grads, recording);
  }
};

// ------------------------------------------------------------------- Python
struct Unlocked {  // other Python threads run meanwhile
  PyThreadState* state = PyEval_SaveThread();
  ~Unlocked() { PyEval_RestoreThread(state); }
};

// An operand.  There is no forward mode: a tensor that carries a tangent is
// refused, since the result would come back without one.
Tensor tensor_arg(PyObject* o) {
  if (o == Py_None) return Tensor();
  if (!THPVariable_Check(o)) throw Failure("a tensor or None expected");
  const Tensor& t = THPVariable_Unpack(o);
  if (t._fw_grad(0).defined()) throw Failure("forward-mode differentiation is not implemented for this operator");
  return t;
}
double number_arg(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return v;
}
long long integer_arg(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}
bool flag_arg(PyObject* o) { return PyObject_IsTrue(o) == 1; }

PyObject* tuple_of(const variable_list& ts) {
  PyObject* r = PyTuple_New((Py_ssize_t)ts.size());
  if (!r) throw python_error();
  for (size_t i = 0; i < ts.size(); ++i) PyTuple_SET_ITEM(r, (Py_ssize_t)i, THPVariable_Wrap(ts[i]));
  return r;
}

// Runs `f` with the exceptions of C++ turned into Python's; the library's
// failures become GfnError.
template <class F>
PyObject* guarded(Py_ssize_t given, Py_ssize_t expected, F f) {
  HANDLE_TH_ERRORS
  if (given != expected || !gfn_error) {
    PyErr_SetString(PyExc_TypeError, "wrong number of arguments, or bind() was not called");
    return nullptr;
  }
  try {
    return f();
  } catch (const Failure& e) {
    PyErr_SetString(gfn_error, e.what());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// layer_norm(x, weight, bias, eps, train) -> y
PyObject* py_layer_norm(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded(n, 5, [&] {
    const Tensor x = tensor_arg(v[0]), w = tensor_arg(v[1]), b = tensor_arg(v[2]);
    const double eps = number_arg(v[3]);
    const bool train = flag_arg(v[4]);
    Tensor y;
    {
      Unlocked u;
      y = train ? NormNode::apply(x, maybe(w), maybe(b), eps) : norm_run(x, w, b, eps, nullptr);
    }
    return THPVariable_Wrap(y);
  });
}

// gated_scan(a, x, h0, want_last, train) -> (h,) or (h, last)
PyObject* py_gated_scan(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded(n, 5, [&] {
    const Tensor a = tensor_arg(v[0]), x = tensor_arg(v[1]), h0 = tensor_arg(v[2]);
    const bool want_last = flag_arg(v[3]), train = flag_arg(v[4]);
    variable_list out;
    {
      Unlocked u;
      if (train) out = GatedNode::apply(maybe(a), x, maybe(h0), want_last);
      else {
        Tensor last, h = gated_run(a, x, h0, want_last ? &last : nullptr, nullptr);
        out = want_last ? variable_list{h, last} : variable_list{h};
      }
    }
    return tuple_of(out);
  });
}

// layer_scan(z, v0, x0, heads, base_dt, want_last, train) -> (x_seq, v_seq) or (x_seq, v_seq, v_last, x_last)
PyObject* py_layer_scan(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded(n, 7, [&] {
    const Tensor z = tensor_arg(v[0]), v0 = tensor_arg(v[1]), x0 = tensor_arg(v[2]);
    const int64_t heads = integer_arg(v[3]);
    const double base_dt = number_arg(v[4]);
    const bool want_last = flag_arg(v[5]), train = flag_arg(v[6]);
    variable_list out;
    {
      Unlocked u;
      out = train ? LayerNode::apply(z, maybe(v0), maybe(x0), heads, base_dt, want_last)
                  : layer_run(z, v0, x0, heads, base_dt, want_last, nullptr);
    }
    return tuple_of(out);
  });
}

// process_logits(x, tokens, tokens_stride, lengths, prompt_lengths, 4 numbers, 4 tensors or None for them,
//                bias, bias_stride, allowed, allowed_stride) -> out
PyObject* py_process_logits(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded(n, 17, [&] {
    const Tensor x = tensor_arg(v[0]), tokens = tensor_arg(v[1]), lengths = tensor_arg(v[3]), prompts = tensor_arg(v[4]);
    const long long ts = integer_arg(v[2]), bs = integer_arg(v[14]), ms = integer_arg(v[16]);
    float num[4];
    Tensor per_row[4];
    for (int i = 0; i < 4; ++i) {
      num[i] = (float)number_arg(v[5 + i]);
      per_row[i] = tensor_arg(v[9 + i]);
    }
    const Tensor bias = tensor_arg(v[13]), allowed = tensor_arg(v[15]);
    Tensor out;
    {
      Unlocked u;
      at::AutoDispatchBelowADInplaceOrView plain;
      const Launch on(x);
      const int B = extent(x.size(0), "process_logits"), V = extent(x.size(1), "process_logits");
      const int T = tokens.defined() ? extent(tokens.size(1), "process_logits") : 0;
      auto longs = [](const Tensor& t) { return static_cast<const long long*>(ptr(t)); };
      out = fresh(x);
      check(api.gfn_process_logits(x.data_ptr(), B > 1 ? x.stride(0) : V, code_of(x), B, V, longs(tokens), ts, T,
                                   longs(lengths), longs(prompts), num[0], fptr(per_row[0]), num[1], fptr(per_row[1]),
                                   num[2], fptr(per_row[2]), num[3], fptr(per_row[3]), fptr(bias), bs, ptr(allowed),
                                   ms, out.data_ptr(), on.stream),
            "gfn_process_logits");
    }
    return THPVariable_Wrap(out);
  });
}

// bind(addresses, error): the entry points of GFN_ENTRIES and the class of the library's errors
PyObject* py_bind(PyObject*, PyObject* const* v, Py_ssize_t n) {
  constexpr Py_ssize_t COUNT = sizeof(Api) / sizeof(void*);
  if (n != 2 || !PyTuple_Check(v[0]) || PyTuple_GET_SIZE(v[0]) != COUNT) {
    PyErr_SetString(PyExc_TypeError, "bind(addresses, error)");
    return nullptr;
  }
  Api a = {};
  Py_ssize_t i = 0;
#define X(name)                                                                      \
  a.name = reinterpret_cast<decltype(a.name)>(PyLong_AsVoidPtr(PyTuple_GET_ITEM(v[0], i++))); \
  if (!a.name) {                                                                     \
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, #name " is missing");   \
    return nullptr;                                                                  \
  }
  GFN_ENTRIES(X)
#undef X
  api = a;
  Py_INCREF(v[1]);
  gfn_error = v[1];
  Py_RETURN_NONE;
}

#define METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_##name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(bind),       METHOD(layer_norm),     METHOD(gated_scan),
                         METHOD(layer_scan), METHOD(process_logits), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_torch_ops", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__torch_ops() { return PyModule_Create(&module_def); }
