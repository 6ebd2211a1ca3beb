// Autograd nodes of the norm, the router and the head loss: the Python module
// lowbit._autograd.
//
// These operators are short: at ordinary sizes a training step's kernels take
// less time than a Python forward and backward around them (the backward runs on
// the engine's thread, where Python first has to be entered).  So their nodes are
// C++.  The kernels stay behind the C-ABI of include/ntlowbit.h: bind() is
// handed the addresses of its functions in the library that lowbit._lib has
// loaded, so this module links to no kernel and there is one library at a time.
// Arguments are checked in Python, where an operator is called.
#include <ATen/ATen.h>
#include <ATen/hip/EmptyTensor.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/utils/object_ptr.h>

#include <algorithm>
#include <memory>
#include <mutex>
#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include "../../../include/ntlowbit.h"

namespace {

using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

struct Abi {
  decltype(&ntlb_last_error) last_error;
  decltype(&ntlb_layer_norm_forward) norm_forward;
  decltype(&ntlb_layer_norm_backward) norm_backward;
  decltype(&ntlb_layer_norm_workspace_bytes) norm_workspace;
  decltype(&ntlb_route_topk) route;
  decltype(&ntlb_route_topk_backward) route_backward;
  decltype(&ntlb_pad_rows) pad_rows;
  decltype(&ntlb_linear_xent_forward) xent_forward;
  decltype(&ntlb_linear_xent_backward) xent_backward;
  decltype(&ntlb_linear_xent_state_bytes) xent_state;
  decltype(&ntlb_linear_xent_workspace_bytes) xent_workspace;
  PyObject* error;  // the package's exception for a failed entry point
} abi = {};

void check(const char* fn, int rc) {
  if (rc == NTLB_OK) return;
  const std::string msg = std::string(fn) + " failed (" + std::to_string(rc) + "): " + abi.last_error();
  if (rc == NTLB_EINVAL) C10_THROW_ERROR(ValueError, msg);
  const PyGILState_STATE gil = PyGILState_Ensure();
  PyErr_SetString(abi.error, msg.c_str());
  python_error err;
  err.persist();
  PyGILState_Release(gil);
  throw err;
}

int dtype_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return NTLB_F32;
    case at::kBFloat16: return NTLB_BF16;
    case at::kHalf: return NTLB_F16;
    default: C10_THROW_ERROR(TypeError, "expected float32, bfloat16 or float16");
  }
}

void* stream_of(const Tensor& t) {
  return (void*)c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream();
}

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// memory of like's device, past the dispatcher
Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) {
  return Tensor(at::detail::empty_cuda(sizes, type, like.device(), std::nullopt));
}
Tensor scratch(int64_t bytes, const Tensor& like) { return fresh({bytes}, at::kByte, like); }

// t as [rows, columns] with unit stride along the columns and rows one behind the
// other (or one row repeated): a copy only where no view gives that.  Of a single
// row torch's own strides may be anything, contiguous() or not.
Tensor rows_of(const Tensor& t) {
  Tensor r = t.dim() == 2 ? t : t.reshape({t.numel() / t.size(-1), t.size(-1)});
  const int64_t n = r.size(1);
  if (r.stride(1) != 1 || (r.stride(0) != 0 && r.stride(0) < n)) r = r.contiguous();
  if (r.size(0) == 1 && r.stride(0) < n) r = r.as_strided({1, n}, {n, 1});
  return r;
}
Tensor shaped(const Tensor& t, at::IntArrayRef sizes) { return t.sizes() == sizes ? t : t.reshape(sizes); }

bool wanted(const Tensor& t) { return t.defined() && t.requires_grad(); }

// No tangents are formed.  One that comes with an argument would be dropped without
// a word: the result would count as constant along it.
template <typename... Ts>
void no_tangent(const char* fn, const Ts&... ts) {
  if (((ts.defined() && ts._fw_grad(/*level=*/0).defined()) || ...))
    C10_THROW_ERROR(NotImplementedError, std::string(fn) + " has no derivative in forward mode");
}

// The gradients are no functions of the graph: where one is being recorded, they
// carry an error for whoever differentiates them
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  for (Tensor& g : grads) {
    if (!g.defined()) continue;
    torch::autograd::DelayedError err("the gradients of this operator cannot be differentiated again", 1);
    g = err({g.detach().set_requires_grad(true)})[0];
  }
  return grads;
}

// A tensor kept for the backward.  The kernels get its address, and saved-tensor
// hooks may hand back anything: its place, type and sizes are looked at when it
// comes back.  Its layout may be another.
class Kept {
 public:
  Kept() = default;
  explicit Kept(const Tensor& t) : v_(t, false) {
    if (!t.defined()) return;
    type_ = t.scalar_type();
    device_ = t.device();
    sizes_ = t.sizes();
  }
  Tensor unpack(const char* what) const {
    const Tensor t = v_.unpack();
    if (device_.is_cpu()) return t;  // undefined when it was kept
    if (!t.defined() || t.device() != device_ || t.scalar_type() != type_ || t.sizes() != at::IntArrayRef(sizes_) ||
        (t.numel() > 0 && !t.data_ptr()))
      C10_THROW_ERROR(Error, std::string("the ") + what + " kept for the backward did not come back as they were: " +
                                 (t.defined() ? t.toString() + c10::str(t.sizes(), " on ", t.device()) : "nothing") +
                                 ", not " + c10::toString(type_) + c10::str(at::IntArrayRef(sizes_), " on ", device_));
    return t;
  }
  void reset() { v_.reset_data(); }

 private:
  SavedVariable v_;
  at::ScalarType type_ = at::kFloat;
  at::Device device_ = at::kCPU;
  at::DimVector sizes_;
};

// What the backward is to read of t: t itself, whose changes in place are then
// noticed, where `used` (its rows) is a view of it, else the copy
Kept kept(const Tensor& t, const Tensor& used) { return Kept(used.is_alias_of(t) ? t : used); }
Tensor dense(const Tensor& t) { return t.defined() ? t.contiguous() : t; }

// The nodes are torch's own kind, not its custom functions, whose context of named
// values and wrapping of results take 3 us more of a router step's 51
template <typename N>
std::shared_ptr<N> make_node(torch::autograd::edge_list edges) {
  std::shared_ptr<N> node(new N(), torch::autograd::deleteNode);
  node->set_next_edges(std::move(edges));
  return node;
}

// ---------------------------------------------------------------------------
struct LayerNorm {
  static int weight_dtype(const Tensor& x, const Tensor& w, const Tensor& b) {
    return dtype_of(w.defined() ? w : b.defined() ? b : x);
  }

  // mr: the rows' means, then 1 / their deviations (undefined: not kept)
  static Tensor run(const Tensor& x2, const Tensor& w, const Tensor& b, double eps, const Tensor& mr) {
    const int64_t T = x2.size(0), H = x2.size(1);
    Tensor y = fresh({T, H}, x2.scalar_type(), x2);
    float* m = mr.defined() ? mr.data_ptr<float>() : nullptr;
    check("ntlb_layer_norm_forward",
          abi.norm_forward(x2.data_ptr(), dtype_of(x2), T, H, x2.stride(0), ptr(w), ptr(b), weight_dtype(x2, w, b),
                           (float)eps, y.data_ptr(), H, m, m ? m + T : nullptr, stream_of(x2)));
    return y;
  }

  struct Backward : Node {
    Kept x, w, b, mr;
    at::DimVector sizes;  // of x, which may be kept as a copy of its rows

    variable_list apply(variable_list&& grads) override {
      const std::lock_guard<std::mutex> lock(mutex_);
      if (!grads[0].defined()) return variable_list(3);
      no_tangent("the gradient of layer_norm", grads[0]);
      const Tensor xt = x.unpack("rows of x"), w0 = w.unpack("values of weight"), b0 = b.unpack("values of bias"),
                   r0 = mr.unpack("rows' means and deviations");
      const c10::DeviceGuard guard(xt.device());
      const at::AutoDispatchBelowADInplaceOrView below;
      const Tensor x2 = rows_of(xt), d2 = rows_of(grads[0]), wt = dense(w0), bt = dense(b0);
      const int64_t T = x2.size(0), H = x2.size(1);
      Tensor dx, dw, db, ws;
      if (task_should_compute_output(0)) dx = fresh({T, H}, x2.scalar_type(), x2);
      if (wt.defined() && task_should_compute_output(1)) dw = fresh({H}, wt.scalar_type(), x2);
      if (bt.defined() && task_should_compute_output(2)) db = fresh({H}, bt.scalar_type(), x2);
      int64_t need = 0;
      if (dw.defined() || db.defined()) {
        need = abi.norm_workspace(dtype_of(x2), T, H);
        ws = scratch(need, x2);
      }
      const Tensor stats = dense(r0);
      const float* m = stats.data_ptr<float>();
      check("ntlb_layer_norm_backward",
            abi.norm_backward(x2.data_ptr(), dtype_of(x2), T, H, x2.stride(0), d2.data_ptr(), d2.stride(0), m, m + T,
                              ptr(wt), weight_dtype(x2, wt, bt), ptr(dx), H, ptr(dw), ptr(db), ptr(ws), need,
                              stream_of(x2)));
      if (dx.defined()) dx = shaped(dx, sizes);
      return once({dx, dw, db});
    }
    void release_variables() override {
      const std::lock_guard<std::mutex> lock(mutex_);
      x.reset();
      w.reset();
      b.reset();
      mr.reset();
    }
    std::string name() const override { return "LayerNormBackward"; }
  };

  static Tensor forward(const Tensor& x, const Tensor& w, const Tensor& b, double eps) {
    const c10::DeviceGuard guard(x.device());
    Tensor y, x2, mr;
    {
      const at::AutoDispatchBelowADInplaceOrView below;
      x2 = rows_of(x);
      mr = fresh({std::max<int64_t>(1, 2 * x2.size(0))}, at::kFloat, x2);
      y = shaped(run(x2, w, b, eps, mr), x.sizes());
    }
    auto node = make_node<Backward>(torch::autograd::collect_next_edges(x, w, b));
    node->x = kept(x, x2);
    node->w = Kept(w);
    node->b = Kept(b);
    node->mr = Kept(mr);
    node->sizes = x.sizes();
    torch::autograd::set_history(y, node);
    return y;
  }
};

// ---------------------------------------------------------------------------
struct RouteConfig {
  int64_t k, sigmoid, groups, kept, renorm;
  double scale;
};

struct Route {
  static std::tuple<Tensor, Tensor> run(const Tensor& z, const Tensor& bias, const RouteConfig& c) {
    const int64_t T = z.size(0);
    Tensor ids = fresh({T, c.k}, at::kInt, z);
    Tensor w = fresh({T, c.k}, at::kFloat, z);
    check("ntlb_route_topk",
          abi.route(z.data_ptr(), dtype_of(z), T, z.size(1), z.stride(0), c.k, (int)c.sigmoid, (const float*)ptr(bias),
                    c.groups, c.kept, (int)c.renorm, (float)c.scale, ids.data_ptr<int32_t>(), w.data_ptr<float>(),
                    stream_of(z)));
    return {ids, w};
  }
  // the results in the logits' leading shape
  static std::tuple<Tensor, Tensor> lead(const Tensor& logits, const std::tuple<Tensor, Tensor>& r, int64_t k) {
    if (logits.dim() == 2) return r;
    std::vector<int64_t> sizes = logits.sizes().vec();
    sizes.back() = k;
    return {shaped(std::get<0>(r), sizes), shaped(std::get<1>(r), sizes)};
  }

  struct Backward : Node {
    Kept z, ids;
    RouteConfig c;
    at::DimVector sizes;  // of the logits, which may be kept as a copy of their rows

    variable_list apply(variable_list&& grads) override {
      const std::lock_guard<std::mutex> lock(mutex_);
      if (!grads[0].defined()) return variable_list(1);
      no_tangent("the gradient of route_tokens", grads[0]);
      const Tensor zt = z.unpack("logits"), i0 = ids.unpack("expert ids");
      const c10::DeviceGuard guard(zt.device());
      const at::AutoDispatchBelowADInplaceOrView below;
      const Tensor z2 = rows_of(zt), it = dense(i0), dw = grads[0].contiguous();
      const int64_t T = z2.size(0), E = z2.size(1);
      Tensor dz = fresh({T, E}, z2.scalar_type(), z2);
      check("ntlb_route_topk_backward",
            abi.route_backward(z2.data_ptr(), dtype_of(z2), T, E, z2.stride(0), c.k, (int)c.sigmoid, (int)c.renorm,
                               (float)c.scale, it.data_ptr<int32_t>(), dw.data_ptr<float>(), dz.data_ptr(), E,
                               stream_of(z2)));
      return once({shaped(dz, sizes)});
    }
    void release_variables() override {
      const std::lock_guard<std::mutex> lock(mutex_);
      z.reset();
      ids.reset();
    }
    std::string name() const override { return "RouteBackward"; }
  };

  static std::tuple<Tensor, Tensor> forward(const Tensor& logits, const Tensor& bias, const RouteConfig& c) {
    const c10::DeviceGuard guard(logits.device());
    Tensor z, ids, w;
    {
      const at::AutoDispatchBelowADInplaceOrView below;
      z = rows_of(logits);
      std::tie(ids, w) = lead(logits, run(z, bias, c), c.k);
    }
    auto node = make_node<Backward>(torch::autograd::collect_next_edges(logits));
    node->z = kept(logits, z);
    node->ids = Kept(ids);
    node->c = c;
    node->sizes = logits.sizes();
    torch::autograd::set_history(w, node);
    return {ids, w};
  }
};

// ---------------------------------------------------------------------------
struct LinearXent {
  static constexpr int64_t MAX_PITCH = 1 << 22;  // of the products' copies
  // whether weight lies in rows of whole 16-byte pieces, as the products take them
  static bool fits(const Tensor& weight) {
    return weight.stride(1) == 1 && weight.stride(0) % 8 == 0 && weight.size(1) % 8 == 0 &&
           weight.stride(0) >= weight.size(1) && weight.stride(0) <= MAX_PITCH && (uintptr_t)weight.data_ptr() % 16 == 0;
  }
  // weight in such rows: a copy where they are not
  static Tensor padded(const Tensor& weight) {
    if (fits(weight)) return weight;
    const c10::DeviceGuard guard(weight.device());
    const at::AutoDispatchBelowADInplaceOrView below;
    const Tensor w = rows_of(weight);
    Tensor out = fresh({w.size(0), (w.size(1) + 7) / 8 * 8}, w.scalar_type(), w);
    check("ntlb_pad_rows", abi.pad_rows((const uint16_t*)w.data_ptr(), w.stride(0), w.size(0), w.size(1),
                                        (uint16_t*)out.data_ptr(), out.size(1), stream_of(w)));
    return out;
  }

  // w: weight in 16-byte rows; reduction 0 none, 1 sum, 2 mean
  static std::tuple<Tensor, Tensor> run(const Tensor& x2, const Tensor& w, const Tensor& targets, int64_t ignore,
                                        int64_t reduction) {
    const int64_t T = x2.size(0), H = x2.size(1), V = w.size(0);
    const Tensor y = targets.reshape({T}).contiguous();
    const Tensor state = scratch(abi.xent_state(T, H), x2);
    const int64_t need = abi.xent_workspace(T, H, V, 0);
    const Tensor ws = scratch(std::max<int64_t>(need, 16), x2);
    Tensor loss = fresh({reduction ? 1 : std::max<int64_t>(T, 1)}, at::kFloat, x2);
    check("ntlb_linear_xent_forward",
          abi.xent_forward((const uint16_t*)x2.data_ptr(), x2.stride(0), (const uint16_t*)w.data_ptr(), w.stride(0),
                           y.data_ptr(), y.scalar_type() == at::kLong, T, H, V, ignore, (int)reduction,
                           loss.data_ptr<float>(), state.data_ptr(), ws.data_ptr(), need, stream_of(x2)));
    return {reduction ? loss.reshape({}) : shaped(T ? loss : loss.slice(0, 0, 0), targets.sizes()), state};
  }

  // the forward's state as the backward takes it
  static Tensor aligned(const Tensor& state) {
    const Tensor s = dense(state);
    return (uintptr_t)s.data_ptr() % 256 == 0 ? s : s.clone();
  }

  struct Backward : Node {
    Kept w, state;
    at::DimVector sizes;  // of hidden
    int64_t T, reduction;

    variable_list apply(variable_list&& grads) override {
      const std::lock_guard<std::mutex> lock(mutex_);
      if (!grads[0].defined()) return variable_list(2);
      no_tangent("the gradient of linear_cross_entropy", grads[0]);
      const Tensor w0 = w.unpack("rows of weight"), s0 = state.unpack("live rows of hidden");
      const c10::DeviceGuard guard(w0.device());
      const at::AutoDispatchBelowADInplaceOrView below;
      const Tensor wt = padded(w0), st = aligned(s0);
      const int64_t H = sizes.back(), V = wt.size(0);
      const Tensor dl = grads[0].reshape({-1}).contiguous();
      Tensor dx, dw;
      if (task_should_compute_output(0)) dx = fresh({T, H}, wt.scalar_type(), wt);
      if (task_should_compute_output(1)) dw = fresh({V, H}, wt.scalar_type(), wt);
      const int64_t need = abi.xent_workspace(T, H, V, 1);
      const Tensor ws = scratch(need, wt);
      check("ntlb_linear_xent_backward",
            abi.xent_backward(st.data_ptr(), (const uint16_t*)wt.data_ptr(), wt.stride(0), T, H, V, (int)reduction,
                              dl.data_ptr<float>(), (uint16_t*)ptr(dx), H, (uint16_t*)ptr(dw), H, ws.data_ptr(), need,
                              stream_of(wt)));
      if (dx.defined()) dx = shaped(dx, sizes);
      return once({dx, dw});
    }
    void release_variables() override {
      const std::lock_guard<std::mutex> lock(mutex_);
      w.reset();
      state.reset();
    }
    std::string name() const override { return "LinearXentBackward"; }
  };

  static Tensor forward(const Tensor& hidden, const Tensor& weight, const Tensor& w, const Tensor& targets,
                        int64_t ignore, int64_t reduction) {
    const c10::DeviceGuard guard(hidden.device());
    Tensor loss, state;
    {
      const at::AutoDispatchBelowADInplaceOrView below;
      std::tie(loss, state) = run(rows_of(hidden), w, targets, ignore, reduction);
    }
    auto node = make_node<Backward>(torch::autograd::collect_next_edges(hidden, weight));
    node->w = Kept(w);
    node->state = Kept(state);
    node->sizes = hidden.sizes();
    node->T = hidden.numel() / hidden.size(-1);
    node->reduction = reduction;
    torch::autograd::set_history(loss, node);
    return loss;
  }
};

// ---------------------------------------------------------------------------
// Python
// ---------------------------------------------------------------------------
Tensor maybe(PyObject* o) { return o == Py_None ? Tensor() : THPVariable_Unpack(o); }

void count(Py_ssize_t n, Py_ssize_t want) {
  if (n != want) C10_THROW_ERROR(TypeError, "wrong number of arguments");
}
int64_t integer(PyObject* o) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}
double real(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return v;
}
struct NoGil {  // kernels are launched without the interpreter's lock
  PyThreadState* save = PyEval_SaveThread();
  ~NoGil() { PyEval_RestoreThread(save); }
};

// layer_norm(x, weight | None, bias | None, eps)
PyObject* py_layer_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 4);
  const Tensor& x = THPVariable_Unpack(a[0]);
  const Tensor w = maybe(a[1]), b = maybe(a[2]);
  const double eps = real(a[3]);
  Tensor y;
  {
    const NoGil nogil;
    no_tangent("layer_norm", x, w, b);
    if (at::GradMode::is_enabled() && (wanted(x) || wanted(w) || wanted(b))) {
      y = LayerNorm::forward(x, w, b, eps);
    } else {
      const at::AutoDispatchBelowADInplaceOrView below;
      const c10::DeviceGuard guard(x.device());
      y = shaped(LayerNorm::run(rows_of(x), w, b, eps, Tensor()), x.sizes());
    }
  }
  return THPVariable_Wrap(y);
  END_HANDLE_TH_ERRORS
}

// route(logits, bias | None, k, sigmoid, groups, kept, renorm, scale) -> (ids, weights)
PyObject* py_route(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 8);
  const Tensor& z = THPVariable_Unpack(a[0]);
  const Tensor bias = maybe(a[1]);
  const RouteConfig c{integer(a[2]), integer(a[3]), integer(a[4]), integer(a[5]), integer(a[6]), real(a[7])};
  std::tuple<Tensor, Tensor> r;
  {
    const NoGil nogil;
    no_tangent("route_tokens", z);
    if (at::GradMode::is_enabled() && wanted(z)) {
      r = Route::forward(z, bias, c);
    } else {
      const at::AutoDispatchBelowADInplaceOrView below;
      const c10::DeviceGuard guard(z.device());
      r = Route::lead(z, Route::run(rows_of(z), bias, c), c.k);
    }
  }
  THPObjectPtr ids(THPVariable_Wrap(std::get<0>(r))), w(THPVariable_Wrap(std::get<1>(r)));
  if (!ids || !w) throw python_error();
  return PyTuple_Pack(2, ids.get(), w.get());
  END_HANDLE_TH_ERRORS
}

// linear_xent(hidden, weight, targets, ignore_index, reduction)
PyObject* py_linear_xent(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 5);
  const Tensor &x = THPVariable_Unpack(a[0]), &weight = THPVariable_Unpack(a[1]), &y = THPVariable_Unpack(a[2]);
  const int64_t ignore = integer(a[3]), reduction = integer(a[4]);
  Tensor loss;
  {
    const NoGil nogil;
    no_tangent("linear_cross_entropy", x, weight);
    const Tensor w = LinearXent::padded(weight);
    if (at::GradMode::is_enabled() && (wanted(x) || wanted(weight))) {
      loss = LinearXent::forward(x, weight, w, y, ignore, reduction);
    } else {
      const at::AutoDispatchBelowADInplaceOrView below;
      const c10::DeviceGuard guard(x.device());
      loss = std::get<0>(LinearXent::run(rows_of(x), w, y, ignore, reduction));
    }
  }
  return THPVariable_Wrap(loss);
  END_HANDLE_TH_ERRORS
}

// bind({name: address, "error": class}): the C-ABI's functions, and what is raised
// where one of them fails for other reasons than its arguments
template <typename F>
void take(PyObject* table, const char* name, F& f) {
  PyObject* v = PyDict_GetItemString(table, name);  // borrowed
  if (!v) C10_THROW_ERROR(ValueError, std::string("no address of ") + name);
  f = reinterpret_cast<F>((uintptr_t)PyLong_AsUnsignedLongLong(v));
  if (PyErr_Occurred()) throw python_error();
}
PyObject* py_bind(PyObject*, PyObject* table) {
  HANDLE_TH_ERRORS
  if (!PyDict_Check(table)) C10_THROW_ERROR(TypeError, "bind takes a dict of addresses");
  Abi a{};
  take(table, "ntlb_last_error", a.last_error);
  take(table, "ntlb_layer_norm_forward", a.norm_forward);
  take(table, "ntlb_layer_norm_backward", a.norm_backward);
  take(table, "ntlb_layer_norm_workspace_bytes", a.norm_workspace);
  take(table, "ntlb_route_topk", a.route);
  take(table, "ntlb_route_topk_backward", a.route_backward);
  take(table, "ntlb_pad_rows", a.pad_rows);
  take(table, "ntlb_linear_xent_forward", a.xent_forward);
  take(table, "ntlb_linear_xent_backward", a.xent_backward);
  take(table, "ntlb_linear_xent_state_bytes", a.xent_state);
  take(table, "ntlb_linear_xent_workspace_bytes", a.xent_workspace);
  PyObject* error = PyDict_GetItemString(table, "error");  // borrowed
  if (!error || !PyExceptionClass_Check(error)) C10_THROW_ERROR(ValueError, "no class of error");
  a.error = Py_NewRef(error);  // for the process's life
  abi = a;
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"bind", py_bind, METH_O, nullptr},
    {"layer_norm", (PyCFunction)(void (*)(void))py_layer_norm, METH_FASTCALL, nullptr},
    {"route", (PyCFunction)(void (*)(void))py_route, METH_FASTCALL, nullptr},
    {"linear_xent", (PyCFunction)(void (*)(void))py_linear_xent, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_autograd", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__autograd(void) { return PyModule_Create(&module); }
