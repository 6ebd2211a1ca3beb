// Autograd nodes of the norms, the router, the head loss and the experts: the Python module
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
  decltype(&ntlb_rms_norm_forward) rms_forward;
  decltype(&ntlb_rms_norm_quant) rms_quant;
  decltype(&ntlb_rms_norm_backward) rms_backward;
  decltype(&ntlb_rms_norm_workspace_bytes) rms_workspace;
  decltype(&ntlb_swiglu_rows) swiglu;
  decltype(&ntlb_swiglu_rows_backward) swiglu_backward;
  decltype(&ntlb_grouped_matmul) grouped;
  decltype(&ntlb_grouped_matmul_dx) grouped_dx;
  decltype(&ntlb_grouped_matmul_dw) grouped_dw;
  decltype(&ntlb_grouped_matmul_workspace_bytes) grouped_workspace;
  decltype(&ntlb_kept_rows) kept_rows;
  decltype(&ntlb_kept_values) kept_values;
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
  // output: t is a result of the node that keeps it, and set_history has been called
  explicit Kept(const Tensor& t, bool output = false) : v_(t, output) {
    if (!t.defined()) return;
    type_ = t.scalar_type();
    device_ = t.device();
    sizes_ = t.sizes();
  }
  Tensor unpack(const char* what, std::shared_ptr<Node> node = nullptr) const {
    const Tensor t = v_.unpack(std::move(node));
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
// What an operator keeps of its input in 8 bits: codes and their tiles' exponents
struct Held {
  Tensor codes, exps;
  // of T rows of `parts` parts of n columns each
  static Held of(int64_t T, int64_t parts, int64_t n, const Tensor& like) {
    const int64_t tiles = (n + 127) / 128;
    // an empty batch keeps one row that nothing writes, so that there is an address
    const int64_t rows = std::max<int64_t>(T, 1) * parts;
    return {fresh({rows, tiles * 128}, at::kByte, like), fresh({rows, tiles}, at::kByte, like)};
  }
};
uint8_t* bytes(const Tensor& t) { return (uint8_t*)ptr(t); }
// codes as the kernels read them
Tensor aligned16(const Tensor& t) {
  const Tensor s = dense(t);
  return !s.defined() || (uintptr_t)s.data_ptr() % 16 == 0 ? s : s.clone();
}

// s = x + residual, y = its norm
struct RmsNorm {
  static int weight_dtype(const Tensor& x, const Tensor& w) { return dtype_of(w.defined() ? w : x); }

  struct Out {
    Tensor y, s;
  };
  static Out run(const Tensor& x2, const Tensor& r2, const Tensor& w, double eps, const Tensor& rstd, const Held& held) {
    const int64_t T = x2.size(0), H = x2.size(1);
    Out o{fresh({T, H}, x2.scalar_type(), x2), {}};
    if (r2.defined()) o.s = fresh({T, H}, x2.scalar_type(), x2);
    check("ntlb_rms_norm_forward",
          abi.rms_forward(x2.data_ptr(), dtype_of(x2), T, H, x2.stride(0), ptr(r2), r2.defined() ? r2.stride(0) : 0,
                          ptr(w), weight_dtype(x2, w), (float)eps, ptr(o.s), H, o.y.data_ptr(), H,
                          rstd.defined() ? rstd.data_ptr<float>() : nullptr, bytes(held.codes), bytes(held.exps),
                          stream_of(x2)));
    return o;
  }
  static Tensor rows(const Tensor& t) { return t.defined() ? rows_of(t) : t; }

  struct Backward : Node {
    Kept s, codes, exps, w, rstd;
    at::DimVector sizes;  // of x
    at::ScalarType type;
    bool summed;          // with a residual: s is a result, with a gradient of its own

    variable_list apply(variable_list&& grads) override {
      const std::lock_guard<std::mutex> lock(mutex_);
      const Tensor ds0 = summed ? grads[1] : Tensor();
      if (!grads[0].defined()) return {ds0, ds0, Tensor()};
      no_tangent("the gradient of rms_norm", grads[0], ds0);
      const Tensor s0 = s.unpack("rows of x", summed ? getptr() : nullptr), c0 = codes.unpack("codes of x"),
                   e0 = exps.unpack("exponents of x"), w0 = w.unpack("values of weight"),
                   r0 = rstd.unpack("rows' deviations");
      const c10::DeviceGuard guard(r0.device());
      const at::AutoDispatchBelowADInplaceOrView below;
      const Tensor s2 = rows(s0), ct = aligned16(c0), et = dense(e0), wt = dense(w0), d2 = rows_of(grads[0]), q2 = rows(ds0);
      const int64_t T = d2.size(0), H = d2.size(1);
      const Tensor dx = fresh({T, H}, type, r0);
      Tensor dw;
      if (wt.defined() && task_should_compute_output(2)) dw = fresh({H}, wt.scalar_type(), r0);
      const int64_t need = abi.rms_workspace(dtype_of(dx), T, H);
      const Tensor ws = scratch(need, r0), stats = dense(r0);
      check("ntlb_rms_norm_backward",
            abi.rms_backward(ptr(s2), dtype_of(dx), T, H, s2.defined() ? s2.stride(0) : 0, bytes(ct), bytes(et),
                             d2.data_ptr(), d2.stride(0), ptr(q2), q2.defined() ? q2.stride(0) : 0,
                             stats.data_ptr<float>(), ptr(wt), weight_dtype(dx, wt), dx.data_ptr(), H, ptr(dw), ptr(ws),
                             need, stream_of(r0)));
      const Tensor out = shaped(dx, sizes);
      return once({task_should_compute_output(0) ? out : Tensor(), task_should_compute_output(1) ? out : Tensor(), dw});
    }
    void release_variables() override {
      const std::lock_guard<std::mutex> lock(mutex_);
      for (Kept* k : {&s, &codes, &exps, &w, &rstd}) k->reset();
    }
    std::string name() const override { return "RmsNormBackward"; }
  };

  static Out forward(const Tensor& x, const Tensor& w, const Tensor& res, double eps, bool keep) {
    const c10::DeviceGuard guard(x.device());
    Tensor x2, rstd;
    Held held;
    Out o;
    {
      const at::AutoDispatchBelowADInplaceOrView below;
      x2 = rows_of(x);
      const int64_t T = x2.size(0);
      rstd = fresh({std::max<int64_t>(1, T)}, at::kFloat, x2);
      if (keep) held = Held::of(T, 1, x2.size(1), x2);
      o = run(x2, rows(res), w, eps, rstd, held);
      o.y = shaped(o.y, x.sizes());
      if (o.s.defined()) o.s = shaped(o.s, x.sizes());
    }
    auto node = make_node<Backward>(torch::autograd::collect_next_edges(x, res, w));
    node->w = Kept(w);
    node->rstd = Kept(rstd);
    node->sizes = x.sizes();
    node->type = x.scalar_type();
    node->summed = res.defined();
    torch::autograd::set_history(o.y, node);
    if (o.s.defined()) torch::autograd::set_history(o.s, node);
    if (keep) {
      node->codes = Kept(held.codes);
      node->exps = Kept(held.exps);
    } else {
      node->s = node->summed ? Kept(o.s, true) : kept(x, x2);
    }
    return o;
  }
};

// ---------------------------------------------------------------------------
struct SwiGlu {
  static Tensor run(const Tensor& x2, int64_t block, const Held& held) {
    const int64_t T = x2.size(0), I = x2.size(1) / 2;
    Tensor h = fresh({T, I}, x2.scalar_type(), x2);
    check("ntlb_swiglu_rows", abi.swiglu(x2.data_ptr(), dtype_of(x2), T, I, x2.stride(0), block, h.data_ptr(), I,
                                         bytes(held.codes), bytes(held.exps), stream_of(x2)));
    return h;
  }
  static Tensor lead(const Tensor& h, const Tensor& x) {
    at::DimVector sizes(x.sizes());
    sizes.back() /= 2;
    return shaped(h, sizes);
  }

  struct Backward : Node {
    Kept x, codes, exps;
    at::DimVector sizes;  // of x
    int64_t block;

    variable_list apply(variable_list&& grads) override {
      const std::lock_guard<std::mutex> lock(mutex_);
      if (!grads[0].defined()) return variable_list(1);
      no_tangent("the gradient of swiglu", grads[0]);
      const Tensor x0 = x.unpack("rows of x"), c0 = codes.unpack("codes of x"), e0 = exps.unpack("exponents of x");
      const c10::DeviceGuard guard(grads[0].device());
      const at::AutoDispatchBelowADInplaceOrView below;
      const Tensor x2 = RmsNorm::rows(x0), ct = aligned16(c0), et = dense(e0), d2 = rows_of(grads[0]);
      const int64_t T = d2.size(0), I = d2.size(1);
      const Tensor dx = fresh({T, 2 * I}, d2.scalar_type(), d2);
      check("ntlb_swiglu_rows_backward",
            abi.swiglu_backward(ptr(x2), dtype_of(d2), T, I, x2.defined() ? x2.stride(0) : 0, block, bytes(ct), bytes(et),
                                d2.data_ptr(), d2.stride(0), dx.data_ptr(), 2 * I, stream_of(d2)));
      return once({shaped(dx, sizes)});
    }
    void release_variables() override {
      const std::lock_guard<std::mutex> lock(mutex_);
      for (Kept* k : {&x, &codes, &exps}) k->reset();
    }
    std::string name() const override { return "SwiGluBackward"; }
  };

  static Tensor forward(const Tensor& x, int64_t block, bool keep) {
    const c10::DeviceGuard guard(x.device());
    Tensor h, x2;
    Held held;
    {
      const at::AutoDispatchBelowADInplaceOrView below;
      x2 = rows_of(x);
      if (keep) held = Held::of(x2.size(0), 2, x2.size(1) / 2, x2);
      h = lead(run(x2, block, held), x);
    }
    auto node = make_node<Backward>(torch::autograd::collect_next_edges(x));
    if (keep) {
      node->codes = Kept(held.codes);
      node->exps = Kept(held.exps);
    } else {
      node->x = kept(x, x2);
    }
    node->sizes = x.sizes();
    node->block = block;
    torch::autograd::set_history(h, node);
    return h;
  }
};

// ---------------------------------------------------------------------------
// y = x W_e^T by rows sorted by expert
struct Grouped {
  static constexpr int64_t MAX_PITCH = 1 << 22;
  static uint16_t* at(const Tensor& t) { return (uint16_t*)ptr(t); }
  static bool pieces(const Tensor& t, int64_t pitch, int64_t cols, bool summed) {
    return t.stride(-1) == 1 && pitch % 8 == 0 && pitch >= cols && pitch <= MAX_PITCH && (uintptr_t)t.data_ptr() % 16 == 0 &&
           (!summed || cols % 8 == 0);
  }
  // [R, C] in rows of whole 16-byte pieces (summed: zero past C): t, or a copy
  static Tensor rows(const Tensor& t, bool summed) {
    if (t.numel() == 0) return t;
    const Tensor r = rows_of(t);
    if (pieces(r, r.stride(0), r.size(1), summed)) return r;
    Tensor out = fresh({r.size(0), (r.size(1) + 7) / 8 * 8}, r.scalar_type(), r);
    check("ntlb_pad_rows", abi.pad_rows(at(r), r.stride(0), r.size(0), r.size(1), at(out), out.size(1), stream_of(r)));
    return out;
  }
  // the same of weights [E, N, K]
  static Tensor weights(const Tensor& w) {
    if (pieces(w, w.stride(1), w.size(2), true) && w.stride(0) >= 0 && w.stride(0) % 8 == 0) return w;
    const int64_t E = w.size(0), N = w.size(1);
    const Tensor r = rows(w.reshape({E * N, w.size(2)}), true);
    return r.as_strided({E, N, r.size(1)}, {N * r.stride(0), r.stride(0), 1});
  }

  static Tensor run(const Tensor& x2, const Tensor& w3, const Tensor& offsets, int64_t N, int64_t K) {
    const int64_t R = x2.size(0);
    Tensor y = fresh({R, N}, x2.scalar_type(), x2), ws;
    const int64_t E = w3.size(0), need = abi.grouped_workspace(R, E, N, K, 0);
    if (need) ws = scratch(need, x2);
    check("ntlb_grouped_matmul", abi.grouped(at(x2), x2.stride(0), at(w3), w3.stride(1), w3.stride(0), offsets.data_ptr<int32_t>(),
                                             R, E, N, K, at(y), N, ptr(ws), need, stream_of(x2)));
    return y;
  }

  struct Backward : Node {
    Kept x, codes, exps, w, offsets;
    int64_t R, E, N, K;

    variable_list apply(variable_list&& grads) override {
      const std::lock_guard<std::mutex> lock(mutex_);
      if (!grads[0].defined()) return variable_list(2);
      no_tangent("the gradient of grouped_matmul", grads[0]);
      const Tensor x0 = x.unpack("rows of x"), c0 = codes.unpack("codes of x"), e0 = exps.unpack("exponents of x"),
                   w0 = w.unpack("values of weight"), o0 = offsets.unpack("offsets");
      const c10::DeviceGuard guard(grads[0].device());
      const at::AutoDispatchBelowADInplaceOrView below;
      const Tensor dy = grads[0], off = dense(o0);
      Tensor dx, dw, d2;
      if (task_should_compute_output(0) && w0.defined()) {
        const Tensor wt = weights(w0);
        d2 = rows(dy, true);
        dx = fresh({R, K}, dy.scalar_type(), dy);
        Tensor ws;
        const int64_t need = abi.grouped_workspace(R, E, N, K, 1);
        if (need) ws = scratch(need, dy);
        check("ntlb_grouped_matmul_dx",
              abi.grouped_dx(at(d2), d2.stride(0), at(wt), wt.stride(1), wt.stride(0), off.data_ptr<int32_t>(), R, E, N, K,
                             at(dx), K, ptr(ws), need, stream_of(dy)));
      }
      if (task_should_compute_output(1) && (x0.defined() || c0.defined())) {
        if (!d2.defined()) d2 = rows(dy, false);
        Tensor x2;
        if (x0.defined()) {
          x2 = rows(x0, false);
        } else {
          const Tensor ct = aligned16(c0), et = dense(e0);
          x2 = fresh({R, (K + 7) / 8 * 8}, dy.scalar_type(), dy);
          check("ntlb_kept_values", abi.kept_values(bytes(ct), bytes(et), R, K, at(x2), x2.size(1), stream_of(dy)));
        }
        dw = fresh({E, N, K}, dy.scalar_type(), dy);
        check("ntlb_grouped_matmul_dw", abi.grouped_dw(at(d2), d2.stride(0), at(x2), x2.stride(0), off.data_ptr<int32_t>(), R,
                                                       E, N, K, at(dw), stream_of(dy)));
      }
      return once({dx, dw});
    }
    void release_variables() override {
      const std::lock_guard<std::mutex> lock(mutex_);
      for (Kept* k : {&x, &codes, &exps, &w, &offsets}) k->reset();
    }
    std::string name() const override { return "GroupedMatmulBackward"; }
  };

  static Tensor forward(const Tensor& x, const Tensor& w, const Tensor& offsets, bool keep) {
    const c10::DeviceGuard guard(x.device());
    const int64_t R = x.size(0), K = x.size(1), E = w.size(0), N = w.size(1);
    Tensor y, x2, w3;
    Held held;
    {
      const at::AutoDispatchBelowADInplaceOrView below;
      x2 = rows(x, true);
      w3 = weights(w);
      if (keep && wanted(w)) {
        held = Held::of(R, 1, K, x);
        check("ntlb_kept_rows", abi.kept_rows(at(x2), x2.stride(0), R, K, bytes(held.codes), bytes(held.exps), stream_of(x)));
      }
      y = run(x2, w3, offsets, N, K);
    }
    auto node = make_node<Backward>(torch::autograd::collect_next_edges(x, w));
    // each operand is kept for the other's gradient
    if (held.codes.defined()) {
      node->codes = Kept(held.codes);
      node->exps = Kept(held.exps);
    } else if (wanted(w)) {
      node->x = kept(x, x2);
    }
    if (wanted(x)) node->w = kept(w, w3);
    node->offsets = Kept(offsets);
    node->R = R;
    node->E = E;
    node->N = N;
    node->K = K;
    torch::autograd::set_history(y, node);
    return y;
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

PyObject* wrap(const Tensor& t) {
  if (!t.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(t);
}
template <size_t N>
PyObject* wrap_all(const Tensor (&ts)[N]) {
  THPObjectPtr out(PyTuple_New(N));
  if (!out) throw python_error();
  for (size_t i = 0; i < N; ++i) {
    PyObject* o = wrap(ts[i]);
    if (!o) throw python_error();
    PyTuple_SET_ITEM(out.get(), i, o);
  }
  return out.release();
}

// rms_norm(x, weight | None, residual | None, eps, keep) -> y, or (y, s) with a residual
PyObject* py_rms_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 5);
  const Tensor& x = THPVariable_Unpack(a[0]);
  const Tensor w = maybe(a[1]), res = maybe(a[2]);
  const double eps = real(a[3]);
  const bool keep = integer(a[4]) != 0;
  RmsNorm::Out o;
  {
    const NoGil nogil;
    no_tangent("rms_norm", x, w, res);
    if (at::GradMode::is_enabled() && (wanted(x) || wanted(w) || wanted(res))) {
      o = RmsNorm::forward(x, w, res, eps, keep);
    } else {
      const at::AutoDispatchBelowADInplaceOrView below;
      const c10::DeviceGuard guard(x.device());
      o = RmsNorm::run(rows_of(x), RmsNorm::rows(res), w, eps, Tensor(), Held());
      o.y = shaped(o.y, x.sizes());
      if (o.s.defined()) o.s = shaped(o.s, x.sizes());
    }
  }
  if (!o.s.defined()) return THPVariable_Wrap(o.y);
  return wrap_all({o.y, o.s});
  END_HANDLE_TH_ERRORS
}

// rms_norm_quant(x, weight | None, residual | None, eps, grid, nan) ->
// (codes, scales by tile, nan rows | None, s | None)
PyObject* py_rms_norm_quant(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 6);
  const Tensor& x = THPVariable_Unpack(a[0]);
  const Tensor w = maybe(a[1]), res = maybe(a[2]);
  const double eps = real(a[3]);
  const int grid = (int)integer(a[4]);
  const bool want_nan = integer(a[5]) != 0;
  Tensor codes, scales, nan, s;
  {
    const NoGil nogil;
    no_tangent("rms_norm_quant", x, w, res);
    const at::AutoDispatchBelowADInplaceOrView below;
    const c10::DeviceGuard guard(x.device());
    const Tensor x2 = rows_of(x), r2 = RmsNorm::rows(res);
    const int64_t T = x2.size(0), H = x2.size(1), tiles = (H + 127) / 128, rp = std::max<int64_t>((T + 3) / 4 * 4, 4);
    codes = fresh({T, tiles * 128}, at::kByte, x2);
    scales = fresh({tiles, rp}, at::kFloat, x2);
    if (want_nan) nan = fresh({T}, at::kInt, x2).zero_();
    if (r2.defined()) s = fresh({T, H}, x2.scalar_type(), x2);
    check("ntlb_rms_norm_quant",
          abi.rms_quant(x2.data_ptr(), dtype_of(x2), T, H, x2.stride(0), ptr(r2), r2.defined() ? r2.stride(0) : 0, ptr(w),
                        RmsNorm::weight_dtype(x2, w), (float)eps, ptr(s), H, grid, bytes(codes), tiles * 128,
                        scales.data_ptr<float>(), 1, rp, nan.defined() ? nan.data_ptr<int32_t>() : nullptr,
                        stream_of(x2)));
    if (s.defined()) s = shaped(s, x.sizes());
  }
  return wrap_all({codes, scales, nan, s});
  END_HANDLE_TH_ERRORS
}

// swiglu(x, block, keep) -> h
PyObject* py_swiglu(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 3);
  const Tensor& x = THPVariable_Unpack(a[0]);
  const int64_t block = integer(a[1]);
  const bool keep = integer(a[2]) != 0;
  Tensor h;
  {
    const NoGil nogil;
    no_tangent("swiglu", x);
    if (at::GradMode::is_enabled() && wanted(x)) {
      h = SwiGlu::forward(x, block, keep);
    } else {
      const at::AutoDispatchBelowADInplaceOrView below;
      const c10::DeviceGuard guard(x.device());
      h = SwiGlu::lead(SwiGlu::run(rows_of(x), block, Held()), x);
    }
  }
  return THPVariable_Wrap(h);
  END_HANDLE_TH_ERRORS
}

// grouped_matmul(x, weight, offsets, keep) -> y
PyObject* py_grouped_matmul(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 4);
  const Tensor &x = THPVariable_Unpack(a[0]), &w = THPVariable_Unpack(a[1]), &offsets = THPVariable_Unpack(a[2]);
  const bool keep = integer(a[3]) != 0;
  Tensor y;
  {
    const NoGil nogil;
    no_tangent("grouped_matmul", x, w);
    if (at::GradMode::is_enabled() && (wanted(x) || wanted(w))) {
      y = Grouped::forward(x, w, offsets, keep);
    } else {
      const at::AutoDispatchBelowADInplaceOrView below;
      const c10::DeviceGuard guard(x.device());
      y = Grouped::run(Grouped::rows(x, true), Grouped::weights(w), offsets, w.size(1), w.size(2));
    }
  }
  return THPVariable_Wrap(y);
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
  take(table, "ntlb_rms_norm_forward", a.rms_forward);
  take(table, "ntlb_rms_norm_quant", a.rms_quant);
  take(table, "ntlb_rms_norm_backward", a.rms_backward);
  take(table, "ntlb_rms_norm_workspace_bytes", a.rms_workspace);
  take(table, "ntlb_swiglu_rows", a.swiglu);
  take(table, "ntlb_swiglu_rows_backward", a.swiglu_backward);
  take(table, "ntlb_grouped_matmul", a.grouped);
  take(table, "ntlb_grouped_matmul_dx", a.grouped_dx);
  take(table, "ntlb_grouped_matmul_dw", a.grouped_dw);
  take(table, "ntlb_grouped_matmul_workspace_bytes", a.grouped_workspace);
  take(table, "ntlb_kept_rows", a.kept_rows);
  take(table, "ntlb_kept_values", a.kept_values);
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
    {"rms_norm", (PyCFunction)(void (*)(void))py_rms_norm, METH_FASTCALL, nullptr},
    {"rms_norm_quant", (PyCFunction)(void (*)(void))py_rms_norm_quant, METH_FASTCALL, nullptr},
    {"grouped_matmul", (PyCFunction)(void (*)(void))py_grouped_matmul, METH_FASTCALL, nullptr},
    {"swiglu", (PyCFunction)(void (*)(void))py_swiglu, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_autograd", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__autograd(void) { return PyModule_Create(&module); }
