// The host side of autograd.linear: checks, allocation and the autograd node of the dense layer (linear.hip) in C++.  A small layer's training step
// is host time: with the node in Python it took 125 us, of which the three kernels of a 64 x 64 layer are 15 and the engine's change of thread 40;
// the rest was the interpreter, in two threads that take turns holding it.
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>
#include <torch/library.h>

#include <numeric>

#include "../../include/s2l_hip.h"

namespace {

using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

struct Library {      // the C ABI's entries, of the library that the package has loaded
  decltype(&s2l_linear_saved_bytes) saved_bytes = nullptr;
  decltype(&s2l_linear_forward_work_bytes) forward_bytes = nullptr;
  decltype(&s2l_linear_backward_work_bytes) backward_bytes = nullptr;
  decltype(&s2l_linear_forward) forward = nullptr;
  decltype(&s2l_linear_backward) backward = nullptr;
} lib;

int dtype_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return S2L_DTYPE_F32;
    case at::kBFloat16: return S2L_DTYPE_BF16;
    case at::kHalf: return S2L_DTYPE_F16;
    default: return -1;
  }
}

struct Rows {      // a tensor [..., n] as rows of dense columns; a view wherever the strides allow it (a lazily negated one is copied)
  Tensor t;
  int64_t rows, ld;
};
Rows rows_of(const Tensor& t) {
  const int64_t n = t.size(-1);
  Tensor r = t.dim() == 2 ? t : t.reshape({-1, n});
  if (r.is_neg()) r = r.resolve_neg();
  if ((n > 1 && r.stride(1) != 1) || (r.size(0) > 1 && r.stride(0) < n)) r = r.contiguous();
  return {r, r.size(0), r.size(0) > 1 ? r.stride(0) : n};
}

void* data(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor bytes(int64_t n, const Tensor& like) { return n ? at::empty({n}, like.options().dtype(at::kByte)) : Tensor(); }
s2l_stream_t stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

bool capturing(hipStream_t stream) {      // (the null stream takes part in no capture, and asking for it would end one)
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  return stream && hipStreamIsCapturing(stream, &status) == hipSuccess && status == hipStreamCaptureStatusActive;
}

void check(int rc, const char* what) {      // the package's own error
  if (!rc) return;
  py::gil_scoped_acquire gil;
  py::module_::import("speech2lip_amd._abi").attr("check")(rc, what);
}

// whether these are what the layer takes
bool fits(const Tensor& x, const Tensor& weight, const Tensor& b, const Tensor& r) {
  const auto like = [&](const Tensor& t) { return t.scalar_type() == x.scalar_type() && t.device() == x.device() && t.layout() == at::kStrided; };
  return dtype_of(x) >= 0 && x.dim() >= 1 && weight.dim() == 2 && like(x) && like(weight) && x.size(-1) == weight.size(1) && weight.size(0) > 0 && weight.size(1) > 0 &&
         (!b.defined() || (like(b) && b.dim() == 1 && b.size(0) == weight.size(0))) &&
         (!r.defined() || (like(r) && r.dim() == x.dim() && r.size(-1) == weight.size(0) && r.sizes().slice(0, r.dim() - 1) == x.sizes().slice(0, x.dim() - 1)));
}

using Forward = std::tuple<Tensor, Tensor>;      // the result, what is kept (or nothing)
Forward forward_launch(const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& residual, int64_t act, double slope, bool keep) {
  const c10::DeviceGuard device(x.device());
  const int dt = dtype_of(x);
  const Rows xr = rows_of(x), wr = rows_of(weight);
  const int64_t n = weight.size(0), k = weight.size(1);
  Rows rr{Tensor(), 0, n};
  if (residual.defined()) rr = rows_of(residual);
  const Tensor b = bias.defined() ? bias.resolve_neg().contiguous() : bias;
  std::vector<int64_t> sizes = x.sizes().vec();
  sizes.back() = n;
  const Tensor out = at::empty(sizes, x.options()), saved = keep ? bytes(lib.saved_bytes(dt, act, xr.rows, n), x) : Tensor();
  const Tensor work = bytes(lib.forward_bytes(dt, act, saved.defined(), xr.rows, k, n), x);
  const int rc = lib.forward(dt, data(xr.t), xr.ld, data(wr.t), wr.ld, data(b), data(rr.t), rr.ld, data(out), n, data(saved), data(work), xr.rows, k, n, act,
                             (float)slope, stream_of(x));
  check(rc, "s2l_linear_forward");
  return {out, saved};
}

using Gradients = std::tuple<Tensor, Tensor, Tensor>;      // of x, weight and bias, where they are needed
Gradients backward_launch(const Tensor& dy, const Tensor& x, const Tensor& weight, const Tensor& saved, at::IntArrayRef x_sizes, at::IntArrayRef w_sizes, int64_t act,
                          double slope, bool need_x, bool need_w, bool need_b) {
  const c10::DeviceGuard device(dy.device());
  const int dt = dtype_of(dy);
  const Rows d = rows_of(dy);
  const int64_t n = w_sizes[0], k = w_sizes[1];
  Rows xr{}, wr{};
  if (need_w) xr = rows_of(x);
  if (need_x) wr = rows_of(weight);
  Tensor dx, dw, db;
  if (need_x) dx = at::empty(x_sizes, dy.options());
  if (need_w) dw = at::empty(w_sizes, dy.options());
  if (need_b) db = at::empty({n}, dy.options());
  const Tensor work = bytes(lib.backward_bytes(dt, act, d.rows, k, n), dy);
  const int rc = lib.backward(dt, data(d.t), d.ld, data(xr.t), need_w ? xr.ld : k, data(wr.t), need_x ? wr.ld : k, data(saved), data(dx), k, data(dw), data(db),
                              data(work), d.rows, k, n, act, (float)slope, stream_of(dy));
  check(rc, "s2l_linear_backward");
  return {dx, dw, db};
}

// The same as operators that torch knows, for whatever watches, records or replaces a call's operators: dispatch modes (make_fx, fake tensors,
// selective checkpoints, counters) and subclasses that dispatch for themselves.  They would see the allocations of the functions above and not their
// launches, and a recorded program would return memory that nothing wrote.  Anybody can call these, so that they check; an absent result is an empty one.
Tensor present(const std::optional<Tensor>& t) { return t.has_value() && t->defined() ? *t : Tensor(); }
Tensor or_empty(const Tensor& t, const Tensor& like) { return t.defined() ? t : at::empty({0}, like.options()); }
Tensor or_none(const Tensor& t, bool wanted) { return wanted ? t : Tensor(); }

Forward linear_forward(const Tensor& x, const Tensor& weight, const std::optional<Tensor>& bias, const std::optional<Tensor>& residual, int64_t act, double slope, bool keep) {
  TORCH_CHECK_VALUE(fits(x, weight, present(bias), present(residual)) && act >= S2L_ACT_NONE && act <= S2L_ACT_SILU,
                    "linear_forward: these are not the layer's operands (shapes, one type, one GPU, activation)");
  const auto [out, saved] = forward_launch(x, weight, present(bias), present(residual), act, slope, keep);
  return {out, saved.defined() ? saved : at::empty({0}, x.options().dtype(at::kByte))};
}
Forward linear_forward_meta(const Tensor& x, const Tensor& weight, const std::optional<Tensor>& bias, const std::optional<Tensor>& residual, int64_t act, double slope, bool keep) {
  std::vector<int64_t> sizes = x.sizes().vec();
  sizes.back() = weight.size(0);
  const int64_t rows = std::accumulate(sizes.begin(), sizes.end() - 1, (int64_t)1, std::multiplies<>());
  return {at::empty(sizes, x.options()), at::empty({keep ? lib.saved_bytes(dtype_of(x), act, rows, weight.size(0)) : 0}, x.options().dtype(at::kByte))};
}
Gradients linear_backward(const Tensor& dy, const std::optional<Tensor>& x, const std::optional<Tensor>& weight, const std::optional<Tensor>& saved, at::IntArrayRef x_sizes,
                          at::IntArrayRef w_sizes, int64_t act, double slope, bool need_x, bool need_w, bool need_b) {
  const auto like = [&](const Tensor& t, at::IntArrayRef sizes) {
    return t.defined() && t.scalar_type() == dy.scalar_type() && t.device() == dy.device() && t.layout() == at::kStrided && t.sizes() == sizes;
  };
  const Tensor xs = present(x), ws = present(weight), kept = present(saved);
  bool fine = dtype_of(dy) >= 0 && act >= S2L_ACT_NONE && act <= S2L_ACT_SILU && w_sizes.size() == 2 && w_sizes[0] > 0 && w_sizes[1] > 0 && !x_sizes.empty() &&
              x_sizes.back() == w_sizes[1] && (need_x || need_w) && (need_w || !need_b);
  if (fine) {
    std::vector<int64_t> y_sizes = x_sizes.vec();
    y_sizes.back() = w_sizes[0];
    const int64_t rows = std::accumulate(y_sizes.begin(), y_sizes.end() - 1, (int64_t)1, std::multiplies<>());
    fine = like(dy, y_sizes) && (!need_w || like(xs, x_sizes)) && (!need_x || like(ws, w_sizes));
    if (fine && lib.saved_bytes(dtype_of(dy), act, rows, w_sizes[0]))
      fine = kept.defined() && kept.scalar_type() == at::kByte && kept.device() == dy.device() && kept.is_contiguous() &&
             kept.numel() == lib.saved_bytes(dtype_of(dy), act, rows, w_sizes[0]);
  }
  TORCH_CHECK_VALUE(fine, "linear_backward: these are not the layer's operands (shapes, one type, one GPU, what the forward kept)");
  const auto [dx, dw, db] = backward_launch(dy, xs, ws, kept, x_sizes, w_sizes, act, slope, need_x, need_w, need_b);
  return {or_empty(dx, dy), or_empty(dw, dy), or_empty(db, dy)};
}
Gradients linear_backward_meta(const Tensor& dy, const std::optional<Tensor>&, const std::optional<Tensor>&, const std::optional<Tensor>&, at::IntArrayRef x_sizes,
                               at::IntArrayRef w_sizes, int64_t, double, bool need_x, bool need_w, bool need_b) {
  const int64_t zero[1] = {0};
  const at::IntArrayRef none(zero, 1), n = w_sizes.slice(0, 1);
  return {at::empty(need_x ? x_sizes : none, dy.options()), at::empty(need_w ? w_sizes : none, dy.options()), at::empty(need_b ? n : none, dy.options())};
}

TORCH_LIBRARY(speech2lip_amd, m) {
  m.def("linear_forward(Tensor x, Tensor weight, Tensor? bias, Tensor? residual, int activation, float slope, bool keep) -> (Tensor, Tensor)");
  m.def("linear_backward(Tensor dy, Tensor? x, Tensor? weight, Tensor? saved, int[] x_sizes, int[] weight_sizes, int activation, float slope, bool need_x, "
        "bool need_weight, bool need_bias) -> (Tensor, Tensor, Tensor)");
}
TORCH_LIBRARY_IMPL(speech2lip_amd, CUDA, m) {
  m.impl("linear_forward", &linear_forward);
  m.impl("linear_backward", &linear_backward);
}
TORCH_LIBRARY_IMPL(speech2lip_amd, Meta, m) {
  m.impl("linear_forward", &linear_forward_meta);
  m.impl("linear_backward", &linear_backward_meta);
}

bool watched(std::initializer_list<const Tensor*> tensors) {
  bool subclass = false;
  for (const Tensor* t : tensors) subclass |= t->defined() && t->key_set().has(c10::DispatchKey::Python);
  return subclass || c10::impl::TorchDispatchModeTLS::any_modes_set();
}

std::optional<Tensor> given(const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }

Forward forward_of(const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& residual, int64_t act, double slope, bool keep) {
  if (!watched({&x, &weight, &bias, &residual})) return forward_launch(x, weight, bias, residual, act, slope, keep);
  static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("speech2lip_amd::linear_forward", "").typed<decltype(linear_forward)>();
  auto [out, saved] = op.call(x, weight, given(bias), given(residual), act, slope, keep);
  return {out, or_none(saved, keep && act != S2L_ACT_NONE)};
}
Gradients backward_of(const Tensor& dy, const Tensor& x, const Tensor& weight, const Tensor& saved, at::IntArrayRef x_sizes, at::IntArrayRef w_sizes, int64_t act,
                      double slope, bool need_x, bool need_w, bool need_b) {
  if (!watched({&dy, &x, &weight, &saved})) return backward_launch(dy, x, weight, saved, x_sizes, w_sizes, act, slope, need_x, need_w, need_b);
  static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("speech2lip_amd::linear_backward", "").typed<decltype(linear_backward)>();
  auto [dx, dw, db] = op.call(dy, given(x), given(weight), given(saved), x_sizes, w_sizes, act, slope, need_x, need_w, need_b);
  return {or_none(dx, need_x), or_none(dw, need_w), or_none(db, need_b)};
}

struct LinearBackward : public Node {
  SavedVariable x, weight, saved;
  int act = 0;
  float slope = 0.f;
  bool released = false;
  std::vector<int64_t> x_sizes, w_sizes;

  std::string name() const override { return "S2LLinearBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    x.reset_data();
    weight.reset_data();
    saved.reset_data();
    released = true;
  }

  // The engine delivers a gradient on the stream on which its receiver was made: it lets that stream wait for this one.  A leaf's receiver lives as long
  // as any graph that holds the leaf, so that an eager graph's makes a captured backward pass reach outside its capture, which torch answers by
  // ending the process.
  void refuse_foreign_edges() {
    for (uint32_t i = 0; i < num_outputs(); ++i) {
      if (!task_should_compute_output(i)) continue;
      const auto stream = next_edge(i).function->stream();
      TORCH_CHECK(!stream || capturing(c10::hip::HIPStreamMasqueradingAsCUDA(*stream).stream()),
                  "linear: this backward pass is being captured, and an input of it is held by a graph made outside the capture (its gradient would be "
                  "delivered on that graph's stream): drop that graph before the capture, or capture with detached leaves");
    }
  }

  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    variable_list out(4);
    const Tensor& dy = grads[0];
    if (!dy.defined()) return out;
    if (capturing(static_cast<hipStream_t>(stream_of(dy)))) refuse_foreign_edges();
    const bool need_x = task_should_compute_output(0), need_b = task_should_compute_output(2), need_w = task_should_compute_output(1) || need_b;
    if (need_x || need_w) {
      TORCH_CHECK(!released, "Trying to backward through the graph a second time (the dense layer's saved values have been freed; "
                             "specify retain_graph=True to go through it again)");
      const Tensor xs = need_w ? x.unpack() : Tensor(), ws = need_x ? weight.unpack() : Tensor(), kept = saved.unpack();
      at::AutoDispatchBelowAutograd below;
      const auto [dx, dw, db] = backward_of(dy, xs, ws, kept, x_sizes, w_sizes, act, slope, need_x, need_w, need_b);      // (the bias gradient is a by-product of dW)
      out[0] = dx;
      if (task_should_compute_output(1)) out[1] = dw;
      out[2] = db;
    }
    if (task_should_compute_output(3)) out[3] = dy;
    if (at::GradMode::is_enabled()) {      // create_graph: the gradients are there, differentiating them again is refused
      variable_list marked;
      for (const Tensor& t : out) marked.push_back(t.defined() ? t.detach().set_requires_grad(true) : Tensor());
      auto error = std::make_shared<torch::autograd::DelayedError>("linear: the backward pass of the dense layer is not differentiable", (int64_t)out.size());
      out = (*error)(std::move(marked));
    }
    return out;
  }
};

// None where the arguments are not what `linear` takes: the caller says what is wrong with them.
py::object linear(const Tensor& x, const Tensor& weight, const std::optional<Tensor>& bias, const std::optional<Tensor>& residual, int act, double slope) {
  const Tensor b = bias.value_or(Tensor()), r = residual.value_or(Tensor());
  TORCH_CHECK_NOT_IMPLEMENTED(!torch::jit::tracer::isTracing(), "linear: not under torch.jit.trace, which would record the allocation of the result and not the launch that writes it");
  if (!x.is_cuda() || !fits(x, weight, b, r)) return py::none();
  const bool need_x = x.requires_grad(), need_w = weight.requires_grad(), need_b = b.defined() && b.requires_grad(), need_r = r.defined() && r.requires_grad();
  const bool grad = at::GradMode::is_enabled() && (need_x || need_w || need_b || need_r);
  for (const Tensor& t : {x, weight, b, r})
    TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(0).defined(), "linear: no forward-mode derivatives");
  Tensor out, saved;
  {
    at::AutoDispatchBelowAutograd below;
    std::tie(out, saved) = forward_of(x, weight, b, r, act, slope, grad && (need_x || need_w || need_b));
  }
  if (grad) {
    auto node = std::shared_ptr<LinearBackward>(new LinearBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(x, weight, b, r));
    if (need_w || need_b) node->x = SavedVariable(x, false);
    if (need_x) node->weight = SavedVariable(weight, false);
    if (saved.defined()) node->saved = SavedVariable(saved, false);
    node->act = act;
    node->slope = (float)slope;
    node->x_sizes = x.sizes().vec();
    node->w_sizes = weight.sizes().vec();
    torch::autograd::set_history(out, node);
  }
  return py::cast(out);
}

void bind(uint64_t saved_bytes, uint64_t forward_bytes, uint64_t backward_bytes, uint64_t forward, uint64_t backward) {
  lib.saved_bytes = reinterpret_cast<decltype(lib.saved_bytes)>(saved_bytes);
  lib.forward_bytes = reinterpret_cast<decltype(lib.forward_bytes)>(forward_bytes);
  lib.backward_bytes = reinterpret_cast<decltype(lib.backward_bytes)>(backward_bytes);
  lib.forward = reinterpret_cast<decltype(lib.forward)>(forward);
  lib.backward = reinterpret_cast<decltype(lib.backward)>(backward);
}

}  // namespace

PYBIND11_MODULE(_linear_ops, m) {
  m.attr("built_for") = "built for torch " S2L_TORCH_VERSION ";";
  m.def("linear", &linear);
  m.def("bind", &bind);
}
