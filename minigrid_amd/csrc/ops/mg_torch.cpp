// mg_torch.cpp — the learning operators as torch sees them (minigrid_amd/ops.py is their documented face): argument checks, result and workspace tensors,
// the calls of the C entries (include/minigrid_ops.h) on the tensors' device and its current stream, and the backward nodes.  In C++ because a
// policy's layers are small: what a call costs on the host is most of what it costs.  The entries are taken from the library that the package has
// loaded; nothing here links against it.
#include <torch/extension.h>

#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPException.h>
#include <c10/hip/HIPStream.h>
#include <dlfcn.h>

#include <unordered_set>

#include "../../../include/minigrid_ops.h"

namespace {

using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
typedef std::optional<Tensor> MaybeTensor;

#define MG_ENTRIES(X) \
  X(mg_ops_last_error) X(mg_op_linear_workspace) X(mg_op_linear) X(mg_op_linear_dz_workspace) X(mg_op_linear_dz) X(mg_op_linear_dx) X(mg_op_linear_dw) \
  X(mg_op_policy_loss_workspace) X(mg_op_policy_loss) X(mg_op_policy_loss_makes_gradient) X(mg_op_policy_loss_with_gradient) X(mg_op_policy_loss_backward) X(mg_op_policy_loss_rescale) X(mg_op_sample_workspace) X(mg_op_sample) X(mg_op_advantages)
struct Entries {
#define X(name) decltype(&::name) name = nullptr;
  MG_ENTRIES(X)
#undef X
} L;

void bind_library(uintptr_t handle) {
#define X(name) \
  L.name = (decltype(&::name))dlsym((void*)handle, #name); \
  if (!L.name) throw std::runtime_error("the loaded library does not hold " #name);
  MG_ENTRIES(X)
#undef X
}

template <class... A> [[noreturn]] void refuse(const A&... a) { throw py::value_error(c10::str(a...)); }

struct HipError : std::runtime_error { using std::runtime_error::runtime_error; };      // minigrid_amd's MiniGridHipError
PyObject* hip_error = nullptr;

void check(int rc) {
  if (rc == MG_OK) return;
  const std::string text = L.mg_ops_last_error();
  if (rc == MG_ERR_INVALID) throw py::value_error(text);
  throw HipError(c10::str("libminigrid_hip error ", rc, ": ", text));
}

int dtype_of(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return MG_DT_F32;
    case at::kBFloat16: return MG_DT_BF16;
    case at::kHalf: return MG_DT_F16;
    case at::kByte: case at::kBool: return MG_DT_U8;
    case at::kDouble: return MG_DT_F64;
    case at::kInt: return MG_DT_I32;
    case at::kLong: return MG_DT_I64;
    default: return -1;
  }
}
bool is_float(at::ScalarType t) { return t == at::kFloat || t == at::kBFloat16 || t == at::kHalf; }

void on_gpu(const char* name, const Tensor& t) {
  if (!t.is_cuda()) refuse(name, " must be on the GPU: minigrid_amd has no CPU fallback");
  if (t.layout() != at::kStrided) refuse(name, " must be a dense tensor");
  // (an optional argument without memory would be taken for one that was not given)
  if (t.numel() && !t.const_data_ptr()) refuse(name, " has no memory: a fake or wrapped tensor cannot be read");
}
void on_gpu(const char* name, const Tensor& t, at::Device dev) {
  on_gpu(name, t);
  if (t.device() != dev) refuse(name, " is on ", t.device(), ", expected ", dev);
}

void* stream_of(at::Device dev) { return (void*)c10::hip::getCurrentHIPStream(dev.index()).stream(); }

Tensor make(at::IntArrayRef shape, at::ScalarType t, at::Device dev) { return at::empty(shape, at::TensorOptions().dtype(t).device(dev)); }
// scratch of a call: given back to the allocator with the call's end, on the call's stream
struct Scratch {
  Tensor t;
  int64_t bytes;
  Scratch(int64_t n, at::Device dev) : bytes(n) { if (n) t = make({n}, at::kByte, dev); }
  void* p() const { return bytes ? t.data_ptr() : nullptr; }
};
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// (a real tensor may carry a minus sign that is still to be applied: its memory does not hold its values)
Tensor values(const Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }

// t as (rows, cols) with contiguous columns and rows that do not overlap: the tensor's own memory where its strides allow it, else a copy
Tensor matrix(const Tensor& signed_t, int64_t cols) {
  const Tensor t = values(signed_t);
  Tensor m = t.dim() == 2 ? t : t.reshape({t.numel() / cols, cols});
  if ((cols > 1 && m.stride(1) != 1) || (m.size(0) > 1 && m.stride(0) < cols)) m = m.contiguous();
  return m;
}
int64_t row_stride(const Tensor& m) { return std::max(m.stride(0), m.size(1)); }     // (the stride of a single row means nothing)

// What the backward pass reads again.  A saved-tensor hook may hand back another tensor than it was given: one of another type, shape or device would be read out of
// its bounds, and is refused; strides are looked at again.
struct Kept {
  SavedVariable saved;
  at::ScalarType type = at::kFloat;
  at::DimVector sizes;
  at::Device dev = at::kCPU;
  void put(const Tensor& t, bool is_output = false) {
    saved = SavedVariable(t, is_output);
    type = t.scalar_type();
    sizes = at::DimVector(t.sizes());
    dev = t.device();
  }
  // the tensor itself where the operator read its memory (a change in place is then noticed), else the copy
  void put(const Tensor& original, const Tensor& used) { put(original.data_ptr() == used.data_ptr() ? original : used); }
  Tensor get(const char* name, std::shared_ptr<Node> owner = nullptr) const {
    const Tensor t = saved.unpack(std::move(owner));
    TORCH_CHECK(t.defined() && t.scalar_type() == type && t.sizes() == at::IntArrayRef(sizes) && t.device() == dev && t.layout() == at::kStrided, name, " was saved as ", type, " ",
                at::IntArrayRef(sizes), " on ", dev, ", and a saved-tensor hook gave back another type, shape or device");
    return t;
  }
  Tensor get_contiguous(const char* name, std::shared_ptr<Node> owner = nullptr) const { return values(get(name, std::move(owner))).contiguous(); }
  void reset_data() { saved.reset_data(); }
};

at::DimVector with_last(at::IntArrayRef lead, int64_t last) {
  at::DimVector s(lead.begin(), lead.end() - 1);
  s.push_back(last);
  return s;
}

// The gradients of a backward pass that is itself recorded depend on what they were made from, but cannot be differentiated again: an error there, not a zero.
variable_list no_second(const char* name, variable_list&& grads, std::initializer_list<const Tensor*> from) {
  if (!at::GradMode::is_enabled()) return std::move(grads);
  torch::autograd::edge_list edges;
  for (const Tensor* t : from)
    if (t->defined() && t->requires_grad()) edges.push_back(torch::autograd::impl::gradient_edge(*t));
  if (edges.empty()) return std::move(grads);
  auto error = std::shared_ptr<torch::autograd::Error>(
      new torch::autograd::Error(c10::str("trying to differentiate ", name, " twice: its gradient is not differentiable"), std::move(edges)), torch::autograd::deleteNode);
  for (auto& g : grads)
    if (g.defined()) {
      g = g.detach();
      torch::autograd::set_history(g, error);
    }
  return std::move(grads);
}

// the capture that a stream takes part in: a number that no other capture has, or 0
uint64_t capture_of(hipStream_t stream) {
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  unsigned long long id = 0;
  C10_HIP_CHECK(hipStreamGetCaptureInfo(stream, &status, &id));
  return status == hipStreamCaptureStatusNone ? 0 : id;
}
uint64_t capture_on(at::Device dev) { return capture_of(c10::hip::getCurrentHIPStream(dev.index()).stream()); }

// A captured step must not meet an eager graph of the same leaves that is still alive, or go on from one: the leaves' gradient nodes (or that graph's own) belong to the
// stream that it was recorded on, the backward pass would wait on that stream from inside the capture, and torch ends the process there.  Said here, where it can
// still be said, of everything that the inputs were made from.
void refuse_capture_beside_eager(at::Device dev, std::initializer_list<const Tensor*> inputs) {
  const uint64_t capture = capture_on(dev);
  if (!capture) return;
  const auto here = c10::hip::getCurrentHIPStream(dev.index()).id();
  // (a stream that has joined the capture belongs to it; the null stream never does, and may not be asked)
  auto inside = [&](const c10::Stream& s) {
    if (s.id() == here) return true;
    const hipStream_t stream = c10::hip::HIPStream(c10::hip::HIPStream::UNCHECKED, s).stream();
    return stream && capture_of(stream) == capture;
  };
  std::vector<std::shared_ptr<Node>> todo;
  std::unordered_set<Node*> seen;
  for (const Tensor* t : inputs) {
    if (!t->defined() || !t->requires_grad()) continue;
    // (a leaf's gradient node is looked at where there is one, not made)
    if (auto node = t->grad_fn() ? t->grad_fn() : torch::autograd::impl::try_get_grad_accumulator(*t)) todo.push_back(std::move(node));
  }
  while (!todo.empty()) {
    const auto node = std::move(todo.back());
    todo.pop_back();
    if (!seen.insert(node.get()).second) continue;
    const auto at = node->stream();
    if (at && !inside(*at))
      refuse("a tensor that requires a gradient is still part of a graph recorded outside of this capture: drop that graph's results before capturing");
    for (const auto& edge : node->next_edges())
      if (edge.function) todo.push_back(edge.function);
  }
}

// A tracer records the tensors that an operator makes and not what fills them: the traced function would return uninitialised memory.
void refuse_tracing(const char* name) {
  typedef c10::impl::TorchDispatchModeTLS Modes;
  if (torch::jit::tracer::isTracing() || (Modes::any_modes_set() && Modes::get_mode(c10::impl::TorchDispatchModeKey::PROXY)))
    refuse(name, " cannot be traced: the trace would not hold the operator (a captured graph does)");
}

// There is no forward-mode derivative: a result without a tangent would be taken for a constant.
void refuse_tangents(const char* name, std::initializer_list<const Tensor*> inputs) {
  for (const Tensor* t : inputs)
    if (t->defined() && torch::autograd::isFwGradDefined(*t)) refuse(name, " has no forward-mode derivative: an argument carries a tangent");
}

// ---- linear ---------------------------------------------------------------------------------------------------------------------------

struct LinearBackward : public Node {
  Kept x, w, z;
  int64_t act = 0;
  at::DimVector x_shape;
  std::string name() const override { return "MinigridLinearBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    x.reset_data();
    w.reset_data();
    z.reset_data();
  }
  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    variable_list out(4);
    if (!grads[0].defined()) return out;
    refuse_tracing("the gradient of linear");
    refuse_tangents("the gradient of linear", {&grads[0]});
    const Tensor x0 = x.get("x"), w0 = w.get("weight"), z0 = act ? z.get_contiguous("what the activation's slope is told from", shared_from_this()) : Tensor();
    const bool want_x = task_should_compute_output(0), want_w = task_should_compute_output(1), want_b = task_should_compute_output(2);
    if (task_should_compute_output(3)) out[3] = grads[0];
    {
      at::AutoDispatchBelowADInplaceOrView below;
      const int64_t n = w0.size(0), k = w0.size(1);
      const at::Device dev = w0.device();
      const auto type = w0.scalar_type();
      const int dt = dtype_of(type);
      const Tensor wm = matrix(w0, k), xm = matrix(x0, k);
      Tensor g = matrix(grads[0], n);
      const int64_t rows = xm.size(0);
      void* st = stream_of(dev);
      int64_t need_dx = 0, need_dw = 0, need_dz = 0;
      check(L.mg_op_linear_workspace(rows, k, n, dt, nullptr, &need_dx, &need_dw));
      const bool want_dz = act && (want_x || want_w);
      if (want_b || want_dz) {
        if (want_b) {
          out[2] = make({n}, type, dev);
          check(L.mg_op_linear_dz_workspace(rows, n, &need_dz));
        }
        const Scratch ws(need_dz, dev);
        const Tensor dz = want_dz ? make({rows, n}, type, dev) : Tensor();
        check(L.mg_op_linear_dz(dev.index(), st, dt, (int)act, rows, n, ptr(g), row_stride(g), ptr(z0), ptr(dz), ptr(out[2]), ws.p(), ws.bytes));
        if (want_dz) g = dz;
      }
      if (want_x) {
        out[0] = make(x_shape, type, dev);
        const Scratch ws(need_dx, dev);
        check(L.mg_op_linear_dx(dev.index(), st, dt, rows, k, n, ptr(g), row_stride(g), ptr(wm), row_stride(wm), ptr(out[0]), ws.p(), ws.bytes));
      }
      if (want_w) {
        out[1] = make({n, k}, type, dev);
        const Scratch ws(need_dw, dev);
        check(L.mg_op_linear_dw(dev.index(), st, dt, dtype_of(xm.scalar_type()), rows, k, n, ptr(g), row_stride(g), ptr(xm), row_stride(xm), ptr(out[1]), ws.p(), ws.bytes));
      }
    }
    return no_second("linear", std::move(out), {&grads[0], &x0, &w0});
  }
};

Tensor linear(const Tensor& x, const Tensor& w, const MaybeTensor& bias, int64_t act, const MaybeTensor& residual) {
  const Tensor b = bias.value_or(Tensor()), r = residual.value_or(Tensor());
  refuse_tracing("linear");
  refuse_tangents("linear", {&x, &w, &b, &r});
  on_gpu("weight", w);
  const at::Device dev = w.device();
  on_gpu("x", x, dev);
  const auto type = w.scalar_type();
  if (!is_float(type) || w.dim() != 2 || w.numel() == 0) refuse("weight must be (n, k) of float32, bfloat16 or float16, n and k at least 1");
  const int64_t n = w.size(0), k = w.size(1);
  if (x.scalar_type() != type && x.scalar_type() != at::kByte) refuse("x must be ", type, " (weight's dtype) or uint8, got ", x.scalar_type());
  if (x.dim() < 1 || x.size(-1) != k) refuse("x must have ", k, " columns, got shape ", x.sizes());
  if (b.defined()) {
    on_gpu("bias", b, dev);
    if (b.scalar_type() != type || b.dim() != 1 || b.size(0) != n) refuse("bias must be (", n, ",) of ", type);
  }
  const at::DimVector shape = with_last(x.sizes(), n);
  if (r.defined()) {
    on_gpu("residual", r, dev);
    if (r.scalar_type() != type || r.sizes() != at::IntArrayRef(shape)) refuse("residual must be ", at::IntArrayRef(shape), " of ", type, ": the result's shape, nothing is broadcast");
  }
  std::shared_ptr<LinearBackward> node;
  if (at::GradMode::is_enabled() && torch::autograd::compute_requires_grad(x, w, b, r)) {
    refuse_capture_beside_eager(dev, {&x, &w, &b, &r});
    node = std::shared_ptr<LinearBackward>(new LinearBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(x, w, b, r));
  }
  // (relu's slope can be told from its result, which is kept instead unless a residual was added: one store fewer)
  const bool from_y = act == MG_ACTIVATION_RELU && !r.defined();
  Tensor y, xm, wm, z;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    xm = matrix(x, k);
    wm = matrix(w, k);
    const Tensor bc = b.defined() ? values(b).contiguous() : b, rm = r.defined() ? matrix(r, n) : r;
    const int64_t rows = xm.size(0);
    const int dt = dtype_of(type);
    y = make(shape, type, dev);
    if (node && act == MG_ACTIVATION_TANH) act = MG_ACTIVATION_TANH_Z32;
    if (node && act && !from_y) z = make({rows, n}, act == MG_ACTIVATION_TANH_Z32 ? at::kFloat : type, dev);
    int64_t need = 0;
    check(L.mg_op_linear_workspace(rows, k, n, dt, &need, nullptr, nullptr));
    const Scratch ws(need, dev);
    check(L.mg_op_linear(dev.index(), stream_of(dev), dt, dtype_of(xm.scalar_type()), (int)act, rows, k, n, ptr(xm), row_stride(xm), ptr(wm), row_stride(wm), ptr(bc),
                         ptr(rm), rm.defined() ? row_stride(rm) : 0, ptr(y), n, ptr(z), ws.p(), ws.bytes));
  }
  if (node) {
    node->x.put(x, xm);
    node->w.put(w, wm);
    node->act = act;
    node->x_shape = at::DimVector(x.sizes());
    torch::autograd::set_history(y, node);
    if (act) node->z.put(from_y ? y : z, from_y);
  }
  return y;
}

// ---- what the row operators share -----------------------------------------------------------------------------------------------------

// one value per row, contiguous; a constant of the operator
Tensor per_row(const char* name, const Tensor& t, at::IntArrayRef shape, at::Device dev, std::initializer_list<at::ScalarType> types) {
  on_gpu(name, t, dev);
  bool fine = t.sizes() == shape;
  if (fine) fine = std::find(types.begin(), types.end(), t.scalar_type()) != types.end();
  if (!fine) refuse(name, " must be ", shape, " of ", at::ArrayRef<at::ScalarType>(types), ", got ", t.sizes(), " of ", t.scalar_type());
  if (t.requires_grad() && at::GradMode::is_enabled()) refuse(name, " is a constant of this operator and gets no gradient: pass ", name, ".detach()");
  at::AutoDispatchBelowADInplaceOrView below;
  return values(t).contiguous();
}

void check_logits(const Tensor& l) {
  on_gpu("logits", l);
  if (!is_float(l.scalar_type()) || l.dim() < 1 || l.size(-1) < 1) refuse("logits must be (..., actions) of float32, bfloat16 or float16");
}

// ---- policy loss ----------------------------------------------------------------------------------------------------------------------

struct PolicyLossBackward : public Node {
  Kept logits, action, mask, save;
  Tensor ready;                // the gradient for the factor 1, until a backward pass hands it out
  bool masked = false;
  uint64_t capture = 0;        // that the forward pass belongs to
  double ent = 0.0;
  at::DimVector shape;
  std::string name() const override { return "MinigridPolicyLossBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    logits.reset_data();
    action.reset_data();
    mask.reset_data();
    save.reset_data();
    ready = Tensor();
  }
  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    variable_list out(1);
    if (!grads[0].defined() || !task_should_compute_output(0)) return out;
    refuse_tracing("the gradient of policy_loss");
    refuse_tangents("the gradient of policy_loss", {&grads[0]});
    const Tensor l0 = logits.get("logits"), a0 = action.get_contiguous("action"), m0 = masked ? mask.get_contiguous("mask") : Tensor(), s0 = save.get_contiguous("the rows' statistics");
    {
      at::AutoDispatchBelowADInplaceOrView below;
      const Tensor l = matrix(l0, shape.back()), factor = values(grads[0]).contiguous();
      const at::Device dev = l.device();
      // (a pass that is captured behind a forward pass outside of its own capture may be replayed several times behind one forward pass, and would then find
      // what it handed out before, as the caller left it)
      const bool made = ready.defined() && capture == capture_on(dev);
      out[0] = made ? std::move(ready) : make(shape, l.scalar_type(), dev);
      ready = Tensor();
      check((made ? L.mg_op_policy_loss_rescale : L.mg_op_policy_loss_backward)(dev.index(), stream_of(dev), dtype_of(l.scalar_type()), l.size(0), l.size(1), ptr(l), row_stride(l), ptr(a0),
                                         dtype_of(a0.scalar_type()), (const uint8_t*)ptr(m0), ent, ptr(s0), (const float*)ptr(factor), ptr(out[0])));
    }
    return no_second("policy_loss", std::move(out), {&grads[0], &l0});
  }
};

std::pair<Tensor, Tensor> policy_loss(const Tensor& logits, const Tensor& action, const Tensor& old_log_prob, const Tensor& advantage, const MaybeTensor& mask,
                                      const MaybeTensor& ref_log_prob, double lo, double hi, double kl, double ent) {
  const Tensor ref_or_none = ref_log_prob.value_or(Tensor());
  refuse_tracing("policy_loss");
  refuse_tangents("policy_loss", {&logits, &old_log_prob, &advantage, &ref_or_none});
  check_logits(logits);
  const at::Device dev = logits.device();
  if (!(lo >= 0.0 && lo <= 1.0 && hi >= 0.0)) refuse("clip must be a number in 0..1 or a pair (lo, hi) with lo in 0..1 and hi >= 0");
  if (kl != 0.0 && !ref_log_prob) refuse("kl_coef needs ref_log_prob");
  const auto lead = logits.sizes().slice(0, logits.dim() - 1);
  const Tensor a = per_row("action", action, lead, dev, {at::kByte, at::kInt, at::kLong}), old = per_row("old_log_prob", old_log_prob, lead, dev, {at::kFloat}),
               adv = per_row("advantage", advantage, lead, dev, {at::kFloat}), ref = ref_log_prob ? per_row("ref_log_prob", *ref_log_prob, lead, dev, {at::kFloat}) : Tensor(),
               m = mask ? per_row("mask", *mask, lead, dev, {at::kBool, at::kByte}) : Tensor();
  std::shared_ptr<PolicyLossBackward> node;
  if (at::GradMode::is_enabled() && logits.requires_grad()) {
    refuse_capture_beside_eager(dev, {&logits});
    node = std::shared_ptr<PolicyLossBackward>(new PolicyLossBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(logits));
  }
  Tensor l, save, loss, stats, grad;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    l = matrix(logits, logits.size(-1));
    const int64_t rows = l.size(0), vocab = l.size(1);
    const Tensor out = make({6}, at::kFloat, dev);
    if (node) save = make({rows + 1, 2}, at::kDouble, dev);
    // (a half-precision loss is scaled before its backward pass: its gradient for the factor 1 would be made in vain)
    if (node && rows && l.scalar_type() != at::kHalf && L.mg_op_policy_loss_makes_gradient(dtype_of(l.scalar_type()), vocab)) grad = make(logits.sizes(), l.scalar_type(), dev);
    int64_t need = 0;
    check(L.mg_op_policy_loss_workspace(rows, vocab, &need));
    const Scratch ws(need, dev);
    check(L.mg_op_policy_loss_with_gradient(dev.index(), stream_of(dev), dtype_of(l.scalar_type()), rows, vocab, ptr(l), row_stride(l), ptr(a), dtype_of(a.scalar_type()),
                              (const float*)ptr(old), (const float*)ptr(adv), (const float*)ptr(ref), (const uint8_t*)ptr(m), lo, hi, kl, ent, (float*)ptr(out), ptr(save),
                              ws.p(), ws.bytes, ptr(grad)));
    loss = out.select(0, 0);
    stats = out.narrow(0, 1, 5);
  }
  if (node) {
    node->logits.put(logits, l);
    node->action.put(action, a);
    node->masked = m.defined();
    if (m.defined()) node->mask.put(*mask, m);
    node->save.put(save);
    node->ready = grad;
    node->capture = capture_on(dev);
    node->ent = ent;
    node->shape = at::DimVector(logits.sizes());
    torch::autograd::set_history(loss, node);
  }
  return {loss, stats};
}

// ---- sampling -------------------------------------------------------------------------------------------------------------------------

std::pair<Tensor, Tensor> sample_actions(const Tensor& logits, const MaybeTensor& uniform) {
  const Tensor uniform_or_none = uniform.value_or(Tensor());
  refuse_tracing("sample_actions");
  refuse_tangents("sample_actions", {&logits, &uniform_or_none});
  check_logits(logits);
  const at::Device dev = logits.device();
  if (logits.requires_grad() && at::GradMode::is_enabled()) refuse("a draw has no gradient: pass logits.detach(), or call it under torch.no_grad()");
  const auto lead = logits.sizes().slice(0, logits.dim() - 1);
  const Tensor u = uniform ? per_row("uniform", *uniform, lead, dev, {at::kFloat}) : Tensor();
  at::AutoDispatchBelowADInplaceOrView below;
  const Tensor l = matrix(logits, logits.size(-1));
  const int64_t rows = l.size(0), vocab = l.size(1);
  const Tensor action = make(lead, vocab <= 256 ? at::kByte : at::kInt, dev), lp = make(lead, at::kFloat, dev);
  int64_t need = 0;
  check(L.mg_op_sample_workspace(rows, vocab, &need));
  const Scratch ws(need, dev);
  check(L.mg_op_sample(dev.index(), stream_of(dev), dtype_of(l.scalar_type()), rows, vocab, ptr(l), row_stride(l), (const float*)ptr(u), ptr(action), (float*)ptr(lp), ws.p(), ws.bytes));
  return {action, lp};
}

// ---- advantages -----------------------------------------------------------------------------------------------------------------------

std::tuple<Tensor, Tensor, Tensor> advantages(const Tensor& reward, const Tensor& value, const Tensor& last_value, const Tensor& terminated, const Tensor& truncated, double gamma,
                                              double lam, bool next_step, const MaybeTensor& done, const MaybeTensor& final_value) {
  const Tensor final_or_none = final_value.value_or(Tensor());
  refuse_tracing("advantages");
  refuse_tangents("advantages", {&reward, &value, &last_value, &final_or_none});
  on_gpu("value", value);
  const at::Device dev = value.device();
  const auto type = value.scalar_type();
  if (value.dim() != 2 || !is_float(type)) refuse("value must be (steps, envs) of float32, bfloat16 or float16");
  const int64_t steps = value.size(0), envs = value.size(1);
  auto grid = [&](const char* name, const Tensor& t, std::initializer_list<at::ScalarType> types) {
    on_gpu(name, t, dev);
    bool fine = t.sizes() == value.sizes();
    if (fine) fine = std::find(types.begin(), types.end(), t.scalar_type()) != types.end();
    if (!fine) refuse(name, " must be ", value.sizes(), " of ", at::ArrayRef<at::ScalarType>(types), ", got ", t.sizes(), " of ", t.scalar_type());
  };
  grid("reward", reward, {at::kDouble, at::kFloat});
  grid("terminated", terminated, {at::kBool, at::kByte});
  grid("truncated", truncated, {at::kBool, at::kByte});
  if (at::GradMode::is_enabled() && (reward.requires_grad() || value.requires_grad() || last_value.requires_grad() || (final_value && final_value->requires_grad())))
    refuse("the advantages have no gradient: pass detached tensors, or call it under torch.no_grad()");
  const Tensor last = per_row("last_value", last_value, {envs}, dev, {type});
  if (final_value) {
    if (next_step) refuse("final_value belongs to autoreset_mode='same_step': with 'next_step' the rows themselves hold it");
    grid("final_value", *final_value, {type});
  }
  if (done && !next_step) refuse("done belongs to autoreset_mode='next_step'");
  const Tensor d = done ? per_row("done", *done, {envs}, dev, {at::kBool, at::kByte}) : Tensor();
  at::AutoDispatchBelowADInplaceOrView below;
  const Tensor adv = make({steps, envs}, at::kFloat, dev), ret = make({steps, envs}, at::kFloat, dev), valid = make({steps, envs}, at::kBool, dev);
  mg_advantages_args a = {};
  a.steps = steps;
  a.envs = envs;
  auto strides = [](int64_t (&s)[2], const Tensor& t) { s[0] = t.stride(0); s[1] = t.stride(1); };
  const Tensor r = values(reward), v = values(value), f = final_value ? values(*final_value) : Tensor();
  a.reward = ptr(r); strides(a.s_reward, r);
  a.value = ptr(v); strides(a.s_value, v);
  if (f.defined()) { a.final_value = ptr(f); strides(a.s_final, f); }
  a.terminated = (const uint8_t*)ptr(terminated); strides(a.s_term, terminated);
  a.truncated = (const uint8_t*)ptr(truncated); strides(a.s_trunc, truncated);
  a.last_value = ptr(last);
  a.done0 = (const uint8_t*)ptr(d);
  a.advantage = (float*)ptr(adv);
  a.ret = (float*)ptr(ret);
  a.valid = (uint8_t*)ptr(valid);
  a.gamma = gamma;
  a.lam = lam;
  a.reward_dtype = dtype_of(reward.scalar_type());
  a.value_dtype = dtype_of(type);
  a.next_step = next_step;
  check(L.mg_op_advantages(dev.index(), stream_of(dev), &a));
  return {adv, ret, valid};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  const auto unlocked = py::call_guard<py::gil_scoped_release>();
  m.def("bind_library", [](uintptr_t handle, py::object error) {
    bind_library(handle);
    hip_error = error.release().ptr();
  });
  py::register_local_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const HipError& e) {
      PyErr_SetString(hip_error, e.what());
    }
  });
  m.def("linear", &linear, unlocked);
  m.def("policy_loss", &policy_loss, unlocked);
  m.def("sample_actions", &sample_actions, unlocked);
  m.def("advantages", &advantages, unlocked);
}
