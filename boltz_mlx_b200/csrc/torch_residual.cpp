// The residual path's binding to PyTorch: tensors in, tensors out, gradients, over the C ABI of
// libtriattn.so (include/triattn.h).  Compiled code instead of ctypes because these operators are short: a
// forward and backward pass through Python functions cost 140 us of host time, several times the kernels'
// own at the usual sizes.  boltz_mlx_b200/residual.py is the public face and checks the numbers (p, seed,
// shared axes); what concerns the tensors is checked here.
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <stdexcept>
#include <string>

#include "triattn.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::variable_list;

namespace {

constexpr int64_t kMaxDim = 8192;

// A refusal with a status of the library (the exception classes of _lib.py), or plain ValueError (code 0).
struct Refused : std::runtime_error {
  int code;
  Refused(int c, const std::string& m) : std::runtime_error(m), code(c) {}
};
[[noreturn]] void value_error(const std::string& m) { throw Refused(0, m); }
[[noreturn]] void unsupported(const std::string& m) { throw Refused(TRIATTN_EUNSUPPORTED, m); }
void check(int rc) {
  if (rc != TRIATTN_OK) throw Refused(rc, triattn_last_error_string());
}

std::string str(at::IntArrayRef s) {
  std::string r = "(";
  for (size_t k = 0; k < s.size(); ++k) r += (k ? ", " : "") + std::to_string(s[k]);
  return r + (s.size() == 1 ? ",)" : ")");
}

int code_of(at::ScalarType t, const char* name) {
  switch (t) {
    case at::kFloat: return TRIATTN_F32;
    case at::kHalf: return TRIATTN_F16;
    case at::kBFloat16: return TRIATTN_BF16;
    default: unsupported(std::string(name) + ": " + c10::toString(t) + " (fp32, fp16 and bf16 are supported)");
  }
}
int code_of(const Tensor& t, const char* name) { return code_of(t.scalar_type(), name); }

void on_gpu(const char* what, const Tensor& x, std::initializer_list<const Tensor*> others) {
  if (!x.is_cuda()) throw std::runtime_error(std::string(what) + " (B200) needs CUDA tensors; there is no CPU path");
  for (const Tensor* t : others)
    if (t->defined() && t->device() != x.device())
      value_error(std::string(what) + ": tensors on " + x.device().str() + " and " + t->device().str());
}

// What PyTorch derives from the operators that it sees, it would derive wrongly from these calls, of which it sees the
// allocation of the results alone: a tracer (torch.jit.trace; make_fx, before dispatch as well) would record uninitialised
// memory, fake tensors have no values to work on (an in-place call would change a real one), and a dual tensor's tangent
// would be lost, which counts as zero.
void refuse_derived(const char* what, std::initializer_list<const Tensor*> ts) {
  using Modes = c10::impl::TorchDispatchModeTLS;
  if (torch::jit::tracer::isTracing() || Modes::get_mode(c10::impl::TorchDispatchModeKey::PROXY) ||
      c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch))
    unsupported(std::string(what) + ": tracing");
  if (Modes::get_mode(c10::impl::TorchDispatchModeKey::FAKE)) unsupported(std::string(what) + ": fake tensors");
  for (const Tensor* t : ts)
    if (t->defined() && t->_fw_grad(0).defined())
      unsupported(std::string(what) + ": forward-mode differentiation (an input has a tangent)");
}

// The three leading sizes of a tensor's rows; tensors of more than four axes have their first ones joined.
struct Rows {
  int64_t n[3];
  int64_t rows, dim;
  explicit Rows(const Tensor& t) {
    const auto s = t.sizes();
    const int lead = (int)s.size() - 1;
    n[0] = n[1] = n[2] = 1;
    for (int k = 0; k < lead; ++k) {
      const int at = lead <= 3 ? k + 3 - lead : (k < lead - 2 ? 0 : k - lead + 3);
      n[at] *= s[k];
    }
    rows = n[0] * n[1] * n[2];
    dim = s.back();
  }
};
// A tensor as the library reads it: a dense last axis, strides of the leading ones (null: dense).
struct View {
  Tensor t;
  int64_t s[3] = {0, 0, 0};
  bool strided = false;
  View() = default;
  View(const Tensor& x) : t(x) {
    if (!t.defined() || t.is_contiguous()) return;
    if (t.dim() > 4) {
      auto shape = t.sizes().slice(t.dim() - 4).vec();
      shape[0] = -1;
      t = t.reshape(shape);  // a view where the strides allow it
    }
    if (t.is_contiguous()) return;
    if (t.stride(-1) != 1 && t.size(-1) != 1) {
      t = t.contiguous();
      return;
    }
    strided = true;
    const int lead = (int)t.dim() - 1;
    for (int k = 0; k < lead; ++k) s[k + 3 - lead] = t.stride(k);
  }
  const int64_t* strides() const { return strided ? s : nullptr; }
  void* ptr() const { return t.defined() ? t.data_ptr() : nullptr; }
};
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
float* stat(const Tensor& st, int k) { return st.defined() ? st.data_ptr<float>() + k * st.size(1) : nullptr; }
void* stream_of(const Tensor& t) { return at::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

struct Draw {
  double p;
  uint64_t seed, offset;
  Tensor state;  // int64 (seed, offset) on the device instead of the two, or undefined
  int share;
  const uint64_t* device_state() const {
    return state.defined() ? reinterpret_cast<const uint64_t*>(state.data_ptr<int64_t>()) : nullptr;
  }
};
Draw draw_of(const char* what, const Tensor& x, double p, uint64_t seed, uint64_t offset, const std::optional<Tensor>& state,
             int share) {
  Draw d{p, seed, offset, state.value_or(Tensor()), share};
  if (d.state.defined() && (d.state.scalar_type() != at::kLong || d.state.numel() != 2 || !d.state.is_contiguous() ||
                            d.state.device() != x.device()))
    value_error(std::string(what) + ": a seed tensor holds (seed, offset) as int64 on " + x.device().str());
  return d;
}

void check_params(const char* what, const Tensor& weight, const Tensor& bias, int64_t dim) {
  for (const Tensor* t : {&weight, &bias}) {
    if (!t->defined()) continue;
    code_of(*t, "weight / bias");
    if (t->dim() != 1 || t->size(0) != dim)
      value_error(std::string(what) + ": weight and bias must be [" + std::to_string(dim) + "], got " + str(t->sizes()));
  }
  if (weight.defined() && bias.defined() && weight.scalar_type() != bias.scalar_type())
    value_error(std::string(what) + ": weight and bias have different types");
}
struct Params {
  Tensor w, b;  // dense, or undefined
  int code = TRIATTN_F32;
  Params(const Tensor& weight, const Tensor& bias) {
    if (weight.defined()) w = weight.contiguous();
    if (bias.defined()) b = bias.contiguous();
    if (w.defined() || b.defined()) code = code_of(w.defined() ? w : b, "weight / bias");
  }
};

void check_dim(const char* what, const Tensor& x, int64_t most) {
  if (x.dim() < 1) value_error(std::string(what) + ": a tensor without axes");
  if (x.size(-1) < 1) value_error(std::string(what) + ": no channels");
  if (x.size(-1) > most)
    unsupported(std::string(what) + ": " + std::to_string(x.size(-1)) + " channels (at most " + std::to_string(most) + ")");
}

Tensor empty(at::IntArrayRef shape, at::ScalarType t, const Tensor& like) {
  return at::empty(shape, like.options().dtype(t));
}

// ---- launches ---------------------------------------------------------------------------------------
Tensor norm_forward(const Tensor& x, const Tensor& weight, const Tensor& bias, double eps, at::ScalarType out_type,
                    Tensor* stats) {
  const c10::cuda::CUDAGuard guard(x.device());
  const Rows r(x);
  const View v(x);
  const Params p(weight, bias);
  Tensor out = empty(x.sizes(), out_type, x);
  Tensor st;
  if (stats) st = *stats = empty({2, r.rows}, at::kFloat, x);
  check(triattn_layer_norm(v.ptr(), code_of(x, "x"), v.strides(), r.n, r.dim, ptr(p.w), ptr(p.b), p.code, (float)eps,
                           out.data_ptr(), code_of(out_type, "out_dtype"), nullptr, stat(st, 0), stat(st, 1), stream_of(x)));
  return out;
}

Tensor add_forward(const Tensor& z, const Tensor& y, const Draw& d, at::ScalarType out_type, const Tensor& into) {
  const c10::cuda::CUDAGuard guard(y.device());
  const Rows r(y);
  const View vz(z), vy(y);
  Tensor out = into.defined() ? into : empty(y.sizes(), out_type, y);
  const int oc = code_of(out_type, "out_dtype");
  check(triattn_dropout_add(vz.ptr(), z.defined() ? code_of(z, "z") : oc, vz.strides(), vy.ptr(), code_of(y, "y"), vy.strides(),
                            r.n, r.dim, d.share, d.p, d.seed, d.offset, d.device_state(), out.data_ptr(), oc,
                            into.defined() ? vz.strides() : nullptr, stream_of(y)));
  return out;
}

std::tuple<Tensor, Tensor> fused_forward(const Tensor& z, const Tensor& y, const Tensor& weight, const Tensor& bias,
                                         double eps, const Draw& d, at::ScalarType out_type, bool trans, Tensor* stats) {
  const c10::cuda::CUDAGuard guard(z.device());
  const Rows r(z);
  const View vz(z), vy(y);
  const Params p(weight, bias);
  Tensor s = empty(z.sizes(), z.scalar_type(), z), h, st;
  int64_t hs[3] = {0, 0, 0};
  if (trans) {  // [B, J, I, C], written through the strides of [B, I, J, C]
    h = empty({z.size(0), z.size(2), z.size(1), z.size(3)}, out_type, z);
    hs[0] = h.stride(0);
    hs[1] = h.stride(2);
    hs[2] = h.stride(1);
  } else {
    h = empty(z.sizes(), out_type, z);
  }
  if (stats) st = *stats = empty({2, r.rows}, at::kFloat, z);
  check(triattn_dropout_add_layer_norm(vz.ptr(), code_of(z, "z"), vz.strides(), vy.ptr(), code_of(y, "y"), vy.strides(), r.n,
                                       r.dim, d.share, d.p, d.seed, d.offset, d.device_state(), ptr(p.w), ptr(p.b), p.code,
                                       (float)eps, s.data_ptr(), nullptr, h.data_ptr(), code_of(out_type, "out_dtype"),
                                       trans ? hs : nullptr, stat(st, 0), stat(st, 1), stream_of(z)));
  return {s, h};
}

struct Gradients {
  Tensor dx, dy, dw, db;
};
// want: dx, dy, dweight, dbias
Gradients norm_backward(const Tensor& dout, const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& st,
                        const Tensor& dsum, const Draw& d, const bool (&want)[4], at::ScalarType y_type) {
  const c10::cuda::CUDAGuard guard(x.device());
  const Rows r(x);
  const View vg(dout), vx(x), vs(dsum);
  const Params p(weight, bias);
  Gradients g;
  if (want[0]) g.dx = empty(x.sizes(), x.scalar_type(), x);
  if (want[1]) g.dy = empty(x.sizes(), y_type, x);
  if (want[2]) g.dw = empty({r.dim}, weight.scalar_type(), x);
  if (want[3]) g.db = empty({r.dim}, bias.scalar_type(), x);
  Tensor ws;
  size_t bytes = 0;
  if (want[2] || want[3]) {
    bytes = triattn_layer_norm_backward_workspace_bytes(r.rows, r.dim);
    ws = empty({(int64_t)bytes}, at::kByte, x);
  }
  check(triattn_layer_norm_backward(vg.ptr(), code_of(dout, "gradient"), vg.strides(), vx.ptr(), code_of(x, "x"), vx.strides(),
                                    r.n, r.dim, ptr(p.w), p.code, stat(st, 0), stat(st, 1), vs.ptr(), vs.strides(), d.share,
                                    d.p, d.seed, d.offset, d.device_state(), ptr(g.dx), ptr(g.dy), code_of(y_type, "y"),
                                    ptr(g.dw), ptr(g.db), bytes ? ptr(ws) : nullptr, bytes, stream_of(x)));
  return g;
}

// The gradients are not differentiable: under create_graph they get a node that says so when it is run.
variable_list once(variable_list grads) {
  if (!c10::GradMode::is_enabled()) return grads;
  variable_list defined;
  for (const Tensor& t : grads)
    if (t.defined()) defined.push_back(t.detach().requires_grad_());
  if (defined.empty()) return grads;
  auto stop = std::make_shared<torch::autograd::DelayedError>(
      "the residual operators are differentiable once: their gradients are not", (int64_t)defined.size());
  variable_list marked = (*stop)(std::move(defined));
  size_t k = 0;
  for (Tensor& t : grads)
    if (t.defined()) t = marked[k++];
  return grads;
}

// ---- gradients --------------------------------------------------------------------------------------
// Nodes of the autograd graph, written out: what torch::autograd::Function keeps of every input and looks up by name
// costs 7 us of a training step's 65.
using torch::autograd::Node;
using torch::autograd::SavedVariable;

struct ResidualNode : Node {
  std::vector<SavedVariable> saved;
  void save(std::initializer_list<const Tensor*> inputs) {
    saved.reserve(inputs.size() + 1);
    for (const Tensor* t : inputs) saved.emplace_back(*t, false);
  }
  variable_list unpack() {
    variable_list r;
    r.reserve(saved.size());
    for (SavedVariable& v : saved) r.push_back(v.unpack(shared_from_this()));
    return r;
  }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (SavedVariable& v : saved) v.reset_data();
  }
};
template <class N>
std::shared_ptr<N> make_node(std::initializer_list<Tensor> inputs) {
  std::shared_ptr<N> node(new N(), torch::autograd::deleteNode);
  torch::autograd::edge_list edges;
  edges.reserve(inputs.size());
  for (const Tensor& t : inputs) edges.push_back(t.defined() ? torch::autograd::impl::gradient_edge(t) : torch::autograd::Edge());
  node->set_next_edges(std::move(edges));
  return node;
}

// x, weight, bias -> out
struct LayerNormNode : ResidualNode {
  std::string name() const override { return "ResidualLayerNormBackward"; }
  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    if (!grads[0].defined()) return variable_list(3);
    refuse_derived("layer_norm's backward pass", {&grads[0]});
    Gradients g;
    {
      at::AutoGradMode off(false);
      const variable_list v = unpack();
      g = norm_backward(grads[0], v[0], v[1], v[2], v[3], Tensor(), Draw{0.0, 0, 0, Tensor(), 0},
                        {task_should_compute_output(0), false, task_should_compute_output(1), task_should_compute_output(2)},
                        v[0].scalar_type());
    }
    return once({g.dx, g.dw, g.db});
  }
};

// z, y -> s.  The seed tensor is saved as a variable, so that a change of it before the backward pass is found out.
struct DropoutAddNode : ResidualNode {
  Draw draw;
  at::ScalarType y_type;
  std::string name() const override { return "ResidualDropoutAddBackward"; }
  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    if (!grads[0].defined()) return variable_list(2);
    if (task_should_compute_output(1)) refuse_derived("dropout_add's backward pass", {&grads[0]});
    Tensor dz, dy;
    {
      at::AutoGradMode off(false);
      draw.state = unpack()[0];
      if (task_should_compute_output(0)) dz = grads[0];
      if (task_should_compute_output(1)) dy = add_forward(Tensor(), grads[0], draw, y_type, Tensor());
      draw.state = Tensor();
    }
    return once({dz, dy});
  }
};

// z, y, weight, bias -> s, h
struct FusedNode : ResidualNode {
  Draw draw;
  at::ScalarType y_type;
  bool trans;
  std::string name() const override { return "ResidualDropoutAddLayerNormBackward"; }
  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    const Tensor &ds = grads[0], &dh = grads[1];
    if (!ds.defined() && !dh.defined()) return variable_list(4);
    bool want[4];
    for (int k = 0; k < 4; ++k) want[k] = task_should_compute_output(k);
    if (dh.defined() || want[1]) refuse_derived("dropout_add_layer_norm's backward pass", {&ds, &dh});
    Gradients g;
    {
      at::AutoGradMode off(false);
      const variable_list v = unpack();  // weight, bias, statistics, seed, s
      draw.state = v[3];
      if (dh.defined()) {
        g = norm_backward(trans ? dh.transpose(1, 2) : dh, v[4], v[0], v[1], v[2], ds, draw, want, y_type);
      } else {  // the norm's result is not used
        if (want[2]) g.dw = at::zeros_like(v[0]);
        if (want[3]) g.db = at::zeros_like(v[1]);
        if (want[0]) g.dx = ds;
        if (want[1]) g.dy = add_forward(Tensor(), ds, draw, y_type, Tensor());
      }
      draw.state = Tensor();
    }
    return once({g.dx, g.dy, g.dw, g.db});
  }
};

Tensor norm_recorded(const Tensor& x, const Tensor& weight, const Tensor& bias, double eps, at::ScalarType out_type) {
  auto node = make_node<LayerNormNode>({x, weight, bias});
  Tensor st, out;
  {
    at::AutoGradMode off(false);
    out = norm_forward(x, weight, bias, eps, out_type, &st);
  }
  node->save({&x, &weight, &bias, &st});
  torch::autograd::set_history(out, node);
  return out;
}

Tensor add_recorded(const Tensor& z, const Tensor& y, const Draw& d) {
  auto node = make_node<DropoutAddNode>({z, y});
  Tensor out;
  {
    at::AutoGradMode off(false);
    out = add_forward(z, y, d, z.defined() ? z.scalar_type() : y.scalar_type(), Tensor());
  }
  node->save({&d.state});
  node->draw = d;
  node->draw.state = Tensor();
  node->y_type = y.scalar_type();
  torch::autograd::set_history(out, node);
  return out;
}

std::tuple<Tensor, Tensor> fused_recorded(const Tensor& z, const Tensor& y, const Tensor& weight, const Tensor& bias, double eps,
                                          const Draw& d, at::ScalarType out_type, bool trans) {
  auto node = make_node<FusedNode>({z, y, weight, bias});
  Tensor st, s, h;
  {
    at::AutoGradMode off(false);
    std::tie(s, h) = fused_forward(z, y, weight, bias, eps, d, out_type, trans, &st);
  }
  node->save({&weight, &bias, &st, &d.state});
  node->draw = d;
  node->draw.state = Tensor();
  node->y_type = y.scalar_type();
  node->trans = trans;
  torch::autograd::set_history(s, node);
  torch::autograd::set_history(h, node);
  node->saved.emplace_back(s, true);
  return {s, h};
}

bool records(std::initializer_list<const Tensor*> ts) {
  if (!c10::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// ---- calls ------------------------------------------------------------------------------------------
using Opt = std::optional<Tensor>;
using Type = std::optional<at::ScalarType>;

// What can be said of the arguments anywhere comes first, that they are on a GPU last.
Tensor layer_norm(const Tensor& x0, const Opt& weight, const Opt& bias, double eps, const Type& out_dtype) {
  const char* what = "layer_norm";
  const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor());
  check_dim(what, x0, kMaxDim);
  code_of(x0, "x");
  const at::ScalarType out = out_dtype.value_or(x0.scalar_type());
  code_of(out, "out_dtype");
  check_params(what, w, b, x0.size(-1));
  refuse_derived(what, {&x0, &w, &b});
  on_gpu(what, x0, {&w, &b});
  const Tensor x = x0.scalar_type() != at::kFloat && out != x0.scalar_type() ? x0.to(at::kFloat) : x0;  // exact
  if (records({&x, &w, &b})) return norm_recorded(x, w, b, eps, out);
  return norm_forward(x, w, b, eps, out, nullptr);
}

void check_pair(const char* what, const Tensor& z, const Tensor& y) {
  if (z.sizes() != y.sizes()) value_error(std::string(what) + ": z is " + str(z.sizes()) + ", y " + str(y.sizes()));
  code_of(z, "z");
  code_of(y, "y");
  if (z.scalar_type() != at::kFloat && y.scalar_type() != z.scalar_type())
    unsupported(std::string(what) + ": y is " + c10::toString(y.scalar_type()) + " on a " + c10::toString(z.scalar_type()) +
                " stream");
}

Tensor dropout(const Tensor& x, double p, uint64_t seed, uint64_t offset, const Opt& state, int share) {
  check_dim("dropout", x, 1 << 30);
  code_of(x, "x");
  const Draw d = draw_of("dropout", x, p, seed, offset, state, share);
  refuse_derived("dropout", {&x});
  on_gpu("dropout", x, {});
  if (records({&x})) return add_recorded(Tensor(), x, d);
  return add_forward(Tensor(), x, d, x.scalar_type(), Tensor());
}

// [first, last] byte of a tensor's values
std::pair<const char*, const char*> span(const Tensor& t) {
  int64_t last = 0;
  for (int64_t k = 0; k < t.dim(); ++k) last += (t.size(k) - 1) * t.stride(k);
  const char* p = static_cast<const char*>(t.data_ptr());
  return {p, p + (last + 1) * t.element_size() - 1};
}

Tensor dropout_add(const Tensor& z, const Tensor& y, double p, uint64_t seed, uint64_t offset, const Opt& state, int share,
                   bool inplace) {
  const char* what = "dropout_add";
  check_pair(what, z, y);
  check_dim(what, z, 1 << 30);
  const Draw d = draw_of(what, z, p, seed, offset, state, share);
  refuse_derived(what, {&z, &y});
  const bool rec = records({&z, &y});
  if (inplace && z.numel()) {
    if (rec) throw std::runtime_error("dropout_add: inplace=True keeps no gradients (use torch.no_grad or detach)");
    if (View(z).ptr() != z.data_ptr())
      value_error("dropout_add: inplace=True needs a z with a dense last axis whose leading axes join into three");
    const auto a = span(z), b = span(y);
    const bool same = y.data_ptr() == z.data_ptr() && y.strides() == z.strides() && y.scalar_type() == z.scalar_type();
    if (!same && a.first <= b.second && b.first <= a.second) value_error("dropout_add: inplace=True, and y overlaps z");
  }
  on_gpu(what, z, {&y});
  if (!inplace) return rec ? add_recorded(z, y, d) : add_forward(z, y, d, z.scalar_type(), Tensor());
  if (z.numel() == 0) return z;
  add_forward(z, y, d, z.scalar_type(), z);
  if (!z.is_inference()) z.unsafeGetTensorImpl()->bump_version();
  return z;
}

std::tuple<Tensor, Tensor> dropout_add_layer_norm(const Tensor& z, const Tensor& y0, const Opt& weight, const Opt& bias,
                                                  double p, uint64_t seed, uint64_t offset, const Opt& state, int share,
                                                  double eps, const Type& out_dtype, bool trans) {
  const char* what = "dropout_add_layer_norm";
  const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor());
  check_pair(what, z, y0);
  check_dim(what, z, kMaxDim);
  const at::ScalarType out = out_dtype.value_or(z.scalar_type());
  code_of(out, "out_dtype");
  if (z.scalar_type() != at::kFloat && out != z.scalar_type())
    unsupported(std::string(what) + ": a " + c10::toString(out) + " result of a " + c10::toString(z.scalar_type()) + " stream");
  if (trans && z.dim() != 4) value_error(std::string(what) + ": trans_out needs [B, I, J, C], got " + str(z.sizes()));
  check_params(what, w, b, z.size(-1));
  const Draw d = draw_of(what, z, p, seed, offset, state, share);
  refuse_derived(what, {&z, &y0, &w, &b});
  on_gpu(what, z, {&y0, &w, &b});
  const Tensor y = y0.scalar_type() != z.scalar_type() && y0.scalar_type() != out ? y0.to(at::kFloat) : y0;  // exact
  if (records({&z, &y, &w, &b})) return fused_recorded(z, y, w, b, eps, d, out, trans);
  return fused_forward(z, y, w, b, eps, d, out, trans, nullptr);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.attr("built_for") = RESIDUAL_BUILT_FOR;  // the build looks for it in the file
  m.def("layer_norm", &layer_norm);
  m.def("dropout", &dropout);
  m.def("dropout_add", &dropout_add);
  m.def("dropout_add_layer_norm", &dropout_add_layer_norm);
  py::register_exception_translator([](std::exception_ptr e) {
    try {
      if (e) std::rethrow_exception(e);
    } catch (const Refused& r) {
      if (r.code == 0) {
        PyErr_SetString(PyExc_ValueError, r.what());
        return;
      }
      const char* name = r.code == TRIATTN_EINVAL || r.code == TRIATTN_ENOSPACE ? "TriAttnInvalid"
                         : r.code == TRIATTN_EUNSUPPORTED                       ? "TriAttnUnsupported"
                                                                                : "TriAttnError";
      const py::object cls = py::module_::import("boltz_mlx_b200._lib").attr(name);
      PyErr_SetObject(cls.ptr(), cls(r.code, r.what()).ptr());
    }
  });
}
