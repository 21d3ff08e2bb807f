// The residual path's binding to PyTorch: tensors in, tensors out, gradients, over the C ABI of
// libtriattn.so (include/triattn.h).  Compiled code instead of ctypes because these operators are short: a
// forward and backward pass through Python functions cost 140 us of host time, several times the kernels'
// own at the usual sizes.  boltz_mlx_b200/residual.py is the public face and checks the numbers (p, seed,
// shared axes); what concerns the tensors is checked here.
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <stdexcept>
#include <string>

#include "triattn.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
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
using Opt = std::optional<Tensor>;
Opt opt(const Tensor& t) { return t.defined() ? Opt(t) : std::nullopt; }  // absent inputs have no edge
// whether the gradient of input `edge` is asked for; edges are counted over the inputs that are there
bool wanted(AutogradContext* ctx, bool there, int& edge) { return there && ctx->needs_input_grad(edge++); }

struct LayerNormFn : torch::autograd::Function<LayerNormFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Opt& w, const Opt& b, double eps,
                        at::ScalarType out_type) {
    const Tensor weight = w.value_or(Tensor()), bias = b.value_or(Tensor());
    Tensor st, out = norm_forward(x, weight, bias, eps, out_type, &st);
    ctx->save_for_backward({x, weight, bias, st});
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    int edge = 0;
    const bool x = wanted(ctx, true, edge), w = wanted(ctx, saved[1].defined(), edge), b = wanted(ctx, saved[2].defined(), edge);
    Gradients g;
    {
      at::AutoGradMode off(false);
      g = norm_backward(grads[0], saved[0], saved[1], saved[2], saved[3], Tensor(), Draw{0.0, 0, 0, Tensor(), 0},
                        {x, false, w, b}, saved[0].scalar_type());
    }
    return once({g.dx, g.dw, g.db, Tensor(), Tensor()});
  }
};

// What a dropout's backward pass keeps of its draw; the seed tensor is saved as a variable, so that a change of
// it in between is found out.
void keep_draw(AutogradContext* ctx, const Draw& d) {
  ctx->saved_data["p"] = d.p;
  ctx->saved_data["seed"] = (int64_t)d.seed;
  ctx->saved_data["offset"] = (int64_t)d.offset;
  ctx->saved_data["share"] = (int64_t)d.share;
}
Draw kept_draw(AutogradContext* ctx, const Tensor& state) {
  return Draw{ctx->saved_data["p"].toDouble(), (uint64_t)ctx->saved_data["seed"].toInt(),
              (uint64_t)ctx->saved_data["offset"].toInt(), state, (int)ctx->saved_data["share"].toInt()};
}

struct DropoutAddFn : torch::autograd::Function<DropoutAddFn> {
  static Tensor forward(AutogradContext* ctx, const Opt& z, const Tensor& y, const Draw& d) {
    ctx->save_for_backward({d.state});
    keep_draw(ctx, d);
    ctx->saved_data["z"] = z.has_value();
    ctx->saved_data["y"] = (int64_t)y.scalar_type();
    return add_forward(z.value_or(Tensor()), y, d, z ? z->scalar_type() : y.scalar_type(), Tensor());
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    int edge = 0;
    const bool z = wanted(ctx, ctx->saved_data["z"].toBool(), edge), y = wanted(ctx, true, edge);
    Tensor dy;
    if (y) {
      at::AutoGradMode off(false);
      dy = add_forward(Tensor(), grads[0], kept_draw(ctx, saved[0]), (at::ScalarType)ctx->saved_data["y"].toInt(), Tensor());
    }
    return once({z ? grads[0] : Tensor(), dy, Tensor()});
  }
};

struct FusedFn : torch::autograd::Function<FusedFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& z, const Tensor& y, const Opt& w, const Opt& b,
                               double eps, const Draw& d, at::ScalarType out_type, bool trans) {
    const Tensor weight = w.value_or(Tensor()), bias = b.value_or(Tensor());
    Tensor st;
    auto [s, h] = fused_forward(z, y, weight, bias, eps, d, out_type, trans, &st);
    ctx->save_for_backward({s, weight, bias, st, d.state});
    keep_draw(ctx, d);
    ctx->saved_data["y"] = (int64_t)y.scalar_type();
    ctx->saved_data["trans"] = trans;
    ctx->set_materialize_grads(false);
    return {s, h};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Draw d = kept_draw(ctx, saved[4]);
    const auto y_type = (at::ScalarType)ctx->saved_data["y"].toInt();
    int edge = 0;
    bool want[4];
    for (int k = 0; k < 4; ++k) want[k] = wanted(ctx, k < 2 || saved[k - 1].defined(), edge);
    const Tensor &ds = grads[0], &dh = grads[1];
    Gradients g;
    {
      at::AutoGradMode off(false);
      if (dh.defined()) {
        g = norm_backward(ctx->saved_data["trans"].toBool() ? dh.transpose(1, 2) : dh, saved[0], saved[1], saved[2], saved[3],
                          ds, d, want, y_type);
      } else {  // the norm's result is not used
        if (want[2]) g.dw = at::zeros_like(saved[1]);
        if (want[3]) g.db = at::zeros_like(saved[2]);
        if (ds.defined()) {
          if (want[0]) g.dx = ds;
          if (want[1]) g.dy = add_forward(Tensor(), ds, d, y_type, Tensor());
        }
      }
    }
    return once({g.dx, g.dy, g.dw, g.db, Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

bool records(std::initializer_list<const Tensor*> ts) {
  if (!c10::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// ---- calls ------------------------------------------------------------------------------------------
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
  on_gpu(what, x0, {&w, &b});
  const Tensor x = x0.scalar_type() != at::kFloat && out != x0.scalar_type() ? x0.to(at::kFloat) : x0;  // exact
  if (records({&x, &w, &b})) return LayerNormFn::apply(x, opt(w), opt(b), eps, out);
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
  on_gpu("dropout", x, {});
  if (records({&x})) return DropoutAddFn::apply(Opt(), x, d);
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
  if (!inplace) return rec ? DropoutAddFn::apply(opt(z), y, d) : add_forward(z, y, d, z.scalar_type(), Tensor());
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
  on_gpu(what, z, {&y0, &w, &b});
  const Tensor y = y0.scalar_type() != z.scalar_type() && y0.scalar_type() != out ? y0.to(at::kFloat) : y0;  // exact
  if (records({&z, &y, &w, &b})) {
    const variable_list r = FusedFn::apply(z, y, opt(w), opt(b), eps, d, out, trans);
    return {r[0], r[1]};
  }
  return fused_forward(z, y, w, b, eps, d, out, trans, nullptr);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
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
