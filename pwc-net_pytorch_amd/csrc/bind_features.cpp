// bind_features.cpp — the feature operators' Python binding (module pwcnet_amd._features_ext):
// argument checks, geometry, allocation and autograd nodes over the C ABI.
//
// A call of these operators on a token or a small map is a few microseconds of GPU work; checks
// and autograd nodes in Python cost 13 us forward and 75 to 150 us with the backward pass, most of
// it in the engine's thread.  The entries are reached through the addresses that pwcnet_amd._lib
// loaded (so one library, wherever it lies, serves both bindings).
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include "../../include/pwc_hotpath.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
namespace py = pybind11;

// ---- the C entries ----
#define PWC_ENTRIES(E)                                                                    \
  E(pwc_last_error) E(pwc_rotary)                                                         \
  E(pwc_layer_norm_forward) E(pwc_layer_norm_backward_workspace_size)                     \
  E(pwc_layer_norm_backward)                                                              \
  E(pwc_linear_forward_workspace_size) E(pwc_linear_forward)                              \
  E(pwc_linear_backward_workspace_size) E(pwc_linear_backward)                            \
  E(pwc_gated_linear_forward_workspace_size) E(pwc_gated_linear_forward)                  \
  E(pwc_gated_linear_backward_workspace_size) E(pwc_gated_linear_backward)

struct Entries {
#define E(name) decltype(&::name) name = nullptr;
  PWC_ENTRIES(E)
#undef E
};
Entries g_entries;
std::atomic<bool> g_bound{false};

const Entries& entries() {
  if (!g_bound.load(std::memory_order_acquire)) {
    py::gil_scoped_acquire gil;  // loads the library (or raises) and calls bind()
    py::module_::import("pwcnet_amd.features").attr("_bind")();
  }
  return g_entries;
}

std::vector<std::string> entry_names() {
  return {
#define E(name) #name,
      PWC_ENTRIES(E)
#undef E
  };
}

void bind(const py::dict& at) {  // (under the interpreter's lock: threads that ask at once, once)
  if (g_bound.load(std::memory_order_acquire)) return;
  Entries e;
#define E(name) e.name = reinterpret_cast<decltype(e.name)>(at[#name].cast<uintptr_t>());
  PWC_ENTRIES(E)
#undef E
  g_entries = e;
  g_bound.store(true, std::memory_order_release);
}

void called(int ok, const char* what) {
  TORCH_CHECK(ok == 1, what, " aborting: ", g_entries.pwc_last_error());
}

// ---- checks ----
int dtype_code(at::ScalarType t) {
  return t == at::kFloat ? PWC_DTYPE_F32 : t == at::kHalf ? PWC_DTYPE_F16
       : t == at::kBFloat16 ? PWC_DTYPE_BF16 : -1;
}

// No tensor that stands for others (torch.func's, a subclass with a dispatch of its own): it has no
// memory, or not the values that its caller means.
void plain(const char* what, const Tensor& t) {
  constexpr c10::DispatchKeySet wrapped({c10::DispatchKey::FuncTorchBatched,
                                         c10::DispatchKey::FuncTorchGradWrapper,
                                         c10::DispatchKey::Functionalize, c10::DispatchKey::Python});
  TORCH_CHECK_TYPE(!t.key_set().has_any(wrapped), what,
                   ": plain tensors only: call torch.ops.pwcnet or pwcnet_amd's functions");
}

void check(const char* what, const Tensor& x, std::initializer_list<const Tensor*> others) {
  // torch.jit.trace would record the outputs' allocation and not the launch that fills them
  TORCH_CHECK(!torch::jit::tracer::isTracing(), what,
              ": not seen by torch.jit.trace: call torch.ops.pwcnet or pwcnet_amd's functions");
  auto one = [&](const Tensor& t) {
    plain(what, t);
    TORCH_CHECK(t.is_cuda(), what, ": pwcnet_amd runs on HIP devices only (got a ", t.device(),
                " tensor); there is no CPU implementation");
    TORCH_CHECK(t.device() == x.device(), what, ": tensors on different devices (", t.device(),
                " vs ", x.device(), ")");
    TORCH_CHECK_TYPE(dtype_code(t.scalar_type()) >= 0, what, ": unsupported dtype ",
                     t.scalar_type());
    TORCH_CHECK_TYPE(t.scalar_type() == x.scalar_type(), what, ": mixed dtypes ",
                     t.scalar_type(), " vs ", x.scalar_type());
    TORCH_CHECK_TYPE(t.layout() == at::kStrided, what, ": dense tensors only");
    TORCH_CHECK_TYPE(!t.is_neg(), what, ": negated views are not read: resolve_neg() first");
  };
  one(x);
  for (const Tensor* t : others)
    if (t->defined()) one(*t);
}

Tensor some(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }
const void* ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* out(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
void* stream_of(const Tensor& t) {
  return (void*)c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

// True: tokens [..., C]; false: a map [B, C, *spatial]
bool by_rows(at::IntArrayRef shape, int64_t channel_dim, const char* what) {
  const int64_t n = (int64_t)shape.size();
  TORCH_CHECK_VALUE(n >= 1 && (channel_dim == 1 || channel_dim == -1 || channel_dim == n - 1) &&
                        !(channel_dim == 1 && n < 2),
                    what, ": channel_dim ", channel_dim, " of a tensor of shape ", shape,
                    " (1 for maps [B, C, *spatial], -1 for tokens [..., C])");
  return channel_dim != 1 || n == 2;
}

// x as the C ABI takes it, copied only where its strides are not those of tokens / images a fixed
// distance apart
struct Matrix {
  Tensor x;
  int layout;
  int64_t B, P, C, stride;
};

int64_t row_stride(const Tensor& x, int64_t C) {  // of the joined leading dimensions, or -1
  if (x.numel() == 0 || (C > 1 && x.stride(-1) != 1)) return -1;
  int64_t stride = -1, span = 0;
  for (int64_t d = x.dim() - 2; d >= 0; --d) {
    if (x.size(d) == 1) continue;
    if (stride < 0)
      stride = x.stride(d);
    else if (x.stride(d) != span)
      return -1;
    span = x.stride(d) * x.size(d);
  }
  if (stride < 0) return C;
  return stride >= C ? stride : -1;
}

Matrix matrix(const Tensor& t, bool rows) {
  Matrix m;
  m.x = t;
  if (rows) {
    m.layout = PWC_LAYOUT_TOKENS;
    m.B = 1;
    m.C = t.size(-1);
    m.P = m.C ? t.numel() / m.C : 0;
    m.stride = m.C;
    if (!t.is_contiguous()) {
      m.stride = row_stride(t, m.C);
      if (m.stride < 0) {
        m.x = t.contiguous();
        m.stride = m.C;
      }
    }
    return m;
  }
  m.layout = PWC_LAYOUT_MAP;
  m.B = t.size(0);
  m.C = t.size(1);
  m.P = 1;
  for (int64_t d = 2; d < t.dim(); ++d) m.P *= t.size(d);
  m.stride = m.C * m.P;
  if (!t.is_contiguous()) {
    if (t.numel() && t.stride(0) >= m.C * m.P && t.select(0, 0).is_contiguous())
      m.stride = t.stride(0);
    else
      m.x = t.contiguous();
  }
  return m;
}

Tensor vector(const char* what, const char* name, const Tensor& v, int64_t n) {
  if (!v.defined()) return v;
  TORCH_CHECK_VALUE(v.dim() == 1 && v.size(0) == n, what, ": ", name, " shape ", v.sizes(),
                    " != [", n, "]");
  return v.contiguous();
}

Tensor workspace(size_t bytes, const Tensor& like) {
  return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : Tensor();
}

int to_int(int64_t v, const char* what) {
  TORCH_CHECK_VALUE(v >= INT_MIN && v <= INT_MAX, what, ": argument ", v,
                    " does not fit the C ABI's int");
  return (int)v;
}

// ---- layer norm ----
struct Norm {
  Tensor y, mean, rstd;
};
Norm norm_forward(const Tensor& x, const Tensor& w, const Tensor& b, double eps,
                  int64_t channel_dim, bool stats) {
  const char* what = "LayerNorm";
  check(what, x, {&w, &b});
  const Matrix m = matrix(x, by_rows(x.sizes(), channel_dim, what));
  TORCH_CHECK_VALUE(m.C > 0, what, ": no channels");
  TORCH_CHECK_VALUE(eps >= 0, what, ": eps ", eps, " is negative");
  const Tensor wv = vector(what, "weight", w, m.C), bv = vector(what, "bias", b, m.C);
  c10::DeviceGuard guard(x.device());
  Norm r;
  r.y = at::empty(x.sizes(), x.options());
  if (stats) {
    r.mean = at::empty({m.B * m.P}, x.options().dtype(at::kFloat));
    r.rstd = at::empty({m.B * m.P}, x.options().dtype(at::kFloat));
  }
  if (r.y.numel())
    called(entries().pwc_layer_norm_forward(ptr(m.x), ptr(wv), ptr(bv), out(r.y), out(r.mean), out(r.rstd),
                                  m.layout, m.B, m.P, to_int(m.C, what), m.stride, (float)eps,
                                  dtype_code(x.scalar_type()), stream_of(x)),
           "LayerNorm_forward");
  return r;
}

struct Needs {
  bool x, w, b;
};
struct Grads {
  Tensor x, w, b;
};
Grads norm_backward(const Tensor& x, const Tensor& w, const Tensor& dy, const Tensor& mean,
                    const Tensor& rstd, int64_t channel_dim, Needs needs) {
  const char* what = "LayerNorm backward";
  check(what, x, {&w, &dy});
  TORCH_CHECK_VALUE(dy.sizes() == x.sizes(), what, ": grad_output shape ", dy.sizes(),
                    " != ", x.sizes());
  const Matrix m = matrix(x, by_rows(x.sizes(), channel_dim, what));
  for (const Tensor* t : {&mean, &rstd})
    TORCH_CHECK_VALUE(t->dim() == 1 && t->size(0) == m.B * m.P && t->scalar_type() == at::kFloat &&
                          t->device() == x.device() && t->is_contiguous(),
                      what, ": mean / rstd are not the forward pass's");
  const Tensor g = dy.contiguous(), wv = vector(what, "weight", w, m.C);
  c10::DeviceGuard guard(x.device());
  Grads r;
  if (needs.x) r.x = at::empty(x.sizes(), x.options());
  if (needs.w) r.w = at::empty({m.C}, x.options());
  if (needs.b) r.b = at::empty({m.C}, x.options());
  const Entries& e = entries();
  const int dt = dtype_code(x.scalar_type()), C = to_int(m.C, what);
  const size_t bytes =
      needs.w || needs.b ? e.pwc_layer_norm_backward_workspace_size(m.layout, m.B, m.P, C, dt) : 0;
  const Tensor ws = workspace(bytes, x);
  called(e.pwc_layer_norm_backward(ptr(m.x), ptr(wv), ptr(g), ptr(mean), ptr(rstd), out(r.x), out(r.w),
                         out(r.b), m.layout, m.B, m.P, C, m.stride, dt, out(ws), bytes,
                         stream_of(x)),
         "LayerNorm_backward");
  return r;
}

// ---- rotary positions ----
using OptInts = std::optional<std::vector<int64_t>>;

Tensor rotary_forward(const Tensor& x, const Tensor& inv_freq, const Tensor& axis,
                      const Tensor& positions, const OptInts& grid, const OptInts& origin,
                      bool interleaved, bool inverse) {
  const char* what = "rotary";
  check(what, x, {});
  for (const Tensor* t : {&inv_freq, &axis, &positions})
    if (t->defined()) {
      plain(what, *t);
      TORCH_CHECK_TYPE(!t->is_neg(), what, ": negated views are not read: resolve_neg() first");
    }
  TORCH_CHECK_VALUE(x.dim() == 4, what, ": expected [B, N, heads, D], got shape ", x.sizes());
  TORCH_CHECK_TYPE(inv_freq.scalar_type() == at::kDouble && axis.scalar_type() == at::kInt, what,
                   ": inv_freq is fp64 and axis int32, got ", inv_freq.scalar_type(), " and ",
                   axis.scalar_type());
  const int64_t B = x.size(0), N = x.size(1), R = inv_freq.numel();
  TORCH_CHECK_VALUE(inv_freq.dim() == 1 && axis.sizes() == inv_freq.sizes() && 2 * R <= x.size(3),
                    what, ": inv_freq ", inv_freq.sizes(), " and axis ", axis.sizes(),
                    ": one value for each of at most ", x.size(3) / 2, " pairs");
  pwc_rotary_shape s = {};
  s.B = B;
  s.N = N;
  s.heads = to_int(x.size(2), what);
  s.D = to_int(x.size(3), what);
  s.pairs = to_int(R, what);
  s.interleaved = interleaved;
  TORCH_CHECK_VALUE(positions.defined() != grid.has_value(), what, ": either positions or grid");
  for (const Tensor* t : {&inv_freq, &axis, &positions})
    TORCH_CHECK(!t->defined() || t->device() == x.device(), what,
                ": tensors on different devices (", t->device(), " vs ", x.device(), ")");
  if (positions.defined()) {
    TORCH_CHECK_VALUE(!origin.has_value(), what, ": origin belongs to grid");
    const auto t = positions.scalar_type();
    TORCH_CHECK_TYPE(t == at::kFloat || t == at::kInt || t == at::kLong, what,
                     ": positions are int32, int64 or fp32, got ", t);
    const int64_t n = positions.dim();
    TORCH_CHECK_VALUE((n == 2 || n == 3) && positions.size(-2) == N &&
                          (n == 2 || positions.size(0) == 1 || positions.size(0) == B) &&
                          positions.size(-1) >= 1 && positions.size(-1) <= 4,
                      what, ": positions shape ", positions.sizes(), " for ", B, " x ", N,
                      " tokens and one to four axes");
    s.axes = (int)positions.size(-1);
    s.position_type = t == at::kFloat ? 0 : t == at::kInt ? 1 : 2;
    s.position_stride[0] = n == 2 || positions.size(0) == 1 ? 0 : positions.stride(0);
    s.position_stride[1] = positions.stride(-2);
    s.position_stride[2] = positions.stride(-1);
  } else {
    const size_t axes = grid->size();
    bool ok = axes >= 1 && axes <= 4 && (!origin.has_value() || origin->size() == axes);
    int64_t n = 1;
    for (int64_t g : *grid) {
      ok = ok && g >= 0 && (n == 0 || g <= INT_MAX / n);
      n = ok ? n * g : 0;
    }
    TORCH_CHECK_VALUE(ok && n == N, what, ": grid ", at::IntArrayRef(*grid), " and origin ",
                      origin.has_value() ? at::IntArrayRef(*origin) : at::IntArrayRef(), " for ",
                      N, " tokens");
    s.axes = (int)axes;
    for (size_t k = 0; k < axes; ++k) {
      s.grid[k] = (*grid)[k];
      s.origin[k] = origin.has_value() ? (*origin)[k] : 0;
    }
  }
  c10::DeviceGuard guard(x.device());
  const Tensor f = inv_freq.contiguous(), a = axis.contiguous(), y = at::empty_like(x);
  for (int k = 0; k < 4; ++k) {
    s.x_stride[k] = x.stride(k);
    s.y_stride[k] = y.stride(k);
  }
  if (y.numel())
    called(entries().pwc_rotary(ptr(x), out(y), ptr(positions), ptr(f), ptr(a), &s, inverse,
                            dtype_code(x.scalar_type()), stream_of(x)),
           what);
  return y;
}

// ---- linear and gated linear ----
constexpr const char* kActivations[] = {"none", "relu", "leaky_relu", "sigmoid",
                                        "tanh", "silu", "gelu", "gelu_tanh"};
int64_t activation_code(const std::string& name) {
  for (int k = 0; k < 8; ++k)
    if (name == kActivations[k]) return k;
  TORCH_CHECK_VALUE(false, "unknown activation '", name,
                    "' (one of none, relu, leaky_relu, sigmoid, tanh, silu, gelu, gelu_tanh)");
}

struct Product {
  Matrix m;
  Tensor w, b;
  int O, K;
  std::vector<int64_t> shape;  // of the output
};
Product product(const char* what, const Tensor& x, const Tensor& w, const Tensor& b,
                int64_t channel_dim, bool gated) {
  const bool rows = by_rows(x.sizes(), channel_dim, what);
  const int64_t ch = rows ? x.dim() - 1 : 1;
  TORCH_CHECK_VALUE(w.dim() == 2 && w.size(1) == x.size(ch) && w.numel() > 0, what,
                    ": weight shape ", w.sizes(), " for ", x.size(ch), " channels");
  TORCH_CHECK_VALUE(!gated || w.size(0) % 2 == 0, what,
                    ": weight [gate; up] has an odd number of rows (", w.size(0), ")");
  Product p;
  p.m = matrix(x, rows);
  p.w = w.contiguous();
  p.b = vector(what, "bias", b, w.size(0));
  p.O = to_int(gated ? w.size(0) / 2 : w.size(0), what);
  p.K = to_int(p.m.C, what);
  to_int(p.m.B * p.m.P, what);
  p.shape = x.sizes().vec();
  p.shape[ch] = p.O;
  return p;
}

Tensor product_forward(bool gated, const Tensor& x, const Tensor& w, const Tensor& b,
                       const Tensor& residual, int64_t act, double slope, int64_t channel_dim) {
  const char* what = gated ? "gated_linear" : "linear";
  check(what, x, {&w, &b, &residual});
  const Product p = product(what, x, w, b, channel_dim, gated);
  Tensor res = residual;
  if (res.defined()) {
    TORCH_CHECK_VALUE(res.sizes() == at::IntArrayRef(p.shape), what, ": residual shape ",
                      res.sizes(), " != ", at::IntArrayRef(p.shape));
    res = res.contiguous();
  }
  c10::DeviceGuard guard(x.device());
  const Tensor y = at::empty(p.shape, x.options());
  if (!y.numel()) return y;
  const int dt = dtype_code(x.scalar_type());
  const Matrix& m = p.m;
  const Entries& e = entries();
  const size_t bytes =
      (gated ? e.pwc_gated_linear_forward_workspace_size : e.pwc_linear_forward_workspace_size)(
          ptr(m.x), ptr(p.w), m.layout, m.B, m.P, p.K, p.O, m.stride, dt);
  const Tensor ws = workspace(bytes, x);
  called(gated ? e.pwc_gated_linear_forward(ptr(m.x), ptr(p.w), ptr(p.b), out(y), m.layout, m.B,
                                            m.P, p.K, p.O, m.stride, (int)act, (float)slope, dt,
                                            out(ws), bytes, stream_of(x))
               : e.pwc_linear_forward(ptr(m.x), ptr(p.w), ptr(p.b), ptr(res), out(y), m.layout,
                                      m.B, m.P, p.K, p.O, m.stride, (int)act, (float)slope, dt,
                                      out(ws), bytes, stream_of(x)),
         what);
  return y;
}

Grads product_backward(bool gated, const Tensor& x, const Tensor& w, const Tensor& b,
                       const Tensor& dy, int64_t act, double slope, int64_t channel_dim,
                       Needs needs) {
  const char* what = gated ? "gated_linear backward" : "linear backward";
  check(what, x, {&w, &b, &dy});
  const Product p = product(what, x, w, b, channel_dim, gated);
  TORCH_CHECK_VALUE(dy.sizes() == at::IntArrayRef(p.shape), what, ": grad_output shape ",
                    dy.sizes(), " != ", at::IntArrayRef(p.shape));
  const Tensor g = dy.contiguous();
  c10::DeviceGuard guard(x.device());
  Grads r;
  if (needs.x) r.x = at::empty(x.sizes(), x.options());
  if (needs.w) r.w = at::empty(p.w.sizes(), x.options());
  if (needs.b) r.b = at::empty({p.w.size(0)}, x.options());
  const Entries& e = entries();
  const Matrix& m = p.m;
  const int dt = dtype_code(x.scalar_type());
  const size_t bytes =
      gated ? e.pwc_gated_linear_backward_workspace_size(ptr(m.x), ptr(p.w), ptr(g), m.layout, m.B,
                                                         m.P, p.K, p.O, m.stride, dt)
            : e.pwc_linear_backward_workspace_size(ptr(m.x), ptr(p.w), ptr(g), m.layout, m.B, m.P,
                                                   p.K, p.O, m.stride, (int)act, dt);
  const Tensor ws = workspace(bytes, x);
  const auto call = gated ? e.pwc_gated_linear_backward : e.pwc_linear_backward;
  called(call(ptr(m.x), ptr(p.w), ptr(p.b), ptr(g), out(r.x), out(r.w), out(r.b), m.layout, m.B,
              m.P, p.K, p.O, m.stride, (int)act, (float)slope, dt, out(ws), bytes, stream_of(x)),
         what);
  return r;
}

// ---- autograd ----
bool wants_grad(std::initializer_list<const Tensor*> ts) {
  // forward-mode derivatives go the same way: the node refuses them
  for (const Tensor* t : ts)
    if (t->defined() && t->_fw_grad(0).defined()) return true;
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// The gradients have no graph of their own: asked for one, they raise when it is walked.
Tensor once(Tensor g) {
  if (!g.defined() || !at::GradMode::is_enabled()) return g;
  g = g.detach();
  g.set_requires_grad(true);
  return std::make_shared<torch::autograd::DelayedError>(
             "pwcnet_amd: trying to differentiate twice a function that can be differentiated once",
             1)
      ->apply({g})[0];
}

// which of x, w, b need a gradient, where the missing ones have no edge
Needs needs_of(AutogradContext* ctx, bool w, bool b) {
  Needs n;
  n.x = ctx->needs_input_grad(0);
  n.w = w && ctx->needs_input_grad(1);
  n.b = b && ctx->needs_input_grad(w ? 2 : 1);
  return n;
}

OptTensor opt(const Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; }

struct NormFunction : torch::autograd::Function<NormFunction> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& w,
                        const OptTensor& b, double eps, int64_t channel_dim) {
    Norm r = norm_forward(x, some(w), some(b), eps, channel_dim, true);
    ctx->save_for_backward({x, some(w), r.mean, r.rstd});
    ctx->saved_data["args"] = std::vector<int64_t>{channel_dim, w.has_value(), b.has_value()};
    return r.y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const auto a = ctx->saved_data["args"].toIntVector();
    Grads g = norm_backward(s[0], s[1], grads[0], s[2], s[3], a[0], needs_of(ctx, a[1], a[2]));
    return {once(g.x), once(g.w), once(g.b), Tensor(), Tensor()};
  }
};

struct RotaryFunction : torch::autograd::Function<RotaryFunction> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& inv_freq,
                        const Tensor& axis, const OptTensor& positions, const OptInts& grid,
                        const OptInts& origin, bool interleaved) {
    ctx->save_for_backward({inv_freq, axis, some(positions)});
    if (grid.has_value()) ctx->saved_data["grid"] = *grid;
    if (origin.has_value()) ctx->saved_data["origin"] = *origin;
    ctx->saved_data["interleaved"] = interleaved;
    return rotary_forward(x, inv_freq, axis, some(positions), grid, origin, interleaved, false);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    OptInts grid, origin;
    if (ctx->saved_data.count("grid")) grid = ctx->saved_data["grid"].toIntVector();
    if (ctx->saved_data.count("origin")) origin = ctx->saved_data["origin"].toIntVector();
    const Tensor g = rotary_forward(grads[0], s[0], s[1], s[2], grid, origin,
                                    ctx->saved_data["interleaved"].toBool(), true);
    return {once(g), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

struct LinearFunction : torch::autograd::Function<LinearFunction> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const OptTensor& b,
                        const OptTensor& residual, int64_t act, double slope,
                        int64_t channel_dim) {
    ctx->save_for_backward({x, w, some(b)});
    ctx->saved_data["args"] =
        std::vector<int64_t>{act, channel_dim, b.has_value(), residual.has_value()};
    ctx->saved_data["slope"] = slope;
    return product_forward(false, x, w, some(b), some(residual), act, slope, channel_dim);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const auto a = ctx->saved_data["args"].toIntVector();
    const Needs n = needs_of(ctx, true, a[2]);
    Grads g;
    if (n.x || n.w || n.b)
      g = product_backward(false, s[0], s[1], s[2], grads[0], a[0],
                           ctx->saved_data["slope"].toDouble(), a[1], n);
    const bool res = a[3] && ctx->needs_input_grad(a[2] ? 3 : 2);
    return {once(g.x), once(g.w), once(g.b), res ? grads[0] : Tensor(), Tensor(), Tensor(),
            Tensor()};
  }
};

struct GatedFunction : torch::autograd::Function<GatedFunction> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const OptTensor& b,
                        int64_t act, double slope, int64_t channel_dim) {
    ctx->save_for_backward({x, w, some(b)});
    ctx->saved_data["args"] = std::vector<int64_t>{act, channel_dim, b.has_value()};
    ctx->saved_data["slope"] = slope;
    return product_forward(true, x, w, some(b), Tensor(), act, slope, channel_dim);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const auto a = ctx->saved_data["args"].toIntVector();
    Grads g = product_backward(true, s[0], s[1], s[2], grads[0], a[0],
                               ctx->saved_data["slope"].toDouble(), a[1],
                               needs_of(ctx, true, a[2]));
    return {once(g.x), once(g.w), once(g.b), Tensor(), Tensor(), Tensor()};
  }
};

// ---- what Python calls ----
Tensor layer_norm(const Tensor& x, const OptTensor& w, const OptTensor& b, double eps,
                  int64_t channel_dim) {
  const Tensor wt = some(w), bt = some(b);
  if (wants_grad({&x, &wt, &bt})) return NormFunction::apply(x, w, b, eps, channel_dim);
  return norm_forward(x, wt, bt, eps, channel_dim, false).y;
}

Tensor rotary(const Tensor& x, const Tensor& inv_freq, const Tensor& axis,
              const OptTensor& positions, const OptInts& grid, const OptInts& origin,
              bool interleaved) {
  TORCH_CHECK_VALUE(!positions.has_value() || !positions->requires_grad(),
                    "rotary: positions have no gradient");
  TORCH_CHECK_VALUE(!at::GradMode::is_enabled() || !inv_freq.requires_grad(),
                    "rotary: inv_freq has no gradient");
  if (wants_grad({&x}))
    return RotaryFunction::apply(x, inv_freq, axis, positions, grid, origin, interleaved);
  return rotary_forward(x, inv_freq, axis, some(positions), grid, origin, interleaved, false);
}

Tensor linear(const Tensor& x, const Tensor& w, const OptTensor& b, const OptTensor& residual,
              const std::string& activation, double slope, int64_t channel_dim) {
  const Tensor bt = some(b), rt = some(residual);
  const int64_t act = activation_code(activation);
  if (wants_grad({&x, &w, &bt, &rt}))
    return LinearFunction::apply(x, w, b, residual, act, slope, channel_dim);
  return product_forward(false, x, w, bt, rt, act, slope, channel_dim);
}

Tensor gated_linear(const Tensor& x, const Tensor& w, const OptTensor& b,
                    const std::string& activation, double slope, int64_t channel_dim) {
  const Tensor bt = some(b);
  const int64_t act = activation_code(activation);
  if (wants_grad({&x, &w, &bt})) return GatedFunction::apply(x, w, b, act, slope, channel_dim);
  return product_forward(true, x, w, bt, Tensor(), act, slope, channel_dim);
}

using Three = std::tuple<OptTensor, OptTensor, OptTensor>;
Three three(const Grads& g) { return {opt(g.x), opt(g.w), opt(g.b)}; }
Needs needs_from(const std::tuple<bool, bool, bool>& n) {
  return {std::get<0>(n), std::get<1>(n), std::get<2>(n)};
}

}  // namespace

PYBIND11_MODULE(_features_ext, m) {
  using All = std::tuple<bool, bool, bool>;
  const auto nogil = py::call_guard<py::gil_scoped_release>();
  const All every(true, true, true);
  m.def("bind", &bind);
  m.def("entries", &entry_names);
  m.def("by_rows", [](const std::vector<int64_t>& shape, int64_t dim, const std::string& what) {
    return by_rows(shape, dim, what.c_str());
  });
  m.def("matrix", [](const Tensor& x, bool rows) {
    const Matrix r = matrix(x, rows);
    return std::make_tuple(r.x.is_same(x), r.layout, r.B, r.P, r.C, r.stride);
  });
  m.def("layer_norm", &layer_norm, py::arg("x"), py::arg("weight") = py::none(),
        py::arg("bias") = py::none(), py::arg("eps") = 1e-5, py::arg("channel_dim") = 1, nogil);
  m.def("rotary", &rotary, py::arg("x"), py::arg("inv_freq"), py::arg("axis"),
        py::arg("positions") = py::none(), py::arg("grid") = py::none(),
        py::arg("origin") = py::none(), py::arg("interleaved") = false, nogil);
  m.def("linear", &linear, py::arg("x"), py::arg("weight"), py::arg("bias") = py::none(),
        py::arg("residual") = py::none(), py::arg("activation") = "none",
        py::arg("negative_slope") = 0.1, py::arg("channel_dim") = 1, nogil);
  m.def("gated_linear", &gated_linear, py::arg("x"), py::arg("weight"),
        py::arg("bias") = py::none(), py::arg("activation") = "silu",
        py::arg("negative_slope") = 0.1, py::arg("channel_dim") = 1, nogil);
  // the passes alone
  m.def(
      "layer_norm_forward",
      [](const Tensor& x, const OptTensor& w, const OptTensor& b, double eps, int64_t dim,
         bool stats) {
        const Norm r = norm_forward(x, some(w), some(b), eps, dim, stats);
        return std::make_tuple(r.y, opt(r.mean), opt(r.rstd));
      },
      py::arg("x"), py::arg("weight") = py::none(), py::arg("bias") = py::none(),
      py::arg("eps") = 1e-5, py::arg("channel_dim") = 1, py::arg("stats") = false, nogil);
  m.def(
      "layer_norm_backward",
      [](const Tensor& x, const OptTensor& w, const Tensor& dy, const Tensor& mean,
         const Tensor& rstd, int64_t dim, const All& needs) {
        return three(norm_backward(x, some(w), dy, mean, rstd, dim, needs_from(needs)));
      },
      py::arg("x"), py::arg("weight"), py::arg("grad_out"), py::arg("mean"), py::arg("rstd"),
      py::arg("channel_dim") = 1, py::arg("needs") = every, nogil);
  m.def(
      "rotary_forward",
      [](const Tensor& x, const Tensor& inv_freq, const Tensor& axis, const OptTensor& positions,
         const OptInts& grid, const OptInts& origin, bool interleaved, bool inverse) {
        return rotary_forward(x, inv_freq, axis, some(positions), grid, origin, interleaved,
                              inverse);
      },
      py::arg("x"), py::arg("inv_freq"), py::arg("axis"), py::arg("positions") = py::none(),
      py::arg("grid") = py::none(), py::arg("origin") = py::none(),
      py::arg("interleaved") = false, py::arg("inverse") = false, nogil);
  m.def(
      "linear_forward",
      [](const Tensor& x, const Tensor& w, const OptTensor& b, const OptTensor& res,
         const std::string& act, double slope, int64_t dim) {
        return product_forward(false, x, w, some(b), some(res), activation_code(act), slope, dim);
      },
      py::arg("x"), py::arg("weight"), py::arg("bias") = py::none(),
      py::arg("residual") = py::none(), py::arg("activation") = "none",
      py::arg("negative_slope") = 0.1, py::arg("channel_dim") = 1, nogil);
  m.def(
      "gated_linear_forward",
      [](const Tensor& x, const Tensor& w, const OptTensor& b, const std::string& act,
         double slope, int64_t dim) {
        return product_forward(true, x, w, some(b), Tensor(), activation_code(act), slope, dim);
      },
      py::arg("x"), py::arg("weight"), py::arg("bias") = py::none(),
      py::arg("activation") = "silu", py::arg("negative_slope") = 0.1,
      py::arg("channel_dim") = 1, nogil);
  for (const bool gated : {false, true})
    m.def(
        gated ? "gated_linear_backward" : "linear_backward",
        [gated](const Tensor& x, const Tensor& w, const OptTensor& b, const Tensor& dy,
                const std::string& act, double slope, int64_t dim, const All& needs) {
          return three(product_backward(gated, x, w, some(b), dy, activation_code(act), slope, dim,
                                        needs_from(needs)));
        },
        py::arg("x"), py::arg("weight"), py::arg("bias"), py::arg("grad_out"),
        py::arg("activation") = gated ? "silu" : "none", py::arg("negative_slope") = 0.1,
        py::arg("channel_dim") = 1, py::arg("needs") = every, nogil);
}
