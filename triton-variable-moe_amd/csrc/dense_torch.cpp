// The dense operators' entry points as torch calls them: checks of the arguments,
// allocation, autograd, and calls of the C entry points (vmoe.h) on the current stream
// of x's device. kernels/dense.py documents the operators; its functions call these.
//
// Compiled because small calls are bound by host work: through ctypes and Python
// autograd functions a layer norm of one token took 9.1 us and a training pass of 4101
// rows 117 us, with 4 and 24 us of kernels.

#include <Python.h>
#include <dlfcn.h>

#include <ATen/ATen.h>
#include <c10/core/InferenceMode.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>

#include <map>
#include <mutex>

#include "vmoe.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> Maybe;

constexpr int64_t kMaxLd = 1 << 20;  // the C entry points' limit

// AssertionError, as the package's other operators raise for tensors on the host.
struct NotOnGpu {
  std::string what;
};

// ---------------------------------------------------------------------------
// Calls of the library: the one that the package has loaded (use(), below), which need
// not be the one beside this module.

#define VMOE_ENTRIES(ENTRY)                                                          \
  ENTRY(vmoe_status_string)                                                          \
  ENTRY(vmoe_layer_norm_max)                                                         \
  ENTRY(vmoe_layer_norm)                                                             \
  ENTRY(vmoe_layer_norm_workspace_bytes)                                             \
  ENTRY(vmoe_layer_norm_backward)                                                    \
  ENTRY(vmoe_dense_arrival_words)                                                    \
  ENTRY(vmoe_linear_workspace_bytes)                                                 \
  ENTRY(vmoe_linear_forward)                                                         \
  ENTRY(vmoe_linear_backward)                                                        \
  ENTRY(vmoe_gated_workspace_bytes)                                                  \
  ENTRY(vmoe_gated_forward)                                                          \
  ENTRY(vmoe_gated_backward)

struct Library {
  bool loaded = false;
#define VMOE_ENTRY(name) decltype(&::name) name = nullptr;
  VMOE_ENTRIES(VMOE_ENTRY)
#undef VMOE_ENTRY
} lib;

PyObject* g_timer = nullptr;  // observer of launches (begin(name), end(name)), or null

void observe(const char* method, const char* name) {
  struct Gil {
    PyGILState_STATE state = PyGILState_Ensure();
    ~Gil() { PyGILState_Release(state); }
  } gil;
  if (!g_timer) return;
  PyObject* r = PyObject_CallMethod(g_timer, method, "s", name);
  if (!r) {  // the observer's own error, for the caller
    python_error error;
    error.persist();
    throw error;
  }
  Py_DECREF(r);
}

template <typename F>
void call(const char* name, F&& f) {
  const bool seen = g_timer != nullptr;
  if (seen) observe("begin", name);
  const int status = f();
  if (seen) observe("end", name);
  if (status == VMOE_OK) return;
  const char* what = lib.vmoe_status_string(status);
  TORCH_CHECK_NOT_IMPLEMENTED(status != VMOE_ERR_UNSUPPORTED, name, ": ", what);
  TORCH_CHECK_VALUE(status != VMOE_ERR_INVALID_ARG, name, ": ", what);
  TORCH_CHECK(false, name, ": ", what, " (status ", status, ")");
}

vmoe_stream_t stream_of(const Tensor& x) {
  return reinterpret_cast<vmoe_stream_t>(c10::hip::getCurrentHIPStream(x.get_device()).stream());
}

// The current stream's arrival words, for products of few rows (which alone use them):
// zero-filled once, and every call leaves them zero. Calls on one stream run in order,
// so they share them. A captured call gets none: its graph may be replayed on any
// stream, beside calls or graphs of the one it was captured on.
uint32_t* words_of(const Tensor& x, int64_t rows, size_t workspace_bytes) {
  if (rows > 64 || !workspace_bytes) return nullptr;
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None)
    return nullptr;
  static std::mutex& lock = *new std::mutex;  // (never destroyed: nor is the memory freed
  static auto& all = *new std::map<std::pair<int64_t, int64_t>, Tensor>;  // at exit)
  const std::pair<int64_t, int64_t> key(x.get_device(),
                                        c10::hip::getCurrentHIPStream(x.get_device()).id());
  const std::lock_guard<std::mutex> held(lock);
  Tensor& t = all[key];
  if (!t.defined()) {
    const c10::InferenceMode normal(false);
    t = at::zeros({lib.vmoe_dense_arrival_words()}, x.options().dtype(at::kInt));
  }
  return static_cast<uint32_t*>(t.mutable_data_ptr());
}

// ---------------------------------------------------------------------------
// Arguments.

void check_type(const Tensor& t, const char* what) {
  TORCH_CHECK_NOT_IMPLEMENTED(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat, what,
                              " must be bfloat16 or float32 (got ", t.scalar_type(), ")");
  TORCH_CHECK_NOT_IMPLEMENTED(t.layout() == at::kStrided, what, " must be a strided tensor");
}
// A tensor's values may be elsewhere (a wrapper's, such as a distributed tensor's) or
// gone (a freed storage): its address is then no address, and the C entry points read
// NULL as "not given".
bool in_memory(const Tensor& t) {
  if (t.numel() == 0) return true;
  if (!t.has_storage()) return false;
  const at::Storage& s = t.storage();
  return s.data() && at::detail::computeStorageNbytes(t.sizes(), t.strides(), t.element_size(),
                                                      t.storage_offset()) <= s.nbytes();
}
void check_memory(const Tensor& t, const char* what) {
  TORCH_CHECK_NOT_IMPLEMENTED(in_memory(t), what, " has no memory here (the values of a wrapper, or "
                              "a storage that was freed)");
}
// x, after the checks that need no device
void check_device(const Tensor& x) {
  if (!x.is_cuda()) throw NotOnGpu{"x must be on CUDA"};
  check_memory(x, "x");
}
void check_like(const Tensor& t, const char* what, const Tensor& x) {
  TORCH_CHECK_VALUE(t.scalar_type() == x.scalar_type(), what, " must have x's type, ",
                    x.scalar_type(), " (got ", t.scalar_type(), ")");
  TORCH_CHECK_VALUE(t.device() == x.device(), what, " must be on x's device, ", x.device(),
                    " (got ", t.device(), ")");
  TORCH_CHECK_NOT_IMPLEMENTED(t.layout() == at::kStrided, what, " must be a strided tensor");
  check_memory(t, what);
}
void check_vector(const Maybe& v, const char* what, int64_t n, const Tensor& x) {
  if (!v) return;
  TORCH_CHECK_VALUE(v->dim() == 1 && v->size(0) == n, what, " must have shape (", n, ",) (got ",
                    v->sizes(), ")");
  check_type(*v, what);
  TORCH_CHECK_VALUE(v->device() == x.device(), what, " must be on x's device, ", x.device(),
                    " (got ", v->device(), ")");
  check_memory(*v, what);
}
void check_residual(const Maybe& r, at::IntArrayRef shape, const Tensor& x) {
  if (!r) return;
  TORCH_CHECK_VALUE(r->sizes() == shape, "residual must have the output's shape ", shape, " (got ",
                    r->sizes(), ")");
  check_like(*r, "residual", x);
}
void check_features(const Tensor& x, int64_t n, const char* what) {
  const int64_t mult = 16 / (int64_t)x.element_size();
  TORCH_CHECK_VALUE(n > 0, what, " must not be empty");
  TORCH_CHECK_NOT_IMPLEMENTED(n % mult == 0, what, " must be a multiple of ", mult, " for ",
                              x.scalar_type(), " (got ", n, ")");
}
// Nothing here knows tangents: a call would drop them.
void check_tangent(const Maybe& t) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t || !t->_fw_grad(0).defined(),
                              "forward-mode derivatives are not supported");
}

int type_of(const Tensor& x) {
  return x.scalar_type() == at::kFloat ? VMOE_DENSE_F32 : VMOE_DENSE_BF16;
}
int f32(const Maybe& v) { return v && v->scalar_type() == at::kFloat; }
const void* ptr(const Maybe& v) { return v ? v->const_data_ptr() : nullptr; }
// What a forward pass has saved.
const void* saved_ptr(const Tensor& v) {
  if (!v.defined()) return nullptr;
  check_memory(v, "a saved tensor");
  return v.const_data_ptr();
}
const float* saved_floats(const Tensor& v) { return static_cast<const float*>(saved_ptr(v)); }
void* out_ptr(const Tensor& v) { return v.defined() ? v.mutable_data_ptr() : nullptr; }
bool aligned(const Tensor& t) { return (reinterpret_cast<uintptr_t>(t.const_data_ptr()) & 15) == 0; }

// A matrix as the kernels read it: element (i, j) at i ld + j (transposed: j ld + i).
struct Mat {
  Tensor t;  // keeps the memory
  int64_t ld = 0;
  int tr = 0;
  const void* p() const { return t.defined() ? t.const_data_ptr() : nullptr; }
};

Tensor fresh(const Tensor& t) { return t.clone(at::MemoryFormat::Contiguous); }
// A view that stands for its negative, as of a conjugate's imaginary part, gets memory
// of its own. (The check again: backward passes read saved tensors and a given gradient.)
Tensor plain(const Tensor& t) {
  check_memory(t, "an operand");
  return t.is_neg() ? t.resolve_neg() : t;
}

// t as rows of `cols` values, contiguous and 16-byte aligned: in place, or a copy.
Mat rows_of(const Tensor& given, int64_t cols) {
  const Tensor t = plain(given);
  Mat m;
  m.t = t.dim() == 2 ? t : t.reshape({-1, cols});
  const int64_t mult = 16 / (int64_t)t.element_size();
  auto fits = [&](const Tensor& q) {
    const int64_t ld = q.stride(0);
    return q.stride(1) == 1 && ld % mult == 0 && ld >= cols && ld <= kMaxLd && aligned(q);
  };
  if (!fits(m.t)) m.t = fresh(m.t);
  m.ld = m.t.size(0) > 1 ? m.t.stride(0) : cols;
  return m;
}

// A weight [in, out]: in place in either order, or a copy in the nearer one.
bool in_order(const Tensor& w, int tr) {  // whether it is read in place
  const int64_t ld = w.stride(tr), mult = 16 / (int64_t)w.element_size();
  return w.stride(1 - tr) == 1 && ld >= w.size(1 - tr) && ld % mult == 0 && ld <= kMaxLd && aligned(w);
}
int weight_order(const Tensor& w) {
  if (in_order(w, 0)) return 0;
  return in_order(w, 1) || (w.stride(0) == 1 && w.stride(1) != 1);
}
Mat weight_of(const Tensor& given, int order = -1) {  // (0 or 1: in that order)
  const Tensor w = plain(given);
  Mat m;
  m.tr = order < 0 ? weight_order(w) : order;
  if (in_order(w, m.tr)) {
    m.t = w;
    m.ld = w.stride(m.tr);
  } else {
    m.t = fresh(m.tr ? w.t() : w);
    m.ld = m.t.size(1);
  }
  return m;
}

// Rows of a norm: contiguous, at any distance (0: one row for all).
Mat norm_rows(const Tensor& given, int64_t d) {
  const Tensor t = plain(given);
  Mat m;
  m.t = t.dim() == 2 ? t : t.reshape({-1, d});
  const int64_t rows = m.t.size(0), s = m.t.stride(0);
  if ((m.t.stride(1) != 1 && d > 1) || (rows > 1 && s < d && s != 0)) m.t = fresh(m.t);
  m.ld = rows > 1 ? m.t.stride(0) : d;
  return m;
}

Maybe contiguous(const Maybe& given) {
  if (!given) return given;
  const Tensor v = plain(*given);
  return v.numel() < 2 || v.stride(0) == 1 ? v : v.contiguous();
}

Tensor empty(at::IntArrayRef shape, const Tensor& x) { return at::empty(shape, x.options()); }
Tensor empty_f32(at::IntArrayRef shape, const Tensor& x) {
  return at::empty(shape, x.options().dtype(at::kFloat));
}
Tensor workspace(size_t bytes, const Tensor& x) {
  return bytes ? at::empty({(int64_t)bytes}, x.options().dtype(at::kByte)) : Tensor();
}
// Uninitialised gradients: of a vector, and of a weight [in, out] in the order the
// kernels read it.
Tensor vector_grad(int64_t n, bool f32, const Tensor& gy) {
  return f32 ? empty_f32({n}, gy) : at::empty({n}, gy.options().dtype(at::kBFloat16));
}
Tensor weight_grad(int64_t in, int64_t out, int tr, const Tensor& gy) {
  return tr ? empty({out, in}, gy).t() : empty({in, out}, gy);
}
int64_t ld_of(const Tensor& g, int tr) {
  return !g.defined() ? 0 : tr ? g.size(0) : g.size(1);
}
void zero(std::initializer_list<Tensor> ts) {
  for (const Tensor& t : ts)
    if (t.defined()) const_cast<Tensor&>(t).zero_();
}

bool recorded(std::initializer_list<const Maybe*> ts) {
  bool any = false;
  for (const Maybe* t : ts) {
    check_tangent(*t);
    any = any || (*t && (*t)->requires_grad());
  }
  return any && at::GradMode::is_enabled();
}

// Gradients as autograd gets them. Where they are recorded themselves (create_graph),
// differentiating them raises.
variable_list gradients(variable_list g) {
  if (!at::GradMode::is_enabled()) return g;
  variable_list in;
  for (const Tensor& t : g)
    if (t.defined()) in.push_back(t.detach().requires_grad_(true));
  if (in.empty()) return g;
  auto delayed = std::make_shared<torch::autograd::DelayedError>(
      "the dense operators' gradients cannot be differentiated again", (int64_t)in.size());
  const variable_list out = (*delayed)(std::move(in));
  size_t i = 0;
  for (Tensor& t : g)
    if (t.defined()) t = out[i++];
  return g;
}

// A forward pass saves what the gradients that can be asked for read, and no more: no
// pre-activations for a residual's gradient, no rows where the weight has none, no bias.
bool wants(const Tensor& t) { return t.requires_grad(); }
bool wants(const Maybe& t) { return t && t->requires_grad(); }
Tensor keep(bool read, const Tensor& t) { return read ? t : Tensor(); }
Tensor keep(bool read, const Maybe& t) { return read && t ? *t : Tensor(); }

// What else a backward pass has to know of its operands, in one value.
struct How {
  bool vector1 = false, vector1_f32 = false;  // a bias (a norm's weight): given, its type
  bool vector2 = false, vector2_f32 = false;  // the second one (a norm's bias)
  bool residual = false;
  bool tr1 = false, tr2 = false;  // weights' orders
  int act = 0;
  int64_t size = 0;  // of a weight: linear's in, a gated block's width
  void save(AutogradContext* ctx) const {
    ctx->saved_data["how"] = size << 16 | act << 8 | vector1 | vector1_f32 << 1 | vector2 << 2 |
                             vector2_f32 << 3 | residual << 4 | tr1 << 5 | tr2 << 6;
  }
  static How of(const AutogradContext* ctx) {
    const int64_t v = ctx->saved_data.at("how").toInt();
    return {bool(v & 1),  bool(v & 2),  bool(v & 4),          bool(v & 8), bool(v & 16),
            bool(v & 32), bool(v & 64), int(v >> 8 & 0xFF), v >> 16};
  }
};

// Which of an operator's tensors need gradients. (Autograd counts the given ones.)
template <size_t N>
std::array<bool, N> needs(const AutogradContext* ctx, const std::array<bool, N>& given) {
  std::array<bool, N> need;
  size_t edge = 0;
  for (size_t i = 0; i < N; ++i) need[i] = given[i] && ctx->needs_input_grad(edge++);
  return need;
}

// ---------------------------------------------------------------------------
// Layer norm.

Tensor norm_forward(const Tensor& x, const Maybe& w_, const Maybe& b_, double eps, Tensor* stats) {
  const c10::DeviceGuard on(x.device());
  const int64_t d = x.size(-1);
  const Mat m = norm_rows(x, d);
  const int64_t rows = m.t.size(0);
  const Maybe w = contiguous(w_), b = contiguous(b_);
  Tensor y = empty(x.sizes(), x);
  if (stats) *stats = empty_f32({rows, 2}, x);
  call("vmoe_layer_norm", [&] {
    return lib.vmoe_layer_norm(type_of(x), m.p(), m.ld, rows, d, ptr(w), f32(w), ptr(b), f32(b),
                               (float)eps, y.mutable_data_ptr(), d,
                               stats ? static_cast<float*>(stats->mutable_data_ptr()) : nullptr,
                               stream_of(x));
  });
  return y;
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Maybe& w, const Maybe& b,
                        double eps) {
    Tensor stats;
    Tensor y = norm_forward(x, w, b, eps, &stats);
    ctx->save_for_backward({x, keep(wants(x), w), stats});
    How{w.has_value(), bool(f32(w)), b.has_value(), bool(f32(b))}.save(ctx);
    return y;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& gys) {
    variable_list out(4);
    {
      const at::AutoGradMode off(false);
      const variable_list s = ctx->get_saved_variables();
      const Tensor &x = s[0], &stats = s[2], &gy = gys[0];
      const How how = How::of(ctx);
      const Maybe w = s[1].defined() ? contiguous(s[1]) : Maybe();
      const auto need = needs<3>(ctx, {true, how.vector1, how.vector2});
      const c10::DeviceGuard on(x.device());
      const int64_t d = x.size(-1), rows = stats.size(0);
      Tensor gx, gw, gb;
      if (need[0]) gx = empty(x.sizes(), x);
      if (need[1]) gw = vector_grad(d, how.vector1_f32, gy);
      if (need[2]) gb = vector_grad(d, how.vector2_f32, gy);
      if (rows == 0) {
        zero({gw, gb});
      } else {
        const Mat m = norm_rows(x, d), g = norm_rows(gy, d);
        const size_t n = need[1] || need[2] ? lib.vmoe_layer_norm_workspace_bytes(rows, d) : 0;
        const Tensor ws = workspace(n, x);
        call("vmoe_layer_norm_backward", [&] {
          return lib.vmoe_layer_norm_backward(
              type_of(x), g.p(), g.ld, m.p(), m.ld, rows, d, ptr(w), f32(w), saved_floats(stats),
              out_ptr(gx), d, out_ptr(gw), how.vector1_f32, out_ptr(gb), how.vector2_f32,
              out_ptr(ws), n, stream_of(x));
        });
      }
      out[0] = gx;
      out[1] = gw;
      out[2] = gb;
    }
    return gradients(std::move(out));
  }
};

Tensor layer_norm(const Tensor& x, const Maybe& w, const Maybe& b, double eps) {
  check_type(x, "x");
  TORCH_CHECK_VALUE(x.dim() > 0, "x must have at least one dimension");
  const int64_t d = x.size(-1);
  TORCH_CHECK_VALUE(d > 0, "the last dimension of x must not be empty");
  TORCH_CHECK_NOT_IMPLEMENTED(d <= lib.vmoe_layer_norm_max(), "rows of at most ", lib.vmoe_layer_norm_max(),
                              " values (got ", d, ")");
  check_vector(w, "weight", d, x);
  check_vector(b, "bias", d, x);
  check_device(x);
  const Maybe mx = x;
  if (recorded({&mx, &w, &b})) return LayerNorm::apply(x, w, b, eps);
  return norm_forward(x, w, b, eps, nullptr);
}

// ---------------------------------------------------------------------------
// Linear layer with a fused epilogue.

Tensor linear_forward(const Tensor& x, const Tensor& w, const Maybe& b_, const Maybe& r, int act,
                      Tensor* z) {
  const c10::DeviceGuard on(x.device());
  const int64_t in = w.size(0), out = w.size(1);
  const Mat m = rows_of(x, in), wm = weight_of(w);
  const Mat rm = r ? rows_of(*r, out) : Mat();
  const Maybe b = contiguous(b_);
  const int64_t rows = m.t.size(0);
  at::DimVector shape(x.sizes());
  shape.back() = out;
  Tensor y = empty(shape, x);
  if (z) *z = empty_f32({rows, out}, x);
  const int type = type_of(x);
  const size_t n = lib.vmoe_linear_workspace_bytes(type, rows, in, out, act, 0);
  const Tensor ws = workspace(n, x);
  call("vmoe_linear_forward", [&] {
    return lib.vmoe_linear_forward(type, m.p(), m.ld, rows, in, out, wm.p(), wm.ld, wm.tr, ptr(b),
                                   f32(b), act, rm.p(), rm.ld, y.mutable_data_ptr(), out,
                                   z ? static_cast<float*>(z->mutable_data_ptr()) : nullptr,
                                   out_ptr(ws), n, words_of(x, rows, n), stream_of(x));
  });
  return y;
}

struct FusedLinear : torch::autograd::Function<FusedLinear> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Maybe& b,
                        const Maybe& r, int64_t act) {
    const bool slope = act && (wants(x) || wants(w) || wants(b));
    // relu's slope follows from the output, unless a residual is in it
    const bool from_y = !r && act == VMOE_DENSE_RELU;
    Tensor z;
    Tensor y = linear_forward(x, w, b, r, (int)act, slope && !from_y ? &z : nullptr);
    ctx->save_for_backward({keep(wants(w), x), keep(wants(x), w), z, keep(slope && from_y, y)});
    How{b.has_value(), bool(f32(b)), false, false, r.has_value(),
        bool(weight_order(plain(w))), false, (int)act, w.size(0)}.save(ctx);
    return y;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& gys) {
    variable_list out(5);
    const How how = How::of(ctx);
    {
      const at::AutoGradMode off(false);
      const variable_list s = ctx->get_saved_variables();
      const Tensor &x = s[0], &w = s[1], &z = s[2], &y = s[3], &gy = gys[0];
      const auto need = needs<4>(ctx, {true, true, how.vector1, how.residual});
      if (need[0] || need[1] || need[2]) {
        const c10::DeviceGuard on(gy.device());
        const int64_t in = how.size, n_out = gy.size(-1);
        Tensor gx, gw, gb;
        if (need[0]) {
          at::DimVector shape(gy.sizes());
          shape.back() = in;
          gx = empty(shape, gy);
        }
        if (need[1]) gw = weight_grad(in, n_out, how.tr1, gy);
        if (need[2]) gb = vector_grad(n_out, how.vector1_f32, gy);
        if (gy.numel() == 0) {
          zero({gw, gb});
        } else {
          const Mat g = rows_of(gy, n_out);
          const Mat m = need[1] ? rows_of(x, in) : Mat(), wm = need[0] ? weight_of(w, how.tr1) : Mat();
          const int64_t rows = g.t.size(0);
          const int type = type_of(gy);
          const size_t n = lib.vmoe_linear_workspace_bytes(type, rows, in, n_out, how.act, 1);
          const Tensor ws = workspace(n, gy);
          call("vmoe_linear_backward", [&] {
            return lib.vmoe_linear_backward(
                type, g.p(), g.ld, m.p(), m.ld, rows, in, n_out, wm.p(), wm.ld, how.tr1, how.act,
                saved_floats(z), saved_ptr(y), n_out, out_ptr(gx), in, out_ptr(gw),
                ld_of(gw, how.tr1), out_ptr(gb), how.vector1_f32, out_ptr(ws), n, stream_of(gy));
          });
        }
        out[0] = gx;
        out[1] = gw;
        out[2] = gb;
      }
    }
    out = gradients(std::move(out));
    if (how.residual) out[3] = gys[0];
    return out;
  }
};

Tensor fused_linear(const Tensor& x, const Tensor& w, const Maybe& b, const Maybe& r, int act) {
  check_type(x, "x");
  TORCH_CHECK_VALUE(x.dim() > 0 && w.dim() == 2 && x.size(-1) == w.size(0),
                    "x [..., in] and weight [in, out] do not fit: ", x.sizes(), ", ", w.sizes());
  check_features(x, w.size(0), "in");
  check_features(x, w.size(1), "out");
  check_like(w, "weight", x);
  check_vector(b, "bias", w.size(1), x);
  at::DimVector shape(x.sizes());
  shape.back() = w.size(1);
  check_residual(r, shape, x);
  check_device(x);
  const Maybe mx = x, mw = w;
  if (recorded({&mx, &mw, &b, &r})) return FusedLinear::apply(x, w, b, r, (int64_t)act);
  return linear_forward(x, w, b, r, act, nullptr);
}

// ---------------------------------------------------------------------------
// Gated block.

Tensor gated_forward(const Tensor& x, const Tensor& w1, const Tensor& w2, const Maybe& b1_,
                     const Maybe& b2_, const Maybe& r, int act, Tensor& h, Tensor* z) {
  const c10::DeviceGuard on(x.device());
  const int64_t width = w2.size(0), d = w2.size(1);
  const Mat m = rows_of(x, d), m1 = weight_of(w1), m2 = weight_of(w2);
  const Mat rm = r ? rows_of(*r, d) : Mat();
  const Maybe b1 = contiguous(b1_), b2 = contiguous(b2_);
  const int64_t rows = m.t.size(0);
  Tensor y = empty(x.sizes(), x);
  h = empty({rows, width}, x);
  if (z) *z = empty_f32({rows, 2 * width}, x);
  const int type = type_of(x);
  const size_t n = lib.vmoe_gated_workspace_bytes(type, rows, d, width, 0);
  const Tensor ws = workspace(n, x);
  call("vmoe_gated_forward", [&] {
    return lib.vmoe_gated_forward(type, m.p(), m.ld, rows, d, width, m1.p(), m1.ld, m1.tr, ptr(b1),
                                  f32(b1), act, m2.p(), m2.ld, m2.tr, ptr(b2), f32(b2), rm.p(), rm.ld,
                                  h.mutable_data_ptr(),
                                  z ? static_cast<float*>(z->mutable_data_ptr()) : nullptr,
                                  y.mutable_data_ptr(), d, out_ptr(ws), n, words_of(x, rows, n),
                                  stream_of(x));
  });
  return y;
}

struct GatedMLP : torch::autograd::Function<GatedMLP> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w1, const Tensor& w2,
                        const Maybe& b1, const Maybe& b2, const Maybe& r, int64_t act) {
    const bool inner = wants(x) || wants(w1) || wants(b1);  // what needs the gradients of g and u
    Tensor h, z;
    Tensor y = gated_forward(x, w1, w2, b1, b2, r, (int)act, h, inner ? &z : nullptr);
    ctx->save_for_backward({keep(wants(w1), x), keep(wants(x), w1), keep(inner, w2),
                            keep(wants(w2), h), z});
    How{b1.has_value(), bool(f32(b1)), b2.has_value(), bool(f32(b2)), r.has_value(),
        bool(weight_order(plain(w1))), bool(weight_order(plain(w2))), (int)act,
        w2.size(0)}.save(ctx);
    return y;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& gys) {
    variable_list out(7);
    const How how = How::of(ctx);
    {
      const at::AutoGradMode off(false);
      const variable_list s = ctx->get_saved_variables();
      const Tensor &x = s[0], &w1 = s[1], &w2 = s[2], &h = s[3], &z = s[4], &gy = gys[0];
      const auto need = needs<6>(ctx, {true, true, true, how.vector1, how.vector2, how.residual});
      const bool inner = need[0] || need[1] || need[3];
      if (inner || need[2] || need[4]) {
        const c10::DeviceGuard on(gy.device());
        const int64_t width = how.size, d = gy.size(-1);
        Tensor gx, gw1, gw2, gb1, gb2;
        if (need[0]) gx = empty(gy.sizes(), gy);
        if (need[1]) gw1 = weight_grad(d, 2 * width, how.tr1, gy);
        if (need[2]) gw2 = weight_grad(width, d, how.tr2, gy);
        if (need[3]) gb1 = vector_grad(2 * width, how.vector1_f32, gy);
        if (need[4]) gb2 = vector_grad(d, how.vector2_f32, gy);
        if (gy.numel() == 0) {
          zero({gw1, gw2, gb1, gb2});
        } else {
          const Mat g = rows_of(gy, d), m = need[1] ? rows_of(x, d) : Mat();
          const Mat m1 = need[0] ? weight_of(w1, how.tr1) : Mat();
          const Mat m2 = inner ? weight_of(w2, how.tr2) : Mat();
          const int64_t rows = g.t.size(0);
          const int type = type_of(gy);
          const size_t n = lib.vmoe_gated_workspace_bytes(type, rows, d, width, 1);
          const Tensor ws = workspace(n, gy);
          call("vmoe_gated_backward", [&] {
            return lib.vmoe_gated_backward(
                type, g.p(), g.ld, m.p(), m.ld, rows, d, width, m1.p(), m1.ld, how.tr1, m2.p(),
                m2.ld, how.tr2, how.act, saved_ptr(h), saved_floats(z), out_ptr(gx), d,
                out_ptr(gw1), ld_of(gw1, how.tr1), out_ptr(gb1), how.vector1_f32, out_ptr(gw2),
                ld_of(gw2, how.tr2), out_ptr(gb2), how.vector2_f32, out_ptr(ws), n,
                stream_of(gy));
          });
        }
        out[0] = gx;
        out[1] = gw1;
        out[2] = gw2;
        out[3] = gb1;
        out[4] = gb2;
      }
    }
    out = gradients(std::move(out));
    if (how.residual) out[5] = gys[0];
    return out;
  }
};

Tensor gated_mlp(const Tensor& x, const Tensor& w1, const Tensor& w2, const Maybe& b1,
                 const Maybe& b2, const Maybe& r, int act) {
  check_type(x, "x");
  TORCH_CHECK_VALUE(x.dim() > 0 && w1.dim() == 2 && w2.dim() == 2 && x.size(-1) == w1.size(0) &&
                        w2.size(1) == w1.size(0) && w1.size(1) == 2 * w2.size(0),
                    "x [..., d], w1 [d, 2 width] and w2 [width, d] do not fit: ", x.sizes(), ", ",
                    w1.sizes(), ", ", w2.sizes());
  check_features(x, w2.size(1), "d");
  check_features(x, w2.size(0), "width");
  check_like(w1, "w1", x);
  check_like(w2, "w2", x);
  check_vector(b1, "bias1", w1.size(1), x);
  check_vector(b2, "bias2", w2.size(1), x);
  check_residual(r, x.sizes(), x);
  check_device(x);
  const Maybe mx = x, m1 = w1, m2 = w2;
  if (recorded({&mx, &m1, &m2, &b1, &b2, &r}))
    return GatedMLP::apply(x, w1, w2, b1, b2, r, (int64_t)act);
  Tensor h;
  return gated_forward(x, w1, w2, b1, b2, r, act, h, nullptr);
}

// ---------------------------------------------------------------------------
// Python.

struct BadType {
  std::string what;
};

const Tensor& tensor(PyObject* o, const char* what) {
  if (!THPVariable_Check(o))
    throw BadType{std::string(what) + " must be a tensor (got " + Py_TYPE(o)->tp_name + ")"};
  return THPVariable_Unpack(o);
}
Maybe maybe(PyObject* o, const char* what) {
  if (o == Py_None) return Maybe();
  return tensor(o, what);
}

struct NoGil {
  PyThreadState* state = PyEval_SaveThread();
  ~NoGil() { PyEval_RestoreThread(state); }
};

// f() reads the arguments and gives the call, which is made without the GIL.
template <typename F>
PyObject* guarded(F&& f) {
  HANDLE_TH_ERRORS
  TORCH_CHECK(lib.loaded, "no library in use");
  try {
    const auto run = f();
    Tensor y;
    {
      const NoGil free;
      y = run();
    }
    return THPVariable_Wrap(y);
  } catch (const NotOnGpu& e) {
    PyErr_SetString(PyExc_AssertionError, e.what.c_str());
  } catch (const BadType& e) {
    PyErr_SetString(PyExc_TypeError, e.what.c_str());
  }
  return nullptr;
  END_HANDLE_TH_ERRORS
}
bool count(Py_ssize_t n, Py_ssize_t want) {
  if (n == want) return true;
  PyErr_Format(PyExc_TypeError, "expected %zd arguments (got %zd)", want, n);
  return false;
}

PyObject* py_layer_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!count(n, 4)) return nullptr;
  const double eps = PyFloat_AsDouble(a[3]);
  if (PyErr_Occurred()) return nullptr;
  return guarded([&] {
    return [x = tensor(a[0], "x"), w = maybe(a[1], "weight"), b = maybe(a[2], "bias"), eps] {
      return layer_norm(x, w, b, eps);
    };
  });
}
PyObject* py_fused_linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!count(n, 5)) return nullptr;
  const long act = PyLong_AsLong(a[4]);
  if (PyErr_Occurred()) return nullptr;
  return guarded([&] {
    return [x = tensor(a[0], "x"), w = tensor(a[1], "weight"), b = maybe(a[2], "bias"),
            r = maybe(a[3], "residual"), act] { return fused_linear(x, w, b, r, (int)act); };
  });
}
PyObject* py_gated_mlp(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!count(n, 7)) return nullptr;
  const long act = PyLong_AsLong(a[6]);
  if (PyErr_Occurred()) return nullptr;
  return guarded([&] {
    return [x = tensor(a[0], "x"), w1 = tensor(a[1], "w1"), w2 = tensor(a[2], "w2"),
            b1 = maybe(a[3], "bias1"), b2 = maybe(a[4], "bias2"), r = maybe(a[5], "residual"),
            act] { return gated_mlp(x, w1, w2, b1, b2, r, (int)act); };
  });
}
// use(handle): calls go to the library that dlopen gave this handle for.
PyObject* py_use(PyObject*, PyObject* handle) {
  HANDLE_TH_ERRORS
  void* h = PyLong_AsVoidPtr(handle);
  if (PyErr_Occurred()) return nullptr;
  TORCH_CHECK(h, "no handle of a library");
  Library found;
#define VMOE_ENTRY(name)                                               \
  found.name = reinterpret_cast<decltype(&::name)>(dlsym(h, #name));   \
  TORCH_CHECK(found.name, "the library has no " #name);
  VMOE_ENTRIES(VMOE_ENTRY)
#undef VMOE_ENTRY
  found.loaded = true;
  lib = found;
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}
PyObject* py_set_timer(PyObject*, PyObject* timer) {
  Py_XINCREF(timer == Py_None ? nullptr : timer);
  Py_XDECREF(g_timer);
  g_timer = timer == Py_None ? nullptr : timer;
  Py_RETURN_NONE;
}

PyMethodDef kMethods[] = {
    {"layer_norm", (PyCFunction)(void (*)(void))py_layer_norm, METH_FASTCALL, nullptr},
    {"fused_linear", (PyCFunction)(void (*)(void))py_fused_linear, METH_FASTCALL, nullptr},
    {"gated_mlp", (PyCFunction)(void (*)(void))py_gated_mlp, METH_FASTCALL, nullptr},
    {"use", py_use, METH_O, nullptr},
    {"set_timer", py_set_timer, METH_O, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_dense", nullptr, -1, kMethods,
                       nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__dense(void) { return PyModule_Create(&kModule); }
