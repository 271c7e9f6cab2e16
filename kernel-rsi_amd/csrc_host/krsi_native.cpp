// Eager path of the public functions in native code: argument tests, output and workspace allocation,
// launch, and the autograd node, for the plain case of each call. The kernels are those of the C ABI;
// what this replaces is the Python around them, whose backward ran in torch's device thread, took
// the interpreter lock there and cost more than the kernels at the smaller sizes (host time of a
// forward and backward of rmsnorm x [256, 1152]: 102 -> 32 us, of which torch takes 20 for any node).
//
// Every function returns None for whatever is not the plain case (tracing, functorch transforms, dispatch
// modes, tensor subclasses, forward-mode duals, layouts that need a copy, arguments that are refused): the
// caller then takes its Python path, which handles it or raises. So no message or rule of
// validation is repeated here, and nothing that the call changes has been touched when None is returned.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <pybind11/pybind11.h>

#include "krsi.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// A status other than KRSI_OK in a forward: nothing was launched, or only what may be launched again; the Python path
// reports it.
struct NotPlain {};

void* stream_of(const Tensor& t) {
  return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream();
}

void forward_status(int rc) {
  if (rc != KRSI_OK) throw NotPlain{};
}

// The module that holds the type of a kernel status as an error, KrsiError, and the assignable workspace cap
// RELPOS_BWD_WORKSPACE_MAX (None or bytes).
PyObject* g_hip_module = nullptr;

// A Python error raised here, as torch's own, which its engine carries between threads. With the
// interpreter lock held.
[[noreturn]] void throw_python_error() {
  python_error err;
  err.persist();
  throw err;
}
void backward_status(int rc) {
  if (rc == KRSI_OK) return;
  pybind11::gil_scoped_acquire lock;
  PyObject* type = g_hip_module ? PyObject_GetAttrString(g_hip_module, "KrsiError") : nullptr;
  if (type) {
    PyErr_SetString(type, krsi_error_string(rc));
    Py_DECREF(type);
  } else if (!PyErr_Occurred()) {
    PyErr_SetString(PyExc_RuntimeError, krsi_error_string(rc));
  }
  throw_python_error();
}

// The status of an operator that changes its arguments: once something may have been launched it is not made again.
void in_place_status(int rc) {
  if (rc == KRSI_ERR_LAUNCH) backward_status(rc);
  forward_status(rc);
}

// KRSI_DTYPE_* of an activation dtype, or -1.
int dtype_code(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return KRSI_DTYPE_BF16;
    case at::kHalf: return KRSI_DTYPE_F16;
    case at::kFloat: return KRSI_DTYPE_F32;
    default: return -1;
  }
}

bool aligned16(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

// No transform, mode or tracer that has to see the call.
bool plain_context() {
  if (torch::jit::tracer::isTracing() || c10::impl::TorchDispatchModeTLS::any_modes_set()) return false;
  const auto on = c10::impl::tls_local_dispatch_key_set().included_;
  return !on.has_any(c10::DispatchKeySet({c10::DispatchKey::FuncTorchDynamicLayerFrontMode,
                                          c10::DispatchKey::FuncTorchDynamicLayerBackMode, c10::DispatchKey::Python,
                                          c10::DispatchKey::Functionalize}));
}
// A strided GPU tensor with storage: no subclass that dispatches, no wrapper, no dual, not nested (whose sizes
// throw).
bool plain(const Tensor& t) {
  if (t.is_nested() || !t.is_cuda() || t.layout() != at::kStrided || !t.has_storage() || t.is_conj() || t.is_neg()) return false;
  const auto keys = t.key_set();
  if (keys.has_any(c10::DispatchKeySet({c10::DispatchKey::Python, c10::DispatchKey::FuncTorchBatched,
                                        c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::Functionalize})))
    return false;
  return !t._fw_grad(0).defined();
}

// A saved tensor can come back from a saved-tensor hook as anything: what a kernel reads by pointer has
// to be where, of the type and of the shape that the forward saved.
void check_saved(const char* name, const Tensor& t, const Tensor& grad, at::ScalarType dtype, at::IntArrayRef sizes) {
  TORCH_CHECK_VALUE(t.is_cuda() && t.device() == grad.device(), "saved ", name, " came back on ", t.device(),
                    ", the gradient is on ", grad.device());
  TORCH_CHECK_TYPE(t.scalar_type() == dtype, "saved ", name, " came back as ", t.scalar_type(), ", not ", dtype);
  TORCH_CHECK_VALUE(t.sizes() == sizes, "saved ", name, " came back with shape ", t.sizes(), ", not ", sizes);
}

// ------------------------------------------------------------------- RMSNorm
struct RmsNormFn : torch::autograd::Function<RmsNormFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, double eps) {
    const int64_t rows = x.size(0), n = x.size(1);
    Tensor y = at::empty_like(x), rstd = at::empty({rows}, x.options().dtype(at::kFloat));
    forward_status(krsi_rmsnorm_fwd(x.data_ptr(), w.data_ptr(), y.data_ptr(), rstd.data_ptr<float>(), rows, (int)n,
                                    (float)eps, dtype_code(x), stream_of(x)));
    ctx->save_for_backward({x, w, rstd});
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor g = grads[0].contiguous(), x = saved[0].contiguous(), w = saved[1].contiguous(),
                 rstd = saved[2].contiguous();
    const int64_t rows = g.size(0), n = g.size(1);
    check_saved("x2d", x, g, g.scalar_type(), {rows, n});
    check_saved("weight", w, g, g.scalar_type(), {n});
    check_saved("rstd", rstd, g, at::kFloat, {rows});
    Tensor dx = at::empty_like(x), dw = at::empty({n}, w.options());
    const size_t bytes = krsi_rmsnorm_bwd_workspace_bytes(rows, (int)n);
    Tensor ws = at::empty({(int64_t)bytes}, x.options().dtype(at::kByte));
    backward_status(krsi_rmsnorm_bwd(g.data_ptr(), x.data_ptr(), w.data_ptr(), rstd.data_ptr<float>(), dx.data_ptr(),
                                     dw.data_ptr(), ws.data_ptr(), bytes, rows, (int)n, dtype_code(x), stream_of(x)));
    return {dx, dw, Tensor()};
  }
};

// --------------------------------------------------------------------- GEGLU
struct GegluFn : torch::autograd::Function<GegluFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& u, int64_t approximate) {
    const int64_t rows = u.size(0), f = u.size(1) / 2;
    Tensor out = at::empty({rows, f}, u.options());
    forward_status(krsi_geglu_fwd(u.data_ptr(), out.data_ptr(), rows, (int)f, (int)approximate, dtype_code(u),
                                  stream_of(u)));
    ctx->save_for_backward({u});
    ctx->saved_data["approximate"] = approximate;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const Tensor g = grads[0].contiguous(), u = ctx->get_saved_variables()[0].contiguous();
    check_saved("u", u, g, g.scalar_type(), {g.size(0), 2 * g.size(1)});
    Tensor du = at::empty_like(u);
    backward_status(krsi_geglu_bwd(g.data_ptr(), u.data_ptr(), du.data_ptr(), u.size(0), (int)(u.size(1) / 2),
                                   (int)ctx->saved_data["approximate"].toInt(), dtype_code(u), stream_of(u)));
    return {du, Tensor()};
  }
};

struct GegluLinearFn : torch::autograd::Function<GegluLinearFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, int64_t approximate) {
    const int64_t rows = x.size(0), k = x.size(1), f = w.size(0) / 2;
    Tensor out = at::empty({rows, f}, x.options());
    forward_status(krsi_geglu_linear_fwd(x.data_ptr(), w.data_ptr(), out.data_ptr(), rows, (int)k, (int)f,
                                         (int)approximate, dtype_code(x), stream_of(x)));
    ctx->save_for_backward({x, w});
    ctx->saved_data["approximate"] = approximate;
    ctx->saved_data["k"] = k;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1];
    const int approximate = (int)ctx->saved_data["approximate"].toInt();
    const int64_t rows = grads[0].size(0), k = ctx->saved_data["k"].toInt(), f = grads[0].size(1);
    check_saved("x", x, grads[0], grads[0].scalar_type(), {rows, k});
    check_saved("weight", w, grads[0], grads[0].scalar_type(), {2 * f, k});
    const Tensor g = grads[0].contiguous(), xc = x.contiguous(), wc = w.contiguous();
    Tensor du = at::empty({rows, 2 * f}, x.options());
    if (aligned16(xc) && aligned16(wc)) {
      backward_status(krsi_geglu_linear_bwd(g.data_ptr(), xc.data_ptr(), wc.data_ptr(), du.data_ptr(), rows, (int)k,
                                            (int)f, approximate, dtype_code(x), stream_of(x)));
    } else {  // a saved tensor that came back elsewhere
      const Tensor u = at::linear(xc, wc);
      backward_status(krsi_geglu_bwd(g.data_ptr(), u.data_ptr(), du.data_ptr(), rows, (int)f, approximate,
                                     dtype_code(x), stream_of(x)));
    }
    const bool need_dx = ctx->needs_input_grad(0), need_dw = ctx->needs_input_grad(1);
    // Not under create_graph, where torch's products carry a graph on.
    if (!at::GradMode::is_enabled() && x.is_contiguous() && w.is_contiguous() &&
        aligned16(x) && aligned16(w) && krsi_geglu_linear_grads_pays(rows, (int)k, (int)f, need_dx, need_dw) == 1) {
      Tensor dx, dw, ws;
      const size_t bytes = krsi_geglu_linear_grads_workspace_bytes(rows, (int)k, (int)f);
      if (bytes) ws = at::empty({(int64_t)bytes}, x.options().dtype(at::kByte));
      if (need_dx) dx = at::empty_like(x);
      if (need_dw) dw = at::empty_like(w);
      backward_status(krsi_geglu_linear_grads(du.data_ptr(), x.data_ptr(), w.data_ptr(),
                                              need_dx ? dx.data_ptr() : nullptr, need_dw ? dw.data_ptr() : nullptr,
                                              bytes ? ws.data_ptr() : nullptr, bytes, rows, (int)k, (int)f,
                                              dtype_code(x), stream_of(x)));
      return {dx, dw, Tensor()};
    }
    return {need_dx ? at::mm(du, w) : Tensor(), need_dw ? at::mm(du.t(), x) : Tensor(), Tensor()};
  }
};

// ------------------------------------------------ relative-position attention
// The workspace of a backward whose full size is `full`: the cap where one is assigned, but no less than
// `least`. Takes the interpreter lock, which torch's device thread owns a state for.
size_t workspace_bytes(size_t full, size_t least) {
  pybind11::gil_scoped_acquire lock;
  if (!g_hip_module) return full;
  try {
    const pybind11::object cap = pybind11::handle(g_hip_module).attr("RELPOS_BWD_WORKSPACE_MAX");
    if (cap.is_none() || !(cap < pybind11::int_(full))) return full;  // raises for what is no number
    const int64_t bytes = pybind11::int_(cap).cast<int64_t>();        // below full, which fits
    return bytes < (int64_t)least ? least : (size_t)bytes;
  } catch (pybind11::error_already_set& e) {
    e.restore();
    throw_python_error();
  }
}

struct Dims {
  int B, S, H, D;
  double scale;
};

Tensor relpos_forward(const Tensor& qkv, const Tensor& pd, const Dims& d, Tensor* out32, Tensor* lse) {
  const Tensor p = pd.contiguous();
  Tensor out = at::empty({(int64_t)d.B * d.S, (int64_t)d.H * d.D}, qkv.options());
  if (out32) {
    *out32 = at::empty(out.sizes(), qkv.options().dtype(at::kFloat));
    *lse = at::empty({(int64_t)d.B * d.H, d.S}, qkv.options().dtype(at::kFloat));
  }
  forward_status(krsi_relpos_fwd(qkv.data_ptr(), qkv.stride(0), p.data_ptr<float>(), out.data_ptr(),
                                 out32 ? out32->data_ptr<float>() : nullptr, lse ? lse->data_ptr<float>() : nullptr,
                                 d.B, d.S, d.H, d.D, (float)d.scale, dtype_code(qkv), stream_of(qkv)));
  return out;
}

struct RelposFn : torch::autograd::Function<RelposFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& qkv, const Tensor& pd, int64_t B, int64_t S, int64_t H,
                        int64_t D, double scale) {
    Tensor out32, lse;
    Tensor out = relpos_forward(qkv, pd, Dims{(int)B, (int)S, (int)H, (int)D, scale}, &out32, &lse);
    ctx->save_for_backward({qkv, pd, out32, lse});
    ctx->saved_data["dims"] = std::vector<int64_t>{B, S, H, D};
    ctx->saved_data["scale"] = scale;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const auto d = ctx->saved_data["dims"].toIntVector();
    const int64_t B = d[0], S = d[1], H = d[2], D = d[3], cols = 3 * H * D;
    const Tensor &qkv = saved[0], dout = grads[0].contiguous(), pd = saved[1].contiguous(),
                 out32 = saved[2].contiguous(), lse = saved[3].contiguous();
    check_saved("qkv", qkv, dout, dout.scalar_type(), {B * S, qkv.dim() == 2 ? qkv.size(1) : cols});
    TORCH_CHECK_VALUE(qkv.size(1) >= cols && qkv.stride(1) == 1, "saved qkv came back with shape ", qkv.sizes(),
                      " and strides ", qkv.strides());
    check_saved("pd", pd, dout, at::kFloat, {H, 2 * S - 1});
    check_saved("out32", out32, dout, at::kFloat, {B * S, H * D});
    check_saved("lse", lse, dout, at::kFloat, {B * H, S});
    // Rows on 16-byte boundaries, which the width of a slice may not give.
    const int64_t per = 16 / qkv.element_size(), width = qkv.size(1), ld = (width + per - 1) / per * per;
    Tensor dqkv = at::empty({B * S, ld}, qkv.options());
    if (ld > width) dqkv = dqkv.narrow(1, 0, width);
    if (width > cols) dqkv.narrow(1, cols, width - cols).zero_();
    Tensor dpd = at::empty({H, 2 * S - 1}, pd.options());
    const size_t bytes = workspace_bytes(krsi_relpos_bwd_workspace_bytes((int)B, (int)S, (int)H, (int)D),
                                         krsi_relpos_bwd_workspace_min_bytes((int)B, (int)S, (int)H, (int)D));
    Tensor ws = at::empty({(int64_t)bytes}, qkv.options().dtype(at::kByte));
    backward_status(krsi_relpos_bwd(dout.data_ptr(), qkv.data_ptr(), qkv.stride(0), pd.data_ptr<float>(),
                                    out32.data_ptr<float>(), lse.data_ptr<float>(), dqkv.data_ptr(), dqkv.stride(0),
                                    dpd.data_ptr<float>(), ws.data_ptr(), bytes, (int)B, (int)S, (int)H, (int)D,
                                    (float)ctx->saved_data["scale"].toDouble(), dtype_code(qkv), stream_of(qkv)));
    return {dqkv, dpd, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

struct BucketFn : torch::autograd::Function<BucketFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& table, const Tensor& bucket, int64_t S) {
    const Tensor t = table.contiguous();
    const int64_t nb = t.size(0), H = t.size(1);
    Tensor pd = at::empty({H, 2 * S - 1}, t.options());
    forward_status(krsi_relpos_bucket_gather(t.data_ptr<float>(), bucket.data_ptr<int32_t>(), pd.data_ptr<float>(),
                                             (int)S, (int)H, (int)nb, stream_of(t)));
    ctx->save_for_backward({bucket});
    ctx->saved_data["dims"] = std::vector<int64_t>{S, nb};
    return pd;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto d = ctx->saved_data["dims"].toIntVector();
    const int64_t S = d[0], nb = d[1];
    const Tensor g = grads[0].contiguous(), bucket = ctx->get_saved_variables()[0].contiguous();
    check_saved("bucket", bucket, g, at::kInt, {2 * S - 1});
    Tensor dtable = at::empty({nb, g.size(0)}, g.options());
    backward_status(krsi_relpos_bucket_sum(g.data_ptr<float>(), bucket.data_ptr<int32_t>(), dtable.data_ptr<float>(),
                                           (int)S, (int)g.size(0), (int)nb, stream_of(g)));
    return {dtable, Tensor(), Tensor()};
  }
};

// ------------------------------------------- query and key norm with rotation
// Each launch below goes to its tensors' device, which need not be the current one.
struct QkArgs {
  int64_t tokens;
  int S, H, KH, D, R;
  int64_t table_rows, ld;
  int position_bytes;
  QkArgs(const std::vector<int64_t>& d, const Tensor& qkv, const Tensor& rope, const Tensor& positions)
      : tokens(d[0]), S((int)d[1]), H((int)d[2]), KH((int)d[3]), D((int)d[4]), R((int)rope.size(1)),
        table_rows(rope.size(0)), ld(qkv.size(0) > 1 ? qkv.stride(0) : qkv.size(1)),
        position_bytes(positions.defined() ? (int)positions.element_size() : 0) {}
};
const void* data_or_null(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

struct QkNormRopeFn : torch::autograd::Function<QkNormRopeFn> {
  static Tensor launch(const Tensor& qkv, const Tensor& wq, const Tensor& wk, const Tensor& rope,
                       const std::optional<Tensor>& given, int64_t tokens, int64_t S, int64_t H, int64_t KH, int64_t D,
                       double eps, int64_t interleaved) {
    const c10::DeviceGuard guard(qkv.device());
    const Tensor positions = given ? *given : Tensor();
    const QkArgs a({tokens, S, H, KH, D}, qkv, rope, positions);
    Tensor out = at::empty({tokens, (H + 2 * KH) * D}, qkv.options());
    forward_status(krsi_qk_norm_rope_fwd(qkv.data_ptr(), a.ld, wq.data_ptr(), wk.data_ptr(), rope.data_ptr<float>(),
                                         data_or_null(positions), out.data_ptr(), tokens, a.S, a.H, a.KH, a.D, a.R,
                                         a.table_rows, a.position_bytes, (float)eps, (int)interleaved, dtype_code(qkv),
                                         stream_of(qkv)));
    return out;
  }
  static Tensor forward(AutogradContext* ctx, const Tensor& qkv, const Tensor& wq, const Tensor& wk, const Tensor& rope,
                        const std::optional<Tensor>& given, int64_t tokens, int64_t S, int64_t H, int64_t KH, int64_t D,
                        double eps, int64_t interleaved) {
    Tensor out = launch(qkv, wq, wk, rope, given, tokens, S, H, KH, D, eps, interleaved);
    ctx->save_for_backward({qkv, wq, wk, rope, given ? *given : Tensor()});
    ctx->saved_data["dims"] = std::vector<int64_t>{tokens, S, H, KH, D, interleaved, qkv.size(1), rope.size(0), rope.size(1),
                                                   given ? (int64_t)given->scalar_type() : (int64_t)-1};
    ctx->saved_data["eps"] = eps;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const c10::DeviceGuard guard(grads[0].device());
    const auto saved = ctx->get_saved_variables();
    const auto dims = ctx->saved_data["dims"].toIntVector();
    const int64_t tokens = dims[0], H = dims[2], KH = dims[3], D = dims[4], heads = (H + 2 * KH) * D;
    const Tensor dy = grads[0].contiguous();
    const Tensor &qkv = saved[0], wq = saved[1].contiguous(), wk = saved[2].contiguous(), rope = saved[3].contiguous();
    const int64_t cols = dims[6], kind = dims[9];
    check_saved("qkv", qkv, dy, dy.scalar_type(), {tokens, cols});
    TORCH_CHECK_VALUE(qkv.stride(1) == 1 && (tokens <= 1 || qkv.stride(0) >= heads), "saved qkv came back with strides ",
                      qkv.strides());
    check_saved("q_weight", wq, dy, dy.scalar_type(), {D});
    check_saved("k_weight", wk, dy, dy.scalar_type(), {D});
    check_saved("rope", rope, dy, at::kFloat, {dims[7], dims[8]});
    Tensor positions;
    if (kind >= 0) {
      positions = saved[4].contiguous();
      check_saved("positions", positions, dy, (at::ScalarType)kind, {tokens});
    }
    const QkArgs a(dims, qkv, rope, positions);
    Tensor dqkv = at::empty({tokens, cols}, qkv.options());
    if (cols > heads) dqkv.narrow(1, heads, cols - heads).zero_();
    Tensor dwq = at::empty({D}, wq.options()), dwk = at::empty({D}, wk.options());
    const size_t bytes = krsi_qk_norm_rope_bwd_workspace_bytes(a.D);
    Tensor ws = at::empty({(int64_t)bytes}, qkv.options().dtype(at::kByte));
    backward_status(krsi_qk_norm_rope_bwd(
        dy.data_ptr(), qkv.data_ptr(), a.ld, wq.data_ptr(), wk.data_ptr(), rope.data_ptr<float>(),
        data_or_null(positions), dqkv.data_ptr(), cols, dwq.data_ptr(), dwk.data_ptr(), ws.data_ptr(), bytes, tokens, a.S,
        a.H, a.KH, a.D, a.R, a.table_rows, a.position_bytes, (float)ctx->saved_data["eps"].toDouble(), (int)dims[5],
        dtype_code(qkv), stream_of(qkv)));
    variable_list out(12);
    out[0] = dqkv, out[1] = dwq, out[2] = dwk;
    return out;
  }
};

// ------------------------------------------------------------ token embedding
struct EmbeddingFn : torch::autograd::Function<EmbeddingFn> {
  static Tensor launch(const Tensor& tokens, const Tensor& table, double scale) {
    const c10::DeviceGuard guard(table.device());
    auto shape = tokens.sizes().vec();
    shape.push_back(table.size(1));
    Tensor out = at::empty(shape, table.options());
    forward_status(krsi_embedding_fwd(tokens.data_ptr(), (int)tokens.element_size(), table.data_ptr(), out.data_ptr(),
                                      tokens.numel(), (int)table.size(0), (int)table.size(1), (float)scale,
                                      dtype_code(table), stream_of(table)));
    return out;
  }
  static Tensor forward(AutogradContext* ctx, const Tensor& tokens, const Tensor& table, double scale, int64_t padding) {
    Tensor out = launch(tokens, table, scale);
    ctx->save_for_backward({tokens});
    ctx->saved_data["shape"] = out.sizes().vec();
    ctx->saved_data["args"] = std::vector<int64_t>{table.size(0), padding, (int64_t)tokens.scalar_type()};
    ctx->saved_data["scale"] = scale;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const c10::DeviceGuard guard(grads[0].device());
    const Tensor dy = grads[0].contiguous(), tokens = ctx->get_saved_variables()[0].contiguous();
    auto shape = ctx->saved_data["shape"].toIntVector();
    const auto args = ctx->saved_data["args"].toIntVector();
    const int64_t V = args[0], D = shape.back();
    shape.pop_back();
    check_saved("tokens", tokens, dy, (at::ScalarType)args[2], shape);
    Tensor dtable = at::empty({V, D}, dy.options());
    const size_t bytes = krsi_embedding_bwd_workspace_bytes(tokens.numel(), (int)V, (int)D);
    Tensor ws = at::empty({(int64_t)bytes}, dy.options().dtype(at::kByte));
    backward_status(krsi_embedding_bwd(dy.data_ptr(), tokens.data_ptr(), (int)tokens.element_size(), dtable.data_ptr(),
                                       ws.data_ptr(), bytes, tokens.numel(), (int)V, (int)D, args[1],
                                       (float)ctx->saved_data["scale"].toDouble(), dtype_code(dy), stream_of(dy)));
    return {Tensor(), dtable, Tensor(), Tensor()};
  }
};

// ----------------------------------- cross entropy of an output projection
struct LinearCrossEntropyFn : torch::autograd::Function<LinearCrossEntropyFn> {
  // The loss and what the backward reads of each row.
  static std::pair<Tensor, Tensor> launch(const Tensor& x, const Tensor& w, const Tensor& targets, int64_t ignore_index,
                                          int64_t reduction) {
    const c10::DeviceGuard guard(x.device());
    const int64_t rows = x.size(0), k = x.size(1), v = w.size(0);
    const auto fp32 = x.options().dtype(at::kFloat);
    Tensor loss = reduction == 0 ? at::empty({rows}, fp32) : at::empty({}, fp32), stats = at::empty({rows + 1}, fp32);
    const size_t bytes = krsi_linear_cross_entropy_fwd_workspace_bytes(rows, (int)k, (int)v);
    Tensor ws = at::empty({(int64_t)bytes}, x.options().dtype(at::kByte));
    forward_status(krsi_linear_cross_entropy_fwd(x.data_ptr(), w.data_ptr(), targets.data_ptr(),
                                                 (int)targets.element_size(), loss.data_ptr<float>(),
                                                 stats.data_ptr<float>(), ws.data_ptr(), bytes, rows, (int)k, (int)v,
                                                 ignore_index, (int)reduction, dtype_code(x), stream_of(x)));
    return {loss, stats};
  }
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Tensor& targets,
                        int64_t ignore_index, int64_t reduction) {
    auto [loss, stats] = launch(x, w, targets, ignore_index, reduction);
    ctx->save_for_backward({x, w, targets, stats});
    ctx->saved_data["args"] = std::vector<int64_t>{x.size(0), x.size(1), w.size(0), ignore_index, reduction,
                                                   (int64_t)targets.scalar_type(), (int64_t)x.scalar_type()};
    return loss;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const c10::DeviceGuard guard(grads[0].device());
    const auto a = ctx->saved_data["args"].toIntVector();
    const int64_t rows = a[0], k = a[1], v = a[2];
    const auto saved = ctx->get_saved_variables();
    const Tensor dout = grads[0].contiguous(), targets = saved[2].contiguous(), stats = saved[3].contiguous();
    Tensor x = saved[0].contiguous(), w = saved[1].contiguous();
    check_saved("x", x, dout, (at::ScalarType)a[6], {rows, k});
    check_saved("weight", w, dout, (at::ScalarType)a[6], {v, k});
    check_saved("targets", targets, dout, (at::ScalarType)a[5], {rows});
    check_saved("stats", stats, dout, at::kFloat, {rows + 1});
    if (!aligned16(x)) x = x.clone();  // a saved tensor that came back elsewhere
    if (!aligned16(w)) w = w.clone();
    Tensor dx, dw;
    if (ctx->needs_input_grad(0)) dx = at::empty({rows, k}, x.options());
    if (ctx->needs_input_grad(1)) dw = at::empty({v, k}, w.options());
    const size_t bytes = krsi_linear_cross_entropy_bwd_workspace_bytes(rows, (int)k, (int)v);
    Tensor ws = at::empty({(int64_t)bytes}, x.options().dtype(at::kByte));
    backward_status(krsi_linear_cross_entropy_bwd(
        dout.data_ptr<float>(), x.data_ptr(), w.data_ptr(), targets.data_ptr(), (int)targets.element_size(),
        stats.data_ptr<float>(), dx.defined() ? dx.data_ptr() : nullptr, dw.defined() ? dw.data_ptr() : nullptr,
        ws.data_ptr(), bytes, rows, (int)k, (int)v, a[3], (int)a[4], dtype_code(x), stream_of(x)));
    return {dx, dw, Tensor(), Tensor(), Tensor()};
  }
};

// ----------------------------------------- residual addition with RMS norm
struct AddRmsNormFn : torch::autograd::Function<AddRmsNormFn> {
  // y, r and, where stats is given, the reciprocal roots.
  static variable_list launch(const Tensor& x, const Tensor& residual, const Tensor& w, double eps, Tensor* stats) {
    const c10::DeviceGuard guard(x.device());
    Tensor y = at::empty_like(x), r = at::empty_like(x);
    if (stats) *stats = at::empty({x.size(0)}, x.options().dtype(at::kFloat));
    forward_status(krsi_add_rmsnorm_fwd(x.data_ptr(), residual.data_ptr(), w.data_ptr(), y.data_ptr(), r.data_ptr(),
                                        stats ? stats->data_ptr<float>() : nullptr, x.size(0), (int)x.size(1), (float)eps,
                                        dtype_code(x), stream_of(x)));
    return {y, r};
  }
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& residual, const Tensor& w,
                               double eps) {
    Tensor rstd;
    variable_list out = launch(x, residual, w, eps, &rstd);
    ctx->save_for_backward({out[1], w, rstd});
    ctx->set_materialize_grads(false);
    ctx->saved_data["shape"] = std::vector<int64_t>{x.size(0), x.size(1), (int64_t)x.scalar_type()};
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return {grads[1], grads[1], Tensor(), Tensor()};  // the stream alone was used
    const c10::DeviceGuard guard(grads[0].device());
    const auto shape = ctx->saved_data["shape"].toIntVector();
    const int64_t rows = shape[0], n = shape[1];
    const at::ScalarType type = (at::ScalarType)shape[2];
    const auto saved = ctx->get_saved_variables();
    const Tensor dy = grads[0].contiguous(), dr = grads[1].defined() ? grads[1].contiguous() : Tensor(),
                 r = saved[0].contiguous(), w = saved[1].contiguous(), rstd = saved[2].contiguous();
    check_saved("r", r, dy, type, {rows, n});
    check_saved("weight", w, dy, type, {n});
    check_saved("rstd", rstd, dy, at::kFloat, {rows});
    Tensor dx = at::empty_like(r), dw = at::empty({n}, w.options());
    const size_t bytes = krsi_add_rmsnorm_bwd_workspace_bytes(rows, (int)n);
    Tensor ws = at::empty({(int64_t)bytes}, r.options().dtype(at::kByte));
    backward_status(krsi_add_rmsnorm_bwd(dy.data_ptr(), dr.defined() ? dr.data_ptr() : nullptr, r.data_ptr(), w.data_ptr(),
                                         rstd.data_ptr<float>(), dx.data_ptr(), dw.data_ptr(), ws.data_ptr(), bytes, rows,
                                         (int)n, dtype_code(r), stream_of(r)));
    return {dx, dx, dw, Tensor()};
  }
};

// ---------------------------------------------------------------- Python entries
// An entry as Python calls it: C++ exceptions, of the argument tests too, become Python ones.
using Args = PyObject* const*;
template <PyObject* (*F)(Args, Py_ssize_t)>
PyObject* entry(PyObject*, Args a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  return F(a, n);
  END_HANDLE_TH_ERRORS
}

// The result of fn, None when the call is not plain.
struct ReleaseLock {  // the interpreter lock, as torch's own bindings release it around an operator
  PyThreadState* state = PyEval_SaveThread();
  ~ReleaseLock() { PyEval_RestoreThread(state); }
};
template <typename Fn>
PyObject* unlocked(Fn&& fn) {
  try {
    Tensor out;
    {
      ReleaseLock released;
      out = fn();
    }
    return THPVariable_Wrap(std::move(out));
  } catch (const NotPlain&) {
    Py_RETURN_NONE;
  }
}

// The same for several tensors, as a tuple; an undefined one is None.
template <typename Fn>
PyObject* unlocked_tuple(Fn&& fn) {
  try {
    variable_list out;
    {
      ReleaseLock released;
      out = fn();
    }
    PyObject* tuple = PyTuple_New((Py_ssize_t)out.size());
    for (size_t i = 0; tuple && i < out.size(); ++i) PyTuple_SET_ITEM(tuple, i, THPVariable_Wrap(std::move(out[i])));
    return tuple;
  } catch (const NotPlain&) {
    Py_RETURN_NONE;
  }
}

bool tensor_arg(PyObject* o, const Tensor** t) {
  if (!THPVariable_CheckExact(o)) return false;  // Tensor or Parameter: a subclass keeps its type in Python
  *t = &THPVariable_Unpack(o);
  return plain(**t);
}
bool int_arg(PyObject* o, int64_t lo, int64_t hi, int64_t* v) {
  if (!PyLong_CheckExact(o)) return false;
  int overflow = 0;
  *v = PyLong_AsLongLongAndOverflow(o, &overflow);
  return !overflow && *v >= lo && *v <= hi;
}
bool float_arg(PyObject* o, double* v) {
  if (!PyFloat_CheckExact(o)) return false;
  *v = PyFloat_AS_DOUBLE(o);
  return true;
}
constexpr int64_t kIntMax = 0x7fffffff;

PyObject* py_rmsnorm(Args a, Py_ssize_t n) {
  const Tensor *x, *w;
  double eps;
  if (n != 3 || !plain_context() || !tensor_arg(a[0], &x) || !tensor_arg(a[1], &w) || !float_arg(a[2], &eps))
    Py_RETURN_NONE;
  if (x->dim() != 2 || !x->is_contiguous() || x->size(0) == 0 || dtype_code(*x) < 0 ||
      w->scalar_type() != x->scalar_type() || w->dim() != 1 || w->size(0) != x->size(1) || !w->is_contiguous() ||
      w->device() != x->device() || x->size(1) > kIntMax)
    Py_RETURN_NONE;
  return unlocked([&] { return RmsNormFn::apply(*x, *w, eps); });
}

PyObject* py_geglu(Args a, Py_ssize_t n) {
  const Tensor* u;
  int64_t approximate;
  if (n != 2 || !plain_context() || !tensor_arg(a[0], &u) || !int_arg(a[1], 0, 1, &approximate)) Py_RETURN_NONE;
  if (u->dim() != 2 || !u->is_contiguous() || u->numel() == 0 || u->size(1) % 2 || dtype_code(*u) < 0 ||
      u->size(1) > kIntMax)
    Py_RETURN_NONE;
  return unlocked([&] { return GegluFn::apply(*u, approximate); });
}

PyObject* py_geglu_linear(Args a, Py_ssize_t n) {
  const Tensor *x, *w;
  int64_t approximate;
  if (n != 3 || !plain_context() || !tensor_arg(a[0], &x) || !tensor_arg(a[1], &w) ||
      !int_arg(a[2], 0, 1, &approximate))
    Py_RETURN_NONE;
  if (x->dim() != 2 || w->dim() != 2 || (x->scalar_type() != at::kBFloat16 && x->scalar_type() != at::kHalf) ||
      w->scalar_type() != x->scalar_type() || w->device() != x->device() || w->size(1) != x->size(1) ||
      x->size(0) == 0 || x->size(1) % 64 || w->size(0) % 128 || x->size(1) > kIntMax || w->size(0) > kIntMax ||
      !x->is_contiguous() || !w->is_contiguous())
    Py_RETURN_NONE;
  return unlocked([&] { return GegluLinearFn::apply(*x, *w, approximate); });
}

PyObject* py_relpos_attention(Args a, Py_ssize_t n) {
  const Tensor *qkv, *pd;
  int64_t B, S, H, D;
  double scale;
  if (n != 7 || !plain_context() || !tensor_arg(a[0], &qkv) || !tensor_arg(a[1], &pd) ||
      !int_arg(a[2], 1, kIntMax, &B) || !int_arg(a[3], 1, kIntMax, &S) || !int_arg(a[4], 1, kIntMax, &H) ||
      !int_arg(a[5], 8, 128, &D) || !float_arg(a[6], &scale))
    Py_RETURN_NONE;
  if (qkv->dim() != 2 || dtype_code(*qkv) < 0 || D % 8 || qkv->stride(1) != 1 ||
      qkv->stride(0) * qkv->element_size() % 16 || !aligned16(*qkv) || qkv->size(0) != B * S ||
      qkv->size(1) / 3 < H * D || pd->scalar_type() != at::kFloat || pd->dim() != 2 || pd->size(0) != H ||
      pd->size(1) != 2 * S - 1 || pd->device() != qkv->device())
    Py_RETURN_NONE;
  if (at::GradMode::is_enabled() && (qkv->requires_grad() || pd->requires_grad()))
    return unlocked([&] { return RelposFn::apply(*qkv, *pd, B, S, H, D, scale); });
  // No backward can follow: the kernels skip the fp32 output and lse it would need.
  return unlocked([&] {
    at::NoGradGuard no_grad;
    return relpos_forward(*qkv, *pd, Dims{(int)B, (int)S, (int)H, (int)D, scale}, nullptr, nullptr);
  });
}

PyObject* py_bucket_table(Args a, Py_ssize_t n) {
  const Tensor *table, *bucket;
  int64_t S;
  if (n != 3 || !plain_context() || !tensor_arg(a[0], &table) || !tensor_arg(a[1], &bucket) ||
      !int_arg(a[2], 1, kIntMax, &S))
    Py_RETURN_NONE;
  if (table->scalar_type() != at::kFloat || table->dim() != 2 || table->numel() == 0 ||
      table->size(0) > kIntMax || table->size(1) > kIntMax || bucket->scalar_type() != at::kInt ||
      bucket->dim() != 1 || bucket->size(0) != 2 * S - 1 || !bucket->is_contiguous() ||
      bucket->device() != table->device())
    Py_RETURN_NONE;
  return unlocked([&] { return BucketFn::apply(*table, *bucket, S); });
}

// Whether the call is recorded for a backward; without that its launch needs no node (bf16 tokens of one step of
// generation: 7.9 -> 6.4 us a call).
bool recorded(std::initializer_list<const Tensor*> inputs) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : inputs)
    if (t->requires_grad()) return true;
  return false;
}

bool index_dtype(const Tensor& t) { return t.scalar_type() == at::kLong || t.scalar_type() == at::kInt; }

PyObject* py_qk_norm_rope(Args a, Py_ssize_t n) {
  const Tensor *qkv, *wq, *wk, *rope, *pos = nullptr;
  int64_t B, S, H, KH, D, interleaved;
  double eps;
  if (n != 12 || !plain_context() || !tensor_arg(a[0], &qkv) || !tensor_arg(a[1], &wq) || !tensor_arg(a[2], &wk) ||
      !tensor_arg(a[3], &rope) || (a[4] != Py_None && !tensor_arg(a[4], &pos)) || !int_arg(a[5], 1, kIntMax, &B) ||
      !int_arg(a[6], 1, kIntMax, &S) || !int_arg(a[7], 1, 65535, &H) || !int_arg(a[8], 1, 65535, &KH) ||
      !int_arg(a[9], 8, 128, &D) || !float_arg(a[10], &eps) || !int_arg(a[11], 0, 1, &interleaved))
    Py_RETURN_NONE;
  const int64_t cols = (H + 2 * KH) * D;
  if (qkv->dim() != 2 || dtype_code(*qkv) < 0 || D % 8 || qkv->size(0) != B * S || qkv->size(1) < cols ||
      qkv->stride(1) != 1 || (qkv->size(0) > 1 && qkv->stride(0) < cols))
    Py_RETURN_NONE;
  for (const Tensor* w : {wq, wk})
    if (w->scalar_type() != qkv->scalar_type() || w->dim() != 1 || w->size(0) != D || !w->is_contiguous() ||
        w->device() != qkv->device())
      Py_RETURN_NONE;
  if (rope->scalar_type() != at::kFloat || rope->dim() != 2 || rope->size(0) < 1 || rope->size(1) < 2 ||
      rope->size(1) > D || rope->size(1) % 2 || !rope->is_contiguous() || rope->requires_grad() ||
      rope->device() != qkv->device() || (!pos && rope->size(0) < S))
    Py_RETURN_NONE;
  if (pos && (!index_dtype(*pos) || pos->dim() != 1 || pos->numel() != B * S || !pos->is_contiguous() ||
              pos->device() != qkv->device()))
    Py_RETURN_NONE;
  const std::optional<Tensor> positions = pos ? std::make_optional(*pos) : std::nullopt;
  return unlocked([&] {
    return recorded({qkv, wq, wk})
               ? QkNormRopeFn::apply(*qkv, *wq, *wk, *rope, positions, B * S, S, H, KH, D, eps, interleaved)
               : QkNormRopeFn::launch(*qkv, *wq, *wk, *rope, positions, B * S, S, H, KH, D, eps, interleaved);
  });
}

PyObject* py_embedding(Args a, Py_ssize_t n) {
  const Tensor *tokens, *table;
  double scale;
  int64_t padding;
  if (n != 4 || !plain_context() || !tensor_arg(a[0], &tokens) || !tensor_arg(a[1], &table) || !float_arg(a[2], &scale) ||
      !int_arg(a[3], -1, kIntMax, &padding))
    Py_RETURN_NONE;
  if (!index_dtype(*tokens) || !tokens->is_contiguous() || tokens->numel() == 0 || table->dim() != 2 ||
      dtype_code(*table) < 0 || table->numel() == 0 || !table->is_contiguous() || table->device() != tokens->device() ||
      table->size(0) > kIntMax || table->size(1) > kIntMax)
    Py_RETURN_NONE;
  return unlocked([&] {
    return recorded({table}) ? EmbeddingFn::apply(*tokens, *table, scale, padding)
                             : EmbeddingFn::launch(*tokens, *table, scale);
  });
}

PyObject* py_linear_cross_entropy(Args a, Py_ssize_t n) {
  const Tensor *x, *w, *targets;
  int64_t ignore_index, reduction;
  if (n != 5 || !plain_context() || !tensor_arg(a[0], &x) || !tensor_arg(a[1], &w) || !tensor_arg(a[2], &targets) ||
      !int_arg(a[3], INT64_MIN, INT64_MAX, &ignore_index) || !int_arg(a[4], 0, 2, &reduction))
    Py_RETURN_NONE;
  if (x->dim() != 2 || w->dim() != 2 || (x->scalar_type() != at::kBFloat16 && x->scalar_type() != at::kHalf) ||
      w->scalar_type() != x->scalar_type() || w->size(1) != x->size(1) || x->numel() == 0 || w->numel() == 0 ||
      x->size(1) % 64 || x->size(1) > kIntMax || w->size(0) > kIntMax || !x->is_contiguous() || !w->is_contiguous() ||
      !aligned16(*x) || !aligned16(*w) || !index_dtype(*targets) || targets->dim() != 1 ||
      targets->size(0) != x->size(0) || !targets->is_contiguous() || w->device() != x->device() ||
      targets->device() != x->device())
    Py_RETURN_NONE;
  return unlocked([&] {
    return recorded({x, w}) ? LinearCrossEntropyFn::apply(*x, *w, *targets, ignore_index, reduction)
                            : LinearCrossEntropyFn::launch(*x, *w, *targets, ignore_index, reduction).first;
  });
}

// x [rows, n], residual (may be null) like it and w [n], contiguous, of one type and device, some rows.
bool plain_rows(const Tensor& x, const Tensor* residual, const Tensor& w) {
  if (x.dim() != 2 || !x.is_contiguous() || x.numel() == 0 || dtype_code(x) < 0 || x.size(1) > kIntMax) return false;
  if (residual && (residual->scalar_type() != x.scalar_type() || residual->sizes() != x.sizes() ||
                   !residual->is_contiguous() || residual->device() != x.device()))
    return false;
  return w.scalar_type() == x.scalar_type() && w.dim() == 1 && w.size(0) == x.size(1) && w.is_contiguous() &&
         w.device() == x.device();
}

PyObject* py_add_rmsnorm(Args a, Py_ssize_t n) {
  const Tensor *x, *residual, *w;
  double eps;
  if (n != 4 || !plain_context() || !tensor_arg(a[0], &x) || !tensor_arg(a[1], &residual) || !tensor_arg(a[2], &w) ||
      !float_arg(a[3], &eps) || !plain_rows(*x, residual, *w))
    Py_RETURN_NONE;
  return unlocked_tuple([&] {
    return recorded({x, residual, w}) ? AddRmsNormFn::apply(*x, *residual, *w, eps)
                                      : AddRmsNormFn::launch(*x, *residual, *w, eps, nullptr);
  });
}

PyObject* py_add_rmsnorm_8bit(Args a, Py_ssize_t n) {
  const Tensor *x, *residual = nullptr, *w;
  double eps;
  if (n != 4 || !plain_context() || !tensor_arg(a[0], &x) || (a[1] != Py_None && !tensor_arg(a[1], &residual)) ||
      !tensor_arg(a[2], &w) || !float_arg(a[3], &eps) || !plain_rows(*x, residual, *w))
    Py_RETURN_NONE;
  return unlocked_tuple([&]() -> variable_list {
    const c10::DeviceGuard guard(x->device());
    Tensor q = at::empty(x->sizes(), x->options().dtype(at::kFloat8_e4m3fn)),
           scale = at::empty({x->size(0)}, x->options().dtype(at::kFloat)), r;
    if (residual) r = at::empty(x->sizes(), x->options());
    forward_status(krsi_add_rmsnorm_8bit(x->data_ptr(), residual ? residual->data_ptr() : nullptr, w->data_ptr(),
                                         q.data_ptr(), scale.data_ptr<float>(), residual ? r.data_ptr() : nullptr,
                                         x->size(0), (int)x->size(1), (float)eps, dtype_code(*x), stream_of(*x)));
    return {q, scale, r};
  });
}

// Codes and scales of the rows of x.
variable_list rows_in_8bit(const Tensor& x) {
  Tensor q = at::empty(x.sizes(), x.options().dtype(at::kFloat8_e4m3fn)),
         scale = at::empty({x.size(0)}, x.options().dtype(at::kFloat));
  forward_status(krsi_quantize_rows(x.data_ptr(), q.data_ptr(), scale.data_ptr<float>(), x.size(0), (int)x.size(1),
                                    dtype_code(x), stream_of(x)));
  return {q, scale};
}

PyObject* py_quantize_rows(Args a, Py_ssize_t n) {
  const Tensor* x;
  if (n != 1 || !plain_context() || !tensor_arg(a[0], &x) || x->dim() != 2 || !x->is_contiguous() || x->numel() == 0 ||
      dtype_code(*x) < 0 || x->size(1) > kIntMax)
    Py_RETURN_NONE;
  return unlocked_tuple([&] {
    at::NoGradGuard no_grad;
    const c10::DeviceGuard guard(x->device());
    return rows_in_8bit(*x);
  });
}

// x in 8 bits with its rows' scales, or (no scales) of another type, brought to 8 bits here.
PyObject* py_linear_8bit(Args a, Py_ssize_t n) {
  const Tensor *x, *w, *w_scale, *x_scale = nullptr;
  int64_t out_dtype;
  if (n != 5 || !plain_context() || !tensor_arg(a[0], &x) || !tensor_arg(a[1], &w) || !tensor_arg(a[2], &w_scale) ||
      (a[3] != Py_None && !tensor_arg(a[3], &x_scale)) || !int_arg(a[4], 0, 2, &out_dtype))
    Py_RETURN_NONE;
  if (x->dim() != 2 || w->dim() != 2 || w->scalar_type() != at::kFloat8_e4m3fn || w->size(1) != x->size(1) ||
      x->numel() == 0 || w->numel() == 0 || x->size(1) % 16 || x->size(1) > kIntMax || w->size(0) > kIntMax ||
      !x->is_contiguous() || !w->is_contiguous() || !aligned16(*w) || w->device() != x->device() ||
      (x_scale ? x->scalar_type() != at::kFloat8_e4m3fn || !aligned16(*x) : dtype_code(*x) < 0))
    Py_RETURN_NONE;
  auto scales = [&](const Tensor* s, int64_t rows) {
    return s->scalar_type() == at::kFloat && s->dim() == 1 && s->size(0) == rows && s->is_contiguous() &&
           s->device() == x->device();
  };
  if (!scales(w_scale, w->size(0)) || (x_scale && !scales(x_scale, x->size(0)))) Py_RETURN_NONE;
  return unlocked([&] {
    at::NoGradGuard no_grad;
    const c10::DeviceGuard guard(x->device());
    variable_list rows = x_scale ? variable_list{*x, *x_scale} : rows_in_8bit(*x);
    const at::ScalarType types[] = {at::kBFloat16, at::kHalf, at::kFloat};
    Tensor out = at::empty({x->size(0), w->size(0)}, x->options().dtype(types[out_dtype]));
    const size_t bytes = krsi_linear_8bit_workspace_bytes(x->size(0), (int)x->size(1), (int)w->size(0));
    Tensor ws;
    if (bytes) ws = at::empty({(int64_t)bytes}, x->options().dtype(at::kByte));
    forward_status(krsi_linear_8bit(rows[0].data_ptr(), w->data_ptr(), rows[1].data_ptr<float>(),
                                    w_scale->data_ptr<float>(), out.data_ptr(), bytes ? ws.data_ptr() : nullptr, bytes, x->size(0), (int)x->size(1),
                                    (int)w->size(0), (int)out_dtype, stream_of(*x)));
    return out;
  });
}

// A list of tensors (or None, where `holes` has none of them) that are plain, contiguous and on one device.
bool list_arg(PyObject* o, bool holes, std::vector<const Tensor*>* out) {
  if (!PyList_CheckExact(o)) return false;
  const Py_ssize_t n = PyList_GET_SIZE(o);
  out->resize(n);
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* item = PyList_GET_ITEM(o, i);
    if (holes && item == Py_None) {
      (*out)[i] = nullptr;
      continue;
    }
    if (!tensor_arg(item, &(*out)[i]) || !(*out)[i]->is_contiguous()) return false;
  }
  return true;
}

Tensor norm_of(const std::vector<const Tensor*>& grads, const Tensor& like, int dtype) {
  std::vector<const void*> ptrs;
  std::vector<int64_t> sizes;
  for (const Tensor* g : grads)
    if (g) {
      ptrs.push_back(g->data_ptr());
      sizes.push_back(g->numel());
    }
  const int count = (int)ptrs.size();
  Tensor norm = at::empty({}, like.options().dtype(at::kFloat));
  const size_t bytes = krsi_grad_norm_workspace_bytes(sizes.data(), count);
  Tensor ws = at::empty({(int64_t)bytes}, like.options().dtype(at::kByte));
  forward_status(krsi_grad_norm(ptrs.data(), sizes.data(), count, norm.data_ptr<float>(), ws.data_ptr(), bytes, dtype,
                                stream_of(like)));
  return norm;
}

PyObject* py_grad_norm(Args a, Py_ssize_t n) {
  std::vector<const Tensor*> grads;
  if (n != 1 || !plain_context() || !list_arg(a[0], true, &grads)) Py_RETURN_NONE;
  const Tensor* first = nullptr;
  for (const Tensor* g : grads) {
    if (!g) continue;
    if (!first) first = g;
    if (g->scalar_type() != first->scalar_type() || g->device() != first->device()) Py_RETURN_NONE;
  }
  if (!first || dtype_code(*first) < 0 || grads.size() > (1u << 20)) Py_RETURN_NONE;
  return unlocked([&] {
    at::NoGradGuard no_grad;
    const c10::DeviceGuard guard(first->device());
    return norm_of(grads, *first, dtype_code(*first));
  });
}

// One step; (norm,) with None for no norm.
PyObject* py_adamw_step(Args a, Py_ssize_t n) {
  std::vector<const Tensor*> params, grads, m, v, masters, scales;
  const Tensor *steps, *lr_at = nullptr, *norm_arg = nullptr;
  double lr = 0, b1, b2, eps, decay, max_norm = 0;
  int64_t seed;
  if (n != 15 || !plain_context() || !list_arg(a[0], false, &params) || !list_arg(a[1], true, &grads) ||
      !list_arg(a[2], false, &m) || !list_arg(a[3], false, &v) || !tensor_arg(a[4], &steps) ||
      (!float_arg(a[5], &lr) && !tensor_arg(a[5], &lr_at)) || !float_arg(a[6], &b1) || !float_arg(a[7], &b2) ||
      !float_arg(a[8], &eps) || !float_arg(a[9], &decay) || (a[10] != Py_None && !list_arg(a[10], false, &masters)) ||
      (a[11] != Py_None && !list_arg(a[11], false, &scales)) || (a[12] != Py_None && !float_arg(a[12], &max_norm)) ||
      (a[13] != Py_None && !tensor_arg(a[13], &norm_arg)) || !int_arg(a[14], 0, 0xffffffff, &seed))
    Py_RETURN_NONE;
  const size_t count = params.size();
  const bool with_masters = a[10] != Py_None, with_scales = a[11] != Py_None, clip = a[12] != Py_None;
  if (!count || count > (1u << 20) || grads.size() != count || m.size() != count || v.size() != count ||
      (with_masters && masters.size() != count) || (with_scales && scales.size() != count))
    Py_RETURN_NONE;
  const auto device = params[0]->device();
  const auto type = params[0]->scalar_type(), state = with_scales ? at::kFloat8_e4m3fn : at::kFloat;
  const int dt = dtype_code(*params[0]);
  auto one = [&](const Tensor* t) { return t->scalar_type() == at::kFloat && t->numel() == 1 && t->device() == device; };
  if (dt < 0 || steps->scalar_type() != at::kInt || steps->dim() != 1 || steps->size(0) != (int64_t)count ||
      !steps->is_contiguous() || steps->device() != device || (lr_at && !one(lr_at)) || (norm_arg && !one(norm_arg)))
    Py_RETURN_NONE;
  const Tensor* first = nullptr;
  std::vector<void*> pp(count), mp(count), vp(count);
  std::vector<const void*> gp(count);
  std::vector<float*> wp(with_masters ? count : 0), sp(with_scales ? count : 0);
  std::vector<int64_t> sizes(count);
  auto fits = [&](const Tensor* t, at::ScalarType kind, const Tensor* p) {
    return t->scalar_type() == kind && t->sizes() == p->sizes() && t->device() == device;
  };
  for (size_t i = 0; i < count; ++i) {
    const Tensor *p = params[i], *g = grads[i];
    if (!fits(p, type, p) || !fits(m[i], state, p) || !fits(v[i], state, p)) Py_RETURN_NONE;
    if (g) {
      if (!first) first = g;
      if (!fits(g, first->scalar_type(), p)) Py_RETURN_NONE;
      // An empty tensor has no address; one that is not null says that its gradient is there.
      gp[i] = g->numel() ? g->data_ptr() : steps->data_ptr();
    }
    pp[i] = p->data_ptr(), mp[i] = m[i]->data_ptr(), vp[i] = v[i]->data_ptr(), sizes[i] = p->numel();
    if (with_masters) {
      if (!fits(masters[i], at::kFloat, p)) Py_RETURN_NONE;
      wp[i] = masters[i]->data_ptr<float>();
    }
    if (with_scales) {
      const Tensor* s = scales[i];
      if (s->scalar_type() != at::kFloat || s->dim() != 2 || s->size(0) != 2 || s->size(1) != (sizes[i] + 255) / 256 ||
          s->device() != device)
        Py_RETURN_NONE;
      sp[i] = s->data_ptr<float>();
    }
  }
  const int gdt = first ? dtype_code(*first) : dt;
  if (gdt != dt && gdt != KRSI_DTYPE_F32) Py_RETURN_NONE;
  return unlocked_tuple([&]() -> variable_list {
    at::NoGradGuard no_grad;
    const c10::DeviceGuard guard(device);
    Tensor norm;
    if (norm_arg) norm = *norm_arg;
    if (clip && !norm.defined()) norm = at::empty({}, params[0]->options().dtype(at::kFloat));
    const size_t bytes = krsi_adamw_workspace_bytes(sizes.data(), (int)count);
    Tensor ws = at::empty({(int64_t)bytes}, params[0]->options().dtype(at::kByte));
    in_place_status(krsi_adamw_step(pp.data(), gp.data(), mp.data(), vp.data(), with_masters ? wp.data() : nullptr,
                                    with_scales ? sp.data() : nullptr, sizes.data(), (int)count, steps->data_ptr<int32_t>(),
                                    lr_at ? lr_at->data_ptr<float>() : nullptr, (float)lr, b1, b2, (float)eps, (float)decay,
                                    norm.defined() ? norm.data_ptr<float>() : nullptr, norm_arg ? 1 : 0, (float)max_norm,
                                    (uint32_t)seed, with_scales ? 8 : 32, dt, gdt, ws.data_ptr(), bytes, stream_of(*params[0])));
    // What a graph has saved of these counts as changed, but for tensors that had no gradient.
    auto changed = [](const Tensor& t) {
      if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
    };
    changed(*steps);
    for (const auto* list : {&params, &m, &v, &masters, &scales})
      for (size_t i = 0; i < list->size(); ++i)
        if (grads[i]) changed(*(*list)[i]);
    return {norm};
  });
}

PyObject* py_set_module(PyObject*, PyObject* m) {
  Py_XDECREF(g_hip_module);
  Py_INCREF(m);
  g_hip_module = m;
  Py_RETURN_NONE;
}

PyMethodDef kMethods[] = {
    {"rmsnorm", (PyCFunction)(void*)entry<py_rmsnorm>, METH_FASTCALL, nullptr},
    {"geglu", (PyCFunction)(void*)entry<py_geglu>, METH_FASTCALL, nullptr},
    {"geglu_linear", (PyCFunction)(void*)entry<py_geglu_linear>, METH_FASTCALL, nullptr},
    {"relpos_attention", (PyCFunction)(void*)entry<py_relpos_attention>, METH_FASTCALL, nullptr},
    {"bucket_table", (PyCFunction)(void*)entry<py_bucket_table>, METH_FASTCALL, nullptr},
    {"qk_norm_rope", (PyCFunction)(void*)entry<py_qk_norm_rope>, METH_FASTCALL, nullptr},
    {"embedding", (PyCFunction)(void*)entry<py_embedding>, METH_FASTCALL, nullptr},
    {"linear_cross_entropy", (PyCFunction)(void*)entry<py_linear_cross_entropy>, METH_FASTCALL, nullptr},
    {"add_rmsnorm", (PyCFunction)(void*)entry<py_add_rmsnorm>, METH_FASTCALL, nullptr},
    {"add_rmsnorm_8bit", (PyCFunction)(void*)entry<py_add_rmsnorm_8bit>, METH_FASTCALL, nullptr},
    {"quantize_rows", (PyCFunction)(void*)entry<py_quantize_rows>, METH_FASTCALL, nullptr},
    {"linear_8bit", (PyCFunction)(void*)entry<py_linear_8bit>, METH_FASTCALL, nullptr},
    {"grad_norm", (PyCFunction)(void*)entry<py_grad_norm>, METH_FASTCALL, nullptr},
    {"adamw_step", (PyCFunction)(void*)entry<py_adamw_step>, METH_FASTCALL, nullptr},
    {"set_module", py_set_module, METH_O, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_krsi_native", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// built_for: the torch, Python and krsi.h this file was compiled against, which its loader compares with its own.
PyMODINIT_FUNC PyInit__krsi_native() {
  PyObject* m = PyModule_Create(&kModule);
  PyObject* v = m ? Py_BuildValue("(siii)", KRSI_TORCH_VERSION, PY_MAJOR_VERSION, PY_MINOR_VERSION, KRSI_ABI_VERSION)
                  : nullptr;
  if (!v || PyModule_AddObject(m, "built_for", v) < 0) {
    Py_XDECREF(v);
    Py_XDECREF(m);
    return nullptr;
  }
  return m;
}
