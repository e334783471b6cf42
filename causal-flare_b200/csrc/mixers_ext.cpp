// Host layer of the convolution, scan and attention operators in native code, as host_ext.cpp is for the FLARE operators: argument
// checks of the usual calls, output and workspace allocation, the argument structs of the C ABI and the autograd nodes.
//
// Why: through Python (autograd.Function, a ctypes struct filled field by field, a size query and an allocation per buffer) a
// single-token call kept the host busy for 20 to 50 us and a training step for 150 to 200 us on a B200 host, more than the kernels of every small
// call take.  Every entry point here returns None for anything but the plain case (empty tensors, types or shapes that must raise, wrapped
// tensors, traces); the Python layer then serves the call and words the errors.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <string.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <climits>
#include <cmath>
#include <optional>
#include <string>

#include "../../include/flare_b200_mixers.h"

namespace {

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Api {
  decltype(&flare_conv_forward) conv_forward = nullptr, conv_backward = nullptr, conv_decode = nullptr;
  decltype(&flare_conv_backward_workspace_bytes) conv_backward_workspace_bytes = nullptr;
  decltype(&flare_scan_forward) scan_forward = nullptr, scan_backward = nullptr, scan_decode = nullptr;
  decltype(&flare_scan_keep_bytes) scan_keep_bytes = nullptr, scan_forward_workspace_bytes = nullptr, scan_backward_workspace_bytes = nullptr;
  decltype(&flare_attention_forward) attention_forward = nullptr, attention_backward = nullptr;
  decltype(&flare_attention_plan_bytes) attention_plan_bytes = nullptr;
  decltype(&flare_attention_forward_workspace_bytes) attention_forward_workspace_bytes = nullptr, attention_backward_workspace_bytes = nullptr;
  decltype(&flare_attention_append) attention_append = nullptr, attention_decode = nullptr;
  decltype(&flare_attention_decode_workspace_bytes) attention_decode_workspace_bytes = nullptr;
  decltype(&flare_status_string) status_string = nullptr;
  decltype(&flare_last_cuda_error) last_cuda_error = nullptr;
} api;

template <typename F>
void take(F& f, const py::dict& table, const char* name) {
  f = reinterpret_cast<F>(table[name].cast<uintptr_t>());
}

void bind(const py::dict& table) {
  decltype(&flare_mixers_abi_sizeof) size = nullptr;
  take(size, table, "flare_mixers_abi_sizeof");
  if (size(0) != sizeof(flare_conv_args_t) || size(1) != sizeof(flare_scan_args_t) || size(2) != sizeof(flare_attention_args_t) ||
      size(3) != sizeof(flare_cache_args_t))
    throw std::runtime_error("the native host layer was built for another version of the library");
  take(api.conv_forward, table, "flare_conv_forward");
  take(api.conv_backward, table, "flare_conv_backward");
  take(api.conv_decode, table, "flare_conv_decode");
  take(api.conv_backward_workspace_bytes, table, "flare_conv_backward_workspace_bytes");
  take(api.scan_forward, table, "flare_scan_forward");
  take(api.scan_backward, table, "flare_scan_backward");
  take(api.scan_decode, table, "flare_scan_decode");
  take(api.scan_keep_bytes, table, "flare_scan_keep_bytes");
  take(api.scan_forward_workspace_bytes, table, "flare_scan_forward_workspace_bytes");
  take(api.scan_backward_workspace_bytes, table, "flare_scan_backward_workspace_bytes");
  take(api.attention_forward, table, "flare_attention_forward");
  take(api.attention_backward, table, "flare_attention_backward");
  take(api.attention_plan_bytes, table, "flare_attention_plan_bytes");
  take(api.attention_forward_workspace_bytes, table, "flare_attention_forward_workspace_bytes");
  take(api.attention_backward_workspace_bytes, table, "flare_attention_backward_workspace_bytes");
  take(api.attention_append, table, "flare_attention_append");
  take(api.attention_decode, table, "flare_attention_decode");
  take(api.attention_decode_workspace_bytes, table, "flare_attention_decode_workspace_bytes");
  take(api.status_string, table, "flare_status_string");
  take(api.last_cuda_error, table, "flare_last_cuda_error");
}

// the exception classes of the Python binding (workspace and CUDA failures: RuntimeError, the rest: ValueError)
void check(int status, const char* what) {
  if (status == FLARE_OK) return;
  std::string msg = std::string(what) + " failed: " + api.status_string(status);
  if (status == FLARE_ERR_CUDA) msg += std::string(": ") + api.last_cuda_error();
  msg += " (status " + std::to_string(status) + ")";
  if (status == FLARE_ERR_WORKSPACE || status == FLARE_ERR_CUDA) throw std::runtime_error(msg);
  throw c10::ValueError({__func__, __FILE__, static_cast<uint32_t>(__LINE__)}, msg);
}

// ---- tensors -----------------------------------------------------------------------------------------------------------

int dtype_code(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return FLARE_F32;
    case at::kBFloat16: return FLARE_BF16;
    case at::kHalf: return FLARE_F16;
    default: return -1;
  }
}

// Dense CUDA storage, and nothing that a call past the Python autograd functions would lose: no wrapper of a function transform or of
// a Python tensor class, no forward-mode tangent.
bool ordinary(const Tensor& t) {
  constexpr c10::DispatchKeySet wrapped({c10::DispatchKey::Python, c10::DispatchKey::FuncTorchBatched,
                                         c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::Functionalize});
  return t.defined() && t.is_cuda() && t.layout() == at::kStrided && !t.key_set().has_any(wrapped) && !t._fw_grad(/*level=*/0).defined();
}
// (an undefined tensor is an argument that was not given)
bool like(const Tensor& t, const Tensor& x) {
  return !t.defined() || (ordinary(t) && t.device() == x.device() && t.scalar_type() == x.scalar_type());
}
bool fp32(const Tensor& t, const Tensor& x) {
  return !t.defined() || (ordinary(t) && t.device() == x.device() && t.scalar_type() == at::kFloat);
}
bool vector(const Tensor& t, int64_t n) { return !t.defined() || (t.dim() == 1 && t.size(0) == n); }
bool same_sizes(const Tensor& t, const Tensor& x) { return !t.defined() || t.sizes() == x.sizes(); }

// an optional argument; false: something else than None or a tensor
bool tensor_or_none(const py::object& o, Tensor* out) {
  if (o.is_none()) return true;
  if (!THPVariable_Check(o.ptr())) return false;
  *out = THPVariable_Unpack(o.ptr());
  return true;
}
// Whole numbers as the kernels read them; false: the Python layer has to look.  Ids of 64 bits need not fit 32: documents are numbered anew,
// in the order of their runs.
bool whole(const py::object& o, const Tensor& x, at::IntArrayRef sizes, Tensor* out, bool ids = false) {
  Tensor t;
  if (!tensor_or_none(o, &t)) return false;
  if (!t.defined()) return true;
  if (!ordinary(t) || t.device() != x.device() || t.sizes() != sizes) return false;
  const auto type = t.scalar_type();
  if (type != at::kInt && type != at::kLong) return false;
  if (type == at::kLong && ids) {
    const int64_t n = t.size(1) - 1;
    Tensor runs = at::zeros(sizes, t.options().dtype(at::kInt));
    if (n > 0) runs.narrow(1, 1, n).copy_(t.narrow(1, 1, n).ne(t.narrow(1, 0, n)).cumsum(1, at::kInt));
    *out = runs.masked_fill_(t.lt(0), -1);
  } else {
    *out = (type == at::kLong ? t.clamp(-1, INT_MAX) : t).to(at::kInt).contiguous();
  }
  return true;
}
// what a kernel wrote in place has a new version: autograd notices graphs that hold the old one
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
Tensor rows(const Tensor& t) { return !t.defined() || t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous(); }
Tensor dense(const Tensor& t) { return t.defined() ? t.contiguous() : t; }
Tensor aligned(const Tensor& t) { return t.is_contiguous() && (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) == 0 ? t : t.clone(at::MemoryFormat::Contiguous); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
template <typename T>
T* ptr(const Tensor& t) { return t.defined() ? reinterpret_cast<T*>(t.data_ptr()) : nullptr; }

bool fits(int64_t n) { return n <= INT_MAX; }
bool tracing() { return torch::jit::tracer::isTracing(); }

flare_stream_t stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }
Tensor bytes(size_t n, const Tensor& x) {
  return n ? at::empty({(int64_t)n}, x.options().dtype(at::kByte).requires_grad(false)) : Tensor();
}
template <typename A>
Tensor workspace(A& a, size_t need, const Tensor& x) {  // (stream-ordered memory: free once the launches are enqueued)
  const Tensor ws = bytes(need, x);
  a.workspace = ptr(ws);
  a.workspace_bytes = need;
  return ws;
}
Tensor new_like(const Tensor& t) { return at::empty(t.sizes(), t.options().requires_grad(false).memory_format(at::MemoryFormat::Contiguous)); }

// (an autograd node takes arguments that may be missing in this form)
using Maybe = std::optional<Tensor>;
Maybe maybe(const Tensor& t) { return t.defined() ? Maybe(t) : Maybe(); }
Tensor given(const Maybe& t) { return t.has_value() ? *t : Tensor(); }

template <typename... Ts>
bool wants_grad(const Ts&... ts) {
  return at::GradMode::is_enabled() && ((ts.defined() && ts.requires_grad()) || ...);
}

// Gradients that cannot be differentiated again say so when somebody tries (what torch's once_differentiable does).
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list marked;
  for (auto& g : grads)
    if (g.defined()) marked.push_back(g.detach().requires_grad_());
  if (marked.empty()) return grads;
  const int n = (int)marked.size();
  auto out = (*std::make_shared<torch::autograd::DelayedError>("trying to differentiate twice a function that was marked with @once_differentiable", n))(
      std::move(marked));
  size_t at = 0;
  for (auto& g : grads)
    if (g.defined()) g = out[at++];
  return grads;
}

bool number(const py::object& o, double* out) {
  PyObject* const f = PyNumber_Float(o.ptr());
  if (f == nullptr) {
    PyErr_Clear();
    return false;
  }
  *out = PyFloat_AS_DOUBLE(f);
  Py_DECREF(f);
  return true;
}

// ---- convolution -------------------------------------------------------------------------------------------------------

int activation_of(const py::object& o) {
  if (o.is_none()) return FLARE_IDENTITY;
  if (PyUnicode_Check(o.ptr()) && PyUnicode_CompareWithASCIIString(o.ptr(), "silu") == 0) return FLARE_SILU;
  return -1;
}
bool plain_conv(const Tensor& x, const Tensor& w, const Tensor& b, int dims) {
  if (tracing() || !ordinary(x) || !ordinary(w) || x.dim() != dims || x.numel() == 0 || dtype_code(x) < 0 || dtype_code(w) < 0) return false;
  const int64_t C = x.size(-1);
  return w.device() == x.device() && like(b, w) && w.dim() == 2 && w.size(0) == C && w.size(1) >= 2 && w.size(1) <= 4 && vector(b, C) &&
         fits(x.size(0)) && fits(C) && (dims == 2 || fits(x.size(1)));
}
// w, b: contiguous
void fill_conv(flare_conv_args_t& a, const Tensor& x, const Tensor& w, const Tensor& b, int act) {
  memset(&a, 0, sizeof(a));
  a.x = x.data_ptr(); a.weight = w.data_ptr(); a.bias = ptr(b);
  a.B = (int32_t)x.size(0); a.N = x.dim() == 3 ? (int32_t)x.size(1) : 1; a.C = (int32_t)x.size(-1); a.W = (int32_t)w.size(1);
  a.x_stride_b = x.stride(0); a.x_stride_n = x.dim() == 3 ? x.stride(1) : 0;
  a.dtype = dtype_code(x); a.weight_dtype = dtype_code(w); a.activation = act;
}
Tensor run_conv(const Tensor& x0, const Tensor& w, const Tensor& b, int act, const Tensor& documents) {
  const Tensor x = rows(x0), wc = dense(w), bc = dense(b), y = new_like(x0);
  flare_conv_args_t a;
  fill_conv(a, x, wc, bc, act);
  a.documents = ptr<int32_t>(documents);
  a.y = y.data_ptr();
  check(api.conv_forward(&a, stream_of(x)), "flare_conv_forward");
  return y;
}

struct ConvNode : public torch::autograd::Function<ConvNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Maybe& b_, int64_t act, const Maybe& documents_) {
    const Tensor b = given(b_), documents = given(documents_);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, w, b, documents});
    ctx->saved_data["act"] = act;
    return {run_conv(x, w, b, (int)act, documents)};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(5);
    if (!grads[0].defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const c10::cuda::CUDAGuard guard(saved[0].device());
    const Tensor x = rows(saved[0]), w = dense(saved[1]), b = dense(saved[2]), dy = rows(grads[0]);
    flare_conv_args_t a;
    fill_conv(a, x, w, b, (int)ctx->saved_data["act"].toInt());
    a.documents = ptr<int32_t>(saved[3]);
    a.dy = dy.data_ptr();
    a.dy_stride_b = dy.stride(0); a.dy_stride_n = dy.stride(1);
    out[0] = new_like(saved[0]);
    out[1] = new_like(saved[1]);
    if (b.defined()) out[2] = new_like(saved[2]);
    a.dx = out[0].data_ptr(); a.dweight = out[1].data_ptr(); a.dbias = ptr(out[2]);
    const Tensor ws = workspace(a, api.conv_backward_workspace_bytes(&a), x);
    check(api.conv_backward(&a, stream_of(x)), "flare_conv_backward");
    return once(out);
  }
};

py::object conv(const Tensor& x, const Tensor& w, const py::object& bias, const py::object& activation, const py::object& documents) {
  Tensor b, ids;
  const int act = activation_of(activation);
  if (act < 0 || !tensor_or_none(bias, &b) || !plain_conv(x, w, b, 3)) return py::none();
  const c10::cuda::CUDAGuard guard(x.device());
  if (!whole(documents, x, x.sizes().slice(0, 2), &ids, true)) return py::none();
  if (wants_grad(x, w, b)) return py::cast(ConvNode::apply(x, w, maybe(b), (int64_t)act, maybe(ids))[0]);
  return py::cast(run_conv(x, w, b, act, ids));
}

py::object conv_prefill(const Tensor& x0, const Tensor& w, const py::object& bias, const py::object& state, const py::object& activation,
                        const py::object& lengths) {
  Tensor b, st, len;
  const int act = activation_of(activation);
  if (act < 0 || !tensor_or_none(bias, &b) || !tensor_or_none(state, &st) || !plain_conv(x0, w, b, 3) || !like(st, x0)) return py::none();
  const int64_t B = x0.size(0), C = x0.size(2), W = w.size(1);
  if (st.defined() && st.sizes() != at::IntArrayRef({B, W - 1, C})) return py::none();
  const c10::cuda::CUDAGuard guard(x0.device());
  if (!whole(lengths, x0, x0.sizes().slice(0, 1), &len)) return py::none();
  const Tensor x = rows(x0), wc = dense(w), bc = dense(b), sc = dense(st), y = new_like(x0);
  const Tensor out = at::empty({B, W - 1, C}, x.options().requires_grad(false));
  flare_conv_args_t a;
  fill_conv(a, x, wc, bc, act);
  a.lengths = ptr<int32_t>(len);
  a.state_in = ptr(sc); a.state_out = out.data_ptr(); a.y = y.data_ptr();
  check(api.conv_forward(&a, stream_of(x)), "flare_conv_forward");
  return py::make_tuple(y, out);
}

py::object conv_decode(const Tensor& x_in, const Tensor& w, const py::object& bias, const py::object& state, const py::object& activation) {
  Tensor b, st;
  const int act = activation_of(activation);
  if (act < 0 || !tensor_or_none(bias, &b) || !tensor_or_none(state, &st) || !st.defined() || !x_in.is_cuda()) return py::none();
  const Tensor x0 = x_in.dim() == 3 && x_in.size(1) == 1 ? x_in.select(1, 0) : x_in;
  if (!plain_conv(x0, w, b, 2) || !like(st, x0) || st.requires_grad() || !st.is_contiguous() || st.sizes() != at::IntArrayRef({x0.size(0), w.size(1) - 1, x0.size(1)}))
    return py::none();
  const c10::cuda::CUDAGuard guard(x0.device());
  const Tensor x = rows(x0), wc = dense(w), bc = dense(b), y = new_like(x_in);
  flare_conv_args_t a;
  fill_conv(a, x, wc, bc, act);
  a.state_out = st.data_ptr(); a.y = y.data_ptr();
  check(api.conv_decode(&a, stream_of(x)), "flare_conv_decode");
  written(st);
  return py::make_tuple(y, state);
}

// ---- scan --------------------------------------------------------------------------------------------------------------

struct ScanInputs {
  Tensor x, dt, A, B, C, D, z, bias;  // B, C: [..., G, S]
  bool softplus = false;
};
bool plain_scan(ScanInputs& s, int dims) {
  const Tensor& x = s.x;
  if (tracing() || !ordinary(x) || x.dim() != dims || x.numel() == 0 || dtype_code(x) < 0) return false;
  if (!s.dt.defined() || !s.A.defined() || !s.B.defined() || !s.C.defined()) return false;
  if (!like(s.dt, x) || !like(s.B, x) || !like(s.C, x) || !like(s.z, x) || !fp32(s.A, x) || !fp32(s.D, x) || !fp32(s.bias, x)) return false;
  const int64_t C = x.size(-1);
  if (s.A.dim() != 2 || s.A.size(0) != C || !same_sizes(s.dt, x) || !same_sizes(s.z, x) || !vector(s.D, C) || !vector(s.bias, C)) return false;
  const int64_t S = s.A.size(1);
  if (S != 8 && S != 16 && S != 32) return false;
  if (s.B.dim() == dims) s.B = s.B.unsqueeze(-2);
  if (s.C.dim() == dims) s.C = s.C.unsqueeze(-2);
  if (s.B.dim() != dims + 1 || s.B.sizes() != s.C.sizes() || s.B.size(-1) != S) return false;
  for (int i = 0; i + 1 < dims; ++i)
    if (s.B.size(i) != x.size(i) || !fits(x.size(i))) return false;
  const int64_t G = s.B.size(-2);
  return G >= 1 && C % G == 0 && fits(C);
}
struct ScanHeld {
  Tensor x, dt, A, B, C, D, z, bias;
};
ScanHeld fill_scan(flare_scan_args_t& a, const ScanInputs& s) {
  ScanHeld h{rows(s.x), rows(s.dt), aligned(s.A), rows(s.B), rows(s.C), dense(s.D), rows(s.z), dense(s.bias)};
  memset(&a, 0, sizeof(a));
  const bool tokens = h.x.dim() == 3;
  a.x = h.x.data_ptr(); a.dt = h.dt.data_ptr(); a.z = ptr(h.z); a.b = h.B.data_ptr(); a.c = h.C.data_ptr();
  a.A = ptr<float>(h.A); a.D = ptr<float>(h.D); a.dt_bias = ptr<float>(h.bias);
  a.B = (int32_t)h.x.size(0); a.N = tokens ? (int32_t)h.x.size(1) : 1; a.C = (int32_t)h.x.size(-1); a.S = (int32_t)h.A.size(1); a.G = (int32_t)h.B.size(-2);
  const auto n = [&](const Tensor& t) { return tokens ? t.stride(1) : 0; };
  a.x_stride_b = h.x.stride(0); a.x_stride_n = n(h.x);
  a.dt_stride_b = h.dt.stride(0); a.dt_stride_n = n(h.dt);
  if (h.z.defined()) { a.z_stride_b = h.z.stride(0); a.z_stride_n = n(h.z); }
  a.b_stride_b = h.B.stride(0); a.b_stride_n = n(h.B); a.b_stride_g = h.B.stride(-2);
  a.c_stride_b = h.C.stride(0); a.c_stride_n = n(h.C); a.c_stride_g = h.C.stride(-2);
  a.dtype = dtype_code(h.x); a.dt_softplus = s.softplus;
  return h;
}

struct ScanNode : public torch::autograd::Function<ScanNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C, const Maybe& D_,
                               const Maybe& z_, const Maybe& bias_, bool softplus, const Maybe& documents_) {
    const Tensor D = given(D_), z = given(z_), bias = given(bias_), documents = given(documents_);
    ctx->set_materialize_grads(false);
    flare_scan_args_t a;
    const ScanHeld h = fill_scan(a, {x, dt, A, B, C, D, z, bias, softplus});
    const Tensor y = new_like(x);
    a.documents = ptr<int32_t>(documents);
    a.y = y.data_ptr();
    const Tensor keep = bytes(api.scan_keep_bytes(&a), x);
    a.keep = ptr<float>(keep);
    const Tensor ws = workspace(a, api.scan_forward_workspace_bytes(&a), x);
    check(api.scan_forward(&a, stream_of(x)), "flare_scan_forward");
    ctx->save_for_backward({x, dt, A, B, C, D, z, bias, documents, keep});
    ctx->saved_data["softplus"] = softplus;
    return {y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(10);
    if (!grads[0].defined()) return out;
    const auto s = ctx->get_saved_variables();
    const c10::cuda::CUDAGuard guard(s[0].device());
    flare_scan_args_t a;
    const ScanHeld h = fill_scan(a, {s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7], ctx->saved_data["softplus"].toBool()});
    const Tensor dy = rows(grads[0]);
    a.documents = ptr<int32_t>(s[8]);
    a.keep = ptr<float>(s[9]);
    a.dy = dy.data_ptr();
    a.dy_stride_b = dy.stride(0); a.dy_stride_n = dy.stride(1);
    for (int i = 0; i < 8; ++i)
      if (s[i].defined()) out[i] = new_like(s[i]);
    a.dx = ptr(out[0]); a.ddt = ptr(out[1]); a.dA = ptr<float>(out[2]); a.db = ptr(out[3]); a.dc = ptr(out[4]);
    a.dD = ptr<float>(out[5]); a.dz = ptr(out[6]); a.ddt_bias = ptr<float>(out[7]);
    const Tensor ws = workspace(a, api.scan_backward_workspace_bytes(&a), s[0]);
    check(api.scan_backward(&a, stream_of(s[0])), "flare_scan_backward");
    return once(out);
  }
};

bool scan_inputs(ScanInputs& s, const py::object& D, const py::object& z, const py::object& bias, int dims) {
  return tensor_or_none(D, &s.D) && tensor_or_none(z, &s.z) && tensor_or_none(bias, &s.bias) && plain_scan(s, dims);
}

py::object scan(const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C, const py::object& D, const py::object& z,
                const py::object& bias, bool softplus, const py::object& documents) {
  ScanInputs s{x, dt, A, B, C, Tensor(), Tensor(), Tensor(), softplus};
  Tensor ids;
  if (!scan_inputs(s, D, z, bias, 3)) return py::none();
  const c10::cuda::CUDAGuard guard(x.device());
  if (!whole(documents, x, x.sizes().slice(0, 2), &ids, true)) return py::none();
  if (wants_grad(x, dt, A, B, C, s.D, s.z, s.bias)) return py::cast(ScanNode::apply(x, dt, A, s.B, s.C, maybe(s.D), maybe(s.z), maybe(s.bias), softplus, maybe(ids))[0]);
  flare_scan_args_t a;
  const ScanHeld h = fill_scan(a, s);
  const Tensor y = new_like(x);
  a.documents = ptr<int32_t>(ids);
  a.y = y.data_ptr();
  const Tensor ws = workspace(a, api.scan_forward_workspace_bytes(&a), x);
  check(api.scan_forward(&a, stream_of(x)), "flare_scan_forward");
  return py::cast(y);
}

bool plain_state(const Tensor& st, const ScanInputs& s) {
  return fp32(st, s.x) && (!st.defined() || (!st.requires_grad() && st.is_contiguous() && (reinterpret_cast<uintptr_t>(st.data_ptr()) & 15u) == 0 &&
                                             st.sizes() == at::IntArrayRef({s.x.size(0), s.x.size(-1), s.A.size(1)})));
}

py::object scan_prefill(const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C, const py::object& state, const py::object& D,
                        const py::object& z, const py::object& bias, bool softplus, const py::object& lengths) {
  ScanInputs s{x, dt, A, B, C, Tensor(), Tensor(), Tensor(), softplus};
  Tensor st, len;
  if (!tensor_or_none(state, &st) || !scan_inputs(s, D, z, bias, 3) || !plain_state(st, s)) return py::none();
  const c10::cuda::CUDAGuard guard(x.device());
  if (!whole(lengths, x, x.sizes().slice(0, 1), &len)) return py::none();
  flare_scan_args_t a;
  const ScanHeld h = fill_scan(a, s);
  const Tensor y = new_like(x), out = at::empty({x.size(0), x.size(2), A.size(1)}, A.options().requires_grad(false));
  a.lengths = ptr<int32_t>(len);
  a.state_in = ptr<float>(st); a.state_out = ptr<float>(out); a.y = y.data_ptr();
  const Tensor ws = workspace(a, api.scan_forward_workspace_bytes(&a), x);
  check(api.scan_forward(&a, stream_of(x)), "flare_scan_forward");
  return py::make_tuple(y, out);
}

py::object scan_decode(const Tensor& x_in, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C, const py::object& state, const py::object& D,
                       const py::object& z, const py::object& bias, bool softplus) {
  Tensor st;
  if (!x_in.is_cuda() || x_in.dim() != 2 || !tensor_or_none(state, &st) || !st.defined()) return py::none();
  ScanInputs s{x_in, dt, A, B, C, Tensor(), Tensor(), Tensor(), softplus};
  if (!scan_inputs(s, D, z, bias, 2) || !plain_state(st, s)) return py::none();
  const c10::cuda::CUDAGuard guard(x_in.device());
  flare_scan_args_t a;
  const ScanHeld h = fill_scan(a, s);
  const Tensor y = new_like(x_in);
  a.state_out = ptr<float>(st); a.y = y.data_ptr();
  check(api.scan_decode(&a, stream_of(x_in)), "flare_scan_decode");
  written(st);
  return py::make_tuple(y, state);
}

// ---- attention -----------------------------------------------------------------------------------------------------------

struct Scores {
  double scale = 0.0, cap = 0.0;
  int64_t window = 0;
  Tensor slopes;
};
// rows that tiled copies can fetch where they are
bool tiled_layout(const Tensor& t) {
  if (t.stride(-1) != 1 || (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u)) return false;
  for (int64_t i = 0; i + 1 < t.dim(); ++i)
    if (t.size(i) > 1 && (t.stride(i) <= 0 || t.stride(i) % 8)) return false;
  return true;
}
Tensor tiled(const Tensor& t) { return tiled_layout(t) ? t : t.clone(at::MemoryFormat::Contiguous); }
int64_t step_of(const Tensor& t, int64_t i) { return t.size(i) > 1 ? t.stride(i) : 0; }

bool plain_attention(const Tensor& q, const Tensor& k, const Tensor& v, int dims) {
  if (tracing() || !ordinary(q) || !ordinary(k) || !ordinary(v) || q.dim() != dims || k.dim() != dims || q.numel() == 0 || k.numel() == 0) return false;
  if ((q.scalar_type() != at::kBFloat16 && q.scalar_type() != at::kHalf) || !like(k, q) || !like(v, q) || k.sizes() != v.sizes()) return false;
  const int64_t D = q.size(-1), H = q.size(-2), J = k.size(-2);
  for (int i = 0; i + 2 < dims; ++i)
    if (q.size(i) != k.size(i) || !fits(q.size(i))) return false;
  return k.size(-1) == D && H % J == 0 && D % 8 == 0 && D <= 128;
}
bool score_inputs(const Tensor& q, const py::object& scale, const py::object& cap, const py::object& slopes, const py::object& window, Scores* s) {
  const int64_t D = q.size(-1);
  if (scale.is_none()) s->scale = D <= 8 ? 1.0 : std::pow((double)D, -0.5);
  else if (!number(scale, &s->scale)) return false;
  if (!(s->scale > 0.0) || std::isinf(s->scale)) return false;
  if (!cap.is_none() && (!number(cap, &s->cap) || !(s->cap > 0.0) || s->cap > 1024.0)) return false;
  if (!window.is_none()) {
    if (!PyLong_Check(window.ptr())) return false;
    int overflow = 0;
    s->window = PyLong_AsLongLongAndOverflow(window.ptr(), &overflow);
    if (overflow || s->window < 1) return false;
    if (s->window > INT_MAX) s->window = INT_MAX;
  }
  if (!tensor_or_none(slopes, &s->slopes) || !fp32(s->slopes, q) || !vector(s->slopes, q.size(-2))) return false;
  if (s->slopes.defined()) s->slopes = s->slopes.detach().contiguous();
  return true;
}
bool truth(const py::object& o, const Tensor& x, Tensor* out) {
  Tensor t;
  if (!tensor_or_none(o, &t)) return false;
  if (!t.defined()) return true;
  if (!ordinary(t) || t.device() != x.device() || t.scalar_type() != at::kBool || t.sizes() != x.sizes().slice(0, 2)) return false;
  *out = t.contiguous();
  return true;
}

void fill_attention(flare_attention_args_t& a, const Tensor& q, const Tensor& k, const Tensor& v, const Scores& s, const Tensor& documents,
                    const Tensor& prefix) {
  memset(&a, 0, sizeof(a));
  a.q = q.data_ptr(); a.k = k.data_ptr(); a.v = v.data_ptr();
  a.documents = ptr<int32_t>(documents); a.prefix = ptr<uint8_t>(prefix); a.slopes = ptr<float>(s.slopes);
  a.B = (int32_t)q.size(0); a.Nq = (int32_t)q.size(1); a.Nk = (int32_t)k.size(1); a.H = (int32_t)q.size(2); a.J = (int32_t)k.size(2); a.D = (int32_t)q.size(3);
  a.q_stride_b = step_of(q, 0); a.q_stride_n = step_of(q, 1); a.q_stride_h = step_of(q, 2);
  a.k_stride_b = step_of(k, 0); a.k_stride_n = step_of(k, 1); a.k_stride_h = step_of(k, 2);
  a.v_stride_b = step_of(v, 0); a.v_stride_n = step_of(v, 1); a.v_stride_h = step_of(v, 2);
  a.scale = (float)s.scale; a.cap = (float)s.cap; a.window = (int32_t)s.window; a.dtype = dtype_code(q);
}

struct AttentionNode : public torch::autograd::Function<AttentionNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q0, const Tensor& k0, const Tensor& v0, double scale, double cap, int64_t window,
                               const Maybe& slopes_, const Maybe& documents_, const Maybe& prefix_) {
    const Tensor slopes = given(slopes_), documents = given(documents_), prefix = given(prefix_);
    ctx->set_materialize_grads(false);
    const Tensor q = tiled(q0), k = tiled(k0), v = tiled(v0), y = new_like(q0);
    flare_attention_args_t a;
    fill_attention(a, q, k, v, {scale, cap, window, slopes}, documents, prefix);
    const Tensor lse = at::empty({q.size(0), q.size(2), (q.size(1) + 127) / 128 * 128}, q.options().dtype(at::kFloat).requires_grad(false));
    a.y = y.data_ptr();
    a.lse = ptr<float>(lse);
    const Tensor plan = bytes(api.attention_plan_bytes(&a), q);
    a.plan = ptr(plan);
    const Tensor ws = workspace(a, api.attention_forward_workspace_bytes(&a), q);
    check(api.attention_forward(&a, stream_of(q)), "flare_attention_forward");
    ctx->save_for_backward({q0, k0, v0, y, lse, slopes, documents, prefix, plan});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["cap"] = cap;
    ctx->saved_data["window"] = window;
    return {y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(9);
    if (!grads[0].defined()) return out;
    const auto s = ctx->get_saved_variables();
    const c10::cuda::CUDAGuard guard(s[0].device());
    const Tensor q = tiled(s[0]), k = tiled(s[1]), v = tiled(s[2]), dy = tiled(grads[0]);
    flare_attention_args_t a;
    fill_attention(a, q, k, v, {ctx->saved_data["scale"].toDouble(), ctx->saved_data["cap"].toDouble(), ctx->saved_data["window"].toInt(), s[5]}, s[6], s[7]);
    a.y = s[3].data_ptr();
    a.lse = ptr<float>(s[4]);
    a.plan = ptr(s[8]);
    a.dy = dy.data_ptr();
    a.dy_stride_b = step_of(dy, 0); a.dy_stride_n = step_of(dy, 1); a.dy_stride_h = step_of(dy, 2);
    for (int i = 0; i < 3; ++i) out[i] = new_like(s[i]);
    a.dq = out[0].data_ptr(); a.dk = out[1].data_ptr(); a.dv = out[2].data_ptr();
    const Tensor ws = workspace(a, api.attention_backward_workspace_bytes(&a), q);
    check(api.attention_backward(&a, stream_of(q)), "flare_attention_backward");
    return once(out);
  }
};

py::object attention(const Tensor& q, const Tensor& k, const Tensor& v, const py::object& scale, const py::object& cap, const py::object& slopes,
                     const py::object& window, const py::object& documents, const py::object& prefix) {
  Scores s;
  Tensor ids, led;
  if (!plain_attention(q, k, v, 4) || !score_inputs(q, scale, cap, slopes, window, &s) || !truth(prefix, q, &led)) return py::none();
  if (!slopes.is_none() && wants_grad(THPVariable_Unpack(slopes.ptr()))) return py::none();  // (they have no gradient)
  const c10::cuda::CUDAGuard guard(q.device());
  if (!whole(documents, q, q.sizes().slice(0, 2), &ids, true)) return py::none();
  if (wants_grad(q, k, v)) return py::cast(AttentionNode::apply(q, k, v, s.scale, s.cap, s.window, maybe(s.slopes), maybe(ids), maybe(led))[0]);
  const Tensor qt = tiled(q), kt = tiled(k), vt = tiled(v), y = new_like(q);
  flare_attention_args_t a;
  fill_attention(a, qt, kt, vt, s, ids, led);
  a.y = y.data_ptr();
  const Tensor ws = workspace(a, api.attention_forward_workspace_bytes(&a), q);
  check(api.attention_forward(&a, stream_of(q)), "flare_attention_forward");
  return py::cast(y);
}

bool plain_caches(const Tensor& q, const Tensor& k, const Tensor& kc, const Tensor& vc) {
  return ordinary(kc) && ordinary(vc) && like(kc, q) && like(vc, q) && kc.dim() == 4 && kc.sizes() == vc.sizes() && kc.size(0) == k.size(0) && kc.size(1) >= 1 &&
         fits(kc.size(1)) && kc.size(2) == k.size(-2) && kc.size(3) == k.size(-1) && tiled_layout(kc) && tiled_layout(vc) && !kc.requires_grad() &&
         !vc.requires_grad();
}
void fill_cache(flare_cache_args_t& a, const Tensor& k, const Tensor& v, const Tensor& kc, const Tensor& vc) {
  memset(&a, 0, sizeof(a));
  a.new_k = k.data_ptr(); a.new_v = v.data_ptr(); a.k_cache = kc.data_ptr(); a.v_cache = vc.data_ptr();
  a.B = (int32_t)kc.size(0); a.L = (int32_t)kc.size(1); a.J = (int32_t)kc.size(2); a.D = (int32_t)kc.size(3);
  const int h = k.dim() == 4 ? 2 : 1;
  a.new_k_stride_b = step_of(k, 0); a.new_k_stride_h = step_of(k, h); a.new_k_stride_n = h == 2 ? step_of(k, 1) : 0;
  a.new_v_stride_b = step_of(v, 0); a.new_v_stride_h = step_of(v, h); a.new_v_stride_n = h == 2 ? step_of(v, 1) : 0;
  a.k_stride_b = step_of(kc, 0); a.k_stride_n = step_of(kc, 1); a.k_stride_h = step_of(kc, 2);
  a.v_stride_b = step_of(vc, 0); a.v_stride_n = step_of(vc, 1); a.v_stride_h = step_of(vc, 2);
  a.dtype = dtype_code(k);
}

py::object attention_prefill(const Tensor& q0, const Tensor& k0, const Tensor& v0, const Tensor& kc, const Tensor& vc, const py::object& cached,
                             const py::object& lengths, const py::object& scale, const py::object& cap, const py::object& slopes, const py::object& window,
                             const py::object& prefix) {
  Scores s;
  Tensor at_, len, led;
  if (!plain_attention(q0, k0, v0, 4) || !plain_caches(q0, k0, kc, vc) || !score_inputs(q0, scale, cap, slopes, window, &s) || !truth(prefix, q0, &led))
    return py::none();
  const c10::cuda::CUDAGuard guard(q0.device());
  const auto batch = q0.sizes().slice(0, 1);
  if (!whole(cached, q0, batch, &at_) || !whole(lengths, q0, batch, &len)) return py::none();
  if (!at_.defined()) at_ = at::zeros(batch, q0.options().dtype(at::kInt).requires_grad(false));
  const Tensor q = tiled(q0), k = tiled(k0), v = tiled(v0), y = new_like(q0);
  flare_cache_args_t c;
  fill_cache(c, k, v, kc, vc);
  c.N = (int32_t)q.size(1);
  c.cached = ptr<int32_t>(at_); c.lengths = ptr<int32_t>(len);
  check(api.attention_append(&c, stream_of(q)), "flare_attention_append");
  written(kc);
  written(vc);
  flare_attention_args_t a;
  fill_attention(a, q, kc, vc, s, Tensor(), led);
  a.cached = ptr<int32_t>(at_); a.lengths = ptr<int32_t>(len); a.y = y.data_ptr();
  const Tensor ws = workspace(a, api.attention_forward_workspace_bytes(&a), q);
  check(api.attention_forward(&a, stream_of(q)), "flare_attention_forward");
  return py::cast(y);
}

py::object attention_decode(const Tensor& q_in, const Tensor& k_in, const Tensor& v_in, const Tensor& kc, const Tensor& vc, const py::object& cached,
                            const py::object& scale, const py::object& cap, const py::object& slopes, const py::object& window) {
  const auto token = [](const Tensor& t) { return t.dim() == 4 && t.size(1) == 1 ? t.select(1, 0) : t; };
  const Tensor q0 = token(q_in), k0 = token(k_in), v0 = token(v_in);
  Scores s;
  Tensor at_;
  if (!plain_attention(q0, k0, v0, 3) || !plain_caches(q0, k0, kc, vc) || !score_inputs(q0, scale, cap, slopes, window, &s)) return py::none();
  const c10::cuda::CUDAGuard guard(q0.device());
  if (!whole(cached, q0, q0.sizes().slice(0, 1), &at_) || !at_.defined()) return py::none();
  const Tensor q = tiled(q0), k = tiled(k0), v = tiled(v0), y = new_like(q_in);
  flare_cache_args_t a;
  fill_cache(a, k, v, kc, vc);
  a.q = q.data_ptr(); a.y = y.data_ptr(); a.H = (int32_t)q.size(1);
  a.q_stride_b = step_of(q, 0); a.q_stride_h = step_of(q, 1);
  a.cached = ptr<int32_t>(at_); a.slopes = ptr<float>(s.slopes);
  a.scale = (float)s.scale; a.cap = (float)s.cap; a.window = (int32_t)s.window;
  const Tensor ws = workspace(a, api.attention_decode_workspace_bytes(&a), q);
  check(api.attention_decode(&a, stream_of(q)), "flare_attention_decode");
  written(kc);
  written(vc);
  return py::cast(y);
}

}  // namespace

PYBIND11_MODULE(_mixers_host, m) {
  m.def("bind", &bind);
  m.def("conv", &conv);
  m.def("conv_prefill", &conv_prefill);
  m.def("conv_decode", &conv_decode);
  m.def("scan", &scan);
  m.def("scan_prefill", &scan_prefill);
  m.def("scan_decode", &scan_decode);
  m.def("attention", &attention);
  m.def("attention_prefill", &attention_prefill);
  m.def("attention_decode", &attention_decode);
}
