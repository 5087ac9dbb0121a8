// The selective scan, the short causal convolution, their steps and the add and layer norm as methods of `vig_host`, over the C ABI.  Host code only.
//
// As in scan_calls.cpp: one native call for tensors of the kind that the kernels take as they are, None for everything else, which selective.py words or converts.
#include "host_calls.h"

#include <torch/csrc/autograd/functions/basic_ops.h>

#include <initializer_list>

namespace vig_host {
namespace {

const void* ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
const float* floats(const Tensor& t) { return t.defined() ? t.const_data_ptr<float>() : nullptr; }
void* out(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
float* out_floats(const Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }
std::optional<Tensor> given(const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }
Tensor held(const std::optional<Tensor>& t) { return t ? *t : Tensor(); }

// an optional tensor of x's device and of a type
bool fits(const Tensor& t, const Tensor& x, at::ScalarType type, at::IntArrayRef sizes) {
  return !t.defined() || (simple(t) && t.device() == x.device() && t.scalar_type() == type && t.sizes() == sizes);
}
// ... a parameter as the kernels read it
bool numbers(const Tensor& t, const Tensor& x, at::IntArrayRef sizes) { return fits(t, x, at::kFloat, sizes) && (!t.defined() || t.is_contiguous()); }
bool sizes_ok(const Tensor& x) { return x.numel() > 0 && x.size(0) <= (1 << 30) && x.size(x.dim() - 1) <= (1 << 18) && (x.dim() < 3 || x.size(1) <= (1 << 24)); }

typedef std::initializer_list<const Tensor*> Given;
bool any_dual(Given ts) {
  for (const Tensor* t : ts)
    if (dual(*t)) return true;
  return false;
}
// whether the call records a gradient; in a capture leaves that another graph holds are refused
bool recorded(Given ts) {
  if (!at::GradMode::is_enabled()) return false;
  bool any = false;
  for (const Tensor* t : ts) any = any || records(*t);
  if (any && c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None)
    for (const Tensor* t : ts) refuse_held_leaf(*t);
  return any;
}
// (create_graph: the gradients' own gradients are refused when they are asked for, and not left out of a sum)
void refuse_second(std::initializer_list<Tensor*> grads, const char* message) {
  if (!at::GradMode::is_enabled()) return;
  variable_list found;
  for (Tensor* t : grads)
    if (t->defined()) found.push_back(t->detach().set_requires_grad(true));
  found = (*std::make_shared<torch::autograd::DelayedError>(message, (int64_t)found.size()))(variable_list(found));
  size_t i = 0;
  for (Tensor* t : grads)
    if (t->defined()) *t = found[i++];
}

// B or C [.., G, N] with its states side by side in rows that do not overlap; anything else is copied
Tensor shared_rows(const Tensor& given, int64_t dims) {
  const Tensor t = given.dim() == dims ? given.unsqueeze(-2) : given;
  const int64_t G = t.size(-2), N = t.size(-1), apart = G > 1 ? (G - 1) * t.stride(-2) + N : N;
  if ((N > 1 && t.stride(-1) != 1) || (G > 1 && t.stride(-2) < N)) return t.contiguous();
  const int64_t next = dims == 3 && t.size(1) > 1 ? t.stride(1) : apart;  // (a token alone is as far from the next as its groups reach)
  return dims == 3 && (next < apart || next > (1 << 18)) ? t.contiguous() : t;
}
struct SharedStrides {  // batch element, token (where there is one), group
  long long v[3];
  explicit SharedStrides(const Tensor& t) {
    const long long G = t.size(-2), N = t.size(-1), group = G > 1 ? t.stride(-2) : N;
    v[0] = t.size(0) == 1 ? 0 : t.stride(0), v[1] = t.dim() == 3 ? group : t.size(1) == 1 ? (G - 1) * group + N : t.stride(1), v[2] = group;
  }
};

struct Scan {
  Tensor x, delta, A, B, C, D, z, bias, h0;
  bool softplus, reverse;
};
bool shared_ok(const Tensor& t, const Tensor& x, int64_t dims) {
  if (!simple(t) || t.device() != x.device() || t.scalar_type() != x.scalar_type() || (t.dim() != dims && t.dim() != dims + 1)) return false;
  return t.sizes().slice(0, dims - 1) == x.sizes().slice(0, dims - 1) && t.size(-1) >= 1 && t.size(-1) <= 64 && (t.dim() == dims || (t.size(-2) >= 1 && x.size(-1) % t.size(-2) == 0));
}
// whether this is a call that the kernels take; dims: 3, or 2 for one token
bool scan_ok(const Scan& s, int64_t dims) {
  const Tensor& x = s.x;
  if (!simple(x) || x.dim() != dims || dtype_code(x) < 0 || !sizes_ok(x) || !s.delta.defined() || !fits(s.delta, x, x.scalar_type(), x.sizes())) return false;
  if (!shared_ok(s.B, x, dims) || !shared_ok(s.C, x, dims) || s.B.sizes() != s.C.sizes() || !fits(s.z, x, x.scalar_type(), x.sizes())) return false;
  const int64_t D = x.size(-1), N = s.B.size(-1);
  return s.A.defined() && numbers(s.A, x, {D, N}) && numbers(s.D, x, {D}) && numbers(s.bias, x, {D}) && fits(s.h0, x, at::kFloat, {x.size(0), D, N});
}
// rows as they are read
void lay(Scan& s) {
  s.x = rows(s.x), s.delta = rows(s.delta), s.B = shared_rows(s.B, 3), s.C = shared_rows(s.C, 3);
  if (s.z.defined()) s.z = rows(s.z);
  if (s.h0.defined()) s.h0 = s.h0.contiguous();
}

struct ScanOut {
  Tensor o, h, kept;
};
ScanOut scan_forward(const Scan& s, bool want_final, bool keep) {
  const c10::DeviceGuard guard(s.x.device());
  const int batch = (int)s.x.size(0), L = (int)s.x.size(1), D = (int)s.x.size(2), N = (int)s.B.size(3), G = (int)s.B.size(2);
  const auto fp32 = s.x.options().dtype(at::kFloat);
  ScanOut r;
  r.o = at::empty({batch, L, D}, s.x.options());
  if (want_final) r.h = at::empty({batch, D, N}, fp32);
  if (keep) r.kept = bytes_like(vig_selective_scan_kept(batch, L, D, N), s.x);
  const size_t need = vig_selective_scan_fwd_workspace(batch, L, D, N, G);
  Tensor ws;
  if (need) ws = bytes_like(need, s.x);
  const Strides sx(s.x), sd(s.delta), sz(s.z.defined() ? s.z : s.x);
  const SharedStrides sb(s.B), sc(s.C);
  check_rc(vig_selective_scan_fwd(ptr(s.x), ptr(s.delta), floats(s.A), ptr(s.B), ptr(s.C), floats(s.D), ptr(s.z), floats(s.bias), floats(s.h0), out(r.o), out_floats(r.h),
                                  static_cast<float*>(out(r.kept)), out(ws), need, batch, L, D, N, G, sx.v, sd.v, sb.v, sc.v, sz.v, s.softplus, s.reverse, dtype_code(s.x),
                                  stream_of(s.x)),
           "vig_selective_scan_fwd");
  return r;
}

struct SelectiveScan : torch::autograd::Function<SelectiveScan> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& delta, const Tensor& A, const Tensor& B, const Tensor& C, const std::optional<Tensor>& D,
                               const std::optional<Tensor>& z, const std::optional<Tensor>& bias, const std::optional<Tensor>& h0, bool softplus, bool reverse, bool want_final) {
    Scan s{x, delta, A, B, C, held(D), held(z), held(bias), held(h0), softplus, reverse};
    lay(s);
    const ScanOut r = scan_forward(s, want_final, true);
    ctx->save_for_backward({s.x, s.delta, s.A, s.B, s.C, s.D, s.z, s.bias, r.kept});
    // (edges are counted over the tensors that are there)
    const int64_t edge = h0 ? 5 + (D ? 1 : 0) + (z ? 1 : 0) + (bias ? 1 : 0) : -1;
    ctx->saved_data["flags"] = std::vector<int64_t>{softplus, reverse, edge, B.dim()};
    ctx->set_materialize_grads(false);
    if (want_final) return {r.o, r.h};
    return {r.o};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto v = ctx->get_saved_variables();
    const auto flags = ctx->saved_data["flags"].toIntVector();
    const Scan s{v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7], Tensor(), flags[0] != 0, flags[1] != 0};
    const c10::DeviceGuard guard(s.x.device());
    const int batch = (int)s.x.size(0), L = (int)s.x.size(1), D = (int)s.x.size(2), N = (int)s.B.size(3), G = (int)s.B.size(2);
    const Tensor d_o = grads[0].defined() ? grads[0].contiguous() : at::zeros({batch, L, D}, s.x.options());
    TORCH_CHECK(d_o.scalar_type() == s.x.scalar_type() && d_o.numel() == s.x.numel(), "d_o must match the output in shape and dtype");
    const Tensor dh = grads.size() > 1 && grads[1].defined() ? grads[1].contiguous() : Tensor();
    const auto io = s.x.options(), fp32 = io.dtype(at::kFloat);
    Tensor dx = at::empty({batch, L, D}, io), ddelta = at::empty({batch, L, D}, io), dB = at::empty({batch, L, G, N}, io), dC = at::empty({batch, L, G, N}, io), dz, dh0;
    if (s.z.defined()) dz = at::empty({batch, L, D}, io);
    if (flags[2] >= 0 && ctx->needs_input_grad(flags[2])) dh0 = at::empty({batch, D, N}, fp32);
    const Tensor params = at::empty({(int64_t)D * (N + 2)}, fp32);
    const size_t need = vig_selective_scan_bwd_workspace(batch, L, D, N, G);
    const Tensor ws = bytes_like(need, s.x);
    const Strides sx(s.x), sd(s.delta), sz(s.z.defined() ? s.z : s.x);
    const SharedStrides sb(s.B), sc(s.C);
    check_rc(vig_selective_scan_bwd(ptr(s.x), ptr(s.delta), floats(s.A), ptr(s.B), ptr(s.C), floats(s.D), ptr(s.z), floats(s.bias), static_cast<const float*>(ptr(v[8])), ptr(d_o),
                                    floats(dh), out(dx), out(ddelta), out(dB), out(dC), out(dz), out_floats(params), out_floats(dh0), out(ws), need, batch, L, D, N, G, sx.v, sd.v,
                                    sb.v, sc.v, sz.v, s.softplus, s.reverse, dtype_code(s.x), stream_of(s.x)),
             "vig_selective_scan_bwd");
    if (flags[3] == 3) dB = dB.squeeze(2), dC = dC.squeeze(2);
    Tensor dA = params.narrow(0, 0, (int64_t)D * N).view({D, N}), dD, dbias;
    if (s.D.defined()) dD = params.narrow(0, (int64_t)D * N, D);
    if (s.bias.defined()) dbias = params.narrow(0, (int64_t)D * (N + 1), D);
    refuse_second({&dx, &ddelta, &dA, &dB, &dC, &dD, &dz, &dbias, &dh0}, "selective_scan has no second derivative");
    return {dx, ddelta, dA, dB, dC, dD, dz, dbias, dh0, Tensor(), Tensor(), Tensor()};
  }
};

PyObject* one_or_pair(Tensor&& o, Tensor&& h, bool want) {
  if (!want) return THPVariable_Wrap(std::move(o));
  PyObject* pair = PyTuple_New(2);
  if (!pair) return nullptr;
  PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(std::move(o)));
  PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(std::move(h)));
  return pair;
}
// the first `count` arguments, tensors or None
bool tensor_args(PyObject* const* a, int count) {
  for (int i = 0; i < count; ++i)
    if (a[i] != Py_None && !is_tensor(a[i])) return false;
  return true;
}

}  // namespace

// selective_scan(x, delta, A, B, C, D, z, delta_bias, initial_state, softplus, reverse, want_final): o or (o, final); None: not of that kind
PyObject* selective_scan(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 12, "selective_scan takes 12 arguments");
  if (!tensor_args(a, 9)) Py_RETURN_NONE;
  Scan s{tensor_arg(a[0]), tensor_arg(a[1]), tensor_arg(a[2]), tensor_arg(a[3]), tensor_arg(a[4]), tensor_arg(a[5]), tensor_arg(a[6]), tensor_arg(a[7]), tensor_arg(a[8]),
         truth(a[9]), truth(a[10])};
  const bool want = truth(a[11]);
  const Given all = {&s.x, &s.delta, &s.A, &s.B, &s.C, &s.D, &s.z, &s.bias, &s.h0};
  if (!s.x.defined() || !s.B.defined() || !s.C.defined() || !scan_ok(s, 3) || observed() || any_dual(all)) Py_RETURN_NONE;
  if (recorded(all)) {
    auto r = SelectiveScan::apply(s.x, s.delta, s.A, s.B, s.C, given(s.D), given(s.z), given(s.bias), given(s.h0), s.softplus, s.reverse, want);
    return one_or_pair(std::move(r[0]), want ? std::move(r[1]) : Tensor(), want);
  }
  lay(s);
  ScanOut r = scan_forward(s, want, false);
  return one_or_pair(std::move(r.o), std::move(r.h), want);
  END_HANDLE_TH_ERRORS
}

// selective_scan_step(x [B, D], delta, A, B, C, D, z, delta_bias, state fp32 in place, softplus): o; None: not of that kind
PyObject* selective_scan_step(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 10, "selective_scan_step takes 10 arguments");
  if (!tensor_args(a, 9)) Py_RETURN_NONE;
  Scan s{tensor_arg(a[0]), tensor_arg(a[1]), tensor_arg(a[2]), tensor_arg(a[3]), tensor_arg(a[4]), tensor_arg(a[5]), tensor_arg(a[6]), tensor_arg(a[7]), tensor_arg(a[8]),
         truth(a[9]), false};
  const Given all = {&s.x, &s.delta, &s.A, &s.B, &s.C, &s.D, &s.z, &s.bias, &s.h0};
  if (!s.x.defined() || !s.B.defined() || !s.C.defined() || !s.h0.defined() || !s.h0.is_contiguous() || !scan_ok(s, 2) || observed() || any_dual(all)) Py_RETURN_NONE;
  if (at::GradMode::is_enabled())
    for (const Tensor* t : all)
      if (records(*t)) Py_RETURN_NONE;
  const c10::DeviceGuard guard(s.x.device());
  const Tensor x = rows(s.x), delta = rows(s.delta), z = s.z.defined() ? rows(s.z) : Tensor(), B = shared_rows(s.B, 2), C = shared_rows(s.C, 2);
  const int batch = (int)x.size(0), D = (int)x.size(1);
  Tensor o = at::empty({batch, D}, x.options());
  auto pitch = [&](const Tensor& t) { return t.defined() && batch > 1 ? (long long)t.stride(0) : (long long)D; };
  const SharedStrides sb(B), sc(C);
  check_rc(vig_selective_scan_step(ptr(x), ptr(delta), floats(s.A), ptr(B), ptr(C), floats(s.D), ptr(z), floats(s.bias), s.h0.data_ptr<float>(), out(o), batch, D, (int)B.size(-1),
                                   (int)B.size(-2), pitch(x), pitch(delta), sb.v, sc.v, pitch(z), s.softplus, dtype_code(x), stream_of(x)),
           "vig_selective_scan_step");
  written(s.h0);
  return THPVariable_Wrap(std::move(o));
  END_HANDLE_TH_ERRORS
}

namespace {

// weight [D, W] or [D, 1, W]
bool taps_ok(const Tensor& w, const Tensor& x) {
  if (!w.defined() || !simple(w) || w.device() != x.device() || w.scalar_type() != at::kFloat || !w.is_contiguous()) return false;
  if (w.dim() != 2 && (w.dim() != 3 || w.size(1) != 1)) return false;
  return w.size(0) == x.size(-1) && w.size(-1) >= 2 && w.size(-1) <= 4;
}

std::pair<Tensor, Tensor> conv_forward(const Tensor& x, const Tensor& w, const Tensor& b, const Tensor& h0, bool silu, bool reverse, bool want_final) {
  const c10::DeviceGuard guard(x.device());
  const int B = (int)x.size(0), L = (int)x.size(1), D = (int)x.size(2), W = (int)w.size(-1);
  std::pair<Tensor, Tensor> r{at::empty({B, L, D}, x.options()), Tensor()};
  if (want_final) r.second = at::empty({B, W - 1, D}, x.options());
  const Strides sx(x);
  check_rc(vig_causal_conv1d_fwd(ptr(x), floats(w), floats(b), ptr(h0), out(r.first), out(r.second), B, L, D, W, sx.v, silu, reverse, dtype_code(x), stream_of(x)),
           "vig_causal_conv1d_fwd");
  return r;
}

struct CausalConv1d : torch::autograd::Function<CausalConv1d> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x0, const Tensor& w, const std::optional<Tensor>& b, const std::optional<Tensor>& h, bool silu, bool reverse,
                               bool want_final) {
    const Tensor x = rows(x0), h0 = h ? h->contiguous() : Tensor();
    auto r = conv_forward(x, w, held(b), h0, silu, reverse, want_final);
    ctx->save_for_backward({x, w, held(b), h0});
    ctx->saved_data["flags"] = std::vector<int64_t>{silu, reverse};
    ctx->set_materialize_grads(false);
    if (want_final) return {r.first, r.second};
    return {r.first};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto v = ctx->get_saved_variables();
    const auto flags = ctx->saved_data["flags"].toIntVector();
    const Tensor &x = v[0], &w = v[1], &b = v[2], &h0 = v[3];
    const c10::DeviceGuard guard(x.device());
    const int B = (int)x.size(0), L = (int)x.size(1), D = (int)x.size(2), W = (int)w.size(-1);
    const Tensor dy = grads[0].defined() ? grads[0].contiguous() : at::zeros({B, L, D}, x.options());
    TORCH_CHECK(dy.scalar_type() == x.scalar_type() && dy.numel() == x.numel(), "dy must match the output in shape and dtype");
    const Tensor dh = grads.size() > 1 && grads[1].defined() ? grads[1].contiguous() : Tensor();
    const bool want = ctx->needs_input_grad(1) || (b.defined() && ctx->needs_input_grad(2));
    Tensor dx = at::empty({B, L, D}, x.options()), dh0, params, ws, dw, db;
    if (h0.defined() && ctx->needs_input_grad(b.defined() ? 3 : 2)) dh0 = at::empty({B, W - 1, D}, x.options());
    size_t need = 0;
    if (want) {
      params = at::empty({(int64_t)D * (W + 1)}, x.options().dtype(at::kFloat));
      need = vig_causal_conv1d_bwd_workspace(B, L, D, W);
      ws = bytes_like(need, x);
    }
    const Strides sx(x);
    check_rc(vig_causal_conv1d_bwd(ptr(x), floats(w), floats(b), ptr(h0), ptr(dy), ptr(dh), out(dx), out(dh0), out_floats(params), out(ws), need, B, L, D, W, sx.v, (int)flags[0],
                                   (int)flags[1], dtype_code(x), stream_of(x)),
             "vig_causal_conv1d_bwd");
    if (want) {
      dw = params.narrow(0, 0, (int64_t)D * W).view(w.sizes());
      if (b.defined()) db = params.narrow(0, (int64_t)D * W, D);
    }
    refuse_second({&dx, &dw, &db, &dh0}, "causal_conv1d has no second derivative");
    return {dx, dw, db, dh0, Tensor(), Tensor(), Tensor()};
  }
};

}  // namespace

// causal_conv1d(x, weight, bias, initial_state, silu, reverse, want_final): y or (y, final); None: not of that kind
PyObject* causal_conv1d(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 7, "causal_conv1d takes 7 arguments");
  if (!tensor_args(a, 4)) Py_RETURN_NONE;
  const Tensor x = tensor_arg(a[0]), w = tensor_arg(a[1]), b = tensor_arg(a[2]), h0 = tensor_arg(a[3]);
  const bool silu = truth(a[4]), reverse = truth(a[5]), want = truth(a[6]);
  if (!x.defined() || !simple(x) || x.dim() != 3 || dtype_code(x) < 0 || !sizes_ok(x) || !taps_ok(w, x) || !numbers(b, x, {x.size(2)}) ||
      !fits(h0, x, x.scalar_type(), {x.size(0), w.size(-1) - 1, x.size(2)}) || observed())
    Py_RETURN_NONE;
  const Given all = {&x, &w, &b, &h0};
  if (any_dual(all)) Py_RETURN_NONE;
  if (recorded(all)) {
    auto r = CausalConv1d::apply(x, w, given(b), given(h0), silu, reverse, want);
    return one_or_pair(std::move(r[0]), want ? std::move(r[1]) : Tensor(), want);
  }
  auto r = conv_forward(rows(x), w, b, h0.defined() ? h0.contiguous() : h0, silu, reverse, want);
  return one_or_pair(std::move(r.first), std::move(r.second), want);
  END_HANDLE_TH_ERRORS
}

// causal_conv1d_step(x [B, D], weight, state in place, bias, silu): y; None: not of that kind
PyObject* causal_conv1d_step(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 5, "causal_conv1d_step takes 5 arguments");
  if (!tensor_args(a, 4)) Py_RETURN_NONE;
  const Tensor x = tensor_arg(a[0]), w = tensor_arg(a[1]), h = tensor_arg(a[2]), b = tensor_arg(a[3]);
  const bool silu = truth(a[4]);
  if (!x.defined() || !h.defined() || !simple(x) || x.dim() != 2 || dtype_code(x) < 0 || !sizes_ok(x) || !taps_ok(w, x) || !numbers(b, x, {x.size(1)}) ||
      !fits(h, x, x.scalar_type(), {x.size(0), w.size(-1) - 1, x.size(1)}) || !h.is_contiguous() || observed())
    Py_RETURN_NONE;
  const Given all = {&x, &w, &h, &b};
  if (any_dual(all)) Py_RETURN_NONE;
  if (at::GradMode::is_enabled())
    for (const Tensor* t : all)
      if (records(*t)) Py_RETURN_NONE;
  const c10::DeviceGuard guard(x.device());
  const Tensor xr = rows(x);
  const int B = (int)x.size(0), D = (int)x.size(1);
  Tensor y = at::empty({B, D}, x.options());
  check_rc(vig_causal_conv1d_step(ptr(xr), floats(w), floats(b), h.data_ptr(), out(y), B, D, (int)w.size(-1), B > 1 ? xr.stride(0) : D, silu, dtype_code(x), stream_of(x)),
           "vig_causal_conv1d_step");
  written(h);
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

namespace {

struct NormOut {
  Tensor y, sum, stats;
};
NormOut norm_forward(const Tensor& x, const Tensor& w, const Tensor& b, const Tensor& residual, double eps, bool keep) {
  const c10::DeviceGuard guard(x.device());
  const int C = (int)x.size(-1);
  const long long n = x.numel() / C;
  NormOut r{at::empty(x.sizes(), x.options()), residual.defined() ? at::empty(x.sizes(), residual.options()) : x, Tensor()};
  if (keep) r.stats = at::empty({n, 2}, x.options().dtype(at::kFloat));
  check_rc(vig_add_layernorm_fwd(ptr(x), ptr(residual), floats(w), floats(b), residual.defined() ? out(r.sum) : nullptr, out(r.y), out_floats(r.stats), n, C, (float)eps, dtype_code(x),
                                 dtype_code(r.sum), stream_of(x)),
           "vig_add_layernorm_fwd");
  return r;
}

struct AddLayerNorm : torch::autograd::Function<AddLayerNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const std::optional<Tensor>& b, const std::optional<Tensor>& residual, double eps) {
    const NormOut r = norm_forward(x.contiguous(), w, held(b), residual ? residual->contiguous() : Tensor(), eps, true);
    ctx->save_for_backward({r.sum, r.stats, w});
    // (edges are counted over the tensors that are there)
    ctx->saved_data["flags"] = std::vector<int64_t>{(int64_t)x.scalar_type(), b.has_value(), residual ? (b ? 3 : 2) : -1};
    ctx->set_materialize_grads(false);
    if (residual) return {r.y, r.sum};
    return {r.y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto v = ctx->get_saved_variables();
    const auto flags = ctx->saved_data["flags"].toIntVector();
    const Tensor &sum = v[0], &stats = v[1], &w = v[2];
    const auto type = (at::ScalarType)flags[0];
    const c10::DeviceGuard guard(sum.device());
    const int C = (int)sum.size(-1);
    const long long n = sum.numel() / C;
    const Tensor dy = grads[0].defined() ? grads[0].contiguous() : at::zeros(sum.sizes(), sum.options().dtype(type));
    const Tensor dsum = grads.size() > 1 && grads[1].defined() ? grads[1].contiguous() : Tensor();
    TORCH_CHECK(dy.scalar_type() == type && dy.numel() == sum.numel() && (!dsum.defined() || dsum.scalar_type() == sum.scalar_type()), "gradients must match the outputs in shape and dtype");
    const bool want = ctx->needs_input_grad(1) || (flags[1] && ctx->needs_input_grad(2));
    Tensor dx = at::empty(sum.sizes(), sum.options().dtype(type)), dres, params, ws, dw, db;
    // (two who want the gradient of one sum get a buffer each: behind views of leaves autograd keeps both as they are, and adds the next pass's to one memory twice)
    const bool second = flags[2] >= 0 && ctx->needs_input_grad(flags[2]);
    if (type != sum.scalar_type() || (second && ctx->needs_input_grad(0))) dres = at::empty(sum.sizes(), sum.options());
    size_t need = 0;
    if (want) {
      params = at::empty({2 * (int64_t)C}, sum.options().dtype(at::kFloat));
      need = vig_add_layernorm_bwd_workspace(n, C);
      ws = bytes_like(need, sum);
    }
    check_rc(vig_add_layernorm_bwd(ptr(sum), floats(stats), floats(w), ptr(dy), ptr(dsum), out(dres), out(dx), out_floats(params), out(ws), need, n, C, dtype_code(dy), dtype_code(sum),
                                   stream_of(sum)),
             "vig_add_layernorm_bwd");
    if (want) {
      dw = params.narrow(0, 0, C);
      if (flags[1]) db = params.narrow(0, C, C);
    }
    if (second && !dres.defined()) dres = std::move(dx);
    refuse_second({&dx, &dw, &db, &dres}, "add_layernorm has no second derivative");
    return {dx, dw, db, dres, Tensor()};
  }
};

}  // namespace

// add_layernorm(x, weight, bias, residual, eps): y, or (y, sum) with a residual; None: not of that kind
PyObject* add_layernorm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 5, "add_layernorm takes 5 arguments");
  if (!tensor_args(a, 4)) Py_RETURN_NONE;
  const Tensor x = tensor_arg(a[0]), w = tensor_arg(a[1]), b = tensor_arg(a[2]), residual = tensor_arg(a[3]);
  const double eps = PyFloat_AsDouble(a[4]);
  if (PyErr_Occurred()) return nullptr;
  if (!x.defined() || !w.defined() || !simple(x) || x.dim() < 1 || dtype_code(x) < 0 || x.numel() == 0 || x.size(-1) > 16384 || x.numel() / x.size(-1) > (1 << 24) ||
      !numbers(w, x, {x.size(-1)}) || !numbers(b, x, {x.size(-1)}) || !(eps >= 0) || observed())
    Py_RETURN_NONE;
  if (residual.defined() && !fits(residual, x, residual.scalar_type() == at::kFloat ? at::kFloat : x.scalar_type(), x.sizes())) Py_RETURN_NONE;
  const Given all = {&x, &w, &b, &residual};
  if (any_dual(all)) Py_RETURN_NONE;
  if (recorded(all)) {
    auto r = AddLayerNorm::apply(x, w, given(b), given(residual), eps);
    return one_or_pair(std::move(r[0]), residual.defined() ? std::move(r[1]) : Tensor(), residual.defined());
  }
  NormOut r = norm_forward(x.contiguous(), w, b, residual.defined() ? residual.contiguous() : residual, eps, false);
  return one_or_pair(std::move(r.y), std::move(r.sum), residual.defined());
  END_HANDLE_TH_ERRORS
}

}  // namespace vig_host
