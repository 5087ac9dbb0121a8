// The gated scan, its step, the update of a list of tensors and the norm of their gradients as methods of `vig_host`, over the C ABI.  Host code only.
//
// As in py_calls.cpp: what bounds a small call is the host.  A list of tensors costs it more than that: 180 parameters with their gradients and two moments
// are 720 addresses, sizes and types, which Python reads in 0.4 ms, twice what the kernels take.
#include "host_calls.h"

#include <c10/hip/HIPGraphsC10Utils.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <deque>
#include <vector>

namespace vig_host {
namespace {

// [B, L, D] (or [B, D]) whose channels lie side by side in rows that do not overlap; anything else is copied.
Tensor rows(const Tensor& t) {
  const int64_t d = t.dim(), pitch = t.stride(d - 2);
  const bool side = t.size(d - 1) == 1 || t.stride(d - 1) == 1;
  return side && (t.size(d - 2) == 1 || (pitch >= t.size(d - 1) && pitch <= (1 << 18))) ? t : t.contiguous();
}
// (batch, token) strides; a row alone is as far from the next as it is wide
struct Strides {
  long long v[2];
  explicit Strides(const Tensor& t) : v{t.size(0) == 1 ? 0 : (long long)t.stride(0), t.size(1) == 1 ? (long long)t.size(2) : (long long)t.stride(1)} {}
};
const void* second(const Tensor& g, bool both) {
  return both ? static_cast<const char*>(g.data_ptr()) + g.size(0) / 2 * g.stride(0) * g.element_size() : nullptr;
}

bool simple(const Tensor& t) { return t.defined() && t.is_cuda() && !t.unsafeGetTensorImpl()->is_python_dispatch() && t.layout() == at::kStrided; }

// What vig_gated_scan_fwd and _bwd take; everything else is ops.py's to word.
bool scan_call(const Tensor& x, const Tensor& g, const Tensor& h0, bool both) {
  if (!simple(x) || !simple(g) || x.dim() != 3 || g.dim() != 3 || g.device() != x.device()) return false;
  if (g.size(0) != x.size(0) * (both ? 2 : 1) || g.size(1) != x.size(1) || g.size(2) != x.size(2)) return false;
  if (dtype_code(x) < 0 || dtype_code(g) < 0) return false;
  if (x.numel() == 0 || x.size(0) > (1 << 30) || x.size(1) > (1 << 24) || x.size(2) > (1 << 18)) return false;
  if (h0.defined() && (both || !simple(h0) || h0.device() != x.device() || h0.scalar_type() != at::kFloat || h0.dim() != 2 || h0.size(0) != x.size(0) ||
                       h0.size(1) != x.size(2)))
    return false;
  return true;
}

struct ScanOutputs {
  Tensor o, final;
};
int scan_forward(const Tensor& x, const Tensor& g, const Tensor& h0, bool both, bool want_final, double out_scale, ScanOutputs& out) {
  const c10::DeviceGuard guard(x.device());
  const int B = (int)x.size(0), L = (int)x.size(1), D = (int)x.size(2);
  out.o = at::empty({B, L, D}, x.options());
  if (want_final) out.final = at::empty({B, D}, x.options().dtype(at::kFloat));
  const size_t need = vig_gated_scan_fwd_workspace(B, L, D, both);
  Tensor ws;
  if (need) ws = bytes_like(need, x);
  const Strides sx(x), sg(g);
  return vig_gated_scan_fwd(x.data_ptr(), g.data_ptr(), second(g, both), h0.defined() ? h0.const_data_ptr<float>() : nullptr, out.o.data_ptr(),
                            want_final ? out.final.data_ptr<float>() : nullptr, need ? ws.data_ptr() : nullptr, need, B, L, D, sx.v, sg.v, (float)out_scale,
                            dtype_code(x), dtype_code(g), stream_of(x));
}

struct GatedScan : torch::autograd::Function<GatedScan> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x0, const Tensor& g0, const std::optional<Tensor>& h, bool both, bool want_final, double out_scale) {
    const Tensor x = rows(x0), g = rows(g0), h0 = h ? h->contiguous() : Tensor();
    ScanOutputs out;
    check_rc(scan_forward(x, g, h0, both, want_final, out_scale, out), "vig_gated_scan_fwd");
    ctx->save_for_backward({x, g, h0});
    ctx->saved_data["both"] = both;
    ctx->saved_data["scale"] = out_scale;
    ctx->set_materialize_grads(false);
    if (want_final) return {out.o, out.final};
    return {out.o};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &g = saved[1], &h0 = saved[2];
    const bool both = ctx->saved_data["both"].toBool();
    const c10::DeviceGuard guard(x.device());
    const int B = (int)x.size(0), L = (int)x.size(1), D = (int)x.size(2);
    const Tensor d_o = grads[0].defined() ? grads[0].contiguous() : at::zeros({B, L, D}, x.options());
    TORCH_CHECK(d_o.scalar_type() == x.scalar_type() && d_o.numel() == x.numel(), "d_o must match the output in shape and dtype");
    const Tensor d_final = grads.size() > 1 && grads[1].defined() ? grads[1].contiguous() : Tensor();
    Tensor dx = at::empty({B, L, D}, x.options()), dg = at::empty({both ? 2 * B : B, L, D}, g.options()), dh0;
    if (h0.defined() && ctx->needs_input_grad(2)) dh0 = at::empty({B, D}, h0.options());
    void* second_dg = both ? static_cast<char*>(dg.data_ptr()) + dg.numel() / 2 * dg.element_size() : nullptr;
    const size_t need = vig_gated_scan_bwd_workspace(B, L, D, both);
    Tensor ws;
    if (need) ws = bytes_like(need, x);
    const Strides sx(x), sg(g);
    check_rc(vig_gated_scan_bwd(x.data_ptr(), g.data_ptr(), second(g, both), h0.defined() ? h0.const_data_ptr<float>() : nullptr, d_o.data_ptr(),
                                d_final.defined() ? d_final.const_data_ptr<float>() : nullptr, dx.data_ptr(), dg.data_ptr(), second_dg,
                                dh0.defined() ? dh0.data_ptr<float>() : nullptr, need ? ws.data_ptr() : nullptr, need, B, L, D, sx.v, sg.v,
                                (float)ctx->saved_data["scale"].toDouble(), dtype_code(x), dtype_code(g), stream_of(x)),
             "vig_gated_scan_bwd");
    if (at::GradMode::is_enabled()) {  // (create_graph: the gradients' own gradients are refused when they are asked for, and not left out of a sum)
      variable_list found;
      for (Tensor* t : {&dx, &dg, &dh0})
        if (t->defined()) found.push_back(t->set_requires_grad(true));
      const auto refuse = std::make_shared<torch::autograd::DelayedError>("gated_scan has no second derivative", (int64_t)found.size());
      found = (*refuse)(variable_list(found));
      dx = found[0], dg = found[1];
      if (dh0.defined()) dh0 = found[2];
    }
    return {dx, dg, dh0, Tensor(), Tensor(), Tensor()};
  }
};

// a tensor of forward-mode differentiation, whose tangent a launch would drop
bool dual(const Tensor& t) { return t.defined() && t._fw_grad(0).defined(); }
bool records(const Tensor& t) { return t.defined() && t.requires_grad(); }

// A leaf's gradient is added up on the stream of the graph that first used it, as long as one lives.  Where that is the default stream a captured backward pass would
// wait there, which breaks the capture in a destructor and ends the process: refused before anything is recorded.
void refuse_held_leaf(const Tensor& t) {
  if (!records(t) || !t.is_leaf()) return;
  const auto held = torch::autograd::impl::try_get_grad_accumulator(t);
  if (!held || !held->stream()) return;
  TORCH_CHECK(held->stream()->id() != c10::hip::getDefaultHIPStream(t.device().index()).id(),
              "gated_scan: a graph recorded on the default stream still holds a leaf that is captured here; drop that graph (its outputs) or detach the leaf first");
}

// What was written behind autograd's back: tensors saved for a backward pass notice.
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

}  // namespace

// gated_scan(x [B, L, D], g, initial state or None, both, want_final): o or (o, final); None: not of that kind
PyObject* gated_scan(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 5, "gated_scan takes 5 arguments");
  if (!is_tensor(a[0]) || !is_tensor(a[1]) || !(a[2] == Py_None || is_tensor(a[2]))) Py_RETURN_NONE;
  const Tensor &x = THPVariable_Unpack(a[0]), &g = THPVariable_Unpack(a[1]), h0 = tensor_arg(a[2]);
  const bool both = PyObject_IsTrue(a[3]), want = PyObject_IsTrue(a[4]);
  if (!scan_call(x, g, h0, both) || (both && want) || observed() || dual(x) || dual(g) || dual(h0)) Py_RETURN_NONE;
  const double out_scale = both ? 0.5 : 1.0;
  Tensor o, final;
  if (at::GradMode::is_enabled() && (records(x) || records(g) || records(h0))) {
    if (c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None)
      for (const Tensor* t : {&x, &g, &h0}) refuse_held_leaf(*t);
    const auto out = GatedScan::apply(x, g, h0.defined() ? std::optional<Tensor>(h0) : std::nullopt, both, want, out_scale);
    o = out[0];
    if (want) final = out[1];
  } else {
    ScanOutputs out;
    const Tensor xr = rows(x), gr = rows(g), hr = h0.defined() ? h0.contiguous() : h0;
    check_rc(scan_forward(xr, gr, hr, both, want, out_scale, out), "vig_gated_scan_fwd");
    o = out.o, final = out.final;
  }
  if (!want) return THPVariable_Wrap(std::move(o));
  PyObject* pair = PyTuple_New(2);
  if (!pair) return nullptr;
  PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(std::move(o)));
  PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(std::move(final)));
  return pair;
  END_HANDLE_TH_ERRORS
}

// refuse_held_leaves(tensors): raises for a leaf that a capture must not take (the caller has asked whether there is one)
PyObject* refuse_held_leaves(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  for (Py_ssize_t i = 0; i < n; ++i) {
    TORCH_CHECK_TYPE(is_tensor(a[i]), "refuse_held_leaves takes tensors");
    refuse_held_leaf(THPVariable_Unpack(a[i]));
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// gated_scan_step(x [B, D], g, state fp32, in place): o; None: not of that kind
PyObject* gated_scan_step(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 3, "gated_scan_step takes 3 arguments");
  for (int i = 0; i < 3; ++i)
    if (!is_tensor(a[i])) Py_RETURN_NONE;
  const Tensor &x = THPVariable_Unpack(a[0]), &g = THPVariable_Unpack(a[1]), &h = THPVariable_Unpack(a[2]);
  if (!simple(x) || !simple(g) || !simple(h) || x.dim() != 2 || g.sizes() != x.sizes() || h.sizes() != x.sizes() || g.device() != x.device() ||
      h.device() != x.device() || dtype_code(x) < 0 || dtype_code(g) < 0 || h.scalar_type() != at::kFloat || !h.is_contiguous() || x.numel() == 0 ||
      x.numel() >= (1LL << 31) - 256 || observed() || dual(x) || dual(g) || dual(h))
    Py_RETURN_NONE;
  if (at::GradMode::is_enabled() && (records(x) || records(g) || records(h))) Py_RETURN_NONE;
  const c10::DeviceGuard guard(x.device());
  const Tensor xr = rows(x), gr = rows(g);
  Tensor o = at::empty(x.sizes(), x.options());
  auto pitch = [](const Tensor& t) { return t.size(0) == 1 ? (long long)t.size(1) : (long long)t.stride(0); };
  check_rc(vig_gated_scan_step(xr.data_ptr(), gr.data_ptr(), h.data_ptr<float>(), o.data_ptr(), (int)x.size(0), (int)x.size(1), pitch(xr), pitch(gr),
                               dtype_code(x), dtype_code(g), stream_of(x)),
           "vig_gated_scan_step");
  written(h);
  return THPVariable_Wrap(std::move(o));
  END_HANDLE_TH_ERRORS
}

namespace {

// The tensors of a list, which holds them for the call; false where something else is among them.
typedef std::vector<const Tensor*> List;
bool tensors(PyObject* o, List& out) {
  if (!PyList_CheckExact(o)) return false;
  const Py_ssize_t n = PyList_GET_SIZE(o);
  out.reserve(n);
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* t = PyList_GET_ITEM(o, i);
    if (!is_tensor(t)) return false;
    out.push_back(&THPVariable_Unpack(t));
  }
  return true;
}
// whether two tensors' elements lie in the same order, without gaps
bool alike(const Tensor& a, const Tensor& b) {
  return &a == &b ? a.is_non_overlapping_and_dense()
                  : a.sizes() == b.sizes() && (a.is_contiguous() ? b.is_contiguous() : a.is_non_overlapping_and_dense() && a.strides() == b.strides());
}

}  // namespace

// adamw(params, grads, moments, moments, scales or None, scales or None, step (int or tensor), lr (float or tensor), beta1, beta2, eps, weight_decay, grad_scale or None,
// seed, first numbers or None): True, or None where ops.py has to see to an argument
PyObject* adamw(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 15, "adamw takes 15 arguments");
  List p, g, m, v, ms, vs;
  const bool bits8 = a[4] != Py_None;
  if (bits8 != (a[5] != Py_None)) Py_RETURN_NONE;
  if (!tensors(a[0], p) || !tensors(a[1], g) || !tensors(a[2], m) || !tensors(a[3], v)) Py_RETURN_NONE;
  if (bits8 && (!tensors(a[4], ms) || !tensors(a[5], vs))) Py_RETURN_NONE;
  const size_t count = p.size();
  if (!count || count > (1u << 30) || g.size() != count || m.size() != count || v.size() != count || (bits8 && (ms.size() != count || vs.size() != count))) Py_RETURN_NONE;
  if (!simple(*p[0]) || observed()) Py_RETURN_NONE;
  const auto dev = p[0]->device();
  auto on_device = [&](PyObject* o, at::ScalarType type, Tensor& t) {  // a number there, or none
    if (!is_tensor(o)) return true;
    t = THPVariable_Unpack(o);
    return simple(t) && t.device() == dev && t.scalar_type() == type && t.numel() == 1;
  };
  Tensor step_t, lr_t, scale_t;
  if (!on_device(a[6], at::kLong, step_t) || !on_device(a[7], at::kFloat, lr_t) || !on_device(a[12], at::kFloat, scale_t)) Py_RETURN_NONE;
  if (a[12] != Py_None && !scale_t.defined()) Py_RETURN_NONE;
  const long long step = step_t.defined() ? 1 : PyLong_AsLongLong(a[6]);
  double x[5];
  for (int i = 0; i < 5; ++i) {
    x[i] = i == 0 && lr_t.defined() ? 0.0 : PyFloat_AsDouble(a[7 + i]);
    if (PyErr_Occurred()) return nullptr;
  }
  const unsigned long long seed = PyLong_AsUnsignedLongLongMask(a[13]);
  if (PyErr_Occurred()) return nullptr;
  std::vector<long long> first;
  if (a[14] != Py_None) {
    if (!PyList_CheckExact(a[14]) || PyList_GET_SIZE(a[14]) != (Py_ssize_t)count) Py_RETURN_NONE;
    first.resize(count);
    for (size_t j = 0; j < count; ++j) first[j] = PyLong_AsLongLong(PyList_GET_ITEM(a[14], j));
    if (PyErr_Occurred()) return nullptr;
  }
  std::vector<void*> pp(count), mp(count), vp(count);
  std::vector<const void*> gp(count);
  std::vector<float*> msp(bits8 ? count : 0), vsp(bits8 ? count : 0);
  std::vector<long long> sizes(count);
  std::vector<int> pd(count), gd(count);
  const auto state = bits8 ? at::kFloat8_e4m3fn : at::kFloat;
  const at::NoGradGuard no_grad;
  const c10::DeviceGuard guard(dev);
  std::deque<Tensor> copies;  // (its elements stay where they are)
  for (size_t j = 0; j < count; ++j) {
    for (const Tensor* t : {p[j], m[j], v[j]})
      if (!simple(*t) || t->device() != dev || !alike(*t, *p[j])) Py_RETURN_NONE;
    if (!simple(*g[j]) || g[j]->device() != dev || g[j]->sizes() != p[j]->sizes()) Py_RETURN_NONE;
    if (!alike(*g[j], *p[j])) {  // (a convolution's weight gradient, channels last)
      copies.push_back(at::empty_like(*p[j], p[j]->options().dtype(g[j]->scalar_type())));
      copies.back().copy_(g[j]->detach());
      g[j] = &copies.back();
    }
    if (m[j]->scalar_type() != state || v[j]->scalar_type() != state) Py_RETURN_NONE;
    sizes[j] = p[j]->numel(), pd[j] = dtype_code(*p[j]), gd[j] = dtype_code(*g[j]);
    if (pd[j] < 0 || gd[j] < 0) Py_RETURN_NONE;
    pp[j] = p[j]->data_ptr(), gp[j] = g[j]->const_data_ptr(), mp[j] = m[j]->data_ptr(), vp[j] = v[j]->data_ptr();
    if (!bits8) continue;
    for (const Tensor* t : {ms[j], vs[j]})
      if (!simple(*t) || t->device() != dev || t->scalar_type() != at::kFloat || !t->is_contiguous() || t->numel() != (sizes[j] + 255) / 256) Py_RETURN_NONE;
    msp[j] = ms[j]->data_ptr<float>(), vsp[j] = vs[j]->data_ptr<float>();
  }
  const int rc = vig_adamw_many(pp.data(), gp.data(), mp.data(), vp.data(), msp.data(), vsp.data(), sizes.data(), first.empty() ? nullptr : first.data(), pd.data(), gd.data(), (int)count, bits8 ? 8 : 32, x[0],
                                x[1], x[2], x[3], x[4], step, lr_t.defined() ? lr_t.const_data_ptr<float>() : nullptr,
                                step_t.defined() ? reinterpret_cast<const long long*>(step_t.const_data_ptr<int64_t>()) : nullptr,
                                scale_t.defined() ? scale_t.const_data_ptr<float>() : nullptr, seed, stream_of(*p[0]));
  if (rc == VIG_EINVAL) Py_RETURN_NONE;
  check_rc(rc, "vig_adamw_many");
  for (const List* list : {&p, &m, &v, &ms, &vs})
    for (const Tensor* t : *list) written(*t);
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// grad_norm(tensors, max_norm or None): (norm, scale or None); None: not of that kind
PyObject* grad_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 2, "grad_norm takes 2 arguments");
  List list;
  if (!tensors(a[0], list) || list.empty() || list.size() > (1u << 30) || !simple(*list[0]) || observed()) Py_RETURN_NONE;
  const Tensor& like = *list[0];
  const bool clip = a[1] != Py_None;
  const double most = clip ? PyFloat_AsDouble(a[1]) : 0.0;
  if (PyErr_Occurred()) return nullptr;
  const size_t count = list.size();
  std::vector<const void*> gp(count);
  std::vector<long long> sizes(count);
  std::vector<int> gd(count);
  for (size_t j = 0; j < count; ++j) {
    const Tensor& g = *list[j];
    if (!simple(g) || g.device() != like.device() || !g.is_non_overlapping_and_dense()) Py_RETURN_NONE;
    gp[j] = g.const_data_ptr(), sizes[j] = g.numel(), gd[j] = dtype_code(g);
    if (gd[j] < 0) Py_RETURN_NONE;
  }
  const c10::DeviceGuard guard(like.device());
  const auto options = like.options().dtype(at::kFloat);
  const size_t need = vig_grad_norm_workspace(sizes.data(), (int)count);
  const Tensor ws = bytes_like(need, like);
  Tensor norm = at::empty({}, options), scale;
  if (clip) scale = at::empty({}, options);
  const int rc = vig_grad_norm(gp.data(), sizes.data(), gd.data(), (int)count, (float)most, norm.data_ptr<float>(), clip ? scale.data_ptr<float>() : nullptr, ws.data_ptr(),
                               need, stream_of(like));
  if (rc == VIG_EINVAL) Py_RETURN_NONE;
  check_rc(rc, "vig_grad_norm");
  PyObject* pair = PyTuple_New(2);
  if (!pair) return nullptr;
  PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(std::move(norm)));
  if (!clip) Py_INCREF(Py_None);
  PyTuple_SET_ITEM(pair, 1, clip ? THPVariable_Wrap(std::move(scale)) : Py_None);
  return pair;
  END_HANDLE_TH_ERRORS
}

}  // namespace vig_host
