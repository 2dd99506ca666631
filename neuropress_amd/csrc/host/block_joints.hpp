// The functions between a decoder block's halves (residual norm and its backward pass), issued from native code.
//
// As in feed_forward.hpp the functions that Python tries first return None for what is not as the kernels want it; Python then checks, reports, copies, and calls them again.
// What the library refuses is an error at once.
#pragma once

namespace {

std::optional<at::Tensor> maybe_tensor(PyObject* o) { return is_none(o) ? std::nullopt : std::optional<at::Tensor>(THPVariable_Unpack(o)); }

PyObject* wrap_or_none(at::Tensor& t) {
  if (t.defined()) return THPVariable_Wrap(std::move(t));
  Py_RETURN_NONE;
}

PyObject* wrap_all(std::initializer_list<at::Tensor> tensors) {
  PyObject* out = PyTuple_New((Py_ssize_t)tensors.size());
  if (!out) return nullptr;
  Py_ssize_t i = 0;
  for (at::Tensor t : tensors) PyTuple_SET_ITEM(out, i++, wrap_or_none(t));
  return out;
}

void* out_or_null(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// Rows of x that share a row of a gate [H], or [..., H] with x's first dimensions and ones behind them; 0: another shape.
int64_t gate_every(const at::Tensor& x, const at::Tensor& gate) {
  const int64_t last = x.dim() - 1, h = x.size(-1);
  if (gate.dim() < 1 || gate.size(-1) != h) return 0;
  if (gate.dim() == 1) return x.numel() / h;
  if (gate.dim() != x.dim()) return 0;
  int64_t i = 0, every = 1;
  while (i < last && gate.size(i) == x.size(i)) ++i;
  for (; i < last; ++i) {
    if (gate.size(i) != 1) return 0;
    every *= x.size(i);
  }
  return every;
}

struct ResidualNormCall {
  at::Tensor x, y, weight, post_weight, gate;  // the last two may be undefined
  double scale, eps;
  int device, m, h, code;
  int64_t every = 1, ldg = 0;
  at::Tensor gate_rows;
  // Of tensors that have been checked.
  ResidualNormCall(const at::Tensor& x_, const at::Tensor& y_, const at::Tensor& weight_, const at::Tensor& post, const at::Tensor& gate_, double scale_, double eps_)
      : x(x_), y(y_), weight(weight_), post_weight(post), gate(gate_), scale(scale_), eps(eps_) {
    device = y.get_device();
    h = (int)y.size(-1);
    m = (int)(y.numel() / h);
    code = dtype_code(y.scalar_type());
    weight = weight.contiguous();
    if (post.defined()) post_weight = post.contiguous();
    if (gate.defined()) {
      every = gate_every(y, gate);
      gate_rows = as_rows(gate, &ldg);
    }
  }
  // stream, normed, post_rstd, rstd
  std::array<at::Tensor, 4> forward(bool stats) const {
    int64_t ldx, ldy;
    const at::Tensor xr = as_rows(x, &ldx), yr = as_rows(y, &ldy);
    std::array<at::Tensor, 4> out;
    out[0] = empty(x.sizes(), x.scalar_type(), device);
    out[1] = empty(x.sizes(), x.scalar_type(), device);
    if (stats) {
      const at::IntArrayRef lead = x.sizes().slice(0, x.dim() - 1);
      if (post_weight.defined()) out[2] = empty(lead, at::kFloat, device);
      out[3] = empty(lead, at::kFloat, device);
    }
    TORCH_CHECK(npamd_residual_norm(xr.const_data_ptr(), ldx, yr.const_data_ptr(), ldy, weight.const_data_ptr(), data_or_null(post_weight), data_or_null(gate_rows), ldg,
                                    (int)every, (float)scale, out[0].data_ptr(), h, out[1].data_ptr(), h, (float*)out_or_null(out[2]), (float*)out_or_null(out[3]), m, h,
                                    (float)eps, code, current_stream(device)) == NPAMD_OK, npamd_last_error());
    return out;
  }
  // The gradients of x, y, weight, post_weight and gate that are needed; `x` is not looked at.
  std::array<at::Tensor, 5> backward(const at::Tensor& dstream, const at::Tensor& dnormed, const at::Tensor& stream, const at::Tensor& post_rstd, const at::Tensor& rstd,
                                     const bool (&need)[5]) const {
    int64_t ldds = 0, lddz = 0, ldy, ldr;
    const at::Tensor ds = dstream.defined() ? as_rows(dstream, &ldds) : at::Tensor(), dz = dnormed.defined() ? as_rows(dnormed, &lddz) : at::Tensor();
    const at::Tensor yr = as_rows(y, &ldy), rr = as_rows(stream, &ldr), pr = post_rstd.defined() ? post_rstd.contiguous() : at::Tensor(), r = rstd.contiguous();
    std::array<at::Tensor, 5> out;
    for (int i = 0; i < 5; ++i) {
      if (!need[i] || (i == 3 && !post_weight.defined()) || (i == 4 && !gate.defined())) continue;
      out[i] = empty(i < 2 ? y.sizes() : i == 4 ? gate.sizes() : weight.sizes(), y.scalar_type(), device);
    }
    const int64_t bytes = npamd_residual_norm_workspace_bytes(m, h, gate.defined() ? (int)every : 0, code);
    at::Tensor scratch;
    if (bytes > 0) scratch = floats(bytes, device);
    TORCH_CHECK(npamd_residual_norm_backward(data_or_null(ds), ldds, data_or_null(dz), lddz, yr.const_data_ptr(), ldy, rr.const_data_ptr(), ldr, weight.const_data_ptr(),
                                             data_or_null(post_weight), data_or_null(gate_rows), ldg, (int)every, (float)scale, (const float*)data_or_null(pr),
                                             r.const_data_ptr<float>(), out_or_null(out[0]), h, out_or_null(out[1]), h, out_or_null(out[2]), out_or_null(out[3]),
                                             out_or_null(out[4]), m, h, code, out_or_null(scratch), bytes, current_stream(device)) == NPAMD_OK, npamd_last_error());
    return out;
  }
};

// The arguments weight, post_weight and gate of a residual norm over x's rows, as the kernels read them.
bool norm_parameters(PyObject* const* args, const Rows& x, int device, at::Tensor (&t)[3]) {
  const void* p;
  const at::ScalarType type = x.t->scalar_type();
  for (int i = 0; i < 3; ++i)
    if (i ? !is_none(args[i]) && !THPVariable_CheckExact(args[i]) : !THPVariable_CheckExact(args[i])) return false;
  if (!vector_of(args[0], device, type, x.width, &p) || !vector_of(args[1], device, type, x.width, &p)) return false;
  t[0] = THPVariable_Unpack(args[0]);
  if (!is_none(args[1])) t[1] = THPVariable_Unpack(args[1]);
  Rows g;
  if (is_none(args[2])) return true;
  if (!rows_argument(args[2], device, &g) || g.code != x.code || !gate_every(*x.t, *g.t)) return false;
  t[2] = *g.t;
  return true;
}

// residual_norm(x, y, weight, post_weight, gate, scale, eps, stats): (stream, normed), with stats (stream, normed, post_rstd, rstd), or None
PyObject* residual_norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 8) {
    PyErr_SetString(PyExc_TypeError, "residual_norm(x, y, weight, post_weight, gate, scale, eps, stats)");
    return nullptr;
  }
  return translated([&]() -> PyObject* {
    const int device = device_of(args[0]);
    Rows x, y;
    at::Tensor t[3];
    if (!PyFloat_Check(args[5]) || !PyFloat_Check(args[6]) || !PyBool_Check(args[7])) Py_RETURN_NONE;
    if (!rows_argument(args[0], device, &x) || !rows_argument(args[1], device, &y) || y.code != x.code || y.t->sizes() != x.t->sizes()) Py_RETURN_NONE;
    if (!norm_parameters(args + 2, x, device, t)) Py_RETURN_NONE;
    const bool stats = args[7] == Py_True;
    auto out = ResidualNormCall(*x.t, *y.t, t[0], t[1], t[2], PyFloat_AS_DOUBLE(args[5]), PyFloat_AS_DOUBLE(args[6])).forward(stats);
    return stats ? wrap_all({out[0], out[1], out[2], out[3]}) : wrap_all({out[0], out[1]});
  });
}

// residual_norm_backward(dstream, dnormed, y, stream, weight, post_weight, gate, scale, post_rstd, rstd, dx?, dy?, dweight?, dpost_weight?, dgate?): the gradients, or None
PyObject* residual_norm_backward(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 15) {
    PyErr_SetString(PyExc_TypeError, "residual_norm_backward(dstream, dnormed, y, stream, weight, post_weight, gate, scale, post_rstd, rstd, 5 booleans)");
    return nullptr;
  }
  return translated([&]() -> PyObject* {
    const int device = device_of(args[2]);
    Rows y, rows;
    at::Tensor t[3], in[3], stat[2];
    if (!PyFloat_Check(args[7]) || !rows_argument(args[2], device, &y)) Py_RETURN_NONE;
    const int from[3] = {0, 1, 3};
    for (int i = 0; i < 3; ++i) {
      if (i < 2 && is_none(args[from[i]])) continue;
      if (!rows_argument(args[from[i]], device, &rows) || rows.code != y.code || rows.t->sizes() != y.t->sizes()) Py_RETURN_NONE;
      in[i] = *rows.t;
    }
    if (!(in[0].defined() || in[1].defined()) || !norm_parameters(args + 4, y, device, t)) Py_RETURN_NONE;
    for (int i = 0; i < 2; ++i) {
      if (i == 0 && !t[1].defined()) continue;
      const at::Tensor* s = readable(args[8 + i], device);
      if (!s || s->scalar_type() != at::kFloat || s->numel() != y.m || !s->is_contiguous()) Py_RETURN_NONE;
      stat[i] = *s;
    }
    bool need[5];
    for (int i = 0; i < 5; ++i) {
      if (!PyBool_Check(args[10 + i])) Py_RETURN_NONE;
      need[i] = args[10 + i] == Py_True;
    }
    auto out = ResidualNormCall(*y.t, *y.t, t[0], t[1], t[2], PyFloat_AS_DOUBLE(args[7]), 0.).backward(in[0], in[1], in[2], stat[0], stat[1], need);
    return wrap_all({out[0], out[1], out[2], out[3], out[4]});
  });
}

// A gradient that a recorded backward pass gives: differentiating it is refused.
at::Tensor final_gradient(const char* message, at::Tensor t) {
  if (!t.defined()) return t;
  return torch::autograd::DelayedError(message, 1).apply(torch::autograd::variable_list{t.requires_grad_(true)})[0];
}

// The residual norm in a recorded graph; arguments that Python has checked.  First derivatives only.
struct ResidualNormNode : torch::autograd::Function<ResidualNormNode> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, const at::Tensor& y, const at::Tensor& weight,
                                                const std::optional<at::Tensor>& post, const std::optional<at::Tensor>& gate, double scale, double eps) {
    const c10::DeviceGuard guard(x.device());
    const auto out = ResidualNormCall(x, y, weight, post.value_or(at::Tensor()), gate.value_or(at::Tensor()), scale, eps).forward(true);
    ctx->set_materialize_grads(false);
    // x itself is needed only where it is a leaf, which a capture asks about.
    ctx->save_for_backward({y, out[0], weight, post.value_or(at::Tensor()), gate.value_or(at::Tensor()), out[2], out[3], x.is_leaf() && x.requires_grad() ? x : at::Tensor()});
    ctx->saved_data["scale"] = scale;
    return {out[0], out[1]};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const torch::autograd::variable_list saved = ctx->get_saved_variables();
    const bool recorded = c10::GradMode::is_enabled();
    torch::autograd::variable_list result(7);
    if (!grads[0].defined() && !grads[1].defined()) return result;
    const at::Tensor &y = saved[0], &stream = saved[1], &weight = saved[2], &post = saved[3], &gate = saved[4];
    const c10::DeviceGuard guard(y.device());
    refuse_foreign_leaves("residual_norm", {saved[7], y, weight, post, gate});
    std::array<at::Tensor, 5> out;
    {
      const c10::AutoGradMode off(false);
      const bool need[5] = {ctx->needs_input_grad(0), ctx->needs_input_grad(1), ctx->needs_input_grad(2), post.defined() && ctx->needs_input_grad(3),
                            gate.defined() && ctx->needs_input_grad(post.defined() ? 4 : 3)};
      out = ResidualNormCall(y, y, weight, post, gate, ctx->saved_data["scale"].toDouble(), 0.).backward(grads[0], grads[1], stream, saved[5], saved[6], need);
    }
    for (int i = 0; i < 5; ++i) result[i] = recorded ? final_gradient("residual_norm: its backward pass cannot be differentiated", out[i]) : out[i];
    return result;
  }
};

// residual_norm_recorded(x, y, weight, post_weight, gate, scale, eps): tensors (or None) that Python has checked, on one device and of one type
PyObject* residual_norm_recorded(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 7 || !THPVariable_Check(args[0]) || !THPVariable_Check(args[1]) || !THPVariable_Check(args[2]) || !PyFloat_Check(args[5]) || !PyFloat_Check(args[6])) {
    PyErr_SetString(PyExc_TypeError, "residual_norm_recorded(x, y, weight, post_weight, gate, scale, eps)");
    return nullptr;
  }
  return translated([&]() -> PyObject* {
    auto out = ResidualNormNode::apply(THPVariable_Unpack(args[0]), THPVariable_Unpack(args[1]), THPVariable_Unpack(args[2]), maybe_tensor(args[3]), maybe_tensor(args[4]),
                                       PyFloat_AS_DOUBLE(args[5]), PyFloat_AS_DOUBLE(args[6]));
    return wrap_all({out[0], out[1]});
  });
}

}  // namespace
