// The functions that join a decoder block's halves (residual norm, gated product, their backward passes, low-rank adapters), issued from native code.
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
    ctx->save_for_backward({y, out[0], weight, post.value_or(at::Tensor()), gate.value_or(at::Tensor()), out[2], out[3]});
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
    refuse_foreign_leaves("residual_norm");
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

// Rows that the tiles can read, of whole 16-byte pieces: t where it lies so, else a copy, its rows padded with zeros.
at::Tensor whole_pieces(const at::Tensor& t, int64_t* ld) {
  const at::Tensor rows = as_rows(t, ld);
  const int64_t k = t.size(-1), m = t.numel() / k, padded = (k + 7) / 8 * 8;
  const void* const p = rows.const_data_ptr();
  if (k == padded && *ld % 8 == 0 && *ld < NPAMD_TILE_MAX_STRIDE && ((uintptr_t)p & 15) == 0) return rows;
  at::Tensor copy = empty({m, padded}, t.scalar_type(), t.get_device());
  TORCH_CHECK(npamd_gather_columns(p, *ld, nullptr, copy.data_ptr(), padded, (int)m, (int)k, current_stream(t.get_device())) == NPAMD_OK, npamd_last_error());
  *ld = padded;
  return copy;
}

at::Tensor last_dimension(const at::Tensor& t, int64_t n) {
  c10::SmallVector<int64_t, 6> sizes(t.sizes().begin(), t.sizes().end());
  sizes.back() = n;
  return empty(sizes, t.scalar_type(), t.get_device());
}

// h and, with keep, pre; of tensors that have been checked.
std::array<at::Tensor, 2> gated_forward(const at::Tensor& x, const at::Tensor& w, const at::Tensor& bias, int activation, bool keep) {
  const int k = (int)x.size(-1), m = (int)(x.numel() / k), n = (int)(w.size(0) / 2), code = dtype_code(x.scalar_type()), device = x.get_device();
  // Odd K or row distances: few tokens read W as it lies, once for every four of them; past that a copy in whole pieces takes less (us as it lies / with the copy: 8 tokens 14336 x 4095 118 / 140,
  // 8192 x 2047 34 / 38; 9 tokens 148 / 141, 46 / 38, 2739 x 2183 23 / 20, but 515 x 2311 8.9 / 13.0; 20 tokens 255 / 143, 75 / 39, 35 / 21, 13.3 / 13.8).
  const bool pieces = m > ((int64_t)n * k >= 1 << 21 ? 8 : 20);
  int64_t ldx, ldw;
  const at::Tensor xr = pieces ? whole_pieces(x, &ldx) : as_rows(x, &ldx), wr = pieces ? whole_pieces(w, &ldw) : as_rows(w, &ldw);
  const at::Tensor b = bias.defined() ? bias.contiguous() : at::Tensor();
  const int columns = pieces ? (k + 7) / 8 * 8 : k;
  std::array<at::Tensor, 2> out{last_dimension(x, n), keep ? last_dimension(x, 2 * (int64_t)n) : at::Tensor()};
  const int64_t bytes = npamd_gated_linear_workspace_bytes(m, n, columns);
  at::Tensor scratch;
  if (bytes > 0) scratch = floats(bytes, device);
  TORCH_CHECK(npamd_gated_linear(xr.const_data_ptr(), ldx, wr.const_data_ptr(), ldw, data_or_null(b), b.defined() ? dtype_code(b.scalar_type()) : NPAMD_F32, activation,
                                 out[0].data_ptr(), n, out_or_null(out[1]), 2 * (int64_t)n, m, n, columns, code, out_or_null(scratch), bytes, current_stream(device)) == NPAMD_OK,
              npamd_last_error());
  return out;
}

// The gradients of x, gate_up and bias that are needed, the last in `bias_type`.
std::array<at::Tensor, 3> gated_backward(const at::Tensor& dh, const at::Tensor& x, const at::Tensor& w, const at::Tensor& pre, int activation, at::ScalarType bias_type,
                                         const bool (&need)[3]) {
  const int k = (int)x.size(-1), m = (int)(x.numel() / k), n = (int)(w.size(0) / 2), code = dtype_code(x.scalar_type()), device = x.get_device();
  int64_t lddh, ldp, ldx = 0, ldw = 0;
  const at::Tensor dhr = as_rows(dh, &lddh), pr = as_rows(pre, &ldp);
  const at::Tensor wr = need[0] ? whole_pieces(w, &ldw) : at::Tensor(), xr = need[1] ? whole_pieces(x, &ldx) : at::Tensor();
  std::array<at::Tensor, 3> out;
  if (need[0]) out[0] = empty(x.sizes(), x.scalar_type(), device);
  if (need[1]) out[1] = empty(w.sizes(), x.scalar_type(), device);
  if (need[2]) out[2] = empty({2 * (int64_t)n}, bias_type, device);
  if (!need[0] && !need[1] && !need[2]) return out;
  const int64_t bytes = npamd_gated_linear_backward_workspace_bytes(m, n, k, need[0], need[1], need[2]);
  const at::Tensor scratch = floats((bytes + 3) / 4 * 4, device);
  TORCH_CHECK(npamd_gated_linear_backward(dhr.const_data_ptr(), lddh, data_or_null(xr), ldx, data_or_null(wr), ldw, pr.const_data_ptr(), ldp, activation, out_or_null(out[0]), k,
                                          out_or_null(out[1]), k, out_or_null(out[2]), dtype_code(bias_type), m, n, k, code, scratch.data_ptr(), bytes,
                                          current_stream(device)) == NPAMD_OK, npamd_last_error());
  return out;
}

// gate_up [2 N, K] for x's rows.
bool gated_weight(PyObject* o, const Rows& x, int device, Rows* w) {
  return x.code != NPAMD_F32 && rows_argument(o, device, w) && w->code == x.code && w->t->dim() == 2 && w->width == x.width && w->m % 2 == 0;
}

int activation_of(PyObject* o) { return PyLong_Check(o) ? (int)PyLong_AsLong(o) : -1; }

// gated_linear(x, gate_up, bias, activation's number, pre?): h, with pre (h, pre), or None
PyObject* gated_linear(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 5) {
    PyErr_SetString(PyExc_TypeError, "gated_linear(x, gate_up, bias, activation, pre)");
    return nullptr;
  }
  return translated([&]() -> PyObject* {
    const int device = device_of(args[0]);
    Rows x, w;
    if (!PyBool_Check(args[4]) || activation_of(args[3]) < 0 || !rows_argument(args[0], device, &x) || !gated_weight(args[1], x, device, &w)) Py_RETURN_NONE;
    const void* p;
    if (!vector_of(args[2], device, x.t->scalar_type(), w.m, &p) && !vector_of(args[2], device, at::kFloat, w.m, &p)) Py_RETURN_NONE;
    const bool keep = args[4] == Py_True;
    auto out = gated_forward(*x.t, *w.t, is_none(args[2]) ? at::Tensor() : THPVariable_Unpack(args[2]), activation_of(args[3]), keep);
    return keep ? wrap_all({out[0], out[1]}) : THPVariable_Wrap(std::move(out[0]));
  });
}

// gated_linear_backward(dh, x, gate_up, pre, activation's number, bias in float32?, dx?, dgate_up?, dbias?): the gradients, or None
PyObject* gated_linear_backward(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 9) {
    PyErr_SetString(PyExc_TypeError, "gated_linear_backward(dh, x, gate_up, pre, activation, 4 booleans)");
    return nullptr;
  }
  return translated([&]() -> PyObject* {
    const int device = device_of(args[1]);
    Rows dh, x, w, pre;
    if (activation_of(args[4]) < 0 || !rows_argument(args[1], device, &x) || !gated_weight(args[2], x, device, &w)) Py_RETURN_NONE;
    if (!rows_argument(args[0], device, &dh) || !rows_argument(args[3], device, &pre) || dh.code != x.code || pre.code != x.code) Py_RETURN_NONE;
    const auto lead = [](const Rows& r) { return r.t->sizes().slice(0, r.t->dim() - 1); };
    if (lead(dh) != lead(x) || lead(pre) != lead(x) || 2 * dh.width != w.m || pre.width != w.m) Py_RETURN_NONE;
    for (int i = 5; i < 9; ++i)
      if (!PyBool_Check(args[i])) Py_RETURN_NONE;
    const bool need[3] = {args[6] == Py_True, args[7] == Py_True, args[8] == Py_True};
    auto out = gated_backward(*dh.t, *x.t, *w.t, *pre.t, activation_of(args[4]), args[5] == Py_True ? at::kFloat : x.t->scalar_type(), need);
    return wrap_all({out[0], out[1], out[2]});
  });
}

// The gated product in a recorded graph; arguments that Python has checked.  First derivatives only.
struct GatedLinearNode : torch::autograd::Function<GatedLinearNode> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w, const std::optional<at::Tensor>& bias, int64_t activation) {
    const c10::DeviceGuard guard(x.device());
    const auto out = gated_forward(x, w, bias.value_or(at::Tensor()), (int)activation, true);
    ctx->save_for_backward({x, w, out[1]});
    ctx->saved_data["activation"] = activation;
    if (bias) ctx->saved_data["bias"] = (int64_t)bias->scalar_type();  // all that its gradient needs of it
    return out[0];
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const torch::autograd::variable_list saved = ctx->get_saved_variables();
    const bool recorded = c10::GradMode::is_enabled();
    const at::Tensor &x = saved[0], &w = saved[1], &pre = saved[2];
    const auto bias = ctx->saved_data.find("bias");
    const bool biased = bias != ctx->saved_data.end();
    const c10::DeviceGuard guard(x.device());
    refuse_foreign_leaves("gated_linear");
    torch::autograd::variable_list result(4);
    std::array<at::Tensor, 3> out;
    {
      const c10::AutoGradMode off(false);
      const bool need[3] = {ctx->needs_input_grad(0), ctx->needs_input_grad(1), biased && ctx->needs_input_grad(2)};
      out = gated_backward(grads[0], x, w, pre, (int)ctx->saved_data["activation"].toInt(), biased ? (at::ScalarType)bias->second.toInt() : at::kFloat, need);
    }
    for (int i = 0; i < 3; ++i) result[i] = recorded ? final_gradient("gated_linear: its backward pass cannot be differentiated", out[i]) : out[i];
    return result;
  }
};

// gated_linear_recorded(x, gate_up, bias, activation's number): tensors (or None) that Python has checked, on one device
PyObject* gated_linear_recorded(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 4 || !THPVariable_Check(args[0]) || !THPVariable_Check(args[1]) || activation_of(args[3]) < 0) {
    PyErr_SetString(PyExc_TypeError, "gated_linear_recorded(x, gate_up, bias, activation)");
    return nullptr;
  }
  return translated([&]() -> PyObject* {
    return THPVariable_Wrap(GatedLinearNode::apply(THPVariable_Unpack(args[0]), THPVariable_Unpack(args[1]), maybe_tensor(args[2]), (int64_t)activation_of(args[3])));
  });
}

// adapter_linear(x, ids, a, b, scale, base, columns of x, columns of y): y, or None; a, b and scale are those of LowRankAdapters, which has checked them
PyObject* adapter_linear(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 8) {
    PyErr_SetString(PyExc_TypeError, "adapter_linear(x, ids, a, b, scale, base, columns of x, columns of y)");
    return nullptr;
  }
  return translated([&]() -> PyObject* {
    const int device = device_of(args[0]);
    Rows x, base{nullptr, 0, 0, 0, 0};
    if (!rows_argument(args[0], device, &x) || !PyLong_Check(args[6]) || !PyLong_Check(args[7]) || x.width != PyLong_AsLong(args[6])) Py_RETURN_NONE;
    const at::Tensor *ids = readable(args[1], device), *a = readable(args[2], device), *b = readable(args[3], device);
    if (!ids || !a || !b || !ids->is_contiguous() || (ids->scalar_type() != at::kInt && ids->scalar_type() != at::kLong)) Py_RETURN_NONE;
    const at::IntArrayRef lead = x.t->sizes().slice(0, x.t->dim() - 1);
    if (ids->dim() > (int64_t)lead.size() || ids->sizes() != lead.slice(0, ids->dim())) Py_RETURN_NONE;
    at::Tensor spread;  // one for each token, where there is one for each sequence of several
    if (ids->numel() != x.m) {
      c10::SmallVector<int64_t, 6> ones(ids->sizes().begin(), ids->sizes().end());
      ones.resize(lead.size(), 1);
      const c10::DeviceGuard guard(x.t->device());
      spread = ids->view(ones).expand(lead).contiguous();
      ids = &spread;
    }
    const void* scale;
    if (a->scalar_type() != x.t->scalar_type() || !vector_of(args[4], device, at::kFloat, a->size(0), &scale)) Py_RETURN_NONE;
    c10::SmallVector<int64_t, 6> sizes(x.t->sizes().begin(), x.t->sizes().end());
    sizes.back() = PyLong_AsLong(args[7]);
    if (!is_none(args[5]) && (!rows_argument(args[5], device, &base) || base.code != x.code || base.t->sizes() != at::IntArrayRef(sizes))) Py_RETURN_NONE;
    const int m = (int)x.m, cols = (int)sizes.back(), rank = (int)a->size(1), adapters = (int)a->size(0);
    const at::Tensor xr = whole_pieces(*x.t, &x.ld);
    const int k = ((int)x.width + 7) / 8 * 8;
    const int64_t bytes = npamd_adapter_linear_workspace_bytes(m, cols, k, rank, adapters);
    at::Tensor scratch, y = empty(sizes, x.t->scalar_type(), device);
    if (bytes > 0) scratch = floats(bytes, device);
    TORCH_CHECK(npamd_adapter_linear(xr.const_data_ptr(), x.ld, ids->const_data_ptr(), ids->scalar_type() == at::kInt ? 32 : 64, a->const_data_ptr(), b->const_data_ptr(),
                                     (const float*)scale, base.t ? base.t->const_data_ptr() : nullptr, base.ld, y.data_ptr(), cols, m, cols, k, rank, adapters, x.code,
                                     out_or_null(scratch), bytes, current_stream(device)) == NPAMD_OK, npamd_last_error());
    return THPVariable_Wrap(std::move(y));
  });
}

}  // namespace
