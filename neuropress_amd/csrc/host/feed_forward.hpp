// The feed-forward half's functions (layer norm and its backward pass, the dense product with an epilogue, the mixture-of-experts layer), issued from native code.
//
// Small calls are bound by the host: through Python's checks and ctypes a layer norm of one row takes 10 us of host time against 2 us of kernel, its backward pass 20.
// These functions take the calls that are as the kernels want them and return None for all others (a tensor of another kind, type, shape, device or layout, something
// that torch follows, an error of the library): the Python function then goes its ordinary way, which copies, checks and reports.
#pragma once

namespace {

bool is_none(PyObject* o) { return o == Py_None; }

// The tensor of an argument: null where it is none that the kernels could read as it lies on the current device.
const at::Tensor* readable(PyObject* o, int device) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  return t.is_cuda() && t.get_device() == device && !tracked(t) ? &t : nullptr;
}

// A contiguous tensor of one type and number of values; *p null for None.  False: neither.
bool vector_of(PyObject* o, int device, at::ScalarType type, int64_t n, const void** p) {
  *p = nullptr;
  if (is_none(o)) return true;
  const at::Tensor* t = readable(o, device);
  if (!t || t->scalar_type() != type || t->dim() != 1 || t->size(0) != n || !t->is_contiguous()) return false;
  *p = t->const_data_ptr();
  return true;
}

bool rows_of(const at::Tensor& t, int64_t* ld) {
  *ld = t.size(-1);
  return t.is_contiguous() || rows_at_one_stride(t, ld);
}

struct Rows {
  const at::Tensor* t;
  int64_t m, width, ld;
  int code;
};

// [..., width] of one of the kernels' types with at least one value, its rows at one distance.
bool rows_argument(PyObject* o, int device, Rows* r) {
  r->t = readable(o, device);
  if (!r->t || r->t->dim() < 1) return false;
  r->code = dtype_code(r->t->scalar_type());
  r->width = r->t->size(-1);
  if (r->code < 0 || r->code == 3 || r->width < 1 || r->width > 1 << 30) return false;
  r->m = r->t->numel() / r->width;
  return r->m >= 1 && r->m <= INT32_MAX && rows_of(*r->t, &r->ld);
}

// The current device where it is the tensor's, else -1.
int device_of(PyObject* o) {
  if (!THPVariable_CheckExact(o) || !THPVariable_Unpack(o).is_cuda()) return -1;
  const int device = THPVariable_Unpack(o).get_device();
  return device == (int)c10::hip::current_device() ? device : -1;
}

at::Tensor floats(int64_t bytes, int device) { return empty({bytes / 4}, at::kFloat, device); }

// layer_norm(x, weight, bias, eps, stats): the output, or (output, mean, rstd) with stats
PyObject* layer_norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 5) {
    PyErr_SetString(PyExc_TypeError, "layer_norm(x, weight, bias, eps, stats)");
    return nullptr;
  }
  return translated([&]() -> PyObject* {
    const int device = device_of(args[0]);
    Rows x;
    const void *weight, *bias;
    if (!PyFloat_Check(args[3]) || !PyBool_Check(args[4]) || !rows_argument(args[0], device, &x)) Py_RETURN_NONE;
    const at::ScalarType type = x.t->scalar_type();
    if (!vector_of(args[1], device, type, x.width, &weight) || !vector_of(args[2], device, type, x.width, &bias)) Py_RETURN_NONE;
    const bool stats = args[4] == Py_True;
    if (!stats && at::isReducedFloatingType(type) && at::autocast::is_autocast_enabled(at::kCUDA)) Py_RETURN_NONE;  // torch norms in f32 there
    at::Tensor y = empty(x.t->sizes(), type, device), mean, rstd;
    if (stats) {
      const at::IntArrayRef rows = x.t->sizes().slice(0, x.t->dim() - 1);
      mean = empty(rows, at::kFloat, device);
      rstd = empty(rows, at::kFloat, device);
    }
    if (npamd_layer_norm(x.t->const_data_ptr(), x.ld, weight, bias, y.data_ptr(), x.width, stats ? mean.data_ptr<float>() : nullptr,
                         stats ? rstd.data_ptr<float>() : nullptr, (int)x.m, (int)x.width, (float)PyFloat_AS_DOUBLE(args[3]), x.code, current_stream(device)) != NPAMD_OK)
      Py_RETURN_NONE;
    if (!stats) return THPVariable_Wrap(std::move(y));
    return Py_BuildValue("(NNN)", THPVariable_Wrap(std::move(y)), THPVariable_Wrap(std::move(mean)), THPVariable_Wrap(std::move(rstd)));
  });
}

// layer_norm_backward(dy, x, weight, mean, rstd, dx?, dweight?, dbias?): (dx, dweight, dbias), None where not asked for
PyObject* layer_norm_backward(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 8) {
    PyErr_SetString(PyExc_TypeError, "layer_norm_backward(dy, x, weight, mean, rstd, dx, dweight, dbias)");
    return nullptr;
  }
  return translated([&]() -> PyObject* {
    const int device = device_of(args[0]);
    Rows dy, x;
    const void* weight;
    if (!rows_argument(args[1], device, &x) || !rows_argument(args[0], device, &dy) || dy.code != x.code || dy.t->sizes() != x.t->sizes()) Py_RETURN_NONE;
    const at::ScalarType type = x.t->scalar_type();
    const at::Tensor *mean = readable(args[3], device), *rstd = readable(args[4], device);
    if (!vector_of(args[2], device, type, x.width, &weight) || !mean || !rstd) Py_RETURN_NONE;
    for (const at::Tensor* t : {mean, rstd})
      if (t->scalar_type() != at::kFloat || t->numel() != x.m || !t->is_contiguous()) Py_RETURN_NONE;
    for (int i = 5; i < 8; ++i)
      if (!PyBool_Check(args[i])) Py_RETURN_NONE;
    const bool need[3] = {args[5] == Py_True, args[6] == Py_True, args[7] == Py_True};
    at::Tensor out[3], scratch;
    if (need[0]) out[0] = empty(x.t->sizes(), type, device);
    for (int i = 1; i < 3; ++i)
      if (need[i]) out[i] = empty({x.width}, type, device);
    const int64_t bytes = need[1] || need[2] ? npamd_layer_norm_workspace_bytes((int)x.m, (int)x.width) : 0;
    if (bytes > 0) scratch = floats(bytes, device);
    auto at = [](const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
    if (npamd_layer_norm_backward(dy.t->const_data_ptr(), dy.ld, x.t->const_data_ptr(), x.ld, weight, mean->const_data_ptr<float>(), rstd->const_data_ptr<float>(),
                                  at(out[0]), x.width, at(out[1]), at(out[2]), (int)x.m, (int)x.width, x.code, at(scratch), bytes, current_stream(device)) != NPAMD_OK)
      Py_RETURN_NONE;
    PyObject* result[3];
    for (int i = 0; i < 3; ++i) {
      result[i] = need[i] ? THPVariable_Wrap(std::move(out[i])) : Py_None;
      if (!need[i]) Py_INCREF(Py_None);
    }
    return Py_BuildValue("(NNN)", result[0], result[1], result[2]);
  });
}

// Rows for a kernel: t where they lie at one distance, else a copy.
at::Tensor as_rows(const at::Tensor& t, int64_t* ld) { return rows_of(t, ld) ? t : (*ld = t.size(-1), t.contiguous()); }

const void* data_or_null(const at::Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }

// Inside a capture torch would go on to leaves whose nodes another graph that is still alive has made on another stream: waiting for that stream there ends the process.  Called in
// a node's backward pass: the leaves are those that its edges lead to, whether it keeps them or not.
void refuse_foreign_leaves(const char* what) {
  const auto stream = c10::hip::getCurrentHIPStream();
  hipStreamCaptureStatus status;
  if (hipStreamIsCapturing(stream.stream(), &status) != hipSuccess) return (void)hipGetLastError();
  if (status == hipStreamCaptureStatusNone) return;
  const auto node = torch::autograd::get_current_node();
  if (!node) return;  // called by itself, not by torch's engine: nothing goes on to the leaves
  for (const torch::autograd::Edge& edge : node->next_edges()) {
    const auto leaf = std::dynamic_pointer_cast<torch::autograd::AccumulateGrad>(edge.function);
    TORCH_CHECK(!leaf || !leaf->stream() || leaf->stream()->id() == stream.id(), what,
                ": a backward pass cannot be captured while a graph of the same leaves from another stream is alive: free it, or make it on the stream of the capture");
  }
}

// Layer norm in a recorded graph; arguments that Python has checked.  First derivatives only: what a backward pass that is itself recorded gives refuses to be differentiated.
struct LayerNormNode : torch::autograd::Function<LayerNormNode> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, const std::optional<at::Tensor>& weight, const std::optional<at::Tensor>& bias,
                            double eps) {
    const c10::DeviceGuard guard(x.device());
    const int device = x.get_device(), h = (int)x.size(-1), m = (int)(x.numel() / h);
    int64_t ld;
    const at::Tensor rows = as_rows(x, &ld), w = weight ? weight->contiguous() : at::Tensor(), b = bias ? bias->contiguous() : at::Tensor();
    const at::IntArrayRef lead = x.sizes().slice(0, x.dim() - 1);
    at::Tensor y = empty(x.sizes(), x.scalar_type(), device), mean = empty(lead, at::kFloat, device), rstd = empty(lead, at::kFloat, device);
    TORCH_CHECK(npamd_layer_norm(rows.const_data_ptr(), ld, data_or_null(w), data_or_null(b), y.data_ptr(), h, mean.data_ptr<float>(), rstd.data_ptr<float>(), m, h,
                                 (float)eps, dtype_code(x.scalar_type()), current_stream(device)) == NPAMD_OK, npamd_last_error());
    ctx->save_for_backward({x, weight ? *weight : at::Tensor(), bias ? *bias : at::Tensor(), mean, rstd});
    return y;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const torch::autograd::variable_list saved = ctx->get_saved_variables();
    const bool recorded = c10::GradMode::is_enabled();
    torch::autograd::variable_list out(4);
    const at::Tensor &x = saved[0], &mean = saved[3], &rstd = saved[4];
    const c10::DeviceGuard guard(x.device());
    refuse_foreign_leaves("layer_norm");
    {
      const c10::AutoGradMode off(false);
      const bool with_w = saved[1].defined(), with_b = saved[2].defined();
      const bool need[3] = {ctx->needs_input_grad(0), with_w && ctx->needs_input_grad(1), with_b && ctx->needs_input_grad(with_w ? 2 : 1)};
      const int device = x.get_device(), h = (int)x.size(-1), m = (int)(x.numel() / h);
      int64_t ldx, lddy;
      const at::Tensor rows = as_rows(x, &ldx), dy = as_rows(grads[0], &lddy), w = saved[1].defined() ? saved[1].contiguous() : at::Tensor();
      if (need[0]) out[0] = empty(x.sizes(), x.scalar_type(), device);
      for (int i = 1; i < 3; ++i)
        if (need[i]) out[i] = empty({h}, x.scalar_type(), device);
      const int64_t bytes = need[1] || need[2] ? npamd_layer_norm_workspace_bytes(m, h) : 0;
      at::Tensor scratch;
      if (bytes > 0) scratch = floats(bytes, device);
      auto at = [](const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
      TORCH_CHECK(npamd_layer_norm_backward(dy.const_data_ptr(), lddy, rows.const_data_ptr(), ldx, data_or_null(w), mean.const_data_ptr<float>(),
                                            rstd.const_data_ptr<float>(), at(out[0]), h, at(out[1]), at(out[2]), m, h, dtype_code(x.scalar_type()), at(scratch), bytes,
                                            current_stream(device)) == NPAMD_OK, npamd_last_error());
    }
    if (recorded) {
      for (at::Tensor& t : out)
        if (t.defined())
          t = torch::autograd::DelayedError("layer_norm: its backward pass cannot be differentiated", 1).apply(torch::autograd::variable_list{t.requires_grad_(true)})[0];
    }
    return out;
  }
};

// layer_norm_recorded(x, weight, bias, eps): tensors (or None) that Python has checked, on one device and of one type
PyObject* layer_norm_recorded(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 4 || !THPVariable_Check(args[0]) || !PyFloat_Check(args[3])) {
    PyErr_SetString(PyExc_TypeError, "layer_norm_recorded(x, weight, bias, eps)");
    return nullptr;
  }
  return translated([&]() -> PyObject* {
    auto maybe = [](PyObject* o) { return THPVariable_Check(o) ? std::optional<at::Tensor>(THPVariable_Unpack(o)) : std::nullopt; };
    const at::Tensor x = THPVariable_Unpack(args[0]);
    const double eps = PyFloat_AS_DOUBLE(args[3]);
    return THPVariable_Wrap(LayerNormNode::apply(x, maybe(args[1]), maybe(args[2]), eps));
  });
}

// dense_linear_act(x, w, bias, activation's number, residual)
PyObject* dense_linear_act(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 5) {
    PyErr_SetString(PyExc_TypeError, "dense_linear_act(x, w, bias, activation, residual)");
    return nullptr;
  }
  return translated([&]() -> PyObject* {
    const int device = device_of(args[0]);
    Rows x, w, res{nullptr, 0, 0, 0, 0};
    if (!rows_argument(args[0], device, &x) || !rows_argument(args[1], device, &w) || !PyLong_Check(args[3])) Py_RETURN_NONE;
    if (x.code == NPAMD_F32 || w.code != x.code || w.t->dim() != 2 || w.width != x.width) Py_RETURN_NONE;
    const at::ScalarType type = x.t->scalar_type();
    c10::SmallVector<int64_t, 6> sizes(x.t->sizes().begin(), x.t->sizes().end());
    sizes.back() = w.m;
    const void* bias;
    const bool wide = !vector_of(args[2], device, type, w.m, &bias);  // not of x's type: float32 then
    if (wide && !vector_of(args[2], device, at::kFloat, w.m, &bias)) Py_RETURN_NONE;
    if (!is_none(args[4]) && (!rows_argument(args[4], device, &res) || res.code != x.code || res.t->sizes() != at::IntArrayRef(sizes))) Py_RETURN_NONE;
    const long activation = PyLong_AsLong(args[3]);
    const hipStream_t st = current_stream(device);
    // Past the GEMV's tokens the tiles take it, which read rows of whole pieces at aligned addresses.
    const int64_t k = x.m > NPAMD_GEMV_MAX_M ? (x.width + 7) / 8 * 8 : x.width;
    const void *xp = x.t->const_data_ptr(), *wp = w.t->const_data_ptr();
    at::Tensor xc, wc;
    auto whole_pieces = [&](Rows& r, const void*& p, at::Tensor& copy) {
      if (x.m <= NPAMD_GEMV_MAX_M || (r.width == k && r.ld % 8 == 0 && r.ld < NPAMD_TILE_MAX_STRIDE && ((uintptr_t)p & 15) == 0)) return true;
      copy = empty({r.m, k}, type, device);
      const bool ok = npamd_gather_columns(p, r.ld, nullptr, copy.data_ptr(), k, (int)r.m, (int)r.width, st) == NPAMD_OK;
      p = copy.const_data_ptr();
      r.ld = k;
      return ok;
    };
    if (!whole_pieces(x, xp, xc) || !whole_pieces(w, wp, wc)) Py_RETURN_NONE;
    const int64_t bytes = npamd_dense_gemm_act_workspace_bytes((int)x.m, (int)w.m, (int)k);
    at::Tensor scratch, y = empty(sizes, type, device);
    if (bytes > 0) scratch = floats(bytes, device);
    if (npamd_dense_gemm_act(xp, x.ld, wp, w.ld, bias, wide ? NPAMD_F32 : x.code, (int)activation,
                             res.t ? res.t->const_data_ptr() : nullptr, res.ld, y.data_ptr(), w.m, (int)x.m, (int)w.m, (int)k, x.code,
                             bytes > 0 ? scratch.data_ptr() : nullptr, bytes, st) != NPAMD_OK)
      Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(y));
  });
}

// moe_layer(x, router, gate_up, its scales, its zero points, down, its scales, its zero points, experts, top_k, hidden, inter, nbits, group_size, renormalize)
PyObject* moe_layer(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 15) {
    PyErr_SetString(PyExc_TypeError, "moe_layer(x, 7 tensors of the experts, 6 numbers, renormalize)");
    return nullptr;
  }
  return translated([&]() -> PyObject* {
    const int device = device_of(args[0]);
    Rows x;
    if (!PyBool_Check(args[14]) || !rows_argument(args[0], device, &x)) Py_RETURN_NONE;
    const void* p[7];
    const at::Tensor* t[7] = {};
    for (int i = 0; i < 7; ++i) {  // of MoEExperts, which has checked them
      if (!is_none(args[1 + i]) && !(t[i] = readable(args[1 + i], device))) Py_RETURN_NONE;
      p[i] = t[i] ? t[i]->const_data_ptr() : nullptr;
    }
    int v[6];
    for (int i = 0; i < 6; ++i) {
      const long l = PyLong_Check(args[8 + i]) ? PyLong_AsLong(args[8 + i]) : -1;
      if (l < 0 || l > INT32_MAX) {
        PyErr_Clear();
        Py_RETURN_NONE;
      }
      v[i] = (int)l;
    }
    const auto [experts, top_k, hidden, inter, nbits, group] = v;
    if (!t[0] || !t[1] || !t[4] || x.width != hidden || x.t->scalar_type() != t[0]->scalar_type()) Py_RETURN_NONE;
    const int64_t bytes = npamd_moe_workspace_bytes((int)x.m, experts, top_k, hidden, inter);
    at::Tensor scratch, y = empty(x.t->sizes(), x.t->scalar_type(), device);
    if (bytes > 0) scratch = floats(bytes, device);
    if (npamd_moe_layer(x.t->const_data_ptr(), x.ld, p[0], p[1], p[2], p[3], p[4], p[5], p[6], y.data_ptr(), hidden, (int)x.m, experts, top_k, hidden, inter, nbits, group,
                        args[14] == Py_True, x.code, bytes > 0 ? scratch.data_ptr() : nullptr, bytes, current_stream(device)) != NPAMD_OK)
      Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(y));
  });
}

}  // namespace
