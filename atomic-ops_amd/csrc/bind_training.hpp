// Native call paths of a training step around the blocks (linear, cross_entropy, AdamW), part of bind.cpp.
// Through Python and ctypes a product with its gradients cost 200 us of host time, a loss with its gradient 130 and an
// update of the benchmark LM's 186 tensors 550.
#pragma once

// The gradients of a node, raising when they are differentiated (as Once above).
struct OnceOnly : torch::autograd::Function<OnceOnly> {
  static variable_list forward(AutogradContext*, at::TensorList, const variable_list& grads) { return grads; }
  static variable_list backward(AutogradContext*, variable_list) {
    TORCH_CHECK(false, "linear and cross_entropy are once differentiable: their gradients cannot be differentiated");
  }
};
void once_only(variable_list* grads, const variable_list& from) {
  if (!at::GradMode::is_enabled()) return;
  variable_list held, in(from);
  for (const Tensor& t : *grads)
    if (t.defined()) held.push_back(t);
  in.push_back(at::empty({0}).requires_grad_(true));
  held = OnceOnly::apply(at::TensorList(in), held);
  size_t i = 0;
  for (Tensor& t : *grads)
    if (t.defined()) t = held[i++];
}

void* at_of(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
bool turned(const Tensor& w) {       // the transposed view of a matrix with whole rows
  return w.stride(0) == 1 && w.stride(1) >= w.size(0) && !(w.stride(1) == 1 && w.size(1) > 1);
}
bool whole_rows(const Tensor& w) { return (w.stride(1) == 1 || w.size(1) == 1) && (w.stride(0) >= w.size(1) || w.size(0) == 1); }
int64_t ld_of(const Tensor& t) { return t.size(0) == 1 ? t.size(1) : t.stride(0); }

// y = act(A B + bias) + residual (gdn2_linear); whether the library took it
bool product(int form, int64_t M, int64_t K, int64_t N, const Tensor& a, int64_t lda, const Tensor& b, int64_t ldb, const Tensor& y,
             int act = 0, const Tensor& bias = {}, const Tensor& res = {}, int64_t ldr = 0, const Tensor& z = {}) {
  gdn2_product p{};
  p.M = (int32_t)M; p.K = (int32_t)K; p.N = (int32_t)N; p.form = form;
  p.dtype = float_kind(a.scalar_type());
  p.out_dtype = float_kind(y.scalar_type());
  p.bias_dtype = bias.defined() ? float_kind(bias.scalar_type()) : 0;
  p.activation = act | (z.defined() && z.scalar_type() == at::kFloat ? GDN2_Z_F32 : 0); p.lda = lda; p.ldb = ldb; p.ldr = ldr;
  p.a = a.data_ptr(); p.b = b.data_ptr(); p.bias = at_of(bias); p.residual = at_of(res);
  p.y = y.data_ptr(); p.z = at_of(z);
  const int64_t bytes = (int64_t)abi.linear_ws(&p);
  const Tensor ws = bytes ? empty_on(y, {bytes}, at::kByte) : Tensor();
  return abi.linear(&p, at_of(ws), stream_of(y.device())) == 0;
}

// Whether the gradients of a product of 16 bits are formed from dz and what its rounding leaves out, and what z is kept in
// (linear.py, _fine and _z_dtype)
bool fine_gradients(int64_t M, int64_t K, int64_t N, at::ScalarType dt) {
  return dt != at::kFloat && 2.0 * (double)M * (double)K * (double)N <= GDN2_LINEAR_FINE && M * K <= GDN2_LINEAR_X;
}
at::ScalarType z_type(int64_t M, int64_t K, int64_t N, at::ScalarType dt) {
  return fine_gradients(M, K, N, dt) || M * N <= GDN2_LINEAR_Z ? at::kFloat : dt;
}

// x (..., in) of whole rows, w (in, out) of whole rows or turned; throws Refused
Tensor linear_forward(const Tensor& x, const Tensor& w, const Tensor& bias, const Tensor& res, int64_t act, bool f32, Tensor* z) {
  const int64_t K = w.size(0), N = w.size(1), M = x.numel() / K;
  c10::DeviceGuard guard(x.device());
  at::DimVector size(x.sizes());
  size.back() = N;
  const Tensor y = empty_on(x, size, f32 ? at::kFloat : x.scalar_type());
  if (z) *z = empty_on(x, {M, N}, z_type(M, K, N, x.scalar_type()));
  const bool t = turned(w);
  if (!product(t ? GDN2_XWT : GDN2_XW, M, K, N, x, row_stride(x, K), w, t ? ld_of(w.t()) : ld_of(w), y, (int)act, bias, res,
               res.defined() ? row_stride(res, N) : 0, z ? *z : Tensor()))
    throw Refused();
  return y;
}

struct Linear : torch::autograd::Function<Linear> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const std::optional<Tensor>& bias,
                        const std::optional<Tensor>& res, int64_t act, bool f32) {
    Tensor z;
    const Tensor y = linear_forward(x, w, bias.value_or(Tensor()), res.value_or(Tensor()), act, f32, act ? &z : nullptr);
    ctx->save_for_backward({x, w, z});
    ctx->saved_data["conf"] = std::vector<int64_t>{act, bias ? (int64_t)bias->scalar_type() : -1, res.has_value(), (int64_t)x.scalar_type()};
    ctx->saved_data["x"] = x.sizes().vec();
    ctx->saved_data["w"] = w.sizes().vec();
    ctx->saved_data["device"] = x.device();
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list gs) {
    variable_list saved = ctx->get_saved_variables();
    const std::vector<int64_t> conf = ctx->saved_data["conf"].toIntVector(), xs = ctx->saved_data["x"].toIntVector(),
                               wsz = ctx->saved_data["w"].toIntVector();
    const c10::Device dev = ctx->saved_data["device"].toDevice();
    const int64_t act = conf[0], K = wsz[0], N = wsz[1];
    const at::ScalarType dt = (at::ScalarType)conf[3];
    Tensor x = saved[0], w = saved[1], z = saved[2];
    auto kept = [&](const Tensor& t, at::IntArrayRef size, at::ScalarType dt) { return t.defined() && t.sizes() == size && t.device() == dev && t.scalar_type() == dt; };
    if (!kept(x, xs, dt) || !row_stride(x, K)) x = restored(x, xs, dt, dev);
    if (!kept(w, wsz, dt) || !(turned(w) || whole_rows(w))) w = restored(w, wsz, dt, dev);
    const int64_t M = x.numel() / K;
    const at::ScalarType zt = z_type(M, K, N, dt);
    if (act && (!kept(z, {M, N}, zt) || !z.is_contiguous())) z = restored(z, {M, N}, zt, dev);
    size_t edge = 2;
    const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1);
    const bool need_b = conf[1] >= 0 && ctx->needs_input_grad(edge++), need_r = conf[2] && ctx->needs_input_grad(edge);
    const Tensor dy = gs[0].contiguous();
    c10::DeviceGuard guard(dev);
    Tensor dz = dy, dx, dw, db;
    const bool own = (act || dy.scalar_type() != dt) && (need_x || need_w), fine = own && fine_gradients(M, K, N, dt);
    if (own || need_b) {
      if (own) dz = empty_on(x, {fine ? 2 * M : M, N}, dt);
      if (need_b) db = empty_on(x, {N}, (at::ScalarType)conf[1]);
      gdn2_slope s{};
      s.M = (int32_t)M; s.N = (int32_t)N; s.dtype = float_kind(dt); s.dy_dtype = float_kind(dy.scalar_type());
      s.bias_dtype = need_b ? float_kind((at::ScalarType)conf[1]) : 0;
      s.activation = (int32_t)act | (zt == at::kFloat ? GDN2_Z_F32 : 0) | (fine ? GDN2_DZ_LOW : 0);
      s.dy = dy.data_ptr(); s.z = act ? z.data_ptr() : nullptr; s.dz = own ? dz.data_ptr() : nullptr; s.dbias = at_of(db);
      const int64_t bytes = (int64_t)abi.slope_ws(&s);
      const Tensor ws = bytes ? empty_on(x, {bytes}, at::kByte) : Tensor();
      TORCH_CHECK(abi.slope(&s, at_of(ws), stream_of(dev)) == 0, "gdn2_linear_slope: ", abi.last_error());
    }
    const bool t = turned(w);
    bool ok = true;
    if (need_x) {
      dx = empty_on(x, x.sizes(), dt);
      ok = product((t ? GDN2_XW : GDN2_XWT) | (fine ? GDN2_HALVES : 0), M, N, K, dz, N, w, t ? ld_of(w.t()) : ld_of(w), dx);
    }
    if (ok && need_w) {
      dw = empty_on(x, t ? at::IntArrayRef{N, K} : at::IntArrayRef{K, N}, dt);
      int64_t rows = M;
      if (fine) {            // (x^T dz is a sum over the rows: over those of both)
        at::NoGradGuard off;
        const Tensor r = x.dim() == 2 ? x : x.view({M, K});
        x = at::cat({r, r});
        rows = 2 * M;
      }
      ok = t ? product(GDN2_XTW, N, rows, K, dz, N, x, row_stride(x, K), dw) : product(GDN2_XTW, K, rows, N, x, row_stride(x, K), dz, N, dw);
      if (t) dw = dw.t();
    }
    TORCH_CHECK(ok, "gdn2_linear: ", abi.last_error());
    variable_list out{dx, dw, db, need_r ? gs[0] : Tensor()};
    once_only(&out, {gs[0], saved[0], saved[1]});
    out.resize(6);
    return out;
  }
};

// linear(x, weight, bias or None, residual or None, activation, whether y is float32) -> y, or None: not a plain call
PyObject* py_linear(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 6) return PyErr_Format(PyExc_TypeError, "linear takes 6 arguments");
  int64_t act;
  if (!THPVariable_Check(args[0]) || !THPVariable_Check(args[1]) || !whole(args[4], &act)) return none();
  const Tensor x = THPVariable_Unpack(args[0]), w = THPVariable_Unpack(args[1]);
  Tensor bias, res;
  for (int i : {2, 3}) {
    if (args[i] == Py_None) continue;
    if (!THPVariable_Check(args[i])) return none();
    (i == 2 ? bias : res) = THPVariable_Unpack(args[i]);
  }
  const bool f32 = args[5] == Py_True;
  if (!plain_mode() || !x.is_cuda() || x.dim() < 1 || x.numel() == 0 || w.dim() != 2 || w.numel() == 0) return none();
  const c10::Device dev = x.device();
  const at::ScalarType dt = x.scalar_type(), od = f32 ? at::kFloat : dt;
  const int64_t K = w.size(0), N = w.size(1);
  if (float_kind(dt) < 0 || x.size(-1) != K || !plain(x, dev) || !plain(w, dev) || w.scalar_type() != dt || !row_stride(x, K) ||
      !(turned(w) || whole_rows(w)) || x.numel() / K > INT32_MAX || K > INT32_MAX || N > INT32_MAX)
    return none();
  if (bias.defined() && (!plain(bias, dev) || (bias.scalar_type() != dt && bias.scalar_type() != at::kFloat) || bias.dim() != 1 ||
                         bias.size(0) != N || !bias.is_contiguous()))
    return none();
  if (res.defined()) {
    if (!plain(res, dev) || res.scalar_type() != od || res.dim() != x.dim() || res.size(-1) != N || !row_stride(res, N)) return none();
    for (int64_t i = 0; i + 1 < x.dim(); ++i)
      if (res.size(i) != x.size(i)) return none();
  }
  const bool grad = recorded({&x, &w, &bias, &res});
  Tensor y;
  bool refused = false;
  unlocked([&] {
    try {
      auto opt = [](const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; };
      y = grad ? Linear::apply(x, w, opt(bias), opt(res), act, f32) : linear_forward(x, w, bias, res, act, f32, nullptr);
    } catch (const Refused&) {
      refused = true;
    }
  });
  return refused ? none() : THPVariable_Wrap(y);
  END_HANDLE_TH_ERRORS
}

// ---- cross-entropy --------------------------------------------------------------------------------------------------

struct LossHow {
  int64_t ignore;
  double smoothing, z;
  int64_t reduction;
};
bool loss_run(const Tensor& x, const Tensor& targets, const LossHow& how, const Tensor& loss, const Tensor& d, const Tensor& up = {}) {
  const int64_t V = x.size(-1), N = x.numel() / V;
  gdn2_loss a{};
  a.rows = (int32_t)N; a.V = (int32_t)V; a.dtype = float_kind(x.scalar_type());
  a.target_type = targets.scalar_type() == at::kInt ? GDN2_FLAG_INT32 : GDN2_FLAG_INT64;
  a.reduction = (int32_t)how.reduction;
  a.upstream_ld = up.defined() && how.reduction == 0;
  a.smoothing = (float)how.smoothing; a.z_loss = (float)how.z; a.ld = row_stride(x, V); a.ignore_index = how.ignore;
  a.logits = x.data_ptr(); a.targets = targets.data_ptr(); a.upstream = f32_at(up); a.loss = f32_at(loss); a.dlogits = at_of(d);
  const Tensor ws = empty_on(x, {(int64_t)abi.loss_ws((int32_t)N)}, at::kByte);
  return abi.cross_entropy(&a, ws.data_ptr(), stream_of(x.device())) == 0;
}
Tensor loss_forward(const Tensor& x, const Tensor& targets, const LossHow& how, Tensor* d) {
  c10::DeviceGuard guard(x.device());
  const Tensor loss = empty_on(x, how.reduction ? at::IntArrayRef{} : targets.sizes(), at::kFloat);
  if (d) *d = empty_on(x, x.sizes(), x.scalar_type());
  if (!loss_run(x, targets, how, loss, d ? *d : Tensor())) throw Refused();
  return loss;
}

// The capture that a stream is in (0: none)
int64_t capture_of(void* stream) {
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  unsigned long long id = 0;
  if (hipStreamGetCaptureInfo(static_cast<hipStream_t>(stream), &status, &id) != hipSuccess) {
    (void)hipGetLastError();
    return 0;
  }
  return status == hipStreamCaptureStatusNone ? 0 : (int64_t)id + 1;
}

struct CrossEntropy : torch::autograd::Function<CrossEntropy> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& targets, int64_t ignore, double e, double z, int64_t reduction) {
    // float16 gradients are formed when the factor of a scaled loss is known: without it they would underflow
    Tensor d;
    const Tensor loss = loss_forward(x, targets, LossHow{ignore, e, z, reduction}, x.scalar_type() == at::kHalf ? nullptr : &d);
    ctx->save_for_backward({x, targets});
    if (d.defined()) ctx->saved_data["grad"] = d;
    ctx->saved_data["how"] = std::vector<int64_t>{ignore, reduction, (int64_t)x.scalar_type(), (int64_t)targets.scalar_type(),
                                                  capture_of(stream_of(x.device()))};
    ctx->saved_data["terms"] = std::vector<double>{e, z};
    ctx->saved_data["size"] = x.sizes().vec();
    ctx->saved_data["device"] = x.device();
    return loss;
  }
  static variable_list backward(AutogradContext* ctx, variable_list gs) {
    const variable_list saved = ctx->get_saved_variables();
    const std::vector<int64_t> how = ctx->saved_data["how"].toIntVector(), size = ctx->saved_data["size"].toIntVector();
    const std::vector<double> terms = ctx->saved_data["terms"].toDoubleVector();
    const c10::Device dev = ctx->saved_data["device"].toDevice();
    const at::ScalarType dt = (at::ScalarType)how[2];
    const Tensor g = gs[0].contiguous();
    c10::DeviceGuard guard(dev);
    Tensor d;
    // (the kept gradient is multiplied where it lies: a graph of the backward pass alone would do so at every replay)
    if (const auto it = ctx->saved_data.find("grad"); it != ctx->saved_data.end() && capture_of(stream_of(dev)) == how[4]) {
      d = it->second.toTensor();
      ctx->saved_data.erase(it);
      const int64_t V = size.back();
      TORCH_CHECK(abi.scale_rows(d.data_ptr(), float_kind(dt), (int)(d.numel() / V), (int)V, f32_at(g), how[1] == 0, stream_of(dev)) == 0,
                  "gdn2_scale_rows: ", abi.last_error());
    } else {                 // float16, a second pass over a kept graph, or another capture than the forward pass's
      Tensor x = saved[0], t = saved[1];
      if (!x.defined() || x.sizes() != at::IntArrayRef(size) || x.device() != dev || x.scalar_type() != dt || !row_stride(x, size.back()))
        x = restored(x, size, dt, dev);
      const at::IntArrayRef rows(size.data(), size.size() - 1);
      if (!t.defined() || t.sizes() != rows || t.device() != dev || t.scalar_type() != (at::ScalarType)how[3] || !t.is_contiguous())
        t = restored(t, rows, (at::ScalarType)how[3], dev);
      d = empty_on(x, size, dt);
      TORCH_CHECK(loss_run(x, t, LossHow{how[0], terms[0], terms[1], how[1]}, Tensor(), d, g), "gdn2_cross_entropy: ", abi.last_error());
    }
    variable_list out{d};
    once_only(&out, {gs[0], saved[0]});
    out.resize(6);
    return out;
  }
};

// cross_entropy(logits, targets, ignore_index, smoothing, z_loss, reduction) -> loss, or None: not a plain call
PyObject* py_cross_entropy(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 6) return PyErr_Format(PyExc_TypeError, "cross_entropy takes 6 arguments");
  int64_t ignore, reduction;
  if (!THPVariable_Check(args[0]) || !THPVariable_Check(args[1]) || !whole(args[2], &ignore) || !PyFloat_Check(args[3]) ||
      !PyFloat_Check(args[4]) || !whole(args[5], &reduction))
    return none();
  const Tensor x = THPVariable_Unpack(args[0]), t = THPVariable_Unpack(args[1]);
  const double e = PyFloat_AS_DOUBLE(args[3]), z = PyFloat_AS_DOUBLE(args[4]);
  if (!plain_mode() || !x.is_cuda() || x.dim() < 1 || x.numel() == 0) return none();
  const c10::Device dev = x.device();
  const int64_t V = x.size(-1);
  if (float_kind(x.scalar_type()) < 0 || !plain(x, dev) || !plain(t, dev) || !row_stride(x, V) || V > INT32_MAX || x.numel() / V > INT32_MAX ||
      (t.scalar_type() != at::kInt && t.scalar_type() != at::kLong) || !t.is_contiguous() || t.dim() != x.dim() - 1)
    return none();
  for (int64_t i = 0; i < t.dim(); ++i)
    if (t.size(i) != x.size(i)) return none();
  const bool grad = recorded({&x});
  Tensor loss;
  bool refused = false;
  unlocked([&] {
    try {
      loss = grad ? CrossEntropy::apply(x, t, ignore, e, z, reduction) : loss_forward(x, t, LossHow{ignore, e, z, reduction}, nullptr);
    } catch (const Refused&) {
      refused = true;
    }
  });
  return refused ? none() : THPVariable_Wrap(loss);
  END_HANDLE_TH_ERRORS
}

// ---- AdamW ----------------------------------------------------------------------------------------------------------

// The tensors of an optimizer's groups (dicts as torch.optim's) with their states; step: those with a gradient, else
// those with a state.  False: something is not as the kernels take it (Python makes states, casts, validates and raises).
// all: how many parameters the groups have.
bool adamw_tensors(PyObject* groups, PyObject* state, int64_t bits, bool step, std::vector<gdn2_adamw_tensor>* out, std::vector<Tensor>* params,
                   int32_t* all = nullptr) {
  static PyObject *const kAvg = PyUnicode_InternFromString("exp_avg"), *const kSq = PyUnicode_InternFromString("exp_avg_sq"),
                         *const kAvgScale = PyUnicode_InternFromString("exp_avg_scale"),
                         *const kSqScale = PyUnicode_InternFromString("exp_avg_sq_scale"),
                         *const kMaster = PyUnicode_InternFromString("master"), *const kStep = PyUnicode_InternFromString("step");
  if (!PyList_Check(groups) || !PyDict_Check(state)) return false;
  int32_t ordinal = 0;
  std::optional<c10::Device> dev;
  for (Py_ssize_t k = 0; k < PyList_GET_SIZE(groups); ++k) {
    PyObject* g = PyList_GET_ITEM(groups, k);
    if (!PyDict_Check(g)) return false;
    PyObject *ps = PyDict_GetItemString(g, "params"), *betas = PyDict_GetItemString(g, "betas");
    PyObject* h[5] = {PyDict_GetItemString(g, "lr"), nullptr, nullptr, PyDict_GetItemString(g, "eps"), PyDict_GetItemString(g, "weight_decay")};
    if (!ps || !PyList_Check(ps) || !betas || !PyTuple_Check(betas) || PyTuple_GET_SIZE(betas) != 2) return false;
    h[1] = PyTuple_GET_ITEM(betas, 0);
    h[2] = PyTuple_GET_ITEM(betas, 1);
    for (PyObject* x : h)
      if (!x || !PyFloat_CheckExact(x)) return false;
    for (Py_ssize_t i = 0; i < PyList_GET_SIZE(ps); ++i, ++ordinal) {
      PyObject* o = PyList_GET_ITEM(ps, i);
      if (!THPVariable_Check(o)) return false;
      const Tensor& p = THPVariable_Unpack(o);
      const Tensor& grad = p.grad();
      if (p.numel() == 0 || (step && !grad.defined())) continue;
      if (!dev) dev = p.device();
      const int kind = float_kind(p.scalar_type());
      if (kind < 0 || !p.is_cuda() || !plain(p, *dev) || !p.is_contiguous()) return false;
      if (step && (!plain(grad, *dev) || grad.scalar_type() != p.scalar_type() || grad.sizes() != p.sizes() || !grad.is_contiguous())) return false;
      PyObject* s = PyDict_GetItemWithError(state, o);
      if (!s) PyErr_Clear();
      if (!s || !PyDict_Check(s) || PyDict_GET_SIZE(s) == 0) {
        if (step) return false;
        continue;
      }
      bool ok = true;
      auto get = [&](PyObject* key, at::ScalarType dt, int64_t size) -> void* {
        PyObject* v = PyDict_GetItemWithError(s, key);
        if (!v) PyErr_Clear();
        if (!v || !THPVariable_Check(v)) return ok = false, nullptr;
        const Tensor& t = THPVariable_Unpack(v);
        if (!plain(t, *dev) || t.scalar_type() != dt || t.numel() != size || !t.is_contiguous()) return ok = false, nullptr;
        return t.data_ptr();
      };
      const int64_t size = p.numel(), blocks = (size + GDN2_ADAMW_BLOCK - 1) / GDN2_ADAMW_BLOCK;
      gdn2_adamw_tensor a{};
      a.p = p.data_ptr();
      a.g = step ? grad.data_ptr() : nullptr;
      a.m = get(kAvg, bits == 8 ? at::kChar : at::kFloat, size);
      a.v = get(kSq, bits == 8 ? at::kByte : at::kFloat, size);
      if (bits == 8) {
        a.m_scale = static_cast<float*>(get(kAvgScale, at::kFloat, blocks));
        a.v_scale = static_cast<float*>(get(kSqScale, at::kFloat, blocks));
      }
      if (kind) a.master = static_cast<float*>(get(kMaster, at::kFloat, size));
      a.step = static_cast<float*>(get(kStep, at::kFloat, 1));
      if (!ok) return false;
      a.numel = size;
      a.ordinal = ordinal;
      a.dtype = kind;
      a.lr = PyFloat_AS_DOUBLE(h[0]); a.beta1 = PyFloat_AS_DOUBLE(h[1]); a.beta2 = PyFloat_AS_DOUBLE(h[2]);
      a.eps = PyFloat_AS_DOUBLE(h[3]); a.weight_decay = PyFloat_AS_DOUBLE(h[4]);
      out->push_back(a);
      params->push_back(p);
    }
  }
  if (all) *all = ordinal;
  return !out->empty();
}

// adamw(groups, state, bits, max_norm or 0.0) -> the norm (True without max_norm), or None: not a plain step
PyObject* py_adamw(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 4) return PyErr_Format(PyExc_TypeError, "adamw takes 4 arguments");
  int64_t bits;
  if (!whole(args[2], &bits) || !PyFloat_Check(args[3]) || !plain_mode()) return none();
  const double max_norm = PyFloat_AS_DOUBLE(args[3]);
  std::vector<gdn2_adamw_tensor> ts;
  std::vector<Tensor> ps;
  if (!adamw_tensors(args[0], args[1], bits, true, &ts, &ps)) return none();
  Tensor norm;
  int status = 0;
  unlocked([&] {
    const c10::Device dev = ps[0].device();
    c10::DeviceGuard guard(dev);
    if (max_norm > 0.0) norm = empty_on(ps[0], {}, at::kFloat);
    const Tensor ws = empty_on(ps[0], {(int64_t)abi.adamw_ws(ts.data(), (int)ts.size())}, at::kByte);
    status = abi.adamw(ts.data(), (int)ts.size(), (int)bits, max_norm, f32_at(norm), ws.data_ptr(), stream_of(dev));
    if (!status)
      for (const Tensor& p : ps) p.unsafeGetTensorImpl()->bump_version();
  });
  if (status) return none();
  if (norm.defined()) return THPVariable_Wrap(norm);
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// adamw_unpack(groups, state, exp_avg, exp_avg_sq): the values of 8-bit states into lists of a tensor for each parameter;
// True, or None: not as the kernel takes them
PyObject* py_adamw_unpack(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 4) return PyErr_Format(PyExc_TypeError, "adamw_unpack takes 4 arguments");
  std::vector<gdn2_adamw_tensor> ts;
  std::vector<Tensor> ps;
  int32_t all = 0;
  if (!plain_mode() || !PyList_Check(args[2]) || !PyList_Check(args[3]) || !adamw_tensors(args[0], args[1], 8, false, &ts, &ps, &all)) return none();
  if (ts.size() != (size_t)all) return none();       // (parameters without a state)
  const c10::Device dev = ps[0].device();
  std::vector<float*> out[2];
  std::vector<Tensor> held;
  for (int k = 0; k < 2; ++k) {
    if ((size_t)PyList_GET_SIZE(args[2 + k]) != ts.size()) return none();
    for (size_t i = 0; i < ts.size(); ++i) {
      PyObject* o = PyList_GET_ITEM(args[2 + k], (Py_ssize_t)i);
      if (!THPVariable_Check(o)) return none();
      const Tensor& t = THPVariable_Unpack(o);
      if (!plain(t, dev) || t.scalar_type() != at::kFloat || t.numel() != ts[i].numel || !t.is_contiguous() || recorded({&t})) return none();
      out[k].push_back(f32_at(t));
      held.push_back(t);
    }
  }
  int status = 0;
  unlocked([&] {
    c10::DeviceGuard guard(dev);
    status = abi.adamw_unpack(ts.data(), (int)ts.size(), out[0].data(), out[1].data(), stream_of(dev));
    if (!status)
      for (const Tensor& t : held) t.unsafeGetTensorImpl()->bump_version();
  });
  if (status) return none();
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}
