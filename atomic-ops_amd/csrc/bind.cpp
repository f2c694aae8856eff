// Native call path of the operator and of the decode step (module atomic_gdn2._bind).
//
// Small calls are bound by the host: through Python and ctypes a gradient evaluation costs about
// 200 us and a decode step 23 us (36 with reset flags to cast) before the GPU matters.  The functions
// here do the same work from C++ (the segment loop, the autograd node, allocation, the C-ABI calls of include/gdn2.h) for plain
// calls: CUDA tensors of one device, the shapes and dtypes the kernels take as they are, no
// dispatch modes, functorch wrappers or forward-mode tangents.  For anything else, and for whatever
// the library refuses, they return None and the caller goes on in Python, which casts, validates
// and raises.  MI355X, per pass: B1 H2 L256 gradient evaluation 209 -> 135 us, B1 H6 decode step
// 23.0 -> 6.4 us, B8 H16 with raw inputs and reset flags 36.4 -> 7.7 us.  The steps of token generation
// (w4, beam, premix_step) come the same way: one row of 512 x 4614 13.0 -> 6.1 us, one token's premix of 4
// rows 36.6 -> 12.7 us, 8.4 with its eight outputs in one allocation.
//
// Nothing is kept between calls but the configuration a caller passed to op().
#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <torch/csrc/Device.h>
#include <torch/csrc/DynamicTypes.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstring>
#include <memory>
#include <string>
#include <vector>

#include "../../include/gdn2.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// The C ABI, by address: the library that atomic_gdn2._lib has loaded.
struct Abi {
  decltype(&gdn2_residual_layout) residual_layout;
  decltype(&gdn2_fwd_workspace_bytes) fwd_ws;
  decltype(&gdn2_bwd_workspace_bytes) bwd_ws;
  decltype(&gdn2_fwd) fwd;
  decltype(&gdn2_fwd_bf16) fwd_bf16;
  decltype(&gdn2_bwd) bwd;
  decltype(&gdn2_decode_from) decode;
  decltype(&gdn2_default_state_ckpt) default_ckpt;
  decltype(&gdn2_w4_workspace_bytes) w4_ws;
  decltype(&gdn2_w4_linear) w4;
  decltype(&gdn2_beam_workspace_bytes) beam_ws;
  decltype(&gdn2_beam_step) beam;
  decltype(&gdn2_lm_premix_step_fwd) premix_step;
  decltype(&gdn2_last_error) last_error;
} abi{};

// The library refused the call: the Python path raises what belongs to it.
struct Refused {};

const c10::DispatchKeySet kUnplain{c10::DispatchKey::Python,          c10::DispatchKey::PythonTLSSnapshot,
                                   c10::DispatchKey::Functionalize,   c10::DispatchKey::FuncTorchBatched,
                                   c10::DispatchKey::Batched,         c10::DispatchKey::FuncTorchGradWrapper,
                                   c10::DispatchKey::FuncTorchVmapMode, c10::DispatchKey::VmapMode,
                                   c10::DispatchKey::FuncTorchDynamicLayerFrontMode,
                                   c10::DispatchKey::FuncTorchDynamicLayerBackMode,
                                   c10::DispatchKey::Negative,        c10::DispatchKey::Conjugate,
                                   c10::DispatchKey::ZeroTensor};

bool plain_mode() {
  const auto tls = c10::impl::tls_local_dispatch_key_set();
  return !tls.included_.has_any(kUnplain);
}
bool plain(const Tensor& t, const c10::Device& dev) {
  return t.defined() && t.layout() == c10::kStrided && t.device() == dev && !t.key_set().has_any(kUnplain) &&
         !t._fw_grad(0).defined();
}

void* stream_of(const c10::Device& dev) {
  return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(dev.index()).stream();
}
Tensor empty_on(const Tensor& like, at::IntArrayRef size, at::ScalarType dt) {
  return at::empty(size, at::TensorOptions().dtype(dt).device(like.device()));
}
// A contiguous tensor on the bytes of base from `at` on (a multiple of 16): several outputs of one call in
// one allocation, at a tenth of the host time of one each.  They share a storage, so this is for outputs
// that a program drops together, or small ones.
Tensor part_of(const Tensor& base, int64_t at, at::IntArrayRef size, at::ScalarType dt) {
  auto impl = c10::make_intrusive<c10::TensorImpl>(c10::Storage(base.storage()), base.key_set(), c10::scalarTypeToTypeMeta(dt));
  impl->set_storage_offset(at / (int64_t)c10::elementSize(dt));
  impl->set_sizes_contiguous(size);
  return Tensor(std::move(impl));
}
int64_t up16(int64_t x) { return (x + 15) / 16 * 16; }
float* f32_at(const Tensor& t, int64_t off = 0) { return t.defined() ? static_cast<float*>(t.data_ptr()) + off : nullptr; }

// One operator configuration: the descriptor without its shape (trivially copyable).
struct Op {
  gdn2_desc base;
  int64_t segment;     // tokens per segment (max_chunks_per_call * bt)

  // base.state_ckpt < 0: the library's choice for the shape
  gdn2_desc training_desc(int64_t B, int64_t H, int64_t L, int64_t D, int64_t seq_ld) const {
    gdn2_desc d = desc(B, H, L, D, seq_ld, base.state_ckpt);
    if (d.state_ckpt < 0) d.state_ckpt = abi.default_ckpt(&d);
    return d;
  }
  gdn2_desc desc(int64_t B, int64_t H, int64_t L, int64_t D, int64_t seq_ld, int ckpt) const {
    gdn2_desc d = base;
    d.B = (int32_t)B;
    d.H = (int32_t)H;
    d.L = (int32_t)L;
    d.D = (int32_t)D;
    d.seq_ld = (int32_t)seq_ld;
    d.state_ckpt = ckpt;
    return d;
  }
};

// A saved tensor as the backward takes it: saved-tensor hooks may give back other dtypes, strides or
// devices (brought back here) or another shape (refused).
Tensor restored(const Tensor& t, at::IntArrayRef size, at::ScalarType dt, const c10::Device& dev) {
  TORCH_CHECK(t.defined() && t.sizes() == size, "saved-tensor hooks gave back another shape than was saved");
  return t.to(dev, dt).contiguous();
}

// The identity on the gradients of a Sequence, as functions of what they were formed from; raises when
// they are differentiated.
struct Once : torch::autograd::Function<Once> {
  static variable_list forward(AutogradContext*, at::TensorList, const variable_list& grads) { return grads; }
  static variable_list backward(AutogradContext*, variable_list) {
    TORCH_CHECK(false, "the GDN-2 operator is once differentiable: its gradients cannot be differentiated");
  }
};

// The whole call as one autograd node: forward and backward run the segment loop over views of the
// full tensors (gdn2_desc.seq_ld), the state carried through h0 / h_final and dh0 / dh_final.
// float32 inputs and clip <= 1e4 (then the reference's final cast of the gradients is the identity).
struct Sequence : torch::autograd::Function<Sequence> {
  // (the node keeps a copy of the configuration: it may outlive the caller's)
  static variable_list forward(AutogradContext* ctx, const Op* op, const Tensor& q, const Tensor& k, const Tensor& v,
                               const Tensor& w, const Tensor& b, const Tensor& g, const std::optional<Tensor>& h0) {
    Tensor xs[6] = {q.contiguous(), k.contiguous(), v.contiguous(), w.contiguous(), b.contiguous(), g.contiguous()};
    Tensor h = h0 ? h0->contiguous() : Tensor();
    const int64_t B = q.size(0), H = q.size(1), L = q.size(2), D = q.size(3);
    c10::DeviceGuard guard(q.device());
    void* stream = stream_of(q.device());
    Tensor o = empty_on(q, {B, H, L, D}, at::kFloat);
    variable_list saved(xs, xs + 6);
    for (int64_t t0 = 0; t0 < L; t0 += op->segment) {
      const gdn2_desc d = op->training_desc(B, H, std::min(L - t0, op->segment), D, L);
      size_t off[GDN2_RES_COUNT], total = 0;
      if (abi.residual_layout(&d, off, &total)) throw Refused();
      Tensor res = empty_on(q, {(int64_t)total}, at::kByte);
      Tensor ws = empty_on(q, {(int64_t)abi.fwd_ws(&d, 1)}, at::kByte);
      Tensor hf = empty_on(q, {B, H, D, D}, at::kFloat);
      const int64_t x = t0 * D;
      if (abi.fwd(&d, f32_at(xs[0], x), f32_at(xs[1], x), f32_at(xs[2], x), f32_at(xs[3], x), f32_at(xs[4], x),
                  f32_at(xs[5], x), f32_at(h), f32_at(o, x), f32_at(hf), res.data_ptr(), ws.data_ptr(), stream))
        throw Refused();
      saved.push_back(res);
      h = hf;
    }
    ctx->save_for_backward(saved);
    ctx->saved_data["op"] = std::string(reinterpret_cast<const char*>(op), sizeof(Op));
    ctx->saved_data["h0"] = h0.has_value() && h0->requires_grad();
    ctx->saved_data["shape"] = std::vector<int64_t>{B, H, L, D};
    ctx->saved_data["device"] = q.device();
    return {o, h};
  }

  static variable_list backward(AutogradContext* ctx, variable_list gs) {
    const variable_list saved = ctx->get_saved_variables();
    Op conf;
    std::memcpy(&conf, ctx->saved_data["op"].toStringRef().data(), sizeof(Op));
    const Op* op = &conf;
    const std::vector<int64_t> shape = ctx->saved_data["shape"].toIntVector();
    const int64_t B = shape[0], H = shape[1], L = shape[2], D = shape[3];
    const c10::Device dev = ctx->saved_data["device"].toDevice();
    c10::DeviceGuard guard(dev);
    void* stream = stream_of(dev);
    Tensor xs[6];
    for (int i = 0; i < 6; ++i) xs[i] = restored(saved[i], shape, at::kFloat, dev);
    Tensor dout = gs[0].to(at::kFloat).contiguous(), dh = gs[1].to(at::kFloat).contiguous();
    Tensor gr[6];
    for (Tensor& t : gr) t = empty_on(xs[0], {B, H, L, D}, at::kFloat);
    const int64_t n_seg = (L + op->segment - 1) / op->segment;
    for (int64_t s = n_seg - 1; s >= 0; --s) {
      const int64_t t0 = s * op->segment, x = t0 * D;
      const gdn2_desc d = op->training_desc(B, H, std::min(L - t0, op->segment), D, L);
      size_t off[GDN2_RES_COUNT], total = 0;
      TORCH_CHECK(abi.residual_layout(&d, off, &total) == 0, "gdn2_bwd: ", abi.last_error());
      const Tensor res = restored(saved[6 + s], {(int64_t)total}, at::kByte, dev);
      Tensor ws = empty_on(xs[0], {(int64_t)abi.bwd_ws(&d)}, at::kByte);
      Tensor dh0 = empty_on(xs[0], {B, H, D, D}, at::kFloat);
      const int st = abi.bwd(&d, f32_at(xs[0], x), f32_at(xs[1], x), f32_at(xs[2], x), f32_at(xs[3], x),
                             f32_at(xs[4], x), f32_at(xs[5], x), res.data_ptr(), f32_at(dout, x), f32_at(dh),
                             f32_at(gr[0], x), f32_at(gr[1], x), f32_at(gr[2], x), f32_at(gr[3], x), f32_at(gr[4], x),
                             f32_at(gr[5], x), f32_at(dh0), ws.data_ptr(), stream);
      TORCH_CHECK(st == 0, "gdn2_bwd: ", abi.last_error());
      dh = dh0;
    }
    variable_list out{gr[0], gr[1], gr[2], gr[3], gr[4], gr[5], ctx->saved_data["h0"].toBool() ? dh : Tensor()};
    if (at::GradMode::is_enabled()) {
      // a backward that keeps its graph: the kernels' gradients have no derivative, and say so when asked
      if (!out.back().defined()) out.pop_back();
      variable_list from(gs);
      from.insert(from.end(), saved.begin(), saved.begin() + 6);
      // (copies made of strided inputs have no history: a leaf of its own keeps the node in the graph)
      from.push_back(at::empty({0}).requires_grad_(true));
      out = Once::apply(at::TensorList(from), out);
      out.resize(7);
    }
    out.insert(out.begin(), Tensor());
    return out;
  }
};

// No gradient: one kernel sequence over all L, float32 or bfloat16 inputs.
variable_list forward_only(const Op* op, const Tensor* in, const Tensor& h0) {
  const bool bf16 = in[0].scalar_type() == at::kBFloat16;
  Tensor xs[6];
  for (int i = 0; i < 6; ++i) xs[i] = in[i].contiguous();
  const Tensor h = h0.defined() ? h0.contiguous() : Tensor();
  const int64_t B = xs[0].size(0), H = xs[0].size(1), L = xs[0].size(2), D = xs[0].size(3);
  c10::DeviceGuard guard(xs[0].device());
  const gdn2_desc d = op->desc(B, H, L, D, 0, 0);
  Tensor o = empty_on(xs[0], {B, H, L, D}, at::kFloat), hf = empty_on(xs[0], {B, H, D, D}, at::kFloat);
  Tensor ws = empty_on(xs[0], {(int64_t)abi.fwd_ws(&d, 0)}, at::kByte);
  void* stream = stream_of(xs[0].device());
  int st;
  if (bf16) {
    auto p = [&](int i) { return static_cast<const uint16_t*>(xs[i].data_ptr()); };
    st = abi.fwd_bf16(&d, p(0), p(1), p(2), p(3), p(4), p(5), f32_at(h), f32_at(o), f32_at(hf), nullptr, ws.data_ptr(), stream);
  } else {
    st = abi.fwd(&d, f32_at(xs[0]), f32_at(xs[1]), f32_at(xs[2]), f32_at(xs[3]), f32_at(xs[4]), f32_at(xs[5]), f32_at(h),
                 f32_at(o), f32_at(hf), nullptr, ws.data_ptr(), stream);
  }
  if (st) throw Refused();
  return {o, hf};
}

// Runs f without the interpreter lock (a launch can block while the device's queue is full).
template <class F>
auto unlocked(F&& f) {
  struct Lock {
    PyThreadState* s = PyEval_SaveThread();
    ~Lock() { PyEval_RestoreThread(s); }
  } lock;
  return f();
}
PyObject* pair(const Tensor& a, const Tensor& b) {
  PyObject* x = THPVariable_Wrap(a);
  PyObject* y = x ? THPVariable_Wrap(b) : nullptr;
  PyObject* t = y ? PyTuple_Pack(2, x, y) : nullptr;
  Py_XDECREF(x);
  Py_XDECREF(y);
  return t;
}
PyObject* none() { Py_RETURN_NONE; }

// bind(addresses): the C ABI's entry points in the order of struct Abi
PyObject* py_bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
  constexpr Py_ssize_t kN = sizeof(Abi) / sizeof(void*);
  if (n != kN) return PyErr_Format(PyExc_TypeError, "bind takes %zd addresses", kN);
  void* p[kN];
  for (Py_ssize_t i = 0; i < kN; ++i) {
    p[i] = PyLong_AsVoidPtr(args[i]);
    if (PyErr_Occurred()) return nullptr;
  }
  std::memcpy(static_cast<void*>(&abi), p, sizeof(abi));
  return none();
}

const char* const kOpName = "atomic_gdn2._bind.op";
void free_op(PyObject* cap) { delete static_cast<Op*>(PyCapsule_GetPointer(cap, kOpName)); }

// op(descriptor bytes, segment tokens): a configuration for sequence()
PyObject* py_op(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 2 || !PyBytes_Check(args[0]) || PyBytes_GET_SIZE(args[0]) != (Py_ssize_t)sizeof(gdn2_desc))
    return PyErr_Format(PyExc_TypeError, "op takes the bytes of a gdn2_desc and a token count");
  Op op;
  std::memcpy(&op.base, PyBytes_AS_STRING(args[0]), sizeof(gdn2_desc));
  op.segment = PyLong_AsLongLong(args[1]);
  if (PyErr_Occurred()) return nullptr;
  if (op.segment < 1) return PyErr_Format(PyExc_ValueError, "segment must be positive");
  return PyCapsule_New(new Op(op), kOpName, free_op);
}

// sequence(op, q, k, v, w, b, g, h0 or None) -> (o, h_final), or None: not a plain call
PyObject* py_sequence(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 8) return PyErr_Format(PyExc_TypeError, "sequence takes 8 arguments");
  const auto* held = static_cast<const Op*>(PyCapsule_GetPointer(args[0], kOpName));
  if (!held) return nullptr;
  const Op op = *held;
  for (int i = 1; i < 7; ++i)
    if (!THPVariable_Check(args[i])) return none();
  if (args[7] != Py_None && !THPVariable_Check(args[7])) return none();
  Tensor x[6], h0;
  for (int i = 0; i < 6; ++i) x[i] = THPVariable_Unpack(args[1 + i]);
  if (args[7] != Py_None) h0 = THPVariable_Unpack(args[7]);
  if (!plain_mode() || !x[0].is_cuda() || x[0].dim() != 4 || x[0].numel() == 0) return none();
  const c10::Device dev = x[0].device();
  const at::ScalarType dt = x[0].scalar_type();
  bool grad = false;
  for (const Tensor& t : x) {
    if (!plain(t, dev) || t.scalar_type() != dt || t.sizes() != x[0].sizes()) return none();
    grad = grad || t.requires_grad();
  }
  const int64_t L = x[0].size(2), D = x[0].size(3);
  for (int i = 0; i < 4; ++i)
    if (x[0].size(i) > INT32_MAX) return none();
  if (L % op.base.bt) return none();
  if (h0.defined()) {
    if (!plain(h0, dev) || h0.scalar_type() != at::kFloat || h0.dim() != 4 || h0.size(0) != x[0].size(0) ||
        h0.size(1) != x[0].size(1) || h0.size(2) != D || h0.size(3) != D)
      return none();
    grad = grad || h0.requires_grad();
  }
  grad = grad && at::GradMode::is_enabled();
  if (dt != at::kFloat && (grad || dt != at::kBFloat16)) return none();
  if (grad && !(op.base.clip <= 1e4)) return none();
  variable_list out;
  bool refused = false;
  unlocked([&] {
    try {
      if (grad)
        out = Sequence::apply(&op, x[0], x[1], x[2], x[3], x[4], x[5], h0.defined() ? std::optional<Tensor>(h0) : std::nullopt);
      else
        out = forward_only(&op, x, h0);
    } catch (const Refused&) {
      refused = true;
    }
  });
  return refused ? none() : pair(out[0], out[1]);
  END_HANDLE_TH_ERRORS
}

// Row indices as the kernels take them: n of int32 or int64 (kind), contiguous on the device.
bool row_indices(const Tensor& t, const c10::Device& dev, int64_t n, int* kind) {
  if (!plain(t, dev) || !t.is_contiguous() || t.dim() != 1 || t.numel() != n) return false;
  *kind = t.scalar_type() == at::kInt ? GDN2_FLAG_INT32 : GDN2_FLAG_INT64;
  return t.scalar_type() == at::kInt || t.scalar_type() == at::kLong;
}

// decode(q, k, v, w, b, g, state, scale, reset or None, state is bf16, tau or None, fuse, a_log or
// None, dt_bias or None[, parents or None]) -> (o, new state), or None: not a plain call
PyObject* py_decode(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 14 && n != 15) return PyErr_Format(PyExc_TypeError, "decode takes 14 or 15 arguments");
  for (int i = 0; i < 7; ++i)
    if (!THPVariable_Check(args[i])) return none();
  for (int i : {8, 12, 13, 14})
    if (i < n && args[i] != Py_None && !THPVariable_Check(args[i])) return none();
  if (!PyFloat_Check(args[7]) || (args[10] != Py_None && !PyFloat_Check(args[10]))) return none();
  Tensor x[7], reset, a_log, dt_bias, parents;
  for (int i = 0; i < 7; ++i) x[i] = THPVariable_Unpack(args[i]);
  if (args[8] != Py_None) reset = THPVariable_Unpack(args[8]);
  const bool sbf = PyObject_IsTrue(args[9]) == 1, fuse = PyObject_IsTrue(args[11]) == 1;
  if (args[12] != Py_None) a_log = THPVariable_Unpack(args[12]);
  if (args[13] != Py_None) dt_bias = THPVariable_Unpack(args[13]);
  if (n == 15 && args[14] != Py_None) parents = THPVariable_Unpack(args[14]);
  if (!plain_mode() || !x[0].is_cuda() || x[0].dim() != 3 || x[0].numel() == 0) return none();
  const c10::Device dev = x[0].device();
  const int64_t B = x[0].size(0), H = x[0].size(1), D = x[0].size(2);
  const at::ScalarType dt = x[0].scalar_type(), sdt = sbf ? at::kBFloat16 : at::kFloat;
  if ((dt != at::kFloat && dt != at::kBFloat16) || (D != 64 && D != 128) || B * H > (int64_t(1) << 22)) return none();
  auto ready = [&](const Tensor& t, at::ScalarType ty) {
    return plain(t, dev) && t.scalar_type() == ty && t.is_contiguous() && (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0;
  };
  for (int i = 0; i < 6; ++i)
    if (!ready(x[i], dt) || x[i].sizes() != x[0].sizes()) return none();
  int from = 0;
  if (parents.defined() && !row_indices(parents, dev, B, &from)) return none();
  if (!ready(x[6], sdt) || x[6].dim() != 4 || (from ? x[6].size(0) < 1 || x[6].size(0) > INT32_MAX : x[6].size(0) != B) || x[6].size(1) != H || x[6].size(2) != D || x[6].size(3) != D)
    return none();
  int kind = 0;
  if (reset.defined()) {
    if (!plain(reset, dev) || !reset.is_contiguous() || reset.numel() != B) return none();
    switch (reset.scalar_type()) {
      case at::kBool: case at::kByte: kind = GDN2_FLAG_BYTE; break;
      case at::kInt: kind = GDN2_FLAG_INT32; break;
      case at::kLong: kind = GDN2_FLAG_INT64; break;
      default: return none();
    }
  }
  if (fuse && !(a_log.defined() && dt_bias.defined() && ready(a_log, at::kFloat) && ready(dt_bias, at::kFloat) &&
                a_log.numel() == H && dt_bias.numel() == D))
    return none();
  gdn2_decode_desc d{};
  d.B = (int32_t)B; d.H = (int32_t)H; d.D = (int32_t)D;
  d.n_tok = d.seq_ld = 1;
  d.in_dtype = d.out_dtype = dt == at::kBFloat16;
  d.state_dtype = sbf;
  d.fuse_prologue = fuse;
  d.cap = args[10] != Py_None;
  d.scale = PyFloat_AS_DOUBLE(args[7]);
  d.stability_tau = d.cap ? PyFloat_AS_DOUBLE(args[10]) : 0.0;
  Tensor o, st;
  int status = 0;
  unlocked([&] {
    c10::DeviceGuard guard(dev);
    o = empty_on(x[0], {B, H, D}, dt);
    st = empty_on(x[0], {B, H, D, D}, sdt);
    auto p = [&](const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
    status = abi.decode(&d, kind, p(x[0]), p(x[1]), p(x[2]), p(x[3]), p(x[4]), p(x[5]),
                        fuse ? f32_at(a_log) : nullptr, fuse ? f32_at(dt_bias) : nullptr, p(reset), from, p(parents),
                        (int)x[6].size(0), p(x[6]), p(o), p(st),
                        stream_of(dev));
  });
  return status ? none() : pair(o, st);
  END_HANDLE_TH_ERRORS
}

bool tensors_of(PyObject* t) {
  if (!PyTuple_Check(t)) return false;
  for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(t); ++i)
    if (!THPVariable_Check(PyTuple_GET_ITEM(t, i))) return false;
  return true;
}
// A whole number of a call's arguments; false with no error set: not one.
bool whole(PyObject* o, int64_t* x) {
  if (!PyLong_CheckExact(o)) return false;
  int over = 0;
  *x = PyLong_AsLongLongAndOverflow(o, &over);
  return !over;
}
// GDN2_F32, GDN2_BF16, GDN2_F16, or -1
int float_kind(at::ScalarType t) { return t == at::kFloat ? 0 : t == at::kBFloat16 ? 1 : t == at::kHalf ? 2 : -1; }
// The stride of t's rows of n elements, t (..., n): t is contiguous or a matrix with whole rows; else 0.
int64_t row_stride(const Tensor& t, int64_t n) {
  if (t.is_contiguous()) return n;
  return t.dim() == 2 && t.stride(1) == 1 && (t.stride(0) >= n || t.size(0) == 1) ? std::max(t.stride(0), n) : 0;
}
// Whether gradients are recorded of one of ts: Python's path has the error for them.
bool recorded(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}
PyObject* tuple_of(std::initializer_list<const Tensor*> ts) {
  PyObject* out = PyTuple_New((Py_ssize_t)ts.size());
  Py_ssize_t i = 0;
  for (const Tensor* t : ts) {
    PyObject* x = out ? THPVariable_Wrap(*t) : nullptr;
    if (!x) {
      Py_XDECREF(out);
      return nullptr;
    }
    PyTuple_SET_ITEM(out, i++, x);
  }
  return out;
}

// w4(x, q, meta, in, out, group, bias or None, residual or None) -> y, or None: not a plain call
PyObject* py_w4(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 8) return PyErr_Format(PyExc_TypeError, "w4 takes 8 arguments");
  int64_t K, N, group;
  if (!THPVariable_Check(args[0]) || !THPVariable_Check(args[1]) || !THPVariable_Check(args[2]) || !whole(args[3], &K) ||
      !whole(args[4], &N) || !whole(args[5], &group))
    return none();
  Tensor x = THPVariable_Unpack(args[0]), q = THPVariable_Unpack(args[1]), meta = THPVariable_Unpack(args[2]), bias, res;
  for (int i : {6, 7}) {
    if (args[i] == Py_None) continue;
    if (!THPVariable_Check(args[i])) return none();
    (i == 6 ? bias : res) = THPVariable_Unpack(args[i]);
  }
  if (!plain_mode() || !x.is_cuda() || x.dim() < 1 || x.numel() == 0 || x.size(-1) != K) return none();
  const c10::Device dev = x.device();
  const at::ScalarType dt = x.scalar_type();
  const int kind = float_kind(dt);
  const int64_t M = x.numel() / K, ldx = row_stride(x, K);
  if (kind < 0 || !ldx || !plain(x, dev) || M > INT32_MAX || K > INT32_MAX || N > INT32_MAX) return none();
  for (const Tensor* t : {&q, &meta})
    if (!plain(*t, dev) || t->scalar_type() != at::kInt || !t->is_contiguous()) return none();
  // (the kernels read by K, N and group: a weight whose tensors have other sizes is not theirs)
  const int64_t blocks = ((N + 15) / 16) * ((K + 127) / 128);
  if (K < 1 || N < 1 || (group != 32 && group != 64 && group != 128) || q.numel() != 256 * blocks ||
      meta.numel() != 16 * (128 / group) * blocks)
    return none();
  if (bias.defined() && (!plain(bias, dev) || bias.scalar_type() != dt || bias.dim() != 1 || bias.size(0) != N || !bias.is_contiguous()))
    return none();
  int64_t ldr = 0;
  if (res.defined()) {
    if (!plain(res, dev) || res.scalar_type() != dt || res.dim() != x.dim() || res.size(-1) != N) return none();
    for (int64_t i = 0; i + 1 < x.dim(); ++i)
      if (res.size(i) != x.size(i)) return none();
    if (!(ldr = row_stride(res, N))) return none();
  }
  if (recorded({&x, &bias, &res})) return none();
  gdn2_w4 a{};
  a.M = (int32_t)M; a.K = (int32_t)K; a.N = (int32_t)N; a.group = (int32_t)group;
  a.dtype = kind; a.ldx = ldx; a.ldr = ldr;
  a.x = x.data_ptr(); a.q = q.data_ptr(); a.meta = meta.data_ptr();
  a.bias = bias.defined() ? bias.data_ptr() : nullptr;
  a.residual = res.defined() ? res.data_ptr() : nullptr;
  Tensor y;
  int status = 0;
  unlocked([&] {
    c10::DeviceGuard guard(dev);
    at::DimVector size(x.sizes());
    size.back() = N;
    y = empty_on(x, size, dt);
    a.y = y.data_ptr();
    const int64_t bytes = (int64_t)abi.w4_ws(&a);
    const Tensor ws = bytes ? empty_on(x, {bytes}, at::kByte) : Tensor();
    status = abi.w4(&a, bytes ? ws.data_ptr() : nullptr, stream_of(dev));
  });
  return status ? none() : THPVariable_Wrap(y);
  END_HANDLE_TH_ERRORS
}

// beam(logits, scores, n, finished or None, eos or -1) -> (tokens, rows, scores[, finished]), or None:
// not a plain call
PyObject* py_beam(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  if (n_args != 5) return PyErr_Format(PyExc_TypeError, "beam takes 5 arguments");
  int64_t n, eos;
  if (!THPVariable_Check(args[0]) || !THPVariable_Check(args[1]) || !whole(args[2], &n) || !whole(args[4], &eos) ||
      (args[3] != Py_None && !THPVariable_Check(args[3])))
    return none();
  const Tensor x = THPVariable_Unpack(args[0]), scores = THPVariable_Unpack(args[1]);
  Tensor fin;
  if (args[3] != Py_None) fin = THPVariable_Unpack(args[3]);
  if (!plain_mode() || !x.is_cuda() || scores.dim() != 2 || scores.numel() == 0 || x.dim() < 2 || x.dim() > 3 || x.numel() == 0)
    return none();
  const c10::Device dev = x.device();
  const int64_t B = scores.size(0), K = scores.size(1), V = x.size(-1), ld = row_stride(x, V);
  const int kind = float_kind(x.scalar_type());
  if (kind < 0 || !ld || !plain(x, dev) || !plain(scores, dev) || scores.scalar_type() != at::kFloat || !scores.is_contiguous())
    return none();
  if (x.dim() == 2 ? x.size(0) != B * K : x.size(0) != B || x.size(1) != K) return none();
  if (fin.defined() && (!plain(fin, dev) || fin.scalar_type() != at::kBool || fin.dim() != 2 || fin.size(0) != B || fin.size(1) != K ||
                        !fin.is_contiguous()))
    return none();
  if (B > 65535 || K > 65535 || V > INT32_MAX || n < 1 || n > std::min<int64_t>(128, K * V) || eos < -1 || eos >= V) return none();
  if (recorded({&x, &scores})) return none();
  gdn2_beam a{};
  a.B = (int32_t)B; a.K = (int32_t)K; a.V = (int32_t)V; a.n = (int32_t)n; a.eos = (int32_t)eos;
  a.dtype = kind; a.ld = ld;
  a.logits = x.data_ptr(); a.scores = f32_at(scores);
  a.finished = fin.defined() ? static_cast<const uint8_t*>(fin.data_ptr()) : nullptr;
  Tensor tokens, rows, out, done;
  int status = 0;
  unlocked([&] {
    c10::DeviceGuard guard(dev);
    const size_t bytes = abi.beam_ws(a.B, a.K, a.V, a.n);
    const int64_t c = up16(8 * B * n), f = up16(4 * B * n);
    const Tensor all = empty_on(x, {2 * c + f + up16(B * n)}, at::kByte);
    tokens = part_of(all, 0, {B, n}, at::kLong);
    rows = part_of(all, c, {B, n}, at::kLong);
    out = part_of(all, 2 * c, {B, n}, at::kFloat);
    if (eos >= 0) done = part_of(all, 2 * c + f, {B, n}, at::kBool);
    const Tensor ws = bytes ? empty_on(x, {(int64_t)bytes}, at::kByte) : Tensor();
    a.tokens = static_cast<int64_t*>(tokens.data_ptr());
    a.rows = static_cast<int64_t*>(rows.data_ptr());
    a.out_scores = f32_at(out);
    a.out_finished = done.defined() ? static_cast<uint8_t*>(done.data_ptr()) : nullptr;
    status = abi.beam(&a, bytes ? ws.data_ptr() : nullptr, stream_of(dev));
  });
  if (status) return none();
  return done.defined() ? tuple_of({&tokens, &rows, &out, &done}) : tuple_of({&tokens, &rows, &out});
  END_HANDLE_TH_ERRORS
}

// premix_step(y, history, (taps of q, k, v, their biases, the gates' biases, decay_b, decay_a), heads, g_max,
// parents or None) -> (q, k, v, w, b, g, gate, history), or None: not a plain call
PyObject* py_premix_step(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 6) return PyErr_Format(PyExc_TypeError, "premix_step takes 6 arguments");
  int64_t H;
  if (!THPVariable_Check(args[0]) || !THPVariable_Check(args[1]) || !tensors_of(args[2]) || PyTuple_GET_SIZE(args[2]) != 10 ||
      !whole(args[3], &H) || !PyFloat_Check(args[4]) || (args[5] != Py_None && !THPVariable_Check(args[5])))
    return none();
  const Tensor y = THPVariable_Unpack(args[0]), past = THPVariable_Unpack(args[1]);
  Tensor parents;
  if (args[5] != Py_None) parents = THPVariable_Unpack(args[5]);
  if (!plain_mode() || !y.is_cuda() || y.dim() != 2 || past.dim() != 3 || y.numel() == 0 || past.numel() == 0 || H < 1 ||
      past.size(1) != 3 || past.size(2) % (3 * H))
    return none();
  const c10::Device dev = y.device();
  const int64_t R = y.size(0), S = past.size(0), C = past.size(2) / 3, D = C / H, ldy = row_stride(y, y.size(1));
  auto ready = [&](const Tensor& t) { return plain(t, dev) && t.scalar_type() == at::kFloat; };
  if ((D != 64 && D != 128) || !ldy || ldy > INT32_MAX || y.size(1) < 6 * C + H || R * H > (int64_t(1) << 28) || S > INT32_MAX ||
      !ready(y) || !ready(past) || !past.is_contiguous())
    return none();
  gdn2_lm_premix_step a{};
  if (parents.defined() ? !row_indices(parents, dev, R, &a.parent_type) : S != R) return none();
  const float* ps[10];
  for (int i = 0; i < 10; ++i) {
    const Tensor& t = THPVariable_Unpack(PyTuple_GET_ITEM(args[2], i));
    const int64_t len = i < 8 ? C : H;
    if (!ready(t) || !t.is_contiguous() || t.dim() != (i < 3 ? 2 : 1) || t.numel() != (i < 3 ? 4 * C : len) || t.size(0) != len)
      return none();
    if (recorded({&t})) return none();
    ps[i] = f32_at(t);
  }
  if (recorded({&y, &past})) return none();
  a.R = (int32_t)R; a.S = (int32_t)S; a.H = (int32_t)H; a.D = (int32_t)D; a.ldy = (int32_t)ldy;
  a.g_max = (float)PyFloat_AS_DOUBLE(args[4]);
  a.y = f32_at(y); a.history = f32_at(past);
  a.parents = parents.defined() ? parents.data_ptr() : nullptr;
  for (int i = 0; i < 3; ++i) {
    a.conv_w[i] = ps[i];
    a.conv_b[i] = ps[3 + i];
  }
  a.gate_b[0] = ps[6]; a.gate_b[1] = ps[7]; a.decay_b = ps[8]; a.decay_a = ps[9];
  Tensor out[6], gate, now;
  int status = 0;
  unlocked([&] {
    c10::DeviceGuard guard(dev);
    const Tensor all = empty_on(y, {7 * R * C}, at::kFloat);      // what the token's next steps consume
    for (int i = 0; i < 6; ++i) {
      out[i] = part_of(all, 4 * i * R * C, {R, H, D}, at::kFloat);
      a.out[i] = f32_at(out[i]);
    }
    gate = part_of(all, 4 * 6 * R * C, {R, C}, at::kFloat);
    now = empty_on(y, {R, 3, 3 * C}, at::kFloat);
    a.og = f32_at(gate);
    a.new_history = f32_at(now);
    status = abi.premix_step(&a, stream_of(dev));
  });
  return status ? none() : tuple_of({&out[0], &out[1], &out[2], &out[3], &out[4], &out[5], &gate, &now});
  END_HANDLE_TH_ERRORS
}

// What a saved tensor looked like (lm_kernels.py): forty of them a block, looked over in Python at 1.5 us
// each, would be a fifth of a small block's host time.
struct Form {
  std::vector<int64_t> sizes;
  at::ScalarType dtype;
  c10::Device device;
};
const char* const kFormsName = "atomic_gdn2._bind.forms";
void free_forms(PyObject* cap) { delete static_cast<std::vector<Form>*>(PyCapsule_GetPointer(cap, kFormsName)); }

// forms(tensors): their sizes, dtypes and devices
PyObject* py_forms(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 1 || !tensors_of(args[0])) return PyErr_Format(PyExc_TypeError, "forms takes a tuple of tensors");
  auto f = std::make_unique<std::vector<Form>>();
  for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(args[0]); ++i) {
    const Tensor& t = THPVariable_Unpack(PyTuple_GET_ITEM(args[0], i));
    f->push_back(Form{t.sizes().vec(), t.scalar_type(), t.device()});
  }
  PyObject* cap = PyCapsule_New(f.get(), kFormsName, free_forms);
  if (cap) f.release();
  return cap;
  END_HANDLE_TH_ERRORS
}

// differ(forms, tensors) -> None when every tensor has its form, contiguous and 16-byte aligned; else
// a list with (sizes, dtype, device) for those that do not, None for the others
PyObject* py_differ(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 2 || !tensors_of(args[1])) return PyErr_Format(PyExc_TypeError, "differ takes forms and a tuple of tensors");
  const auto* f = static_cast<const std::vector<Form>*>(PyCapsule_GetPointer(args[0], kFormsName));
  if (!f) return nullptr;
  if ((Py_ssize_t)f->size() != PyTuple_GET_SIZE(args[1])) return PyErr_Format(PyExc_ValueError, "another number of tensors");
  auto same = [&](const Tensor& t, const Form& o) {
    return t.layout() == c10::kStrided && t.sizes() == at::IntArrayRef(o.sizes) && t.scalar_type() == o.dtype &&
           t.device() == o.device && t.is_contiguous() && (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0;
  };
  bool all = true;
  for (size_t i = 0; i < f->size() && all; ++i) all = same(THPVariable_Unpack(PyTuple_GET_ITEM(args[1], i)), (*f)[i]);
  if (all) return none();
  PyObject* out = PyList_New((Py_ssize_t)f->size());
  for (size_t i = 0; out && i < f->size(); ++i) {
    const Form& o = (*f)[i];
    PyObject* x = Py_None;
    if (same(THPVariable_Unpack(PyTuple_GET_ITEM(args[1], i)), o)) {
      Py_INCREF(x);
    } else {
      PyObject *sz = PyTuple_New((Py_ssize_t)o.sizes.size()), *dev = THPDevice_New(o.device);
      for (size_t k = 0; sz && k < o.sizes.size(); ++k) PyTuple_SET_ITEM(sz, (Py_ssize_t)k, PyLong_FromLongLong(o.sizes[k]));
      PyObject* dt = reinterpret_cast<PyObject*>(torch::getTHPDtype(o.dtype));
      x = sz && dev ? PyTuple_Pack(3, sz, dt, dev) : nullptr;
      Py_XDECREF(sz);
      Py_XDECREF(dev);
      if (!x) {
        Py_DECREF(out);
        return nullptr;
      }
    }
    PyList_SET_ITEM(out, (Py_ssize_t)i, x);
  }
  return out;
  END_HANDLE_TH_ERRORS
}

// dense(tensors, x) -> whether each is as the kernels read it: float32, on x's device, contiguous,
// 16-byte aligned, not empty
PyObject* py_dense(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 2 || !tensors_of(args[0]) || !THPVariable_Check(args[1])) return PyErr_Format(PyExc_TypeError, "dense takes a tuple of tensors and a tensor");
  const c10::Device dev = THPVariable_Unpack(args[1]).device();
  for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(args[0]); ++i) {
    const Tensor& t = THPVariable_Unpack(PyTuple_GET_ITEM(args[0], i));
    if (t.layout() != c10::kStrided || t.device() != dev || t.scalar_type() != at::kFloat || t.numel() == 0 || !t.is_contiguous() ||
        (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) != 0)
      Py_RETURN_FALSE;
  }
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"bind", (PyCFunction)(void (*)())py_bind, METH_FASTCALL, "bind(*addresses)"},
    {"op", (PyCFunction)(void (*)())py_op, METH_FASTCALL, "op(desc, segment)"},
    {"sequence", (PyCFunction)(void (*)())py_sequence, METH_FASTCALL, "sequence(op, q, k, v, w, b, g, h0)"},
    {"forms", (PyCFunction)(void (*)())py_forms, METH_FASTCALL, "forms(tensors)"},
    {"differ", (PyCFunction)(void (*)())py_differ, METH_FASTCALL, "differ(forms, tensors)"},
    {"dense", (PyCFunction)(void (*)())py_dense, METH_FASTCALL, "dense(tensors, x)"},
    {"decode", (PyCFunction)(void (*)())py_decode, METH_FASTCALL, "decode(...)"},
    {"w4", (PyCFunction)(void (*)())py_w4, METH_FASTCALL, "w4(x, q, meta, in, out, group, bias, residual)"},
    {"beam", (PyCFunction)(void (*)())py_beam, METH_FASTCALL, "beam(logits, scores, n, finished, eos)"},
    {"premix_step", (PyCFunction)(void (*)())py_premix_step, METH_FASTCALL, "premix_step(y, history, weights, heads, g_max, parents)"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module{PyModuleDef_HEAD_INIT, "_bind", "native call path of the operator", -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__bind(void) { return PyModule_Create(&module); }
