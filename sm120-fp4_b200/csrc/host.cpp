// Host side of the quantiser calls that are host time for the most part (16 x 2048 bf16: 2.4 us on the GPU, 11.5 us from Python, of which three allocations
// 4.8, the ctypes call 1.1 and the launch 2.5; 5.7 us this way): argument checks, allocations and the library call in one call into native code. Each function takes plain CUDA
// tensors on the current device only and returns None for whatever it does not take - the caller's general path, with its checks and errors, is then
// the one that runs -, the error code of the library as an int, or the outputs.
#include <Python.h>
#include <ATen/ATen.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/variable.h>

namespace {

using OwnScale = int (*)(const void*, int, int, int, int, void*, void*, void*, int, void*, long long, void*);
using Quantize = int (*)(const void*, int, const int*, int, int, const void*, int, void*, void*, int, void*);
OwnScale own_scale = nullptr;
Quantize quantize = nullptr;
long long one_cluster = 0;   // values of a matrix up to which own_scale needs no workspace

// Nothing that would see the torch calls of the general path: function and dispatch modes, functorch transforms, functionalisation.
bool plain_call() {
  using c10::DispatchKey;
  return !at::impl::torch_function_mode_enabled() && !c10::impl::tls_is_dispatch_key_included(DispatchKey::Python) &&
         !c10::impl::tls_is_dispatch_key_included(DispatchKey::PythonTLSSnapshot) &&
         !c10::impl::tls_is_dispatch_key_included(DispatchKey::FuncTorchDynamicLayerFrontMode) &&
         !c10::impl::tls_is_dispatch_key_included(DispatchKey::FuncTorchDynamicLayerBackMode) &&
         !c10::impl::tls_is_dispatch_key_included(DispatchKey::Functionalize);
}

bool plain_tensor(const at::Tensor& t) {
  using c10::DispatchKey;
  const c10::DispatchKeySet k = t.key_set();
  return t.is_cuda() && t.layout() == at::kStrided && !k.has(DispatchKey::Python) && !k.has(DispatchKey::FuncTorchBatched) && !k.has(DispatchKey::FuncTorchGradWrapper) &&
         !k.has(DispatchKey::Functionalize) && !k.has(DispatchKey::Negative) && !k.has(DispatchKey::ZeroTensor);
}

// a matrix the kernels take as it is: bf16 or fp32, whole blocks of 16, contiguous, on the current device
bool plain_matrix(const at::Tensor& x) {
  return plain_tensor(x) && x.dim() == 2 && (x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kFloat) && x.size(0) > 0 && x.size(1) > 0 && x.size(1) % 16 == 0 &&
         x.is_contiguous() && x.get_device() == c10::cuda::current_device();
}

at::Tensor bytes(int64_t rows, int64_t cols, const at::Tensor& like) { return at::empty({rows, cols}, at::TensorOptions().dtype(at::kByte).device(like.device())); }

// Python runs on meanwhile, as under torch's own calls: an allocation may wait for the device, and the device for a callback that wants the interpreter.
struct Released {
  PyThreadState* state = PyEval_SaveThread();
  ~Released() { PyEval_RestoreThread(state); }
};

PyObject* outputs(int rc, const at::Tensor& packed, const at::Tensor& sf, PyObject* scale) {   // takes over the reference to scale
  if (rc) {
    Py_XDECREF(scale);
    return PyLong_FromLong(rc);
  }
  PyObject *p = THPVariable_Wrap(packed), *s = THPVariable_Wrap(sf), *t = p && s && scale ? PyTuple_New(3) : nullptr;
  if (!t) {
    Py_XDECREF(p), Py_XDECREF(s), Py_XDECREF(scale);
    return nullptr;
  }
  PyTuple_SET_ITEM(t, 0, p), PyTuple_SET_ITEM(t, 1, s), PyTuple_SET_ITEM(t, 2, scale);
  return t;
}

// bind(address of b200moe_quantize_nvfp4_own_scale, of b200moe_quantize_nvfp4, one_cluster)
PyObject* py_bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 3) {
    PyErr_SetString(PyExc_TypeError, "bind takes two addresses and a size");
    return nullptr;
  }
  void *a = PyLong_AsVoidPtr(args[0]), *b = PyLong_AsVoidPtr(args[1]);
  const long long c = PyLong_AsLongLong(args[2]);
  if (PyErr_Occurred()) return nullptr;
  own_scale = (OwnScale)a, quantize = (Quantize)b, one_cluster = c;
  Py_RETURN_NONE;
}

// quantize_own_scale(x): one matrix small enough to need no workspace, its own global scale, row-major block scales
PyObject* py_quantize_own_scale(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 1 || !own_scale || !THPVariable_CheckExact(args[0]) || !plain_call()) Py_RETURN_NONE;
  const at::Tensor x = THPVariable_Unpack(args[0]);
  if (!plain_matrix(x) || x.numel() > one_cluster) Py_RETURN_NONE;
  const int64_t rows = x.size(0), k = x.size(1);
  at::Tensor packed, sf, gs;
  int rc;
  {
    Released released;
    packed = bytes(rows, k / 2, x), sf = bytes(rows, k / 16, x), gs = at::empty({1}, at::TensorOptions().dtype(at::kFloat).device(x.device()));
    rc = own_scale(x.data_ptr(), x.scalar_type() == at::kFloat, 1, (int)rows, (int)k, gs.data_ptr(), packed.data_ptr(), sf.data_ptr(), 0, nullptr, 0,
                   (void*)c10::cuda::getCurrentCUDAStream().stream());
  }
  return outputs(rc, packed, sf, THPVariable_Wrap(gs));
  END_HANDLE_TH_ERRORS
}

// quantize_128x4(x, global_scale): block scales in the 128x4 swizzle
PyObject* py_quantize_128x4(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 2 || !quantize || !THPVariable_CheckExact(args[0]) || !THPVariable_CheckExact(args[1]) || !plain_call()) Py_RETURN_NONE;
  const at::Tensor x = THPVariable_Unpack(args[0]), gs = THPVariable_Unpack(args[1]);
  if (!plain_matrix(x) || !plain_tensor(gs) || gs.scalar_type() != at::kFloat || gs.dim() != 1 || gs.size(0) != 1 || gs.device() != x.device()) Py_RETURN_NONE;
  const int64_t rows = x.size(0), k = x.size(1);
  if (rows > 0x7fffffff - 128 || k > 0x7fffffff) Py_RETURN_NONE;
  at::Tensor packed, sf;
  int rc;
  {
    Released released;
    packed = bytes(rows, k / 2, x), sf = bytes((rows + 127) / 128 * 128, (k / 16 + 3) / 4 * 4, x);
    rc = quantize(x.data_ptr(), x.scalar_type() == at::kFloat, nullptr, (int)rows, (int)k, gs.data_ptr(), 0, packed.data_ptr(), sf.data_ptr(), 1,
                  (void*)c10::cuda::getCurrentCUDAStream().stream());
  }
  Py_INCREF(args[1]);
  return outputs(rc, packed, sf, args[1]);
  END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------------------------------------------- router and FP8 operators
// The same for the router from logits, its balance loss and the FP8 operators: what gate.py and fp8.py do for plain tensors, gradients included, as nodes of
// the autograd engine that call the library: a training step of the gate of 16384 x 128 logits takes 58 us instead of 100, of which the engine's hand-over to its device
// thread and back takes 37 for any operator.
struct Ops {
  int (*gate)(const void*, int, long long, int, int, int, int, void*, void*, void*);
  int (*gate_backward)(const void*, const void*, const void*, const void*, int, long long, int, int, int, int, void*, void*);
  long long (*balance_workspace_bytes)(int, int);
  int (*balance_loss)(const void*, int, long long, int, int, const void*, int, void*, void*, void*, void*, long long, void*);
  int (*balance_backward)(const void*, const void*, int, long long, int, int, const void*, int, const void*, const void*, void*, void*);
  long long (*quantize_fp8_workspace_bytes)(int, int, int);
  int (*quantize_fp8)(const void*, int, long long, int, const void*, int, int, void*, long long, void*, void*, long long, void*);
  int (*quantize_fp8_blocks)(const void*, int, int, int, int, void*, long long, void*, void*);
  int (*matmul_fp8)(const void*, long long, const void*, const void*, long long, const void*, int, int, int, void*, int, long long, void*);
  int (*matmul_fp8_experts)(const void*, long long, const void*, int, const void*, long long, const void*, int, const void*, const void*, int, int, int, void*, int, long long,
                            int, void*);
  const char* (*error_string)(int);
} ops = {};
constexpr int64_t kMaxExperts = 512, kMaxTopK = 16, kMaxSize = 1ll << 30;

void* raw_stream() { return (void*)c10::cuda::getCurrentCUDAStream().stream(); }
int dtype_code(at::ScalarType t) { return t == at::kBFloat16 ? 0 : t == at::kFloat ? 1 : t == at::kHalf ? 2 : -1; }
at::Tensor fresh(at::IntArrayRef size, at::ScalarType t, const at::Tensor& like) { return at::empty(size, at::TensorOptions().dtype(t).device(like.device())); }
bool here(const at::Tensor& t) { return plain_tensor(t) && t.get_device() == c10::cuda::current_device(); }
bool plain_logits(const at::Tensor& x) {
  return here(x) && !x._fw_grad(0).defined() && x.dim() == 2 && dtype_code(x.scalar_type()) >= 0 && x.size(0) > 0 && x.size(0) <= kMaxSize && x.size(1) > 0 && x.size(1) <= kMaxExperts && x.stride(1) == 1 &&
         (x.stride(0) >= x.size(1) || x.size(0) == 1);
}
long long row_stride(const at::Tensor& x) { return std::max(x.stride(0), x.size(1)); }
// (the FP8 calls have no derivatives: inputs that ask for one are refused on the general path)
bool no_gradient(const at::Tensor& t) { return !(t.requires_grad() && at::GradMode::is_enabled()) && !t._fw_grad(0).defined(); }
bool vector_of(const at::Tensor& t, at::ScalarType type) { return here(t) && t.dim() == 1 && t.scalar_type() == type && t.is_contiguous(); }
void checked(int rc, const char* what) {      // (the message as one string: no streams)
  if (rc) TORCH_CHECK(false, std::string(what) + ": " + ops.error_string(rc) + " (" + std::to_string(rc) + ")");
}
// The gradient of a gradient is not there: whoever asks for it is told so.
at::Tensor once(at::Tensor out, const char* what) {
  if (!at::GradMode::is_enabled()) return out;
  auto error = std::make_shared<torch::autograd::DelayedError>(std::string(what) + " is differentiable once", 1);
  return (*error)({out.detach().requires_grad_(true)})[0];
}

// A gradient with its values in memory as they read: the sign of a negated view is a mark beside them, and some gradients are zeros without memory.
at::Tensor stored(const at::Tensor& grad) {
  at::Tensor t = grad.detach();
  if (t._is_zerotensor()) t = t.clone();
  return t.resolve_neg().contiguous();
}

// A saved tensor as the forward pass saw it. Hooks on saved tensors may give back another one, whose memory would be read as if it were the first.
at::Tensor unpacked(const torch::autograd::SavedVariable& saved, at::IntArrayRef size, at::ScalarType type, const at::Tensor& grad, const char* what,
                    std::shared_ptr<torch::autograd::Node> made_by = nullptr) {
  const at::Tensor t = saved.unpack(std::move(made_by));
  TORCH_CHECK(t.layout() == at::kStrided && t.device() == grad.device() && t.scalar_type() == type && t.sizes() == size,
              std::string(what) + " backward: a hook gave back a saved tensor of another size, type or device");
  if (plain_tensor(t) && (t.is_contiguous() || (t.dim() == 2 && t.stride(1) == 1 && t.stride(0) >= t.size(1)))) return t;
  return stored(t);
}

// A leaf's gradient is handed over on the stream on which its accumulator was made. Where an eager graph keeps that alive, a backward pass that is being captured
// on another stream would have the engine wait across the two, which ends the process: refused while it still can be.
void check_capture(const at::Tensor& x, const char* what) {
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None || !x.is_leaf()) return;
  const auto node = torch::autograd::impl::try_get_grad_accumulator(x);
  if (!node) return;
  const auto made_on = node->stream();
  TORCH_CHECK(!made_on || *made_on == c10::cuda::getCurrentCUDAStream().unwrap(),
              std::string(what) + ": a graph of the same leaf that was made on another stream is still alive; drop its outputs before a capture that takes gradients");
}

using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

// Nodes of their own instead of torch::autograd::Function: a training step of the gate takes 6 us less host time.
template <typename N> std::shared_ptr<N> node_of(const at::Tensor& x) {
  auto node = std::shared_ptr<N>(new N(), torch::autograd::deleteNode);
  node->set_next_edges(torch::autograd::collect_next_edges(x));
  return node;
}

int run_gate(const at::Tensor& x, int64_t k, bool renormalize, at::Tensor& weights, at::Tensor& ids) {
  weights = fresh({x.size(0), k}, at::kFloat, x), ids = fresh({x.size(0), k}, at::kInt, x);
  return ops.gate(x.data_ptr(), dtype_code(x.scalar_type()), row_stride(x), (int)x.size(0), (int)x.size(1), (int)k, renormalize, weights.data_ptr(), ids.data_ptr(), raw_stream());
}
struct GateBackward : torch::autograd::Node {
  SavedVariable weights, ids, x;      // (normalised weights do not depend on the experts left out: no x)
  int64_t tokens = 0, e = 0, k = 0;
  at::ScalarType dtype = at::kFloat;
  bool renormalize = true;
  std::string name() const override { return "TopKGateBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    weights.reset_data(), ids.reset_data(), x.reset_data();
  }
  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    if (!grads[0].defined() || !task_should_compute_output(0)) return {at::Tensor()};
    const at::Tensor grad = stored(grads[0]), w = unpacked(weights, {tokens, k}, at::kFloat, grad, "top_k_gate", shared_from_this()).contiguous(),
                     i = unpacked(ids, {tokens, k}, at::kInt, grad, "top_k_gate").contiguous(),
                     l = renormalize ? at::Tensor() : unpacked(x, {tokens, e}, dtype, grad, "top_k_gate");
    const at::Tensor out = fresh({w.size(0), e}, dtype, w);
    checked(ops.gate_backward(grad.data_ptr(), w.data_ptr(), i.data_ptr(), l.defined() ? l.data_ptr() : nullptr, dtype_code(dtype), l.defined() ? row_stride(l) : e, (int)w.size(0),
                              (int)e, (int)w.size(1), renormalize, out.data_ptr(), raw_stream()),
            "top_k_gate backward");
    return {once(out, "top_k_gate")};
  }
};
int gate_with_grad(const at::Tensor& x, int64_t k, bool renormalize, at::Tensor& weights, at::Tensor& ids) {
  const auto node = node_of<GateBackward>(x);
  if (const int rc = run_gate(x, k, renormalize, weights, ids)) return rc;
  node->tokens = x.size(0), node->e = x.size(1), node->k = k, node->dtype = x.scalar_type(), node->renormalize = renormalize;
  torch::autograd::set_history(weights, node);
  node->weights = SavedVariable(weights, true), node->ids = SavedVariable(ids, false);
  if (!renormalize) node->x = SavedVariable(x, false);
  return 0;
}

int run_balance(const at::Tensor& x, const at::Tensor& ids, at::Tensor& loss, at::Tensor& counts, at::Tensor& stats) {
  const int tokens = (int)x.size(0), e = (int)x.size(1);
  const long long bytes = ops.balance_workspace_bytes(tokens, e);
  if (bytes < 0) return (int)bytes;
  const at::Tensor ws = fresh({(bytes + 3) / 4}, at::kFloat, x);
  loss = fresh({}, at::kFloat, x), counts = fresh({e}, at::kInt, x), stats = fresh({2}, at::kFloat, x);
  return ops.balance_loss(x.data_ptr(), dtype_code(x.scalar_type()), row_stride(x), tokens, e, ids.data_ptr(), (int)ids.size(1), loss.data_ptr(), counts.data_ptr(), stats.data_ptr(),
                          ws.data_ptr(), bytes, raw_stream());
}
struct BalanceBackward : torch::autograd::Node {
  SavedVariable x, ids, counts, stats;
  int64_t tokens = 0, e = 0, k = 0;
  at::ScalarType dtype = at::kFloat;
  std::string name() const override { return "BalanceLossBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    x.reset_data(), ids.reset_data(), counts.reset_data(), stats.reset_data();
  }
  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    if (!grads[0].defined() || !task_should_compute_output(0)) return {at::Tensor()};
    const at::Tensor grad = stored(grads[0]), l = unpacked(x, {tokens, e}, dtype, grad, "balance_loss"), i = unpacked(ids, {tokens, k}, at::kInt, grad, "balance_loss").contiguous(),
                     c = unpacked(counts, {e}, at::kInt, grad, "balance_loss"), s = unpacked(stats, {2}, at::kFloat, grad, "balance_loss");
    const at::Tensor out = fresh({l.size(0), l.size(1)}, l.scalar_type(), l);
    checked(ops.balance_backward(grad.data_ptr(), l.data_ptr(), dtype_code(l.scalar_type()), row_stride(l), (int)l.size(0), (int)l.size(1), i.data_ptr(), (int)i.size(1), c.data_ptr(),
                                 s.data_ptr(), out.data_ptr(), raw_stream()),
            "balance_loss backward");
    return {once(out, "balance_loss")};
  }
};
int balance_with_grad(const at::Tensor& x, const at::Tensor& ids, at::Tensor& loss, at::Tensor& counts, at::Tensor& stats) {
  const auto node = node_of<BalanceBackward>(x);
  if (const int rc = run_balance(x, ids, loss, counts, stats)) return rc;
  node->tokens = x.size(0), node->e = x.size(1), node->k = ids.size(1), node->dtype = x.scalar_type();
  torch::autograd::set_history(loss, node);
  node->x = SavedVariable(x, false), node->ids = SavedVariable(ids, false), node->counts = SavedVariable(counts, false), node->stats = SavedVariable(stats, false);
  return 0;
}

PyObject* pair(int rc, const at::Tensor& a, const at::Tensor& b) {
  if (rc) return PyLong_FromLong(rc);
  PyObject *p = THPVariable_Wrap(a), *q = THPVariable_Wrap(b), *t = p && q ? PyTuple_New(2) : nullptr;
  if (!t) {
    Py_XDECREF(p), Py_XDECREF(q);
    return nullptr;
  }
  PyTuple_SET_ITEM(t, 0, p), PyTuple_SET_ITEM(t, 1, q);
  return t;
}
bool tensors(PyObject* const* args, Py_ssize_t n) {
  for (Py_ssize_t i = 0; i < n; ++i)
    if (!THPVariable_CheckExact(args[i])) return false;
  return ops.gate && plain_call();
}

// bind_ops(addresses of the library's functions in the order of Ops)
PyObject* py_bind_ops(PyObject*, PyObject* const* args, Py_ssize_t n) {
  constexpr Py_ssize_t count = sizeof(Ops) / sizeof(void*);
  void* at[count];
  if (n != count) {
    PyErr_SetString(PyExc_TypeError, "bind_ops takes the addresses of the operators");
    return nullptr;
  }
  for (Py_ssize_t i = 0; i < n; ++i) at[i] = PyLong_AsVoidPtr(args[i]);
  if (PyErr_Occurred()) return nullptr;
  memcpy(&ops, at, sizeof ops);
  Py_RETURN_NONE;
}

// top_k_gate(logits, k, renormalize)
PyObject* py_top_k_gate(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 3 || !tensors(args, 1) || !PyLong_CheckExact(args[1]) || !PyBool_Check(args[2])) Py_RETURN_NONE;
  const at::Tensor x = THPVariable_Unpack(args[0]);
  int over = 0;
  const long long k = PyLong_AsLongLongAndOverflow(args[1], &over);
  if (over || !plain_logits(x) || k < 1 || k > kMaxTopK || k > x.size(1)) Py_RETURN_NONE;
  const bool renormalize = args[2] == Py_True;
  at::Tensor weights, ids;
  int rc = 0;
  {
    Released released;
    if (x.requires_grad() && at::GradMode::is_enabled()) {
      check_capture(x, "top_k_gate");
      rc = gate_with_grad(x, k, renormalize, weights, ids);
    } else {
      rc = run_gate(x, k, renormalize, weights, ids);
    }
  }
  return pair(rc, weights, ids);
  END_HANDLE_TH_ERRORS
}

// check_capture(logits, name of the call), for calls that take the general path
PyObject* py_check_capture(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const char* what = n == 2 && THPVariable_Check(args[0]) && PyUnicode_Check(args[1]) ? PyUnicode_AsUTF8(args[1]) : nullptr;
  if (!what) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_TypeError, "check_capture takes a tensor and a name");
    return nullptr;
  }
  check_capture(THPVariable_Unpack(args[0]), what);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// balance_loss(logits, ids)
PyObject* py_balance_loss(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 2 || !tensors(args, 2)) Py_RETURN_NONE;
  const at::Tensor x = THPVariable_Unpack(args[0]), ids = THPVariable_Unpack(args[1]);
  if (!plain_logits(x) || !here(ids) || ids.dim() != 2 || ids.scalar_type() != at::kInt || !ids.is_contiguous() || ids.size(0) != x.size(0) || ids.size(1) < 1 || ids.size(1) > 32 ||
      ids.numel() > 0x7fffffff)
    Py_RETURN_NONE;
  at::Tensor loss, counts, stats;
  int rc = 0;
  {
    Released released;
    if (x.requires_grad() && at::GradMode::is_enabled()) {
      check_capture(x, "balance_loss");
      rc = balance_with_grad(x, ids, loss, counts, stats);
    } else {
      rc = run_balance(x, ids, loss, counts, stats);
    }
  }
  return pair(rc, loss, counts);
  END_HANDLE_TH_ERRORS
}

// quantize_fp8(x, src_row or None)
PyObject* py_quantize_fp8(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 2 || !tensors(args, args[1] == Py_None ? 1 : 2)) Py_RETURN_NONE;
  const at::Tensor x = THPVariable_Unpack(args[0]), src = args[1] == Py_None ? at::Tensor() : THPVariable_Unpack(args[1]);
  if (!here(x) || !no_gradient(x) || x.dim() != 2 || dtype_code(x.scalar_type()) < 0 || x.size(0) < 1 || x.size(1) < 1 || x.size(0) > kMaxSize || x.size(1) > kMaxSize || x.stride(1) != 1 ||
      (x.stride(0) < x.size(1) && x.size(0) > 1) || (src.defined() && (!vector_of(src, at::kInt) || src.size(0) > kMaxSize)))
    Py_RETURN_NONE;
  const int64_t k = x.size(1), rows = src.defined() ? src.size(0) : x.size(0), ld = (k + 15) & ~15ll;
  at::Tensor codes, scales;
  int rc;
  {
    Released released;
    codes = at::empty_strided({rows, k}, {ld, 1}, at::TensorOptions().dtype(at::kFloat8_e4m3fn).device(x.device())), scales = fresh({rows, (k + 127) / 128}, at::kFloat, x);
    const long long bytes = src.defined() ? ops.quantize_fp8_workspace_bytes((int)x.size(0), (int)rows, (int)k) : 0;
    const at::Tensor ws = bytes > 0 ? fresh({bytes / 4}, at::kInt, x) : at::Tensor();
    rc = ops.quantize_fp8(x.data_ptr(), dtype_code(x.scalar_type()), x.size(0) > 1 ? x.stride(0) : ld, (int)x.size(0), src.defined() ? src.data_ptr() : nullptr, (int)rows, (int)k,
                          codes.data_ptr(), ld, scales.data_ptr(), bytes > 0 ? ws.data_ptr() : nullptr, bytes, raw_stream());
  }
  return pair(rc, codes, scales);
  END_HANDLE_TH_ERRORS
}

// quantize_fp8_weight(w): a matrix or stacked ones
PyObject* py_quantize_fp8_weight(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 1 || !tensors(args, 1)) Py_RETURN_NONE;
  const at::Tensor w = THPVariable_Unpack(args[0]);
  if (!here(w) || !no_gradient(w) || (w.dim() != 2 && w.dim() != 3) || dtype_code(w.scalar_type()) < 0 || w.numel() < 1 || !w.is_contiguous() || w.size(-1) > kMaxSize || w.size(-2) > 65535 * 128 ||
      w.size(0) > kMaxSize)
    Py_RETURN_NONE;
  const int64_t e = w.dim() == 3 ? w.size(0) : 1, rows = w.size(-2), k = w.size(-1), ld = (k + 15) & ~15ll, nb = (rows + 127) / 128, kb = (k + 127) / 128;
  at::Tensor codes, scales;
  int rc;
  {
    Released released;
    const auto options = at::TensorOptions().dtype(at::kFloat8_e4m3fn).device(w.device());
    codes = w.dim() == 3 ? at::empty_strided({e, rows, k}, {rows * ld, ld, 1}, options) : at::empty_strided({rows, k}, {ld, 1}, options);
    scales = w.dim() == 3 ? fresh({e, nb, kb}, at::kFloat, w) : fresh({nb, kb}, at::kFloat, w);
    rc = ops.quantize_fp8_blocks(w.data_ptr(), dtype_code(w.scalar_type()), (int)e, (int)rows, (int)k, codes.data_ptr(), ld, scales.data_ptr(), raw_stream());
  }
  return pair(rc, codes, scales);
  END_HANDLE_TH_ERRORS
}

// bytes between rows of codes that the products take as they are, 0 for others
int64_t codes_stride(const at::Tensor& t) {
  if (!here(t) || !no_gradient(t) || t.scalar_type() != at::kFloat8_e4m3fn) return 0;
  const int64_t k = t.size(-1), ld = t.size(-2) > 1 ? t.stride(-2) : (k + 15) & ~15ll;
  return k >= 1 && k <= kMaxSize && (t.stride(-1) == 1 || k == 1) && ld >= k && ld % 16 == 0 && (uintptr_t)t.data_ptr() % 16 == 0 ? ld : 0;
}
bool scales_of(const at::Tensor& s, at::IntArrayRef size) { return here(s) && no_gradient(s) && s.scalar_type() == at::kFloat && s.sizes() == size && s.is_contiguous(); }

// matmul_fp8(a, a_scale, w, w_scale, dtype), matmul_fp8_experts(a, a_scale, w, w_scale, experts, offsets, dtype): a new output
PyObject* matmul(PyObject* const* args, bool experts) {
  HANDLE_TH_ERRORS
  const int count = experts ? 6 : 4;
  if (!tensors(args, count) || !THPDtype_Check(args[count])) Py_RETURN_NONE;
  const at::ScalarType type = reinterpret_cast<THPDtype*>(args[count])->scalar_type;
  const at::Tensor a = THPVariable_Unpack(args[0]), sa = THPVariable_Unpack(args[1]), w = THPVariable_Unpack(args[2]), sw = THPVariable_Unpack(args[3]);
  if (dtype_code(type) < 0 || a.dim() != 2 || w.dim() != (experts ? 3 : 2) || a.size(1) != w.size(-1)) Py_RETURN_NONE;
  const int64_t lda = codes_stride(a), ldw = codes_stride(w), m = a.size(0), n = w.size(-2), k = a.size(1), g = (k + 127) / 128;
  if (!lda || !ldw || m < 1 || n < 1 || m > kMaxSize || n > kMaxSize || !scales_of(sa, {m, g})) Py_RETURN_NONE;
  at::Tensor table, offsets;
  if (experts) {
    table = THPVariable_Unpack(args[4]), offsets = THPVariable_Unpack(args[5]);
    const int64_t e = w.size(0);
    if (e < 1 || e > kMaxSize || (e > 1 && w.stride(0) != n * ldw) || !scales_of(sw, {e, (n + 127) / 128, g}) || !vector_of(table, at::kInt) || !vector_of(offsets, at::kInt) ||
        table.size(0) < 1 || table.size(0) > 1024 || offsets.size(0) != table.size(0) + 1)
      Py_RETURN_NONE;
  } else if (!scales_of(sw, {(n + 127) / 128, g})) {
    Py_RETURN_NONE;
  }
  at::Tensor out;
  int rc;
  {
    Released released;
    out = fresh({m, n}, type, a);
    if (experts)
      rc = ops.matmul_fp8_experts(a.data_ptr(), lda, sa.data_ptr(), (int)m, w.data_ptr(), ldw, sw.data_ptr(), (int)w.size(0), table.data_ptr(), offsets.data_ptr(), (int)table.size(0),
                                  (int)n, (int)k, out.data_ptr(), dtype_code(type), n, 1, raw_stream());
    else
      rc = ops.matmul_fp8(a.data_ptr(), lda, sa.data_ptr(), w.data_ptr(), ldw, sw.data_ptr(), (int)m, (int)n, (int)k, out.data_ptr(), dtype_code(type), n, raw_stream());
  }
  return rc ? PyLong_FromLong(rc) : THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}
PyObject* py_matmul_fp8(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 5) Py_RETURN_NONE;
  return matmul(args, false);
}
PyObject* py_matmul_fp8_experts(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 7) Py_RETURN_NONE;
  return matmul(args, true);
}

PyMethodDef methods[] = {{"bind", (PyCFunction)(void (*)(void))py_bind, METH_FASTCALL, nullptr},
                         {"quantize_own_scale", (PyCFunction)(void (*)(void))py_quantize_own_scale, METH_FASTCALL, nullptr},
                         {"quantize_128x4", (PyCFunction)(void (*)(void))py_quantize_128x4, METH_FASTCALL, nullptr},
                         {"bind_ops", (PyCFunction)(void (*)(void))py_bind_ops, METH_FASTCALL, nullptr},
                         {"check_capture", (PyCFunction)(void (*)(void))py_check_capture, METH_FASTCALL, nullptr},
                         {"top_k_gate", (PyCFunction)(void (*)(void))py_top_k_gate, METH_FASTCALL, nullptr},
                         {"balance_loss", (PyCFunction)(void (*)(void))py_balance_loss, METH_FASTCALL, nullptr},
                         {"quantize_fp8", (PyCFunction)(void (*)(void))py_quantize_fp8, METH_FASTCALL, nullptr},
                         {"quantize_fp8_weight", (PyCFunction)(void (*)(void))py_quantize_fp8_weight, METH_FASTCALL, nullptr},
                         {"matmul_fp8", (PyCFunction)(void (*)(void))py_matmul_fp8, METH_FASTCALL, nullptr},
                         {"matmul_fp8_experts", (PyCFunction)(void (*)(void))py_matmul_fp8_experts, METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host(void) {   // (nothing of torch: the caller compares the version before anything else)
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "torch_version", B200_TORCH_VERSION)) Py_CLEAR(m);
  return m;
}
