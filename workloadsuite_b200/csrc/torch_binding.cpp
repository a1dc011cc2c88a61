// The short way from PyTorch tensors to the C ABI of ssd_b200.h.  A call of a few microseconds on the GPU (one decoded
// token, a small layer) is otherwise bound by what Python spends on attribute look-ups, ctypes marshalling and context
// managers: 15-20 us per call, against 2-3 us here.
// Every function returns None when the call is not plainly valid for the kernels (other dtypes, shapes that disagree,
// tensors that have to be copied first, a code that says so); the Python wrapper then goes its long way, which copies what
// has to be copied or raises.  Nothing is decided here that the long way would decide otherwise.  A CUDA error is raised
// here: work may have been enqueued by then, and a step made again would advance the state twice.
#include <Python.h>

#include <atomic>
#include <mutex>

#include <ATen/ATen.h>
#include <c10/core/InferenceMode.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>

#include "ssd_b200.h"

namespace {

using at::Tensor;

// The entry points stand between HANDLE_TH_ERRORS and END_HANDLE_TH_ERRORS from their first line on: what PyTorch's C++ throws
// (a nested tensor has no sizes, an allocation runs out of memory) becomes the Python exception that PyTorch itself raises
// for it, and would end the process if it left the entry point.

// entry points of the library that the Python side has loaded
decltype(&ssd_b200_forward) f_forward;
decltype(&ssd_b200_workspace_bytes) f_workspace;
decltype(&ssd_b200_step_strided) f_step;
decltype(&ssd_b200_conv1d_silu) f_conv;
decltype(&ssd_b200_dt_prologue) f_dt;
decltype(&ssd_b200_conv1d_silu_workspace_bytes) f_conv_workspace;
decltype(&ssd_b200_conv1d_silu_backward) f_conv_backward;
decltype(&ssd_b200_gated_scan_workspace_bytes) f_gated_workspace;
decltype(&ssd_b200_gated_scan) f_gated;
decltype(&ssd_b200_gated_scan_backward) f_gated_backward;
decltype(&ssd_b200_gated_step) f_gated_step;
decltype(&ssd_b200_norm_workspace_bytes) f_norm_workspace;
decltype(&ssd_b200_rms_norm) f_norm;
decltype(&ssd_b200_rms_norm_backward) f_norm_backward;
decltype(&ssd_b200_gated_rms_norm) f_gated_norm;
decltype(&ssd_b200_gated_rms_norm_backward) f_gated_norm_backward;
PyObject* f_raise;   // raises the Python exception of an error code

constexpr int kMaxDevices = 64;
Tensor* g_workspace[kMaxDevices];   // scratch of the runs that leave results for a later one (never shrinks)
std::atomic<Tensor*> g_status[kMaxDevices];   // the kernels' status word

int dtype_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return SSD_DTYPE_F32;
    case at::kHalf: return SSD_DTYPE_F16;
    case at::kBFloat16: return SSD_DTYPE_BF16;
    default: return -1;
  }
}

// The tensor behind a Python object: false for anything but a plain tensor; None gives an undefined tensor.
bool get(PyObject* o, const Tensor** out, bool optional = false) {
  static const Tensor none;
  if (o == Py_None) {
    *out = &none;
    return optional;
  }
  if (!THPVariable_CheckExact(o)) return false;
  *out = &THPVariable_Unpack(o);
  return true;
}

bool shaped(const Tensor& t, std::initializer_list<int64_t> s) { return t.sizes() == at::IntArrayRef(s.begin(), s.size()); }
bool inner(const Tensor& t) { return t.stride(-1) == 1 || t.size(-1) == 1; }

// The result of a call that returned `rc`: None, for the long way, unless that could enqueue work twice.
PyObject* declined(int rc) {
  if (rc != SSD_ERR_CUDA) Py_RETURN_NONE;
  Py_XDECREF(PyObject_CallFunction(f_raise, "i", rc));
  return nullptr;
}

struct Where {
  c10::cuda::OptionalCUDAGuard guard;
  c10::Device dev;
  explicit Where(const Tensor& t) : dev(t.device()) { if (c10::cuda::current_device() != dev.index()) guard.set_device(dev); }
  bool here(const Tensor& t) const { return !t.defined() || t.device() == dev; }
  void* stream() const { return c10::cuda::getCurrentCUDAStream(dev.index()).stream(); }
};

// Made once, by whichever thread asks first: autograd's threads do too, which do not hold the interpreter.  Zeroed before anybody has it, on a
// stream of its own, in memory of no pool, so that a capture that is under way records none of it and no replay clears it.
Tensor& status_word(int dev) {
  if (Tensor* t = g_status[dev].load(std::memory_order_acquire)) return *t;
  static std::mutex making;
  const std::lock_guard<std::mutex> lock(making);
  if (Tensor* t = g_status[dev].load(std::memory_order_acquire)) return *t;
  constexpr int kWords = 1024;
  const c10::cuda::CUDAGuard guard((c10::DeviceIndex)dev);
  const c10::cuda::CUDAStreamCaptureModeGuard relaxed(cudaStreamCaptureModeRelaxed);
  const c10::InferenceMode plain(false);   // (it is cleared outside of such a mode)
  void* at = nullptr;
  cudaStream_t stream = nullptr;
  C10_CUDA_CHECK(cudaMalloc(&at, kWords * sizeof(int32_t)));
  C10_CUDA_CHECK(cudaStreamCreateWithFlags(&stream, cudaStreamNonBlocking));
  C10_CUDA_CHECK(cudaMemsetAsync(at, 0, kWords * sizeof(int32_t), stream));
  C10_CUDA_CHECK(cudaStreamSynchronize(stream));
  C10_CUDA_CHECK(cudaStreamDestroy(stream));
  const c10::Device device(c10::kCUDA, (c10::DeviceIndex)dev);
  Tensor* t = new Tensor(at::for_blob(at, {kWords}).options(at::TensorOptions().dtype(at::kInt).device(device)).target_device(device).make_tensor());
  g_status[dev].store(t, std::memory_order_release);
  return *t;
}
Tensor& workspace(int dev, int64_t bytes) {
  if (!g_workspace[dev] || g_workspace[dev]->numel() < bytes) {
    delete g_workspace[dev];
    g_workspace[dev] = nullptr;
    g_workspace[dev] = new Tensor(at::empty({bytes}, at::TensorOptions().dtype(at::kByte).device(at::kCUDA, dev)));
  }
  return *g_workspace[dev];
}

// Strides of the three outer axes; a size-1 axis gets its contiguous stride (its own is arbitrary and may break the
// 16-byte rule of TMA descriptors).
void strides4(const Tensor& t, int64_t* st) {
  int64_t in = t.size(3);
  for (int d = 2; d >= 0; --d) {
    st[d] = t.size(d) == 1 ? in : t.stride(d);
    in = std::max(in, st[d] * t.size(d));
  }
}
void strides3(const Tensor& t, int64_t* st) {
  for (int d = 0; d < 3; ++d) st[d] = t.stride(d);
}

// step(x, a, B, C, state, dt, D, z, out) -> y
PyObject* py_step(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const Tensor *x, *a, *B, *C, *state, *dt, *D, *z, *out;
  if (n != 9 || !get(o[0], &x) || !get(o[1], &a) || !get(o[2], &B) || !get(o[3], &C) || !get(o[4], &state) ||
      !get(o[5], &dt, true) || !get(o[6], &D, true) || !get(o[7], &z, true) || !get(o[8], &out, true) || !x->is_cuda() ||
      x->dim() != 3 || B->dim() != 3 || state->dim() != 4)
    Py_RETURN_NONE;
  const int dtype = dtype_of(*x);
  const int64_t b = x->size(0), h = x->size(1), p = x->size(2), g = B->size(1), ns = B->size(2);
  const auto st = x->scalar_type();
  if (dtype < 0 || g <= 0 || h % g != 0 || !inner(*x) || !inner(*B)) Py_RETURN_NONE;
  if (a->scalar_type() != at::kFloat || !shaped(*a, {b, h}) || B->scalar_type() != st || !shaped(*B, {b, g, ns}) ||
      C->scalar_type() != st || !shaped(*C, {b, g, ns}) || !inner(*C) || state->scalar_type() != at::kFloat ||
      !shaped(*state, {b, h, ns, p}) || !state->is_contiguous())
    Py_RETURN_NONE;
  if (dt->defined() && (dt->scalar_type() != st || !shaped(*dt, {b, h}))) Py_RETURN_NONE;
  if (z->defined() && (z->scalar_type() != st || !shaped(*z, {b, h, p}) || !inner(*z))) Py_RETURN_NONE;
  if (D->defined() && (!shaped(*D, {h}) || !D->is_contiguous() || (D->scalar_type() != st && D->scalar_type() != at::kFloat)))
    Py_RETURN_NONE;
  if (out->defined() && (out->scalar_type() != st || !shaped(*out, {b, h, p}) || !out->is_contiguous())) Py_RETURN_NONE;
  Where w(*x);
  if (!w.here(*a) || !w.here(*B) || !w.here(*C) || !w.here(*state) || !w.here(*dt) || !w.here(*D) || !w.here(*z) || !w.here(*out))
    Py_RETURN_NONE;
  Tensor y = out->defined() ? *out : at::empty({b, h, p}, x->options());
  SsdStepArgs s = {};
  s.x = x->data_ptr(); s.a = static_cast<const float*>(a->data_ptr()); s.B = B->data_ptr(); s.C = C->data_ptr();
  s.state = static_cast<float*>(state->data_ptr()); s.y = y.data_ptr();
  s.batch = (int)b; s.nheads = (int)h; s.headdim = (int)p; s.dstate = (int)ns; s.ngroups = (int)g; s.dtype = dtype;
  for (int d = 0; d < 2; ++d) {
    s.x_stride[d] = x->stride(d); s.a_stride[d] = a->stride(d); s.b_stride[d] = B->stride(d); s.c_stride[d] = C->stride(d);
  }
  if (dt->defined()) { s.dt = dt->data_ptr(); s.dt_stride[0] = dt->stride(0); s.dt_stride[1] = dt->stride(1); }
  if (z->defined()) { s.z = z->data_ptr(); s.z_stride[0] = z->stride(0); s.z_stride[1] = z->stride(1); }
  if (D->defined()) { s.D = D->data_ptr(); s.d_in_dtype = D->scalar_type() == st && st != at::kFloat; }
  if (const int rc = f_step(&s, w.stream())) return declined(rc);
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// dt_prologue(dt_raw, dt_bias, A_log) -> (dt, A_dt)
PyObject* py_dt(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const Tensor *r, *bias, *al;
  if (n != 3 || !get(o[0], &r) || !get(o[1], &bias, true) || !get(o[2], &al) || !r->is_cuda() || r->dim() != 3) Py_RETURN_NONE;
  const int dtype = dtype_of(*r);
  const int64_t b = r->size(0), l = r->size(1), h = r->size(2);
  if (dtype < 0 || r->stride(2) != 1 || al->scalar_type() != at::kFloat || !shaped(*al, {h}) || !al->is_contiguous()) Py_RETURN_NONE;
  if (bias->defined() && (!shaped(*bias, {h}) || bias->scalar_type() != r->scalar_type() || !bias->is_contiguous())) Py_RETURN_NONE;
  Where w(*r);
  if (!w.here(*bias) || !w.here(*al)) Py_RETURN_NONE;
  Tensor dt = at::empty({b, l, h}, r->options());
  Tensor A = at::empty({b, l, h}, r->options().dtype(at::kFloat));
  if (const int rc = f_dt(r->data_ptr(), r->stride(0), r->stride(1), bias->defined() ? bias->data_ptr() : nullptr,
                          static_cast<const float*>(al->data_ptr()), dt.data_ptr(), static_cast<float*>(A.data_ptr()), (int)b,
                          (int)l, (int)h, dtype, w.stream()))
    return declined(rc);
  PyObject* t = PyTuple_New(2);
  if (!t) return nullptr;
  PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(std::move(dt)));
  PyTuple_SET_ITEM(t, 1, THPVariable_Wrap(std::move(A)));
  return t;
  END_HANDLE_TH_ERRORS
}

// forward(X, A, B, C, chunk, dt, initial_states, D, z, out, return_final_state) -> Y or (Y, final_state)
PyObject* py_forward(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const Tensor *X, *A, *B, *C, *dt, *init, *D, *z, *out;
  if (n != 11 || !get(o[0], &X) || !get(o[1], &A) || !get(o[2], &B) || !get(o[3], &C) || !PyLong_CheckExact(o[4]) ||
      !get(o[5], &dt, true) || !get(o[6], &init, true) || !get(o[7], &D, true) || !get(o[8], &z, true) ||
      !get(o[9], &out, true) || !X->is_cuda() || X->dim() != 4 || A->dim() != 3 || B->dim() != 4)
    Py_RETURN_NONE;
  int over = 0;
  const long long chunk = PyLong_AsLongLongAndOverflow(o[4], &over);
  const bool want_final = o[10] == Py_True;
  const int dtype = dtype_of(*X);
  const auto st = X->scalar_type();
  const int64_t b = X->size(0), s = X->size(1), h = X->size(2), p = X->size(3), g = B->size(2), ns = B->size(3);
  if (dtype < 0 || over || chunk <= 0 || chunk > 0x7fffffff || g <= 0 || h % g != 0 || !inner(*X) || !inner(*B) ||
      A->scalar_type() != at::kFloat || !shaped(*A, {b, s, h}) || B->scalar_type() != st || !shaped(*B, {b, s, g, ns}) ||
      C->scalar_type() != st || C->sizes() != B->sizes() || !inner(*C))
    Py_RETURN_NONE;
  if (dt->defined() && (dt->scalar_type() != st || !shaped(*dt, {b, s, h}))) Py_RETURN_NONE;
  if (init->defined() && (init->scalar_type() != at::kFloat || !shaped(*init, {b, h, ns, p}) || !init->is_contiguous())) Py_RETURN_NONE;
  if (D->defined() && (!shaped(*D, {h}) || !D->is_contiguous() || (D->scalar_type() != st && D->scalar_type() != at::kFloat)))
    Py_RETURN_NONE;
  if (z->defined() && (z->scalar_type() != st || z->sizes() != X->sizes() || !inner(*z))) Py_RETURN_NONE;
  if (out->defined() && (out->scalar_type() != st || out->sizes() != X->sizes() || !inner(*out))) Py_RETURN_NONE;
  Where w(*X);
  if (!w.here(*A) || !w.here(*B) || !w.here(*C) || !w.here(*dt) || !w.here(*init) || !w.here(*D) || !w.here(*z) || !w.here(*out))
    Py_RETURN_NONE;
  Tensor Y = out->defined() ? *out : at::empty({b, s, h, p}, X->options());
  Tensor fin;
  if (want_final) fin = at::empty({b, h, ns, p}, X->options().dtype(at::kFloat));
  SsdArgs a = {};
  a.X = X->data_ptr(); a.A = static_cast<const float*>(A->data_ptr()); a.B = B->data_ptr(); a.C = C->data_ptr(); a.Y = Y.data_ptr();
  if (dt->defined()) { a.dt = dt->data_ptr(); strides3(*dt, a.dt_stride); }
  if (init->defined()) a.initial_state = static_cast<const float*>(init->data_ptr());
  if (want_final) a.final_state = static_cast<float*>(fin.data_ptr());
  if (D->defined()) {
    a.D = static_cast<const float*>(D->data_ptr());
    if (D->scalar_type() != at::kFloat) a.flags |= SSD_FLAG_D_IN_DTYPE;
  }
  if (z->defined()) { a.Z = z->data_ptr(); strides4(*z, a.z_stride); }
  a.status = static_cast<int32_t*>(status_word(w.dev.index()).data_ptr());
  a.batch = (int)b; a.seqlen = (int)s; a.nheads = (int)h; a.headdim = (int)p; a.dstate = (int)ns; a.ngroups = (int)g;
  a.chunk = (int)chunk; a.dtype = dtype;
  strides4(*X, a.x_stride); strides3(*A, a.a_stride); strides4(*B, a.b_stride); strides4(*C, a.c_stride); strides4(Y, a.y_stride);
  const size_t need = f_workspace(&a);
  Tensor ws;   // from the current stream's memory: calls on other streams have their own
  if (need) {
    ws = at::empty({(int64_t)need}, X->options().dtype(at::kByte));
    a.workspace = ws.data_ptr();
    a.workspace_bytes = need;
  }
  if (const int rc = f_forward(&a, w.stream())) return declined(rc);
  if (!want_final) return THPVariable_Wrap(std::move(Y));
  PyObject* t = PyTuple_New(2);
  if (!t) return nullptr;
  PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(std::move(Y)));
  PyTuple_SET_ITEM(t, 1, THPVariable_Wrap(std::move(fin)));
  return t;
  END_HANDLE_TH_ERRORS
}

// ---- a recurrent block's other pieces: gradients and norms ----

// A tuple of tensors; undefined ones are None.
PyObject* tuple_of(std::initializer_list<Tensor> ts) {
  PyObject* t = PyTuple_New((Py_ssize_t)ts.size());
  if (!t) return nullptr;
  Py_ssize_t i = 0;
  for (const Tensor& v : ts) PyTuple_SET_ITEM(t, i++, v.defined() ? THPVariable_Wrap(v) : (Py_INCREF(Py_None), Py_None));
  return t;
}
Tensor scratch(const Tensor& like, size_t bytes) {   // from the current stream's memory
  return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : Tensor();
}
template <typename T = void>
T* ptr(const Tensor& t) { return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr; }
bool real(PyObject* o, float* v) {
  if (!PyFloat_CheckExact(o)) return false;
  *v = (float)PyFloat_AS_DOUBLE(o);
  return true;
}
bool fits(int64_t n) { return n > 0 && n <= 0x7fffffff; }
bool whole(PyObject* o, int* v) {   // a number of 32 bits
  if (!PyLong_CheckExact(o)) return false;
  int over = 0;
  const long n = PyLong_AsLongAndOverflow(o, &over);
  *v = (int)n;
  return over == 0 && n == (long)*v;
}
// fp32, whole and contiguous, or not given
bool plain32(const Tensor& t, std::initializer_list<int64_t> s) {
  return !t.defined() || (t.scalar_type() == at::kFloat && shaped(t, s) && t.is_contiguous());
}
bool like3(const Tensor& t, const Tensor& x) { return t.scalar_type() == x.scalar_type() && t.sizes() == x.sizes() && inner(t); }
void two(const Tensor& t, int64_t* st) {
  if (!t.defined()) return;
  st[0] = t.stride(0);
  st[1] = t.stride(1);
}

// The operators below are recorded for autograd here too: a node in Python costs a training step of a small layer more than its kernels.
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using Maybe = std::optional<Tensor>;

bool records(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}
// Forward-mode gradients and function transforms have no kernels: what carries one goes the long way, which says so.
bool tangents(std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    if (t->defined() && (t->_fw_grad(0).defined() || t->key_set().has(c10::DispatchKey::FuncTorchBatched) ||
                         t->key_set().has(c10::DispatchKey::FuncTorchGradWrapper)))
      return true;
  return false;
}
// A tensor that a kernel has written over: a backward pass that saved it is to notice.
void written(const Tensor& t) {
  if (t.defined() && !t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
Maybe maybe(const Tensor& t) { return t.defined() ? Maybe(t) : std::nullopt; }
Tensor given(const Maybe& t) { return t ? *t : Tensor(); }
// A gradient whose innermost axis is not contiguous (a sum's is expanded) is copied once.
Tensor usable(const Tensor& t) { return !t.defined() || inner(t) ? t : t.contiguous(); }
// Outside of entry points that hold the interpreter: what a refused or failed call raises.
void must(bool fits, int rc, const char* what) {
  TORCH_CHECK_NOT_IMPLEMENTED(fits, what, ": sizes or strides outside what the kernels cover");
  TORCH_CHECK(rc == 0, what, ": the library returned code ", rc);
}
// Gradients are not differentiable themselves: to differentiate them is an error, as with once_differentiable in Python.
variable_list once(variable_list grads, const char* what) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list there;
  for (Tensor& g : grads)
    if (g.defined()) there.push_back(g.detach().requires_grad_(true));
  auto error = std::make_shared<torch::autograd::DelayedError>(std::string(what) + " is not twice differentiable", (int)there.size());
  there = (*error)(std::move(there));
  size_t n = 0;
  for (Tensor& g : grads)
    if (g.defined()) g = there[n++];
  return grads;
}

// ---- gated scan ----

// What the forward and the backward both check and fill in.
bool gated_args(const Tensor& x, const Tensor& i, const Tensor& r, const Tensor& decay, const Tensor& init, const Tensor& reset, float rate,
                const Where& w, SsdGatedScanArgs* a) {
  const int64_t b = x.size(0), s = x.size(1), d = x.size(2);
  if (!fits(b) || !fits(s) || !fits(d) || !inner(x) || !like3(i, x) || !like3(r, x) || decay.scalar_type() != at::kFloat ||
      !shaped(decay, {d}) || !decay.is_contiguous() || !plain32(init, {b, d}) ||
      (reset.defined() && (reset.scalar_type() != at::kBool || !shaped(reset, {b, s}))) || !w.here(i) || !w.here(r) || !w.here(decay) ||
      !w.here(init) || !w.here(reset))
    return false;
  a->x = x.data_ptr(); a->input_gate = i.data_ptr(); a->decay_gate = r.data_ptr();
  a->decay = ptr<float>(decay);
  a->initial_state = ptr<float>(init);
  a->reset = ptr<uint8_t>(reset);
  a->status = ptr<int32_t>(status_word(w.dev.index()));
  a->rate = rate;
  a->batch = (int)b; a->seqlen = (int)s; a->channels = (int)d; a->dtype = dtype_of(x);
  two(x, a->x_stride); two(i, a->input_gate_stride); two(r, a->decay_gate_stride); two(reset, a->reset_stride);
  return true;
}

struct Gated {
  Tensor y, fin, pieces;
};
bool gated_forward(const Tensor& x, const Tensor& i, const Tensor& r, const Tensor& decay, const Tensor& init, const Tensor& reset,
                   const Tensor& out, float rate, int wait_ms, bool keep, Gated* g, int* rc) {
  Where w(x);
  SsdGatedScanArgs a = {};
  if (!gated_args(x, i, r, decay, init, reset, rate, w, &a)) return false;
  if (out.defined() && (out.dim() != 3 || !like3(out, x) || !w.here(out))) return false;
  a.wait_limit_ms = wait_ms;
  const auto f32 = x.options().dtype(at::kFloat);
  g->y = out.defined() ? out : at::empty(x.sizes(), x.options());
  g->fin = at::empty({x.size(0), x.size(2)}, f32);
  if (keep) g->pieces = at::empty({x.size(0), (x.size(1) + 63) / 64, x.size(2)}, f32);
  a.y = g->y.data_ptr(); a.final_state = ptr<float>(g->fin); a.pieces = ptr<float>(g->pieces);
  two(g->y, a.y_stride);
  const size_t need = f_gated_workspace(&a, 0);
  const Tensor ws = scratch(x, need);
  a.workspace = ptr(ws);
  a.workspace_bytes = need;
  *rc = f_gated(&a, w.stream());
  written(out);
  return true;
}
bool gated_backward(const Tensor& x, const Tensor& i, const Tensor& r, const Tensor& decay, const Tensor& reset, const Tensor& pieces,
                    const Tensor& dy, const Tensor& dfin, float rate, bool want_dinit, variable_list* out, int* rc) {
  Where w(x);
  SsdGatedScanArgs a = {};
  if (!gated_args(x, i, r, decay, Tensor(), reset, rate, w, &a)) return false;
  const int64_t b = x.size(0), s = x.size(1), d = x.size(2);
  if (!like3(dy, x) || !w.here(dy) || !plain32(dfin, {b, d}) || !w.here(dfin) || !plain32(pieces, {b, (s + 63) / 64, d}) || !w.here(pieces))
    return false;
  const auto f32 = x.options().dtype(at::kFloat);
  Tensor dx = at::empty(x.sizes(), x.options()), di = at::empty(x.sizes(), x.options()), dr = at::empty(x.sizes(), x.options());
  Tensor dd = at::empty({d}, f32), dh;
  if (want_dinit) dh = at::empty({b, d}, f32);
  a.pieces = ptr<float>(pieces); a.dy = dy.data_ptr(); a.dfinal_state = ptr<float>(dfin);
  a.dx = dx.data_ptr(); a.dinput_gate = di.data_ptr(); a.ddecay_gate = dr.data_ptr(); a.ddecay = ptr<float>(dd); a.dinitial_state = ptr<float>(dh);
  two(dy, a.dy_stride); two(dx, a.dx_stride); two(di, a.dinput_gate_stride); two(dr, a.ddecay_gate_stride);
  const size_t need = f_gated_workspace(&a, 1);
  const Tensor ws = scratch(x, need);
  a.workspace = ptr(ws);
  a.workspace_bytes = need;
  *rc = f_gated_backward(&a, w.stream());
  *out = {dx, di, dr, dd, dh};
  return true;
}

struct GatedNode : torch::autograd::Function<GatedNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& i, const Tensor& r, const Tensor& decay, const Maybe& init,
                               const Maybe& reset, double rate, int64_t wait_ms, int* rc) {
    Gated g;
    *rc = 1;   // (declined)
    if (!gated_forward(x, i, r, decay, given(init), given(reset), Tensor(), (float)rate, (int)wait_ms, true, &g, rc) || *rc) return {};
    ctx->save_for_backward({x, i, r, decay, given(reset), g.pieces});
    ctx->saved_data["rate"] = rate;
    ctx->saved_data["state"] = init.has_value();
    ctx->set_materialize_grads(false);
    return {g.y, g.fin};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined() && !grads[1].defined()) return variable_list(9);
    const auto saved = ctx->get_saved_variables();
    const Tensor& x = saved[0];
    const Tensor dy = grads[0].defined() ? usable(grads[0]) : at::zeros(x.sizes(), x.options());
    const Tensor dfin = grads[1].defined() ? grads[1].contiguous() : Tensor();
    variable_list out;
    int rc = 0;
    const bool ok = gated_backward(x, saved[1], saved[2], saved[3], saved[4], saved[5], dy, dfin, (float)ctx->saved_data["rate"].toDouble(),
                                   ctx->saved_data["state"].toBool(), &out, &rc);
    must(ok, rc, "gated_scan");
    out.resize(9);
    return once(std::move(out), "gated_scan");
  }
};

// gated_scan(x, input_gate, decay_gate, decay, initial_state, reset, out, rate, wait_limit_ms) -> (y, final_state)
PyObject* py_gated(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const Tensor *x, *i, *r, *decay, *init, *reset, *out;
  float rate;
  int wait_ms;
  if (n != 9 || !get(o[0], &x) || !get(o[1], &i) || !get(o[2], &r) || !get(o[3], &decay) || !get(o[4], &init, true) ||
      !get(o[5], &reset, true) || !get(o[6], &out, true) || !real(o[7], &rate) || !whole(o[8], &wait_ms) || !x->is_cuda() ||
      x->dim() != 3 || i->dim() != 3 || r->dim() != 3 || dtype_of(*x) < 0)
    Py_RETURN_NONE;
  if (tangents({x, i, r, decay, init})) Py_RETURN_NONE;
  int rc = 0;
  if (records({x, i, r, decay, init})) {
    if (out->defined()) Py_RETURN_NONE;
    const variable_list v = GatedNode::apply(*x, *i, *r, *decay, maybe(*init), maybe(*reset), (double)rate, (int64_t)wait_ms, &rc);
    return rc ? declined(rc) : tuple_of({v[0], v[1]});
  }
  Gated g;
  if (!gated_forward(*x, *i, *r, *decay, *init, *reset, *out, rate, wait_ms, false, &g, &rc)) Py_RETURN_NONE;
  return rc ? declined(rc) : tuple_of({g.y, g.fin});
  END_HANDLE_TH_ERRORS
}

// gated_step(x, input_gate, decay_gate, decay, state, out_state, out, rate) -> y
PyObject* py_gated_step(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const Tensor *x, *i, *r, *decay, *state, *state_out, *out;
  float rate;
  if (n != 8 || !get(o[0], &x) || !get(o[1], &i) || !get(o[2], &r) || !get(o[3], &decay) || !get(o[4], &state) ||
      !get(o[5], &state_out, true) || !get(o[6], &out, true) || !real(o[7], &rate) || !x->is_cuda() || x->dim() != 2 || i->dim() != 2 ||
      r->dim() != 2 || dtype_of(*x) < 0)
    Py_RETURN_NONE;
  const int64_t b = x->size(0), d = x->size(1);
  auto like = [&](const Tensor& t) { return t.scalar_type() == x->scalar_type() && t.sizes() == x->sizes() && inner(t); };
  if (!fits(b) || !fits(d) || !like(*x) || !like(*i) || !like(*r) || decay->scalar_type() != at::kFloat || !shaped(*decay, {d}) ||
      !decay->is_contiguous() || !plain32(*state, {b, d}) || !plain32(*state_out, {b, d}) || (out->defined() && (out->dim() != 2 || !like(*out))))
    Py_RETURN_NONE;
  Where w(*x);
  if (!w.here(*i) || !w.here(*r) || !w.here(*decay) || !w.here(*state) || !w.here(*state_out) || !w.here(*out)) Py_RETURN_NONE;
  Tensor y = out->defined() ? *out : at::empty({b, d}, x->options());
  SsdGatedStepArgs a = {};
  a.x = x->data_ptr(); a.input_gate = i->data_ptr(); a.decay_gate = r->data_ptr(); a.decay = ptr<float>(*decay);
  a.state = ptr<float>(*state);
  a.state_out = state_out->defined() ? ptr<float>(*state_out) : ptr<float>(*state);
  a.y = y.data_ptr();
  a.rate = rate;
  a.batch = (int)b; a.channels = (int)d; a.dtype = dtype_of(*x);
  a.x_stride = x->stride(0); a.input_gate_stride = i->stride(0); a.decay_gate_stride = r->stride(0); a.y_stride = y.stride(0);
  if (const int rc = f_gated_step(&a, w.stream())) return declined(rc);
  written(state_out->defined() ? *state_out : *state);
  written(*out);
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// ---- norms ----

// Rows of [..., d] that lie one stride apart.
bool rows_of(const Tensor& t, int64_t* rows, int64_t* stride) {
  if (t.dim() < 1 || !inner(t)) return false;
  int64_t n = 1, st = t.size(-1);
  for (int64_t k = t.dim() - 2; k >= 0; --k) {
    if (t.size(k) == 1) continue;
    if (n == 1) st = t.stride(k);
    else if (t.stride(k) != st * n) return false;
    n *= t.size(k);
  }
  *rows = n;
  *stride = st;
  return true;
}
Tensor usable_rows(const Tensor& t) {
  int64_t n, st;
  return !t.defined() || rows_of(t, &n, &st) ? t : t.contiguous();
}
// The operands of a norm: checked against x, with their strides.
struct NormCall {
  const Tensor& x;
  Where w;
  SsdNormArgs a = {};
  bool ok = true;
  explicit NormCall(const Tensor& t) : x(t), w(t) {
    a.d = (int)t.size(-1);
    a.dtype = dtype_of(t);
    a.residual_dtype = a.dtype;
    a.groups = 1;
    ok = fits(t.size(-1)) && rows_of(t, &a.rows, &a.x_stride) && a.rows > 0;
    a.x = t.data_ptr();
  }
  void* rows(const Tensor& t, at::ScalarType type, int64_t* stride) {
    if (!t.defined()) return nullptr;
    int64_t n = 0;
    ok = ok && t.scalar_type() == type && t.sizes() == x.sizes() && w.here(t) && rows_of(t, &n, stride);
    return t.data_ptr();
  }
  void* vector(const Tensor& t, int bit) {
    if (!t.defined()) return nullptr;
    ok = ok && shaped(t, {(int64_t)a.d}) && t.is_contiguous() && w.here(t) && (t.scalar_type() == at::kFloat || t.scalar_type() == x.scalar_type());
    if (t.scalar_type() == x.scalar_type()) a.vectors_in_dtype |= bit;
    return t.data_ptr();
  }
  Tensor fresh(void** at, int64_t* stride) {   // a result like x
    Tensor t = at::empty(x.sizes(), x.options());
    *at = t.data_ptr();
    *stride = a.d;
    return t;
  }
  Tensor scratch_of() {
    a.workspace_bytes = f_norm_workspace(&a);
    Tensor ws = scratch(x, a.workspace_bytes);
    a.workspace = ptr(ws);
    return ws;
  }
};
bool norm_operand(const Tensor& x) { return x.is_cuda() && x.dim() >= 1 && dtype_of(x) >= 0; }

struct Normed {
  Tensor y, r, inv, invp;
};
bool norm_forward(const Tensor& x, const Tensor& wt, const Tensor& res, const Tensor& post, const Tensor& scale, const Tensor& out, float eps,
                  bool keep, Normed* v, int* rc) {
  NormCall c(x);
  c.a.weight = c.vector(wt, 1);
  c.a.post_weight = c.vector(post, 2);
  c.a.scale = c.vector(scale, 4);
  if (res.defined()) {
    if (dtype_of(res) < 0) return false;
    c.a.residual_dtype = dtype_of(res);
    c.a.residual = c.rows(res, res.scalar_type(), &c.a.residual_stride);
  }
  c.a.y = c.rows(out, x.scalar_type(), &c.a.y_stride);
  if (!c.ok) return false;
  v->y = out.defined() ? out : c.fresh(&c.a.y, &c.a.y_stride);
  if (res.defined()) {
    v->r = at::empty(x.sizes(), res.options());
    c.a.residual_out = v->r.data_ptr();
    c.a.residual_out_stride = c.a.d;
  }
  const auto f32 = x.options().dtype(at::kFloat);
  if (keep) v->inv = at::empty({c.a.rows}, f32);
  if (keep && post.defined()) v->invp = at::empty({c.a.rows}, f32);
  c.a.inv_rms = ptr<float>(v->inv);
  c.a.inv_rms_post = ptr<float>(v->invp);
  c.a.eps = eps;
  *rc = f_norm(&c.a, c.w.stream());
  written(out);
  return true;
}
// like: x, or where nothing of it is read a tensor of its shape and type
bool norm_backward(const Tensor& like, const Tensor& wt, const Tensor& r, const Tensor& post, const Tensor& scale, const Tensor& inv,
                   const Tensor& invp, const Tensor& dy, const Tensor& dr, variable_list* out, int* rc) {
  NormCall c(like);
  c.a.weight = c.vector(wt, 1);
  c.a.post_weight = c.vector(post, 2);
  c.a.scale = c.vector(scale, 4);
  if (r.defined()) {
    c.a.residual_dtype = dtype_of(r);
    c.a.residual_out = c.rows(r, r.scalar_type(), &c.a.residual_out_stride);
    c.a.dresidual_out = c.rows(dr, r.scalar_type(), &c.a.dresidual_out_stride);
  }
  c.a.dy = c.rows(dy, like.scalar_type(), &c.a.dy_stride);
  c.a.inv_rms = ptr<float>(inv);
  c.a.inv_rms_post = ptr<float>(invp);
  if (!c.ok) return false;
  Tensor dx = c.fresh(&c.a.dx, &c.a.dx_stride), dres, dw = at::empty({(int64_t)c.a.d}, wt.options()), dpost, dscale;
  if (r.defined()) {
    // without a norm or a scale behind the block its gradient is the residual's; of one type they are one tensor
    if (!post.defined() && !scale.defined() && r.scalar_type() == like.scalar_type()) {
      dres = dx;
    } else {
      dres = at::empty(like.sizes(), r.options());
      c.a.dresidual = dres.data_ptr();
      c.a.dresidual_stride = c.a.d;
    }
  }
  if (post.defined()) dpost = at::empty({(int64_t)c.a.d}, post.options());
  if (scale.defined()) dscale = at::empty({(int64_t)c.a.d}, scale.options());
  c.a.dweight = dw.data_ptr(); c.a.dpost_weight = ptr(dpost); c.a.dscale = ptr(dscale);
  const Tensor ws = c.scratch_of();
  *rc = f_norm_backward(&c.a, c.w.stream());
  *out = {dx, dw, dres, dpost, dscale};
  return true;
}

struct NormNode : torch::autograd::Function<NormNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& wt, const Maybe& res, const Maybe& post, const Maybe& scale,
                               double eps, int* rc) {
    Normed v;
    *rc = 1;
    if (!norm_forward(x, wt, given(res), given(post), given(scale), Tensor(), (float)eps, true, &v, rc) || *rc) return {};
    // the block's output itself is needed again only behind a norm or a scale, or where it is what is normalised
    ctx->save_for_backward({post || scale || !res ? x : Tensor(), wt, v.r, given(post), given(scale), v.inv, v.invp});
    ctx->saved_data["type"] = (int64_t)x.scalar_type();
    ctx->set_materialize_grads(false);
    if (v.r.defined()) return {v.y, v.r};
    return {v.y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const Tensor gr = grads.size() > 1 ? grads[1] : Tensor();
    if (!grads[0].defined() && !gr.defined()) return variable_list(7);
    const auto s = ctx->get_saved_variables();
    const Tensor& of = s[0].defined() ? s[0] : s[2];
    const auto type = (at::ScalarType)ctx->saved_data["type"].toInt();
    const Tensor dy = grads[0].defined() ? usable_rows(grads[0]) : at::zeros(of.sizes(), of.options().dtype(type));
    variable_list out;
    int rc = 0;
    const bool ok = norm_backward(s[0].defined() ? s[0] : dy, s[1], s[2], s[3], s[4], s[5], s[6], dy, usable_rows(gr), &out, &rc);
    must(ok, rc, "rms_norm");
    out.resize(7);
    return once(std::move(out), "rms_norm");
  }
};

// rms_norm(x, weight, residual, post_weight, scale, out, eps) -> (y, residual_out or None)
PyObject* py_norm(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const Tensor *x, *wt, *res, *post, *scale, *out;
  float eps;
  if (n != 7 || !get(o[0], &x) || !get(o[1], &wt) || !get(o[2], &res, true) || !get(o[3], &post, true) || !get(o[4], &scale, true) ||
      !get(o[5], &out, true) || !real(o[6], &eps) || !norm_operand(*x) || tangents({x, wt, res, post, scale}))
    Py_RETURN_NONE;
  int rc = 0;
  if (records({x, wt, res, post, scale})) {
    if (out->defined()) Py_RETURN_NONE;
    const variable_list v = NormNode::apply(*x, *wt, maybe(*res), maybe(*post), maybe(*scale), (double)eps, &rc);
    return rc ? declined(rc) : tuple_of({v[0], v.size() > 1 ? v[1] : Tensor()});
  }
  Normed v;
  if (!norm_forward(*x, *wt, *res, *post, *scale, *out, eps, false, &v, &rc)) Py_RETURN_NONE;
  return rc ? declined(rc) : tuple_of({v.y, v.r});
  END_HANDLE_TH_ERRORS
}

bool gated_norm_forward(const Tensor& x, const Tensor& z, const Tensor& wt, const Tensor& out, float eps, int64_t groups, bool first, bool keep,
                        Normed* v, int* rc) {
  NormCall c(x);
  if (groups <= 0 || groups > c.a.d) return false;
  c.a.groups = (int)groups;
  c.a.norm_first = first;
  c.a.weight = c.vector(wt, 1);
  c.a.z = c.rows(z, x.scalar_type(), &c.a.z_stride);
  c.a.y = c.rows(out, x.scalar_type(), &c.a.y_stride);
  if (!c.ok) return false;
  v->y = out.defined() ? out : c.fresh(&c.a.y, &c.a.y_stride);
  if (keep) v->inv = at::empty({c.a.rows, groups}, x.options().dtype(at::kFloat));
  c.a.inv_rms = ptr<float>(v->inv);
  c.a.eps = eps;
  *rc = f_gated_norm(&c.a, c.w.stream());
  written(out);
  return true;
}

struct GatedNormNode : torch::autograd::Function<GatedNormNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& z, const Tensor& wt, double eps, int64_t groups, bool first,
                               int* rc) {
    Normed v;
    *rc = 1;
    if (!gated_norm_forward(x, z, wt, Tensor(), (float)eps, groups, first, true, &v, rc) || *rc) return {};
    ctx->save_for_backward({x, z, wt, v.inv});
    ctx->saved_data["groups"] = groups;
    ctx->saved_data["first"] = first;
    return {v.y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    NormCall c(s[0]);
    c.a.groups = (int)ctx->saved_data["groups"].toInt();
    c.a.norm_first = ctx->saved_data["first"].toBool();
    c.a.weight = c.vector(s[2], 1);
    c.a.z = c.rows(s[1], s[0].scalar_type(), &c.a.z_stride);
    const Tensor dy = usable_rows(grads[0]);
    c.a.dy = c.rows(dy, s[0].scalar_type(), &c.a.dy_stride);
    c.a.inv_rms = ptr<float>(s[3]);
    must(c.ok, 0, "gated_rms_norm");
    Tensor dx = c.fresh(&c.a.dx, &c.a.dx_stride), dz = c.fresh(&c.a.dz, &c.a.dz_stride), dw = at::empty({(int64_t)c.a.d}, s[2].options());
    c.a.dweight = dw.data_ptr();
    const Tensor ws = c.scratch_of();
    must(true, f_gated_norm_backward(&c.a, c.w.stream()), "gated_rms_norm");
    return once({dx, dz, dw, Tensor(), Tensor(), Tensor(), Tensor()}, "gated_rms_norm");
  }
};

// gated_rms_norm(x, z, weight, out, eps, groups, norm_first) -> y
PyObject* py_gated_norm(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const Tensor *x, *z, *wt, *out;
  float eps;
  int groups;
  if (n != 7 || !get(o[0], &x) || !get(o[1], &z) || !get(o[2], &wt) || !get(o[3], &out, true) || !real(o[4], &eps) ||
      !whole(o[5], &groups) || !norm_operand(*x) || tangents({x, z, wt}))
    Py_RETURN_NONE;
  const bool first = o[6] == Py_True;
  int rc = 0;
  if (records({x, z, wt})) {
    if (out->defined()) Py_RETURN_NONE;
    const variable_list v = GatedNormNode::apply(*x, *z, *wt, (double)eps, (int64_t)groups, first, &rc);
    return rc ? declined(rc) : THPVariable_Wrap(v[0]);
  }
  Normed v;
  if (!gated_norm_forward(*x, *z, *wt, *out, eps, groups, first, false, &v, &rc)) Py_RETURN_NONE;
  return rc ? declined(rc) : THPVariable_Wrap(v.y);
  END_HANDLE_TH_ERRORS
}

// ---- conv1d + SiLU ----

bool conv_operands(const Tensor& x, const Tensor& w, const Tensor& bias, const Tensor& out) {
  if (x.dim() != 3) return false;
  const int64_t d = x.size(2);
  const auto st = x.scalar_type();
  return dtype_of(x) >= 0 && x.stride(2) == 1 && d > 0 && w.scalar_type() == st && w.is_contiguous() && w.dim() >= 2 && w.size(0) == d &&
         w.numel() == d * w.size(-1) && (!bias.defined() || (shaped(bias, {d}) && bias.scalar_type() == st && bias.is_contiguous())) &&
         (!out.defined() || (out.scalar_type() == st && out.sizes() == x.sizes() && inner(out)));
}
bool conv_forward(const Tensor& x, const Tensor& w, const Tensor& bias, const Tensor& out, Tensor* y, int* rc) {
  if (!conv_operands(x, w, bias, out)) return false;
  Where q(x);
  if (!q.here(w) || !q.here(bias) || !q.here(out)) return false;
  *y = out.defined() ? out : at::empty(x.sizes(), x.options());
  *rc = f_conv(x.data_ptr(), w.data_ptr(), ptr(bias), y->data_ptr(), (int)x.size(0), (int)x.size(1), (int)x.size(2), (int)w.size(-1), dtype_of(x),
               x.stride(0), x.stride(1), y->stride(0), y->stride(1), q.stream());
  written(out);
  return true;
}
// What the gradient reads two channels at a time of; other views are copied once.
Tensor usable_pairs(const Tensor& t) {
  const bool ok = t.stride(2) == 1 && t.stride(0) % 2 == 0 && t.stride(1) % 2 == 0 &&
                  reinterpret_cast<uintptr_t>(t.data_ptr()) % (2 * t.element_size()) == 0;
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);   // (a single row counts as contiguous wherever it starts)
}

struct ConvNode : torch::autograd::Function<ConvNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Maybe& bias, int* rc) {
    Tensor y;
    *rc = 1;
    if (!conv_forward(x, w, given(bias), Tensor(), &y, rc) || *rc) return {};
    ctx->save_for_backward({x, w, given(bias)});
    return {y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const Tensor x = usable_pairs(s[0]), dy = usable_pairs(grads[0]);
    const Tensor &w = s[1], &bias = s[2];
    Where q(x);
    const int b = (int)x.size(0), l = (int)x.size(1), d = (int)x.size(2), taps = (int)w.size(-1);
    Tensor dx = at::empty(x.sizes(), x.options()), dw = at::empty(w.sizes(), w.options()), db;
    if (bias.defined()) db = at::empty({(int64_t)d}, bias.options());
    const size_t need = f_conv_workspace(b, l, d, taps);
    const Tensor ws = scratch(x, need);
    must(true, f_conv_backward(x.data_ptr(), w.data_ptr(), ptr(bias), dy.data_ptr(), dx.data_ptr(), dw.data_ptr(), ptr(db), ptr(ws), need, b, l, d,
                               taps, dtype_of(x), x.stride(0), x.stride(1), dy.stride(0), dy.stride(1), dx.stride(0), dx.stride(1),
                               ptr<int32_t>(status_word(q.dev.index())), q.stream()),
         "conv1d_silu");
    return once({dx, dw, db, Tensor()}, "conv1d_silu");
  }
};

// conv1d_silu(x, weight, bias, out) -> y
PyObject* py_conv(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const Tensor *x, *w, *bias, *out;
  if (n != 4 || !get(o[0], &x) || !get(o[1], &w) || !get(o[2], &bias, true) || !get(o[3], &out, true) || !x->is_cuda() ||
      tangents({x, w, bias}))
    Py_RETURN_NONE;
  int rc = 0;
  Tensor y;
  if (!out->defined() && records({x, w, bias})) {
    const variable_list v = ConvNode::apply(*x, *w, maybe(*bias), &rc);
    return rc ? declined(rc) : THPVariable_Wrap(v[0]);
  }
  if (!conv_forward(*x, *w, *bias, *out, &y, &rc)) Py_RETURN_NONE;
  return rc ? declined(rc) : THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// workspace(device_index, bytes), status_word(device_index): the tensors that the long way uses too
PyObject* py_workspace(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 2) Py_RETURN_NONE;
  const long dev = PyLong_AsLong(o[0]);
  const long long bytes = PyLong_AsLongLong(o[1]);
  if (PyErr_Occurred() || dev < 0 || dev >= kMaxDevices) return PyErr_Occurred() ? nullptr : (Py_INCREF(Py_None), Py_None);
  return THPVariable_Wrap(workspace((int)dev, bytes));
  END_HANDLE_TH_ERRORS
}
PyObject* py_status(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 1) Py_RETURN_NONE;
  const long dev = PyLong_AsLong(o[0]);
  if (PyErr_Occurred() || dev < 0 || dev >= kMaxDevices) return PyErr_Occurred() ? nullptr : (Py_INCREF(Py_None), Py_None);
  return THPVariable_Wrap(status_word((int)dev));
  END_HANDLE_TH_ERRORS
}

// init(addresses in the loaded library, in the order of the entry points above, and the function that raises the exception of an
// error code)
template <typename F>
void bind(F& f, PyObject* address) { f = reinterpret_cast<F>(PyLong_AsVoidPtr(address)); }
PyObject* py_init(PyObject*, PyObject* const* o, Py_ssize_t n) {
  if (n != 17) {
    PyErr_SetString(PyExc_TypeError, "init takes sixteen addresses and a function");
    return nullptr;
  }
  bind(f_forward, o[0]); bind(f_workspace, o[1]); bind(f_step, o[2]); bind(f_conv, o[3]); bind(f_dt, o[4]);
  bind(f_conv_workspace, o[5]); bind(f_conv_backward, o[6]);
  bind(f_gated_workspace, o[7]); bind(f_gated, o[8]); bind(f_gated_backward, o[9]); bind(f_gated_step, o[10]);
  bind(f_norm_workspace, o[11]); bind(f_norm, o[12]); bind(f_norm_backward, o[13]); bind(f_gated_norm, o[14]); bind(f_gated_norm_backward, o[15]);
  if (PyErr_Occurred()) return nullptr;
  Py_INCREF(o[16]);
  Py_XSETREF(f_raise, o[16]);
  Py_RETURN_NONE;
}

#define FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(f)), METH_FASTCALL, nullptr
PyMethodDef methods[] = {{"init", FAST(py_init)}, {"step", FAST(py_step)}, {"dt_prologue", FAST(py_dt)},
                         {"conv1d_silu", FAST(py_conv)}, {"gated_scan", FAST(py_gated)}, {"gated_step", FAST(py_gated_step)},
                         {"rms_norm", FAST(py_norm)}, {"gated_rms_norm", FAST(py_gated_norm)},
                         {"forward", FAST(py_forward)}, {"workspace", FAST(py_workspace)},
                         {"status_word", FAST(py_status)}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "ssd_b200_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_ssd_b200_torch(void) { return PyModule_Create(&module); }
