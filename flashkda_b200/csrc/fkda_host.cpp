// The host path of `flash_kda.fwd` and of the operators round it: argument checks, scratch memory and the launch in one native call.
//
// A decode step costs a few microseconds on the GPU; the checks written in Python (some ninety attribute reads), a
// torch.empty, a ctypes structure and a device guard cost 20 of the 26 us that such a call took.  The same conditions are
// read here from the tensor objects directly.  This file only decides "everything is in order" and then calls the C ABI
// (include/fkda.h); whenever anything is not, it reports that and the caller walks the Python checks, which own the order
// and the wording of the errors (the reference's TORCH_CHECKs, csrc/flash_kda.cpp:44-174).
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/fkda.h"

namespace {

// A plain tensor (no subclass with behaviour of its own) on the GPU, contiguous; nullptr otherwise.
const at::Tensor* cuda_tensor(PyObject* o, at::ScalarType type) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  return t.is_cuda() && t.scalar_type() == type && t.is_contiguous() && t.has_storage() ? &t : nullptr;
}

// fwd_fast(q, k, v, g, beta, scale, out, A_log, dt_bias, lower_bound, initial_state, final_state, cu_seqlens)
// -> True: launched; False: not an ordinary call, nothing was done; str: the library's error message.
PyObject* fwd_fast(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 13) Py_RETURN_FALSE;
  const at::Tensor* main[6];
  const int at_main[6] = {0, 1, 2, 3, 4, 6};      // q k v g beta out
  for (int i = 0; i < 6; ++i)
    if ((main[i] = cuda_tensor(a[at_main[i]], at::kBFloat16)) == nullptr) Py_RETURN_FALSE;
  const at::Tensor *A_log = cuda_tensor(a[7], at::kFloat), *dt_bias = cuda_tensor(a[8], at::kFloat);
  if (A_log == nullptr || dt_bias == nullptr) Py_RETURN_FALSE;
  const at::Tensor& q = *main[0];
  if (q.dim() != 4) Py_RETURN_FALSE;
  const int64_t B = q.size(0), T = q.size(1), H = q.size(2), D = q.size(3);
  for (int i : {1, 2, 3, 5})
    if (main[i]->sizes() != q.sizes()) Py_RETURN_FALSE;
  const at::Tensor& beta = *main[4];
  if (D != 128 || beta.dim() != 3 || beta.size(0) != B || beta.size(1) != T || beta.size(2) != H) Py_RETURN_FALSE;
  if (A_log->dim() != 1 || A_log->size(0) != H || dt_bias->dim() != 2 || dt_bias->size(0) != H || dt_bias->size(1) != D) Py_RETURN_FALSE;
  const c10::Device dev = q.device();
  for (const at::Tensor* t : {main[1], main[2], main[3], main[4], main[5], A_log, dt_bias})
    if (t->device() != dev) Py_RETURN_FALSE;
  int64_t N = B;
  const at::Tensor* cu = nullptr;
  if (a[12] != Py_None) {
    if ((cu = cuda_tensor(a[12], at::kLong)) == nullptr || B != 1 || cu->dim() != 1 || cu->numel() < 2 || cu->device() != dev) Py_RETURN_FALSE;
    N = cu->numel() - 1;
  }
  const at::Tensor* state[2] = {nullptr, nullptr};
  int state_dtype = FKDA_STATE_NONE;
  for (int i = 0; i < 2; ++i) {
    if (a[10 + i] == Py_None) continue;
    const at::Tensor* s = cuda_tensor(a[10 + i], at::kFloat);
    const int type = s != nullptr ? FKDA_STATE_FP32 : FKDA_STATE_BF16;
    if (s == nullptr && (s = cuda_tensor(a[10 + i], at::kBFloat16)) == nullptr) Py_RETURN_FALSE;
    if (state_dtype != FKDA_STATE_NONE && state_dtype != type) Py_RETURN_FALSE;
    if (s->dim() != 4 || s->size(0) != N || s->size(1) != H || s->size(2) != D || s->size(3) != D || s->device() != dev) Py_RETURN_FALSE;
    state[i] = s;
    state_dtype = type;
  }
  if (!PyFloat_CheckExact(a[5]) || !PyFloat_CheckExact(a[9])) Py_RETURN_FALSE;

  fkda_fwd_params p{};
  p.q = q.data_ptr();
  p.k = main[1]->data_ptr();
  p.v = main[2]->data_ptr();
  p.g = main[3]->data_ptr();
  p.beta = beta.data_ptr();
  p.out = main[5]->data_ptr();
  p.A_log = static_cast<const float*>(A_log->data_ptr());
  p.dt_bias = static_cast<const float*>(dt_bias->data_ptr());
  p.initial_state = state[0] != nullptr ? state[0]->data_ptr() : nullptr;
  p.final_state = state[1] != nullptr ? state[1]->data_ptr() : nullptr;
  p.cu_seqlens = cu != nullptr ? static_cast<const int64_t*>(cu->data_ptr()) : nullptr;
  p.B = B;
  p.T = T;
  p.H = H;
  p.N = N;
  p.scale = static_cast<float>(PyFloat_AS_DOUBLE(a[5]));
  p.lower_bound = static_cast<float>(PyFloat_AS_DOUBLE(a[9]));
  p.state_dtype = state_dtype;
  p.flags = FKDA_FLAG_STATUS_UNREAD;      // the scratch memory is not the caller's: nobody can read its status word

  char message[512];
  bool failed = false;
  try {
    c10::cuda::CUDAGuard guard(dev);
    int64_t bytes = 0;
    if (fkda_fwd_scratch_bytes(&p, &bytes) != FKDA_OK) Py_RETURN_FALSE;
    // freed when the call returns: the caching allocator hands a block only to later work of the same stream
    // (none for a decode step, where asking for it would be a tenth of the call)
    c10::DataPtr ws;
    if (bytes > 0) ws = c10::cuda::CUDACachingAllocator::get()->allocate(static_cast<size_t>(bytes));
    p.workspace = ws.get();
    p.workspace_bytes = bytes;
    void* stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = fkda_fwd(&p, stream);
    Py_END_ALLOW_THREADS
    if (rc != FKDA_OK) {
      snprintf(message, sizeof(message), "flash_kda: %s (code %d)", fkda_last_error(), rc);
      failed = true;
    }
  } catch (const c10::OutOfMemoryError&) {
    Py_RETURN_FALSE;                       // the Python path meets the same and raises torch's own exception
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
  if (failed) return PyUnicode_FromString(message);
  Py_RETURN_TRUE;
}

// ---- the operators round the recurrence ------------------------------------------------------------------------------------
// The same division of labour: True = launched; False = not in order, or not understood here, nothing was done; a str = the library's
// error message.

PyObject* launched(int rc) {
  if (rc == FKDA_OK) Py_RETURN_TRUE;
  char message[600];
  snprintf(message, sizeof(message), "flash_kda: %s (code %d)", fkda_last_error(), rc);
  return PyUnicode_FromString(message);
}
// A plain tensor on the GPU; nullptr otherwise.
const at::Tensor* any_tensor(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  return t.is_cuda() && t.has_storage() ? &t : nullptr;
}
// ... of that type, [B, T, ...] with dense tokens.
const at::Tensor* tokens(PyObject* o, at::ScalarType type, int dims) {
  const at::Tensor* t = any_tensor(o);
  if (t == nullptr || t->scalar_type() != type || t->dim() != dims) return nullptr;
  int64_t dense = 1;
  for (int i = dims - 1; i >= 2; --i) {
    if (t->size(i) != 1 && t->stride(i) != dense) return nullptr;
    dense *= t->size(i);
  }
  return t;
}
// ... contiguous, bf16 or fp32.
const at::Tensor* parameter(PyObject* o, int32_t* dtype) {
  const at::Tensor* t = any_tensor(o);
  if (t == nullptr || !t->is_contiguous()) return nullptr;
  *dtype = t->scalar_type() == at::kFloat ? FKDA_STATE_FP32 : t->scalar_type() == at::kBFloat16 ? FKDA_STATE_BF16 : FKDA_STATE_NONE;
  return *dtype != FKDA_STATE_NONE ? t : nullptr;
}
bool is_shape(const at::Tensor& t, std::initializer_list<int64_t> want) { return t.sizes() == at::IntArrayRef(want); }
bool number(PyObject* o, double* v) {
  if (!PyFloat_CheckExact(o)) return false;
  *v = PyFloat_AS_DOUBLE(o);
  return true;
}
// cu_seqlens or None: the sequences, or a batch of them.
bool sequences(PyObject* o, int64_t B, c10::Device dev, const int64_t** cu, int64_t* N) {
  *N = B;
  *cu = nullptr;
  if (o == Py_None) return true;
  const at::Tensor* t = cuda_tensor(o, at::kLong);
  if (t == nullptr || B != 1 || t->dim() != 1 || t->numel() < 2 || t->device() != dev) return false;
  *cu = static_cast<const int64_t*>(t->data_ptr());
  *N = t->numel() - 1;
  return true;
}
// A contiguous state of that shape and device, or None (nullptr in `data`); its type in `dtype`.
bool state_of(PyObject* o, std::initializer_list<int64_t> want, c10::Device dev, void** data, int32_t* dtype) {
  *data = nullptr;
  if (o == Py_None) return true;
  int32_t type;
  const at::Tensor* t = parameter(o, &type);
  if (t == nullptr || t->device() != dev || !is_shape(*t, want) || (*dtype != FKDA_STATE_NONE && *dtype != type)) return false;
  *data = t->data_ptr();
  *dtype = type;
  return true;
}
template <class Launch>
PyObject* on_device(c10::Device dev, Launch launch) {
  try {
    c10::cuda::CUDAGuard guard(dev);
    void* stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
    return launch(stream);
  } catch (const c10::OutOfMemoryError&) {
    Py_RETURN_FALSE;                       // the Python path meets the same and raises torch's own exception
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}
template <class Params>
PyObject* simple_launch(c10::Device dev, int (*fn)(const Params*, void*), const Params& p) {
  return on_device(dev, [&](void* stream) {
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = fn(&p, stream);
    Py_END_ALLOW_THREADS
    return launched(rc);
  });
}
#define FKDA_STRIDES(p, name, t) \
  p.name##_batch_stride = (t)->stride(0); \
  p.name##_token_stride = (t)->stride(1)

// short_conv_fast(x, weight, out, bias, initial_state, final_state, cu_seqlens, silu)
PyObject* short_conv_fast(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 8 || !PyBool_Check(a[7])) Py_RETURN_FALSE;
  fkda_conv_params p{};
  const at::Tensor *x = tokens(a[0], at::kBFloat16, 3), *out = tokens(a[2], at::kBFloat16, 3), *weight = parameter(a[1], &p.weight_dtype);
  if (x == nullptr || out == nullptr || weight == nullptr || x->sizes() != out->sizes()) Py_RETURN_FALSE;
  const c10::Device dev = x->device();
  p.B = x->size(0);
  p.T = x->size(1);
  p.C = x->size(2);
  if (weight->dim() != 2 || weight->size(0) != p.C || out->device() != dev || weight->device() != dev) Py_RETURN_FALSE;
  p.width = static_cast<int32_t>(weight->size(1) > 4 ? 0 : weight->size(1));
  if (a[3] != Py_None) {
    int32_t type;
    const at::Tensor* bias = parameter(a[3], &type);
    if (bias == nullptr || type != p.weight_dtype || bias->device() != dev || !is_shape(*bias, {p.C})) Py_RETURN_FALSE;
    p.bias = bias->data_ptr();
  }
  if (!sequences(a[6], p.B, dev, &p.cu_seqlens, &p.N)) Py_RETURN_FALSE;
  void *in, *fin;
  int32_t type = FKDA_STATE_BF16;
  if (!state_of(a[4], {p.N, p.width - 1, p.C}, dev, &in, &type) || !state_of(a[5], {p.N, p.width - 1, p.C}, dev, &fin, &type)) Py_RETURN_FALSE;
  p.x = x->data_ptr();
  p.weight = weight->data_ptr();
  p.out = out->data_ptr();
  p.initial_state = in;
  p.final_state = fin;
  FKDA_STRIDES(p, x, x);
  FKDA_STRIDES(p, out, out);
  p.silu = a[7] == Py_True;
  return simple_launch(dev, fkda_short_conv, p);
}

// ssm_fwd_fast(x, dt, B, C, out, A_log, dt_bias, D, initial_state, final_state, cu_seqlens)
PyObject* ssm_fwd_fast(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 11) Py_RETURN_FALSE;
  const at::Tensor *x = tokens(a[0], at::kBFloat16, 4), *dt = tokens(a[1], at::kBFloat16, 3), *b = tokens(a[2], at::kBFloat16, 4),
                   *c = tokens(a[3], at::kBFloat16, 4), *out = tokens(a[4], at::kBFloat16, 4);
  if (x == nullptr || dt == nullptr || b == nullptr || c == nullptr || out == nullptr) Py_RETURN_FALSE;
  const c10::Device dev = x->device();
  fkda_ssm_params p{};
  p.B = x->size(0);
  p.T = x->size(1);
  p.H = x->size(2);
  p.P = x->size(3);
  p.G = b->size(2);
  p.Ns = b->size(3);
  if (out->sizes() != x->sizes() || c->sizes() != b->sizes() || b->size(0) != p.B || b->size(1) != p.T || !is_shape(*dt, {p.B, p.T, p.H})) Py_RETURN_FALSE;
  for (const at::Tensor* t : {dt, b, c, out})
    if (t->device() != dev) Py_RETURN_FALSE;
  const float** const per_head[3] = {&p.A_log, &p.dt_bias, &p.D};
  for (int i = 0; i < 3; ++i) {
    if (i == 2 && a[7] == Py_None) continue;
    const at::Tensor* t = cuda_tensor(a[5 + i], at::kFloat);
    if (t == nullptr || t->device() != dev || !is_shape(*t, {p.H})) Py_RETURN_FALSE;
    *per_head[i] = static_cast<const float*>(t->data_ptr());
  }
  if (!sequences(a[10], p.B, dev, &p.cu_seqlens, &p.N)) Py_RETURN_FALSE;
  void *in, *fin;
  if (!state_of(a[8], {p.N, p.H, p.P, p.Ns}, dev, &in, &p.state_dtype) || !state_of(a[9], {p.N, p.H, p.P, p.Ns}, dev, &fin, &p.state_dtype)) Py_RETURN_FALSE;
  p.x = x->data_ptr();
  p.dt = dt->data_ptr();
  p.Bm = b->data_ptr();
  p.Cm = c->data_ptr();
  p.out = out->data_ptr();
  p.initial_state = in;
  p.final_state = fin;
  FKDA_STRIDES(p, x, x);
  FKDA_STRIDES(p, dt, dt);
  FKDA_STRIDES(p, B, b);
  FKDA_STRIDES(p, C, c);
  FKDA_STRIDES(p, out, out);
  p.flags = FKDA_FLAG_STATUS_UNREAD;
  return on_device(dev, [&](void* stream) -> PyObject* {
    if (fkda_ssm_scratch_bytes(&p, &p.workspace_bytes) != FKDA_OK) Py_RETURN_FALSE;
    c10::DataPtr ws;                       // (freed when the call returns, as in fwd_fast)
    if (p.workspace_bytes > 0) ws = c10::cuda::CUDACachingAllocator::get()->allocate(static_cast<size_t>(p.workspace_bytes));
    p.workspace = ws.get();
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = fkda_ssm_fwd(&p, stream);
    Py_END_ALLOW_THREADS
    return launched(rc);
  });
}

// gated_norm_fast(x, gate, weight, out, eps, act, gate_first)
PyObject* gated_norm_fast(PyObject*, PyObject* const* a, Py_ssize_t n) {
  double eps;
  if (n != 7 || !number(a[4], &eps) || !PyUnicode_CheckExact(a[5]) || !PyBool_Check(a[6])) Py_RETURN_FALSE;
  fkda_gated_norm_params p{};
  const at::Tensor *x = tokens(a[0], at::kBFloat16, 4), *gate = tokens(a[1], at::kBFloat16, 4), *out = tokens(a[3], at::kBFloat16, 4),
                   *weight = parameter(a[2], &p.weight_dtype);
  if (x == nullptr || gate == nullptr || out == nullptr || weight == nullptr) Py_RETURN_FALSE;
  const c10::Device dev = x->device();
  p.B = x->size(0);
  p.T = x->size(1);
  p.H = x->size(2);
  p.D = x->size(3);
  p.weight_per_head = weight->dim() == 2;
  if (gate->sizes() != x->sizes() || out->sizes() != x->sizes() || !(p.weight_per_head ? is_shape(*weight, {p.H, p.D}) : is_shape(*weight, {p.D}))) Py_RETURN_FALSE;
  for (const at::Tensor* t : {gate, out, weight})
    if (t->device() != dev) Py_RETURN_FALSE;
  p.silu = PyUnicode_CompareWithASCIIString(a[5], "silu") == 0;
  if (!p.silu && PyUnicode_CompareWithASCIIString(a[5], "sigmoid") != 0) Py_RETURN_FALSE;
  p.x = x->data_ptr();
  p.gate = gate->data_ptr();
  p.weight = weight->data_ptr();
  p.out = out->data_ptr();
  FKDA_STRIDES(p, x, x);
  FKDA_STRIDES(p, gate, gate);
  FKDA_STRIDES(p, out, out);
  p.eps = static_cast<float>(eps);
  p.gate_first = a[6] == Py_True;
  return simple_launch(dev, fkda_gated_norm, p);
}

// add_norm_fast(x, residual, weight, out, residual_out, scale, eps)
PyObject* add_norm_fast(PyObject*, PyObject* const* a, Py_ssize_t n) {
  double scale, eps;
  if (n != 7 || !number(a[5], &scale) || !number(a[6], &eps)) Py_RETURN_FALSE;
  fkda_add_norm_params p{};
  const at::Tensor *x = tokens(a[0], at::kBFloat16, 3), *out = tokens(a[3], at::kBFloat16, 3), *weight = parameter(a[2], &p.weight_dtype);
  if (x == nullptr || out == nullptr || weight == nullptr) Py_RETURN_FALSE;
  const at::Tensor* residual = tokens(a[1], at::kFloat, 3);
  const at::ScalarType type = residual != nullptr ? at::kFloat : at::kBFloat16;
  if (residual == nullptr) residual = tokens(a[1], type, 3);
  const at::Tensor* residual_out = tokens(a[4], type, 3);
  if (residual == nullptr || residual_out == nullptr) Py_RETURN_FALSE;
  const c10::Device dev = x->device();
  p.B = x->size(0);
  p.T = x->size(1);
  p.D = x->size(2);
  for (const at::Tensor* t : {out, residual, residual_out})
    if (t->sizes() != x->sizes() || t->device() != dev) Py_RETURN_FALSE;
  if (!is_shape(*weight, {p.D}) || weight->device() != dev) Py_RETURN_FALSE;
  p.x = x->data_ptr();
  p.residual = residual->data_ptr();
  p.weight = weight->data_ptr();
  p.out = out->data_ptr();
  p.residual_out = residual_out->data_ptr();
  FKDA_STRIDES(p, x, x);
  FKDA_STRIDES(p, residual, residual);
  FKDA_STRIDES(p, out, out);
  FKDA_STRIDES(p, residual_out, residual_out);
  p.scale = static_cast<float>(scale);
  p.eps = static_cast<float>(eps);
  p.residual_dtype = type == at::kFloat ? FKDA_STATE_FP32 : FKDA_STATE_BF16;
  return simple_launch(dev, fkda_add_norm, p);
}

PyMethodDef methods[] = {
    {"fwd_fast", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(fwd_fast)), METH_FASTCALL,
     "checks an ordinary flash_kda.fwd call and launches it"},
    {"short_conv_fast", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(short_conv_fast)), METH_FASTCALL, "the same for short_conv"},
    {"ssm_fwd_fast", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(ssm_fwd_fast)), METH_FASTCALL, "the same for ssm_fwd"},
    {"gated_norm_fast", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(gated_norm_fast)), METH_FASTCALL, "the same for gated_norm"},
    {"add_norm_fast", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(add_norm_fast)), METH_FASTCALL, "the same for add_norm"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fkda_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fkda_host(void) {
  PyObject* m = PyModule_Create(&module);
  // the torch whose headers this was compiled against: another one may lay out a tensor differently (checked by the loader)
  if (m != nullptr && PyModule_AddStringConstant(m, "torch_version", FKDA_TORCH_VERSION) != 0) Py_CLEAR(m);
  return m;
}
