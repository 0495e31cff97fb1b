// Small calls from Python without the interpreter between the check of the arguments and the launch: lm2exp and lt2exp on
// ordinary CUDA tensors, for the sizes that one launch of the direct kernels takes.  A call of 4 us on the device took 17 us
// of Python (shape and stride objects, ctypes conversions); here 5.  The operators around them, which have one kernel for
// all sizes or a rule inside the library, are here for ordinary tensors of any size.
//
// All functions return None, having done nothing, for every call that is not such a one: other tensor types and modes,
// wrong shapes, larger problems.  The Python code behind them then does what it would have done without them.
#include <Python.h>

#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/ops/empty.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <c10/util/SmallVector.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <limits>
#include <utility>

#include "../../include/triturus_b200.h"

namespace {

// No tracing, no transform (vmap, grad, functionalisation) and no Python mode that would want to see the operations.
bool plain_mode() {
  using c10::DispatchKey;
  const c10::DispatchKeySet inc = c10::impl::tls_local_dispatch_key_set().included_;
  return !inc.has(DispatchKey::Python) && !inc.has(DispatchKey::Tracer) && !inc.has(DispatchKey::Functionalize) &&
         !inc.has(DispatchKey::FuncTorchDynamicLayerFrontMode) && !inc.has(DispatchKey::FuncTorchDynamicLayerBackMode) &&
         !at::impl::torch_function_mode_enabled();
}

// A float32 CUDA tensor that is nothing but its storage, shape and strides: the dispatch keys are those of an ordinary (or an
// inference) tensor, so no wrapper, lazy conjugation or negation, quantisation, subclass.
const at::Tensor* plain_object(PyObject* o) {
  using c10::DispatchKey;
  static const c10::DispatchKeySet ordinary(
      {DispatchKey::CUDA, DispatchKey::AutogradCUDA, DispatchKey::ADInplaceOrView, DispatchKey::AutocastCUDA});
  static const c10::DispatchKeySet inference({DispatchKey::CUDA, DispatchKey::AutocastCUDA});
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  const c10::DispatchKeySet ks = t.key_set();
  if (ks != ordinary && ks != inference) return nullptr;
  return t.layout() == at::kStrided && t.numel() != 0 ? &t : nullptr;
}

const at::Tensor* plain_tensor(PyObject* o, int64_t dim) {
  const at::Tensor* t = plain_object(o);
  return t != nullptr && t->scalar_type() == at::kFloat && t->dim() == dim ? t : nullptr;
}

// The library's code for an element type, or -1.
int type_code(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return TRITURUS_B200_TYPE_F32;
    case at::kBFloat16: return TRITURUS_B200_TYPE_BF16;
    case at::kHalf: return TRITURUS_B200_TYPE_F16;
    default: return -1;
  }
}

// Rows of consecutive elements at one distance, without a copy: that distance, or -1 where the strides may be something else.
int64_t row_stride(const at::Tensor& t) {
  if (t.is_contiguous()) return t.size(-1);
  return t.dim() == 2 && t.stride(1) == 1 ? t.stride(0) : -1;
}

bool int_arg(PyObject* o, int* v) {
  const long x = PyLong_AsLong(o);
  if (x == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  *v = static_cast<int>(x);
  return *v == x;
}

struct ThreadsRun {  // without the interpreter lock, for the time of a launch: it waits where the queue of the stream is full
  PyThreadState* state = PyEval_SaveThread();
  ~ThreadsRun() { PyEval_RestoreThread(state); }
};

PyObject* none() { Py_RETURN_NONE; }

at::Tensor new_result(const at::Tensor& like, int64_t r, int64_t i, int64_t k) {
  return at::empty({r, i, k}, at::TensorOptions().dtype(at::kFloat).device(like.device()));
}

// Set by the Python side.
PyObject* error_class = nullptr;  // what it raises for a code of the library
double copy_flop_rows = 0.0;      // problems of more operations than this get a padded copy of an operand that no tensor map
double copy_flop_strided = 0.0;   // describes: of rows of consecutive floats, and of other views

PyObject* failed(const char* what, int rc) {
  PyErr_Format(error_class != nullptr ? error_class : PyExc_RuntimeError, "%s failed with code %d: %s", what, rc, triturus_b200_strerror(rc));
  return nullptr;
}

// lm2exp(a, b, precision, variant)
PyObject* lm2exp(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  int precision, variant;
  if (nargs != 4 || !int_arg(args[2], &precision) || !int_arg(args[3], &variant) || variant != 0 || !plain_mode()) return none();
  const at::Tensor* a = plain_tensor(args[0], 3);
  const at::Tensor* b = a != nullptr ? plain_tensor(args[1], 3) : nullptr;
  if (b == nullptr || a->device() != b->device() || a->get_device() != c10::cuda::current_device()) return none();
  const int64_t R = a->size(0), I = a->size(1), J = a->size(2), K = b->size(2);
  if (b->size(0) != R || b->size(1) != J) return none();
  const int64_t* as = a->strides().data();
  const int64_t* bs = b->strides().data();
  const float* ap = a->const_data_ptr<float>();
  const float* bp = b->const_data_ptr<float>();
  const int small = triturus_b200_lm2exp_small_f32(ap, bp, nullptr, R, I, J, K, as, bs, nullptr, precision, nullptr);
  if (small <= 0) return none();
  // (the copies are the Python side's; with them the call is one of the large kernels)
  const double flop = 2.0 * static_cast<double>(R) * static_cast<double>(I) * static_cast<double>(J) * static_cast<double>(K);
  if ((small & 2) != 0 && flop > (as[2] == 1 ? copy_flop_rows : copy_flop_strided)) return none();
  if ((small & 4) != 0 && flop > (bs[2] == 1 ? copy_flop_rows : copy_flop_strided)) return none();
  at::Tensor out = new_result(*a, R, I, K);
  float* op = out.mutable_data_ptr<float>();
  const auto stream = c10::cuda::getCurrentCUDAStream(a->get_device()).stream();
  int rc;
  {
    ThreadsRun unlocked;
    rc = triturus_b200_lm2exp_small_f32(ap, bp, op, R, I, J, K, as, bs, out.strides().data(), precision, stream);
  }
  if (rc != TRITURUS_B200_OK) return failed("triturus_b200_lm2exp_small_f32", rc);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// lt2exp(w, a, b, precision, variant)
PyObject* lt2exp(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  int precision, variant;
  if (nargs != 5 || !int_arg(args[3], &precision) || !int_arg(args[4], &variant) || !plain_mode()) return none();
  const at::Tensor* w = plain_tensor(args[0], 4);
  const at::Tensor* a = w != nullptr ? plain_tensor(args[1], 3) : nullptr;
  const at::Tensor* b = a != nullptr ? plain_tensor(args[2], 3) : nullptr;
  if (b == nullptr || w->device() != a->device() || a->device() != b->device() || a->get_device() != c10::cuda::current_device())
    return none();
  const int64_t R = w->size(0), S = w->size(1), I = w->size(2), J = w->size(3), K = a->size(2);
  if (a->size(0) != R || a->size(1) != I || b->size(0) != R || b->size(1) != J || b->size(2) != K) return none();
  const int64_t* ws = w->strides().data();
  if (I > 1 && J > 1 && ws[2] != J * ws[3]) return none();  // (I and J are not one dimension: refused, as the reference's view does)
  const float* wp = w->const_data_ptr<float>();
  const uint64_t bits = (reinterpret_cast<uintptr_t>(wp) >> 2) | static_cast<uint64_t>(J | ws[0] | ws[1] | ws[2]);
  const int odd = ws[3] != 1 || (bits & 1) != 0;
  if (triturus_b200_lt2exp_direct(R, S, I, J, K, precision, variant, odd) != 1) return none();
  at::Tensor out = new_result(*a, R, S, K);
  const float *ap = a->const_data_ptr<float>(), *bp = b->const_data_ptr<float>();
  float* op = out.mutable_data_ptr<float>();
  const auto stream = c10::cuda::getCurrentCUDAStream(a->get_device()).stream();
  int rc;
  {
    ThreadsRun unlocked;
    rc = triturus_b200_lt2exp_direct_f32(wp, ap, bp, op, R, S, I, J, K, ws, a->strides().data(), b->strides().data(), out.strides().data(),
                                         precision, nullptr, nullptr, nullptr, stream);
  }
  if (rc != TRITURUS_B200_OK) return failed("triturus_b200_lt2exp_direct_f32", rc);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// None, or a vector of `n` elements of x's type or 32 bits on x's device; sets *type to its code.  False: not an ordinary one.
bool weight_arg(PyObject* o, const at::Tensor& x, int64_t n, const at::Tensor** t, int* type) {
  *t = nullptr;
  if (o == Py_None) return true;
  const at::Tensor* w = plain_object(o);
  if (w == nullptr || w->dim() != 1 || w->size(0) != n || (n != 1 && w->stride(0) != 1) || w->device() != x.device()) return false;
  const int code = type_code(*w);
  if (code != TRITURUS_B200_TYPE_F32 && w->scalar_type() != x.scalar_type()) return false;
  if (*type >= 0 && *type != code) return false;
  *type = code;
  *t = w;
  return true;
}

const void* data_of(const at::Tensor* t) { return t != nullptr ? t->const_data_ptr() : nullptr; }

at::Tensor empty_on(const at::Tensor& like, at::IntArrayRef shape, at::ScalarType type) {
  return at::empty(shape, at::TensorOptions().dtype(type).device(like.device()));
}

PyObject* tuple3(at::Tensor* a, at::Tensor* b, at::Tensor* c) {
  PyObject* out = PyTuple_New(3);
  if (out == nullptr) return nullptr;
  at::Tensor* all[3] = {a, b, c};
  for (int i = 0; i < 3; ++i) PyTuple_SET_ITEM(out, i, all[i] != nullptr ? THPVariable_Wrap(std::move(*all[i])) : Py_NewRef(Py_None));
  return out;
}

// A tensor of forward-mode differentiation, which looks like any other.
bool has_tangent(const at::Tensor* t) { return t != nullptr && t->_fw_grad(0).defined(); }

// layer_norm(x, weight, bias, eps, return_stats)
PyObject* layer_norm(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 5 || !PyFloat_Check(args[3]) || !PyBool_Check(args[4]) || !plain_mode()) return none();
  const at::Tensor* x = plain_object(args[0]);
  if (x == nullptr || x->dim() < 1 || x->get_device() != c10::cuda::current_device()) return none();
  const int type = type_code(*x);
  const int64_t stride = row_stride(*x), width = x->size(-1), rows = x->numel() / width;
  const at::Tensor *weight, *bias;
  int weight_type = -1;
  if (type < 0 || stride < 0 || !weight_arg(args[1], *x, width, &weight, &weight_type) || !weight_arg(args[2], *x, width, &bias, &weight_type))
    return none();
  if (has_tangent(x) || has_tangent(weight) || has_tangent(bias)) return none();  // (refused there)
  const bool stats = args[4] == Py_True;
  at::Tensor y = empty_on(*x, x->sizes(), x->scalar_type()), mean, rstd;
  float *mp = nullptr, *rp = nullptr;
  if (stats) {
    const at::IntArrayRef lead = x->sizes().slice(0, x->dim() - 1);
    mean = empty_on(*x, lead, at::kFloat);
    rstd = empty_on(*x, lead, at::kFloat);
    mp = mean.mutable_data_ptr<float>();
    rp = rstd.mutable_data_ptr<float>();
  }
  const auto stream = c10::cuda::getCurrentCUDAStream(x->get_device()).stream();
  int rc;
  {
    ThreadsRun unlocked;
    rc = triturus_b200_layer_norm(x->const_data_ptr(), data_of(weight), data_of(bias), y.mutable_data_ptr(), mp, rp, rows, width, stride, type,
                                  weight_type < 0 ? type : weight_type, static_cast<float>(PyFloat_AS_DOUBLE(args[3])), stream);
  }
  if (rc != TRITURUS_B200_OK) return failed("triturus_b200_layer_norm", rc);
  return stats ? tuple3(&y, &mean, &rstd) : THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// layer_norm_backward(dy, x, mean, rstd, weight, weight_grad, bias_grad)
PyObject* layer_norm_backward(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 7 || !PyBool_Check(args[5]) || !PyBool_Check(args[6]) || !plain_mode()) return none();
  const at::Tensor* x = plain_object(args[1]);
  const at::Tensor* dy = x != nullptr ? plain_object(args[0]) : nullptr;
  const at::Tensor* mean = dy != nullptr ? plain_object(args[2]) : nullptr;
  const at::Tensor* rstd = mean != nullptr ? plain_object(args[3]) : nullptr;
  if (rstd == nullptr || x->dim() < 1 || x->get_device() != c10::cuda::current_device()) return none();
  const int type = type_code(*x);
  if (type < 0 || dy->scalar_type() != x->scalar_type() || dy->sizes() != x->sizes() || dy->device() != x->device()) return none();
  const at::IntArrayRef lead = x->sizes().slice(0, x->dim() - 1);
  for (const at::Tensor* t : {mean, rstd})
    if (t->scalar_type() != at::kFloat || t->sizes() != lead || !t->is_contiguous() || t->device() != x->device()) return none();
  const int64_t x_stride = row_stride(*x), dy_stride = row_stride(*dy), width = x->size(-1), rows = x->numel() / width;
  const at::Tensor* weight;
  int weight_type = -1;
  if (x_stride < 0 || dy_stride < 0 || !weight_arg(args[4], *x, width, &weight, &weight_type)) return none();
  const at::ScalarType kind = weight != nullptr ? weight->scalar_type() : x->scalar_type();
  const bool want_weight = args[5] == Py_True, want_bias = args[6] == Py_True;
  at::Tensor dx = empty_on(*x, x->sizes(), x->scalar_type()), dweight, dbias;
  if (want_weight) dweight = empty_on(*x, {width}, kind);
  if (want_bias) dbias = empty_on(*x, {width}, kind);
  const size_t bytes = triturus_b200_layer_norm_backward_workspace_bytes(rows, width, type);
  at::Tensor ws = empty_on(*x, {static_cast<int64_t>(bytes)}, at::kByte);
  const auto stream = c10::cuda::getCurrentCUDAStream(x->get_device()).stream();
  int rc;
  {
    ThreadsRun unlocked;
    rc = triturus_b200_layer_norm_backward(dy->const_data_ptr(), x->const_data_ptr(), data_of(weight), mean->const_data_ptr<float>(),
                                           rstd->const_data_ptr<float>(), dx.mutable_data_ptr(), want_weight ? dweight.mutable_data_ptr() : nullptr,
                                           want_bias ? dbias.mutable_data_ptr() : nullptr, rows, width, dy_stride, x_stride, type,
                                           weight_type < 0 ? type : weight_type, ws.mutable_data_ptr(), bytes, stream);
  }
  if (rc != TRITURUS_B200_OK) return failed("triturus_b200_layer_norm_backward", rc);
  return tuple3(&dx, want_weight ? &dweight : nullptr, want_bias ? &dbias : nullptr);
  END_HANDLE_TH_ERRORS
}

// clip_grad_norm(grads, max_norm, norm_type, scale): a list or tuple of dense tensors and None
PyObject* clip_grad_norm(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 4 || !(PyList_CheckExact(args[0]) || PyTuple_CheckExact(args[0])) || !PyFloat_CheckExact(args[1]) || !PyFloat_CheckExact(args[2]) ||
      !plain_mode())
    return none();
  const double max_norm = PyFloat_AS_DOUBLE(args[1]), norm_type = PyFloat_AS_DOUBLE(args[2]);
  const bool scale = args[3] == Py_True;
  if (norm_type != 2.0 && !(std::isinf(norm_type) && norm_type > 0)) return none();
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(args[0]);
  c10::SmallVector<void*, 64> data;
  c10::SmallVector<int64_t, 64> numels;
  c10::SmallVector<int, 64> types;
  c10::SmallVector<at::Tensor, 64> tensors;  // held: while other Python threads run, the list may lose its own
  c10::SmallVector<std::pair<uintptr_t, uintptr_t>, 64> ranges;
  c10::DeviceIndex device = -1;
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* o = PySequence_Fast_GET_ITEM(args[0], i);
    if (o == Py_None) continue;
    const at::Tensor* t = plain_object(o);
    const int type = t != nullptr ? type_code(*t) : -1;
    if (t != nullptr && device < 0) device = c10::cuda::current_device();  // (not asked where there is no GPU)
    if (type < 0 || t->get_device() != device || !t->is_non_overlapping_and_dense() || (scale && (t->requires_grad() || has_tangent(t)))) return none();
    void* p = const_cast<void*>(t->const_data_ptr());
    const uintptr_t at = reinterpret_cast<uintptr_t>(p);
    data.push_back(p);
    numels.push_back(t->numel());
    types.push_back(type);
    tensors.push_back(*t);
    if (scale) ranges.emplace_back(at, at + t->numel() * t->element_size());
  }
  if (tensors.empty()) return none();
  std::sort(ranges.begin(), ranges.end());
  for (size_t i = 1; i < ranges.size(); ++i)
    if (ranges[i].first < ranges[i - 1].second) return none();
  const int64_t count = static_cast<int64_t>(tensors.size());
  const size_t bytes = triturus_b200_clip_grad_norm_workspace_bytes(count);
  at::Tensor norm = empty_on(tensors[0], {}, at::kFloat);
  at::Tensor ws = empty_on(tensors[0], {static_cast<int64_t>(bytes / 8)}, at::kDouble);
  float* np = norm.mutable_data_ptr<float>();
  const auto stream = c10::cuda::getCurrentCUDAStream(device).stream();
  int rc;
  {
    ThreadsRun unlocked;
    rc = triturus_b200_clip_grad_norm(data.data(), numels.data(), types.data(), count, max_norm, norm_type != 2.0, scale, np,
                                      ws.mutable_data_ptr(), bytes, stream);
  }
  if (rc != TRITURUS_B200_OK) return failed("triturus_b200_clip_grad_norm", rc);
  if (scale)
    for (const at::Tensor& t : tensors)
      if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
  return THPVariable_Wrap(std::move(norm));
  END_HANDLE_TH_ERRORS
}

// A parameter of sample: a number in [least, most], None (`off`), or a contiguous tensor of the rows' shape.
bool sample_arg(PyObject* o, const at::Tensor& logits, at::ScalarType kind, double least, double most, const void** array, double* number) {
  *array = nullptr;
  if (o == Py_None) return true;
  if (PyFloat_CheckExact(o) || PyLong_CheckExact(o)) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) {
      PyErr_Clear();
      return false;
    }
    *number = v;
    return v >= least && v <= most && (kind != at::kInt || PyLong_CheckExact(o));
  }
  const at::Tensor* t = plain_object(o);
  if (t == nullptr || t->scalar_type() != kind || t->device() != logits.device() || !t->is_contiguous()) return false;
  if (t->sizes() != logits.sizes().slice(0, logits.dim() - 1)) return false;
  *array = t->const_data_ptr();
  return true;
}

// sample(logits, noise, temperature, top_k, top_p, min_p, return_logprob)
PyObject* sample(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 7 || !PyBool_Check(args[6]) || args[2] == Py_None || !plain_mode()) return none();
  const at::Tensor* logits = plain_object(args[0]);
  const at::Tensor* noise = logits != nullptr ? plain_object(args[1]) : nullptr;
  if (noise == nullptr || logits->dim() < 1 || logits->get_device() != c10::cuda::current_device()) return none();
  const int type = type_code(*logits);
  if (type < 0 || noise->scalar_type() != at::kFloat || noise->sizes() != logits->sizes() || noise->device() != logits->device()) return none();
  const int64_t stride = row_stride(*logits), noise_stride = row_stride(*noise), symbols = logits->size(-1), rows = logits->numel() / symbols;
  const void *temperature, *top_k, *top_p, *min_p;
  double t0 = 1.0, k0 = 0.0, p0 = 1.0, m0 = 0.0;
  if (stride < 0 || noise_stride < 0 || !sample_arg(args[2], *logits, at::kFloat, 0.0, std::numeric_limits<float>::max(), &temperature, &t0) ||
      !sample_arg(args[3], *logits, at::kInt, 1.0, std::numeric_limits<int32_t>::max(), &top_k, &k0) ||
      !sample_arg(args[4], *logits, at::kFloat, 0.0, 1.0, &top_p, &p0) || !sample_arg(args[5], *logits, at::kFloat, 0.0, 1.0, &min_p, &m0))
    return none();
  const at::IntArrayRef lead = logits->sizes().slice(0, logits->dim() - 1);
  const bool want = args[6] == Py_True;
  at::Tensor token = empty_on(*logits, lead, at::kLong), logprob;
  float* lp = nullptr;
  if (want) {
    logprob = empty_on(*logits, lead, at::kFloat);
    lp = logprob.mutable_data_ptr<float>();
  }
  const auto stream = c10::cuda::getCurrentCUDAStream(logits->get_device()).stream();
  int rc;
  {
    ThreadsRun unlocked;
    rc = triturus_b200_sample(logits->const_data_ptr(), noise->const_data_ptr<float>(), token.mutable_data_ptr<int64_t>(), lp, rows, symbols, stride,
                              noise_stride, type, static_cast<const float*>(temperature), static_cast<float>(t0),
                              static_cast<const int32_t*>(top_k), static_cast<int32_t>(k0), static_cast<const float*>(top_p),
                              static_cast<float>(p0), static_cast<const float*>(min_p), static_cast<float>(m0), stream);
  }
  if (rc != TRITURUS_B200_OK) return failed("triturus_b200_sample", rc);
  if (!want) return THPVariable_Wrap(std::move(token));
  PyObject* out = PyTuple_New(2);
  if (out == nullptr) return nullptr;
  PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(std::move(token)));
  PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(std::move(logprob)));
  return out;
  END_HANDLE_TH_ERRORS
}

// Symbols: 64- or 32-bit whole numbers, one after the other, on `like`'s device.
const at::Tensor* token_arg(PyObject* o, const at::Tensor& like) {
  const at::Tensor* t = plain_object(o);
  if (t == nullptr || (t->scalar_type() != at::kLong && t->scalar_type() != at::kInt)) return nullptr;
  return t->is_contiguous() && t->device() == like.device() ? t : nullptr;
}
// None (-1) or a symbol below `symbols`.
bool padding_arg(PyObject* o, int64_t symbols, int64_t* padding) {
  *padding = -1;
  if (o == Py_None) return true;
  if (!PyLong_CheckExact(o)) return false;
  *padding = PyLong_AsLongLong(o);
  if (*padding == -1 && PyErr_Occurred()) PyErr_Clear();
  return *padding >= 0 && *padding < symbols;
}
bool scale_arg(PyObject* o, float* scale) {
  if (!PyFloat_CheckExact(o)) return false;
  *scale = static_cast<float>(PyFloat_AS_DOUBLE(o));
  return std::isfinite(*scale);
}

// embedding(tokens, weight, scale, padding_idx)
PyObject* embedding(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  float scale;
  int64_t padding;
  if (nargs != 4 || !scale_arg(args[2], &scale) || !plain_mode()) return none();
  const at::Tensor* weight = plain_object(args[1]);
  if (weight == nullptr || weight->dim() != 2 || weight->get_device() != c10::cuda::current_device()) return none();
  const at::Tensor* tokens = token_arg(args[0], *weight);
  const int type = type_code(*weight);
  const int64_t stride = row_stride(*weight), symbols = weight->size(0), width = weight->size(1);
  if (tokens == nullptr || type < 0 || stride < 0 || !padding_arg(args[3], symbols, &padding) || has_tangent(weight)) return none();
  at::DimVector shape(tokens->sizes());
  shape.push_back(width);
  at::Tensor y = empty_on(*weight, shape, weight->scalar_type());
  const auto stream = c10::cuda::getCurrentCUDAStream(weight->get_device()).stream();
  int rc;
  {
    ThreadsRun unlocked;
    rc = triturus_b200_embedding(tokens->const_data_ptr(), static_cast<int>(tokens->element_size()), weight->const_data_ptr(), y.mutable_data_ptr(),
                                 tokens->numel(), symbols, width, stride, type, scale, stream);
  }
  if (rc != TRITURUS_B200_OK) return failed("triturus_b200_embedding", rc);
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// embedding_backward(dy, tokens, symbols, scale, padding_idx)
PyObject* embedding_backward(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  float scale;
  int64_t padding;
  if (nargs != 5 || !PyLong_CheckExact(args[2]) || !scale_arg(args[3], &scale) || !plain_mode()) return none();
  const int64_t symbols = PyLong_AsLongLong(args[2]);
  if (symbols == -1 && PyErr_Occurred()) PyErr_Clear();
  const at::Tensor* dy = plain_object(args[0]);
  if (symbols < 1 || dy == nullptr || dy->dim() < 1 || dy->get_device() != c10::cuda::current_device()) return none();
  const at::Tensor* tokens = token_arg(args[1], *dy);
  const int type = type_code(*dy);
  const int64_t stride = row_stride(*dy), width = dy->size(-1);
  if (tokens == nullptr || type < 0 || stride < 0 || tokens->sizes() != dy->sizes().slice(0, dy->dim() - 1) ||
      !padding_arg(args[4], symbols, &padding) || has_tangent(dy))
    return none();
  const int64_t count = tokens->numel();
  const size_t bytes = triturus_b200_embedding_backward_workspace_bytes(count, symbols, width, type);
  if (bytes == 0) return none();  // (sizes that the library refuses)
  at::Tensor dweight = empty_on(*dy, {symbols, width}, dy->scalar_type());
  at::Tensor ws = empty_on(*dy, {static_cast<int64_t>(bytes)}, at::kByte);
  const auto stream = c10::cuda::getCurrentCUDAStream(dy->get_device()).stream();
  int rc;
  {
    ThreadsRun unlocked;
    rc = triturus_b200_embedding_backward(dy->const_data_ptr(), tokens->const_data_ptr(), static_cast<int>(tokens->element_size()),
                                          dweight.mutable_data_ptr(), count, symbols, width, stride, type, scale, padding, ws.mutable_data_ptr(), bytes, stream);
  }
  if (rc != TRITURUS_B200_OK) return failed("triturus_b200_embedding_backward", rc);
  return THPVariable_Wrap(std::move(dweight));
  END_HANDLE_TH_ERRORS
}

// The operands of the cross entropy: x [..., D], weight [V, D] of its type, targets of x's leading shape.
struct EntropyOperands {
  const at::Tensor *x, *weight, *target;
  int64_t rows, symbols, width, x_stride, weight_stride;
  int type;
};
bool entropy_operands(PyObject* const* args, EntropyOperands* o) {
  o->x = plain_object(args[0]);
  o->weight = o->x != nullptr ? plain_object(args[1]) : nullptr;
  if (o->weight == nullptr || o->x->dim() < 1 || o->weight->dim() != 2 || o->x->get_device() != c10::cuda::current_device()) return false;
  o->target = token_arg(args[2], *o->x);
  o->type = type_code(*o->x);
  o->width = o->x->size(-1);
  if (o->target == nullptr || o->type < 0 || o->weight->scalar_type() != o->x->scalar_type() || o->weight->device() != o->x->device() ||
      o->weight->size(1) != o->width || o->target->sizes() != o->x->sizes().slice(0, o->x->dim() - 1))
    return false;
  o->rows = o->target->numel();
  o->symbols = o->weight->size(0);
  o->x_stride = row_stride(*o->x);
  o->weight_stride = row_stride(*o->weight);
  return o->x_stride >= 0 && o->weight_stride >= 0 && !has_tangent(o->x) && !has_tangent(o->weight);
}
bool int64_arg(PyObject* o, int64_t* v) {
  if (!PyLong_CheckExact(o)) return false;
  *v = PyLong_AsLongLong(o);
  if (*v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return true;
}
PyObject* tuple2(at::Tensor* a, at::Tensor* b) {
  PyObject* out = PyTuple_New(2);
  if (out == nullptr) return nullptr;
  at::Tensor* all[2] = {a, b};
  for (int i = 0; i < 2; ++i) PyTuple_SET_ITEM(out, i, all[i] != nullptr ? THPVariable_Wrap(std::move(*all[i])) : Py_NewRef(Py_None));
  return out;
}

// linear_cross_entropy(x, weight, target, reduction, ignore_index, status) -> (loss, lse); status: address of the device's status word
PyObject* linear_cross_entropy(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  int reduction;
  int64_t ignore, status;
  EntropyOperands o;
  if (nargs != 6 || !int_arg(args[3], &reduction) || !int64_arg(args[4], &ignore) || !int64_arg(args[5], &status) || !plain_mode() ||
      !entropy_operands(args, &o))
    return none();
  at::Tensor lse = empty_on(*o.x, o.target->sizes(), at::kFloat);
  at::Tensor loss = empty_on(*o.x, reduction == TRITURUS_B200_REDUCTION_NONE ? o.target->sizes() : at::IntArrayRef(), at::kFloat);
  const void *xp = o.x->const_data_ptr(), *wp = o.weight->const_data_ptr();
  const size_t bytes = triturus_b200_linear_cross_entropy_workspace_bytes(xp, wp, o.rows, o.symbols, o.width, o.x_stride, o.weight_stride, o.type);
  if (bytes == 0) return none();  // (sizes that the library refuses)
  at::Tensor ws = empty_on(*o.x, {static_cast<int64_t>(bytes)}, at::kByte);
  const auto stream = c10::cuda::getCurrentCUDAStream(o.x->get_device()).stream();
  int rc;
  {
    ThreadsRun unlocked;
    rc = triturus_b200_linear_cross_entropy(xp, wp, o.target->const_data_ptr(), static_cast<int>(o.target->element_size()), loss.mutable_data_ptr<float>(),
                                            lse.mutable_data_ptr<float>(), o.rows, o.symbols, o.width, o.x_stride, o.weight_stride, o.type, reduction, ignore,
                                            ws.mutable_data_ptr(), bytes, reinterpret_cast<int32_t*>(status), stream);
  }
  if (rc != TRITURUS_B200_OK) return failed("triturus_b200_linear_cross_entropy", rc);
  return tuple2(&loss, &lse);
  END_HANDLE_TH_ERRORS
}

// linear_cross_entropy_backward(x, weight, target, dloss, lse, reduction, ignore_index, x_grad, weight_grad, status) -> (dx or None, dweight or None)
PyObject* linear_cross_entropy_backward(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  int reduction;
  int64_t ignore, status;
  EntropyOperands o;
  if (nargs != 10 || !int_arg(args[5], &reduction) || !int64_arg(args[6], &ignore) || !PyBool_Check(args[7]) || !PyBool_Check(args[8]) ||
      !int64_arg(args[9], &status) || !plain_mode() || !entropy_operands(args, &o))
    return none();
  const at::Tensor* dloss = plain_object(args[3]);
  const at::Tensor* lse = plain_object(args[4]);
  if (dloss == nullptr || lse == nullptr) return none();
  for (const at::Tensor* t : {dloss, lse})
    if (t->scalar_type() != at::kFloat || !t->is_contiguous() || t->device() != o.x->device() || has_tangent(t)) return none();
  if (lse->sizes() != o.target->sizes() || dloss->sizes() != (reduction == TRITURUS_B200_REDUCTION_NONE ? o.target->sizes() : at::IntArrayRef())) return none();
  const bool want_x = args[7] == Py_True, want_weight = args[8] == Py_True;
  at::Tensor dx, dweight;
  if (want_x) dx = empty_on(*o.x, o.x->sizes(), o.x->scalar_type());
  if (want_weight) dweight = empty_on(*o.x, o.weight->sizes(), o.x->scalar_type());
  const void *xp = o.x->const_data_ptr(), *wp = o.weight->const_data_ptr();
  const size_t bytes = triturus_b200_linear_cross_entropy_backward_workspace_bytes(xp, wp, o.rows, o.symbols, o.width, o.x_stride, o.weight_stride, o.type);
  if (bytes == 0) return none();
  at::Tensor ws = empty_on(*o.x, {static_cast<int64_t>(bytes)}, at::kByte);
  const auto stream = c10::cuda::getCurrentCUDAStream(o.x->get_device()).stream();
  int rc;
  {
    ThreadsRun unlocked;
    rc = triturus_b200_linear_cross_entropy_backward(
        dloss->const_data_ptr<float>(), xp, wp, o.target->const_data_ptr(), static_cast<int>(o.target->element_size()), lse->const_data_ptr<float>(),
        want_x ? dx.mutable_data_ptr() : nullptr, want_weight ? dweight.mutable_data_ptr() : nullptr, o.rows, o.symbols, o.width, o.x_stride, o.weight_stride,
        o.type, reduction, ignore, ws.mutable_data_ptr(), bytes, reinterpret_cast<int32_t*>(status), stream);
  }
  if (rc != TRITURUS_B200_OK) return failed("triturus_b200_linear_cross_entropy_backward", rc);
  return tuple2(want_x ? &dx : nullptr, want_weight ? &dweight : nullptr);
  END_HANDLE_TH_ERRORS
}

// set_up(error_class, copy_flop_rows, copy_flop_strided)
PyObject* set_up(PyObject*, PyObject* args) {
  PyObject* cls;
  if (!PyArg_ParseTuple(args, "Odd", &cls, &copy_flop_rows, &copy_flop_strided)) return nullptr;
  Py_XDECREF(error_class);
  error_class = Py_NewRef(cls);
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"set_up", set_up, METH_VARARGS, "set_up(error_class, copy_flop_rows, copy_flop_strided)"},
    {"lm2exp", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(lm2exp)), METH_FASTCALL, "lm2exp(a, b, precision, variant) -> Tensor or None"},
    {"lt2exp", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(lt2exp)), METH_FASTCALL, "lt2exp(w, a, b, precision, variant) -> Tensor or None"},
    {"layer_norm", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(layer_norm)), METH_FASTCALL,
     "layer_norm(x, weight, bias, eps, return_stats) -> Tensor, tuple or None"},
    {"layer_norm_backward", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(layer_norm_backward)), METH_FASTCALL,
     "layer_norm_backward(dy, x, mean, rstd, weight, weight_grad, bias_grad) -> tuple or None"},
    {"clip_grad_norm", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(clip_grad_norm)), METH_FASTCALL,
     "clip_grad_norm(grads, max_norm, norm_type, scale) -> Tensor or None"},
    {"sample", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(sample)), METH_FASTCALL,
     "sample(logits, noise, temperature, top_k, top_p, min_p, return_logprob) -> Tensor, tuple or None"},
    {"embedding", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(embedding)), METH_FASTCALL,
     "embedding(tokens, weight, scale, padding_idx) -> Tensor or None"},
    {"embedding_backward", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(embedding_backward)), METH_FASTCALL,
     "embedding_backward(dy, tokens, symbols, scale, padding_idx) -> Tensor or None"},
    {"linear_cross_entropy", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(linear_cross_entropy)), METH_FASTCALL,
     "linear_cross_entropy(x, weight, target, reduction, ignore_index, status) -> tuple or None"},
    {"linear_cross_entropy_backward", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(linear_cross_entropy_backward)), METH_FASTCALL,
     "linear_cross_entropy_backward(x, weight, target, dloss, lse, reduction, ignore_index, x_grad, weight_grad, status) -> tuple or None"},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", "Small calls of triturus_b200 from C++.", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host() { return PyModule_Create(&module); }
