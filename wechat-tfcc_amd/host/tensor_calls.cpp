// CPython module behind the operators of the package on torch tensors: the plain case of each - contiguous tensors of
// the documented types on the current device - from the Python call to the launch without going back to Python.  A
// small operator is bound by that way, not by the GPU: through ctypes a call cost 11 us of which the launch is 3.
// Every function returns None for what it leaves to the Python form of the operator (other layouts and ranks, batches,
// mismatches and whatever the library refuses), which carries the checks and raises the errors.
#include <Python.h>

#include <ATen/Functions.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <limits>

#include "tfcc_rocm.h"

namespace {

using at::Tensor;

// The caller keeps the reference; nullptr: not a tensor this module takes (one without memory of its own, as inside
// torch.func transforms, is none).
const Tensor* plain(PyObject* o, at::ScalarType type, c10::DeviceIndex device) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda() || !t.has_storage() || t.layout() != at::kStrided || t.scalar_type() != type || t.get_device() != device || !t.is_contiguous()) return nullptr;
  return &t;
}

const Tensor* plain_scalar(PyObject* o, c10::DeviceIndex device) {
  const Tensor* t = plain(o, at::kFloat, device);
  return t && t->dim() == 1 && t->numel() == 1 ? t : nullptr;
}

Tensor empty(at::IntArrayRef shape, at::ScalarType type, c10::DeviceIndex device) {
  return at::detail::empty_cuda(shape, type, c10::Device(c10::kCUDA, device), std::nullopt);
}

// The two ends of a range: two tensors over one allocation.  Taking and giving back the second was 0.3 us of a call that the host bounds:
// quantize of 1 x 64 4.8 -> 4.5 us, 1 x 64 x 64 product 5.0 -> 4.7; the four calls of a quantized layer gain 1.5 to 2 % (24.8 -> 24.4, 21 -> 20.4).
struct Range {
  Tensor low, high;
  explicit Range(c10::DeviceIndex device) : low(empty({2}, at::kFloat, device)) {
    high = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(low.storage()), c10::DispatchKeySet(c10::DispatchKey::CUDA), low.dtype());
    high.unsafeGetTensorImpl()->set_storage_offset(1);
    high.unsafeGetTensorImpl()->set_sizes_contiguous({1});
    low.unsafeGetTensorImpl()->set_sizes_contiguous({1});
  }
};

template <class T = void>
T* data(const Tensor* t) { return t ? static_cast<T*>(t->unsafeGetTensorImpl()->mutable_data()) : nullptr; }
template <class T = void>
T* data(const Tensor& t) { return data<T>(&t); }

bool fits(int64_t v) { return v > 0 && v <= 0x7fffffff; }

// the device of the first operand, where that is the current one; -1 (which no GPU tensor has) otherwise
struct Here {
  c10::DeviceIndex device = -1;
  explicit Here(PyObject* first) {
    if (!THPVariable_CheckExact(first) || !THPVariable_Unpack(first).is_cuda()) return;
    const c10::DeviceIndex d = THPVariable_Unpack(first).get_device();
    if (d == c10::hip::current_device()) device = d;
  }
  void* stream() const { return c10::hip::getCurrentHIPStream(device).stream(); }
};

// The launch itself runs without the interpreter lock, as through ctypes.  What is thrown on the way - a data pointer
// that cannot be had, memory of the library's own bookkeeping - becomes a Python error only with the lock held again.
struct Unlocked {
  PyThreadState* state = PyEval_SaveThread();
  ~Unlocked() { PyEval_RestoreThread(state); }
};
template <class F>
int launch(F&& f) {
  Unlocked unlocked;
  return f();
}

PyObject* wrap(Tensor t) { return THPVariable_Wrap(std::move(t)); }

PyObject* pack(std::initializer_list<PyObject*> items) {
  PyObject* r = PyTuple_New(static_cast<Py_ssize_t>(items.size()));
  Py_ssize_t i = 0;
  for (PyObject* o : items) {
    if (o == nullptr) {
      for (PyObject* p : items) Py_XDECREF(p);
      Py_XDECREF(r);
      return nullptr;
    }
    ++i;
  }
  if (r == nullptr) return nullptr;
  i = 0;
  for (PyObject* o : items) PyTuple_SET_ITEM(r, i++, o);
  return r;
}

PyObject* none() { Py_RETURN_NONE; }

// blas_matmul(a, b, bias or None)
PyObject* blas_matmul(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 3) return none();
  Here here(args[0]);
  const Tensor* a = plain(args[0], at::kFloat, here.device);
  const Tensor* b = plain(args[1], at::kFloat, here.device);
  const Tensor* bias = args[2] == Py_None ? nullptr : plain(args[2], at::kFloat, here.device);
  if (!a || !b || (args[2] != Py_None && !bias)) return none();
  const int64_t ra = a->dim(), rb = b->dim();
  if (ra < 2 || (rb != 2 && rb != ra)) return none();
  const int64_t m = a->size(ra - 2), k = a->size(ra - 1), cols = b->size(rb - 1);
  if (b->size(rb - 2) != k || (bias && (bias->dim() != 1 || bias->size(0) != cols))) return none();
  if (a->numel() == 0 || b->numel() == 0) return none();
  int64_t batch = 1;
  at::DimVector shape(a->sizes().begin(), a->sizes().end());
  for (int64_t i = 0; i + 2 < ra; ++i) {
    if (rb != 2 && b->size(i) != a->size(i)) return none();
    batch *= a->size(i);
  }
  if (!fits(m) || !fits(k) || !fits(cols) || !fits(batch)) return none();
  shape[ra - 1] = cols;
  Tensor out = empty(shape, at::kFloat, here.device);
  const uint64_t sa = ra == 2 && rb != 2 ? 0 : static_cast<uint64_t>(m) * k, sb = rb == 2 && ra != 2 ? 0 : static_cast<uint64_t>(k) * cols;
  void* stream = here.stream();
  if (launch([&] {
        return tfcc_rocm_sgemm_strided_batched(stream, data<float>(a), sa, data<float>(b), sb, data<float>(bias), data<float>(out),
                                               static_cast<uint64_t>(m) * cols, static_cast<unsigned>(m), static_cast<unsigned>(cols),
                                               static_cast<unsigned>(k), static_cast<unsigned>(batch));
      }) != TFCC_ROCM_OK)
    return none();
  return wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// reduce_sum(a, row)
PyObject* reduce_sum(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 2 || !THPVariable_CheckExact(args[0]) || !PyBool_Check(args[1])) return none();
  Here here(args[0]);
  const at::ScalarType type = THPVariable_Unpack(args[0]).scalar_type();
  if (type != at::kByte && type != at::kChar) return none();
  const Tensor* a = plain(args[0], type, here.device);
  if (!a || a->dim() != 2 || !fits(a->size(0)) || !fits(a->size(1))) return none();
  const bool row = args[1] == Py_True;
  const unsigned r = static_cast<unsigned>(a->size(0)), c = static_cast<unsigned>(a->size(1));
  Tensor out = empty({row ? a->size(0) : a->size(1)}, at::kInt, here.device);
  void* stream = here.stream();
  const int code = type == at::kByte ? TFCC_ROCM_U8 : TFCC_ROCM_S8;
  if (launch([&] {
        return (row ? tfcc_rocm_reduce_sum_rows : tfcc_rocm_reduce_sum_cols)(stream, data(a), code, 1, r, c, data<int32_t>(out));
      }) != TFCC_ROCM_OK)
    return none();
  return wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// The descriptor of a 2-D quantized product from the eight leading arguments of both forms below; false: not plain.
bool describe(PyObject* const* args, const Here& here, tfcc_rocm_qgemm_desc& d) {
  const Tensor* a = plain(args[0], at::kByte, here.device);
  const Tensor* ra = plain(args[1], at::kInt, here.device);
  const Tensor *minA = plain_scalar(args[2], here.device), *maxA = plain_scalar(args[3], here.device);
  const Tensor* b = plain(args[4], at::kChar, here.device);
  const Tensor* rb = plain(args[5], at::kInt, here.device);
  const Tensor *minB = plain_scalar(args[6], here.device), *maxB = plain_scalar(args[7], here.device);
  if (!a || !ra || !minA || !maxA || !b || !rb || !minB || !maxB) return false;
  if (a->dim() != 2 || b->dim() != 2 || ra->dim() != 1 || rb->dim() != 1) return false;
  const int64_t m = a->size(0), k = a->size(1), n = b->size(1);
  if (!fits(m) || !fits(k) || !fits(n) || b->size(0) != k || ra->size(0) != m || rb->size(0) != n) return false;
  d.a = data<uint8_t>(a);
  d.b = data<int8_t>(b);
  d.rowsum_a = data<int32_t>(ra);
  d.colsum_b = data<int32_t>(rb);
  d.stride_c = static_cast<uint64_t>(m) * n;
  d.m = static_cast<unsigned>(m);
  d.n = static_cast<unsigned>(n);
  d.k = static_cast<unsigned>(k);
  d.batch = 1;
  d.min_a = data<float>(minA);
  d.max_a = data<float>(maxA);
  d.min_b = data<float>(minB);
  d.max_b = data<float>(maxB);
  return true;
}

// quantization_matmul(a, reduce_a, min_a, max_a, b, reduce_b, min_b, max_b)
PyObject* quantization_matmul(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 8) return none();
  Here here(args[0]);
  tfcc_rocm_qgemm_desc d{};
  if (!describe(args, here, d)) return none();
  Tensor c = empty({d.m, d.n}, at::kInt, here.device);
  Range range(here.device);
  d.min_c = data<float>(range.low);
  d.max_c = data<float>(range.high);
  void* stream = here.stream();
  if (launch([&] { return tfcc_rocm_gemm_u8s8s32(stream, &d, data<int32_t>(c)); }) != TFCC_ROCM_OK) return none();
  return pack({wrap(std::move(c)), wrap(std::move(range.low)), wrap(std::move(range.high))});
  END_HANDLE_TH_ERRORS
}

// quantization_matmul_requantize(... the eight above, min_out, max_out, want_acc, colsum_exact)
PyObject* quantization_matmul_requantize(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 12 || !PyBool_Check(args[10]) || !PyBool_Check(args[11])) return none();
  Here here(args[0]);
  tfcc_rocm_qgemm_desc d{};
  if (!describe(args, here, d)) return none();
  const Tensor *minOut = plain_scalar(args[8], here.device), *maxOut = plain_scalar(args[9], here.device);
  if (!minOut || !maxOut) return none();
  Tensor q = empty({d.m, d.n}, at::kByte, here.device), c;
  Range range(here.device);
  if (args[10] == Py_True) c = empty({d.m, d.n}, at::kInt, here.device);
  d.min_c = data<float>(range.low);
  d.max_c = data<float>(range.high);
  d.colsum_b_is_exact = args[11] == Py_True ? 1 : 0;
  void* stream = here.stream();
  if (launch([&] {
        return tfcc_rocm_gemm_u8s8s32_requant_u8(stream, &d, c.defined() ? data<int32_t>(c) : nullptr, data<uint8_t>(q), 0.0, 0.0, 0.0, 0,
                                                 data<float>(minOut), data<float>(maxOut));
      }) != TFCC_ROCM_OK)
    return none();
  PyObject* acc = c.defined() ? wrap(std::move(c)) : none();
  return pack({wrap(std::move(q)), acc, wrap(std::move(range.low)), wrap(std::move(range.high))});
  END_HANDLE_TH_ERRORS
}

struct Skinny {
  const Tensor *a, *ra, *rb, *scale;
  int32_t offsetA, offsetB;
  float scaleA;
};

bool skinny_offsets(PyObject* oa, PyObject* ob, PyObject* sa, Skinny& s) {
  if (!PyLong_CheckExact(oa) || !PyLong_CheckExact(ob) || !PyFloat_CheckExact(sa)) return false;
  int overflow = 0;
  const long long x = PyLong_AsLongLongAndOverflow(oa, &overflow);
  if (overflow || x < INT32_MIN || x > INT32_MAX) return false;
  const long long y = PyLong_AsLongLongAndOverflow(ob, &overflow);
  if (overflow || y < INT32_MIN || y > INT32_MAX) return false;
  s.offsetA = static_cast<int32_t>(x);
  s.offsetB = static_cast<int32_t>(y);
  s.scaleA = static_cast<float>(PyFloat_AS_DOUBLE(sa));
  return true;
}

bool skinny_tensors(PyObject* a, PyObject* ra, PyObject* rb, PyObject* scale, const Here& here, Skinny& s) {
  s.a = plain(a, at::kByte, here.device);
  s.ra = plain(ra, at::kInt, here.device);
  s.rb = plain(rb, at::kInt, here.device);
  s.scale = plain(scale, at::kFloat, here.device);
  return s.a && s.ra && s.rb && s.scale && s.a->dim() == 2 && fits(s.a->size(0)) && fits(s.a->size(1)) && s.ra->numel() >= s.a->size(0);
}

// gemv_dequant(a, b, reduce_a, reduce_b, offset_a, offset_b, scale_a, scale_b, want_acc, colsum_exact)
PyObject* gemv_dequant(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 10 || !PyBool_Check(args[8]) || !PyBool_Check(args[9])) return none();
  Here here(args[0]);
  Skinny s;
  const Tensor* b = plain(args[1], at::kChar, here.device);
  if (!b || b->dim() != 2 || !skinny_tensors(args[0], args[2], args[3], args[7], here, s) || !skinny_offsets(args[4], args[5], args[6], s)) return none();
  const int64_t m = s.a->size(0), k = s.a->size(1), cols = b->size(1);
  if (b->size(0) != k || !fits(cols) || s.rb->numel() < cols || s.scale->numel() < cols) return none();
  Tensor acc, out = empty({m, cols}, at::kFloat, here.device);
  if (args[8] == Py_True) acc = empty({m, cols}, at::kInt, here.device);
  void* stream = here.stream();
  const unsigned flags = args[9] == Py_True ? TFCC_ROCM_GEMV_COLSUM_B_IS_EXACT : 0;
  if (launch([&] {
        return tfcc_rocm_gemv_u8s8s32_flags(stream, data<uint8_t>(s.a), data<int8_t>(b), data<int32_t>(s.ra), data<int32_t>(s.rb), s.offsetA,
                                            s.offsetB, static_cast<unsigned>(m), static_cast<unsigned>(cols), static_cast<unsigned>(k),
                                            acc.defined() ? data<int32_t>(acc) : nullptr, s.scaleA, data<float>(s.scale), data<float>(out), flags);
      }) != TFCC_ROCM_OK)
    return none();
  PyObject* accObject = acc.defined() ? wrap(std::move(acc)) : none();
  return pack({wrap(std::move(out)), accObject});
  END_HANDLE_TH_ERRORS
}

// gemv_dequant_packed(a, packed, n, reduce_a, reduce_b, offset_a, offset_b, scale_a, scale_b, want_acc)
PyObject* gemv_dequant_packed(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 10 || !PyBool_Check(args[9]) || !PyLong_CheckExact(args[2])) return none();
  Here here(args[0]);
  Skinny s;
  const Tensor* packed = plain(args[1], at::kByte, here.device);
  int overflow = 0;
  const long long cols = PyLong_AsLongLongAndOverflow(args[2], &overflow);
  if (overflow || !fits(cols) || !packed || !skinny_tensors(args[0], args[3], args[4], args[8], here, s) ||
      !skinny_offsets(args[5], args[6], args[7], s))
    return none();
  const int64_t m = s.a->size(0), k = s.a->size(1);
  if (s.rb->numel() < cols || s.scale->numel() < cols ||
      static_cast<size_t>(packed->numel()) < tfcc_rocm_gemv_packed_size(static_cast<unsigned>(cols), static_cast<unsigned>(k)))
    return none();
  Tensor acc, out = empty({m, cols}, at::kFloat, here.device);
  if (args[9] == Py_True) acc = empty({m, cols}, at::kInt, here.device);
  void* stream = here.stream();
  if (launch([&] {
        return tfcc_rocm_gemv_u8s8s32_packed(stream, data<uint8_t>(s.a), data(packed), data<int32_t>(s.ra), data<int32_t>(s.rb), s.offsetA,
                                             s.offsetB, static_cast<unsigned>(m), static_cast<unsigned>(cols), static_cast<unsigned>(k),
                                             acc.defined() ? data<int32_t>(acc) : nullptr, s.scaleA, data<float>(s.scale), data<float>(out));
      }) != TFCC_ROCM_OK)
    return none();
  PyObject* accObject = acc.defined() ? wrap(std::move(acc)) : none();
  return pack({wrap(std::move(out)), accObject});
  END_HANDLE_TH_ERRORS
}

// -1: a type the quantization kernels do not take
int quantized_code(at::ScalarType t) {
  switch (t) {
    case at::kChar: return TFCC_ROCM_S8;
    case at::kByte: return TFCC_ROCM_U8;
    case at::kShort: return TFCC_ROCM_S16;
    case at::kInt: return TFCC_ROCM_S32;
    default: return -1;
  }
}

// quantize(a, out_dtype): the form that takes the range from the data
PyObject* quantize(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 2 || !THPDtype_Check(args[1])) return none();
  Here here(args[0]);
  const at::ScalarType type = reinterpret_cast<THPDtype*>(args[1])->scalar_type;
  const int code = quantized_code(type);
  const Tensor* a = plain(args[0], at::kFloat, here.device);
  if (!a || code < 0 || a->numel() == 0) return none();
  Tensor out = empty(a->sizes(), type, here.device);
  Range range(here.device);
  void* stream = here.stream();
  if (launch([&] {
        return tfcc_rocm_quantize_minmax(stream, data<float>(a), static_cast<uint64_t>(a->numel()), data(out), code, data<float>(range.low),
                                         data<float>(range.high));
      }) != TFCC_ROCM_OK)
    return none();
  return pack({wrap(std::move(out)), wrap(std::move(range.low)), wrap(std::move(range.high))});
  END_HANDLE_TH_ERRORS
}

// dequantize(a, min, max)
PyObject* dequantize(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 3 || !THPVariable_CheckExact(args[0])) return none();
  Here here(args[0]);
  const at::ScalarType type = THPVariable_Unpack(args[0]).scalar_type();
  const int code = quantized_code(type);
  if (code < 0) return none();
  const Tensor* a = plain(args[0], type, here.device);
  const Tensor *lo = plain_scalar(args[1], here.device), *hi = plain_scalar(args[2], here.device);
  if (!a || !lo || !hi || a->numel() == 0) return none();
  Tensor out = empty(a->sizes(), at::kFloat, here.device);
  void* stream = here.stream();
  if (launch([&] {
        return tfcc_rocm_dequantize(stream, data(a), code, static_cast<uint64_t>(a->numel()), data<float>(lo), data<float>(hi), data<float>(out));
      }) != TFCC_ROCM_OK)
    return none();
  return wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// A tensor as above but for its strides, of which the last is one.
const Tensor* rows_of(PyObject* o, at::ScalarType type, int64_t dims, c10::DeviceIndex device) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda() || !t.has_storage() || t.layout() != at::kStrided || t.scalar_type() != type || t.get_device() != device || t.is_neg()) return nullptr;
  return t.dim() == dims && t.numel() > 0 && t.numel() <= INT32_MAX * int64_t{256} && t.stride(dims - 1) == 1 ? &t : nullptr;
}

// int32 or int64 [count]; the type's code, -1: neither
int integers(PyObject* o, int64_t count, c10::DeviceIndex device, const Tensor** t) {
  for (const auto& [type, code] : {std::pair{at::kInt, TFCC_ROCM_S32}, std::pair{at::kLong, TFCC_ROCM_S64}})
    if ((*t = plain(o, type, device)) != nullptr) return (*t)->dim() == 1 && (*t)->numel() == count ? code : -1;
  return -1;
}

bool number(PyObject* o, int64_t* v) {
  if (!PyLong_CheckExact(o)) return false;
  int overflow = 0;
  const long long x = PyLong_AsLongLongAndOverflow(o, &overflow);
  *v = x;
  return !overflow && x >= 0 && x <= INT32_MAX;
}

// The memory of a paged cache: a tuple of two tensors of float32, or of two of int8, or of uint8 with two integers of 4 bits in each, and two of scales.
bool cache_of(PyObject* o, c10::DeviceIndex device, tfcc_rocm_paged_cache& c) {
  if (!PyTuple_CheckExact(o)) return false;
  const Py_ssize_t n = PyTuple_GET_SIZE(o);
  if (n != 2 && n != 4) return false;
  at::ScalarType type = n == 4 ? at::kChar : at::kFloat;
  const Tensor* keys = rows_of(PyTuple_GET_ITEM(o, 0), type, 4, device);
  if (!keys && n == 4) keys = rows_of(PyTuple_GET_ITEM(o, 0), type = at::kByte, 4, device);
  const Tensor* values = rows_of(PyTuple_GET_ITEM(o, 1), type, 4, device);
  if (!keys || !values || keys->sizes() != values->sizes() || keys->strides() != values->strides()) return false;
  if (!fits(keys->size(0)) || !fits(keys->size(1)) || !fits(keys->size(2)) || !fits(keys->size(3))) return false;
  c.keys = data(keys);
  c.values = data(values);
  c.type = type == at::kChar ? TFCC_ROCM_S8 : type == at::kByte ? TFCC_ROCM_S4 : TFCC_ROCM_F32;
  c.pages = static_cast<unsigned>(keys->size(0));
  c.heads = static_cast<unsigned>(keys->size(1));
  c.page_size = static_cast<unsigned>(keys->size(2));
  c.size = static_cast<unsigned>(keys->size(3));
  if (type == at::kByte) {
    if (c.size > 1024) return false;
    c.size *= 2;
  }
  c.page_stride = keys->stride(0);
  c.head_stride = keys->stride(1);
  c.row_stride = keys->stride(2);
  if (n == 2) return true;
  const Tensor* key_scales = plain(PyTuple_GET_ITEM(o, 2), at::kFloat, device);
  const Tensor* value_scales = plain(PyTuple_GET_ITEM(o, 3), at::kFloat, device);
  if (!key_scales || !value_scales || key_scales->dim() != 3 || value_scales->sizes() != key_scales->sizes() ||
      key_scales->sizes() != keys->sizes().slice(0, 3) || key_scales->strides() != value_scales->strides())
    return false;
  c.key_scales = data<float>(key_scales);
  c.value_scales = data<float>(value_scales);
  c.scale_page_stride = key_scales->stride(0);
  c.scale_head_stride = key_scales->stride(1);
  c.scale_row_stride = key_scales->stride(2);
  return true;
}

// rotary(q, k or None, positions, frequencies, interleaved, magnitude)
PyObject* rotary(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 6 || !PyBool_Check(args[4]) || !PyFloat_CheckExact(args[5])) return none();
  Here here(args[0]);
  const Tensor* in[2] = {rows_of(args[0], at::kFloat, 3, here.device), nullptr};
  const Tensor *positions, *frequencies = plain(args[3], at::kDouble, here.device);
  if (!in[0] || !frequencies || frequencies->dim() != 1) return none();
  const int64_t tokens = in[0]->size(0), size = in[0]->size(2), half = frequencies->size(0);
  if (args[1] != Py_None) {
    in[1] = rows_of(args[1], at::kFloat, 3, here.device);
    if (!in[1] || in[1]->size(0) != tokens || in[1]->size(2) != size) return none();
  }
  tfcc_rocm_rotary_desc d{};
  d.position_type = integers(args[2], tokens, here.device, &positions);
  if (d.position_type < 0 || half < 1 || half > size / 2 || !fits(tokens) || !fits(size)) return none();
  Tensor out[2];
  for (int i = 0; i < 2 && in[i]; ++i) {
    if (!fits(in[i]->size(1))) return none();
    out[i] = empty(in[i]->sizes(), at::kFloat, here.device);
    d.in[i] = data<float>(in[i]);
    d.out[i] = data<float>(out[i]);
    d.heads[i] = static_cast<unsigned>(in[i]->size(1));
    d.in_token_stride[i] = in[i]->stride(0);
    d.in_head_stride[i] = in[i]->stride(1);
    d.out_token_stride[i] = static_cast<uint64_t>(in[i]->size(1)) * size;
    d.out_head_stride[i] = size;
  }
  d.tokens = static_cast<unsigned>(tokens);
  d.size = static_cast<unsigned>(size);
  d.part = static_cast<unsigned>(2 * half);
  d.positions = data(positions);
  d.frequencies = data<double>(frequencies);
  d.magnitude = static_cast<float>(PyFloat_AS_DOUBLE(args[5]));
  d.interleaved = args[4] == Py_True ? 1 : 0;
  void* stream = here.stream();
  if (launch([&] { return tfcc_rocm_rotary_f32(stream, &d); }) != TFCC_ROCM_OK) return none();
  PyObject* second = in[1] ? wrap(std::move(out[1])) : none();
  return pack({wrap(std::move(out[0])), second});
  END_HANDLE_TH_ERRORS
}

// cache_write(cache, keys, values, slots): True where it was done
PyObject* cache_write(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 4) return none();
  Here here(args[1]);
  tfcc_rocm_paged_cache c{};
  const Tensor* keys = rows_of(args[1], at::kFloat, 3, here.device);
  const Tensor* values = rows_of(args[2], at::kFloat, 3, here.device);
  if (!keys || !values || keys->sizes() != values->sizes() || !cache_of(args[0], here.device, c)) return none();
  if (keys->size(1) != c.heads || keys->size(2) != c.size || !fits(keys->size(0))) return none();
  const Tensor* slots;
  const int type = integers(args[3], keys->size(0), here.device, &slots);
  if (type < 0) return none();
  void* stream = here.stream();
  if (launch([&] {
        return tfcc_rocm_cache_write(stream, &c, data<float>(keys), keys->stride(0), keys->stride(1), data<float>(values), values->stride(0),
                                     values->stride(1), static_cast<unsigned>(keys->size(0)), data(slots), type);
      }) != TFCC_ROCM_OK)
    return none();
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// cache_read(cache, table, starts, tokens)
PyObject* cache_read(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 4) return none();
  Here here(args[1]);
  tfcc_rocm_paged_cache c{};
  const Tensor* table = rows_of(args[1], at::kInt, 2, here.device);
  const Tensor* starts = plain(args[2], at::kInt, here.device);
  int64_t tokens;
  if (!table || !starts || !number(args[3], &tokens) || tokens == 0 || !cache_of(args[0], here.device, c)) return none();
  if (starts->dim() != 1 || starts->size(0) != table->size(0) + 1 || !fits(table->size(0)) || !fits(table->size(1))) return none();
  Tensor keys = empty({tokens, c.heads, c.size}, at::kFloat, here.device), values = empty({tokens, c.heads, c.size}, at::kFloat, here.device);
  void* stream = here.stream();
  if (launch([&] {
        return tfcc_rocm_cache_read(stream, &c, data<int32_t>(table), table->stride(0), static_cast<unsigned>(table->size(1)),
                                    static_cast<unsigned>(table->size(0)), data<int32_t>(starts), static_cast<unsigned>(tokens),
                                    data<float>(keys), data<float>(values));
      }) != TFCC_ROCM_OK)
    return none();
  return pack({wrap(std::move(keys)), wrap(std::move(values))});
  END_HANDLE_TH_ERRORS
}

// cache_copy(cache, sources, destinations, rows or None): True where it was done
PyObject* cache_copy(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 4 || !THPVariable_CheckExact(args[1])) return none();
  Here here(args[1]);
  tfcc_rocm_paged_cache c{};
  const int64_t runs = THPVariable_Unpack(args[1]).numel();
  const Tensor *sources, *destinations, *rows = args[3] == Py_None ? nullptr : plain(args[3], at::kInt, here.device);
  const int type = integers(args[1], runs, here.device, &sources);
  if (type < 0 || integers(args[2], runs, here.device, &destinations) != type || !fits(runs) || !cache_of(args[0], here.device, c)) return none();
  if (args[3] != Py_None && (!rows || rows->dim() != 1 || rows->size(0) != runs)) return none();
  void* stream = here.stream();
  if (launch([&] { return tfcc_rocm_cache_copy(stream, &c, data(sources), data(destinations), type, data<int32_t>(rows), static_cast<unsigned>(runs)); }) != TFCC_ROCM_OK)
    return none();
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// paged_attention(q, cache, table, starts, lengths, scale, causal, window, max_length, cap, slopes or None, prefixes or None)
PyObject* paged_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 12 || !PyFloat_CheckExact(args[5]) || !PyBool_Check(args[6]) || !PyFloat_CheckExact(args[9])) return none();
  Here here(args[0]);
  tfcc_rocm_paged_attention_desc d{};
  const Tensor* q = rows_of(args[0], at::kFloat, 3, here.device);
  const Tensor* table = rows_of(args[2], at::kInt, 2, here.device);
  const Tensor *starts = plain(args[3], at::kInt, here.device), *lengths = plain(args[4], at::kInt, here.device);
  int64_t window, most;
  if (!q || !table || !starts || !lengths || !number(args[7], &window) || !number(args[8], &most) || !cache_of(args[1], here.device, d.cache)) return none();
  const int64_t batch = table->size(0);
  if (lengths->dim() != 1 || lengths->size(0) != batch || starts->dim() != 1 || starts->size(0) != batch + 1) return none();
  if (!fits(q->size(0)) || !fits(q->size(1)) || q->size(2) != d.cache.size || !fits(batch) || !fits(table->size(1))) return none();
  const double cap = PyFloat_AS_DOUBLE(args[9]);
  if (!(cap >= 0)) return none();
  // (one below float32's smallest number is that: rounded to 0 it would be none)
  tfcc_rocm_attention_scores scores{static_cast<float>(cap > 0 ? std::max<double>(cap, std::numeric_limits<float>::denorm_min()) : 0), nullptr, nullptr};
  if (args[10] != Py_None) {
    const Tensor* slopes = plain(args[10], at::kFloat, here.device);
    if (!slopes || slopes->dim() != 1 || slopes->size(0) != q->size(1)) return none();
    scores.slopes = data<float>(slopes);
  }
  if (args[11] != Py_None) {
    const Tensor* prefixes = plain(args[11], at::kInt, here.device);
    if (!prefixes || prefixes->dim() != 1 || prefixes->size(0) != batch) return none();
    scores.prefixes = data<int32_t>(prefixes);
  }
  Tensor out = empty(q->sizes(), at::kFloat, here.device);
  d.q = data<float>(q);
  d.out = data<float>(out);
  d.q_token_stride = q->stride(0);
  d.q_head_stride = q->stride(1);
  d.out_token_stride = static_cast<uint64_t>(q->size(1)) * q->size(2);
  d.out_head_stride = q->size(2);
  d.tokens = static_cast<unsigned>(q->size(0));
  d.heads = static_cast<unsigned>(q->size(1));
  d.batch = static_cast<unsigned>(batch);
  d.starts = data<int32_t>(starts);
  d.lengths = data<int32_t>(lengths);
  d.table = data<int32_t>(table);
  d.table_stride = table->stride(0);
  d.table_width = static_cast<unsigned>(table->size(1));
  d.max_length = static_cast<unsigned>(most);
  d.scale = static_cast<float>(PyFloat_AS_DOUBLE(args[5]));
  d.causal = args[6] == Py_True ? 1 : 0;
  d.window = static_cast<unsigned>(window);
  Tensor workspace;
  d.workspace_bytes = tfcc_rocm_paged_attention_workspace(&d);
  if (d.workspace_bytes > 0) {
    workspace = empty({static_cast<int64_t>(d.workspace_bytes)}, at::kByte, here.device);
    d.workspace = data(workspace);
  }
  void* stream = here.stream();
  if (launch([&] { return tfcc_rocm_paged_attention_scores_f32(stream, &d, &scores); }) != TFCC_ROCM_OK) return none();
  return wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// sample(logits, random, temperature, top_k, top_p, min_p), the last four or None
PyObject* sample(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 6) return none();
  Here here(args[0]);
  const Tensor* logits = rows_of(args[0], at::kFloat, 2, here.device);
  if (!logits || !fits(logits->size(0)) || !fits(logits->size(1))) return none();
  const int64_t rows = logits->size(0);
  const Tensor* given[5] = {};
  for (int i = 0; i < 5; ++i) {
    if (args[1 + i] == Py_None && i > 0) continue;
    given[i] = plain(args[1 + i], i == 2 ? at::kInt : at::kFloat, here.device);
    if (!given[i] || given[i]->dim() != 1 || given[i]->size(0) != rows) return none();
  }
  tfcc_rocm_sample_desc d{};
  Tensor tokens = empty({rows}, at::kLong, here.device), probabilities = empty({rows}, at::kFloat, here.device), workspace;
  d.logits = data<float>(logits);
  d.row_stride = logits->stride(0);
  d.rows = static_cast<unsigned>(rows);
  d.length = static_cast<unsigned>(logits->size(1));
  d.random = data<float>(given[0]);
  d.temperature = data<float>(given[1]);
  d.top_k = data<int32_t>(given[2]);
  d.top_p = data<float>(given[3]);
  d.min_p = data<float>(given[4]);
  d.tokens = data<int64_t>(tokens);
  d.probabilities = data<float>(probabilities);
  d.workspace_bytes = tfcc_rocm_sample_workspace(d.rows, d.length);
  if (d.workspace_bytes > 0) {
    workspace = empty({static_cast<int64_t>(d.workspace_bytes)}, at::kByte, here.device);
    d.workspace = data(workspace);
  }
  void* stream = here.stream();
  if (launch([&] { return tfcc_rocm_sample_f32(stream, &d); }) != TFCC_ROCM_OK) return none();
  return pack({wrap(std::move(tokens)), wrap(std::move(probabilities))});
  END_HANDLE_TH_ERRORS
}

// rms_norm(x, weight, eps, residual or None, quantized)
PyObject* rms_norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 5 || !PyFloat_CheckExact(args[2]) || !PyBool_Check(args[4])) return none();
  const double eps = PyFloat_AS_DOUBLE(args[2]);
  if (eps != 0 && !(static_cast<float>(eps) > 0)) return none();
  Here here(args[0]);
  const Tensor *x = plain(args[0], at::kFloat, here.device), *weight = plain(args[1], at::kFloat, here.device);
  const Tensor* residual = args[3] == Py_None ? nullptr : plain(args[3], at::kFloat, here.device);
  if (!x || !weight || (args[3] != Py_None && !residual) || x->dim() < 1 || x->numel() == 0 || weight->dim() != 1) return none();
  const int64_t width = x->size(x->dim() - 1), rows = x->numel() / width;
  if (weight->size(0) != width || (residual && residual->sizes() != x->sizes()) || !fits(width) || !fits(rows)) return none();
  tfcc_rocm_rms_norm_desc d{};
  Tensor sum, out, scales, sums;
  if (residual) sum = empty(x->sizes(), at::kFloat, here.device);
  d.x = data<float>(x);
  d.weight = data<float>(weight);
  d.residual = data<float>(residual);
  d.sum = residual ? data<float>(sum) : nullptr;
  d.rows = static_cast<unsigned>(rows);
  d.width = static_cast<unsigned>(width);
  d.eps = static_cast<float>(eps);
  d.x_row_stride = d.residual_row_stride = d.sum_row_stride = d.out_row_stride = d.steps_row_stride = static_cast<uint64_t>(width);
  const bool quantized = args[4] == Py_True;
  out = empty(x->sizes(), quantized ? at::kByte : at::kFloat, here.device);
  if (quantized) {
    const at::IntArrayRef shape = x->sizes().slice(0, x->dim() - 1);
    scales = empty(shape, at::kFloat, here.device);
    sums = empty(shape, at::kInt, here.device);
    d.steps = data<uint8_t>(out);
    d.scales = data<float>(scales);
    d.sums = data<int32_t>(sums);
  } else {
    d.out = data<float>(out);
  }
  void* stream = here.stream();
  if (launch([&] { return tfcc_rocm_rms_norm_f32(stream, &d); }) != TFCC_ROCM_OK) return none();
  PyObject* held = residual ? wrap(std::move(sum)) : none();
  if (quantized) return pack({wrap(std::move(out)), wrap(std::move(scales)), wrap(std::move(sums)), held});
  return pack({wrap(std::move(out)), held});
  END_HANDLE_TH_ERRORS
}

// dequantize_rows(a, scales, offset, column_scales or None)
PyObject* dequantize_rows(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 4 || !THPVariable_CheckExact(args[0]) || !PyLong_CheckExact(args[2])) return none();
  Here here(args[0]);
  const at::ScalarType type = THPVariable_Unpack(args[0]).scalar_type();
  const int code = quantized_code(type);
  const Tensor *a = plain(args[0], type, here.device), *scales = plain(args[1], at::kFloat, here.device);
  const Tensor* columns = args[3] == Py_None ? nullptr : plain(args[3], at::kFloat, here.device);
  if (!a || !scales || (args[3] != Py_None && !columns) || code < 0 || a->dim() < 1 || a->numel() == 0) return none();
  const int64_t width = a->size(a->dim() - 1), rows = a->numel() / width;
  if (scales->sizes() != a->sizes().slice(0, a->dim() - 1) || (columns && (columns->dim() != 1 || columns->size(0) != width)) || !fits(width) || !fits(rows)) return none();
  int overflow = 0;
  const long long offset = PyLong_AsLongLongAndOverflow(args[2], &overflow);
  if (overflow || offset < INT32_MIN || offset > INT32_MAX) return none();
  Tensor out = empty(a->sizes(), at::kFloat, here.device);
  void* stream = here.stream();
  if (launch([&] {
        return tfcc_rocm_dequantize_rows(stream, data(a), code, static_cast<unsigned>(rows), static_cast<unsigned>(width), static_cast<int32_t>(offset),
                                         data<float>(scales), data<float>(columns), data<float>(out));
      }) != TFCC_ROCM_OK)
    return none();
  return wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

#define TENSOR_CALL(NAME) {#NAME, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(NAME)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {TENSOR_CALL(blas_matmul), TENSOR_CALL(reduce_sum), TENSOR_CALL(quantization_matmul),
                         TENSOR_CALL(quantization_matmul_requantize), TENSOR_CALL(gemv_dequant), TENSOR_CALL(gemv_dequant_packed),
                         TENSOR_CALL(quantize), TENSOR_CALL(dequantize), TENSOR_CALL(rotary),
                         TENSOR_CALL(cache_write), TENSOR_CALL(cache_read), TENSOR_CALL(cache_copy), TENSOR_CALL(paged_attention), TENSOR_CALL(sample),
                         TENSOR_CALL(rms_norm), TENSOR_CALL(dequantize_rows), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensor_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensor_calls(void) { return PyModule_Create(&module); }
