// The serving operators' ordinary eager calls, from Python to the C ABI without
// Python in between: their smallest calls take a few microseconds on the device,
// and checking and marshalling them in Python takes longer than that.
//
// Each function does the call when everything about it is ordinary -- plain
// strided CUDA tensors of the expected shapes and types, laid out as the C ABI
// wants them, nothing watching (no dispatch mode, tracer or functorch level, no
// gradient asked for) -- and returns None, with nothing done, when it is not.
// The public functions (mxwave_b200/linear.py, kvcache.py) then take their
// general path, which copies, dispatches or raises.  So no check lives here alone.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>

#include "../../include/mxwave_b200.h"

namespace {

int dtype_code(at::ScalarType t) {
  return t == at::kBFloat16 ? MXW_BF16 : t == at::kHalf ? MXW_F16 : t == at::kFloat ? MXW_F32 : -1;
}

// Whether something records or transforms operators on this thread: each such
// thing adds keys to those that every call dispatches through.
bool watched() {
  constexpr c10::DispatchKeySet always({c10::DispatchKey::BackendSelect, c10::DispatchKey::ADInplaceOrView});
  return !(c10::impl::tls_local_dispatch_key_set().included_ - always).empty();
}

// A plain tensor with memory of its own kind, or null.
const at::Tensor* plain(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  return t.has_storage() && t.layout() == at::kStrided && !t.is_neg() && !t.is_conj() ? &t : nullptr;
}
const at::Tensor* on_cuda(PyObject* o) {
  const at::Tensor* t = plain(o);
  return t && t->is_cuda() ? t : nullptr;
}
bool wants_gradient(const at::Tensor* t) { return t && ((c10::GradMode::is_enabled() && t->requires_grad()) || t->_fw_grad(0).defined()); }
bool aligned16(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }
bool bytes_like(const at::Tensor& t, int64_t dim) { return t.scalar_type() == at::kByte && t.dim() == dim && t.is_contiguous(); }

// Rows of `width` elements that are contiguous and do not overlap, whatever the
// leading dimensions; `ld`: from one to the next.
bool as_rows(const at::Tensor& t, int64_t width, int64_t rows, int64_t& ld) {
  if (t.is_contiguous()) {
    ld = width;
    return true;
  }
  if (t.dim() != 2 || (width > 1 && t.stride(1) != 1) || (rows > 1 && t.stride(0) < width)) return false;
  ld = rows > 1 ? t.stride(0) : width;
  return true;
}

PyObject* none() { Py_RETURN_NONE; }

PyObject* linear(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 6 || watched()) return none();
  const at::Tensor *x = on_cuda(args[0]), *packed = on_cuda(args[1]), *scales = on_cuda(args[2]);
  const at::Tensor* bias = args[3] == Py_None ? nullptr : on_cuda(args[3]);
  const at::Tensor* residual = args[4] == Py_None ? nullptr : on_cuda(args[4]);
  if (!x || !packed || !scales || (!bias && args[3] != Py_None) || (!residual && args[4] != Py_None)) return none();
  if (wants_gradient(x) || wants_gradient(bias) || wants_gradient(residual) || x->dim() < 1) return none();
  const int code = dtype_code(x->scalar_type());
  const auto device = x->device();
  const int64_t inner = x->size(-1);
  if ((code != MXW_BF16 && code != MXW_F16) || inner == 0 || inner % 32 != 0) return none();
  if (!bytes_like(*packed, 2) || !bytes_like(*scales, 2) || !aligned16(*packed)) return none();
  const int64_t outs = packed->size(0), rows = x->numel() / inner;
  if (packed->size(1) != inner / 2 || scales->size(0) != outs || scales->size(1) != inner / 32) return none();
  if (packed->device() != device || scales->device() != device || rows == 0 || outs == 0) return none();
  int64_t ldx = 0, ldr = 0;
  if (!as_rows(*x, inner, rows, ldx)) return none();
  if (bias && (bias->dim() != 1 || bias->size(0) != outs || bias->scalar_type() != x->scalar_type() || bias->device() != device || !bias->is_contiguous()))
    return none();
  c10::SmallVector<int64_t, 5> shape(x->sizes().begin(), x->sizes().end());
  shape.back() = outs;
  if (residual && (residual->sizes() != c10::IntArrayRef(shape) || residual->scalar_type() != x->scalar_type() || residual->device() != device ||
                   !as_rows(*residual, outs, rows, ldr)))
    return none();
  const long act = PyLong_AsLong(args[5]);
  const c10::cuda::CUDAGuard guard(device);
  at::Tensor y = at::empty(shape, x->options());
  const size_t need = mxw_linear_workspace_size(rows, inner, code);
  at::Tensor workspace = need > 16 ? at::empty({static_cast<int64_t>(need)}, packed->options()) : *packed;
  const int status = mxw_linear_mxfp4(x->data_ptr(), code, rows, inner, ldx, packed->data_ptr<uint8_t>(), scales->data_ptr<uint8_t>(), outs,
                                      bias ? bias->data_ptr() : nullptr, static_cast<int>(act), residual ? residual->data_ptr() : nullptr,
                                      residual ? ldr : outs, y.data_ptr(), workspace.data_ptr(), need, nullptr,
                                      c10::cuda::getCurrentCUDAStream(device.index()).stream());
  return status == MXW_OK ? THPVariable_Wrap(std::move(y)) : none();
  END_HANDLE_TH_ERRORS
}

struct Pool {
  const at::Tensor *codes, *scales;
  int64_t pages, heads, page, dim;
};

// One layer of a cache (`lead` 0), or all of them (1).
bool as_pool(PyObject* codes, PyObject* scales, int64_t lead, Pool& p) {
  p.codes = on_cuda(codes);
  p.scales = on_cuda(scales);
  if (!p.codes || !p.scales || !bytes_like(*p.codes, 5 + lead) || !bytes_like(*p.scales, 5 + lead)) return false;
  const auto c = p.codes->sizes(), s = p.scales->sizes();
  for (int64_t i = 0; i < 4 + lead; ++i)
    if (c[i] != s[i]) return false;
  p.pages = c[lead];
  p.heads = c[lead + 2];
  p.page = c[lead + 3];
  p.dim = 2 * c[lead + 4];
  return c[lead + 1] == 2 && s[lead + 4] * 32 == p.dim && (p.dim == 64 || p.dim == 128) && p.scales->device() == p.codes->device() &&
         aligned16(*p.codes) && aligned16(*p.scales);
}

// What an in-place operator does to its tensors' version counters (inference tensors have none).
void written(const Pool& p) {
  for (const at::Tensor* t : {p.codes, p.scales})
    if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}

bool index_like(const at::Tensor* t, at::ScalarType type, int64_t dim, c10::Device device) {
  return t && t->scalar_type() == type && t->dim() == dim && t->device() == device && t->is_contiguous();
}

PyObject* append(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Pool p;
  if (n != 5 || watched() || !as_pool(args[0], args[1], 0, p)) return none();
  const at::Tensor *key = on_cuda(args[2]), *value = on_cuda(args[3]), *slots = on_cuda(args[4]);
  const auto device = p.codes->device();
  if (!key || !value || !index_like(slots, at::kLong, 1, device)) return none();
  const int code = dtype_code(key->scalar_type());
  if (code < 0 || value->scalar_type() != key->scalar_type() || key->device() != device || value->device() != device) return none();
  if (key->dim() != 3 || key->size(1) != p.heads || key->size(2) != p.dim || value->sizes() != key->sizes() || slots->size(0) != key->size(0))
    return none();
  if (key->stride(2) != 1 || value->stride(2) != 1) return none();
  const c10::cuda::CUDAGuard guard(device);
  const int status = mxw_kv_append(p.codes->data_ptr<uint8_t>(), p.scales->data_ptr<uint8_t>(), p.pages, p.heads, p.page, p.dim, key->data_ptr(),
                                   value->data_ptr(), code, key->stride(0), key->stride(1), value->stride(0), value->stride(1),
                                   slots->data_ptr<int64_t>(), slots->size(0), c10::cuda::getCurrentCUDAStream(device.index()).stream());
  if (status != MXW_OK) return none();
  written(p);
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

PyObject* gather(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Pool p;
  if (n != 4 || watched() || !as_pool(args[0], args[1], 0, p) || !THPDtype_Check(args[3])) return none();
  const at::Tensor* slots = on_cuda(args[2]);
  const auto device = p.codes->device();
  const at::ScalarType type = reinterpret_cast<THPDtype*>(args[3])->scalar_type;
  const int code = dtype_code(type);
  if (code < 0 || !index_like(slots, at::kLong, 1, device)) return none();
  const c10::cuda::CUDAGuard guard(device);
  const auto options = p.codes->options().dtype(type);
  at::Tensor key = at::empty({slots->size(0), p.heads, p.dim}, options), value = at::empty({slots->size(0), p.heads, p.dim}, options);
  const int status = mxw_kv_gather(p.codes->data_ptr<uint8_t>(), p.scales->data_ptr<uint8_t>(), p.pages, p.heads, p.page, p.dim,
                                   slots->data_ptr<int64_t>(), slots->size(0), code, key.data_ptr(), value.data_ptr(),
                                   c10::cuda::getCurrentCUDAStream(device.index()).stream());
  if (status != MXW_OK) return none();
  PyObject* k = THPVariable_Wrap(std::move(key));
  PyObject* v = THPVariable_Wrap(std::move(value));
  return Py_BuildValue("(NN)", k, v);
  END_HANDLE_TH_ERRORS
}

PyObject* copy_pages(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Pool p;
  if (n != 4 || watched() || !as_pool(args[0], args[1], 1, p)) return none();
  const at::Tensor *source = plain(args[2]), *target = plain(args[3]);
  if (!index_like(source, at::kLong, 1, c10::Device(c10::kCPU)) || !index_like(target, at::kLong, 1, c10::Device(c10::kCPU)) ||
      source->size(0) != target->size(0))
    return none();
  const auto device = p.codes->device();
  const c10::cuda::CUDAGuard guard(device);
  const int64_t rows = 2 * p.heads * p.page;
  const int status = mxw_copy_pages(p.codes->data_ptr<uint8_t>(), p.scales->data_ptr<uint8_t>(), p.codes->size(0), p.pages, rows * p.dim / 2,
                                    rows * p.dim / 32, source->data_ptr<int64_t>(), target->data_ptr<int64_t>(), source->size(0),
                                    c10::cuda::getCurrentCUDAStream(device.index()).stream());
  if (status != MXW_OK) return none();
  written(p);
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// (query, codes, scales, table, lengths, query_start, max_length, max_queries, softmax_scale or None, causal, window, return_lse)
PyObject* attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Pool p;
  if (n != 12 || watched() || !as_pool(args[1], args[2], 0, p)) return none();
  const at::Tensor *query = on_cuda(args[0]), *table = on_cuda(args[3]), *lengths = on_cuda(args[4]), *start = on_cuda(args[5]);
  const auto device = p.codes->device();
  if (!query || wants_gradient(query) || query->dim() != 3 || query->device() != device || query->stride(2) != 1) return none();
  const int code = dtype_code(query->scalar_type());
  const int64_t tokens = query->size(0), heads = query->size(1);
  if ((code != MXW_BF16 && code != MXW_F16) || query->size(2) != p.dim || tokens == 0 || heads == 0 || p.heads == 0 || heads % p.heads != 0)
    return none();
  if (!index_like(table, at::kInt, 2, device) || !index_like(lengths, at::kInt, 1, device) || !index_like(start, at::kInt, 1, device)) return none();
  const int64_t seqs = table->size(0), width = table->size(1);
  if (seqs == 0 || lengths->size(0) != seqs || start->size(0) != seqs + 1) return none();
  for (int i : {6, 7, 10})
    if (!PyLong_CheckExact(args[i])) return none();
  const long long max_length = PyLong_AsLongLong(args[6]), max_queries = PyLong_AsLongLong(args[7]), window = PyLong_AsLongLong(args[10]);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    return none();
  }
  const double scale = args[8] == Py_None ? 1.0 / std::sqrt(static_cast<double>(p.dim)) : PyFloat_CheckExact(args[8]) ? PyFloat_AS_DOUBLE(args[8]) : 0.0;
  const bool causal = PyObject_IsTrue(args[9]) == 1, want_lse = PyObject_IsTrue(args[11]) == 1;
  if (max_length < 0 || max_queries < 0 || window < 0 || (window > 0 && !causal) || !(scale > 0.0) || !std::isfinite(scale)) return none();
  const c10::cuda::CUDAGuard guard(device);
  at::Tensor out = at::empty({tokens, heads, p.dim}, query->options());
  at::Tensor lse = want_lse ? at::empty({tokens, heads}, query->options().dtype(at::kFloat)) : at::Tensor();
  const size_t need = mxw_paged_attention_workspace_size(seqs, heads, p.heads, p.dim, max_length, max_queries);
  at::Tensor workspace = need > 16 ? at::empty({static_cast<int64_t>(need)}, p.codes->options()) : *p.codes;
  const int status = mxw_paged_attention(query->data_ptr(), code, tokens, heads, query->stride(0), query->stride(1), p.codes->data_ptr<uint8_t>(),
                                         p.scales->data_ptr<uint8_t>(), p.pages, p.heads, p.page, p.dim, table->data_ptr<int32_t>(), width, width,
                                         lengths->data_ptr<int32_t>(), start->data_ptr<int32_t>(), seqs, max_length, max_queries, scale, causal ? 1 : 0,
                                         window, out.data_ptr(), want_lse ? lse.data_ptr<float>() : nullptr, workspace.data_ptr(), need, nullptr,
                                         c10::cuda::getCurrentCUDAStream(device.index()).stream());
  if (status != MXW_OK) return none();
  PyObject* o = THPVariable_Wrap(std::move(out));
  if (!want_lse) return o;
  PyObject* l = THPVariable_Wrap(std::move(lse));
  return Py_BuildValue("(NN)", o, l);
  END_HANDLE_TH_ERRORS
}

#define MXW_METHOD(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {MXW_METHOD(linear), MXW_METHOD(append), MXW_METHOD(gather), MXW_METHOD(copy_pages), MXW_METHOD(attention),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_binding", "Ordinary eager calls of the serving operators.", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding() { return PyModule_Create(&module); }
