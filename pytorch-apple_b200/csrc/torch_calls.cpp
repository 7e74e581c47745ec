// The calls of paged_attention.py and sampling.py from torch tensors to the library, as a CPython module.
//
// Checking the tensors, making the output and the workspace and filling the argument structure costs 10 us in Python, more than most of these
// kernels run; here it costs one.  Every function takes the address of the library's entry point first, or minus the address of a stand-in of the
// test-suite, which works on host memory, and returns the output tensor, 1 where the tensors do not fit together (the caller says what it has
// seen), or the library's negative code.  Work goes to the current stream of the tensors' device, with that device current.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <cmath>
#include <optional>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/b200nn.h"

namespace {

using at::Tensor;

// The tensor an argument is, or nullptr for None
const Tensor* tensor(PyObject* o) { return o == Py_None ? nullptr : &THPVariable_Unpack(o); }
bool is_tensor(PyObject* o) { return THPVariable_Check(o); }
bool is_optional(PyObject* o) { return o == Py_None || THPVariable_Check(o); }
void* address(const Tensor* t) { return t ? t->data_ptr() : nullptr; }

int code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return B200_F32;
    case at::kHalf: return B200_F16;
    case at::kBFloat16: return B200_BF16;
    default: return -1;
  }
}

bool dense(const Tensor& t, const Tensor& with, at::ScalarType type, at::IntArrayRef sizes) {
  return t.scalar_type() == type && t.sizes() == sizes && t.is_contiguous() && t.device() == with.device();
}
// [tokens, heads, dims] with contiguous dims
bool heads(const Tensor& t, const Tensor& with, int64_t tokens) {
  return t.dim() == 3 && t.scalar_type() == with.scalar_type() && (t.size(2) <= 1 || t.stride(2) == 1) && t.size(0) == tokens && t.device() == with.device();
}
bool pages(const Tensor& k, const Tensor& v, const Tensor& with, int64_t dims) {
  return k.dim() == 4 && k.sizes() == v.sizes() && k.strides() == v.strides() && k.scalar_type() == with.scalar_type() && v.scalar_type() == with.scalar_type() &&
         k.size(3) == dims && k.stride(3) == 1 && k.device() == with.device() && v.device() == with.device() && k.size(0) > 0 && k.size(1) > 0 && k.size(2) > 0;
}
Tensor made(const Tensor& like, at::IntArrayRef sizes, at::ScalarType type) { return at::empty(sizes, like.options().dtype(type).requires_grad(false)); }
void* stream_of(const Tensor& t) { return t.is_cuda() ? static_cast<void*>(c10::cuda::getCurrentCUDAStream(t.device().index()).stream()) : nullptr; }

// The entry point that `a` stands for, as a function; nullptr: it does not take tensors on the device that `t` is on
template <typename F> F* entry(PyObject* a, const Tensor& t) {
  const int64_t at = PyLong_AsLongLong(a);
  return t.is_cuda() == (at > 0) ? reinterpret_cast<F*>(at > 0 ? at : -at) : nullptr;
}

PyObject* one() { return PyLong_FromLong(1); }

// address, q, k, v, cos, sin, k_pages, v_pages, slots, q_out
PyObject* paged_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 10 || !is_optional(a[1]) || !is_tensor(a[2]) || !is_tensor(a[3]) || !is_optional(a[4]) || !is_optional(a[5]) || !is_tensor(a[6]) ||
      !is_tensor(a[7]) || !is_tensor(a[8]) || !is_optional(a[9])) return one();
  const Tensor *q = tensor(a[1]), *cos = tensor(a[4]), *sin = tensor(a[5]), *given = tensor(a[9]);
  const Tensor &k = *tensor(a[2]), &v = *tensor(a[3]), &kp = *tensor(a[6]), &vp = *tensor(a[7]), &slots = *tensor(a[8]);
  auto* const call = entry<int(const b200_paged_append_args*, void*)>(a[0], k);
  if (!call || k.dim() != 3 || code(k.scalar_type()) < 0) return one();
  const int64_t N = k.size(0), Hkv = k.size(1), D = k.size(2);
  if (!heads(k, k, N) || !heads(v, k, N) || v.sizes() != k.sizes() || !pages(kp, vp, k, D) || kp.size(1) != Hkv || !dense(slots, k, at::kLong, {N})) return one();
  if (q && (!heads(*q, k, N) || q->size(2) != D)) return one();
  if (given && (!q || !dense(*given, k, k.scalar_type(), q->sizes()))) return one();
  if (!cos != !sin) return one();
  if (cos && (code(cos->scalar_type()) < 0 || !dense(*cos, k, cos->scalar_type(), {N, D}) || !dense(*sin, k, cos->scalar_type(), {N, D}))) return one();
  const c10::OptionalDeviceGuard guard(k.is_cuda() ? std::optional<c10::Device>(k.device()) : std::nullopt);
  Tensor out;
  if (q) out = given ? *given : made(k, q->sizes(), k.scalar_type());
  if (N > 0) {
    b200_paged_append_args args = {};
    args.q = address(q); args.k = k.data_ptr(); args.v = v.data_ptr(); args.cos_t = address(cos); args.sin_t = address(sin);
    args.q_out = q ? out.data_ptr() : nullptr; args.k_pages = kp.data_ptr(); args.v_pages = vp.data_ptr();
    args.slots = static_cast<const int64_t*>(slots.data_ptr());
    args.n_tokens = N; args.num_pages = kp.size(0);
    for (int i = 0; i < 2; ++i) {
      args.q_strides[i] = q ? q->stride(i) : 0;
      args.k_strides[i] = k.stride(i);
      args.v_strides[i] = v.stride(i);
    }
    for (int i = 0; i < 3; ++i) args.kv_strides[i] = kp.stride(i);
    args.Hq = q ? static_cast<int32_t>(q->size(1)) : 0;
    args.Hkv = static_cast<int32_t>(Hkv); args.D = static_cast<int32_t>(D); args.page_size = static_cast<int32_t>(kp.size(2));
    args.table_dtype = cos ? code(cos->scalar_type()) : 0;
    args.dtype = code(k.scalar_type());
    if (const int rc = call(&args, stream_of(k))) return PyLong_FromLong(rc);
  }
  if (!q) Py_RETURN_NONE;
  if (given) return Py_NewRef(a[9]);
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// address, address of the workspace's size, q, k_pages, v_pages, q_start, kv_len, page_table, max_q, scale (NaN: 1 / sqrt(D)), window, out
PyObject* paged_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 12 || !is_tensor(a[2]) || !is_tensor(a[3]) || !is_tensor(a[4]) || !is_tensor(a[5]) || !is_tensor(a[6]) || !is_tensor(a[7]) || !is_optional(a[11]))
    return one();
  const Tensor &q = *tensor(a[2]), &kp = *tensor(a[3]), &vp = *tensor(a[4]), &start = *tensor(a[5]), &len = *tensor(a[6]), &table = *tensor(a[7]);
  const Tensor* given = tensor(a[11]);
  int64_t max_q = PyLong_AsLongLong(a[8]);
  const int64_t window = PyLong_AsLongLong(a[10]);
  const double scale = PyFloat_AsDouble(a[9]);
  if (PyErr_Occurred()) return nullptr;
  auto* const call = entry<int(const b200_attn_paged_args*, void*)>(a[0], q);
  auto* const size = entry<int64_t(int64_t, int, int, int)>(a[1], q);
  if (!call || !size || q.dim() != 3 || code(q.scalar_type()) < 0 || table.dim() != 2) return one();
  const int64_t N = q.size(0), Hq = q.size(1), D = q.size(2), B = table.size(0);
  if (!heads(q, q, N) || !pages(kp, vp, q, D) || !dense(start, q, at::kInt, {B + 1}) || !dense(len, q, at::kInt, {B}) ||
      !dense(table, q, at::kInt, table.sizes()) || (given && !dense(*given, q, q.scalar_type(), q.sizes()))) return one();
  const c10::OptionalDeviceGuard guard(q.is_cuda() ? std::optional<c10::Device>(q.device()) : std::nullopt);
  const Tensor out = given ? *given : made(q, q.sizes(), q.scalar_type());
  if (N > 0 && B > 0) {
    // (0 tells the library that no sequence has a token, and it launches nothing: an output made here would come back as it was allocated)
    if (max_q == 0) max_q = 1;
    // from the allocator on every call: a captured graph gets a workspace of its own, calls on other streams theirs
    const int64_t need = size(max_q, static_cast<int>(Hq), static_cast<int>(kp.size(1)), static_cast<int>(D));
    const Tensor space = made(q, {need}, at::kByte);
    b200_attn_paged_args args = {};
    args.q = q.data_ptr(); args.k_pages = kp.data_ptr(); args.v_pages = vp.data_ptr(); args.out = out.data_ptr();
    args.q_start = static_cast<const int32_t*>(start.data_ptr()); args.kv_len = static_cast<const int32_t*>(len.data_ptr());
    args.page_table = static_cast<const int32_t*>(table.data_ptr());
    args.workspace = space.data_ptr(); args.workspace_bytes = need;
    args.B = B; args.n_tokens = N; args.max_q = max_q; args.num_pages = kp.size(0); args.table_stride = table.size(1);
    for (int i = 0; i < 2; ++i) args.q_strides[i] = q.stride(i);
    for (int i = 0; i < 3; ++i) args.kv_strides[i] = kp.stride(i);
    args.window = window;
    args.Hq = static_cast<int32_t>(Hq); args.Hkv = static_cast<int32_t>(kp.size(1)); args.D = static_cast<int32_t>(D);
    args.page_size = static_cast<int32_t>(kp.size(2)); args.dtype = code(q.scalar_type());
    args.scale = static_cast<float>(scale == scale ? scale : 1. / std::sqrt(static_cast<double>(D)));
    if (const int rc = call(&args, stream_of(q))) return PyLong_FromLong(rc);
  }
  if (given) return Py_NewRef(a[11]);
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// address, logits, uniform, temperature, top_k, top_p, min_p, out
PyObject* sample_rows(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 8 || !is_tensor(a[1]) || !is_tensor(a[2])) return one();
  for (int i = 3; i < 8; ++i)
    if (!is_optional(a[i])) return one();
  const Tensor& x = *tensor(a[1]);
  auto* const call = entry<int(const void*, int64_t*, int64_t, int64_t, int64_t, const float*, const int32_t*, const float*, const float*, const float*, int, void*)>(a[0], x);
  if (!call || x.dim() != 2 || code(x.scalar_type()) < 0 || x.size(1) < 1 || (x.size(1) > 1 && x.stride(1) != 1)) return one();
  const int64_t rows = x.size(0);
  for (int i = 2; i < 8; ++i) {
    const at::ScalarType type = i == 4 ? at::kInt : i == 7 ? at::kLong : at::kFloat;
    if (const Tensor* t = tensor(a[i]))
      if (!dense(*t, x, type, {rows})) return one();
  }
  const c10::OptionalDeviceGuard guard(x.is_cuda() ? std::optional<c10::Device>(x.device()) : std::nullopt);
  const Tensor out = tensor(a[7]) ? *tensor(a[7]) : made(x, {rows}, at::kLong);
  if (rows > 0) {
    const int rc = call(x.data_ptr(), static_cast<int64_t*>(out.data_ptr()), rows, x.size(1), x.stride(0), static_cast<const float*>(address(tensor(a[3]))),
                        static_cast<const int32_t*>(address(tensor(a[4]))), static_cast<const float*>(address(tensor(a[5]))),
                        static_cast<const float*>(address(tensor(a[6]))), static_cast<const float*>(address(tensor(a[2]))), code(x.scalar_type()), stream_of(x));
    if (rc) return PyLong_FromLong(rc);
  }
  if (a[7] != Py_None) return Py_NewRef(a[7]);
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"paged_append", reinterpret_cast<PyCFunction>(paged_append), METH_FASTCALL, nullptr},
    {"paged_attention", reinterpret_cast<PyCFunction>(paged_attention), METH_FASTCALL, nullptr},
    {"sample_rows", reinterpret_cast<PyCFunction>(sample_rows), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "b200_torch_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// Looked for in the file before it is loaded: torch's and the interpreter's versions
extern "C" __attribute__((used, visibility("default"))) const char b200_torch_calls_built_for[] = B200_BUILT_FOR;

PyMODINIT_FUNC PyInit_b200_torch_calls(void) { return PyModule_Create(&module); }
