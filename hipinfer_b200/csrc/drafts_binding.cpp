// attention_shared and verify_drafts for arguments that are as they should be: checks, allocations and the library's call without the
// interpreter (kernels/drafts.py calls these first; where they answer None, its own checks say what is wrong). A call's host time is what bounds
// the small ones: 14.5 us for the attention and 20 for the verification through the interpreter, of which the launches are 5.
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

namespace {

// What kernels/drafts.py keeps of a plan: its sizes, and the array that the library's call reads (SharedLaunch in attention_shared.cu).
struct Plan {
  int64_t rows, width, kv_heads, page_size, head_dim, dtype, requests, most_keys, workspace, ctas, numbers, launch;
  double scale;
};
typedef int (*AttendFn)(const void*, long, const void*, const void*, long, const int*, int, const int*, const void*, float*, void*, float, int, int*, void*);
typedef int (*VerifyFn)(const void*, int, long, int, int, const int*, const int*, const int*, int, int, const float*, const float*, const float*, long,
                        const void*, int, long, long, void*, int*, int*, float*, void*);
typedef int (*WorkspaceFn)(int, int, int, int);
AttendFn attend_fn;
VerifyFn verify_fn;
WorkspaceFn workspace_fn;
constexpr int64_t MAX_DRAFTS = 63;

const at::Tensor* tensor(PyObject* x) {          // a strided one on the GPU
  if (!THPVariable_Check(x)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(x);
  return t.is_cuda() && t.layout() == at::kStrided ? &t : nullptr;
}
int type_code(const at::Tensor& t) { return t.scalar_type() == at::kFloat ? 0 : t.scalar_type() == at::kBFloat16 ? 1 : -1; }
bool vector(const at::Tensor& t, at::ScalarType type, int64_t n) { return t.scalar_type() == type && t.numel() == n && t.is_contiguous(); }
at::Tensor empty(at::IntArrayRef size, at::ScalarType type, c10::Device device) {
  return at::detail::empty_cuda(size, type, device, c10::nullopt);
}

PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 3) return PyErr_Format(PyExc_TypeError, "three addresses are expected");
  attend_fn = (AttendFn)PyLong_AsVoidPtr(a[0]);
  verify_fn = (VerifyFn)PyLong_AsVoidPtr(a[1]);
  workspace_fn = (WorkspaceFn)PyLong_AsVoidPtr(a[2]);
  if (PyErr_Occurred()) return nullptr;
  Py_RETURN_NONE;
}

// (q, keys, values, block table, address of a Plan, out or None, scale or None, address of the status word): the output; None for arguments
// that this does not take; the code of a call that failed
PyObject* attend(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 8) return PyErr_Format(PyExc_TypeError, "eight arguments are expected");
  const at::Tensor *q = tensor(a[0]), *k = tensor(a[1]), *v = tensor(a[2]), *table = tensor(a[3]);
  if (!q || !k || !v || !table) Py_RETURN_NONE;
  const Plan& p = *(const Plan*)PyLong_AsVoidPtr(a[4]);
  const int64_t pages = k->dim() == 4 ? k->size(0) : 0;
  const auto paged = [&](const at::Tensor& t) {
    return t.dim() == 4 && t.size(0) == pages && t.size(1) == p.kv_heads && t.size(2) == p.page_size && t.size(3) == p.head_dim && type_code(t) == p.dtype &&
           t.is_contiguous();
  };
  if (q->dim() != 2 || q->size(0) != p.rows || q->size(1) != p.width || q->stride(1) != 1 || type_code(*q) != p.dtype || !p.rows || !paged(*k) || !paged(*v) ||
      table->dim() != 2 || table->scalar_type() != at::kInt || table->stride(1) != 1 || table->size(0) != p.requests ||
      table->size(1) * p.page_size < p.most_keys)
    Py_RETURN_NONE;
  at::Tensor out;
  if (a[5] == Py_None) {
    out = empty({p.rows, p.width}, q->scalar_type(), q->device());
  } else {
    const at::Tensor* given = tensor(a[5]);
    if (!given || given->dim() != 2 || given->size(0) != p.rows || given->size(1) != p.width || type_code(*given) != p.dtype || !given->is_contiguous())
      Py_RETURN_NONE;
    out = *given;
  }
  double scale = p.scale;
  if (a[6] != Py_None && (scale = PyFloat_AsDouble(a[6])) == -1.0 && PyErr_Occurred()) return nullptr;
  at::Tensor ws;
  if (p.workspace) ws = empty({p.workspace}, at::kFloat, q->device());
  const int64_t ld = q->stride(0), size = p.dtype ? 2 : 4;
  const uintptr_t all = (uintptr_t)q->const_data_ptr() | (uintptr_t)k->const_data_ptr() | (uintptr_t)v->const_data_ptr() | (uintptr_t)out.const_data_ptr();
  const int r = attend_fn(q->const_data_ptr(), (long)ld, k->const_data_ptr(), v->const_data_ptr(), (long)pages, (const int*)table->const_data_ptr(),
                          (int)table->stride(0), (const int*)p.numbers, (const void*)p.launch, ws.defined() ? (float*)ws.mutable_data_ptr() : nullptr,
                          out.mutable_data_ptr(), (float)scale, (ld * size) % 16 == 0 && all % 16 == 0, (int*)PyLong_AsVoidPtr(a[7]),
                          c10::cuda::getCurrentCUDAStream().stream());
  if (r) return PyLong_FromLong(r);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// The arguments of ops.verify_drafts: its three results, or as above
PyObject* verify(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 8) return PyErr_Format(PyExc_TypeError, "eight arguments are expected");
  const at::Tensor* t[7];
  for (int i = 0; i < 7; i++)
    if (!(t[i] = tensor(a[i]))) Py_RETURN_NONE;
  const at::Tensor &logits = *t[0], &start = *t[1], &n_drafts = *t[2], &drafts = *t[3], &temperature = *t[4], &uniform = *t[5], &noise = *t[6];
  if (logits.dim() != 2 || drafts.dim() != 2 || noise.dim() != 2) Py_RETURN_NONE;
  const int64_t T = logits.size(0), V = logits.size(1), R = drafts.size(0), K = drafts.size(1);
  const int dt = type_code(logits);
  if (dt < 0 || !R || !V || R > 65535 || T > 0x7fffffff || V > 1 << 30 || K > MAX_DRAFTS || (V > 1 && logits.stride(1) != 1) || !vector(drafts, at::kInt, R * K) ||
      !vector(start, at::kInt, R) || !vector(n_drafts, at::kInt, R) || !vector(temperature, at::kFloat, R) || !vector(uniform, at::kFloat, R * K) ||
      noise.scalar_type() != at::kFloat || noise.size(0) != R || noise.size(1) != V || (V > 1 && noise.stride(1) != 1))
    Py_RETURN_NONE;
  const at::Tensor* probs = nullptr;
  if (a[7] != Py_None) {
    probs = tensor(a[7]);
    if (!probs || probs->dim() != 3 || probs->size(0) != R || probs->size(1) != K || probs->size(2) != V || type_code(*probs) < 0 || (V > 1 && probs->stride(2) != 1))
      Py_RETURN_NONE;
    if (!K) probs = nullptr;
  }
  const int floats = workspace_fn((int)R, (int)K, (int)V, dt);
  if (floats < 0) Py_RETURN_NONE;
  const c10::Device device = logits.device();
  at::Tensor tokens = empty({R, K + 1}, at::kInt, device), counts = empty({R}, at::kInt, device), logprobs = empty({R, K + 1}, at::kFloat, device),
             ws = empty({floats}, at::kFloat, device);
  const int r = verify_fn(logits.const_data_ptr(), dt, (long)logits.stride(0), (int)T, (int)V, (const int*)start.const_data_ptr(),
                          (const int*)n_drafts.const_data_ptr(), (const int*)drafts.const_data_ptr(), (int)R, (int)K, (const float*)temperature.const_data_ptr(),
                          (const float*)uniform.const_data_ptr(), (const float*)noise.const_data_ptr(), (long)noise.stride(0),
                          probs ? probs->const_data_ptr() : nullptr, probs ? type_code(*probs) : 0, probs ? (long)probs->stride(0) : 0,
                          probs ? (long)probs->stride(1) : 0, ws.mutable_data_ptr(), (int*)tokens.mutable_data_ptr(), (int*)counts.mutable_data_ptr(),
                          (float*)logprobs.mutable_data_ptr(), c10::cuda::getCurrentCUDAStream().stream());
  if (r) return PyLong_FromLong(r);
  PyObject* out = PyTuple_New(3);
  if (!out) return nullptr;
  PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(std::move(tokens)));
  PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(std::move(counts)));
  PyTuple_SET_ITEM(out, 2, THPVariable_Wrap(std::move(logprobs)));
  return out;
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {{"bind", (PyCFunction)(void*)bind, METH_FASTCALL, nullptr},
                         {"attend", (PyCFunction)(void*)attend, METH_FASTCALL, nullptr},
                         {"verify", (PyCFunction)(void*)verify, METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "hipinfer_b200_drafts_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_hipinfer_b200_drafts_binding() { return PyModule_Create(&module_def); }
