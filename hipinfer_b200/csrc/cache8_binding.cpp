// The operators of a cache in 8 bits, and copying pages, for arguments that are as they should be: checks, allocations and the library's calls
// without the interpreter (kernels/cache8.py calls these first; where they answer None, its own checks say what is wrong). A decode step's calls
// are bounded by their host time: the attention's is 4 us, 17 through the interpreter, 20 and 60 with portions; copying 500 pages took 200.
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <vector>

namespace {

// What kernels/cache8.py keeps of a Cache8: its tensors live as long as it does.
struct Cache {
  int64_t k, v, k_scale, v_scale, pages, kv_heads, page_size, head_dim, code, device;
};
// What it makes of a step's lengths for one call: how the rows are cut into tiles.
struct Cut {
  int64_t rows, requests, n_tiles, nt, ranks, group, window, max_pos;
};
// And how a step's portions go through the flash kernel: their pages (`pages` of the block table's places, of `scales` blocks), the portions' lengths, on the
// device, and the kernel's status word.
struct Portions {
  int64_t rows, requests, width, pages, scales, limit, max_q_len, group, window, max_pos, index, places, base, q_start, q_len, ctx_len, status;
};
typedef int (*StoreFn)(const void*, const void*, long, long, int, const int*, int, int, int, int, long, int, void*, void*, float*, float*, void*);
typedef int (*ExpandFn)(const void*, const void*, const float*, const float*, int, const int*, long, long, int, int, int, void*, void*, int, void*);
typedef int (*AttendFn)(const void*, int, long, const void*, const void*, const float*, const float*, int, long, int, int, int, const int*, long, int, int,
                        const int*, const int*, int, int, int, int, int, float, void*, int, void*);
typedef int (*PortionsFn)(const void*, const void*, const float*, const float*, int, const int*, const int*, long, long, int, int, int, float, void*, void*,
                          void*, int, void*);
typedef int (*FlashFn)(const void*, const void*, const void*, long, const int*, int, const int*, const int*, const int*, void*, int, int, int, int, int, int, int,
                       int, int, int*, const void*, const int*, long, void*);
typedef int (*CopyFn)(const long*, int, const int*, const int*, int, void*);
StoreFn store_fn;
ExpandFn expand_fn;
AttendFn attend_fn;
PortionsFn portions_fn;
FlashFn flash_fn;
CopyFn copy_fn;

const at::Tensor* tensor(PyObject* x, int64_t device) {          // a strided one on that GPU
  if (!THPVariable_Check(x)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(x);
  return t.is_cuda() && t.layout() == at::kStrided && t.get_device() == device ? &t : nullptr;
}
int type_code(const at::Tensor& t) { return t.scalar_type() == at::kFloat ? 0 : t.scalar_type() == at::kBFloat16 ? 1 : -1; }
bool ints(const at::Tensor& t, int64_t dim) { return t.scalar_type() == at::kInt && t.dim() == dim && t.is_contiguous(); }
const Cache* cache(PyObject* address) {                          // null for one on another device than the current one
  const Cache* c = (const Cache*)PyLong_AsVoidPtr(address);
  return c && c->device == (int64_t)c10::cuda::current_device() ? c : nullptr;
}
// What a call of the cache8 library gave, to the interpreter: 0, or 1 where it failed (the library's own is -1, which here says that the flash kernel's did).
PyObject* code(int r) { return PyLong_FromLong(r ? 1 : 0); }
void* stream() { return c10::cuda::getCurrentCUDAStream().stream(); }
at::Tensor empty(at::IntArrayRef size, at::ScalarType type, const at::Tensor& like) {
  return at::detail::empty_cuda(size, type, like.device(), c10::nullopt);
}

PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 6) return PyErr_Format(PyExc_TypeError, "six addresses are expected");
  store_fn = (StoreFn)PyLong_AsVoidPtr(a[0]);
  expand_fn = (ExpandFn)PyLong_AsVoidPtr(a[1]);
  attend_fn = (AttendFn)PyLong_AsVoidPtr(a[2]);
  copy_fn = (CopyFn)PyLong_AsVoidPtr(a[3]);
  portions_fn = (PortionsFn)PyLong_AsVoidPtr(a[4]);
  flash_fn = (FlashFn)PyLong_AsVoidPtr(a[5]);
  if (PyErr_Occurred()) return nullptr;
  Py_RETURN_NONE;
}

// (keys, values, slot map, address of a Cache): 0, or 1 for a call that failed; None for arguments that this does not take
PyObject* store(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 4) return PyErr_Format(PyExc_TypeError, "four arguments are expected");
  const Cache* c = cache(a[3]);
  if (!c) Py_RETURN_NONE;
  const at::Tensor *k = tensor(a[0], c->device), *v = tensor(a[1], c->device), *slots = tensor(a[2], c->device);
  if (!k || !v || !slots || k->dim() != 2 || v->dim() != 2 || k->size(1) != c->kv_heads * c->head_dim || k->sizes() != v->sizes() || type_code(*k) < 0 ||
      type_code(*k) != type_code(*v) || k->stride(1) != 1 || v->stride(1) != 1 || !ints(*slots, 1) || slots->size(0) != k->size(0) || k->size(0) > 0x7fffffff ||
      !k->size(0) || !c->pages)
    Py_RETURN_NONE;
  return code(store_fn(k->const_data_ptr(), v->const_data_ptr(), (long)k->stride(0), (long)v->stride(0), type_code(*k),
                                  (const int*)slots->const_data_ptr(), (int)k->size(0), (int)c->kv_heads, (int)c->page_size, (int)c->head_dim, (long)c->pages,
                                  (int)c->code, (void*)c->k, (void*)c->v, (float*)c->k_scale, (float*)c->v_scale, stream()));
  END_HANDLE_TH_ERRORS
}

// (pages, address of a Cache, the results' type as type_code has it): keys and values; or as above
PyObject* expand(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 3) return PyErr_Format(PyExc_TypeError, "three arguments are expected");
  const Cache* c = cache(a[1]);
  if (!c) Py_RETURN_NONE;
  const at::Tensor* pages = tensor(a[0], c->device);
  if (!pages || !ints(*pages, 1) || !pages->size(0) || !c->pages) Py_RETURN_NONE;
  const at::ScalarType type = PyLong_AsLong(a[2]) == 0 ? at::kFloat : at::kBFloat16;
  const int64_t count = pages->size(0);
  at::Tensor k = empty({count, c->kv_heads, c->page_size, c->head_dim}, type, *pages), v = empty(k.sizes(), type, *pages);
  const int r = expand_fn((const void*)c->k, (const void*)c->v, (const float*)c->k_scale, (const float*)c->v_scale, (int)c->code,
                          (const int*)pages->const_data_ptr(), (long)count, (long)c->pages, (int)c->kv_heads, (int)c->page_size, (int)c->head_dim,
                          k.mutable_data_ptr(), v.mutable_data_ptr(), type_code(k), stream());
  if (r) return code(r);
  PyObject* out = PyTuple_New(2);
  if (!out) return nullptr;
  PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(std::move(k)));
  PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(std::move(v)));
  return out;
  END_HANDLE_TH_ERRORS
}

// (q, address of a Cache, block table, positions, tiles or None, address of a Cut, scale, out or None, address of Portions or 0): the output; or as above.
// With portions the Cut is of the other rows, 0 where there are none; -1: the flash kernel's call failed.
PyObject* attend(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 9) return PyErr_Format(PyExc_TypeError, "nine arguments are expected");
  const Cache* c = cache(a[1]);
  if (!c) Py_RETURN_NONE;
  const Portions* flash = (const Portions*)PyLong_AsVoidPtr(a[8]);
  const Cut* others = (const Cut*)PyLong_AsVoidPtr(a[5]);
  if (!flash && !others) Py_RETURN_NONE;
  const Cut cut = others ? *others : Cut{flash->rows, flash->requests, 0, 1, 1, flash->group, flash->window, flash->max_pos};
  const at::Tensor *q = tensor(a[0], c->device), *table = tensor(a[2], c->device), *pos = tensor(a[3], c->device);
  const at::Tensor* tiles = a[4] == Py_None ? nullptr : tensor(a[4], c->device);
  const int64_t width = c->kv_heads * cut.group * c->head_dim;
  if (!q || !table || !pos || (!tiles && a[4] != Py_None) || q->dim() != 2 || q->size(0) != cut.rows || !cut.rows || q->size(1) != width || q->stride(1) != 1 ||
      type_code(*q) < 0 || !ints(*table, 2) || table->size(0) != cut.requests ||
      table->size(1) * c->page_size <= cut.max_pos || !ints(*pos, 1) || pos->size(0) != cut.rows ||
      (tiles && (!ints(*tiles, 2) || tiles->size(0) != cut.n_tiles || tiles->size(1) != 4)))
    Py_RETURN_NONE;
  if (flash && (!q->is_contiguous() || q->scalar_type() != at::kBFloat16 || ((uintptr_t)q->const_data_ptr() & 15) || table->size(1) != flash->width)) Py_RETURN_NONE;
  const double scale = PyFloat_AsDouble(a[6]);
  if (scale == -1.0 && PyErr_Occurred()) return nullptr;
  at::Tensor out;
  if (a[7] == Py_None) {
    out = empty({cut.rows, width}, q->scalar_type(), *q);
  } else {
    const at::Tensor* given = tensor(a[7], c->device);
    if (!given || given->sizes() != q->sizes() || given->scalar_type() != q->scalar_type() || !given->is_contiguous()) Py_RETURN_NONE;
    out = *given;
    if (flash && ((uintptr_t)out.const_data_ptr() & 15)) Py_RETURN_NONE;
  }
  int r = !others ? 0 : attend_fn(q->const_data_ptr(), type_code(*q), (long)q->stride(0), (const void*)c->k, (const void*)c->v, (const float*)c->k_scale,
                          (const float*)c->v_scale, (int)c->code, (long)c->pages, (int)c->kv_heads, (int)c->page_size, (int)c->head_dim,
                          (const int*)table->const_data_ptr(), (long)table->size(1), (int)cut.requests, (int)table->size(1),
                          (const int*)pos->const_data_ptr(), tiles ? (const int*)tiles->const_data_ptr() : nullptr, (int)cut.n_tiles, (int)cut.nt,
                          (int)cut.ranks, (int)cut.group, (int)cut.window, (float)scale, out.mutable_data_ptr(), flash ? 1 : 0, stream());
  if (!r && flash) {
    at::Tensor k = empty({flash->pages, c->kv_heads, c->page_size, c->head_dim}, at::kBFloat16, *q), v = empty(k.sizes(), at::kBFloat16, *q);
    at::Tensor scales = empty({c->kv_heads, flash->scales, 4}, at::kFloat, *q);
    r = portions_fn((const void*)c->k, (const void*)c->v, (const float*)c->k_scale, (const float*)c->v_scale, (int)c->code, (const int*)table->const_data_ptr(),
                    (const int*)flash->index, (long)flash->pages, (long)c->pages, (int)c->kv_heads, (int)c->page_size, (int)c->head_dim, (float)scale,
                    k.mutable_data_ptr(), v.mutable_data_ptr(), scales.mutable_data_ptr(), others ? 1 : 0, stream());
    if (!r) {
      r = flash_fn(q->const_data_ptr(), k.const_data_ptr(), v.const_data_ptr(), (long)flash->pages, (const int*)flash->places, (int)flash->width,
                   (const int*)flash->q_start, (const int*)flash->q_len, (const int*)flash->ctx_len, out.mutable_data_ptr(), (int)cut.rows, (int)cut.requests,
                   (int)flash->max_q_len, (int)(c->kv_heads * cut.group), (int)c->kv_heads, (int)c->head_dim, (int)c->page_size, (int)cut.window,
                   (int)flash->limit, (int*)flash->status, scales.const_data_ptr(), (const int*)flash->base, (long)flash->scales, stream());
      if (r) return PyLong_FromLong(-1);
    }
  }
  if (r) return code(r);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

bool numbers(PyObject* list, int64_t end, std::vector<int>& out) {      // pages of a list or tuple of ints, all of 0 .. end - 1
  PyObject* const* item = PySequence_Fast_ITEMS(list);
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(list);
  out.resize(n);
  for (Py_ssize_t i = 0; i < n; i++) {
    if (!PyLong_CheckExact(item[i])) return false;
    int over = 0;
    const long x = PyLong_AsLongAndOverflow(item[i], &over);
    if (over || x < 0 || x >= end) return false;
    out[i] = (int)x;
  }
  return true;
}

// (planes, sources, targets), each a list or tuple: 0, or 1 for a call that failed; None for arguments that this does not take
PyObject* copy(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 3) return PyErr_Format(PyExc_TypeError, "three arguments are expected");
  for (int i = 0; i < 3; i++)
    if (!PyList_CheckExact(a[i]) && !PyTuple_CheckExact(a[i])) Py_RETURN_NONE;
  const Py_ssize_t planes = PySequence_Fast_GET_SIZE(a[0]), pairs = PySequence_Fast_GET_SIZE(a[1]);
  if (!planes || !pairs || pairs != PySequence_Fast_GET_SIZE(a[2])) Py_RETURN_NONE;
  const int64_t device = c10::cuda::current_device();
  int64_t pages = 0x7fffffff;
  std::vector<long> plane;
  plane.reserve(5 * planes);
  for (Py_ssize_t i = 0; i < planes; i++) {
    const at::Tensor* t = tensor(PySequence_Fast_GET_ITEM(a[0], i), device);
    if (!t || t->dim() < 2 || !t->numel() || !t->is_contiguous()) Py_RETURN_NONE;
    const long size = (long)t->element_size();
    for (long x : {(long)t->const_data_ptr(), (long)t->size(0), (long)t->stride(0) * size, (long)t->stride(1) * size, (long)t->stride(1) * size}) plane.push_back(x);
    pages = std::min(pages, t->size(1));
  }
  std::vector<int> src, dst;
  if (!numbers(a[1], pages, src) || !numbers(a[2], pages, dst)) Py_RETURN_NONE;
  std::vector<bool> target(pages);
  for (int p : dst) {
    if (target[p]) Py_RETURN_NONE;
    target[p] = true;
  }
  for (int p : src)
    if (target[p]) Py_RETURN_NONE;
  return code(copy_fn(plane.data(), (int)planes, src.data(), dst.data(), (int)pairs, stream()));
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {{"bind", (PyCFunction)(void*)bind, METH_FASTCALL, nullptr},     {"store", (PyCFunction)(void*)store, METH_FASTCALL, nullptr},
                         {"expand", (PyCFunction)(void*)expand, METH_FASTCALL, nullptr}, {"attend", (PyCFunction)(void*)attend, METH_FASTCALL, nullptr},
                         {"copy", (PyCFunction)(void*)copy, METH_FASTCALL, nullptr},     {nullptr, nullptr, 0, nullptr}};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "hipinfer_b200_cache8_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_hipinfer_b200_cache8_binding() { return PyModule_Create(&module_def); }
