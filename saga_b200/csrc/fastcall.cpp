// Host calls of the 4-bit cache operators without Python between the tensors
// and the C ABI. A call that is right in every respect is made here, and its
// outputs are returned; for any other this returns None, and the Python layer
// (saga_b200/kv4.py) makes the same call or raises the error that fits. The
// kernels are reached through the addresses that the Python layer binds, so
// this module does not link the CUDA library.
//
// What it saves: a call of these operators is two launches of about 2.5 us, and
// built in Python the descriptor, the checks and the outputs took longer
// (page_tables of 64 requests: 19 us, 9 us from here).
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/utils/pybind.h>
#include <torch/version.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAStream.h>

#include <cmath>
#include <map>
#include <vector>

#include "../../include/saga_b200.h"

namespace {

decltype(&saga_kv4_write) f_write;
decltype(&saga_kv4_read) f_read;
decltype(&saga_kv4_workspace_bytes) f_workspace;
decltype(&saga_kv4_decode) f_decode;
decltype(&saga_kv4_select) f_select;
decltype(&saga_page_tables) f_tables;

// A pool as the Python layer describes it once.
struct Pool {
  SagaKv4Pool desc;
  int index;
  int32_t* status;
  std::map<std::vector<int64_t>, size_t> sizes;  // workspace bytes per op and shapes
};

// A workspace for one call on the current stream: one is kept per (device,
// stream): a call makes all its launches before another thread can make one here,
// since it holds Python's lock throughout. A call under capture gets one
// of its own from the graph's memory: graphs captured on one stream may be
// replayed on several. The kernels do not care what a workspace holds.
std::map<std::pair<int, cudaStream_t>, at::Tensor>& scratches() {
  static auto* m = new std::map<std::pair<int, cudaStream_t>, at::Tensor>();  // outlives CUDA's teardown
  return *m;
}
at::Tensor scratch(int index, cudaStream_t stream, size_t nbytes) {
  auto take = [&](size_t n) {
    return at::empty({(int64_t)n}, at::TensorOptions().dtype(at::kByte).device(at::kCUDA, index));
  };
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None) return take(nbytes);
  at::Tensor& have = scratches()[{index, stream}];
  if (!have.defined()) have = take(std::max(nbytes, (size_t)1 << 20));
  else if ((size_t)have.numel() < nbytes) have = take(std::max(nbytes, 2 * (size_t)have.numel()));
  return have;
}

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16: return SAGA_BF16;
    case at::kHalf: return SAGA_FP16;
    case at::kFloat: return SAGA_FP32;
    default: return -1;
  }
}

// The argument as a plain strided CUDA tensor of the device, or NULL.
const at::Tensor* tensor(PyObject* o, int index) {
  if (!THPVariable_Check(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda() || t.layout() != at::kStrided || t.get_device() != index) return nullptr;
  if (t.unsafeGetTensorImpl()->is_python_dispatch() || t.is_neg() || t.is_conj()) return nullptr;
  return &t;
}
// The address of a contiguous tensor of these sizes, or false.
template <class T>
bool ints(PyObject* o, int index, at::ScalarType type, at::IntArrayRef sizes, T** p) {
  const at::Tensor* t = tensor(o, index);
  if (!t || t->scalar_type() != type || t->sizes() != sizes || !t->is_contiguous()) return false;
  *p = reinterpret_cast<T*>(t->data_ptr());
  return true;
}
bool table(PyObject* o, int index, int64_t B, int32_t** p, int64_t* stride, int32_t* width) {
  const at::Tensor* t = tensor(o, index);
  if (!t || t->scalar_type() != at::kInt || t->dim() != 2 || t->size(0) < B || t->numel() == 0 || t->stride(1) != 1 ||
      t->size(1) > INT32_MAX)
    return false;
  *p = reinterpret_cast<int32_t*>(t->data_ptr());
  *stride = t->stride(0);
  *width = (int32_t)t->size(1);
  return true;
}
bool rows(PyObject* o, const Pool& p, int64_t T, int heads, at::ScalarType type, const at::Tensor** out) {
  const at::Tensor* t = tensor(o, p.index);
  if (!t || t->scalar_type() != type || t->dim() != 3 || t->size(0) != T || t->size(1) != heads ||
      t->size(2) != p.desc.D || t->stride(2) != 1)
    return false;
  *out = t;
  return true;
}

Pool* pool_of(PyObject* o) { return reinterpret_cast<Pool*>(PyCapsule_GetPointer(o, "saga_kv4_pool")); }
bool on_device(int index) { return c10::cuda::current_device() == index; }
cudaStream_t stream_of(int index) { return c10::cuda::getCurrentCUDAStream(index).stream(); }
at::TensorOptions options(int index, at::ScalarType t) {
  return at::TensorOptions().dtype(t).device(at::kCUDA, index);
}

// C++ exceptions become Python's.
template <class F>
PyObject* guarded(F f) {
  try {
    return f();
  } catch (const std::exception& e) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}
#define SLOW_PATH Py_RETURN_NONE

PyObject* py_bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 6) return PyErr_Format(PyExc_TypeError, "bind takes six addresses");
  f_write = reinterpret_cast<decltype(f_write)>(PyLong_AsVoidPtr(a[0]));
  f_read = reinterpret_cast<decltype(f_read)>(PyLong_AsVoidPtr(a[1]));
  f_workspace = reinterpret_cast<decltype(f_workspace)>(PyLong_AsVoidPtr(a[2]));
  f_decode = reinterpret_cast<decltype(f_decode)>(PyLong_AsVoidPtr(a[3]));
  f_select = reinterpret_cast<decltype(f_select)>(PyLong_AsVoidPtr(a[4]));
  f_tables = reinterpret_cast<decltype(f_tables)>(PyLong_AsVoidPtr(a[5]));
  if (PyErr_Occurred()) return nullptr;
  Py_RETURN_NONE;
}

// pool(address of a SagaKv4Pool, device index, address of the status word)
PyObject* py_pool(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 3) return PyErr_Format(PyExc_TypeError, "pool takes three arguments");
  const void* desc = PyLong_AsVoidPtr(a[0]);
  const int index = (int)PyLong_AsLong(a[1]);
  void* status = PyLong_AsVoidPtr(a[2]);
  if (PyErr_Occurred()) return nullptr;
  Pool* p = new Pool{*reinterpret_cast<const SagaKv4Pool*>(desc), index, reinterpret_cast<int32_t*>(status), {}};
  return PyCapsule_New(p, "saga_kv4_pool",
                       [](PyObject* c) { delete reinterpret_cast<Pool*>(PyCapsule_GetPointer(c, "saga_kv4_pool")); });
}

// write(pool, k, v, slots) -> True
PyObject* py_write(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 4) return PyErr_Format(PyExc_TypeError, "write takes four arguments");
  return guarded([&]() -> PyObject* {
    Pool* p = pool_of(a[0]);
    if (!p) return nullptr;
    const at::Tensor *s = tensor(a[3], p->index), *k, *v;
    if (!s || s->scalar_type() != at::kLong || s->dim() != 1 || s->numel() == 0 || !s->is_contiguous()) SLOW_PATH;
    const int64_t T = s->numel();
    const at::Tensor* k0 = tensor(a[1], p->index);
    if (!k0 || !rows(a[1], *p, T, p->desc.Hk, k0->scalar_type(), &k) ||
        !rows(a[2], *p, T, p->desc.Hv, k0->scalar_type(), &v))
      SLOW_PATH;
    const int dt = dtype_code(k->scalar_type());
    if (dt < 0 || !on_device(p->index)) SLOW_PATH;
    if (f_write(&p->desc, dt, T, k->data_ptr(), k->stride(0), k->stride(1), v->data_ptr(), v->stride(0), v->stride(1),
                reinterpret_cast<const int64_t*>(s->data_ptr()), p->status, stream_of(p->index)))
      SLOW_PATH;
    Py_RETURN_TRUE;
  });
}

// read(pool, slots, dtype) -> (k, v)
PyObject* py_read(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 3) return PyErr_Format(PyExc_TypeError, "read takes three arguments");
  return guarded([&]() -> PyObject* {
    Pool* p = pool_of(a[0]);
    if (!p) return nullptr;
    const at::Tensor* s = tensor(a[1], p->index);
    if (!s || s->scalar_type() != at::kLong || s->dim() != 1 || s->numel() == 0 || !s->is_contiguous() ||
        !THPDtype_Check(a[2]) || !on_device(p->index))
      SLOW_PATH;
    const at::ScalarType type = reinterpret_cast<THPDtype*>(a[2])->scalar_type;
    const int dt = dtype_code(type);
    if (dt < 0) SLOW_PATH;
    const int64_t T = s->numel(), D = p->desc.D, hk = p->desc.Hk, hv = p->desc.Hv;
    at::Tensor k = at::empty({T, hk, D}, options(p->index, type)), v = at::empty({T, hv, D}, options(p->index, type));
    if (f_read(&p->desc, dt, T, reinterpret_cast<const int64_t*>(s->data_ptr()), k.data_ptr(), hk * D, D, v.data_ptr(),
               hv * D, D, p->status, stream_of(p->index)))
      SLOW_PATH;
    return PyTuple_Pack(2, py::reinterpret_steal<py::object>(THPVariable_Wrap(std::move(k))).ptr(),
                        py::reinterpret_steal<py::object>(THPVariable_Wrap(std::move(v))).ptr());
  });
}

// The arguments that decode and select share.
bool attention(Pool* p, PyObject* query, PyObject* page_table, PyObject* lens, SagaKv4Args* c, const at::Tensor** out) {
  const at::Tensor* q = tensor(query, p->index);
  if (!q || q->dim() != 4 || q->size(2) != 1 || q->size(3) != p->desc.D || q->stride(3) != 1 || q->numel() == 0 ||
      q->size(0) > INT32_MAX || q->size(1) > INT32_MAX)
    return false;
  const int dt = dtype_code(q->scalar_type());
  if (dt < 0 || !on_device(p->index)) return false;
  c->pool = p->desc;
  c->dtype = dt;
  c->B = (int32_t)q->size(0);
  c->Hq = (int32_t)q->size(1);
  c->q = q->data_ptr();
  c->q_sb = q->stride(0);
  c->q_sh = q->stride(1);
  c->status = p->status;
  int32_t *pt, *l;
  if (!table(page_table, p->index, c->B, &pt, &c->pt_sb, &c->max_pages) ||
      !ints(lens, p->index, at::kInt, {c->B}, &l))
    return false;
  c->page_table = pt;
  c->lens = l;
  *out = q;
  return true;
}
int run(Pool* p, SagaKv4Args* c, int op) {
  size_t& bytes = p->sizes[{op, c->dtype, c->B, c->Hq, c->max_pages, c->top}];
  if (!bytes) bytes = f_workspace(c, op);
  if (!bytes) return -1;
  cudaStream_t st = stream_of(p->index);
  const at::Tensor ws = scratch(p->index, st, bytes);
  c->workspace = ws.data_ptr();
  c->workspace_bytes = bytes;
  return op == SAGA_KV4_DECODE ? f_decode(c, st) : f_select(c, st);
}

// decode(pool, query, page_table, lens, scaling, starts, blocks, counts) -> out
PyObject* py_decode(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 8) return PyErr_Format(PyExc_TypeError, "decode takes eight arguments");
  return guarded([&]() -> PyObject* {
    Pool* p = pool_of(a[0]);
    if (!p) return nullptr;
    SagaKv4Args c = {};
    const at::Tensor* q;
    if (!attention(p, a[1], a[2], a[3], &c, &q)) SLOW_PATH;
    if (a[4] == Py_None) {
      c.scaling = (float)(1.0 / std::sqrt((double)p->desc.D));
    } else {
      if (!PyFloat_Check(a[4])) SLOW_PATH;
      c.scaling = (float)PyFloat_AS_DOUBLE(a[4]);
    }
    if (a[5] != Py_None) {
      int32_t* s;
      if (!ints(a[5], p->index, at::kInt, {c.B}, &s)) SLOW_PATH;
      c.starts = s;
    }
    if (a[6] != Py_None || a[7] != Py_None) {
      const at::Tensor* b = a[6] == Py_None ? nullptr : tensor(a[6], p->index);
      if (!b || b->dim() != 3 || b->size(2) == 0 || b->size(2) > INT32_MAX) SLOW_PATH;
      c.top = (int32_t)b->size(2);
      if (!ints(a[6], p->index, at::kInt, {c.B, p->desc.Hk, c.top}, &c.blocks) ||
          !ints(a[7], p->index, at::kInt, {c.B, p->desc.Hk}, &c.counts))
        SLOW_PATH;
    }
    at::Tensor out = at::empty({c.B, c.Hq, 1, p->desc.D}, options(p->index, q->scalar_type()));
    c.out = out.data_ptr();
    c.o_sb = (int64_t)c.Hq * p->desc.D;
    c.o_sh = p->desc.D;
    if (run(p, &c, SAGA_KV4_DECODE)) SLOW_PATH;
    return THPVariable_Wrap(std::move(out));
  });
}

// select(pool, query, page_table, lens, top, keep_first, keep_last) -> (blocks, counts)
PyObject* py_select(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 7) return PyErr_Format(PyExc_TypeError, "select takes seven arguments");
  return guarded([&]() -> PyObject* {
    Pool* p = pool_of(a[0]);
    if (!p) return nullptr;
    SagaKv4Args c = {};
    const at::Tensor* q;
    if (!attention(p, a[1], a[2], a[3], &c, &q)) SLOW_PATH;
    int32_t* to[3] = {&c.top, &c.keep_first, &c.keep_last};
    for (int i = 0; i < 3; ++i) {
      if (!PyLong_CheckExact(a[4 + i])) SLOW_PATH;
      const long x = PyLong_AsLong(a[4 + i]);
      if (PyErr_Occurred()) {
        PyErr_Clear();
        SLOW_PATH;
      }
      if (x < 0 || x > INT32_MAX) SLOW_PATH;
      *to[i] = (int32_t)x;
    }
    if (c.top == 0) SLOW_PATH;
    at::Tensor blocks = at::empty({c.B, p->desc.Hk, c.top}, options(p->index, at::kInt));
    at::Tensor counts = at::empty({c.B, p->desc.Hk}, options(p->index, at::kInt));
    c.blocks = reinterpret_cast<int32_t*>(blocks.data_ptr());
    c.counts = reinterpret_cast<int32_t*>(counts.data_ptr());
    if (run(p, &c, SAGA_KV4_SELECT)) SLOW_PATH;
    return PyTuple_Pack(2, py::reinterpret_steal<py::object>(THPVariable_Wrap(std::move(blocks))).ptr(),
                        py::reinterpret_steal<py::object>(THPVariable_Wrap(std::move(counts))).ptr());
  });
}

// tables(page_table, lens, new_lens, free_pages, free_state, num_tokens, page_len, lens_out, free_state_out,
// address of the status word) -> (slots, positions, offsets, lens, free_state)
PyObject* py_tables(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 10) return PyErr_Format(PyExc_TypeError, "tables takes ten arguments");
  return guarded([&]() -> PyObject* {
    if (!THPVariable_Check(a[0]) || !THPVariable_Unpack(a[0]).is_cuda()) SLOW_PATH;
    const int index = THPVariable_Unpack(a[0]).get_device();
    const at::Tensor *lens = tensor(a[1], index), *ring = tensor(a[3], index);
    if (!lens || lens->dim() != 1 || lens->numel() == 0 || !ring || ring->dim() != 1 || ring->numel() == 0 ||
        lens->numel() > INT32_MAX || ring->numel() > INT32_MAX || !on_device(index) || !PyLong_CheckExact(a[5]) ||
        !PyLong_CheckExact(a[6]))
      SLOW_PATH;
    const int64_t B = lens->numel();
    SagaPageTableArgs c = {};
    c.num_tokens = PyLong_AsLongLong(a[5]);
    const long pl = PyLong_AsLong(a[6]);
    if (PyErr_Occurred()) {
      PyErr_Clear();
      SLOW_PATH;
    }
    if (c.num_tokens < 0 || c.num_tokens > INT32_MAX || pl < 0 || pl > INT32_MAX) SLOW_PATH;
    c.B = (int32_t)B;
    c.page_len = (int32_t)pl;
    c.ring = (int32_t)ring->numel();
    int32_t *l, *nl, *fs;
    if (!table(a[0], index, B, &c.page_table, &c.pt_sb, &c.max_pages) || !ints(a[1], index, at::kInt, {B}, &l) ||
        !ints(a[2], index, at::kInt, {B}, &nl) || !ints(a[3], index, at::kInt, {c.ring}, &c.free_pages) ||
        !ints(a[4], index, at::kInt, {2}, &fs))
      SLOW_PATH;
    c.lens = l;
    c.new_lens = nl;
    c.free_state = fs;
    at::Tensor lens_out, state_out;
    if (a[7] == Py_None) lens_out = at::empty({B}, options(index, at::kInt));
    else if (ints(a[7], index, at::kInt, {B}, &c.lens_out)) lens_out = THPVariable_Unpack(a[7]);
    else SLOW_PATH;
    if (a[8] == Py_None) state_out = at::empty({2}, options(index, at::kInt));
    else if (ints(a[8], index, at::kInt, {2}, &c.free_state_out)) state_out = THPVariable_Unpack(a[8]);
    else SLOW_PATH;
    at::Tensor slots = at::empty({c.num_tokens}, options(index, at::kLong));
    at::Tensor positions = at::empty({c.num_tokens}, options(index, at::kInt));
    at::Tensor offsets = at::empty({B + 1}, options(index, at::kInt));
    c.lens_out = reinterpret_cast<int32_t*>(lens_out.data_ptr());
    c.free_state_out = reinterpret_cast<int32_t*>(state_out.data_ptr());
    c.slots = reinterpret_cast<int64_t*>(slots.data_ptr());
    c.positions = reinterpret_cast<int32_t*>(positions.data_ptr());
    c.offsets = reinterpret_cast<int32_t*>(offsets.data_ptr());
    c.status = reinterpret_cast<int32_t*>(PyLong_AsVoidPtr(a[9]));
    cudaStream_t st = stream_of(index);
    c.workspace_bytes = 16 * (size_t)B;
    const at::Tensor ws = scratch(index, st, c.workspace_bytes);
    c.workspace = ws.data_ptr();
    if (f_tables(&c, st)) SLOW_PATH;
    PyObject* r = PyTuple_New(5);
    if (!r) return nullptr;
    PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(std::move(slots)));
    PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(std::move(positions)));
    PyTuple_SET_ITEM(r, 2, THPVariable_Wrap(std::move(offsets)));
    PyTuple_SET_ITEM(r, 3, THPVariable_Wrap(std::move(lens_out)));
    PyTuple_SET_ITEM(r, 4, THPVariable_Wrap(std::move(state_out)));
    return r;
  });
}

#define METHOD(name) \
  { #name, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_##name)), METH_FASTCALL, nullptr }
PyMethodDef methods[] = {METHOD(bind), METHOD(pool), METHOD(write), METHOD(read), METHOD(decode),
                         METHOD(select), METHOD(tables), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fastcall", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fastcall(void) {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "torch_version", TORCH_VERSION)) Py_CLEAR(m);
  return m;
}
