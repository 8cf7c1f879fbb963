// binding.cpp — CPython functions behind butterfly_b200.paged: argument checks, output tensors and
// the C call in one step.  The kernels of a serving step take 2 to 10 us, and the same work in
// Python (a ctypes call, packed descriptors, torch.empty) took 7 to 19 us a call.
// The C entry points come in as addresses (init), from the library that ctypes has loaded.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <string>

#include "../../include/bna_b200.h"

namespace {

decltype(&bna_paged_reserve) g_reserve = nullptr;
decltype(&bna_paged_append) g_append = nullptr;
decltype(&bna_paged_decode) g_decode = nullptr;

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) throw torch::TypeError(std::string(name) + " must be a torch.Tensor");
  return THPVariable_Unpack(o);
}

void need(bool ok, const char* what) { TORCH_CHECK_VALUE(ok, what); }

void need_cuda(std::initializer_list<const at::Tensor*> xs) {
  for (const at::Tensor* x : xs) need(x->is_cuda(), "butterfly_b200 kernels run on CUDA tensors only (no CPU path)");
  const auto dev = (*xs.begin())->get_device();
  for (const at::Tensor* x : xs) need(x->get_device() == dev, "all tensors must be on the same CUDA device");
}

void need_ints(const at::Tensor& x, int dim, const char* name) {
  if (x.scalar_type() != at::kInt || x.dim() != dim || (x.size(-1) > 1 && x.stride(-1) != 1))
    TORCH_CHECK_VALUE(false, name, " must be a ", dim, "-D int32 tensor with a contiguous last dim");
}

bna_tensor4 view4(const at::Tensor& x, const char* name) {
  TORCH_CHECK_VALUE(x.dim() == 4, name, " must be a 4-D tensor, got ", x.dim(), " dims");
  bna_tensor4 t;
  t.data = x.data_ptr();
  for (int i = 0; i < 4; ++i) {
    t.size[i] = x.size(i);
    t.stride[i] = x.stride(i);
  }
  return t;
}

int32_t dtype_code(const at::Tensor& x) {
  if (x.scalar_type() == at::kBFloat16) return BNA_BF16;
  TORCH_CHECK_VALUE(x.scalar_type() == at::kHalf, "paged cache kernels take bfloat16 or float16 tensors");
  return BNA_F16;
}

int64_t integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}

void* address(PyObject* o) {
  void* p = PyLong_AsVoidPtr(o);
  if (!p && PyErr_Occurred()) throw python_error();
  return p;
}

void arity(Py_ssize_t n, Py_ssize_t want) {
  if (n != want) throw torch::TypeError("wrong number of arguments");
}

at::Tensor empty(const at::Tensor& like, at::IntArrayRef size, at::ScalarType type) {
  return at::empty(size, like.options().dtype(type));
}

// n elements of `type` at byte `offset` of a byte buffer, sharing its storage (a fraction of the
// time of an allocation).
at::Tensor part(const at::Tensor& bytes, int64_t offset, int64_t n, at::ScalarType type) {
  auto impl = c10::make_intrusive<at::TensorImpl>(c10::Storage(bytes.storage()), bytes.key_set(),
                                                  caffe2::TypeMeta::fromScalarType(type));
  impl->set_sizes_contiguous({n});
  impl->set_storage_offset(bytes.storage_offset() + offset / (int64_t)c10::elementSize(type));
  return at::Tensor(std::move(impl));
}

PyObject* tuple_of(std::initializer_list<at::Tensor> ts) {
  PyObject* r = PyTuple_New((Py_ssize_t)ts.size());
  if (!r) throw python_error();
  Py_ssize_t i = 0;
  for (const at::Tensor& t : ts) PyTuple_SET_ITEM(r, i++, THPVariable_Wrap(t));
  return r;
}

// init(reserve, append, decode): addresses of the C entry points.
PyObject* init(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arity(n, 3);
  g_reserve = reinterpret_cast<decltype(g_reserve)>(address(a[0]));
  g_append = reinterpret_cast<decltype(g_append)>(address(a[1]));
  g_decode = reinterpret_cast<decltype(g_decode)>(address(a[2]));
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// The functions below return their tensors, or the status of a refused call as an int.

// reserve(lens, add, block_table, free_pages, num_free, page_size, num_tokens, stream, keep): `keep`
// [B + 1] int32 (or None) gets the new lengths and stack height after the kernel, which may have
// read the old ones from there (its CTAs read them at different times, so it cannot write there).
PyObject* reserve(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arity(n, 9);
  const at::Tensor &lens = tensor(a[0], "lens"), &add = tensor(a[1], "add"), &table = tensor(a[2], "block_table"),
                   &free_pages = tensor(a[3], "free_pages"), &num_free = tensor(a[4], "num_free");
  need_cuda({&lens, &add, &table, &free_pages, &num_free});
  const c10::DeviceGuard guard(lens.device());
  need_ints(lens, 1, "lens");
  need_ints(add, 1, "add");
  need_ints(table, 2, "block_table");
  need_ints(free_pages, 1, "free_pages");
  need_ints(num_free, 1, "num_free");
  const int64_t B = table.size(0), width = table.size(1), page_size = integer(a[5]), tokens = integer(a[6]);
  need(lens.size(0) == B && add.size(0) == B && num_free.size(0) == 1 && tokens >= 0,
       "lens and add must have block_table's rows, num_free one entry, num_tokens must be >= 0");
  const at::Tensor* keep = a[8] == Py_None ? nullptr : &tensor(a[8], "keep");
  if (keep) {
    need_cuda({&lens, keep});
    need_ints(*keep, 1, "keep");
    need(keep->size(0) == B + 1, "keep must have one entry more than block_table has rows");
  }
  need(B <= INT32_MAX && width <= INT32_MAX && free_pages.size(0) <= INT32_MAX && page_size >= 0 && page_size <= INT32_MAX,
       "paged_reserve: sizes beyond 32 bits");
  // one allocation for what lives on as the cache's state, one for the step's tokens
  const int64_t round = (tokens + 1) / 2 * 16;  // slots, to a multiple of 16 bytes
  const at::Tensor state = empty(lens, {4 * B + 4 + B}, at::kByte), step = empty(lens, {round + 4 * tokens}, at::kByte);
  at::Tensor out = part(state, 0, B, at::kInt), left = part(state, 4 * B, 1, at::kInt), granted = part(state, 4 * B + 4, B, at::kBool),
             slots = part(step, 0, tokens, at::kLong), positions = part(step, round, tokens, at::kInt);
  if (B == 0) left.copy_(num_free);  // (no request: the call writes nothing)
  const int st = g_reserve(static_cast<const int32_t*>(lens.data_ptr()), static_cast<const int32_t*>(add.data_ptr()), (int32_t)B,
                           static_cast<int32_t*>(table.data_ptr()), B > 1 ? table.stride(0) : width, (int32_t)width,
                           static_cast<int32_t*>(free_pages.data_ptr()), (int32_t)free_pages.size(0),
                           static_cast<const int32_t*>(num_free.data_ptr()), (int32_t)page_size,
                           static_cast<int32_t*>(out.data_ptr()), static_cast<int32_t*>(left.data_ptr()),
                           static_cast<uint8_t*>(granted.data_ptr()), static_cast<int64_t*>(slots.data_ptr()),
                           static_cast<int32_t*>(positions.data_ptr()), tokens, address(a[7]));
  if (st != BNA_OK) return PyLong_FromLong(st);
  if (keep) keep->copy_(part(state, 0, B + 1, at::kInt));
  return tuple_of({out, left, slots, positions, granted});
  END_HANDLE_TH_ERRORS
}

// append(k, v, k_pages, v_pages, slot_map, stream): k / v [tokens, Hkv, dh]
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arity(n, 6);
  const at::Tensor &k = tensor(a[0], "k"), &v = tensor(a[1], "v"), &kp = tensor(a[2], "k_pages"), &vp = tensor(a[3], "v_pages"),
                   &slots = tensor(a[4], "slot_map");
  need_cuda({&k, &v, &kp, &vp, &slots});
  const c10::DeviceGuard guard(k.device());
  need(k.dim() == 3 && v.dim() == 3, "k and v must be [tokens, Hkv, dh]");
  const auto dt = k.scalar_type();
  need(v.scalar_type() == dt && kp.scalar_type() == dt && vp.scalar_type() == dt, "k, v and the pools must have one dtype");
  need(slots.scalar_type() == at::kLong && slots.dim() == 1 && slots.size(0) == k.size(0) &&
           (slots.size(0) <= 1 || slots.stride(0) == 1),
       "slot_map must be a contiguous int64 tensor with one entry per token");
  bna_tensor4 rows[2];
  const at::Tensor* src[2] = {&k, &v};
  for (int i = 0; i < 2; ++i) {
    const at::Tensor& x = *src[i];
    rows[i] = bna_tensor4{x.data_ptr(), {1, x.size(1), x.size(0), x.size(2)}, {0, x.stride(1), x.stride(0), x.stride(2)}};
  }
  bna_tensor4 tkp = view4(kp, "k_pages"), tvp = view4(vp, "v_pages");
  return PyLong_FromLong(g_append(&rows[0], &rows[1], &tkp, &tvp, static_cast<const int64_t*>(slots.data_ptr()), dtype_code(k),
                                  address(a[5])));
  END_HANDLE_TH_ERRORS
}

// decode(q, k_pages, v_pages, block_table, lens, k_new, v_new, active, window, scale, want_lse, workspace, stream)
PyObject* decode(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arity(n, 13);
  const at::Tensor &q = tensor(a[0], "q"), &kp = tensor(a[1], "k_pages"), &vp = tensor(a[2], "v_pages"),
                   &table = tensor(a[3], "block_table"), &lens = tensor(a[4], "lens"), &ws = tensor(a[11], "workspace");
  need_cuda({&q, &kp, &vp, &table, &lens, &ws});
  const c10::DeviceGuard guard(q.device());
  const bna_tensor4 tq = view4(q, "q");
  bna_tensor4 tkp = view4(kp, "k_pages"), tvp = view4(vp, "v_pages");
  const int64_t B = q.size(0), Hq = q.size(1), Tq = q.size(2), dh = q.size(3);
  const auto dt = q.scalar_type();
  need(kp.scalar_type() == dt && vp.scalar_type() == dt, "the pools must have q's dtype");
  need_ints(table, 2, "block_table");
  need_ints(lens, 1, "lens");
  need(table.size(0) == B && lens.size(0) == B, "block_table and lens must have one row per request");
  need(table.size(1) <= INT32_MAX, "block_table: too many columns");
  need(ws.scalar_type() == at::kByte && ws.is_contiguous(), "workspace must be a contiguous uint8 tensor (decode_workspace)");
  const bool has_k = a[5] != Py_None, has_v = a[6] != Py_None;
  need(has_k == has_v, "k_new and v_new go together");
  bna_tensor4 tkn, tvn;
  if (has_k) {
    const at::Tensor &kn = tensor(a[5], "k_new"), &vn = tensor(a[6], "v_new");
    need_cuda({&q, &kn, &vn});
    need(kn.scalar_type() == dt && vn.scalar_type() == dt, "q, k_new, v_new dtype mismatch");
    tkn = view4(kn, "k_new");
    tvn = view4(vn, "v_new");
  }
  const uint8_t* active = nullptr;
  if (a[7] != Py_None) {
    const at::Tensor& x = tensor(a[7], "active");
    need_cuda({&q, &x});
    need(x.scalar_type() == at::kBool && x.dim() == 1 && x.size(0) == B && x.is_contiguous(),
         "active must be a contiguous bool tensor with one entry per request");
    active = static_cast<const uint8_t*>(x.data_ptr());
    need(has_k, "active says which requests have k_new / v_new rows");
  }
  const int64_t window = integer(a[8]);
  need(window >= 0 && window <= INT32_MAX, "window must be in [0, 2^31) (0: every key)");
  const double scale = PyFloat_AsDouble(a[9]);
  if (scale == -1.0 && PyErr_Occurred()) throw python_error();
  const int want_lse = PyObject_IsTrue(a[10]);
  if (want_lse < 0) throw python_error();
  const int32_t code = dtype_code(q);
  at::Tensor out = empty(q, {B, Hq, Tq, dh}, dt), lse;
  if (want_lse) lse = empty(q, {B, Hq, Tq}, at::kFloat);
  bna_tensor4 to = view4(out, "out");
  const int st = g_decode(&tq, &tkp, &tvp, has_k ? &tkn : nullptr, has_k ? &tvn : nullptr, active, &to,
                          want_lse ? static_cast<float*>(lse.data_ptr()) : nullptr, Hq * Tq, Tq, code,
                          static_cast<const int32_t*>(table.data_ptr()), table.stride(0), (int32_t)table.size(1),
                          static_cast<const int32_t*>(lens.data_ptr()), (int32_t)window, (float)scale, ws.data_ptr(), ws.numel(),
                          address(a[12]));
  if (st != BNA_OK) return PyLong_FromLong(st);
  if (want_lse) return tuple_of({out, lse});
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyCFunction fast() {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F));
}

PyMethodDef methods[] = {{"init", fast<init>(), METH_FASTCALL, nullptr},
                         {"reserve", fast<reserve>(), METH_FASTCALL, nullptr},
                         {"append", fast<append>(), METH_FASTCALL, nullptr},
                         {"decode", fast<decode>(), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__native(void) { return PyModule_Create(&module); }
