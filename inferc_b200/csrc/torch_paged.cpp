// Python binding of the paged-cache entry points over torch tensors: the
// argument checks, output and scratch allocation and the call itself, for
// inferc_b200/paged.py. These operators run once per layer and decode step,
// where checking some ten tensors attribute by attribute from Python took
// longer (11 us) than the kernels run; everything else of the library is bound
// by ctypes (lib.py).
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/extension.h>

#include <map>
#include <optional>

#include "../../include/inferc_dev.h"

namespace {

constexpr const char* kHandle = "inferc_b200.PagedKV";

// A cache descriptor as PagedKV made it, with what the checks compare to. It keeps its
// tensors alive.
struct Handle {
  InfercPagedKv kv;
  at::Tensor k, v, table, lens;
  at::ScalarType type;
  int dev;
  int64_t capacity;
  std::map<std::pair<int64_t, bool>, int64_t> scratch;  // by (query heads, with weights)
};

// A status of the C ABI, on its way to inferc_b200.lib.check.
struct Status {
  int code;
};

void ok(int code) {
  if (code != INFERC_OK) throw Status{code};
}

template <typename Fn>
PyObject* guarded(Fn&& fn) {
  try {
    return fn();
  } catch (const Status& s) {
    PyObject* lib = PyImport_ImportModule("inferc_b200.lib");
    if (lib) {
      Py_XDECREF(PyObject_CallMethod(lib, "check", "i", s.code));
      Py_DECREF(lib);
    }
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "inferc_b200: unknown status");
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

int dtype_code(at::ScalarType t) {
  return t == at::kFloat ? 1 : t == at::kHalf ? 10 : t == at::kBFloat16 ? 16 : 0;
}

const at::Tensor& tensor(PyObject* o, const char* op, const char* what) {
  TORCH_CHECK(THPVariable_Check(o), op, ": ", what, " must be a tensor");
  return THPVariable_Unpack(o);
}

const at::Tensor* maybe(PyObject* o, const char* op, const char* what) {
  return o == Py_None ? nullptr : &tensor(o, op, what);
}

double number(PyObject* o) {
  const double x = PyFloat_AsDouble(o);
  if (x == -1.0 && PyErr_Occurred()) throw std::runtime_error("");
  return x;
}

int64_t integer(PyObject* o) {
  const int64_t x = PyLong_AsLongLong(o);
  if (x == -1 && PyErr_Occurred()) throw std::runtime_error("");
  return x;
}

Handle& handle(PyObject* o) {
  auto* h = static_cast<Handle*>(PyCapsule_GetPointer(o, kHandle));
  if (!h) throw std::runtime_error("");
  // x.data = y, x.set_(y), a resize: the tensor is the same, its old memory may be another's
  auto same = [](const at::Tensor& t, const void* p, const char* what) {
    TORCH_CHECK(t.const_data_ptr() == p, "PagedKV: the memory of ", what,
                " was replaced; make another view");
  };
  same(h->k, h->kv.k, "k_cache");
  same(h->v, h->kv.v, "v_cache");
  same(h->table, h->kv.page_table, "page_table");
  same(h->lens, h->kv.lens, "lens");
  return *h;
}

void arity(Py_ssize_t got, Py_ssize_t want) {
  TORCH_CHECK(got == want, "expected ", want, " arguments, got ", got);
}

// A [rows, heads, dim] tensor of the operator's type, device and sizes (-1: any).
struct Rows {
  void* p = nullptr;
  int64_t row = 0, head = 0;
};
Rows rows_of(const char* op, const char* what, const at::Tensor& t, at::ScalarType type, int dev,
             int64_t rows, int64_t heads, int64_t dim) {
  TORCH_CHECK(t.scalar_type() == type && t.is_cuda() && t.get_device() == dev, op, ": ", what,
              " must be ", type, " on CUDA device ", dev);
  TORCH_CHECK(t.dim() == 3 && t.size(2) == dim && (rows < 0 || t.size(0) == rows) &&
                  (heads < 0 || t.size(1) == heads),
              op, ": ", what, " must be [", rows, ", ", heads, ", ", dim, "] (-1: any), got ",
              t.sizes());
  TORCH_CHECK(t.stride(2) == 1, op, ": the last dimension of ", what, " must be contiguous");
  return {t.data_ptr(), t.stride(0), t.stride(1)};
}

template <typename T>
T* flat(const char* op, const char* what, const at::Tensor& t, at::ScalarType type,
        at::IntArrayRef shape, int dev) {
  TORCH_CHECK(t.scalar_type() == type && t.is_cuda() && t.get_device() == dev &&
                  t.sizes() == shape && t.is_contiguous(),
              op, ": ", what, " must be a contiguous ", type, " tensor ", shape, " on CUDA device ",
              dev);
  return static_cast<T*>(t.data_ptr());
}

Rows weights_of(const char* op, const char* what, const at::Tensor& t, const Handle& h) {
  TORCH_CHECK(t.scalar_type() == at::kFloat && t.is_cuda() && t.get_device() == h.dev &&
                  t.dim() == 3 && t.size(0) == h.kv.batch && t.size(1) == h.kv.kv_heads &&
                  t.size(2) >= h.capacity && (t.size(2) <= 1 || t.stride(2) == 1),
              op, ": ", what, " must be float32 [", h.kv.batch, ", ", h.kv.kv_heads, ", >= ",
              h.capacity, "] on CUDA device ", h.dev, ", contiguous in its last dimension");
  return {t.data_ptr(), t.stride(0), t.stride(1)};
}

at::Tensor empty(at::IntArrayRef shape, at::ScalarType type, int dev) {
  return at::detail::empty_cuda(shape, type, at::Device(at::kCUDA, dev), std::nullopt);
}

void* stream(int dev) { return c10::cuda::getCurrentCUDAStream(dev).stream(); }

// gammas, eps, tables, positions and layout as QKNormRotary takes them.
InfercHeadRotary rotary_of(const char* op, PyObject* const* a, int dev, int64_t dim,
                           int64_t tokens) {
  InfercHeadRotary r{};
  const at::Tensor *gq = maybe(a[0], op, "q_gamma"), *gk = maybe(a[1], op, "k_gamma");
  const at::Tensor *cos = maybe(a[3], op, "cos"), *sin = maybe(a[4], op, "sin");
  const at::Tensor* pos = maybe(a[5], op, "positions");
  if (gq) r.q_gamma = flat<float>(op, "q_gamma", *gq, at::kFloat, {dim}, dev);
  if (gk) r.k_gamma = flat<float>(op, "k_gamma", *gk, at::kFloat, {dim}, dev);
  r.eps = (float)number(a[2]);
  TORCH_CHECK(!cos == !sin, op, ": cos and sin come together");
  if (cos) {
    TORCH_CHECK(cos->dim() == 2 && cos->size(0) >= 1 && cos->size(1) >= 1 &&
                    2 * cos->size(1) <= dim,
                op, ": cos and sin must be [positions, rotary_dim / 2], rotary_dim at most "
                "head_dim");
    r.cos = flat<float>(op, "cos", *cos, at::kFloat, cos->sizes(), dev);
    r.sin = flat<float>(op, "sin", *sin, at::kFloat, cos->sizes(), dev);
    r.table_len = cos->size(0);
    r.table_stride = cos->size(1);
    r.rotary_dim = (int32_t)(2 * cos->size(1));
  }
  if (pos) r.positions = flat<int32_t>(op, "positions", *pos, at::kInt, {tokens}, dev);
  const int interleaved = PyObject_IsTrue(a[6]);
  if (interleaved < 0) throw std::runtime_error("");
  r.interleaved = interleaved;
  return r;
}

const int32_t* cu_of(const char* op, PyObject* o, const Handle& h, int64_t tokens) {
  if (const at::Tensor* cu = maybe(o, op, "cu_tokens"))
    return flat<int32_t>(op, "cu_tokens", *cu, at::kInt, {h.kv.batch + 1}, h.dev);
  TORCH_CHECK(tokens == h.kv.batch, op, ": without cu_tokens there is one token per sequence");
  return nullptr;
}

// (k_cache, v_cache, page_table, lens) -> handle
PyObject* make(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    arity(n, 4);
    const char* op = "PagedKV";
    const at::Tensor &k = tensor(a[0], op, "k_cache"), &v = tensor(a[1], op, "v_cache");
    const at::Tensor &table = tensor(a[2], op, "page_table"), &lens = tensor(a[3], op, "lens");
    TORCH_CHECK(k.is_cuda(), op, ": tensors must be on a CUDA device");
    TORCH_CHECK(dtype_code(k.scalar_type()) != 0, op,
                ": caches must be float32, float16 or bfloat16");
    TORCH_CHECK(k.dim() == 4 && v.sizes() == k.sizes() && v.scalar_type() == k.scalar_type() &&
                    v.device() == k.device(),
                op, ": k_cache and v_cache must be alike, [pages, kv_heads, page, head_dim]");
    TORCH_CHECK(k.size(1) >= 1 && k.size(2) >= 1, op,
                ": caches must have a key head and a position per page at least");
    TORCH_CHECK(k.stride(3) == 1 && v.stride(3) == 1, op,
                ": the caches' last dimension must be contiguous");
    TORCH_CHECK(table.dim() == 2 && table.scalar_type() == at::kInt &&
                    table.device() == k.device() && (table.size(1) <= 1 || table.stride(1) == 1),
                op, ": page_table must be int32 [batch, max_pages] with contiguous rows");
    TORCH_CHECK(lens.dim() == 1 && lens.scalar_type() == at::kInt && lens.device() == k.device() &&
                    lens.size(0) == table.size(0) && lens.is_contiguous(),
                op, ": lens must be a contiguous int32 tensor [batch]");
    auto h = std::make_unique<Handle>();
    h->type = k.scalar_type();
    h->dev = k.get_device();
    h->k = k;
    h->v = v;
    h->table = table;
    h->lens = lens;
    InfercPagedKv& kv = h->kv;
    kv = InfercPagedKv{};
    kv.k = k.data_ptr();
    kv.v = v.data_ptr();
    kv.page_table = static_cast<const int32_t*>(table.data_ptr());
    kv.lens = static_cast<const int32_t*>(lens.data_ptr());
    kv.k_page_stride = k.stride(0);
    kv.k_head_stride = k.stride(1);
    kv.k_token_stride = k.stride(2);
    kv.v_page_stride = v.stride(0);
    kv.v_head_stride = v.stride(1);
    kv.v_token_stride = v.stride(2);
    kv.num_pages = k.size(0);
    kv.kv_heads = k.size(1);
    kv.page_size = k.size(2);
    kv.batch = table.size(0);
    kv.max_pages = table.size(1);
    kv.table_stride = kv.batch <= 1 ? std::max(table.stride(0), kv.max_pages) : table.stride(0);
    kv.head_dim = (int32_t)k.size(3);
    kv.dtype = dtype_code(h->type);
    h->capacity = kv.max_pages * kv.page_size;
    PyObject* c = PyCapsule_New(h.get(), kHandle, [](PyObject* o) {
      delete static_cast<Handle*>(PyCapsule_GetPointer(o, kHandle));
    });
    if (c) h.release();
    return c;
  });
}

// (handle, q, scale, weights, out) -> out
PyObject* attend(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    arity(n, 5);
    const char* op = "PagedDecodeAttention";
    Handle& h = handle(a[0]);
    const at::Tensor& q = tensor(a[1], op, "q");
    const int64_t dim = h.kv.head_dim, batch = h.kv.batch;
    const Rows rq = rows_of(op, "q", q, h.type, h.dev, batch, -1, dim);
    const int64_t heads = q.size(1);
    TORCH_CHECK(heads >= 1 && heads % h.kv.kv_heads == 0, op,
                ": the query heads must be a multiple of kv_heads");
    const float scale = a[2] == Py_None ? 1.0f / std::sqrt((float)dim) : (float)number(a[2]);
    Rows rw;
    const at::Tensor* w = maybe(a[3], op, "weights");
    if (w) rw = weights_of(op, "weights", *w, h);
    const c10::cuda::OptionalCUDAGuard guard(at::Device(at::kCUDA, h.dev));
    at::Tensor out;
    if (const at::Tensor* given = maybe(a[4], op, "out")) out = *given;
    else out = empty({batch, heads, dim}, h.type, h.dev);
    const Rows ro = rows_of(op, "out", out, h.type, h.dev, batch, heads, dim);
    auto [size, fresh] = h.scratch.try_emplace({heads, w != nullptr}, -1);
    if (fresh) {
      size->second = inferc_dev_paged_decode_attention_workspace(&h.kv, heads, w != nullptr);
      if (size->second < 0) {
        h.scratch.erase(size);
        throw Status{INFERC_ERR_INVALID};
      }
    }
    // scratch of this call alone, in stream order, so that calls on other streams may overlap
    c10::DataPtr ws;
    if (size->second) ws = c10::cuda::CUDACachingAllocator::get()->allocate(size->second);
    ok(inferc_dev_paged_decode_attention(&h.kv, rq.p, rq.row, rq.head, heads, scale, ro.p, ro.row,
                                         ro.head, static_cast<float*>(rw.p), rw.row, rw.head,
                                         ws.get(), size->second, stream(h.dev)));
    return THPVariable_Wrap(std::move(out));
  });
}

// (handle, k, v, cu_tokens)
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    arity(n, 4);
    const char* op = "PagedKVAppend";
    const Handle& h = handle(a[0]);
    const at::Tensor &k = tensor(a[1], op, "k"), &v = tensor(a[2], op, "v");
    const int64_t dim = h.kv.head_dim, hk = h.kv.kv_heads;
    const Rows rk = rows_of(op, "k", k, h.type, h.dev, -1, hk, dim);
    const int64_t tokens = k.size(0);
    const Rows rv = rows_of(op, "v", v, h.type, h.dev, tokens, hk, dim);
    const int32_t* cu = cu_of(op, a[3], h, tokens);
    const c10::cuda::OptionalCUDAGuard guard(at::Device(at::kCUDA, h.dev));
    ok(inferc_dev_paged_kv_append(&h.kv, nullptr, nullptr, 0, 0, rk.p, rk.row, rk.head, rv.p,
                                  rv.row, rv.head, nullptr, 0, 0, 0, cu, tokens, stream(h.dev)));
    Py_RETURN_NONE;
  });
}

// (handle, q, k, v, q_gamma, k_gamma, eps, cos, sin, positions, interleaved, cu_tokens, q_out)
PyObject* norm_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    arity(n, 13);
    const char* op = "QKNormRotaryAppend";
    const Handle& h = handle(a[0]);
    const at::Tensor& q = tensor(a[1], op, "q");
    const at::Tensor &k = tensor(a[2], op, "k"), &v = tensor(a[3], op, "v");
    const int64_t dim = h.kv.head_dim, hk = h.kv.kv_heads;
    const Rows rq = rows_of(op, "q", q, h.type, h.dev, -1, -1, dim);
    const int64_t tokens = q.size(0), heads = q.size(1);
    const Rows rk = rows_of(op, "k", k, h.type, h.dev, tokens, hk, dim);
    const Rows rv = rows_of(op, "v", v, h.type, h.dev, tokens, hk, dim);
    const InfercHeadRotary rot = rotary_of(op, a + 4, h.dev, dim, tokens);
    const int32_t* cu = cu_of(op, a[11], h, tokens);
    const c10::cuda::OptionalCUDAGuard guard(at::Device(at::kCUDA, h.dev));
    at::Tensor out;
    if (const at::Tensor* given = maybe(a[12], op, "q_out")) out = *given;
    else out = empty({tokens, heads, dim}, h.type, h.dev);
    const Rows ro = rows_of(op, "q_out", out, h.type, h.dev, tokens, heads, dim);
    ok(inferc_dev_paged_kv_append(&h.kv, &rot, rq.p, rq.row, rq.head, rk.p, rk.row, rk.head, rv.p,
                                  rv.row, rv.head, ro.p, ro.row, ro.head, heads, cu, tokens,
                                  stream(h.dev)));
    return THPVariable_Wrap(std::move(out));
  });
}

// (q, k, q_gamma, k_gamma, eps, cos, sin, positions, interleaved, q_out, k_out) -> (q_out, k_out)
PyObject* norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    arity(n, 11);
    const char* op = "QKNormRotary";
    const at::Tensor &q = tensor(a[0], op, "q"), &k = tensor(a[1], op, "k");
    const at::ScalarType type = q.scalar_type();
    TORCH_CHECK(q.is_cuda() && dtype_code(type) != 0 && q.dim() == 3, op,
                ": q must be [tokens, heads, head_dim], float32, float16 or bfloat16, on a CUDA "
                "device");
    const int dev = q.get_device();
    const int64_t tokens = q.size(0), heads = q.size(1), dim = q.size(2);
    const Rows rq = rows_of(op, "q", q, type, dev, -1, -1, dim);
    const Rows rk = rows_of(op, "k", k, type, dev, tokens, -1, dim);
    const int64_t hk = k.size(1);
    const InfercHeadRotary rot = rotary_of(op, a + 2, dev, dim, tokens);
    const c10::cuda::OptionalCUDAGuard guard(at::Device(at::kCUDA, dev));
    at::Tensor qo, ko;
    if (const at::Tensor* given = maybe(a[9], op, "q_out")) qo = *given;
    else qo = empty({tokens, heads, dim}, type, dev);
    if (const at::Tensor* given = maybe(a[10], op, "k_out")) ko = *given;
    else ko = empty({tokens, hk, dim}, type, dev);
    const Rows ro = rows_of(op, "q_out", qo, type, dev, tokens, heads, dim);
    const Rows so = rows_of(op, "k_out", ko, type, dev, tokens, hk, dim);
    ok(inferc_dev_qk_norm_rotary(&rot, dtype_code(type), rq.p, rq.row, rq.head, rk.p, rk.row,
                                 rk.head, ro.p, ro.row, ro.head, so.p, so.row, so.head, tokens,
                                 heads, hk, dim, stream(dev)));
    return PyTuple_Pack(2, py::reinterpret_steal<py::object>(THPVariable_Wrap(std::move(qo))).ptr(),
                        py::reinterpret_steal<py::object>(THPVariable_Wrap(std::move(ko))).ptr());
  });
}

// (handle, weights, keep, recent, dst_table, weights_out, lens_out, kept)
//   -> (lens_out, kept, weights_out)
PyObject* evict(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    arity(n, 8);
    const char* op = "PagedKVEvict";
    const Handle& h = handle(a[0]);
    const at::Tensor& w = tensor(a[1], op, "weights");
    const int64_t keep = integer(a[2]), recent = integer(a[3]), batch = h.kv.batch;
    TORCH_CHECK(keep >= 1 && recent >= 0 && recent <= keep, op,
                ": keep must be at least 1 and recent in [0, keep]");
    const Rows rw = weights_of(op, "weights", w, h);
    Rows wo;
    const at::Tensor* given_w = maybe(a[5], op, "weights_out");
    if (given_w) wo = weights_of(op, "weights_out", *given_w, h);
    const int32_t* dst = nullptr;
    int64_t dst_pages = 0, dst_stride = 0;
    if (const at::Tensor* t = maybe(a[4], op, "dst_table")) {
      TORCH_CHECK(t->scalar_type() == at::kInt && t->is_cuda() && t->get_device() == h.dev &&
                      t->dim() == 2 && t->size(0) == batch &&
                      (t->size(1) <= 1 || t->stride(1) == 1),
                  op, ": dst_table must be int32 [batch, pages] with contiguous rows on CUDA device ",
                  h.dev);
      dst = static_cast<const int32_t*>(t->data_ptr());
      dst_pages = t->size(1);
      dst_stride = batch <= 1 ? std::max(t->stride(0), dst_pages) : t->stride(0);
    }
    const c10::cuda::OptionalCUDAGuard guard(at::Device(at::kCUDA, h.dev));
    at::Tensor lens, kept;
    if (const at::Tensor* given = maybe(a[6], op, "lens_out")) lens = *given;
    else lens = empty({batch}, at::kInt, h.dev);
    if (const at::Tensor* given = maybe(a[7], op, "kept")) kept = *given;
    else kept = empty({batch, h.kv.kv_heads, keep}, at::kInt, h.dev);
    int32_t* pl = flat<int32_t>(op, "lens_out", lens, at::kInt, {batch}, h.dev);
    int32_t* pk = flat<int32_t>(op, "kept", kept, at::kInt, {batch, h.kv.kv_heads, keep}, h.dev);
    ok(inferc_dev_paged_kv_evict(&h.kv, dst, dst_pages, dst_stride, static_cast<float*>(rw.p),
                                 rw.row, rw.head, static_cast<float*>(wo.p), wo.row, wo.head, keep,
                                 recent, pl, pk, stream(h.dev)));
    return PyTuple_Pack(3,
                        py::reinterpret_steal<py::object>(THPVariable_Wrap(std::move(lens))).ptr(),
                        py::reinterpret_steal<py::object>(THPVariable_Wrap(std::move(kept))).ptr(),
                        given_w ? a[5] : a[1]);
  });
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyMethodDef method(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F)), METH_FASTCALL,
          nullptr};
}

PyMethodDef kMethods[] = {method<make>("make"),
                          method<attend>("attend"),
                          method<append>("append"),
                          method<norm_append>("norm_append"),
                          method<norm>("norm"),
                          method<evict>("evict"),
                          {nullptr, nullptr, 0, nullptr}};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_paged", nullptr, -1, kMethods, nullptr, nullptr,
                       nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__paged(void) { return PyModule_Create(&kModule); }
