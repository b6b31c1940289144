// torch_paged.cpp - the PyTorch side of the paged KV-cache operators: checks of
// the tensors, outputs and workspaces, and the call of the C ABI
// (include/ddq_b200.h), as a CPython module.
//
// A step's kernels take 2 to 15 us; the same checks in Python with a ctypes call
// took 16 to 30 us of the host a call.  This module knows nothing of CUDA
// kernels: it gets the addresses of the library's entry points from bind().
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/TensorImpl.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>

#include "../../include/ddq_b200.h"

namespace {

struct Entries {
  decltype(&ddq_plan_step) plan_step = nullptr;
  decltype(&ddq_paged_rope_kv) rope_kv = nullptr;
  decltype(&ddq_paged_prefill_attention_workspace_size) prefill_size = nullptr;
  decltype(&ddq_paged_decode_attention_workspace_size) decode_size = nullptr;
  decltype(&ddq_paged_prefill_attention) prefill = nullptr;
  decltype(&ddq_paged_decode_attention) decode = nullptr;
  decltype(&ddq_status_string) status_string = nullptr;
} g;

void check_status(int st, const char* what) {
  TORCH_CHECK(st == DDQ_OK, what, ": ", g.status_string(st), " (ddq status ", st, ")");
}

const at::Tensor& tensor(PyObject* o, const char* what, const char* name) {
  TORCH_CHECK(THPVariable_Check(o), what, ": ", name, " must be a tensor");
  return THPVariable_Unpack(o);
}

int64_t integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}

double real(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return v;
}

void check_page_size(int64_t ps, const char* what) {
  TORCH_CHECK(ps >= DDQ_PAGE_SIZE_MIN && ps <= DDQ_PAGE_SIZE_MAX && (ps & (ps - 1)) == 0, what,
              ": page_size must be a power of two from ", DDQ_PAGE_SIZE_MIN, " to ",
              DDQ_PAGE_SIZE_MAX);
}

bool vec(const at::Tensor& t, at::ScalarType type, c10::Device dev) {
  return t.scalar_type() == type && t.device() == dev && t.dim() == 1 && t.is_contiguous();
}

// Element stride of dimension i; a dimension of one element has no stride that
// matters (torch leaves any there).
int64_t stride(const at::Tensor& t, int i) {
  return t.size(i) > 1 ? t.stride(i) : t.size(-1);
}

// The unit inner stride (or an inner dimension of one element).
bool inner1(const at::Tensor& t) { return t.size(-1) == 1 || t.stride(-1) == 1; }

struct Pool {
  ddq_paged_cache c;
  c10::Device dev;
  at::ScalarType type;
};

Pool pool(const at::Tensor& k, const at::Tensor& v, const char* what) {
  TORCH_CHECK(k.is_cuda() && (k.scalar_type() == at::kHalf || k.scalar_type() == at::kBFloat16) &&
                  k.dim() == 4,
              what, ": k_pages must be fp16 or bf16 CUDA [P, Hkv, page_size, D]");
  TORCH_CHECK(v.scalar_type() == k.scalar_type() && v.device() == k.device() &&
                  v.sizes() == k.sizes(),
              what, ": k_pages and v_pages must have the same type and shape");
  check_page_size(k.size(2), what);
  TORCH_CHECK(k.size(3) == 64 || k.size(3) == 128, what, ": head_dim must be 64 or 128");
  const int64_t a = stride(k, 0), b = stride(k, 1), r = stride(k, 2);
  TORCH_CHECK(k.stride(3) == 1 && (a | b | r) % 8 == 0, what,
              ": pages need a unit inner stride and outer strides that are multiples of 8");
  TORCH_CHECK(v.stride(3) == 1 && stride(v, 0) == a && stride(v, 1) == b && stride(v, 2) == r,
              what, ": k_pages and v_pages must have the same strides");
  return Pool{ddq_paged_cache{k.data_ptr(), v.data_ptr(), k.size(0), k.size(2), k.size(1),
                              k.size(3), a, b, r,
                              k.scalar_type() == at::kHalf ? DDQ_DTYPE_F16 : DDQ_DTYPE_BF16},
              k.device(), k.scalar_type()};
}

void* stream_of(c10::Device dev) { return c10::cuda::getCurrentCUDAStream(dev.index()).stream(); }

at::Tensor empty(at::IntArrayRef shape, at::ScalarType type, c10::Device dev) {
  return at::empty(shape, at::TensorOptions().dtype(type).device(dev));
}

PyObject* plan_step(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  constexpr const char* W = "plan_step";
  TORCH_CHECK(n == 8, W, ": 8 arguments");
  const at::Tensor& cached = tensor(a[0], W, "cached");
  const at::Tensor& fresh = tensor(a[1], W, "new");
  const at::Tensor& table = tensor(a[2], W, "block_table");
  const at::Tensor& free_pages = tensor(a[3], W, "free_pages");
  const int64_t ps = integer(a[4]), T = integer(a[5]), prefix = integer(a[7]);
  const bool has_head = a[6] != Py_None;
  const c10::Device dev = cached.device();
  const int64_t R = cached.numel();
  TORCH_CHECK(cached.is_cuda() && vec(cached, at::kInt, dev), W,
              ": cached must be int32 CUDA [R]");
  TORCH_CHECK(vec(fresh, at::kInt, dev) && fresh.numel() == R, W,
              ": new must be int32 CUDA [R]");
  TORCH_CHECK(table.scalar_type() == at::kInt && table.device() == dev && table.dim() == 2 &&
                  table.size(0) == R && table.size(1) > 0 && inner1(table) &&
                  (R == 1 || table.stride(0) >= table.size(1)),
              W, ": block_table must be int32 CUDA [R, width] with distinct rows");
  TORCH_CHECK(vec(free_pages, at::kInt, dev), W, ": free_pages must be int32 CUDA [F]");
  const int32_t* head = nullptr;
  if (has_head) {
    const at::Tensor& h = tensor(a[6], W, "free_head");
    TORCH_CHECK(vec(h, at::kInt, dev) && h.numel() == 1, W, ": free_head must be int32 CUDA [1]");
    head = h.data_ptr<int32_t>();
  }
  TORCH_CHECK(R >= 1, W, ": at least one request");
  check_page_size(ps, W);
  TORCH_CHECK(T >= 0 && prefix >= 0, W, ": negative count");
  c10::cuda::OptionalCUDAGuard guard;
  if (dev.index() != c10::cuda::current_device()) guard.set_device(dev);
  // one allocation for all outputs (six took a third of the call)
  const int64_t words = 4 * T + (R + 1) + R + 1 + T;  // int32
  const at::Tensor base = empty({(words + 1) / 2}, at::kLong, dev);
  int64_t at32 = 0;
  auto part = [&](int64_t count, at::ScalarType type) {
    auto impl = c10::make_intrusive<c10::TensorImpl>(
        c10::Storage(base.storage()), c10::DispatchKeySet(c10::DispatchKey::CUDA),
        c10::scalarTypeToTypeMeta(type));
    const int64_t size = type == at::kLong ? 2 : 1;
    impl->set_storage_offset(at32 / size);
    impl->set_sizes_contiguous({count});
    at32 += count * size;
    return at::Tensor(std::move(impl));
  };
  at::Tensor slots = part(T, at::kLong), positions = part(T, at::kLong);
  at::Tensor cu = part(R + 1, at::kInt), lens = part(R, at::kInt), out_head = part(1, at::kInt),
             seq = part(T, at::kInt);
  check_status(
      g.plan_step(cached.data_ptr<int32_t>(), fresh.data_ptr<int32_t>(),
                  table.data_ptr<int32_t>(), R > 1 ? table.stride(0) : table.size(1),
                  table.size(1), free_pages.data_ptr<int32_t>(), free_pages.numel(), head, ps,
                  prefix, cu.data_ptr<int32_t>(), lens.data_ptr<int32_t>(),
                  slots.data_ptr<int64_t>(), positions.data_ptr<int64_t>(),
                  seq.data_ptr<int32_t>(), out_head.data_ptr<int32_t>(), R, T, stream_of(dev)),
      W);
  PyObject* t = PyTuple_New(6);
  if (!t) throw python_error();
  PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(std::move(cu)));
  PyTuple_SET_ITEM(t, 1, THPVariable_Wrap(std::move(lens)));
  PyTuple_SET_ITEM(t, 2, THPVariable_Wrap(std::move(slots)));
  PyTuple_SET_ITEM(t, 3, THPVariable_Wrap(std::move(positions)));
  PyTuple_SET_ITEM(t, 4, THPVariable_Wrap(std::move(seq)));
  PyTuple_SET_ITEM(t, 5, THPVariable_Wrap(std::move(out_head)));
  return t;
  END_HANDLE_TH_ERRORS
}

PyObject* rope_kv_write(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  constexpr const char* W = "rope_kv_write";
  TORCH_CHECK(n == 11, W, ": 11 arguments");
  const Pool p = pool(tensor(a[1], W, "k_pages"), tensor(a[2], W, "v_pages"), W);
  const at::Tensor& qkv = tensor(a[0], W, "qkv");
  const at::Tensor& cos = tensor(a[3], W, "cos");
  const at::Tensor& sin = tensor(a[4], W, "sin");
  const at::Tensor& slots = tensor(a[5], W, "slots");
  const at::Tensor& positions = tensor(a[6], W, "positions");
  const int64_t hq = integer(a[7]), hkv = integer(a[8]), d = integer(a[9]);
  TORCH_CHECK(hkv == p.c.Hkv && d == p.c.D && hq >= 1 && hq <= 1024, W,
              ": heads do not match the pages");
  const int64_t width = (hq + 2 * hkv) * d;
  TORCH_CHECK(qkv.scalar_type() == p.type && qkv.device() == p.dev && qkv.dim() == 2 &&
                  qkv.size(1) == width && qkv.stride(1) == 1,
              W, ": qkv must be [T, (Hq + 2 Hkv) * D] of the pages' type, unit inner stride");
  TORCH_CHECK(cos.scalar_type() == at::kFloat && cos.device() == p.dev && cos.dim() == 2 &&
                  cos.size(1) == d && cos.is_contiguous() && sin.scalar_type() == at::kFloat &&
                  sin.device() == p.dev && sin.sizes() == cos.sizes() && sin.is_contiguous(),
              W, ": cos and sin must be contiguous fp32 CUDA [max_pos, D]");
  const int64_t T = qkv.size(0);
  TORCH_CHECK(vec(slots, at::kLong, p.dev) && slots.numel() == T, W,
              ": slots must be int64 CUDA [T]");
  TORCH_CHECK(vec(positions, at::kLong, p.dev) && positions.numel() == T, W,
              ": positions must be int64 CUDA [T]");
  c10::cuda::OptionalCUDAGuard guard;
  if (p.dev.index() != c10::cuda::current_device()) guard.set_device(p.dev);
  at::Tensor out;
  if (a[10] == Py_None) {
    out = empty({T, hq, d}, p.type, p.dev);
  } else {
    out = tensor(a[10], W, "out");
    TORCH_CHECK(out.scalar_type() == p.type && out.device() == p.dev && out.is_contiguous() &&
                    out.dim() == 3 && out.size(0) == T && out.size(1) == hq && out.size(2) == d,
                W, ": out must be contiguous [T, Hq, D] of the pages' type");
  }
  check_status(g.rope_kv(qkv.data_ptr(), T > 1 ? qkv.stride(0) : width, &p.c,
                         cos.data_ptr<float>(), sin.data_ptr<float>(), cos.size(0),
                         slots.data_ptr<int64_t>(), positions.data_ptr<int64_t>(),
                         out.data_ptr(), T, hq, stream_of(p.dev)),
               W);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// What the two attention calls have in common: q, out, table, lengths, slopes.
struct Attn {
  const at::Tensor& q;
  const at::Tensor& table;
  const at::Tensor& lens;
  const float* slopes;
  float scale, cap;
  const int32_t* prefix_pages;
  int64_t prefix_len;
  at::Tensor out;
  int64_t table_stride;
};

Attn attention_args(const Pool& p, const at::Tensor& q, const at::Tensor& table,
                    const at::Tensor& lens, int64_t rows, PyObject* scale, PyObject* softcap,
                    PyObject* slopes, PyObject* prefix_pages, PyObject* prefix_len,
                    PyObject* out, const char* W) {
  TORCH_CHECK(q.scalar_type() == p.type && q.device() == p.dev && q.dim() == 3 &&
                  q.size(2) == p.c.D && q.size(1) >= 1 && q.size(1) % p.c.Hkv == 0 &&
                  q.stride(2) == 1,
              W, ": q must be [T, Hq, D] of the pages' type, Hq a multiple of Hkv");
  if (rows < 0) rows = q.size(0);
  TORCH_CHECK(table.scalar_type() == at::kInt && table.device() == p.dev && table.dim() == 2 &&
                  table.size(0) == rows && table.size(1) > 0 && inner1(table) &&
                  (rows <= 1 || table.stride(0) >= table.size(1)),
              W, ": block_table must be int32 CUDA [requests, width], its rows apart");
  TORCH_CHECK(vec(lens, at::kInt, p.dev) && lens.numel() == rows, W,
              ": lens must be int32 CUDA [requests]");
  Attn r{q, table, lens, nullptr, (float)real(scale), (float)real(softcap), nullptr,
         integer(prefix_len), at::Tensor(), rows > 1 ? table.stride(0) : table.size(1)};
  if (slopes != Py_None) {
    const at::Tensor& s = tensor(slopes, W, "slopes");
    TORCH_CHECK(vec(s, at::kFloat, p.dev) && s.numel() == q.size(1), W,
                ": slopes must be fp32 CUDA [Hq]");
    r.slopes = s.data_ptr<float>();
  }
  TORCH_CHECK(std::isfinite(r.cap) && r.cap >= 0.f, W,
              ": softcap must be finite and not negative");
  TORCH_CHECK(std::isfinite(r.scale), W, ": scale must be finite");
  TORCH_CHECK(r.prefix_len >= 0, W, ": prefix_len must not be negative");
  if (r.prefix_len > 0) {
    TORCH_CHECK(prefix_pages != Py_None, W, ": prefix_len needs prefix_pages");
    const at::Tensor& t = tensor(prefix_pages, W, "prefix_pages");
    TORCH_CHECK(vec(t, at::kInt, p.dev), W, ": prefix_pages must be int32 CUDA [pages]");
    TORCH_CHECK(t.numel() * p.c.page_size >= r.prefix_len, W,
                ": prefix_pages holds fewer than prefix_len keys");
    r.prefix_pages = t.data_ptr<int32_t>();
  }
  if (out != Py_None) {
    r.out = tensor(out, W, "out");
    TORCH_CHECK(r.out.scalar_type() == p.type && r.out.device() == p.dev &&
                    r.out.sizes() == q.sizes() && r.out.stride(2) == 1,
                W, ": out must have the shape and type of q");
  }
  return r;
}

// Partial results of a split key axis: from the caching allocator for each call,
// so that calls on different streams and captured graphs never share it.
at::Tensor workspace(size_t bytes, c10::Device dev) {
  return bytes ? empty({(int64_t)bytes}, at::kByte, dev) : at::Tensor();
}

PyObject* prefill_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  constexpr const char* W = "prefill_attention";
  TORCH_CHECK(n == 13, W, ": 13 arguments");
  const Pool p = pool(tensor(a[1], W, "k_pages"), tensor(a[2], W, "v_pages"), W);
  const at::Tensor& cu = tensor(a[4], W, "cu_new");
  TORCH_CHECK(vec(cu, at::kInt, p.dev) && cu.numel() >= 1, W,
              ": cu_new must be int32 CUDA [R + 1]");
  const int64_t R = cu.numel() - 1;
  Attn r = attention_args(p, tensor(a[0], W, "q"), tensor(a[3], W, "block_table"),
                          tensor(a[5], W, "lens"), R, a[6], a[7], a[8], a[10], a[11], a[12], W);
  const int32_t* bidir = nullptr;
  if (a[9] != Py_None) {
    const at::Tensor& b = tensor(a[9], W, "bidir");
    TORCH_CHECK(vec(b, at::kInt, p.dev) && b.numel() == R, W, ": bidir must be int32 CUDA [R]");
    bidir = b.data_ptr<int32_t>();
  }
  c10::cuda::OptionalCUDAGuard guard;
  if (p.dev.index() != c10::cuda::current_device()) guard.set_device(p.dev);
  if (!r.out.defined()) r.out = empty(r.q.sizes(), p.type, p.dev);
  const int64_t T = r.q.size(0), Hq = r.q.size(1), width = r.table.size(1);
  const size_t bytes =
      g.prefill_size(T, R, Hq, p.c.Hkv, p.c.D, width, p.c.page_size, r.prefix_len);
  at::Tensor ws = workspace(bytes, p.dev);
  check_status(
      g.prefill(r.q.data_ptr(), stride(r.q, 0), stride(r.q, 1), &p.c, r.table.data_ptr<int32_t>(),
                r.table_stride, width, cu.data_ptr<int32_t>(), r.lens.data_ptr<int32_t>(), bidir,
                r.prefix_pages, r.prefix_len, r.slopes, r.scale, r.cap, r.out.data_ptr(),
                stride(r.out, 0), stride(r.out, 1), T, R, Hq,
                ws.defined() ? ws.data_ptr() : nullptr, bytes, stream_of(p.dev)),
      W);
  return THPVariable_Wrap(std::move(r.out));
  END_HANDLE_TH_ERRORS
}

PyObject* decode_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  constexpr const char* W = "decode_attention";
  TORCH_CHECK(n == 11, W, ": 11 arguments");
  const Pool p = pool(tensor(a[1], W, "k_pages"), tensor(a[2], W, "v_pages"), W);
  Attn r = attention_args(p, tensor(a[0], W, "q"), tensor(a[3], W, "block_table"),
                          tensor(a[4], W, "lens"), -1, a[5], a[8], a[9], a[6], a[7], a[10], W);
  c10::cuda::OptionalCUDAGuard guard;
  if (p.dev.index() != c10::cuda::current_device()) guard.set_device(p.dev);
  if (!r.out.defined()) r.out = empty(r.q.sizes(), p.type, p.dev);
  const int64_t B = r.q.size(0), Hq = r.q.size(1), width = r.table.size(1);
  const size_t bytes =
      g.decode_size(B, Hq, p.c.Hkv, p.c.D, width, p.c.page_size, r.prefix_len);
  at::Tensor ws = workspace(bytes, p.dev);
  check_status(
      g.decode(r.q.data_ptr(), stride(r.q, 0), stride(r.q, 1), &p.c, r.table.data_ptr<int32_t>(),
               r.table_stride, width, r.lens.data_ptr<int32_t>(), r.prefix_pages, r.prefix_len,
               r.slopes, r.scale, r.cap, r.out.data_ptr(), stride(r.out, 0), stride(r.out, 1), B,
               Hq, ws.defined() ? ws.data_ptr() : nullptr, bytes, stream_of(p.dev)),
      W);
  return THPVariable_Wrap(std::move(r.out));
  END_HANDLE_TH_ERRORS
}

// bind(addresses of the entry points, in the order of Entries)
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK(n == 7, "bind: 7 addresses");
  void* p[7];
  for (int i = 0; i < 7; ++i) p[i] = reinterpret_cast<void*>(integer(a[i]));
  g.plan_step = reinterpret_cast<decltype(g.plan_step)>(p[0]);
  g.rope_kv = reinterpret_cast<decltype(g.rope_kv)>(p[1]);
  g.prefill_size = reinterpret_cast<decltype(g.prefill_size)>(p[2]);
  g.decode_size = reinterpret_cast<decltype(g.decode_size)>(p[3]);
  g.prefill = reinterpret_cast<decltype(g.prefill)>(p[4]);
  g.decode = reinterpret_cast<decltype(g.decode)>(p[5]);
  g.status_string = reinterpret_cast<decltype(g.status_string)>(p[6]);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

#define DDQ_FAST(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), \
                     METH_FASTCALL, nullptr}
PyMethodDef methods[] = {DDQ_FAST(bind),
                         DDQ_FAST(plan_step),
                         DDQ_FAST(rope_kv_write),
                         DDQ_FAST(prefill_attention),
                         DDQ_FAST(decode_attention),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_paged", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__paged() { return PyModule_Create(&module); }
