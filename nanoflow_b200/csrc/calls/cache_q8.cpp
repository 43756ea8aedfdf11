// Calls of the 8-bit cache's kernels from Python (module nanoflow_b200.ops._cache_q8): the checks of arguments that the C ABI cannot
// make, the parameter block, and the launch on the tensors' device and its current stream. In C++ because a kernel of a few
// microseconds waits for its call: through ctypes a decode call took 25 us of the host's time, here 0.4 and 2.5 to 3 for its launch.
//
// Functions take positional arguments only; nanoflow_b200/ops/cache_q8.py gives them names, defaults and documentation. The kernel
// library is loaded there, too, and hands over its entry points' addresses.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <initializer_list>
#include <stdexcept>
#include <string>

#include "kernels.h"

namespace {

using at::Tensor;

struct Entries {
  int (*append)(const nfk_rope_append_q8_params*, cudaStream_t) = nullptr;
  int (*read)(const nfk_kv_read_q8_params*, cudaStream_t) = nullptr;
  int (*decode)(const nfk_attn_q8_params*, cudaStream_t) = nullptr;
} entries;

constexpr int kPage = 16;

[[noreturn]] void refuse(const char* what, const std::string& why) { throw std::runtime_error(std::string(what) + ": " + why); }

const char* name_of(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16: return "bfloat16";
    case at::kFloat: return "float32";
    case at::kInt: return "int32";
    case at::kByte: return "uint8";
    default: return "";
  }
}

const Tensor& tensor(const char* what, const char* name, PyObject* o) {
  if (!THPVariable_Check(o)) refuse(what, std::string(name) + " must be a tensor");
  return THPVariable_Unpack(o);
}
// A contiguous tensor of one type on the cache's device.
const Tensor& checked(const char* what, const char* name, PyObject* o, at::ScalarType type, c10::Device device) {
  const Tensor& t = tensor(what, name, o);
  if (t.scalar_type() != type || t.device() != device || !t.is_contiguous())
    refuse(what, std::string(name) + " must be a contiguous " + name_of(type) + " tensor on " + device.str());
  return t;
}
const Tensor* optional(const char* what, const char* name, PyObject* o, at::ScalarType type, c10::Device device) {
  return o == Py_None ? nullptr : &checked(what, name, o, type, device);
}
int whole(PyObject* o, const char* what, const char* name) {
  const long v = PyLong_AsLong(o);
  if ((v == -1 && PyErr_Occurred()) || v < INT32_MIN || v > INT32_MAX) {
    PyErr_Clear();
    refuse(what, std::string(name) + " must be an int of 32 bits");
  }
  return static_cast<int>(v);
}
float real(PyObject* o, const char* what, const char* name) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    refuse(what, std::string(name) + " must be a number");
  }
  return static_cast<float>(v);
}
int count(const char* what, const Tensor& t, const char* name) {
  if (t.numel() > INT32_MAX) refuse(what, std::string(name) + " has too many entries");
  return static_cast<int>(t.numel());
}
const Tensor* status_word(const char* what, PyObject* o, c10::Device device) {
  const Tensor* t = optional(what, "status", o, at::kInt, device);
  if (t != nullptr && t->numel() < 1) refuse(what, "status must have a word");
  return t;
}
unsigned int* word(const Tensor* t) { return t == nullptr ? nullptr : static_cast<unsigned int*>(t->data_ptr()); }

struct Cache {
  const Tensor& pool;
  const Tensor& scale;
  int pages, kv_heads, head_dim, kind;
  c10::Device device;
};
Cache cache(const char* what, PyObject* pool_arg, PyObject* scale_arg) {
  const Tensor& pool = tensor(what, "kv_pool", pool_arg);
  const Tensor& scale = tensor(what, "kv_scale", scale_arg);
  const bool e4m3 = pool.scalar_type() == at::kFloat8_e4m3fn;
  if ((!e4m3 && pool.scalar_type() != at::kChar) || pool.dim() != 5 || !pool.is_contiguous() || !pool.is_cuda())
    refuse(what, "kv_pool must be a contiguous CUDA float8_e4m3fn or int8 [pages, 2, kv_heads, 16, head_dim]");
  if (pool.size(1) != 2 || pool.size(3) != kPage || (pool.size(4) != 64 && pool.size(4) != 128) || pool.size(0) < 1 || pool.size(2) < 1 ||
      pool.size(0) > INT32_MAX || pool.size(2) > 65536)
    refuse(what, "pages hold 16 tokens of keys and of values, head_dim is 64 or 128");
  if (scale.scalar_type() != at::kFloat || !scale.is_contiguous() || scale.sizes() != pool.sizes().slice(0, 4))
    refuse(what, "kv_scale must be a contiguous float32 [pages, 2, kv_heads, 16]");
  if (scale.device() != pool.device()) refuse(what, "tensors on more than one device");
  return Cache{pool, scale, static_cast<int>(pool.size(0)), static_cast<int>(pool.size(2)), static_cast<int>(pool.size(4)),
               e4m3 ? NFK_Q8_E4M3 : NFK_Q8_INT8, pool.device()};
}

// What a kernel writes must not lie over anything else that it reads or writes. (Null: a tensor that the call goes without.)
void apart(const char* what, std::initializer_list<const Tensor*> written, std::initializer_list<const Tensor*> read) {
  struct Span {
    const char *begin, *end;
  } spans[16];
  int n = 0, n_written = 0;
  const auto add = [&](const Tensor* t) {
    if (t == nullptr || t->numel() == 0) return;
    int64_t last = 0;
    for (int64_t d = 0; d < t->dim(); ++d) last += (t->size(d) - 1) * t->stride(d);
    const char* begin = static_cast<const char*>(t->data_ptr());
    spans[n++] = Span{begin, begin + (last + 1) * t->element_size()};
  };
  if (written.size() + read.size() > 16) refuse(what, "too many tensors");
  for (const Tensor* t : written) add(t);
  n_written = n;
  for (const Tensor* t : read) add(t);
  for (int i = 0; i < n_written; ++i)
    for (int j = i + 1; j < n; ++j)
      if (spans[i].begin < spans[j].end && spans[j].begin < spans[i].end) refuse(what, "tensors overlap, and one of them is written");
}

template <class P>
void launch(const char* name, int (*entry)(const P*, cudaStream_t), const P& p, c10::Device device) {
  if (entry == nullptr) refuse(name, "the kernel library is not loaded");
  c10::cuda::OptionalCUDAGuard guard;
  if (device.index() != c10::cuda::current_device()) guard.set_device(device);       // whichever device is the current one
  const int rc = entry(&p, c10::cuda::getCurrentCUDAStream(device.index()).stream());
  if (rc == 0) return;
  refuse(name, rc == 1 ? "bad argument (shape / alignment / size limit)" : rc == 2 ? "CUDA call failed" : "unsupported configuration");
}

// Arguments as they come, and no C++ exception beyond this module.
template <class F>
PyObject* guarded(Py_ssize_t have, Py_ssize_t want, F f) {
  if (have != want) {
    PyErr_Format(PyExc_TypeError, "%zd arguments expected, %zd given", want, have);
    return nullptr;
  }
  try {
    f();
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown error");
    return nullptr;
  }
  Py_RETURN_NONE;
}

// qkv, q_out, kv_pool, kv_scale, inv_freq, positions, token_req, kv_indptr, kv_indices, q_heads, kv_heads, head_dim, q_off, k_off,
// v_off, q_norm, k_norm, eps, cos_sin, status, early_start
PyObject* rope_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 21, [&] {
    const char* what = "rope_append_q8";
    const Cache c = cache(what, a[2], a[3]);
    const Tensor& qkv = tensor(what, "qkv", a[0]);
    nfk_rope_append_q8_params p = {};
    p.q_heads = whole(a[9], what, "q_heads");
    p.kv_heads = whole(a[10], what, "kv_heads");
    p.head_dim = whole(a[11], what, "head_dim");
    p.q_off = whole(a[12], what, "q_off");
    p.k_off = whole(a[13], what, "k_off");
    p.v_off = whole(a[14], what, "v_off");
    p.eps = real(a[17], what, "eps");
    if (qkv.scalar_type() != at::kBFloat16 || qkv.dim() != 2 || qkv.device() != c.device || (qkv.size(1) > 1 && qkv.stride(1) != 1) ||
        qkv.size(0) > INT32_MAX || qkv.size(1) > INT32_MAX)
      refuse(what, "qkv must be a bfloat16 [T, columns] with unit inner stride on " + c.device.str());
    if (c.kv_heads != p.kv_heads || c.head_dim != p.head_dim || p.q_heads < 1 || p.q_heads > 65536) refuse(what, "kv_pool does not have these heads");
    const int64_t T = qkv.size(0), columns = qkv.size(1), hd = p.head_dim;
    if (p.q_off < 0 || p.q_off + p.q_heads * hd > columns || p.k_off < 0 || p.k_off + p.kv_heads * hd > columns || p.v_off < 0 ||
        p.v_off + p.kv_heads * hd > columns)
      refuse(what, "heads lie outside qkv's columns");
    const Tensor& q_out = checked(what, "q_out", a[1], at::kBFloat16, c.device);
    if (q_out.numel() != T * p.q_heads * hd) refuse(what, "q_out must be [T, q_heads * head_dim]");
    const Tensor& inv_freq = checked(what, "inv_freq", a[4], at::kFloat, c.device);
    const Tensor& positions = checked(what, "positions", a[5], at::kInt, c.device);
    const Tensor& token_req = checked(what, "token_req", a[6], at::kInt, c.device);
    const Tensor& kv_indptr = checked(what, "kv_indptr", a[7], at::kInt, c.device);
    const Tensor& kv_indices = checked(what, "kv_indices", a[8], at::kInt, c.device);
    if (positions.numel() != T || token_req.numel() != T || kv_indptr.numel() < 2)
      refuse(what, "positions and token_req have an entry per token, kv_indptr one per request and one more");
    if (inv_freq.numel() != hd / 2) refuse(what, "inv_freq must be float32 [head_dim/2]");
    const Tensor* q_norm = optional(what, "q_norm", a[15], at::kBFloat16, c.device);
    const Tensor* k_norm = optional(what, "k_norm", a[16], at::kBFloat16, c.device);
    if ((q_norm != nullptr && q_norm->numel() != hd) || (k_norm != nullptr && k_norm->numel() != hd)) refuse(what, "norms must be [head_dim]");
    const Tensor* cos_sin = optional(what, "cos_sin", a[18], at::kFloat, c.device);
    if (cos_sin != nullptr && cos_sin->numel() < T * hd) refuse(what, "cos_sin must be [T, head_dim/2, 2]");
    const Tensor* status = status_word(what, a[19], c.device);
    apart(what, {&q_out, &c.pool, &c.scale, status}, {&qkv, &inv_freq, &positions, &token_req, &kv_indptr, &kv_indices, q_norm, k_norm, cos_sin});
    p.qkv = qkv.data_ptr();
    p.ld_qkv = T > 1 ? qkv.stride(0) : (columns + 7) / 8 * 8;
    p.q_out = q_out.data_ptr();
    p.kv_pool = c.pool.data_ptr();
    p.kv_scale = static_cast<float*>(c.scale.data_ptr());
    p.inv_freq = static_cast<const float*>(inv_freq.data_ptr());
    p.cos_sin = cos_sin != nullptr ? static_cast<const float*>(cos_sin->data_ptr()) : nullptr;
    p.positions = static_cast<const int*>(positions.data_ptr());
    p.token_req = static_cast<const int*>(token_req.data_ptr());
    p.kv_indptr = static_cast<const int*>(kv_indptr.data_ptr());
    p.kv_indices = static_cast<const int*>(kv_indices.data_ptr());
    p.q_norm = q_norm != nullptr ? q_norm->data_ptr() : nullptr;
    p.k_norm = k_norm != nullptr ? k_norm->data_ptr() : nullptr;
    p.T = static_cast<int>(T);
    p.num_pages = c.pages;
    p.num_reqs = count(what, kv_indptr, "kv_indptr") - 1;
    p.num_indices = count(what, kv_indices, "kv_indices");
    p.kind = c.kind;
    p.status = word(status);
    p.early_start = whole(a[20], what, "early_start");
    if (T > 0) launch("nfk_rope_append_q8", entries.append, p, c.device);
  });
}

// kv_pool, kv_scale, page_ids, out, status, early_start
PyObject* read(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 6, [&] {
    const char* what = "kv_read_q8";
    const Cache c = cache(what, a[0], a[1]);
    const Tensor& page_ids = checked(what, "page_ids", a[2], at::kInt, c.device);
    const Tensor& out = checked(what, "out", a[3], at::kBFloat16, c.device);
    if (out.dim() != 5 || out.size(0) != page_ids.numel() || out.sizes().slice(1) != c.pool.sizes().slice(1))
      refuse(what, "out must be [pages, 2, kv_heads, 16, head_dim]");
    const Tensor* status = status_word(what, a[4], c.device);
    apart(what, {&out, status}, {&c.pool, &c.scale, &page_ids});
    nfk_kv_read_q8_params p = {};
    p.kv_pool = c.pool.data_ptr();
    p.kv_scale = static_cast<const float*>(c.scale.data_ptr());
    p.out = out.data_ptr();
    p.page_ids = static_cast<const int*>(page_ids.data_ptr());
    p.n_pages = count(what, page_ids, "page_ids");
    p.kv_heads = c.kv_heads;
    p.head_dim = c.head_dim;
    p.num_pages = c.pages;
    p.kind = c.kind;
    p.status = word(status);
    p.early_start = whole(a[5], what, "early_start");
    if (p.n_pages > 0) launch("nfk_kv_read_q8", entries.read, p, c.device);
  });
}

// what, q, out, kv_pool, kv_scale, qo_indptr, kv_indptr, kv_indices, kv_last_page_len, prefix_pages, prefix_len, q_heads, req_begin,
// req_count, sm_scale, num_ctas, workspace, status, early_start
PyObject* decode(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 19, [&] {
    const char* what = PyUnicode_AsUTF8(a[0]);
    if (what == nullptr) {
      PyErr_Clear();
      refuse("attn_decode_q8", "bad name");
    }
    const Cache c = cache(what, a[3], a[4]);
    const Tensor& q = checked(what, "q", a[1], at::kBFloat16, c.device);
    const Tensor& out = checked(what, "out", a[2], at::kBFloat16, c.device);
    nfk_attn_q8_params p = {};
    p.prefix_len = whole(a[10], what, "prefix_len");
    p.q_heads = whole(a[11], what, "q_heads");
    p.req_begin = whole(a[12], what, "req_begin");
    p.req_count = whole(a[13], what, "req_count");
    p.kv_heads = c.kv_heads;
    p.head_dim = c.head_dim;
    p.num_pages = c.pages;
    p.kind = c.kind;
    p.sm_scale = a[14] == Py_None ? (c.head_dim == 128 ? 0.08838834764831845f : 0.125f) : real(a[14], what, "sm_scale");
    p.num_ctas = whole(a[15], what, "num_ctas");
    if (p.q_heads < 1 || p.q_heads % p.kv_heads != 0 || p.q_heads / p.kv_heads > 16)
      refuse(what, "up to 16 query heads share a KV head, all KV heads the same number");
    if (q.dim() < 2 || q.size(0) * p.q_heads * p.head_dim != q.numel() || q.size(0) > INT32_MAX || out.sizes() != q.sizes())
      refuse(what, "q and out must be [tokens, q_heads * head_dim]");
    if (p.prefix_len < 0) refuse(what, "prefix_len must not be negative");
    const Tensor& qo_indptr = checked(what, "qo_indptr", a[5], at::kInt, c.device);
    const Tensor& kv_indptr = checked(what, "kv_indptr", a[6], at::kInt, c.device);
    const Tensor& kv_indices = checked(what, "kv_indices", a[7], at::kInt, c.device);
    const Tensor& last = checked(what, "kv_last_page_len", a[8], at::kInt, c.device);
    const int64_t end = static_cast<int64_t>(p.req_begin) + p.req_count;
    if (p.req_begin < 0 || p.req_count < 0 || qo_indptr.numel() < end || kv_indptr.numel() < end + 1 || last.numel() < end)
      refuse(what, "requests " + std::to_string(p.req_begin) + " to " + std::to_string(end) + " are not all listed");
    const Tensor* pages = nullptr;
    if (p.prefix_len > 0) {
      pages = &checked(what, "prefix_pages", a[9], at::kInt, c.device);
      if (pages->numel() < (static_cast<int64_t>(p.prefix_len) + kPage - 1) / kPage) refuse(what, "prefix_pages lists fewer pages than prefix_len needs");
      p.prefix_pages = static_cast<const int*>(pages->data_ptr());
    }
    if (a[16] == Py_None) refuse(what, "needs a workspace (decode_workspace_q8)");
    const Tensor& workspace = checked(what, "workspace", a[16], at::kByte, c.device);
    const Tensor* status = status_word(what, a[17], c.device);
    apart(what, {&out, &workspace, status}, {&q, &c.pool, &c.scale, &qo_indptr, &kv_indptr, &kv_indices, &last, pages});
    p.q = q.data_ptr();
    p.out = out.data_ptr();
    p.kv_pool = c.pool.data_ptr();
    p.kv_scale = static_cast<const float*>(c.scale.data_ptr());
    p.qo_indptr = static_cast<const int*>(qo_indptr.data_ptr());
    p.kv_indptr = static_cast<const int*>(kv_indptr.data_ptr());
    p.kv_indices = static_cast<const int*>(kv_indices.data_ptr());
    p.kv_last_page_len = static_cast<const int*>(last.data_ptr());
    p.num_tokens = static_cast<int>(q.size(0));
    p.num_indices = count(what, kv_indices, "kv_indices");
    p.workspace = workspace.data_ptr();
    p.workspace_bytes = workspace.numel();
    p.status = word(status);
    p.early_start = whole(a[18], what, "early_start");
    if (p.req_count > 0) launch(what, entries.decode, p, c.device);
  });
}

// addresses of nfk_rope_append_q8, nfk_kv_read_q8, nfk_attn_decode_q8
PyObject* connect(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 3, [&] {
    void* at[3];
    for (int i = 0; i < 3; ++i) {
      at[i] = PyLong_AsVoidPtr(a[i]);
      if (at[i] == nullptr) {
        PyErr_Clear();
        refuse("connect", "addresses expected");
      }
    }
    entries.append = reinterpret_cast<decltype(entries.append)>(at[0]);
    entries.read = reinterpret_cast<decltype(entries.read)>(at[1]);
    entries.decode = reinterpret_cast<decltype(entries.decode)>(at[2]);
  });
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyMethodDef method(const char* name) {
  return PyMethodDef{name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F)), METH_FASTCALL, nullptr};
}
PyMethodDef methods[] = {method<connect>("connect"), method<rope_append>("rope_append"), method<read>("read"), method<decode>("decode"),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_cache_q8", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__cache_q8() { return PyModule_Create(&module); }
