// Python binding of the KV-cache operators: checks torch tensors and calls the
// C ABI (include/scalesweep_b200.h).  These calls sit between every layer's
// GEMMs at decode sizes, where the checks and allocations in Python cost more
// than the kernels (a one-token cache write: 23 us of host time through
// ctypes, 6 us through here).
#include <Python.h>

#include <cmath>
#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <stdexcept>
#include <string>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/scalesweep_b200.h"

namespace {

struct ValueError : std::runtime_error {
  using std::runtime_error::runtime_error;
};

[[noreturn]] __attribute__((format(printf, 1, 2))) void bad(const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  throw ValueError(buf);
}

std::string shape_of(const at::Tensor& t) {
  std::string s = "[";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + "]";
}

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) bad("%s must be a tensor", name);
  return THPVariable_Unpack(o);
}

int64_t integer(PyObject* o, const char* name) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    bad("%s must be an integer", name);
  }
  return v;
}

bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) {
    PyErr_Clear();
    bad("a flag must be true or false");
  }
  return v != 0;
}

void check_status(int st) {
  if (st == SSW_OK) return;
  const char* msg = ssw_last_error();
  if (!msg || !*msg) msg = ssw_status_string(st);
  if (st == SSW_ERR_INVALID_ARGUMENT) throw ValueError(msg);
  throw std::runtime_error(msg);
}

void on(const at::Tensor& t, const char* name, const c10::Device& dev) {
  if (t.device() != dev)
    bad("%s must be on %s, got %s", name, dev.str().c_str(), t.device().str().c_str());
}

int dtype_code(at::ScalarType t) {
  if (t == at::kBFloat16) return SSW_DTYPE_BF16;
  if (t == at::kHalf) return SSW_DTYPE_F16;
  bad("input dtype must be torch.bfloat16 or torch.float16, got %s", c10::toString(t));
}

// The dimensions and inner strides of a cache, from its last five axes.
struct CacheShape {
  int64_t pages, heads, page, half;
};

CacheShape check_cache_tensors(const at::Tensor& codes, const at::Tensor& scales, int64_t dims) {
  if (codes.dim() != dims || scales.dim() != dims)
    bad("codes and scales must be [%snum_pages, 2, kv_heads, page_size, ..] tensors",
        dims == 6 ? "layers, " : "");
  if (codes.scalar_type() != at::kByte || scales.scalar_type() != at::kFloat8_e4m3fn)
    bad("codes must be uint8 and scales float8_e4m3fn, got %s and %s",
        c10::toString(codes.scalar_type()), c10::toString(scales.scalar_type()));
  const auto c = codes.sizes(), s = scales.sizes();
  const int64_t o = dims - 5;
  const CacheShape r{c[o], c[o + 2], c[o + 3], c[o + 4]};
  bool same = c[o + 1] == 2 && r.half % 8 == 0 && s[o + 4] == r.half / 8;
  for (int64_t i = 0; i < dims - 1; ++i) same = same && c[i] == s[i];
  if (!same)
    bad("codes must be [num_pages, 2, kv_heads, page_size, head_size/2] and scales "
        "[.., head_size/16], got %s and %s",
        shape_of(codes).c_str(), shape_of(scales).c_str());
  if (!codes.is_cuda()) bad("codes must be a CUDA tensor (there is no CPU implementation)");
  on(scales, "scales", codes.device());
  const auto cs = codes.strides(), ss = scales.strides();
  const int64_t srow = r.half / 8;
  if (cs[o + 1] != r.heads * r.page * r.half || cs[o + 2] != r.page * r.half ||
      cs[o + 3] != r.half || cs[o + 4] != 1 || ss[o + 1] != r.heads * r.page * srow ||
      ss[o + 2] != r.page * srow || ss[o + 3] != srow || ss[o + 4] != 1)
    bad("codes and scales must be contiguous within a page");
  return r;
}

ssw_kv_cache cache_of(const at::Tensor& codes, const at::Tensor& scales, const at::Tensor& mult) {
  const CacheShape r = check_cache_tensors(codes, scales, 5);
  if (mult.scalar_type() != at::kFloat || mult.dim() != 1 || mult.size(0) != 2 ||
      mult.device() != codes.device() || mult.stride(0) != 1)
    bad("kv_input_scale must be a contiguous float32 tensor of shape [2] on %s",
        codes.device().str().c_str());
  ssw_kv_cache c;
  c.codes = static_cast<uint8_t*>(codes.data_ptr());
  c.scales = static_cast<uint8_t*>(scales.data_ptr());
  c.codes_page_stride = codes.stride(0);
  c.scales_page_stride = scales.stride(0);
  c.input_scale = static_cast<const float*>(mult.data_ptr());
  c.num_pages = r.pages;
  c.page_size = (int32_t)r.page;
  c.kv_heads = (int32_t)r.heads;
  c.head_size = (int32_t)(2 * r.half);
  return c;
}

ssw_kv_heads heads_of(const at::Tensor& t, const char* name, int64_t tokens, int64_t heads,
                      int64_t d, at::ScalarType dtype, const c10::Device& dev) {
  if (t.dim() != 3 || t.size(0) != tokens || t.size(1) != heads || t.size(2) != d ||
      t.scalar_type() != dtype)
    bad("%s must be a %s tensor of shape [%lld, %lld, %lld], got %s %s", name, c10::toString(dtype),
        (long long)tokens, (long long)heads, (long long)d, c10::toString(t.scalar_type()),
        shape_of(t).c_str());
  on(t, name, dev);
  // the stride of an axis of length 1 says nothing, and may be anything
  const int64_t st = tokens > 1 ? t.stride(0) : 0, sh = heads > 1 ? t.stride(1) : 0;
  if (t.stride(2) != 1 || st % 8 || sh % 8)
    bad("%s: the last dimension must be contiguous, the other strides multiples of 8", name);
  return {t.data_ptr(), st, sh};
}

// These calls bypass autograd, so a gradient that is asked for would be lost
// without a word.
void check_no_gradient(const at::Tensor& t, const char* name) {
  if (c10::GradMode::is_enabled() && t.requires_grad())
    bad("%s requires a gradient, which this operator does not have: call it under torch.no_grad()",
        name);
  if (at::isFloatingType(t.scalar_type()) && t._fw_grad(0).defined())
    bad("%s carries a forward-mode gradient, which this operator does not have", name);
}

// An output whose elements share memory would be written in no order.
void check_distinct(const at::Tensor& t, const char* name) {
  for (int64_t i = 0; i < t.dim(); ++i)
    if (t.size(i) > 1 && t.stride(i) == 0) bad("%s must not be an expanded tensor", name);
}

void* vector_of(const at::Tensor& t, const char* name, at::ScalarType dtype, int64_t n,
                const c10::Device& dev) {
  if (t.scalar_type() != dtype || t.dim() != 1 || t.size(0) != n || t.device() != dev ||
      (n > 1 && t.stride(0) != 1))
    bad("%s must be a contiguous %s tensor of shape [%lld] on %s", name,
        dtype == at::kInt ? "int32" : "int64", (long long)n, dev.str().c_str());
  return t.data_ptr();
}

at::Tensor empty(at::IntArrayRef sizes, at::ScalarType dtype, const c10::Device& dev) {
  return at::detail::empty_cuda(sizes, dtype, dev, c10::nullopt);
}

void* stream_of(const c10::Device& dev) {
  return c10::cuda::getCurrentCUDAStream(dev.index()).stream();
}

template <typename F>
PyObject* guarded(F&& f) {
  try {
    return f();
  } catch (const ValueError& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
  } catch (const c10::OutOfMemoryError& e) {
    PyObject* torch = PyImport_ImportModule("torch");
    PyObject* type = torch ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
    if (type) PyErr_SetString(type, e.what_without_backtrace());
    Py_XDECREF(type);
    Py_XDECREF(torch);
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

void expect(Py_ssize_t have, Py_ssize_t want) {
  if (have != want) bad("expected %zd arguments, got %zd", want, have);
}

// write(query, key, value, positions, cos_sin_cache, slot_mapping, kv_input_scale, codes, scales,
//       is_neox, query_out or None) -> query_out
PyObject* write(PyObject*, PyObject* const* x, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    expect(n, 11);
    const at::Tensor &query = tensor(x[0], "query"), &key = tensor(x[1], "key"),
                     &value = tensor(x[2], "value"), &positions = tensor(x[3], "positions"),
                     &table = tensor(x[4], "cos_sin_cache"), &slots = tensor(x[5], "slot_mapping"),
                     &mult = tensor(x[6], "kv_input_scale"), &codes = tensor(x[7], "codes"),
                     &scales = tensor(x[8], "scales");
    const ssw_kv_cache cache = cache_of(codes, scales, mult);
    const c10::Device dev = codes.device();
    check_no_gradient(query, "query");
    check_no_gradient(key, "key");
    check_no_gradient(value, "value");
    check_no_gradient(table, "cos_sin_cache");
    check_no_gradient(mult, "kv_input_scale");
    if (query.dim() != 3)
      bad("query must be [T, heads, head_size], got shape %s", shape_of(query).c_str());
    const int64_t tokens = query.size(0), hq = query.size(1), d = query.size(2);
    if (d != cache.head_size)
      bad("query has head size %lld, the cache %d", (long long)d, cache.head_size);
    const at::ScalarType type = query.scalar_type();
    const int dtype = dtype_code(type);
    const ssw_kv_heads q = heads_of(query, "query", tokens, hq, d, type, dev);
    const ssw_kv_heads k = heads_of(key, "key", tokens, cache.kv_heads, d, type, dev);
    const ssw_kv_heads v = heads_of(value, "value", tokens, cache.kv_heads, d, type, dev);
    const void* pos = vector_of(positions, "positions", at::kLong, tokens, dev);
    const void* slot = vector_of(slots, "slot_mapping", at::kLong, tokens, dev);
    if (table.scalar_type() != at::kFloat || table.dim() != 2 || table.device() != dev ||
        !table.is_contiguous())
      bad("cos_sin_cache must be a contiguous float32 tensor [max_position, rotary_dim] on %s",
          dev.str().c_str());
    if (hq > 65536 || table.size(1) > 65536) bad("too many heads or rotary dimensions");
    const c10::cuda::CUDAGuard guard(dev);
    const at::Tensor out =
        x[10] == Py_None ? empty({tokens, hq, d}, type, dev) : tensor(x[10], "query_out");
    const ssw_kv_heads o = heads_of(out, "query_out", tokens, hq, d, type, dev);
    check_distinct(out, "query_out");
    check_no_gradient(out, "query_out");
    check_status(ssw_rotary_scalesweep_mse_nvfp4_kv_write(
        &cache, dtype, tokens, (int)hq, &q, &k, &v, &o, static_cast<const int64_t*>(pos),
        static_cast<const float*>(table.data_ptr()), table.size(0), (int)table.size(1),
        truth(x[9]), static_cast<const int64_t*>(slot), stream_of(dev)));
    if (x[10] != Py_None) {
      Py_INCREF(x[10]);
      return x[10];
    }
    return THPVariable_Wrap(out);
  });
}

// gather(codes, scales, kv_input_scale, slot_mapping, dtype) -> (key, value)
PyObject* gather(PyObject*, PyObject* const* x, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    expect(n, 5);
    const at::Tensor &codes = tensor(x[0], "codes"), &scales = tensor(x[1], "scales"),
                     &mult = tensor(x[2], "kv_input_scale"), &slots = tensor(x[3], "slot_mapping");
    if (!THPDtype_Check(x[4])) bad("dtype must be torch.bfloat16 or torch.float16");
    const at::ScalarType type = reinterpret_cast<THPDtype*>(x[4])->scalar_type;
    const int dtype = dtype_code(type);
    const ssw_kv_cache cache = cache_of(codes, scales, mult);
    const c10::Device dev = codes.device();
    check_no_gradient(mult, "kv_input_scale");
    const int64_t tokens = slots.numel();
    const void* slot = vector_of(slots, "slot_mapping", at::kLong, tokens, dev);
    const c10::cuda::CUDAGuard guard(dev);
    const at::Tensor key = empty({tokens, cache.kv_heads, cache.head_size}, type, dev);
    const at::Tensor value = empty({tokens, cache.kv_heads, cache.head_size}, type, dev);
    check_status(ssw_nvfp4_kv_gather(&cache, dtype, tokens, static_cast<const int64_t*>(slot),
                                     key.data_ptr(), value.data_ptr(), stream_of(dev)));
    PyObject* k = THPVariable_Wrap(key);
    PyObject* v = THPVariable_Wrap(value);
    PyObject* r = k && v ? PyTuple_Pack(2, k, v) : nullptr;
    Py_XDECREF(k);
    Py_XDECREF(v);
    return r;
  });
}

// attend(query, codes, scales, kv_input_scale, block_table, seq_lens, query_start, max_query_len,
//        max_seq_len, softmax_scale or None, causal, window or None, out or None, return_lse,
//        status or None) -> out, or (out, lse)
PyObject* attend(PyObject*, PyObject* const* x, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    expect(n, 15);
    const at::Tensor &query = tensor(x[0], "query"), &codes = tensor(x[1], "codes"),
                     &scales = tensor(x[2], "scales"), &mult = tensor(x[3], "kv_input_scale"),
                     &table = tensor(x[4], "block_table"), &lens = tensor(x[5], "seq_lens"),
                     &start = tensor(x[6], "query_start");
    const ssw_kv_cache cache = cache_of(codes, scales, mult);
    const c10::Device dev = codes.device();
    check_no_gradient(query, "query");
    check_no_gradient(mult, "kv_input_scale");
    if (query.dim() != 3)
      bad("query must be [T, heads, head_size], got shape %s", shape_of(query).c_str());
    const int64_t tokens = query.size(0), hq = query.size(1), d = query.size(2);
    if (d != cache.head_size)
      bad("query has head size %lld, the cache %d", (long long)d, cache.head_size);
    const at::ScalarType type = query.scalar_type();
    const int dtype = dtype_code(type);
    const ssw_kv_heads q = heads_of(query, "query", tokens, hq, d, type, dev);
    if (table.dim() != 2 || table.scalar_type() != at::kInt || table.device() != dev)
      bad("block_table must be an int32 tensor [sequences, pages] on %s", dev.str().c_str());
    const int64_t seqs = table.size(0), columns = table.size(1);
    if (columns > 1 && table.stride(1) != 1) bad("block_table's rows must be contiguous");
    if (seqs >= (1ll << 31) || columns >= (1ll << 31) || hq > 65536) bad("sizes must be below 2^31");
    ssw_kv_attention a = {};
    a.block_table = static_cast<const int32_t*>(table.data_ptr());
    a.block_table_stride = seqs > 1 ? table.stride(0) : columns;
    a.seq_lens = static_cast<const int32_t*>(vector_of(lens, "seq_lens", at::kInt, seqs, dev));
    a.query_start =
        static_cast<const int32_t*>(vector_of(start, "query_start", at::kInt, seqs + 1, dev));
    if (x[14] != Py_None) {
      const at::Tensor& s = tensor(x[14], "status");
      if (s.scalar_type() != at::kInt || s.device() != dev || s.numel() < 1)
        bad("status must be an int32 tensor on %s", dev.str().c_str());
      a.status = static_cast<int32_t*>(s.data_ptr());
    }
    const int64_t max_q = integer(x[7], "max_query_len"), max_s = integer(x[8], "max_seq_len");
    if (max_q < 1 || max_s < 1 || max_q > (1 << 30) || max_s > (1 << 30))
      bad("max_query_len and max_seq_len must be positive and at most 2^30 (got %lld, %lld)",
          (long long)max_q, (long long)max_s);
    double scale = 1.0 / std::sqrt((double)d);
    if (x[9] != Py_None) {
      scale = PyFloat_AsDouble(x[9]);
      if (scale == -1.0 && PyErr_Occurred()) {
        PyErr_Clear();
        bad("softmax_scale must be a number");
      }
    }
    int64_t window = -1;
    if (x[11] != Py_None) {
      window = integer(x[11], "window");
      if (window < 0) bad("window must not be negative, got %lld", (long long)window);
      if (window > (1 << 30)) window = 1 << 30;
    }
    const bool want_lse = truth(x[13]);
    a.tokens = tokens;
    a.seqs = (int32_t)seqs;
    a.block_table_columns = (int32_t)columns;
    a.q_heads = (int32_t)hq;
    a.max_query_len = (int32_t)max_q;
    a.max_seq_len = (int32_t)max_s;
    a.causal = truth(x[10]);
    a.window = (int32_t)window;
    a.softmax_scale = (float)scale;
    const c10::cuda::CUDAGuard guard(dev);
    const at::Tensor out =
        x[12] == Py_None ? empty({tokens, hq, d}, type, dev) : tensor(x[12], "out");
    const ssw_kv_heads o = heads_of(out, "out", tokens, hq, d, type, dev);
    check_distinct(out, "out");
    check_no_gradient(out, "out");
    at::Tensor lse, workspace;
    if (want_lse) {
      lse = empty({tokens, hq}, at::kFloat, dev);
      a.lse = static_cast<float*>(lse.data_ptr());
    }
    const int64_t need = ssw_nvfp4_paged_attention_workspace_bytes(&cache, &a, dtype);
    if (need < 0) check_status(SSW_ERR_INVALID_ARGUMENT);
    // from the caching allocator: reused only by work behind this call on its stream
    if (need > 0) workspace = empty({need / 4}, at::kFloat, dev);
    check_status(ssw_nvfp4_paged_attention(&cache, &a, dtype, &q, &o,
                                           need > 0 ? workspace.data_ptr() : nullptr, need,
                                           stream_of(dev)));
    PyObject* po;
    if (x[12] != Py_None) {
      Py_INCREF(x[12]);
      po = x[12];
    } else {
      po = THPVariable_Wrap(out);
    }
    if (!want_lse || !po) return po;
    PyObject* pl = THPVariable_Wrap(lse);
    PyObject* r = pl ? PyTuple_Pack(2, po, pl) : nullptr;
    Py_DECREF(po);
    Py_XDECREF(pl);
    return r;
  });
}

// ---- page tables: a capsule of the structs, and the tensors it points into
struct Pages {
  ssw_kv_pages tables;
  ssw_kv_pool pool;
  c10::Device device{c10::kCUDA, 0};
  at::Tensor keep[6];
};

constexpr const char* kCapsule = "scalesweep_b200.kv_pages";

const Pages& pages_of(PyObject* o) {
  void* p = PyCapsule_GetPointer(o, kCapsule);
  if (!p) {
    PyErr_Clear();
    bad("not the page tables of a cache");
  }
  return *static_cast<Pages*>(p);
}

// pages(codes, scales, block_table, seq_lens, refcount, status or None) -> (capsule, status)
PyObject* pages(PyObject*, PyObject* const* x, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    expect(n, 6);
    const at::Tensor &codes = tensor(x[0], "codes"), &scales = tensor(x[1], "scales"),
                     &table = tensor(x[2], "block_table"), &lens = tensor(x[3], "seq_lens"),
                     &refs = tensor(x[4], "refcount");
    const bool layered = codes.dim() == 6;
    const CacheShape r = check_cache_tensors(codes, scales, layered ? 6 : 5);
    const c10::Device dev = codes.device();
    if (table.dim() != 2 || table.scalar_type() != at::kInt || table.device() != dev ||
        (table.size(1) > 1 && table.stride(1) != 1))
      bad("block_table must be an int32 tensor [max_seqs, columns] with contiguous rows on %s",
          dev.str().c_str());
    const int64_t seqs = table.size(0), columns = table.size(1);
    if (r.pages >= (1ll << 31) || seqs >= (1ll << 31) || columns >= (1ll << 31))
      bad("sizes must be below 2^31");
    check_distinct(table, "block_table");
    if (layered && codes.size(0) > 1 && (codes.stride(0) == 0 || scales.stride(0) == 0))
      bad("codes and scales must not be expanded tensors");
    const c10::cuda::CUDAGuard guard(dev);
    Pages p;
    p.device = dev;
    p.tables.refcount = static_cast<int32_t*>(vector_of(refs, "refcount", at::kInt, r.pages, dev));
    p.tables.block_table = static_cast<int32_t*>(table.data_ptr());
    p.tables.table_stride = seqs > 1 ? table.stride(0) : columns;
    p.tables.seq_lens = static_cast<int32_t*>(vector_of(lens, "seq_lens", at::kInt, seqs, dev));
    at::Tensor status;
    if (x[5] == Py_None) {
      status = empty({1}, at::kInt, dev);
      if (cudaMemsetAsync(status.data_ptr(), 0, 4, static_cast<cudaStream_t>(stream_of(dev))) !=
          cudaSuccess)
        throw std::runtime_error("kv_pages: cudaMemsetAsync failed");
    } else {
      status = tensor(x[5], "status");
    }
    p.tables.status = static_cast<int32_t*>(vector_of(status, "status", at::kInt, 1, dev));
    p.tables.num_pages = (int32_t)r.pages;
    p.tables.max_seqs = (int32_t)seqs;
    p.tables.columns = (int32_t)columns;
    p.tables.page_size = (int32_t)r.page;
    const int64_t nc = 2 * r.heads * r.page * r.half, ns = nc / 8, o = layered ? 1 : 0;
    p.pool.codes = static_cast<uint8_t*>(codes.data_ptr());
    p.pool.scales = static_cast<uint8_t*>(scales.data_ptr());
    p.pool.codes_layer_stride = layered ? codes.stride(0) : 0;
    p.pool.scales_layer_stride = layered ? scales.stride(0) : 0;
    p.pool.codes_page_stride = r.pages > 1 ? codes.stride(o) : nc;
    p.pool.scales_page_stride = r.pages > 1 ? scales.stride(o) : ns;
    p.pool.codes_page_bytes = nc;
    p.pool.scales_page_bytes = ns;
    p.pool.num_pages = r.pages;
    p.pool.layers = layered ? (int32_t)codes.size(0) : 1;
    const at::Tensor* all[6] = {&codes, &scales, &table, &lens, &refs, &status};
    for (int i = 0; i < 6; ++i) p.keep[i] = *all[i];
    PyObject* cap = PyCapsule_New(new Pages(std::move(p)), kCapsule, [](PyObject* o) {
      delete static_cast<Pages*>(PyCapsule_GetPointer(o, kCapsule));
    });
    PyObject* st = cap ? THPVariable_Wrap(status) : nullptr;
    PyObject* res = st ? PyTuple_Pack(2, cap, st) : nullptr;
    Py_XDECREF(cap);
    Py_XDECREF(st);
    return res;
  });
}

at::Tensor workspace_of(const Pages& p, int64_t n, int64_t tokens, int64_t pages) {
  const int64_t b = ssw_kv_pages_workspace_bytes(n, tokens, p.tables.page_size, pages);
  if (b < 0) bad("total_tokens must not be negative");
  return empty({b / 4}, at::kInt, p.device);
}

const int32_t* index_of(PyObject* o, const char* name, int64_t n, const Pages& p) {
  return static_cast<const int32_t*>(vector_of(tensor(o, name), name, at::kInt, n, p.device));
}

// pages_extend(pages, seqs, new_tokens, total_tokens) -> slots
PyObject* pages_extend(PyObject*, PyObject* const* x, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    expect(n, 4);
    const Pages& p = pages_of(x[0]);
    const int64_t count = tensor(x[1], "seqs").numel(), total = integer(x[3], "total_tokens");
    const int32_t* seqs = index_of(x[1], "seqs", count, p);
    const int32_t* more = index_of(x[2], "new_tokens", count, p);
    if (total < 0 || total >= (1ll << 30)) bad("total_tokens must be in 0..2^30-1");
    const c10::cuda::CUDAGuard guard(p.device);
    const at::Tensor slots = empty({total}, at::kLong, p.device);
    const at::Tensor ws = workspace_of(p, count, total, 0);
    check_status(ssw_kv_pages_extend(&p.tables, count, seqs, more, total,
                                     static_cast<int64_t*>(slots.data_ptr()), ws.data_ptr(),
                                     ws.numel() * 4, stream_of(p.device)));
    return THPVariable_Wrap(slots);
  });
}

// pages_fork(pages, parents, children)
PyObject* pages_fork(PyObject*, PyObject* const* x, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    expect(n, 3);
    const Pages& p = pages_of(x[0]);
    const int64_t count = tensor(x[1], "parents").numel();
    const int32_t* parents = index_of(x[1], "parents", count, p);
    const int32_t* children = index_of(x[2], "children", count, p);
    const c10::cuda::CUDAGuard guard(p.device);
    const at::Tensor ws = workspace_of(p, count, 0, 0);
    check_status(ssw_kv_pages_fork(&p.tables, &p.pool, count, parents, children, ws.data_ptr(),
                                   ws.numel() * 4, stream_of(p.device)));
    Py_RETURN_NONE;
  });
}

// pages_free(pages, seqs)
PyObject* pages_free(PyObject*, PyObject* const* x, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    expect(n, 2);
    const Pages& p = pages_of(x[0]);
    const int64_t count = tensor(x[1], "seqs").numel();
    const int32_t* seqs = index_of(x[1], "seqs", count, p);
    const c10::cuda::CUDAGuard guard(p.device);
    check_status(ssw_kv_pages_free(&p.tables, count, seqs, stream_of(p.device)));
    Py_RETURN_NONE;
  });
}

// pages_compact(pages)
PyObject* pages_compact(PyObject*, PyObject* const* x, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    expect(n, 1);
    const Pages& p = pages_of(x[0]);
    const c10::cuda::CUDAGuard guard(p.device);
    const at::Tensor ws = workspace_of(p, 0, 0, p.tables.num_pages);
    check_status(ssw_kv_pages_compact(&p.tables, &p.pool, ws.data_ptr(), ws.numel() * 4,
                                      stream_of(p.device)));
    Py_RETURN_NONE;
  });
}

// pages_copy(pages, source, target)
PyObject* pages_copy(PyObject*, PyObject* const* x, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    expect(n, 3);
    const Pages& p = pages_of(x[0]);
    const int64_t count = tensor(x[1], "source").numel();
    const int32_t* source = index_of(x[1], "source", count, p);
    const int32_t* target = index_of(x[2], "target", count, p);
    const c10::cuda::CUDAGuard guard(p.device);
    check_status(ssw_kv_pages_copy(&p.pool, count, source, target, stream_of(p.device)));
    Py_RETURN_NONE;
  });
}

PyMethodDef kMethods[] = {
#define SSW_METHOD(f) {#f, reinterpret_cast<PyCFunction>(f), METH_FASTCALL, nullptr}
    SSW_METHOD(write),        SSW_METHOD(gather),     SSW_METHOD(attend),
    SSW_METHOD(pages),        SSW_METHOD(pages_extend), SSW_METHOD(pages_fork),
    SSW_METHOD(pages_free),   SSW_METHOD(pages_compact), SSW_METHOD(pages_copy),
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_kv_binding", nullptr, -1, kMethods};

}  // namespace

PyMODINIT_FUNC PyInit__kv_binding(void) { return PyModule_Create(&kModule); }
