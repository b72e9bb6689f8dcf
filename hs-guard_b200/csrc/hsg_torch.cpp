// Tensor side of draft scoring and of the 8-bit cache (CPython extension module _hsg_torch over libhsg.so and torch's C++ tensors).
//
// hs_guard_b200.drafts documents these functions; here their arguments are checked, their outputs allocated and the
// argument structs of include/hsg.h filled. The same steps in Python cost 6 to 15 us a call, several times what the
// smallest calls take on the GPU; here they cost 1 to 2.
//
// Every argument is positional and every function METH_FASTCALL. A wrong argument raises ValueError before anything is
// queued; what the library refuses goes through hs_guard_b200._lib.check, torch's own failures (out of memory) through
// torch's translation.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/LegacyTypeDispatch.h>
#include <ATen/core/grad_mode.h>
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cstdarg>
#include <cstdio>
#include <limits>

#include "../../include/hsg.h"

namespace {

using at::Tensor;

struct Refused {  // a ValueError's text
  char text[256];
};

[[noreturn]] void refuse(const char* fmt, ...) {
  Refused r;
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(r.text, sizeof(r.text), fmt, ap);
  va_end(ap);
  throw r;
}

const char* name_of(at::ScalarType t) { return c10::toString(t); }

const Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) refuse("%s must be a tensor", name);
  const Tensor& t = THPVariable_Unpack(o);
  // outputs are made below autograd: a gradient would be lost in silence
  if (t.requires_grad() && at::GradMode::is_enabled())
    refuse("%s requires a gradient and there is no backward pass: call under torch.no_grad()", name);
  return t;
}

// What a call changes in place, for those who compare version counters.
void changed(PyObject* o) {
  const Tensor& t = THPVariable_Unpack(o);
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// A tensor on the calls' device, of these dimensions and this type, its last dimension contiguous.
const Tensor& shaped(PyObject* o, const char* name, int64_t ndim, at::ScalarType dtype, at::Device device) {
  const Tensor& t = tensor(o, name);
  if (t.scalar_type() != dtype || t.device() != device || t.dim() != ndim || t.layout() != at::kStrided)
    refuse("%s must be a %d-d %s tensor on %s", name, (int)ndim, name_of(dtype), device.str().c_str());
  if (t.stride(-1) != 1 && t.size(-1) > 1) refuse("%s must be contiguous in its last dimension", name);
  return t;
}

// The data of a contiguous 1-d tensor; size < 0: any.
template <typename P>
P* vector(PyObject* o, const char* name, at::ScalarType dtype, at::Device device, int64_t size = -1) {
  const Tensor& t = shaped(o, name, 1, dtype, device);
  if (size >= 0 && t.size(0) != size) refuse("%s must have %lld elements, got %lld", name, (long long)size, (long long)t.size(0));
  return static_cast<P*>(t.data_ptr());
}

int32_t* error_word(PyObject* o, at::Device device) {
  return o == Py_None ? nullptr : vector<int32_t>(o, "err", at::kInt, device, 1);
}

at::Device device_of(const Tensor& t, const char* name) {
  if (!t.is_cuda()) refuse("%s must be a CUDA tensor", name);
  return t.device();
}

// A Python integer, or what converts to one without loss as numpy's do. Not a tensor, whose conversion would wait for the GPU.
int32_t whole(PyObject* o, const char* name, int64_t lo, int64_t hi) {
  PyObject* index = PyLong_Check(o) ? (Py_INCREF(o), o) : THPVariable_Check(o) ? nullptr : PyNumber_Index(o);
  int overflow = 0;
  const long long v = index ? PyLong_AsLongLongAndOverflow(index, &overflow) : 0;
  const bool good = index && !overflow && v >= lo && v <= hi;
  Py_XDECREF(index);
  PyErr_Clear();
  if (!good) refuse("%s must be an integer in [%lld, %lld]", name, (long long)lo, (long long)hi);
  return (int32_t)v;
}

float real(PyObject* o, const char* name) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    refuse("%s must be a number", name);
  }
  return (float)v;
}

int32_t small(int64_t v, const char* name) {
  if (v > INT32_MAX) refuse("%s is beyond 32 bits", name);
  return (int32_t)v;
}

int32_t code_of(at::ScalarType t) {
  return t == at::kFloat ? HSG_DT_F32 : t == at::kHalf ? HSG_DT_F16 : t == at::kBFloat16 ? HSG_DT_BF16 : -1;
}
bool is_16(at::ScalarType t) { return t == at::kHalf || t == at::kBFloat16; }

// k and v [pages, page_size, heads, dim], alike in strides.
hsg_page_cache page_cache(PyObject* ko, PyObject* vo, int64_t heads, int64_t dim, at::ScalarType dtype, at::Device device) {
  const Tensor &k = shaped(ko, "k_cache", 4, dtype, device), &v = shaped(vo, "v_cache", 4, dtype, device);
  if (v.sizes() != k.sizes() || v.strides() != k.strides() || k.size(2) != heads || k.size(3) != dim)
    refuse("k_cache and v_cache must be alike, [pages, page_size, %lld, %lld]", (long long)heads, (long long)dim);
  return hsg_page_cache{k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), k.stride(2), small(k.size(0), "pages"),
                        small(k.size(1), "page_size")};
}

struct Heads {
  int32_t tokens, hq, hkv, dim;
};
Heads heads_of(const Tensor& q, const Tensor& k, const Tensor& v) {
  if (k.sizes() != v.sizes() || k.size(0) != q.size(0) || k.size(2) != q.size(2))
    refuse("k and v must be alike, [tokens, kv heads, dim] with q's tokens and dim");
  return {small(q.size(0), "tokens"), small(q.size(1), "heads"), small(k.size(1), "kv heads"), small(q.size(2), "dim")};
}

Tensor empty(at::IntArrayRef sizes, at::ScalarType dtype, at::Device device) {
  return at::empty(sizes, at::TensorOptions().dtype(dtype).device(device));
}

// A contiguous tensor of these sizes over `base`'s storage from the offset-th element (of this type) on: a view operator costs
// several times as much.
Tensor part(const Tensor& base, at::ScalarType dtype, int64_t offset, at::IntArrayRef sizes) {
  Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::TensorImpl::VIEW, c10::Storage(base.storage()), base.key_set(),
                                                      c10::scalarTypeToTypeMeta(dtype));
  t.unsafeGetTensorImpl()->set_storage_offset(offset);
  t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
  return t;
}
Tensor part(const Tensor& base, at::ScalarType dtype, int64_t offset, int64_t n) {
  return part(base, dtype, offset, at::IntArrayRef(&n, 1));
}

void* stream_of(at::Device device) { return c10::cuda::getCurrentCUDAStream(device.index()).stream(); }

struct LibraryError {
  int rc;
};
void done(int rc) {
  if (rc != HSG_OK) throw LibraryError{rc};
}

// Runs `body`; the exceptions that it may end with become Python's.
template <typename F>
PyObject* guarded(Py_ssize_t n, Py_ssize_t want, F body) {
  HANDLE_TH_ERRORS
  if (n != want) {
    PyErr_Format(PyExc_TypeError, "%zd arguments, %zd are wanted", n, want);
    return nullptr;
  }
  try {
    // the outputs have no gradients: their creation skips autograd's dispatch
    const at::AutoDispatchBelowADInplaceOrView below;
    return body();
  } catch (const Refused& r) {
    PyErr_SetString(PyExc_ValueError, r.text);
    return nullptr;
  } catch (const LibraryError& e) {  // raises by itself
    PyObject* lib = PyImport_ImportModule("hs_guard_b200._lib");
    PyObject* r = lib ? PyObject_CallMethod(lib, "check", "i", e.rc) : nullptr;
    Py_XDECREF(lib);
    Py_XDECREF(r);
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "libhsg failed");
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

template <typename... T>
PyObject* tuple_of(const T&... t) {
  PyObject* r = PyTuple_New(sizeof...(T));
  if (!r) return nullptr;
  Py_ssize_t i = 0;
  bool ok = true;
  auto put = [&](const Tensor& x) {
    PyObject* o = THPVariable_Wrap(x);
    if (!o) ok = false;
    PyTuple_SET_ITEM(r, i++, o);
  };
  (put(t), ...);
  if (!ok) {
    Py_DECREF(r);
    return nullptr;
  }
  return r;
}

// advance_tables(lens, delta, table, ring, counters, page_size, capacity, err) -> the six tensors of Tables
PyObject* advance_tables(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 8, [&]() -> PyObject* {
    const at::Device device = device_of(tensor(a[0], "lens"), "lens");
    hsg_tables_args s{};
    s.size = sizeof(s);
    s.lens = vector<int32_t>(a[0], "lens", at::kInt, device);
    const int64_t rows = THPVariable_Unpack(a[0]).size(0);
    if (rows > HSG_MAX_TABLE_ROWS) refuse("at most %d requests a call, got %lld", HSG_MAX_TABLE_ROWS, (long long)rows);
    s.delta = vector<int32_t>(a[1], "delta", at::kInt, device, rows);
    const Tensor& table = shaped(a[2], "table", 2, at::kInt, device);
    if (table.size(0) != rows) refuse("table must have %lld rows, got %lld", (long long)rows, (long long)table.size(0));
    s.table = static_cast<int32_t*>(table.data_ptr());
    s.width = small(table.size(1), "the table's width");
    s.table_stride = rows > 1 ? table.stride(0) : s.width;
    s.ring = vector<int32_t>(a[3], "ring", at::kInt, device);
    s.ring_size = small(THPVariable_Unpack(a[3]).size(0), "the ring");
    s.counters = vector<int64_t>(a[4], "counters", at::kLong, device, 2);
    s.page_size = whole(a[5], "page_size", 1, INT32_MAX);
    s.capacity = whole(a[6], "capacity", 0, INT32_MAX - 3);
    s.err = error_word(a[7], device);
    s.rows = (int32_t)rows;
    // one allocation for what a caller keeps until the next call (counters, lengths, offsets) and one for the three lists,
    // each of which begins on a 16-byte boundary
    const int64_t room = ((int64_t)s.capacity + 3) / 4 * 4;
    const Tensor kept = empty({4 + 2 * rows + 1}, at::kInt, device), lists = empty({3 * room}, at::kInt, device);
    int32_t* base = static_cast<int32_t*>(kept.data_ptr());
    s.counters_out = reinterpret_cast<int64_t*>(base);
    s.lens_out = base + 4;
    s.cu = s.lens_out + rows;
    s.slots = static_cast<int32_t*>(lists.data_ptr());
    s.token_rows = s.slots + room;
    s.positions = s.token_rows + room;
    s.stream = stream_of(device);
    const c10::cuda::CUDAGuard guard(device);
    done(hsg_advance_tables(&s));
    changed(a[2]);
    changed(a[3]);
    return tuple_of(part(kept, at::kInt, 4, rows), part(kept, at::kLong, 0, 2), part(kept, at::kInt, 4 + rows, rows + 1),
                    part(lists, at::kInt, 0, s.capacity), part(lists, at::kInt, room, s.capacity),
                    part(lists, at::kInt, 2 * room, s.capacity));
  });
}

// plan_tree(parents, cu, lens, max_tree, err) -> (positions, mask)
PyObject* plan_tree(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 5, [&]() -> PyObject* {
    const at::Device device = device_of(tensor(a[0], "parents"), "parents");
    hsg_tree_args s{};
    s.size = sizeof(s);
    s.words = (whole(a[3], "max_tree", 1, HSG_MAX_TREE) + 31) / 32;
    s.parents = vector<int32_t>(a[0], "parents", at::kInt, device);
    s.lens = vector<int32_t>(a[2], "lens", at::kInt, device);
    s.tokens = small(THPVariable_Unpack(a[0]).size(0), "tokens");
    s.rows = small(THPVariable_Unpack(a[2]).size(0), "rows");
    s.cu = vector<int32_t>(a[1], "cu", at::kInt, device, (int64_t)s.rows + 1);
    s.err = error_word(a[4], device);
    const Tensor positions = empty({s.tokens}, at::kInt, device), mask = empty({s.tokens, s.words}, at::kInt, device);
    s.positions = static_cast<int32_t*>(positions.data_ptr());
    s.mask = static_cast<uint32_t*>(mask.data_ptr());
    s.stream = stream_of(device);
    const c10::cuda::CUDAGuard guard(device);
    if (s.rows == 0) {  // the library has nothing to do: every token is one of no request
      positions.fill_(-1);
      mask.zero_();
    } else {
      done(hsg_plan_tree(&s));
    }
    return tuple_of(positions, mask);
  });
}

// The arguments that both forms of norm_rope begin with: q, k, v, q_weight, k_weight, inv_freq, positions, eps.
hsg_norm_rope_args norm_args(PyObject* const* a, at::ScalarType out, Tensor& q_out) {
  const Tensor& q0 = tensor(a[0], "q");
  const at::Device device = device_of(q0, "q");
  const at::ScalarType in = q0.scalar_type();
  hsg_norm_rope_args s{};
  s.size = sizeof(s);
  s.in_dtype = code_of(in);
  if (s.in_dtype < 0) refuse("q, k and v must be fp32, fp16 or bf16");
  const Tensor &q = shaped(a[0], "q", 3, in, device), &k = shaped(a[1], "k", 3, in, device), &v = shaped(a[2], "v", 3, in, device);
  const Heads h = heads_of(q, k, v);
  s.q = q.data_ptr();
  s.k = k.data_ptr();
  s.v = v.data_ptr();
  s.q_token_stride = q.stride(0);
  s.q_head_stride = q.stride(1);
  s.k_token_stride = k.stride(0);
  s.k_head_stride = k.stride(1);
  s.v_token_stride = v.stride(0);
  s.v_head_stride = v.stride(1);
  s.q_weight = vector<float>(a[3], "q_weight", at::kFloat, device, h.dim);
  s.k_weight = vector<float>(a[4], "k_weight", at::kFloat, device, h.dim);
  s.inv_freq = vector<float>(a[5], "inv_freq", at::kFloat, device);
  s.rot = small(2 * THPVariable_Unpack(a[5]).size(0), "inv_freq");
  s.positions = vector<int32_t>(a[6], "positions", at::kInt, device, h.tokens);
  s.eps = real(a[7], "eps");
  s.tokens = h.tokens;
  s.hq = h.hq;
  s.hkv = h.hkv;
  s.dim = h.dim;
  s.out_dtype = code_of(out);
  q_out = empty({h.tokens, h.hq, h.dim}, out, device);
  s.q_out = q_out.data_ptr();
  s.stream = stream_of(device);
  return s;
}

// norm_rope(<norm_args>, dtype, err) -> (q, k, v)
PyObject* norm_rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 10, [&]() -> PyObject* {
    if (!THPDtype_Check(a[8]) || !is_16(reinterpret_cast<THPDtype*>(a[8])->scalar_type))
      refuse("dtype must be torch.float16 or torch.bfloat16");
    const at::ScalarType out = reinterpret_cast<THPDtype*>(a[8])->scalar_type;
    Tensor q_out;
    hsg_norm_rope_args s = norm_args(a, out, q_out);
    const at::Device device = q_out.device();
    const Tensor k_out = empty({s.tokens, s.hkv, s.dim}, out, device), v_out = empty({s.tokens, s.hkv, s.dim}, out, device);
    s.k_out = k_out.data_ptr();
    s.v_out = v_out.data_ptr();
    s.err = error_word(a[9], device);
    const c10::cuda::CUDAGuard guard(device);
    done(hsg_norm_rope(&s));
    return tuple_of(q_out, k_out, v_out);
  });
}

// norm_rope_store(<norm_args>, k_cache, v_cache, slots, err) -> q
PyObject* norm_rope_store(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 12, [&]() -> PyObject* {
    const at::ScalarType out = tensor(a[8], "k_cache").scalar_type();
    if (!is_16(out)) refuse("the cache must be fp16 or bf16");
    Tensor q_out;
    hsg_norm_rope_args s = norm_args(a, out, q_out);
    const at::Device device = q_out.device();
    s.cache = page_cache(a[8], a[9], s.hkv, s.dim, out, device);
    // without tokens there are no slots to point at, and nothing to do
    s.slots = vector<int32_t>(a[10], "slots", at::kInt, device, s.tokens);
    s.err = error_word(a[11], device);
    const c10::cuda::CUDAGuard guard(device);
    done(hsg_norm_rope(&s));
    changed(a[8]);
    changed(a[9]);
    return THPVariable_Wrap(q_out);
  });
}

// tree_attention(q, k, v, k_cache, v_cache, table, lens, cu, scale, max_tree, mask, positions, window, workspace, err)
//   -> (out, lse)
PyObject* tree_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 15, [&]() -> PyObject* {
    const Tensor& q0 = tensor(a[0], "q");
    const at::Device device = device_of(q0, "q");
    const at::ScalarType dtype = q0.scalar_type();
    if (!is_16(dtype)) refuse("q, k, v and the cache must be fp16 or bf16");
    const Tensor &q = shaped(a[0], "q", 3, dtype, device), &k = shaped(a[1], "k", 3, dtype, device),
                 &v = shaped(a[2], "v", 3, dtype, device);
    const Heads h = heads_of(q, k, v);
    hsg_tree_attention_args s{};
    s.size = sizeof(s);
    s.q = q.data_ptr();
    s.k = k.data_ptr();
    s.v = v.data_ptr();
    s.q_token_stride = q.stride(0);
    s.q_head_stride = q.stride(1);
    s.k_token_stride = k.stride(0);
    s.k_head_stride = k.stride(1);
    s.v_token_stride = v.stride(0);
    s.v_head_stride = v.stride(1);
    s.cache = page_cache(a[3], a[4], h.hkv, h.dim, dtype, device);
    const Tensor& table = shaped(a[5], "table", 2, at::kInt, device);
    s.rows = small(table.size(0), "rows");
    s.width = small(table.size(1), "the table's width");
    s.table = static_cast<const int32_t*>(table.data_ptr());
    s.table_stride = s.rows > 1 ? table.stride(0) : s.width;
    s.lens = vector<int32_t>(a[6], "lens", at::kInt, device, s.rows);
    s.cu = vector<int32_t>(a[7], "cu", at::kInt, device, (int64_t)s.rows + 1);
    s.scale = real(a[8], "scale");
    s.max_tree = whole(a[9], "max_tree", 1, HSG_MAX_TREE);
    if (a[10] != Py_None) {
      const Tensor& mask = shaped(a[10], "mask", 2, at::kInt, device);
      if (mask.size(0) != h.tokens || !mask.is_contiguous()) refuse("mask must be contiguous, [%d, words]", h.tokens);
      s.words = small(mask.size(1), "the mask's words");
      s.mask = static_cast<const uint32_t*>(mask.data_ptr());
    }
    if (a[11] != Py_None) s.positions = vector<int32_t>(a[11], "positions", at::kInt, device, h.tokens);
    s.window = whole(a[12], "window", 0, INT32_MAX);
    Tensor workspace;
    if (a[13] == Py_None) workspace = empty({(int64_t)hsg_tree_attention_workspace(h.dim)}, at::kByte, device);
    else workspace = shaped(a[13], "workspace", 1, at::kByte, device);
    s.workspace = workspace.data_ptr();
    s.workspace_bytes = workspace.numel();
    s.err = error_word(a[14], device);
    const Tensor out = empty({h.tokens, h.hq, h.dim}, dtype, device), lse = empty({h.tokens, h.hq}, at::kFloat, device);
    s.out = out.data_ptr();
    s.lse = static_cast<float*>(lse.data_ptr());
    s.tokens = h.tokens;
    s.hq = h.hq;
    s.hkv = h.hkv;
    s.dim = h.dim;
    s.dtype = code_of(dtype);
    s.stream = stream_of(device);
    const c10::cuda::CUDAGuard guard(device);
    if (s.rows == 0) {  // the library has nothing to do: no token sees anything
      out.zero_();
      lse.fill_(-std::numeric_limits<float>::infinity());
    } else {
      done(hsg_tree_attention(&s));
    }
    return tuple_of(out, lse);
  });
}

// store_rows(k, v, k_cache, v_cache, slots, source, err)
PyObject* store_rows(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 7, [&]() -> PyObject* {
    const Tensor& k0 = tensor(a[0], "k");
    const at::Device device = device_of(k0, "k");
    const at::ScalarType dtype = k0.scalar_type();
    if (!is_16(dtype)) refuse("k, v and the cache must be fp16 or bf16");
    const Tensor &k = shaped(a[0], "k", 3, dtype, device), &v = shaped(a[1], "v", 3, dtype, device);
    if (k.sizes() != v.sizes()) refuse("k and v must be alike, [rows, kv heads, dim]");
    hsg_store_args s{};
    s.size = sizeof(s);
    s.k = k.data_ptr();
    s.v = v.data_ptr();
    s.k_token_stride = k.stride(0);
    s.k_head_stride = k.stride(1);
    s.v_token_stride = v.stride(0);
    s.v_head_stride = v.stride(1);
    s.cache = page_cache(a[2], a[3], k.size(1), k.size(2), dtype, device);
    s.slots = vector<int32_t>(a[4], "slots", at::kInt, device);
    s.count = small(THPVariable_Unpack(a[4]).size(0), "slots");
    s.rows = small(k.size(0), "rows");
    s.heads = small(k.size(1), "heads");
    s.dim = small(k.size(2), "dim");
    if (a[5] != Py_None) s.source = vector<int32_t>(a[5], "source", at::kInt, device, s.count);
    else if (s.count > s.rows) refuse("%d slots for %d rows", s.count, s.rows);
    s.err = error_word(a[6], device);
    s.stream = stream_of(device);
    const c10::cuda::CUDAGuard guard(device);
    done(hsg_store_rows(&s));
    changed(a[2]);
    changed(a[3]);
    Py_RETURN_NONE;
  });
}

// k_cache and v_cache [pages, page_size, heads, dim] e4m3, alike in strides, and their scales [pages, blocks, heads].
hsg_cache8 cache8(PyObject* ko, PyObject* vo, PyObject* kso, PyObject* vso, int64_t heads, int64_t dim, at::Device device) {
  const Tensor &k = shaped(ko, "k_cache", 4, at::kFloat8_e4m3fn, device), &v = shaped(vo, "v_cache", 4, at::kFloat8_e4m3fn, device);
  const Tensor &ks = shaped(kso, "k_scale", 3, at::kFloat, device), &vs = shaped(vso, "v_scale", 3, at::kFloat, device);
  if (v.sizes() != k.sizes() || v.strides() != k.strides() || k.size(2) != heads || k.size(3) != dim)
    refuse("k_cache and v_cache must be alike, [pages, page_size, %lld, %lld]", (long long)heads, (long long)dim);
  const int64_t blocks = ks.size(1);
  if (vs.sizes() != ks.sizes() || !ks.is_contiguous() || !vs.is_contiguous() || ks.size(0) != k.size(0) || ks.size(2) != heads ||
      blocks < 1 || k.size(1) % blocks)
    refuse("k_scale and v_scale must be contiguous, [pages, blocks of a page, %lld]", (long long)heads);
  return hsg_cache8{k.data_ptr(), v.data_ptr(), static_cast<float*>(ks.data_ptr()), static_cast<float*>(vs.data_ptr()),
                    k.stride(0), k.stride(1), k.stride(2), small(k.size(0), "pages"), small(k.size(1), "page_size"),
                    small(k.size(1) / blocks, "block"), 0};
}

bool truth(PyObject* o, const char* name) {
  if (o != Py_True && o != Py_False) refuse("%s must be True or False", name);
  return o == Py_True;
}

// append_8bit(k, v, k_cache, v_cache, k_scale, v_scale, slots, source, positions, inv_freq, interleaved, rope_scale, q, err)
//   -> q or None
PyObject* append_8bit(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 14, [&]() -> PyObject* {
    const Tensor& k0 = tensor(a[0], "k");
    const at::Device device = device_of(k0, "k");
    const at::ScalarType dtype = k0.scalar_type();
    if (!is_16(dtype)) refuse("q, k and v must be fp16 or bf16");
    const Tensor &k = shaped(a[0], "k", 3, dtype, device), &v = shaped(a[1], "v", 3, dtype, device);
    if (k.sizes() != v.sizes()) refuse("k and v must be alike, [rows, kv heads, dim]");
    hsg_append8_args s{};
    s.size = sizeof(s);
    s.k = k.data_ptr();
    s.v = v.data_ptr();
    s.k_token_stride = k.stride(0);
    s.k_head_stride = k.stride(1);
    s.v_token_stride = v.stride(0);
    s.v_head_stride = v.stride(1);
    s.rows = small(k.size(0), "rows");
    s.hkv = small(k.size(1), "kv heads");
    s.dim = small(k.size(2), "dim");
    s.dtype = code_of(dtype);
    s.cache = cache8(a[2], a[3], a[4], a[5], s.hkv, s.dim, device);
    s.slots = vector<int32_t>(a[6], "slots", at::kInt, device);
    s.count = small(THPVariable_Unpack(a[6]).size(0), "slots");
    if (a[7] != Py_None) s.source = vector<int32_t>(a[7], "source", at::kInt, device, s.count);
    else if (s.count > s.rows) refuse("%d slots for %d rows", s.count, s.rows);
    if ((a[8] == Py_None) != (a[9] == Py_None)) refuse("positions and inv_freq go together");
    if (a[9] != Py_None) {
      s.positions = vector<int32_t>(a[8], "positions", at::kInt, device, s.count);
      s.inv_freq = vector<float>(a[9], "inv_freq", at::kFloat, device);
      s.rot = small(2 * THPVariable_Unpack(a[9]).size(0), "inv_freq");
    }
    s.interleaved = truth(a[10], "interleaved");
    s.rope_scale = real(a[11], "rope_scale");
    s.err = error_word(a[13], device);
    Tensor q_out;
    if (a[12] != Py_None) {
      if (a[7] != Py_None) refuse("q goes with entries in order, not with a source");
      const Tensor& q = shaped(a[12], "q", 3, dtype, device);
      if (q.size(0) != s.count || q.size(2) != s.dim) refuse("q must be [%d, heads, %d]", s.count, s.dim);
      s.hq = small(q.size(1), "heads");
      if (s.hq < 1) refuse("q must have heads");
      s.q = q.data_ptr();
      s.q_token_stride = q.stride(0);
      s.q_head_stride = q.stride(1);
      q_out = empty({s.count, s.hq, s.dim}, dtype, device);
      s.q_out = q_out.data_ptr();
    }
    s.stream = stream_of(device);
    const c10::cuda::CUDAGuard guard(device);
    done(hsg_append8(&s));
    for (int i = 2; i < 6; ++i) changed(a[i]);
    if (a[12] == Py_None) Py_RETURN_NONE;
    return THPVariable_Wrap(q_out);
  });
}

// attention_8bit(q, k_cache, v_cache, k_scale, v_scale, table, lens, cu, scale, max_new, mask, positions, window, sinks, workspace,
//   err) -> (out, lse)
PyObject* attention_8bit(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 16, [&]() -> PyObject* {
    const Tensor& q0 = tensor(a[0], "q");
    const at::Device device = device_of(q0, "q");
    const at::ScalarType dtype = q0.scalar_type();
    if (!is_16(dtype)) refuse("q must be fp16 or bf16");
    const Tensor& q = shaped(a[0], "q", 3, dtype, device);
    hsg_attention8_args s{};
    s.size = sizeof(s);
    s.q = q.data_ptr();
    s.q_token_stride = q.stride(0);
    s.q_head_stride = q.stride(1);
    s.tokens = small(q.size(0), "tokens");
    s.hq = small(q.size(1), "heads");
    s.dim = small(q.size(2), "dim");
    const Tensor& codes = tensor(a[1], "k_cache");
    if (codes.dim() != 4) refuse("k_cache must be a 4-d tensor");
    s.hkv = small(codes.size(2), "kv heads");
    s.cache = cache8(a[1], a[2], a[3], a[4], s.hkv, s.dim, device);
    const Tensor& table = shaped(a[5], "table", 2, at::kInt, device);
    s.rows = small(table.size(0), "rows");
    s.width = small(table.size(1), "the table's width");
    s.table = static_cast<const int32_t*>(table.data_ptr());
    s.table_stride = s.rows > 1 ? table.stride(0) : s.width;
    s.lens = vector<int32_t>(a[6], "lens", at::kInt, device, s.rows);
    s.cu = vector<int32_t>(a[7], "cu", at::kInt, device, (int64_t)s.rows + 1);
    s.scale = real(a[8], "scale");
    s.max_new = whole(a[9], "max_new", 1, HSG_MAX_NEW);
    if (a[10] != Py_None) {
      const Tensor& mask = shaped(a[10], "mask", 2, at::kInt, device);
      if (mask.size(0) != s.tokens || !mask.is_contiguous()) refuse("mask must be contiguous, [%d, words]", s.tokens);
      s.words = small(mask.size(1), "the mask's words");
      s.mask = static_cast<const uint32_t*>(mask.data_ptr());
    }
    if (a[11] != Py_None) s.positions = vector<int32_t>(a[11], "positions", at::kInt, device, s.tokens);
    s.window = whole(a[12], "window", 0, INT32_MAX);
    s.sinks = whole(a[13], "sinks", 0, INT32_MAX);
    Tensor workspace;
    if (a[14] == Py_None) workspace = empty({(int64_t)hsg_attention8_workspace(s.dim, s.tokens, s.hq)}, at::kByte, device);
    else workspace = shaped(a[14], "workspace", 1, at::kByte, device);
    s.workspace = workspace.data_ptr();
    s.workspace_bytes = workspace.numel();
    s.err = error_word(a[15], device);
    const Tensor out = empty({s.tokens, s.hq, s.dim}, dtype, device), lse = empty({s.tokens, s.hq}, at::kFloat, device);
    s.out = out.data_ptr();
    s.lse = static_cast<float*>(lse.data_ptr());
    s.dtype = code_of(dtype);
    s.stream = stream_of(device);
    const c10::cuda::CUDAGuard guard(device);
    if (s.rows == 0) {  // the library has nothing to do: no token sees anything
      out.zero_();
      lse.fill_(-std::numeric_limits<float>::infinity());
    } else {
      done(hsg_attention8(&s));
    }
    return tuple_of(out, lse);
  });
}

// token_logprobs(logits, given, top, temperature, err) -> the five tensors of Logprobs
PyObject* token_logprobs(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 5, [&]() -> PyObject* {
    const Tensor& x0 = tensor(a[0], "logits");
    const at::Device device = device_of(x0, "logits");
    hsg_logprobs_args s{};
    s.size = sizeof(s);
    s.dtype = code_of(x0.scalar_type());
    if (s.dtype < 0) refuse("logits must be fp32, fp16 or bf16");
    const Tensor& x = shaped(a[0], "logits", 2, x0.scalar_type(), device);
    s.logits = x.data_ptr();
    s.row_stride = x.stride(0);
    s.rows = small(x.size(0), "rows");
    s.vocab = small(x.size(1), "the vocabulary");
    bool flat = false;
    if (a[1] != Py_None) {
      flat = tensor(a[1], "given").dim() == 1;
      const Tensor& given = shaped(a[1], "given", flat ? 1 : 2, at::kInt, device);
      if (given.size(0) != s.rows || !given.is_contiguous()) refuse("given must be contiguous, [%d] or [%d, tokens]", s.rows, s.rows);
      s.n_given = flat ? 1 : small(given.size(1), "given");
      s.given = static_cast<const int32_t*>(given.data_ptr());
    }
    s.top = whole(a[2], "top", 0, HSG_MAX_TOP);
    s.temperature = real(a[3], "temperature");
    s.err = error_word(a[4], device);
    const int64_t rows = s.rows, at_lse = rows, at_given = 2 * rows, at_top = at_given + rows * s.n_given, at_ids = at_top + rows * s.top;
    const Tensor all = empty({at_ids + rows * s.top}, at::kFloat, device);
    float* base = static_cast<float*>(all.data_ptr());
    s.entropy = base;
    s.lse = base + at_lse;
    s.logprobs = base + at_given;
    s.top_logprobs = base + at_top;
    s.top_ids = reinterpret_cast<int32_t*>(base + at_ids);
    s.stream = stream_of(device);
    const c10::cuda::CUDAGuard guard(device);
    done(hsg_token_logprobs(&s));
    const int64_t n_given = s.n_given, top = s.top;
    return tuple_of(flat ? part(all, at::kFloat, at_given, rows) : part(all, at::kFloat, at_given, at::IntArrayRef({rows, n_given})),
                    part(all, at::kFloat, 0, rows), part(all, at::kFloat, at_lse, rows),
                    part(all, at::kFloat, at_top, at::IntArrayRef({rows, top})),
                    part(all, at::kInt, at_ids, at::IntArrayRef({rows, top})));
  });
}

#define FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(f))
PyMethodDef methods[] = {{"advance_tables", FAST(advance_tables), METH_FASTCALL, nullptr},
                         {"plan_tree", FAST(plan_tree), METH_FASTCALL, nullptr},
                         {"norm_rope", FAST(norm_rope), METH_FASTCALL, nullptr},
                         {"norm_rope_store", FAST(norm_rope_store), METH_FASTCALL, nullptr},
                         {"tree_attention", FAST(tree_attention), METH_FASTCALL, nullptr},
                         {"store_rows", FAST(store_rows), METH_FASTCALL, nullptr},
                         {"append_8bit", FAST(append_8bit), METH_FASTCALL, nullptr},
                         {"attention_8bit", FAST(attention_8bit), METH_FASTCALL, nullptr},
                         {"token_logprobs", FAST(token_logprobs), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_hsg_torch", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__hsg_torch() { return PyModule_Create(&module); }
