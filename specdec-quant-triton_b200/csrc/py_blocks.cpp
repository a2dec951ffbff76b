// py_blocks.cpp -- the Python binding of the block-scaled cache's operators (specq/_native.so).
//
// A verification step calls these operators for a few microseconds of GPU work each, and a call
// through ctypes with its argument checks in Python costs 14-28 us of host time.  Here the checks
// read the tensors' metadata directly and the C ABI of include/specq.h is called through pointers
// that specq/_lib.py binds at load (so SPECQ_LIB selects the library for both).  The checks and the
// errors are those of the rest of the package: TypeError and ValueError before any launch, ValueError
// or SpecqError from a code that the library returns.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/zeros.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <string>

#include "specq.h"

namespace {

using at::Tensor;

struct Table {
  decltype(&specq_rope) rope;
  decltype(&specq_block_append) block_append;
  decltype(&specq_block_attention) block_attention;
  decltype(&specq_block_attention_workspace) block_attention_workspace;
  decltype(&specq_block_compact) block_compact;
  decltype(&specq_pages_release) pages_release;
  decltype(&specq_pages_reserve) pages_reserve;
  decltype(&specq_pages_fork) pages_fork;
  decltype(&specq_last_error) last_error;
} lib;
PyObject* specq_error = nullptr;   // specq.SpecqError

struct Refused {                   // a check failed: a Python exception of this type and message
  PyObject* type;
  std::string text;
};
struct Raised {};                  // a Python exception is set already

[[noreturn]] void refuse(PyObject* type, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  throw Refused{type, buf};
}
#define BAD_VALUE(...) refuse(PyExc_ValueError, __VA_ARGS__)
#define BAD_TYPE(...) refuse(PyExc_TypeError, __VA_ARGS__)

std::string shape(const Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + ")";
}
const char* dtype(const Tensor& t) { return c10::toString(t.scalar_type()); }

const Tensor& tensor(const char* who, const char* what, PyObject* o) {
  if (!THPVariable_Check(o)) BAD_TYPE("%s: %s must be a tensor, got %s", who, what, Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}
const Tensor* optional(const char* who, const char* what, PyObject* o) { return o == Py_None ? nullptr : &tensor(who, what, o); }

int integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Raised{};
  if (v < INT32_MIN || v > INT32_MAX) BAD_VALUE("integer %lld does not fit 32 bits", v);
  return static_cast<int>(v);
}
int integer_or(PyObject* o, int otherwise) { return o == Py_None ? otherwise : integer(o); }

int size32(const char* who, int64_t n) {
  if (n > INT32_MAX) BAD_VALUE("%s: a dimension of %lld", who, static_cast<long long>(n));
  return static_cast<int>(n);
}

int layout_code(const char* who, PyObject* o) {
  if (PyUnicode_Check(o)) {
    if (PyUnicode_CompareWithASCIIString(o, "half") == 0) return SPECQ_ROPE_HALF;
    if (PyUnicode_CompareWithASCIIString(o, "interleaved") == 0) return SPECQ_ROPE_INTERLEAVED;
  }
  BAD_VALUE("%s: layout must be 'half' or 'interleaved'", who);
}

int row_code(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kHalf: return SPECQ_DTYPE_F16;
    case at::kBFloat16: return SPECQ_DTYPE_BF16;
    case at::kFloat: return SPECQ_DTYPE_F32;
    default: return -1;
  }
}
int cache_code(const Tensor& t) { return t.scalar_type() == at::kChar ? SPECQ_CACHE_INT8 : SPECQ_CACHE_E4M3; }

void rows3(const char* who, const char* what, const Tensor& t, bool with_f32) {
  const int c = row_code(t);
  if (c < 0 || (c == SPECQ_DTYPE_F32 && !with_f32))
    BAD_TYPE("%s: %s must be float16, bfloat16%s, got %s", who, what, with_f32 ? " or float32" : "", dtype(t));
  if (t.dim() != 3 || (t.stride(2) != 1 && t.size(2) > 1))
    BAD_VALUE("%s: %s must be [rows, heads, dim] with unit inner stride, got %s", who, what, shape(t).c_str());
}

// A tensor that a kernel writes: no two of its elements share memory by a stride of 0.
void written(const char* who, const char* what, const Tensor& t) {
  for (int64_t i = 0; i < t.dim(); ++i)
    if (t.stride(i) == 0 && t.size(i) > 1) BAD_VALUE("%s: %s is written and must not be expanded (dimension %lld)", who, what, (long long)i);
}

// int32, `dims` dimensions, at least n0 (and n1) long (-1: any), unit inner stride
void int32s(const char* who, const char* what, const Tensor& t, int dims, int64_t n0, int64_t n1 = -1) {
  if (t.scalar_type() != at::kInt) BAD_TYPE("%s: %s must be int32, got %s", who, what, dtype(t));
  if (t.dim() != dims || (n0 >= 0 && t.size(0) < n0) || (dims == 2 && n1 >= 0 && t.size(1) < n1))
    BAD_VALUE("%s: %s is too small or of another rank: %s", who, what, shape(t).c_str());
  if (t.size(dims - 1) > 1 && t.stride(dims - 1) != 1) BAD_VALUE("%s: %s needs unit inner stride", who, what);
}

struct Cache {
  const Tensor &kc, &vc, &ks, &vs;
  int d;                 // index of the page dimension: 1 with layers, else 0
  int64_t L, P, page, H, D;
  int64_t sl() const { return d ? kc.stride(0) : 0; }
  int64_t s_sl() const { return d ? ks.stride(0) : 0; }
};

Cache cache(const char* who, PyObject* const* a, bool layers, bool writes = true) {
  const Tensor &kc = tensor(who, "kc", a[0]), &vc = tensor(who, "vc", a[1]), &ks = tensor(who, "ks", a[2]), &vs = tensor(who, "vs", a[3]);
  if ((kc.scalar_type() != at::kChar && kc.scalar_type() != at::kFloat8_e4m3fn) || vc.scalar_type() != kc.scalar_type())
    BAD_TYPE("%s: kc and vc must both be int8 or both float8_e4m3fn, got %s and %s", who, dtype(kc), dtype(vc));
  if (ks.scalar_type() != at::kFloat || vs.scalar_type() != at::kFloat) BAD_TYPE("%s: ks and vs must be float32", who);
  const int dims = layers && kc.dim() == 5 ? 5 : 4, d = dims - 4;
  if (kc.dim() != dims || vc.sizes() != kc.sizes() || vc.strides() != kc.strides())
    BAD_VALUE("%s: kc and vc must be alike with %d dimensions, got %s and %s", who, dims, shape(kc).c_str(), shape(vc).c_str());
  if (kc.stride(dims - 1) != 1) BAD_VALUE("%s: the cache needs unit stride along D", who);
  bool ok = ks.dim() == dims - 2 && vs.sizes() == ks.sizes() && vs.strides() == ks.strides();
  for (int i = 0; ok && i <= d; ++i) ok = ks.size(i) == kc.size(i);
  if (!ok || ks.size(d + 1) != kc.size(d + 2))
    BAD_VALUE("%s: ks and vs must be alike, one scale for each page and head of %s, got %s and %s", who, shape(kc).c_str(),
              shape(ks).c_str(), shape(vs).c_str());
  if (writes) {              // vc and vs are alike
    written(who, "the cache", kc);
    written(who, "the cache's scales", ks);
  }
  return Cache{kc, vc, ks, vs, d, d ? kc.size(0) : 1, kc.size(d), kc.size(d + 1), kc.size(d + 2), kc.size(d + 3)};
}

// every tensor on one CUDA device
void same_device(const char* who, std::initializer_list<const Tensor*> ts) {
  const Tensor* first = nullptr;
  for (const Tensor* t : ts) {
    if (t == nullptr) continue;
    if (!t->is_cuda()) BAD_VALUE("specq kernels take CUDA tensors (there is no CPU path)");
    if (first == nullptr) {
      first = t;
      const int now = static_cast<int>(c10::cuda::current_device());   // whose stream the call uses
      if (t->get_device() != now) BAD_VALUE("%s: tensors on cuda:%d, the current device is cuda:%d", who, t->get_device(), now);
    } else if (t->get_device() != first->get_device()) {
      BAD_VALUE("%s: tensors on different devices", who);
    }
  }
}

void rotary_table(const char* who, const Tensor& t, int64_t D) {
  if (t.scalar_type() != at::kFloat || t.dim() != 2 || !t.is_contiguous()) BAD_TYPE("%s: table must be a contiguous float32 [n_pos, rot]", who);
  if (t.size(0) < 1 || t.size(1) < 2 || t.size(1) % 2 || t.size(1) > D)
    BAD_VALUE("%s: table %s needs positions and an even rot <= %lld", who, shape(t).c_str(), static_cast<long long>(D));
}

// A plan whose first n values the kernels read.
const int32_t* plan_of(const char* who, const Tensor* plan, int n) {
  if (plan == nullptr) return nullptr;
  if (plan->scalar_type() != at::kInt) BAD_TYPE("%s: plan must be int32, got %s", who, dtype(*plan));
  if (plan->numel() < n || !plan->is_contiguous()) BAD_VALUE("%s: plan must be contiguous, %d values or more, got %s", who, n, shape(*plan).c_str());
  return static_cast<const int32_t*>(plan->data_ptr());
}

template <typename T>
T* ptr(const Tensor& t) { return static_cast<T*>(t.data_ptr()); }
template <typename T>
T* ptr(const Tensor* t) { return t == nullptr ? nullptr : static_cast<T*>(t->data_ptr()); }

void* stream() { return c10::cuda::getCurrentCUDAStream().stream(); }

void check(int rc) {
  if (rc == SPECQ_OK) return;
  const char* msg = lib.last_error();
  if (rc == SPECQ_ERR_INVALID_ARG) BAD_VALUE("libspecq: %s", msg);
  PyObject* e = PyObject_CallFunction(specq_error, "is", rc, msg);
  if (e != nullptr) {
    PyErr_SetObject(specq_error, e);
    Py_DECREF(e);
  }
  throw Raised{};
}

// A new output like x; rows that the call does not reach (all = false) are zeros.
Tensor new_rows(const Tensor& x, bool all) { return all ? at::empty(x.sizes(), x.options()) : at::zeros(x.sizes(), x.options()); }

Tensor new_int32(const Tensor& like, int64_t n) { return at::empty({n}, like.options().dtype(at::kInt)); }

PyObject* wrap(const Tensor& t) { return THPVariable_Wrap(t); }
PyObject* none() { Py_RETURN_NONE; }

// ---- the operators: positional arguments in the order of specq/blocks.py ---------------------------
PyObject* rope(PyObject* const* a) {
  const char* who = "rope";
  const int lay = layout_code(who, a[3]);
  const Tensor &x = tensor(who, "x", a[0]), &pos = tensor(who, "pos", a[1]), &table = tensor(who, "table", a[2]);
  rows3(who, "x", x, true);
  rotary_table(who, table, x.size(2));
  int32s(who, "pos", pos, 1, x.size(0));
  const int inverse = PyObject_IsTrue(a[4]);
  if (inverse < 0) throw Raised{};
  const Tensor* given = optional(who, "out", a[5]);
  const Tensor* plan = optional(who, "plan", a[6]);
  const int32_t* plan_at = plan_of(who, plan, 1);
  if (given != nullptr) {
    rows3(who, "out", *given, true);
    if (given->scalar_type() != x.scalar_type() || given->sizes() != x.sizes())
      BAD_VALUE("rope: out must be %s %s, got %s %s", dtype(x), shape(x).c_str(), dtype(*given), shape(*given).c_str());
    written(who, "out", *given);
  }
  if (c10::GradMode::is_enabled()) {
    if (given != nullptr && (x.requires_grad() || given->requires_grad())) BAD_VALUE("rope: no out for a tensor that requires grad");
    if (table.requires_grad()) BAD_VALUE("rope: the table has no gradient");
    if (x.requires_grad()) Py_RETURN_NOTIMPLEMENTED;   // specq/blocks.py records the gradient and calls again
  }
  same_device(who, {&x, &pos, &table, given, plan});
  const Tensor out = given != nullptr ? *given : new_rows(x, plan == nullptr);
  check(lib.rope(x.data_ptr(), x.stride(0), x.stride(1), out.data_ptr(), out.stride(0), out.stride(1), row_code(x), ptr<int32_t>(pos),
                 ptr<float>(table), size32(who, table.size(0)), size32(who, x.size(0)), size32(who, x.size(1)), size32(who, x.size(2)),
                 size32(who, table.size(1)), lay, inverse, plan_at, stream()));
  return wrap(out);
}

PyObject* kv_append_blocks(PyObject* const* a) {
  // k, v, kc, vc, ks, vs, block_tbl, ctx_len, q_len, q, q_out, table, pos, layout, plan, n_seqs, ql_max
  const char* who = "kv_append_blocks";
  const int lay = layout_code(who, a[13]);
  const Cache c = cache(who, a + 2, false);
  const Tensor &k = tensor(who, "k", a[0]), &v = tensor(who, "v", a[1]);
  rows3(who, "k", k, false);
  rows3(who, "v", v, false);
  const Tensor &tbl = tensor(who, "block_tbl", a[6]), &ctx = tensor(who, "ctx_len", a[7]);
  int32s(who, "block_tbl", tbl, 2, -1);
  int32s(who, "ctx_len", ctx, 1, tbl.size(0));
  const int B = size32(who, tbl.size(0)), q_len = integer(a[8]);
  const int n_seqs = integer_or(a[15], B), ql_max = integer_or(a[16], q_len);
  if (n_seqs < 0 || n_seqs > B || q_len < 0 || q_len > ql_max)
    BAD_VALUE("%s: n_seqs=%d of %d, q_len=%d of %d", who, n_seqs, B, q_len, ql_max);
  const Tensor* plan = optional(who, "plan", a[14]);
  const int32_t* plan_at = plan_of(who, plan, 2);
  const int64_t need = plan != nullptr ? static_cast<int64_t>(B) * ql_max : static_cast<int64_t>(n_seqs) * q_len;
  auto kv = [&](const char* what, const Tensor& t) {
    if (t.scalar_type() != k.scalar_type() || t.size(1) != c.H || t.size(2) != c.D || t.size(0) < need)
      BAD_VALUE("%s: %s must be %s [>= %lld, %lld, %lld], got %s %s", who, what, dtype(k), (long long)need, (long long)c.H,
                (long long)c.D, dtype(t), shape(t).c_str());
  };
  kv("k", k);
  kv("v", v);
  const Tensor *q = optional(who, "q", a[9]), *q_given = optional(who, "q_out", a[10]), *table = optional(who, "table", a[11]),
               *pos = optional(who, "pos", a[12]);
  if (table != nullptr) rotary_table(who, *table, c.D);
  else if (q != nullptr || pos != nullptr) BAD_VALUE("%s: q and pos need a rotary table", who);
  if (pos != nullptr) int32s(who, "pos", *pos, 1, need);
  if (q != nullptr) {
    rows3(who, "q", *q, false);
    if (q->scalar_type() != k.scalar_type() || q->size(2) != c.D || q->size(0) < need)
      BAD_VALUE("%s: q must be %s [>= %lld, H, %lld], got %s %s", who, dtype(k), (long long)need, (long long)c.D, dtype(*q),
                shape(*q).c_str());
    if (q_given != nullptr) {
      rows3(who, "q_out", *q_given, false);
      if (q_given->scalar_type() != q->scalar_type() || q_given->sizes() != q->sizes())
        BAD_VALUE("%s: q_out must be %s %s", who, dtype(*q), shape(*q).c_str());
      written(who, "q_out", *q_given);
    }
  } else if (q_given != nullptr) {
    BAD_VALUE("%s: q_out without q", who);
  }
  same_device(who, {&c.kc, &c.vc, &c.ks, &c.vs, &k, &v, q, q_given, table, pos, &tbl, &ctx, plan});
  Tensor q_out;
  if (q != nullptr) q_out = q_given != nullptr ? *q_given : new_rows(*q, plan == nullptr && q->size(0) == need);
  const bool qs = q != nullptr;
  check(lib.block_append(
      k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), qs ? q->data_ptr() : nullptr,
      qs ? q->stride(0) : 0, qs ? q->stride(1) : 0, qs ? q_out.data_ptr() : nullptr, qs ? q_out.stride(0) : 0,
      qs ? q_out.stride(1) : 0, row_code(k), ptr<float>(table), table ? size32(who, table->size(0)) : 0,
      table ? size32(who, table->size(1)) : 0, lay, ptr<int32_t>(pos), c.kc.data_ptr(), c.vc.data_ptr(), c.kc.stride(0),
      c.kc.stride(1), c.kc.stride(2), cache_code(c.kc), size32(who, c.P), ptr<float>(c.ks), ptr<float>(c.vs), c.ks.stride(0),
      c.ks.stride(1), ptr<int32_t>(tbl), tbl.stride(0), size32(who, tbl.size(1)), ptr<int32_t>(ctx), plan_at, B, n_seqs,
      q_len, ql_max, qs ? size32(who, q->size(1)) : 0, size32(who, c.H), size32(who, c.D), size32(who, c.page), stream()));
  return qs ? wrap(q_out) : none();
}

PyObject* paged_attention_blocks(PyObject* const* a) {
  // q, kc, vc, ks, vs, block_tbl, ctx_len, q_len, tree, sm_scale, out, plan, n_seqs, ql_max
  const char* who = "paged_attention_blocks";
  const Cache c = cache(who, a + 1, false, false);
  const Tensor& q = tensor(who, "q", a[0]);
  if (q.scalar_type() != at::kHalf && q.scalar_type() != at::kBFloat16)
    BAD_TYPE("%s: q must be float16 or bfloat16, got %s", who, dtype(q));
  const Tensor &tbl = tensor(who, "block_tbl", a[5]), &ctx = tensor(who, "ctx_len", a[6]);
  int32s(who, "block_tbl", tbl, 2, -1);
  int32s(who, "ctx_len", ctx, 1, tbl.size(0));
  const int B = size32(who, tbl.size(0));
  const bool packed = q.dim() == 3;
  if (packed ? a[7] == Py_None : q.dim() != 4) {
    if (packed) BAD_VALUE("%s: packed queries need q_len", who);
    BAD_VALUE("%s: q must have 3 or 4 dimensions, got %s", who, shape(q).c_str());
  }
  const Tensor* plan = optional(who, "plan", a[11]);
  const int32_t* plan_at = plan_of(who, plan, 2);
  const int q_len = packed ? integer(a[7]) : integer_or(a[7], size32(who, q.size(1)));
  if (!packed && (q.size(0) < B || q.size(1) < q_len))
    BAD_VALUE("%s: q is %s for %d sequences of %d tokens", who, shape(q).c_str(), B, q_len);
  const int n_seqs = integer_or(a[12], B);
  const int ql_max = integer_or(a[13], packed || plan == nullptr ? q_len : size32(who, q.size(1)));
  if (n_seqs < 0 || n_seqs > B || q_len < 0 || q_len > ql_max || (!packed && plan != nullptr && q.size(1) < ql_max))
    BAD_VALUE("%s: n_seqs=%d of %d, q_len=%d of %d, q %s", who, n_seqs, B, q_len, ql_max, shape(q).c_str());
  if (packed && q.size(0) < (plan != nullptr ? static_cast<int64_t>(B) * ql_max : static_cast<int64_t>(n_seqs) * q_len))
    BAD_VALUE("%s: %lld packed rows for %d sequences of %d tokens", who, (long long)q.size(0), B, ql_max);
  // to the kernels a batch stride of 0 says packed rows
  if (!packed && q.stride(0) == 0 && (plan != nullptr ? B : n_seqs) > 1)
    BAD_VALUE("%s: q is expanded over the sequences (its stride is 0); give each sequence its rows", who);
  const int64_t H = q.size(-2);
  if (q.size(-1) != c.D || c.H == 0 || H % c.H)
    BAD_VALUE("%s: q heads (%lld, %lld) do not fit the cache's (%lld, %lld)", who, (long long)H, (long long)q.size(-1), (long long)c.H,
              (long long)c.D);
  const Tensor *given = optional(who, "out", a[10]), *tree = optional(who, "tree", a[8]);
  if (given != nullptr && (given->scalar_type() != q.scalar_type() || given->sizes() != q.sizes()))
    BAD_VALUE("%s: out must be %s %s, got %s %s", who, dtype(q), shape(q).c_str(), dtype(*given), shape(*given).c_str());
  if (given != nullptr) written(who, "out", *given);
  if (q.stride(-1) != 1 || (given != nullptr && given->stride(-1) != 1)) BAD_VALUE("%s: q and out need unit stride along D", who);
  float sm = 1.f / std::sqrt(static_cast<float>(c.D));
  if (a[9] != Py_None) {
    const double v = PyFloat_AsDouble(a[9]);
    if (v == -1.0 && PyErr_Occurred()) throw Raised{};
    if (!(v > 0)) BAD_VALUE("%s: sm_scale=%g must be positive", who, v);
    sm = static_cast<float>(v);
  }
  if (tree != nullptr && (tree->scalar_type() != at::kLong || tree->dim() != 2 || tree->size(0) < B || tree->size(1) < ql_max))
    BAD_VALUE("%s: tree must be int64 [>= %d, >= %d], got %s %s", who, B, ql_max, dtype(*tree), shape(*tree).c_str());
  same_device(who, {&c.kc, &c.vc, &c.ks, &c.vs, &q, given, &tbl, &ctx, tree, plan});
  const bool all = plan == nullptr && n_seqs == B &&
                   (packed ? q.size(0) == static_cast<int64_t>(B) * q_len : q.size(0) == B && q.size(1) == q_len);
  const Tensor out = given != nullptr ? *given : new_rows(q, all);
  int64_t bytes = 0;
  const int cols = size32(who, tbl.size(1)), h = size32(who, H), hk = size32(who, c.H), D = size32(who, c.D), page = size32(who, c.page);
  check(lib.block_attention_workspace(B, n_seqs, q_len, ql_max, h, hk, D, page, cols, plan != nullptr, &bytes));
  // from torch's allocator on the current stream: nothing outlives the call but what its launches need
  Tensor ws;
  if (bytes > 0) ws = at::empty({bytes}, q.options().dtype(at::kByte));
  const int o = packed ? 0 : 1;
  check(lib.block_attention(
      q.data_ptr(), packed ? 0 : q.stride(0), q.stride(o), q.stride(o + 1), row_code(q), c.kc.data_ptr(), c.vc.data_ptr(), c.kc.stride(0),
      c.kc.stride(1), c.kc.stride(2), cache_code(c.kc), size32(who, c.P), ptr<float>(c.ks), ptr<float>(c.vs), c.ks.stride(0), c.ks.stride(1),
      ptr<int32_t>(tbl), tbl.stride(0), cols, ptr<int32_t>(ctx), tree ? reinterpret_cast<const uint64_t*>(tree->data_ptr()) : nullptr,
      tree ? tree->stride(0) : 0, tree ? tree->stride(1) : 0, sm, out.data_ptr(), packed ? 0 : out.stride(0), out.stride(o),
      out.stride(o + 1), plan_at, B, n_seqs, q_len, ql_max, h, hk, D, page, bytes > 0 ? ws.data_ptr() : nullptr, bytes, stream()));
  return wrap(out);
}

PyObject* kv_compact_blocks(PyObject* const* a) {
  // kc, vc, ks, vs, block_tbl, ctx_len, q_len, accept, n_accept, ctx_out
  const char* who = "kv_compact_blocks";
  const Cache c = cache(who, a, true);
  const Tensor &tbl = tensor(who, "block_tbl", a[4]), &ctx = tensor(who, "ctx_len", a[5]), &acc = tensor(who, "accept", a[7]),
               &n_acc = tensor(who, "n_accept", a[8]);
  int32s(who, "block_tbl", tbl, 2, -1);
  const int64_t B = tbl.size(0);
  int32s(who, "ctx_len", ctx, 1, B);
  int32s(who, "accept", acc, 2, B);
  int32s(who, "n_accept", n_acc, 1, B);
  const int q_len = integer(a[6]);
  if (q_len < 0) BAD_VALUE("%s: q_len=%d", who, q_len);
  if (c.L == 0) BAD_VALUE("%s: a cache without layers", who);
  const Tensor* given = optional(who, "ctx_out", a[9]);
  if (given != nullptr) int32s(who, "ctx_out", *given, 1, B);
  same_device(who, {&c.kc, &c.vc, &c.ks, &c.vs, &tbl, &ctx, &acc, &n_acc, given});
  const Tensor out = given != nullptr ? *given : new_int32(ctx, B);
  const int d = c.d;
  check(lib.block_compact(c.kc.data_ptr(), c.vc.data_ptr(), c.sl(), c.kc.stride(d), c.kc.stride(d + 1), c.kc.stride(d + 2), cache_code(c.kc),
                          size32(who, c.L), size32(who, c.P), ptr<float>(c.ks), ptr<float>(c.vs), c.s_sl(), c.ks.stride(d),
                          c.ks.stride(d + 1), ptr<int32_t>(tbl), tbl.stride(0), size32(who, tbl.size(1)), ptr<int32_t>(ctx),
                          ptr<int32_t>(acc), acc.stride(0), size32(who, acc.size(1)), ptr<int32_t>(n_acc), ptr<int32_t>(out),
                          size32(who, B), q_len, size32(who, c.H), size32(who, c.D), size32(who, c.page), stream()));
  return wrap(out);
}

struct Pool {
  const Tensor &ref, &tbl, &held;
  int P, S, C;
  int64_t ld;
};

Pool pool(const char* who, PyObject* const* a) {
  const Tensor &ref = tensor(who, "ref", a[0]), &tbl = tensor(who, "tbl", a[1]), &held = tensor(who, "held", a[2]);
  int32s(who, "ref", ref, 1, -1);
  int32s(who, "tbl", tbl, 2, -1);
  int32s(who, "held", held, 1, tbl.size(0));
  const int C = size32(who, tbl.size(1));
  return Pool{ref, tbl, held, size32(who, ref.size(0)), size32(who, tbl.size(0)), C, tbl.size(0) > 1 ? tbl.stride(0) : C > 0 ? C : 1};
}

PyObject* pages_release(PyObject* const* a) {
  const char* who = "pages_release";
  const Pool p = pool(who, a);
  const Tensor& drop = tensor(who, "drop", a[3]);
  if ((drop.scalar_type() != at::kBool && drop.scalar_type() != at::kByte) || drop.dim() != 1 || drop.size(0) < p.S ||
      (drop.size(0) > 1 && drop.stride(0) != 1))
    BAD_VALUE("%s: drop must be a contiguous bool [%d], got %s %s", who, p.S, dtype(drop), shape(drop).c_str());
  same_device(who, {&p.ref, &p.tbl, &p.held, &drop});
  check(lib.pages_release(ptr<int32_t>(p.ref), p.P, ptr<int32_t>(p.tbl), p.ld, ptr<int32_t>(p.held), p.S, p.C, ptr<uint8_t>(drop), stream()));
  return none();
}

PyObject* pages_reserve(PyObject* const* a) {
  // ref, tbl, held, want_len, page, short
  const char* who = "pages_reserve";
  const Pool p = pool(who, a);
  const Tensor& want = tensor(who, "want_len", a[3]);
  int32s(who, "want_len", want, 1, p.S);
  const int page = integer(a[4]);
  if (page < 1) BAD_VALUE("%s: page=%d", who, page);
  const Tensor* given = optional(who, "short", a[5]);
  if (given != nullptr) int32s(who, "short", *given, 1, 1);
  same_device(who, {&p.ref, &p.tbl, &p.held, &want, given});
  const Tensor out = given != nullptr ? *given : new_int32(p.ref, 1);
  check(lib.pages_reserve(ptr<int32_t>(p.ref), p.P, ptr<int32_t>(p.tbl), p.ld, ptr<int32_t>(p.held), p.S, p.C, ptr<int32_t>(want), page,
                          ptr<int32_t>(out), stream()));
  return wrap(out);
}

PyObject* pages_fork(PyObject* const* a) {
  // kc, vc, ks, vs, ref, tbl, held, parent, length, short
  const char* who = "pages_fork";
  const Cache c = cache(who, a, true);
  const Pool p = pool(who, a + 4);
  const Tensor &parent = tensor(who, "parent", a[7]), &length = tensor(who, "length", a[8]);
  int32s(who, "parent", parent, 1, p.S);
  int32s(who, "length", length, 1, p.S);
  if (c.P < p.P) BAD_VALUE("%s: a pool of %d pages over a cache of %lld", who, p.P, (long long)c.P);
  const Tensor* given = optional(who, "short", a[9]);
  if (given != nullptr) int32s(who, "short", *given, 1, 1);
  same_device(who, {&p.ref, &c.kc, &c.vc, &c.ks, &c.vs, &p.tbl, &p.held, &parent, &length, given});
  const Tensor out = given != nullptr ? *given : new_int32(p.ref, 1);
  const Tensor scratch = new_int32(p.ref, static_cast<int64_t>(p.S) * (p.C + 2));
  const int d = c.d;
  check(lib.pages_fork(c.kc.data_ptr(), c.vc.data_ptr(), c.sl(), c.kc.stride(d), c.kc.stride(d + 1), c.kc.stride(d + 2), size32(who, c.L),
                       ptr<float>(c.ks), ptr<float>(c.vs), c.s_sl(), c.ks.stride(d), c.ks.stride(d + 1), ptr<int32_t>(p.ref), p.P,
                       ptr<int32_t>(p.tbl), p.ld, ptr<int32_t>(p.held), p.S, p.C, ptr<int32_t>(parent), ptr<int32_t>(length),
                       ptr<int32_t>(scratch), ptr<int32_t>(out), size32(who, c.H), size32(who, c.D), size32(who, c.page), stream()));
  return wrap(out);
}

// No C++ exception leaves an entry: a failed check, an out-of-memory of torch's allocator or any other
// becomes the Python exception.
template <PyObject* (*F)(PyObject* const*), int N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "%d arguments expected, got %zd", N, n);
    return nullptr;
  }
  if (lib.rope == nullptr) {
    PyErr_SetString(PyExc_RuntimeError, "the library is not bound");
    return nullptr;
  }
  try {
    return F(args);
  } catch (const Refused& r) {
    PyErr_SetString(r.type, r.text.c_str());
  } catch (const Raised&) {
  } catch (const c10::OutOfMemoryError& e) {
    PyErr_SetString(PyExc_MemoryError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 2 || !PyDict_Check(args[0])) {
    PyErr_SetString(PyExc_TypeError, "bind(addresses, error type)");
    return nullptr;
  }
  Table t = {};
  const struct { const char* name; void** at; } names[] = {
      {"specq_rope", reinterpret_cast<void**>(&t.rope)},
      {"specq_block_append", reinterpret_cast<void**>(&t.block_append)},
      {"specq_block_attention", reinterpret_cast<void**>(&t.block_attention)},
      {"specq_block_attention_workspace", reinterpret_cast<void**>(&t.block_attention_workspace)},
      {"specq_block_compact", reinterpret_cast<void**>(&t.block_compact)},
      {"specq_pages_release", reinterpret_cast<void**>(&t.pages_release)},
      {"specq_pages_reserve", reinterpret_cast<void**>(&t.pages_reserve)},
      {"specq_pages_fork", reinterpret_cast<void**>(&t.pages_fork)},
      {"specq_last_error", reinterpret_cast<void**>(&t.last_error)},
  };
  for (const auto& e : names) {
    PyObject* v = PyDict_GetItemString(args[0], e.name);
    if (v == nullptr) {
      PyErr_Format(PyExc_KeyError, "%s", e.name);
      return nullptr;
    }
    *e.at = PyLong_AsVoidPtr(v);
    if (PyErr_Occurred()) return nullptr;
  }
  Py_INCREF(args[1]);
  Py_XSETREF(specq_error, args[1]);
  lib = t;
  Py_RETURN_NONE;
}

#define FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL
PyMethodDef methods[] = {
    {"bind", FAST(bind), "bind(addresses, error type): the library's entry points"},
    {"rope", FAST((entry<rope, 7>)), nullptr},
    {"kv_append_blocks", FAST((entry<kv_append_blocks, 17>)), nullptr},
    {"paged_attention_blocks", FAST((entry<paged_attention_blocks, 14>)), nullptr},
    {"kv_compact_blocks", FAST((entry<kv_compact_blocks, 10>)), nullptr},
    {"pages_release", FAST((entry<pages_release, 4>)), nullptr},
    {"pages_reserve", FAST((entry<pages_reserve, 6>)), nullptr},
    {"pages_fork", FAST((entry<pages_fork, 10>)), nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_native", "binding of the block-scaled cache's operators", -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__native(void) { return PyModule_Create(&module); }
