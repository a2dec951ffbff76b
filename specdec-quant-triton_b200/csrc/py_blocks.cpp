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
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <optional>
#include <string>
#include <vector>

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
  decltype(&specq_pages_trim) pages_trim;
  decltype(&specq_qk_norm_rope) qk_norm_rope;
  decltype(&specq_qk_norm_rope_grad) qk_norm_rope_grad;
  decltype(&specq_qk_norm_rope_grad_workspace) qk_norm_rope_grad_workspace;
  decltype(&specq_beam_select) beam_select;
  decltype(&specq_beam_select_workspace) beam_select_workspace;
  decltype(&specq_beam_reorder) beam_reorder;
  decltype(&specq_attention_mass) attention_mass;
  decltype(&specq_attention_mass_workspace) attention_mass_workspace;
  decltype(&specq_block_evict) block_evict;
  decltype(&specq_block_evict_workspace) block_evict_workspace;
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

// The call has written these tensors of the caller: a backward pass that saved one is to know.
void wrote(std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    if (t != nullptr && !t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}

// Forward-mode differentiation has no form here: a tensor that carries a tangent is refused, since the result would have none.
void no_tangent(const char* who, std::initializer_list<const Tensor*> ts) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const Tensor* t : ts)
    if (t != nullptr && t->_fw_grad(0).defined()) BAD_VALUE("%s: no forward-mode gradient; unpack the dual tensor", who);
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
  no_tangent(who, {&x, &table, given});
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
  wrote({given});
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
  wrote({&c.kc, &c.vc, &c.ks, &c.vs, q_given});
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
  wrote({given});
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
  wrote({&c.kc, &c.vc, &c.ks, &c.vs, given});
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
  // ref, tbl, held, drop, length, page
  const char* who = "pages_release";
  const Pool p = pool(who, a);
  const Tensor& drop = tensor(who, "drop", a[3]);
  if ((drop.scalar_type() != at::kBool && drop.scalar_type() != at::kByte) || drop.dim() != 1 || drop.size(0) < p.S ||
      (drop.size(0) > 1 && drop.stride(0) != 1))
    BAD_VALUE("%s: drop must be a contiguous bool [%d], got %s %s", who, p.S, dtype(drop), shape(drop).c_str());
  const Tensor* length = optional(who, "length", a[4]);
  if ((length == nullptr) != (a[5] == Py_None)) BAD_VALUE("%s: length and page go together", who);
  if (length == nullptr) {
    same_device(who, {&p.ref, &p.tbl, &p.held, &drop});
    check(lib.pages_release(ptr<int32_t>(p.ref), p.P, ptr<int32_t>(p.tbl), p.ld, ptr<int32_t>(p.held), p.S, p.C, ptr<uint8_t>(drop), stream()));
    wrote({&p.ref, &p.tbl, &p.held});
    return none();
  }
  int32s(who, "length", *length, 1, p.S);
  const int page = integer(a[5]);
  if (page < 1) BAD_VALUE("%s: page=%d", who, page);
  same_device(who, {&p.ref, &p.tbl, &p.held, &drop, length});
  check(lib.pages_trim(ptr<int32_t>(p.ref), p.P, ptr<int32_t>(p.tbl), p.ld, ptr<int32_t>(p.held), p.S, p.C, ptr<uint8_t>(drop),
                       ptr<int32_t>(*length), page, stream()));
  wrote({&p.ref, &p.tbl, &p.held});
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
  wrote({&p.ref, &p.tbl, &p.held, given});
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
  wrote({&c.kc, &c.vc, &c.ks, &c.vs, &p.ref, &p.tbl, &p.held, given});
  return wrap(out);
}

// ---- heads: norm and turn ---------------------------------------------------------------------------
// q and k rows with their weights and angles, as qk_norm_rope and its gradient take them.
struct Heads {
  const Tensor &q, &k, &pos, &table;
  const Tensor *qw, *kw, *plan;
  float eps;
  int layout;
};

Heads heads(const char* who, PyObject* q_, PyObject* k_, PyObject* qw_, PyObject* kw_, PyObject* pos_, PyObject* table_, PyObject* eps_,
            PyObject* layout_, PyObject* plan_) {
  const int lay = layout_code(who, layout_);
  const Tensor &q = tensor(who, "q", q_), &k = tensor(who, "k", k_), &pos = tensor(who, "pos", pos_), &table = tensor(who, "table", table_);
  rows3(who, "q", q, true);
  rows3(who, "k", k, true);
  if (k.scalar_type() != q.scalar_type() || k.size(0) != q.size(0) || k.size(2) != q.size(2))
    BAD_VALUE("%s: q and k must be of one type, with as many rows and elements a head, got %s %s and %s %s", who, dtype(q),
              shape(q).c_str(), dtype(k), shape(k).c_str());
  const Tensor *qw = optional(who, "q_weight", qw_), *kw = optional(who, "k_weight", kw_);
  int f32 = -1;
  for (const Tensor* w : {qw, kw}) {
    if (w == nullptr) continue;
    if (w->scalar_type() != q.scalar_type() && w->scalar_type() != at::kFloat)
      BAD_TYPE("%s: weights must be %s or float32, got %s", who, dtype(q), dtype(*w));
    if (w->dim() != 1 || w->size(0) != q.size(2) || (w->size(0) > 1 && w->stride(0) != 1))
      BAD_VALUE("%s: weights must be contiguous [%lld], got %s", who, (long long)q.size(2), shape(*w).c_str());
    const int is = w->scalar_type() == at::kFloat;
    if (f32 >= 0 && f32 != is) BAD_TYPE("%s: both weights must be of one type", who);
    f32 = is;
  }
  rotary_table(who, table, q.size(2));
  int32s(who, "pos", pos, 1, q.size(0));
  const double eps = PyFloat_AsDouble(eps_);
  if (eps == -1.0 && PyErr_Occurred()) throw Raised{};
  if (!(static_cast<float>(eps) > 0.f) || !(eps < 3e38)) BAD_VALUE("%s: eps=%g must be positive and finite", who, eps);
  const Tensor* plan = optional(who, "plan", plan_);
  plan_of(who, plan, 1);
  return Heads{q, k, pos, table, qw, kw, plan, static_cast<float>(eps), lay};
}

PyObject* pack(std::initializer_list<Tensor> ts) {    // undefined tensors become None
  PyObject* out = PyTuple_New(static_cast<Py_ssize_t>(ts.size()));
  if (out == nullptr) throw Raised{};
  Py_ssize_t i = 0;
  for (const Tensor& t : ts) {
    PyObject* o = t.defined() ? wrap(t) : none();
    if (o == nullptr) {
      Py_DECREF(out);
      throw Raised{};
    }
    PyTuple_SET_ITEM(out, i++, o);
  }
  return out;
}

int64_t stride_of(const Tensor& t, int i) { return t.defined() ? t.stride(i) : 0; }
void* raw(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor or_none(const Tensor* t) { return t == nullptr ? Tensor() : *t; }
std::optional<Tensor> maybe(const Tensor* t) { return t == nullptr ? std::nullopt : std::optional<Tensor>(*t); }

// The launch of checked tensors (undefined: not given); the library's code.
int launch_qk_norm_rope(const Tensor& q, const Tensor& k, const Tensor& qw, const Tensor& kw, const Tensor& pos, const Tensor& table,
                        const Tensor& plan, float eps, int layout, const Tensor& q_out, const Tensor& k_out) {
  const int f32 = (qw.defined() && qw.scalar_type() == at::kFloat) || (kw.defined() && kw.scalar_type() == at::kFloat);
  return lib.qk_norm_rope(q.data_ptr(), q.stride(0), q.stride(1), q_out.data_ptr(), q_out.stride(0), q_out.stride(1), k.data_ptr(),
                          k.stride(0), k.stride(1), k_out.data_ptr(), k_out.stride(0), k_out.stride(1), row_code(q), raw(qw), raw(kw),
                          f32, eps, ptr<int32_t>(pos), ptr<float>(table), static_cast<int>(table.size(0)), static_cast<int>(q.size(0)),
                          static_cast<int>(q.size(1)), static_cast<int>(k.size(1)), static_cast<int>(q.size(2)),
                          static_cast<int>(table.size(1)), layout, static_cast<const int32_t*>(raw(plan)), stream());
}

// Both outputs with the gradients of q, k and the weights.  The backward pass runs without the interpreter's lock, so its errors
// are C++ exceptions of torch's engine.
struct QkNormRope : torch::autograd::Function<QkNormRope> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& q, const Tensor& k,
                                                const std::optional<Tensor>& qw_, const std::optional<Tensor>& kw_, const Tensor& pos,
                                                const Tensor& table, const std::optional<Tensor>& plan_, double eps, int64_t layout) {
    const Tensor qw = qw_.value_or(Tensor()), kw = kw_.value_or(Tensor()), plan = plan_.value_or(Tensor());
    ctx->save_for_backward({q, k, qw, kw, pos, table, plan});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["layout"] = layout;
    const bool all = !plan.defined();
    const Tensor q_out = new_rows(q, all), k_out = new_rows(k, all);
    check(launch_qk_norm_rope(q, k, qw, kw, pos, table, plan, static_cast<float>(eps), static_cast<int>(layout), q_out, k_out));
    return {q_out, k_out};
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &q = saved[0], &k = saved[1], &qw = saved[2], &kw = saved[3], &pos = saved[4], &table = saved[5], &plan = saved[6];
    auto dense = [](const Tensor& g) { return g.stride(2) == 1 || g.size(2) == 1 ? g : g.contiguous(); };
    const Tensor gq = dense(grads[0]), gk = dense(grads[1]);
    const bool all = !plan.defined();
    const int T = static_cast<int>(q.size(0)), H = static_cast<int>(q.size(1)), HK = static_cast<int>(k.size(1)), D = static_cast<int>(q.size(2));
    Tensor dq, dk, dqw, dkw, ws;
    if (ctx->needs_input_grad(0)) dq = new_rows(q, all);
    if (ctx->needs_input_grad(1)) dk = new_rows(k, all);
    // (weights that are not there are no edges of the graph)
    if (qw.defined() && ctx->needs_input_grad(2)) dqw = at::empty(qw.sizes(), qw.options());
    if (kw.defined() && ctx->needs_input_grad(qw.defined() ? 3 : 2)) dkw = at::empty(kw.sizes(), kw.options());
    int64_t bytes = 0;
    int rc = SPECQ_OK;
    if (dqw.defined() || dkw.defined()) rc = lib.qk_norm_rope_grad_workspace(T, H, HK, D, &bytes);
    // from torch's allocator on the current stream, as the attention's
    if (rc == SPECQ_OK && bytes > 0) ws = at::empty({bytes}, q.options().dtype(at::kByte));
    const int f32 = (qw.defined() && qw.scalar_type() == at::kFloat) || (kw.defined() && kw.scalar_type() == at::kFloat);
    if (rc == SPECQ_OK)
      rc = lib.qk_norm_rope_grad(q.data_ptr(), q.stride(0), q.stride(1), gq.data_ptr(), gq.stride(0), gq.stride(1), raw(dq), stride_of(dq, 0),
                                 stride_of(dq, 1), k.data_ptr(), k.stride(0), k.stride(1), gk.data_ptr(), gk.stride(0), gk.stride(1), raw(dk),
                                 stride_of(dk, 0), stride_of(dk, 1), row_code(q), raw(qw), raw(kw), raw(dqw), raw(dkw), f32,
                                 static_cast<float>(ctx->saved_data["eps"].toDouble()), ptr<int32_t>(pos), ptr<float>(table),
                                 static_cast<int>(table.size(0)), T, H, HK, D, static_cast<int>(table.size(1)),
                                 static_cast<int>(ctx->saved_data["layout"].toInt()), static_cast<const int32_t*>(raw(plan)), raw(ws), bytes,
                                 stream());
    if (rc != SPECQ_OK) throw std::runtime_error(std::string("libspecq: ") + lib.last_error());
    torch::autograd::variable_list out = {dq, dk, dqw, dkw};
    if (c10::GradMode::is_enabled()) {     // the gradients are no graph of their own: differentiating them is an error, not a zero
      for (Tensor& t : out)
        if (t.defined()) t.set_requires_grad(true);
      auto stop = std::make_shared<torch::autograd::DelayedError>("qk_norm_rope is differentiable once", 4);
      out = (*stop)(std::move(out));
    }
    out.resize(9);
    return out;
  }
};

// Whether two [T, H, D] tensors of one type share no memory: apart altogether, or columns of one buffer by rows or by heads.
bool apart(const Tensor& a, const Tensor& b) {
  if (a.numel() == 0 || b.numel() == 0) return true;
  const int64_t es = a.element_size();
  auto head = [&](const Tensor& t) { return (t.size(1) - 1) * t.stride(1) + t.size(2); };
  auto span = [&](const Tensor& t) { return (t.size(0) - 1) * t.stride(0) + head(t); };
  const int64_t lo = (static_cast<char*>(a.data_ptr()) - static_cast<char*>(b.data_ptr())) / es;
  if (lo >= span(b) || -lo >= span(a)) return true;
  auto beside = [&](int64_t stride, int64_t in_a, int64_t in_b) {
    if (stride <= 0) return false;
    const int64_t off = ((lo % stride) + stride) % stride;
    return off >= in_b && off + in_a <= stride;
  };
  const int64_t s0 = a.stride(0), s1 = a.stride(1);
  if (s0 != b.stride(0)) return false;
  return beside(s0, head(a), head(b)) || (s1 == b.stride(1) && s1 > 0 && s0 % s1 == 0 && beside(s1, a.size(2), b.size(2)));
}

// The same elements in the same places.
bool same_place(const Tensor& a, const Tensor& b) {
  return a.data_ptr() == b.data_ptr() && (a.size(0) < 2 || a.stride(0) == b.stride(0)) && (a.size(1) < 2 || a.stride(1) == b.stride(1));
}

PyObject* qk_norm_rope(PyObject* const* a) {
  // q, k, q_weight, k_weight, pos, table, eps, layout, q_out, k_out, plan
  const char* who = "qk_norm_rope";
  const Heads x = heads(who, a[0], a[1], a[2], a[3], a[4], a[5], a[6], a[7], a[10]);
  const Tensor *q_given = optional(who, "q_out", a[8]), *k_given = optional(who, "k_out", a[9]);
  auto out_like = [&](const char* what, const Tensor* out, const Tensor& in) {
    if (out == nullptr) return;
    rows3(who, what, *out, true);
    if (out->scalar_type() != in.scalar_type() || out->sizes() != in.sizes())
      BAD_VALUE("%s: %s must be %s %s, got %s %s", who, what, dtype(in), shape(in).c_str(), dtype(*out), shape(*out).c_str());
    written(who, what, *out);
  };
  out_like("q_out", q_given, x.q);
  out_like("k_out", k_given, x.k);
  for (int64_t n : {x.q.size(0), x.q.size(1), x.k.size(1), x.q.size(2), x.table.size(0)}) size32(who, n);
  no_tangent(who, {&x.q, &x.k, x.qw, x.kw, &x.table, q_given, k_given});
  bool needs = false;
  if (c10::GradMode::is_enabled()) {
    needs = x.q.requires_grad() || x.k.requires_grad() || (x.qw != nullptr && x.qw->requires_grad()) ||
            (x.kw != nullptr && x.kw->requires_grad());
    if ((q_given != nullptr || k_given != nullptr) &&
        (needs || (q_given != nullptr && q_given->requires_grad()) || (k_given != nullptr && k_given->requires_grad())))
      BAD_VALUE("%s: no q_out or k_out where a gradient is wanted", who);
    if (x.table.requires_grad()) BAD_VALUE("%s: the table has no gradient", who);
  }
  if (q_given != nullptr && ((!same_place(*q_given, x.q) && !apart(*q_given, x.q)) || !apart(*q_given, x.k)))
    BAD_VALUE("%s: q_out may be q, and else shares no memory with q and k", who);
  if (k_given != nullptr && ((!same_place(*k_given, x.k) && !apart(*k_given, x.k)) || !apart(*k_given, x.q)))
    BAD_VALUE("%s: k_out may be k, and else shares no memory with q and k", who);
  if (q_given != nullptr && k_given != nullptr && !apart(*q_given, *k_given)) BAD_VALUE("%s: q_out and k_out share memory", who);
  same_device(who, {&x.q, &x.k, &x.pos, &x.table, x.qw, x.kw, q_given, k_given, x.plan});
  const Tensor qw = or_none(x.qw), kw = or_none(x.kw), plan = or_none(x.plan);
  if (needs) {
    const auto out = QkNormRope::apply(x.q, x.k, maybe(x.qw), maybe(x.kw), x.pos, x.table, maybe(x.plan), static_cast<double>(x.eps),
                                       static_cast<int64_t>(x.layout));
    return pack({out[0], out[1]});
  }
  const bool all = x.plan == nullptr;
  const Tensor q_out = q_given != nullptr ? *q_given : new_rows(x.q, all), k_out = k_given != nullptr ? *k_given : new_rows(x.k, all);
  check(launch_qk_norm_rope(x.q, x.k, qw, kw, x.pos, x.table, plan, x.eps, x.layout, q_out, k_out));
  wrote({q_given, k_given});
  return pack({q_out, k_out});
}

// ---- beams ------------------------------------------------------------------------------------------
PyObject* beam_select(PyObject* const* a) {
  // logits, scores, n, done, pad, beams
  const char* who = "beam_select";
  const Tensor &x = tensor(who, "logits", a[0]), &scores = tensor(who, "scores", a[1]);
  if (row_code(x) < 0) BAD_TYPE("%s: logits must be float16, bfloat16 or float32, got %s", who, dtype(x));
  if (x.dim() != 2 || (x.size(1) > 1 && x.stride(1) != 1)) BAD_VALUE("%s: logits must be [rows, vocabulary] with unit inner stride, got %s", who, shape(x).c_str());
  if (scores.scalar_type() != at::kFloat || scores.numel() != x.size(0) || !scores.is_contiguous() || scores.dim() > 2)
    BAD_VALUE("%s: scores must be contiguous float32 [requests, beams] of %lld rows, got %s %s", who, (long long)x.size(0), dtype(scores),
              shape(scores).c_str());
  if (a[5] == Py_None && scores.dim() != 2) BAD_VALUE("%s: give beams, or scores as [requests, beams]", who);
  const int K = a[5] == Py_None ? size32(who, scores.size(1)) : integer(a[5]);
  if (K < 1 || x.size(0) % K || (scores.dim() == 2 && scores.size(1) != K)) BAD_VALUE("%s: %lld rows of scores %s are no requests of %d beams", who, (long long)x.size(0), shape(scores).c_str(), K);
  const int n = integer_or(a[2], K), pad = integer(a[4]), V = size32(who, x.size(1)), B = size32(who, x.size(0) / K);
  if (n < 1 || V < 1) BAD_VALUE("%s: n=%d of a vocabulary of %d", who, n, V);
  if (x.size(0) > 1 && x.stride(0) < V) BAD_VALUE("%s: logits' rows overlap (stride %lld of %d tokens); give each beam its row", who, (long long)x.stride(0), V);
  const Tensor* done = optional(who, "done", a[3]);
  if (done != nullptr && ((done->scalar_type() != at::kBool && done->scalar_type() != at::kByte) || done->numel() != x.size(0) || !done->is_contiguous()))
    BAD_VALUE("%s: done must be a contiguous bool of %lld rows, got %s %s", who, (long long)x.size(0), dtype(*done), shape(*done).c_str());
  if (pad < 0 || pad >= V) BAD_VALUE("%s: pad=%d is no token of %d", who, pad, V);
  if (c10::GradMode::is_enabled() && (x.requires_grad() || scores.requires_grad())) BAD_VALUE("%s: no gradient; detach logits and scores", who);
  no_tangent(who, {&x, &scores});
  same_device(who, {&x, &scores, done});
  const Tensor out = at::empty({B, n}, scores.options()), parent = at::empty({B, n}, scores.options().dtype(at::kInt)),
               token = at::empty({B, n}, scores.options().dtype(at::kInt));
  int64_t bytes = 0;
  check(lib.beam_select_workspace(B, K, V, n, row_code(x), &bytes));
  Tensor ws;
  if (bytes > 0) ws = at::empty({bytes}, x.options().dtype(at::kByte));
  check(lib.beam_select(x.data_ptr(), x.size(0) > 1 ? x.stride(0) : V, row_code(x), ptr<float>(scores), ptr<uint8_t>(done), pad, ptr<float>(out),
                        ptr<int32_t>(parent), ptr<int32_t>(token), B, K, V, n, bytes > 0 ? ws.data_ptr() : nullptr, bytes, stream()));
  return pack({out, parent, token});
}

PyObject* beam_reorder(PyObject* const* a) {
  // states, parent, beams
  const char* who = "beam_reorder";
  if (!PyList_Check(a[0]) && !PyTuple_Check(a[0])) BAD_TYPE("%s: states must be a list or a tuple of tensors", who);
  const Tensor& parent = tensor(who, "parent", a[1]);
  if (parent.scalar_type() != at::kInt || !parent.is_contiguous() || parent.dim() < 1 || parent.dim() > 2)
    BAD_VALUE("%s: parent must be contiguous int32 [rows] or [requests, beams], got %s %s", who, dtype(parent), shape(parent).c_str());
  const int K = a[2] == Py_None && parent.dim() == 2 ? size32(who, parent.size(1)) : a[2] == Py_None ? 0 : integer(a[2]);
  const int64_t R = parent.numel();
  if (K < 1 || R % K) BAD_VALUE("%s: %lld rows are no requests of %d beams (give beams, or parent as [requests, beams])", who, (long long)R, K);
  const Py_ssize_t count = PySequence_Fast_GET_SIZE(a[0]);
  PyObject** items = PySequence_Fast_ITEMS(a[0]);
  std::vector<void*> at_(count);
  std::vector<int64_t> stride(count), bytes(count);
  for (Py_ssize_t i = 0; i < count; ++i) {
    const Tensor& t = tensor(who, "a state", items[i]);
    if (t.dim() < 1 || t.size(0) != R) BAD_VALUE("%s: state %zd is %s for %lld rows", who, i, shape(t).c_str(), (long long)R);
    int64_t inner = 1;                                   // a row is one run of memory
    for (int64_t d = t.dim() - 1; d > 0; --d) {
      if (t.size(d) > 1 && t.stride(d) != inner) BAD_VALUE("%s: state %zd's rows must be contiguous, strides of %s", who, i, shape(t).c_str());
      inner *= t.size(d);
    }
    if (R > 1 && inner > 0 && t.stride(0) < inner) BAD_VALUE("%s: state %zd is written and its rows must not share memory", who, i);
    if (c10::GradMode::is_enabled() && t.requires_grad()) BAD_VALUE("%s: state %zd requires grad; it is written in place", who, i);
    no_tangent(who, {&t});
    at_[i] = t.data_ptr();
    stride[i] = t.stride(0) * t.element_size();
    bytes[i] = inner * t.element_size();
    const char *lo_ = static_cast<char*>(at_[i]), *par = static_cast<char*>(parent.data_ptr());
    if (bytes[i] > 0 && lo_ < par + R * 4 && par < lo_ + (R - 1) * stride[i] + bytes[i])
      BAD_VALUE("%s: state %zd and parent share memory", who, i);
    for (Py_ssize_t j = 0; j < i && bytes[i] > 0; ++j) {     // columns of one buffer are two states, shared bytes are not
      if (bytes[j] == 0) continue;
      const int64_t lo = static_cast<char*>(at_[i]) - static_cast<char*>(at_[j]);
      const int64_t span_i = (R - 1) * stride[i] + bytes[i], span_j = (R - 1) * stride[j] + bytes[j];
      if (lo >= span_j || -lo >= span_i) continue;
      bool apart = false;
      if (stride[i] == stride[j] && R > 1) {
        const int64_t s = stride[i], off = ((lo % s) + s) % s;
        apart = off >= bytes[j] && off + bytes[i] <= s;
      }
      if (!apart) BAD_VALUE("%s: states %zd and %zd share memory", who, j, i);
    }
  }
  for (Py_ssize_t i = 0; i < count; ++i) same_device(who, {&parent, &THPVariable_Unpack(items[i])});
  same_device(who, {&parent});
  check(lib.beam_reorder(at_.data(), stride.data(), bytes.data(), size32(who, count), ptr<int32_t>(parent), size32(who, R / K), K, stream()));
  for (Py_ssize_t i = 0; i < count; ++i) wrote({&THPVariable_Unpack(items[i])});
  return none();
}

// ---- a bounded cache --------------------------------------------------------------------------------
// mass: float32, one run of at least `tokens` for each sequence and KV head (and layer)
void mass_of(const char* who, const Tensor& m, bool layers, int64_t L, int64_t B, int64_t H, int64_t tokens) {
  const int d = layers ? 1 : 0;
  if (m.scalar_type() != at::kFloat) BAD_TYPE("%s: mass must be float32, got %s", who, dtype(m));
  if (m.dim() != 3 + d || (d && m.size(0) != L) || m.size(d) < B || m.size(d + 1) != H || m.size(d + 2) < tokens)
    BAD_VALUE("%s: mass must be [%s%lld, %lld, >= %lld], got %s", who, d ? (std::to_string(L) + ", ").c_str() : "", (long long)B, (long long)H,
              (long long)tokens, shape(m).c_str());
  if (m.size(d + 2) > 1 && m.stride(d + 2) != 1) BAD_VALUE("%s: mass needs unit stride along the tokens", who);
  written(who, "mass", m);
  if (c10::GradMode::is_enabled() && m.requires_grad()) BAD_VALUE("%s: mass requires grad; it is written in place", who);
  no_tangent(who, {&m});
}

PyObject* attention_mass_blocks(PyObject* const* a) {
  // q, kc, ks, block_tbl, ctx_len, mass, q_len, n_rows, decay, sm_scale
  const char* who = "attention_mass_blocks";
  PyObject* const keys[4] = {a[1], a[1], a[2], a[2]};
  const Cache c = cache(who, keys, false, false);
  const Tensor& q = tensor(who, "q", a[0]);
  if (q.scalar_type() != at::kHalf && q.scalar_type() != at::kBFloat16)
    BAD_TYPE("%s: q must be float16 or bfloat16, got %s", who, dtype(q));
  const Tensor &tbl = tensor(who, "block_tbl", a[3]), &ctx = tensor(who, "ctx_len", a[4]), &mass = tensor(who, "mass", a[5]);
  int32s(who, "block_tbl", tbl, 2, -1);
  int32s(who, "ctx_len", ctx, 1, tbl.size(0));
  const int B = size32(who, tbl.size(0)), cols = size32(who, tbl.size(1));
  const bool packed = q.dim() == 3;
  if (packed ? a[6] == Py_None : q.dim() != 4) {
    if (packed) BAD_VALUE("%s: packed queries need q_len", who);
    BAD_VALUE("%s: q must have 3 or 4 dimensions, got %s", who, shape(q).c_str());
  }
  const int q_len = packed ? integer(a[6]) : integer_or(a[6], size32(who, q.size(1)));
  if (q_len < 0 || (packed ? q.size(0) < static_cast<int64_t>(B) * q_len : q.size(0) < B || q.size(1) < q_len))
    BAD_VALUE("%s: q is %s for %d sequences of %d tokens", who, shape(q).c_str(), B, q_len);
  if (!packed && q.stride(0) == 0 && B > 1) BAD_VALUE("%s: q is expanded over the sequences (its stride is 0); give each sequence its rows", who);
  const int64_t H = q.size(-2);
  if (q.size(-1) != c.D || c.H == 0 || H < 1 || H % c.H)
    BAD_VALUE("%s: q heads (%lld, %lld) do not fit the cache's (%lld, %lld)", who, (long long)H, (long long)q.size(-1), (long long)c.H, (long long)c.D);
  if (q.stride(-1) != 1) BAD_VALUE("%s: q needs unit stride along D", who);
  const Tensor* n_rows = optional(who, "n_rows", a[7]);
  if (n_rows != nullptr) int32s(who, "n_rows", *n_rows, 1, B);
  mass_of(who, mass, false, 1, B, c.H, static_cast<int64_t>(cols) * c.page);
  const double decay = PyFloat_AsDouble(a[8]);
  if (decay == -1.0 && PyErr_Occurred()) throw Raised{};
  if (!(decay >= 0 && decay <= 1)) BAD_VALUE("%s: decay=%g must be in 0..1", who, decay);
  float sm = 1.f / std::sqrt(static_cast<float>(c.D));
  if (a[9] != Py_None) {
    const double v = PyFloat_AsDouble(a[9]);
    if (v == -1.0 && PyErr_Occurred()) throw Raised{};
    if (!(v > 0) || !(v < 2e38)) BAD_VALUE("%s: sm_scale=%g must be positive and finite", who, v);
    sm = static_cast<float>(v);
  }
  same_device(who, {&c.kc, &c.ks, &q, &tbl, &ctx, n_rows, &mass});
  const int h = size32(who, H), hk = size32(who, c.H), D = size32(who, c.D), page = size32(who, c.page);
  int64_t bytes = 0;
  check(lib.attention_mass_workspace(B, q_len, h, hk, D, page, cols, &bytes));
  Tensor ws;
  if (bytes > 0) ws = at::empty({bytes}, q.options().dtype(at::kByte));
  const int o = packed ? 0 : 1;
  // to the kernels a batch stride of 0 says packed rows; one sequence is one either way
  check(lib.attention_mass(q.data_ptr(), packed ? 0 : q.stride(0), q.stride(o), q.stride(o + 1), row_code(q), c.kc.data_ptr(), c.kc.stride(0),
                           c.kc.stride(1), c.kc.stride(2), cache_code(c.kc), size32(who, c.P), ptr<float>(c.ks), c.ks.stride(0), c.ks.stride(1),
                           ptr<int32_t>(tbl), tbl.stride(0), cols, ptr<int32_t>(ctx), ptr<int32_t>(n_rows), sm, static_cast<float>(decay),
                           ptr<float>(mass), mass.stride(0), mass.stride(1), B, q_len, h, hk, D, page, bytes > 0 ? ws.data_ptr() : nullptr, bytes,
                           stream()));
  wrote({&mass});
  Py_INCREF(a[5]);
  return a[5];
}

PyObject* kv_evict_blocks(PyObject* const* a) {
  // kc, vc, ks, vs, block_tbl, ctx_len, mass, keep, recent, ref, ctx_out
  const char* who = "kv_evict_blocks";
  const Cache c = cache(who, a, true);
  const Tensor &tbl = tensor(who, "block_tbl", a[4]), &ctx = tensor(who, "ctx_len", a[5]), &mass = tensor(who, "mass", a[6]);
  int32s(who, "block_tbl", tbl, 2, -1);
  const int64_t B = tbl.size(0);
  int32s(who, "ctx_len", ctx, 1, B);
  if (c.L == 0) BAD_VALUE("%s: a cache without layers", who);
  // K and V are moved side by side
  if ((c.kc.numel() > 0 && c.kc.data_ptr() == c.vc.data_ptr()) || (c.ks.numel() > 0 && c.ks.data_ptr() == c.vs.data_ptr()))
    BAD_VALUE("%s: kc and vc, and ks and vs, must not be the same memory", who);
  int keep = integer(a[7]), recent = integer(a[8]);
  if (keep < 1 || recent < 0 || recent > keep) BAD_VALUE("%s: keep=%d, of these the newest recent=%d", who, keep, recent);
  // more than the table has room for: no row has as many, and none needs a place for them
  keep = static_cast<int>(std::min<int64_t>(keep, std::max<int64_t>(1, tbl.size(1) * c.page)));
  recent = std::min(recent, keep);
  mass_of(who, mass, c.d != 0, c.L, B, c.H, tbl.size(1) * c.page);
  const Tensor *ref = optional(who, "ref", a[9]), *given = optional(who, "ctx_out", a[10]);
  if (ref != nullptr) int32s(who, "ref", *ref, 1, c.P);
  if (given != nullptr) int32s(who, "ctx_out", *given, 1, B);
  same_device(who, {&c.kc, &c.vc, &c.ks, &c.vs, &tbl, &ctx, &mass, ref, given});
  const Tensor out = given != nullptr ? *given : new_int32(ctx, B);
  const int L = size32(who, c.L), b = size32(who, B), h = size32(who, c.H), d = c.d;
  if (b == 0 || h == 0) return wrap(out);
  int64_t bytes = 0;
  check(lib.block_evict_workspace(L, b, h, keep, &bytes));
  const Tensor ws = at::empty({bytes}, c.kc.options().dtype(at::kByte));
  check(lib.block_evict(c.kc.data_ptr(), c.vc.data_ptr(), c.sl(), c.kc.stride(d), c.kc.stride(d + 1), c.kc.stride(d + 2), cache_code(c.kc), L,
                        size32(who, c.P), ptr<float>(c.ks), ptr<float>(c.vs), c.s_sl(), c.ks.stride(d), c.ks.stride(d + 1), ptr<int32_t>(tbl),
                        tbl.stride(0), size32(who, tbl.size(1)), ptr<int32_t>(ctx), ptr<int32_t>(ref), ptr<float>(mass), d ? mass.stride(0) : 0,
                        mass.stride(d), mass.stride(d + 1), keep, recent, ptr<int32_t>(out), b, h, size32(who, c.D), size32(who, c.page),
                        ws.data_ptr(), bytes, stream()));
  wrote({&c.kc, &c.vc, &c.ks, &c.vs, &mass, given});
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
      {"specq_pages_trim", reinterpret_cast<void**>(&t.pages_trim)},
      {"specq_qk_norm_rope", reinterpret_cast<void**>(&t.qk_norm_rope)},
      {"specq_qk_norm_rope_grad", reinterpret_cast<void**>(&t.qk_norm_rope_grad)},
      {"specq_qk_norm_rope_grad_workspace", reinterpret_cast<void**>(&t.qk_norm_rope_grad_workspace)},
      {"specq_beam_select", reinterpret_cast<void**>(&t.beam_select)},
      {"specq_beam_select_workspace", reinterpret_cast<void**>(&t.beam_select_workspace)},
      {"specq_beam_reorder", reinterpret_cast<void**>(&t.beam_reorder)},
      {"specq_attention_mass", reinterpret_cast<void**>(&t.attention_mass)},
      {"specq_attention_mass_workspace", reinterpret_cast<void**>(&t.attention_mass_workspace)},
      {"specq_block_evict", reinterpret_cast<void**>(&t.block_evict)},
      {"specq_block_evict_workspace", reinterpret_cast<void**>(&t.block_evict_workspace)},
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
    {"qk_norm_rope", FAST((entry<qk_norm_rope, 11>)), nullptr},
    {"beam_select", FAST((entry<beam_select, 6>)), nullptr},
    {"beam_reorder", FAST((entry<beam_reorder, 3>)), nullptr},
    {"attention_mass_blocks", FAST((entry<attention_mass_blocks, 10>)), nullptr},
    {"kv_evict_blocks", FAST((entry<kv_evict_blocks, 11>)), nullptr},
    {"pages_release", FAST((entry<pages_release, 6>)), nullptr},
    {"pages_reserve", FAST((entry<pages_reserve, 6>)), nullptr},
    {"pages_fork", FAST((entry<pages_fork, 10>)), nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_native", "binding of the block-scaled cache's operators", -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__native(void) { return PyModule_Create(&module); }
