// CPython entry points that take torch tensors: the operators of a decode step
// beside the Linears (polylora_amd.paged, polylora_amd.logits).
//
// Their smallest calls take 4 us on the GPU, and checking ten tensor arguments
// from Python alone takes twice that.  Here a call is one look at each tensor,
// the output's allocation and the library's function.  Errors are Python's:
// ValueError and TypeError for arguments, RuntimeError for what the library
// refuses; no C++ exception leaves a function.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <exception>
#include <optional>
#include <string>

#include "../../include/polylora_hip.h"

namespace {

struct Refusal {
  PyObject* type;
  std::string what;
};
[[noreturn]] void value_error(const std::string& what) { throw Refusal{PyExc_ValueError, what}; }
[[noreturn]] void type_error(const std::string& what) { throw Refusal{PyExc_TypeError, what}; }
[[noreturn]] void runtime_error(const std::string& what) { throw Refusal{PyExc_RuntimeError, what}; }
// A Python error that is set already.
struct Raised {};

std::string shape_text(at::IntArrayRef s) {
  std::string r = "[";
  for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
  return r + "]";
}
std::string type_text(at::ScalarType t) {
  switch (t) {
    case at::kFloat:
      return "torch.float32";
    case at::kHalf:
      return "torch.float16";
    case at::kBFloat16:
      return "torch.bfloat16";
    case at::kInt:
      return "torch.int32";
    case at::kLong:
      return "torch.int64";
    case at::kFloat8_e4m3fn:
      return "torch.float8_e4m3fn";
    default:
      return std::string("of type ") + toString(t);
  }
}

// No argument may be part of a graph that wants derivatives: none of the calls has any.
void check_no_grad(const at::Tensor& t, const char* name) {
  if (t.requires_grad() && c10::GradMode::is_enabled())
    runtime_error(std::string(name) + " requires a gradient, and the call has no backward: call it under torch.no_grad()");
  if (t._fw_grad(0).defined() && c10::AutogradState::get_tls_state().get_fw_grad_mode())
    runtime_error(std::string(name) + " carries a tangent, and the call has no forward derivative");
}

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) type_error(std::string(name) + " must be a torch.Tensor");
  const at::Tensor& t = THPVariable_Unpack(o);
  check_no_grad(t, name);
  return t;
}
const at::Tensor* maybe(PyObject* o, const char* name) {
  return o == Py_None ? nullptr : &tensor(o, name);
}
int64_t integer(PyObject* o) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Raised{};
  return v;
}
double real(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Raised{};
  return v;
}

// The library's 32-bit sizes.
int32_t size32(int64_t n, const char* name) {
  if (n > INT32_MAX) value_error(std::string(name) + " has a size of " + std::to_string(n));
  return (int32_t)n;
}

int32_t dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat:
      return PL_F32;
    case at::kBFloat16:
      return PL_BF16;
    case at::kHalf:
      return PL_F16;
    default:
      type_error("polylora_amd kernels support float32, bfloat16 and float16, not " + type_text(t));
  }
}

// The tensor that sets the call's GPU is on one.
void check_lead(const at::Tensor& t, const char* what) {
  if (!t.is_cuda())
    runtime_error(std::string(what) +
                  ": polylora_amd computes only on a ROCm GPU through its HIP library; got a CPU "
                  "tensor (there is no CPU fallback)");
}
// Launches go to the current GPU: the tensor's, for as long as this lives.
class OnDevice {
 public:
  explicit OnDevice(const at::Tensor& t) {
    if (c10::impl::getDeviceGuardImpl(c10::DeviceType::CUDA)->getDevice() != t.device()) guard_.emplace(t.device());
  }

 private:
  std::optional<c10::DeviceGuard> guard_;
};

void check_type(const at::Tensor& t, const char* name, at::ScalarType type, int device) {
  if (t.scalar_type() != type)
    type_error(std::string(name) + " must be " + type_text(type) + ", not " + type_text(t.scalar_type()));
  if (!t.is_cuda() || t.get_device() != device)
    value_error(std::string(name) + " is not on the GPU of the other arguments");
}
void check_shape(const at::Tensor& t, const char* name, at::IntArrayRef want) {
  if (t.sizes() != want)
    value_error(std::string(name) + " must have shape " + shape_text(want) + ", not " + shape_text(t.sizes()));
}
void check_dense(const at::Tensor& t, const char* name) {
  if (!t.is_contiguous()) value_error(std::string(name) + " must be contiguous");
}
void check_last(const at::Tensor& t, const char* name) {
  if (t.numel() && t.size(-1) > 1 && t.stride(-1) != 1)
    value_error(std::string("the last dimension of ") + name + " must be contiguous");
}
// A contiguous int32 or fp32 vector of n elements; null where the tensor is.
template <typename E>
const E* vector(const at::Tensor* t, const char* name, at::ScalarType type, int device, int64_t n) {
  if (!t) return nullptr;
  check_type(*t, name, type, device);
  check_shape(*t, name, {n});
  check_dense(*t, name);
  return static_cast<const E*>(t->const_data_ptr());
}

void check_status(int rc, const char* what) {
  if (rc)
    runtime_error(std::string(what) + " failed (status " + std::to_string(rc) + "): " + pl_last_error());
}

// The cache arguments of both calls over a paged cache.  A written cache that
// shares its memory until then (a lazy clone) gets its own.
struct Cache {
  int32_t code, num_pages, page_size, kv_heads, max_pages;
  void *key, *value;
  const int64_t *key_strides, *value_strides;
  const int32_t* table;
  int64_t table_ld;
  const float *k_scale, *v_scale;
};

Cache check_cache(const at::Tensor& key, const at::Tensor& value, const at::Tensor& table, int64_t rows,
                  int64_t dim, at::ScalarType type, int device, const at::Tensor* k_scale,
                  const at::Tensor* v_scale, bool written) {
  if (key.dim() != 4 || key.sizes() != value.sizes())
    value_error("the caches must be [pages, kv_heads, page_size, head_dim], both alike, not " +
                shape_text(key.sizes()) + " and " + shape_text(value.sizes()));
  const int64_t kv_heads = key.size(1), page_size = key.size(2);
  if (key.size(3) != dim)
    value_error("the caches hold heads of " + std::to_string(key.size(3)) + " elements, not " +
                std::to_string(dim));
  Cache c;
  c.k_scale = c.v_scale = nullptr;
  if (key.scalar_type() == type) {
    c.code = dtype_code(type);
    if (k_scale || v_scale) value_error("scales belong to an 8-bit cache");
  } else if (key.scalar_type() == at::kFloat8_e4m3fn && type != at::kFloat) {
    c.code = PL_F8E4M3;
    if (!k_scale || !v_scale) value_error("an 8-bit cache needs k_scale and v_scale");
    c.k_scale = vector<float>(k_scale, "k_scale", at::kFloat, device, kv_heads);
    c.v_scale = vector<float>(v_scale, "v_scale", at::kFloat, device, kv_heads);
  } else {
    type_error("a cache holds the model's dtype (" + type_text(type) +
               ") or, for 16-bit models, torch.float8_e4m3fn, not " + type_text(key.scalar_type()));
  }
  if (value.scalar_type() != key.scalar_type())
    type_error("the caches must have one dtype, not " + type_text(key.scalar_type()) + " and " +
               type_text(value.scalar_type()));
  check_type(key, "key_cache", key.scalar_type(), device);
  check_type(value, "value_cache", key.scalar_type(), device);
  check_last(key, "the caches");
  check_last(value, "the caches");
  if (page_size < 16 || (page_size & (page_size - 1)))
    value_error("a page must hold a power of two of at least 16 tokens, not " + std::to_string(page_size));
  check_type(table, "page_table", at::kInt, device);
  if (table.dim() != 2 || table.size(0) != rows)
    value_error("page_table must be [" + std::to_string(rows) + ", pages], not " + shape_text(table.sizes()));
  check_last(table, "page_table");
  c.num_pages = size32(key.size(0), "the cache"), c.page_size = size32(page_size, "a page");
  c.kv_heads = size32(kv_heads, "the cache"), c.max_pages = size32(table.size(1), "page_table");
  c.key = written ? key.mutable_data_ptr() : const_cast<void*>(key.const_data_ptr());
  c.value = written ? value.mutable_data_ptr() : const_cast<void*>(value.const_data_ptr());
  c.key_strides = key.strides().data(), c.value_strides = value.strides().data();
  c.table = static_cast<const int32_t*>(table.const_data_ptr());
  // a table of one row or column may have any stride there
  c.table_ld = rows > 1 ? table.stride(0) : table.size(1);
  return c;
}

// (q, k, v, key_cache, value_cache, page_table, past_lens, cos, sin, seq_lens, interleaved, k_scale, v_scale,
//  k_out, stream) -> the rotated q
PyObject* rope_append(PyObject* const* a) {
  const at::Tensor &q = tensor(a[0], "q"), &k = tensor(a[1], "k"), &v = tensor(a[2], "v");
  const at::Tensor &cos = tensor(a[7], "cos"), &sin = tensor(a[8], "sin");
  const at::Tensor* k_out = maybe(a[13], "k_out");
  check_lead(q, "rope_append");
  const int device = q.get_device();
  const OnDevice current(q);
  if (q.dim() != 4 || k.dim() != 4 || q.size(0) != k.size(0) || q.size(1) != k.size(1) || q.size(3) != k.size(3))
    value_error("q and k must be [rows, M, heads, dim] and [rows, M, kv_heads, dim], not " +
                shape_text(q.sizes()) + " and " + shape_text(k.sizes()));
  const int64_t rows = q.size(0), m = q.size(1), heads = q.size(2), dim = q.size(3), kv_heads = k.size(2);
  const at::ScalarType type = q.scalar_type();
  const int32_t code = dtype_code(type);
  check_type(k, "k", type, device);
  check_type(v, "v", type, device);
  check_shape(v, "v", k.sizes());
  for (const at::Tensor* t : {&q, &k, &v}) check_last(*t, "q, k and v");
  const Cache c = check_cache(tensor(a[3], "key_cache"), tensor(a[4], "value_cache"), tensor(a[5], "page_table"),
                              rows, dim, type, device, maybe(a[11], "k_scale"), maybe(a[12], "v_scale"), true);
  if (c.kv_heads != kv_heads || kv_heads == 0 || heads % kv_heads)
    value_error(std::to_string(heads) + " heads and " + std::to_string(kv_heads) + " key heads over a cache of " +
                std::to_string(c.kv_heads));
  const int32_t* past = vector<int32_t>(&tensor(a[6], "past_lens"), "past_lens", at::kInt, device, rows);
  const int32_t* seq = vector<int32_t>(maybe(a[9], "seq_lens"), "seq_lens", at::kInt, device, rows);
  check_type(cos, "cos", at::kFloat, device);
  check_type(sin, "sin", at::kFloat, device);
  if (cos.dim() != 2) value_error("cos must be [positions, rot / 2], not " + shape_text(cos.sizes()));
  check_shape(sin, "sin", cos.sizes());
  check_dense(cos, "cos");
  check_dense(sin, "sin");
  const int64_t half = cos.size(1);
  if (2 * half > dim)
    value_error("cos and sin rotate " + std::to_string(2 * half) + " elements of heads of " + std::to_string(dim));
  if (k_out) {
    check_type(*k_out, "k_out", type, device);
    check_shape(*k_out, "k_out", k.sizes());
    check_dense(*k_out, "k_out");
  }
  const int interleaved = PyObject_IsTrue(a[10]);
  if (interleaved < 0) throw Raised{};
  void* stream = PyLong_AsVoidPtr(a[14]);
  const int32_t r32 = size32(rows, "q"), m32 = size32(m, "q"), h32 = size32(heads, "q"), d32 = size32(dim, "q");
  const int32_t p32 = size32(cos.size(0), "cos");
  at::Tensor out = at::empty(q.sizes(), q.options());
  int rc;
  Py_BEGIN_ALLOW_THREADS;
  rc = pl_rope_append(code, c.code, q.const_data_ptr(), q.strides().data(), k.const_data_ptr(), k.strides().data(),
                      v.const_data_ptr(), v.strides().data(), out.data_ptr(), k_out ? k_out->data_ptr() : nullptr,
                      c.key, c.key_strides, c.value, c.value_strides, c.num_pages, c.page_size, c.table, c.table_ld,
                      c.max_pages, past, seq, r32, m32, h32, c.kv_heads, d32,
                      static_cast<const float*>(cos.const_data_ptr()), static_cast<const float*>(sin.const_data_ptr()),
                      p32, (int32_t)(2 * half), interleaved, c.k_scale, c.v_scale, stream);
  Py_END_ALLOW_THREADS;
  check_status(rc, "pl_rope_append");
  return THPVariable_Wrap(std::move(out));
}

// (q, key_cache, value_cache, page_table, lens, scale, window, k_scale, v_scale, out, workspace, workspace_bytes,
//  counters, counter_ints, stream) -> out; scale and window may be None
PyObject* paged_attention(PyObject* const* a) {
  const at::Tensor& q = tensor(a[0], "q");
  check_lead(q, "paged_attention");
  const int device = q.get_device();
  const OnDevice current(q);
  if (q.dim() != 3) value_error("q must be [rows, heads, dim], not " + shape_text(q.sizes()));
  const int64_t rows = q.size(0), heads = q.size(1), dim = q.size(2);
  const at::ScalarType type = q.scalar_type();
  const int32_t code = dtype_code(type);
  check_last(q, "q");
  const Cache c = check_cache(tensor(a[1], "key_cache"), tensor(a[2], "value_cache"), tensor(a[3], "page_table"),
                              rows, dim, type, device, maybe(a[7], "k_scale"), maybe(a[8], "v_scale"), false);
  if (c.kv_heads == 0 || heads % c.kv_heads)
    value_error(std::to_string(heads) + " heads over a cache of " + std::to_string(c.kv_heads) + " key heads");
  const int32_t* lens = vector<int32_t>(&tensor(a[4], "lens"), "lens", at::kInt, device, rows);
  const double scale = a[5] == Py_None ? 1.0 / std::sqrt((double)dim) : real(a[5]);
  int64_t window = 0;
  if (a[6] != Py_None) {
    window = integer(a[6]);
    if (window < 1) value_error("window must be at least one token, not " + std::to_string(window));
    if (window > INT32_MAX) window = 0;  // no row is that long
  }
  const at::Tensor* given = maybe(a[9], "out");
  if (given) {
    check_type(*given, "out", type, device);
    check_shape(*given, "out", q.sizes());
    check_dense(*given, "out");
  }
  void *workspace = PyLong_AsVoidPtr(a[10]), *counters = PyLong_AsVoidPtr(a[12]), *stream = PyLong_AsVoidPtr(a[14]);
  const int64_t workspace_bytes = integer(a[11]), counter_ints = integer(a[13]);
  const int32_t r32 = size32(rows, "q"), h32 = size32(heads, "q"), d32 = size32(dim, "q");
  at::Tensor out = given ? *given : at::empty(q.sizes(), q.options());
  int rc;
  Py_BEGIN_ALLOW_THREADS;
  rc = pl_paged_attention(code, c.code, q.const_data_ptr(), q.strides().data(), c.key, c.key_strides, c.value,
                          c.value_strides, c.num_pages, c.page_size, c.table, c.table_ld, c.max_pages, lens, r32, h32,
                          c.kv_heads, d32, (float)scale, (int32_t)window, c.k_scale, c.v_scale, out.data_ptr(),
                          workspace, workspace_bytes, static_cast<int32_t*>(counters), counter_ints, stream);
  Py_END_ALLOW_THREADS;
  check_status(rc, "pl_paged_attention");
  if (given) return Py_NewRef(a[9]);
  return THPVariable_Wrap(std::move(out));
}

// A list per row [rows, n], or one [n] that all rows share (row stride 0).
struct List {
  const void* p = nullptr;
  int32_t n = 0;
  int64_t ld = 0;
};
List list(const at::Tensor& t, const char* name, at::ScalarType type, int device, int64_t rows) {
  check_type(t, name, type, device);
  if (t.dim() < 1 || t.dim() > 2 || (t.dim() == 2 && t.size(0) != rows))
    value_error(std::string(name) + " must be [" + std::to_string(rows) + ", n], or [n] for all rows, not " +
                shape_text(t.sizes()));
  check_last(t, name);
  // the stride of a single row says nothing
  return {t.const_data_ptr(), size32(t.size(-1), name), t.dim() == 2 && rows > 1 ? t.stride(0) : 0};
}

// (logits, tokens, lens, prompt_lens, repetition, presence, frequency, bias_ids, bias_values, allowed, out,
//  stream) -> out
PyObject* adjust_logits(PyObject* const* a) {
  const at::Tensor& logits = tensor(a[0], "logits");
  check_lead(logits, "adjust_logits");
  const int device = logits.get_device();
  const OnDevice current(logits);
  if (logits.dim() != 2) value_error("logits must be [rows, vocab], not " + shape_text(logits.sizes()));
  const int64_t rows = logits.size(0), vocab = logits.size(1);
  const at::ScalarType type = logits.scalar_type();
  const int32_t code = dtype_code(type);
  check_last(logits, "logits");
  const at::Tensor* given = maybe(a[10], "out");
  if (given) {
    if (given->scalar_type() != at::kFloat && given->scalar_type() != type)
      type_error("out must be torch.float32 or " + type_text(type) + ", not " + type_text(given->scalar_type()));
    check_type(*given, "out", given->scalar_type(), device);
    check_shape(*given, "out", logits.sizes());
    check_last(*given, "out");
  }
  const at::Tensor *tokens = maybe(a[1], "tokens"), *lens = maybe(a[2], "lens");
  const at::Tensor* prompt_lens = maybe(a[3], "prompt_lens");
  const at::Tensor *repetition = maybe(a[4], "repetition"), *presence = maybe(a[5], "presence");
  const at::Tensor* frequency = maybe(a[6], "frequency");
  List history;
  int32_t token_bytes = 0;
  if (!tokens) {
    if (lens || prompt_lens) value_error("lens and prompt_lens count tokens, which are missing");
    if (repetition || presence || frequency) value_error("penalties need the tokens they are for");
  } else {
    if (tokens->scalar_type() != at::kLong && tokens->scalar_type() != at::kInt)
      type_error("tokens must be torch.int64 or torch.int32, not " + type_text(tokens->scalar_type()));
    if (!lens) value_error("tokens need lens, the number of them in each row");
    history = list(*tokens, "tokens", tokens->scalar_type(), device, rows);
    token_bytes = (int32_t)tokens->element_size();
  }
  const int32_t* lens_p = vector<int32_t>(lens, "lens", at::kInt, device, rows);
  const int32_t* prompt_p = vector<int32_t>(prompt_lens, "prompt_lens", at::kInt, device, rows);
  const float* repetition_p = vector<float>(repetition, "repetition", at::kFloat, device, rows);
  const float* presence_p = vector<float>(presence, "presence", at::kFloat, device, rows);
  const float* frequency_p = vector<float>(frequency, "frequency", at::kFloat, device, rows);
  const at::Tensor *bias_ids = maybe(a[7], "bias_ids"), *bias_values = maybe(a[8], "bias_values");
  if (!bias_ids != !bias_values) value_error("bias_ids and bias_values go together");
  List ids, values;
  if (bias_ids) {
    ids = list(*bias_ids, "bias_ids", at::kInt, device, rows);
    values = list(*bias_values, "bias_values", at::kFloat, device, rows);
    if (ids.n != values.n || ids.ld != values.ld)
      value_error("bias_ids and bias_values must have one shape and row stride");
  }
  List masks;
  if (const at::Tensor* allowed = maybe(a[9], "allowed")) {
    masks = list(*allowed, "allowed", at::kInt, device, rows);
    if ((int64_t)masks.n * 32 < vocab)
      value_error("allowed has " + std::to_string(masks.n) + " words a row for a vocabulary of " +
                  std::to_string(vocab));
  }
  void* stream = PyLong_AsVoidPtr(a[11]);
  const int32_t r32 = size32(rows, "logits"), v32 = size32(vocab, "logits");
  at::Tensor out = given ? *given : at::empty(logits.sizes(), logits.options().dtype(at::kFloat));
  const int32_t out_code = dtype_code(out.scalar_type());
  int rc;
  Py_BEGIN_ALLOW_THREADS;
  rc = pl_adjust_logits(code, out_code, logits.const_data_ptr(), logits.stride(0), out.data_ptr(), out.stride(0), r32,
                        v32, history.p, token_bytes, history.ld, history.n, lens_p, prompt_p, repetition_p, presence_p,
                        frequency_p, static_cast<const int32_t*>(ids.p), static_cast<const float*>(values.p), ids.ld,
                        ids.n, static_cast<const int32_t*>(masks.p), masks.ld, stream);
  Py_END_ALLOW_THREADS;
  check_status(rc, "pl_adjust_logits");
  if (given) return Py_NewRef(a[10]);
  return THPVariable_Wrap(std::move(out));
}

// (stream) -> pl_stream_capture_id of it
PyObject* stream_capture_id(PyObject* const* a) {
  void* stream = PyLong_AsVoidPtr(a[0]);
  if (!stream && PyErr_Occurred()) throw Raised{};
  return PyLong_FromLongLong(pl_stream_capture_id(stream));
}

template <PyObject* (*Fn)(PyObject* const*), Py_ssize_t N>
PyObject* guarded(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "%zd arguments given, %zd taken", n, N);
    return nullptr;
  }
  try {
    return Fn(args);
  } catch (const Refusal& r) {
    PyErr_SetString(r.type, r.what.c_str());
  } catch (const Raised&) {
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
  }
  return nullptr;
}

template <PyObject* (*Fn)(PyObject* const*), Py_ssize_t N>
constexpr PyMethodDef method(const char* name) {
  return {name, (PyCFunction)(void (*)(void)) & guarded<Fn, N>, METH_FASTCALL, nullptr};
}

PyMethodDef methods[] = {method<rope_append, 15>("rope_append"), method<paged_attention, 15>("paged_attention"),
                         method<adjust_logits, 12>("adjust_logits"),
                         method<stream_capture_id, 1>("stream_capture_id"), {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensor_calls", nullptr, -1, methods,
                      nullptr,               nullptr,         nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensor_calls(void) { return PyModule_Create(&module); }
