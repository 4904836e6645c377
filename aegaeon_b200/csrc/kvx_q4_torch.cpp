// Python entry points of the 4-bit cache (aegaeon_b200.q4_cache).
//
// A decode turn calls write and attention once per layer, and the kernels of a
// small batch take a few microseconds: checking the tensors in Python and
// marshalling their arguments through ctypes took 9 us a call more.  This module does
// the checks on the C++ tensors, allocates the results and calls libkvx.so
// through the addresses that bind() was given, so both routes reach the same
// library instance.
//
// Refusals raise here (ValueError, TypeError); a status that the library
// returns goes back to the caller as an int, for aegaeon_b200._lib.check.
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <algorithm>
#include <cmath>
#include <string>

#include "../../include/kvx.h"

namespace {

decltype(&kvx_q4_write) g_write = nullptr;
decltype(&kvx_q4_read) g_read = nullptr;
decltype(&kvx_q4_attention) g_attention = nullptr;
decltype(&kvx_q4_attention_workspace) g_workspace = nullptr;

// A refusal: the Python exception and its message.
struct Refused {
  PyObject* type;
  std::string message;
};
[[noreturn]] void value_error(const std::string& m) { throw Refused{PyExc_ValueError, m}; }
[[noreturn]] void type_error(const std::string& m) { throw Refused{PyExc_TypeError, m}; }
#define REQUIRE(condition, message) \
  do {                              \
    if (!(condition)) value_error(message); \
  } while (0)

std::string shape(c10::IntArrayRef s) {
  std::string r = "[";
  for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
  return r + "]";
}

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) type_error(std::string(name) + " must be a tensor");
  const at::Tensor& t = THPVariable_Unpack(o);
  if (t.layout() != c10::kStrided) type_error(std::string(name) + " must be a dense tensor");
  if (t.requires_grad() && c10::GradMode::is_enabled())
    throw Refused{PyExc_RuntimeError, std::string(name) + " requires a gradient: the 4-bit "
                                      "cache's operators have none (detach it, or use no_grad)"};
  if (t._fw_grad(0).defined() && c10::AutogradState::get_tls_state().get_fw_grad_mode())
    throw Refused{PyExc_RuntimeError, std::string(name) + " carries a forward-mode gradient: the "
                                      "4-bit cache's operators have none"};
  return t;
}

int type_code(c10::ScalarType t) {
  return t == at::kBFloat16 ? KVX_DTYPE_BF16 : t == at::kHalf ? KVX_DTYPE_FP16
         : t == at::kFloat  ? KVX_DTYPE_FP32 : -1;
}

bool head_dim_ok(int64_t d) { return d == 64 || d == 128 || d == 256; }

struct CacheView {
  void *key, *value;
  int64_t stride, blocks, heads, block, dim;
  c10::Device device;
};

CacheView cache_of(const at::Tensor& k, const at::Tensor& v, int64_t dim) {
  REQUIRE(head_dim_ok(dim), "head_dim must be 64, 128 or 256, got " + std::to_string(dim));
  if (k.scalar_type() != at::kByte || v.scalar_type() != at::kByte)
    type_error("cache pages must be uint8 tensors");
  REQUIRE(k.dim() == 3 && v.sizes() == k.sizes(),
          "key and value pages must have one shape, [num_blocks, kv_heads, bytes]");
  REQUIRE(k.is_cuda() && v.device() == k.device(),
          "key and value pages must be on one CUDA device");
  const int64_t blocks = k.size(0), heads = k.size(1), size = k.size(2), token = dim / 2 + 4;
  REQUIRE(heads > 0 && size > 0 && size % (16 * token) == 0,
          std::to_string(size) + " bytes for each of " + std::to_string(heads) +
              " heads are no multiple of 16 tokens of " + std::to_string(token) +
              " bytes (head_dim " + std::to_string(dim) + ")");
  REQUIRE(k.stride(2) == 1 && v.stride(2) == 1 &&
              (heads == 1 || (k.stride(1) == size && v.stride(1) == size)),
          "the bytes of a page must be contiguous");
  REQUIRE(blocks <= 1 || k.stride(0) == v.stride(0),
          "key and value pages must have the same stride");
  return CacheView{k.data_ptr(), v.data_ptr(), blocks > 1 ? k.stride(0) : heads * size,
                   blocks, heads, size / token, dim, k.device()};
}

int check_rows(const at::Tensor& key, const at::Tensor& value, int64_t tokens,
               const CacheView& c) {
  const int kind = type_code(key.scalar_type());
  if (kind < 0 || value.scalar_type() != key.scalar_type())
    type_error("key and value must both be bfloat16, float16 or float32");
  const int64_t want[3] = {tokens, c.heads, c.dim};
  REQUIRE(key.sizes() == c10::IntArrayRef(want) && value.sizes() == key.sizes(),
          "key and value must be [tokens, kv_heads, head_dim] = " + shape(want) + ", got " +
              shape(key.sizes()) + " and " + shape(value.sizes()));
  REQUIRE(key.device() == c.device && value.device() == c.device,
          "key and value must be on the device of the cache");
  REQUIRE(key.stride(2) == 1 && value.stride(2) == 1, "the elements of a row must be contiguous");
  return kind;
}

// The bytes of a tensor: runs of `run` bytes at base + sums of multiples of the strides,
// largest stride first.  Neighbouring dimensions that lie like one are one.
struct Extent {
  static constexpr int kMost = 8;
  const char* base = nullptr;
  int64_t run = 0, span = 0;  // of one run; from the first byte to behind the last
  int dims = 0;
  int64_t size[kMost], stride[kMost];
  bool known = true;  // false: more dimensions than this can hold

  explicit Extent(const at::Tensor& t) {
    if (t.numel() == 0) return;
    base = static_cast<const char*>(t.const_data_ptr());
    run = t.element_size();
    std::pair<int64_t, int64_t> d[16];  // (stride, size)
    int n = 0;
    if (t.dim() > 16) known = false;
    for (int64_t i = 0; known && i < t.dim(); ++i)
      if (t.size(i) > 1) d[n++] = {t.stride(i) * t.element_size(), t.size(i)};
    std::sort(d, d + n);
    for (int i = 0; i < n; ++i) {
      if (dims == 0 && d[i].first == run) {
        run *= d[i].second;
      } else if (dims > 0 && d[i].first == stride[dims - 1] * size[dims - 1]) {
        size[dims - 1] *= d[i].second;
      } else if (dims == kMost) {
        known = false;
      } else {
        stride[dims] = d[i].first, size[dims] = d[i].second;
        ++dims;
      }
    }
    std::reverse(stride, stride + dims);
    std::reverse(size, size + dims);
    span = span_from(0);
  }
  int64_t span_from(int d) const {
    int64_t n = run;
    for (; d < dims; ++d) n += (size[d] - 1) * stride[d];
    return n;
  }
  // Whether no byte is in two of its runs, which is so where each stride passes
  // all that lies inside it.
  bool apart() const {
    for (int d = 0; d < dims; ++d)
      if (stride[d] < span_from(d + 1)) return false;
    return known;
  }
};

// Whether x from dimension dx on, at 0, and y from dy on, at `at`, share a byte.  Takes
// the larger of the two outermost strides (both at once where they are one) and
// follows those steps alone that bring the spans together.  After `left` steps the answer
// is yes: refusing such strides is better than racing.
bool meet(const Extent& x, int dx, const Extent& y, int dy, int64_t at, int* left) {
  const int64_t nx = x.span_from(dx), ny = y.span_from(dy);
  if (at >= nx || -at >= ny) return false;
  if ((dx == x.dims && dy == y.dims) || --*left < 0) return true;
  const int64_t sx = dx < x.dims ? x.stride[dx] : 0, sy = dy < y.dims ? y.stride[dy] : 0;
  const int64_t s = std::max(sx, sy);
  if (s == 0) return true;  // outermost dimensions that do not move
  const int ix = dx + (sx == s), iy = dy + (sy == s);
  // at + k s, k from -(steps of x) to the steps of y
  const int64_t low = sx == s ? -(x.size[dx] - 1) : 0, high = sy == s ? y.size[dy] - 1 : 0;
  const int64_t mx = x.span_from(ix), my = y.span_from(iy);
  // the steps with -my < at + k s < mx
  auto floor_div = [](int64_t a, int64_t b) { return a / b - (a % b < 0); };
  const int64_t first = std::max(low, floor_div(-my - at, s) + 1);
  const int64_t last = std::min(high, -floor_div(at - mx, s) - 1);
  for (int64_t k = first; k <= last; ++k) {
    if (meet(x, ix, y, iy, at + k * s, left)) return true;
    if (*left < 0) return true;
  }
  return false;
}

// First byte of a tensor and the one behind its last.
std::pair<const char*, const char*> range(const at::Tensor& t) {
  const char* base = static_cast<const char*>(t.const_data_ptr());
  if (t.numel() == 0) return {base, base};
  int64_t last = 0;
  for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
  return {base, base + (last + 1) * t.element_size()};
}

// Whether two tensors share bytes (yes, too, where their strides make it too long to tell).
bool overlap(const at::Tensor& a, const at::Tensor& b) {
  const auto ra = range(a), rb = range(b);  // of most pairs they tell
  if (ra.first == ra.second || rb.first == rb.second || ra.second <= rb.first ||
      rb.second <= ra.first)
    return false;
  const Extent x(a), y(b);
  if (!x.known || !y.known) return true;
  int left = 10000;
  return meet(x, 0, y, 0, y.base - x.base, &left);
}

// An output must have one place for each element and share none with the inputs.
void check_output(const at::Tensor& t, const char* name,
                  std::initializer_list<std::pair<const at::Tensor*, const char*>> others) {
  REQUIRE(t.is_non_overlapping_and_dense() || Extent(t).apart(),
          std::string("the elements of ") + name + " overlap one another");
  for (const auto& [other, what] : others)
    REQUIRE(!overlap(t, *other), std::string(name) + " must not overlap " + what);
}

int64_t check_slots(const at::Tensor& s, c10::Device device) {
  REQUIRE(s.scalar_type() == at::kLong && s.dim() == 1 && s.is_contiguous(),
          "slots must be a contiguous int64 tensor of one dimension");
  REQUIRE(s.device() == device, "slots must be on the device of the cache");
  return s.size(0);
}

// Tells autograd that a tensor was written to.  An inference tensor has no counter.
void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// Runs f with the device current and its current stream.
template <class F>
int on_device(c10::Device device, F f) {
  c10::cuda::OptionalCUDAGuard guard;
  if (c10::cuda::current_device() != device.index()) guard.set_device(device);
  void* stream = c10::cuda::getCurrentCUDAStream(device.index()).stream();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = f(stream);
  Py_END_ALLOW_THREADS
  return rc;
}

bool count(Py_ssize_t got, Py_ssize_t want, const char* name) {
  if (got != want) {
    PyErr_Format(PyExc_TypeError, "%s() takes %zd arguments", name, want);
    return false;
  }
  if (!g_write) {
    PyErr_SetString(PyExc_RuntimeError, "kvx q4 module used before bind()");
    return false;
  }
  return true;
}

int64_t integer(PyObject* o, const char* name) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    type_error(std::string(name) + " must be an integer");
  }
  return v;
}

#define BEGIN_CALL \
  HANDLE_TH_ERRORS \
  try {
#define END_CALL                                  \
  }                                               \
  catch (const Refused& r) {                      \
    PyErr_SetString(r.type, r.message.c_str());   \
    return nullptr;                               \
  }                                               \
  END_HANDLE_TH_ERRORS

// bind(write, read, attention, attention_workspace): addresses in libkvx.so
PyObject* py_bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 4) {
    PyErr_SetString(PyExc_TypeError, "bind() takes 4 function addresses");
    return nullptr;
  }
  void* p[4];
  for (int i = 0; i < 4; ++i) {
    p[i] = PyLong_AsVoidPtr(args[i]);
    if (!p[i]) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "null function address");
      return nullptr;
    }
  }
  g_read = reinterpret_cast<decltype(g_read)>(p[1]);
  g_attention = reinterpret_cast<decltype(g_attention)>(p[2]);
  g_workspace = reinterpret_cast<decltype(g_workspace)>(p[3]);
  g_write = reinterpret_cast<decltype(g_write)>(p[0]);
  Py_RETURN_NONE;
}

// write(key, value, key_pages, value_pages, slots) -> status
PyObject* py_write(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (!count(n, 5, "write")) return nullptr;
  BEGIN_CALL
  const at::Tensor &key = tensor(args[0], "key"), &value = tensor(args[1], "value");
  const at::Tensor &slots = tensor(args[4], "slots");
  REQUIRE(key.dim() == 3, "key must be [tokens, kv_heads, head_dim]");
  const CacheView c = cache_of(tensor(args[2], "key_pages"), tensor(args[3], "value_pages"),
                               key.size(2));
  const int64_t tokens = check_slots(slots, c.device);
  const int kind = check_rows(key, value, tokens, c);
  const at::Tensor &key_pages = THPVariable_Unpack(args[2]),
                   &value_pages = THPVariable_Unpack(args[3]);
  check_output(key_pages, "key pages to write to",
               {{&value_pages, "the value pages"}, {&key, "key"}, {&value, "value"},
                {&slots, "slots"}});
  check_output(value_pages, "value pages to write to",
               {{&key, "key"}, {&value, "value"}, {&slots, "slots"}});
  if (tokens == 0) return PyLong_FromLong(0);
  written(key_pages), written(value_pages);
  return PyLong_FromLong(on_device(c.device, [&](void* stream) {
    return g_write(key.data_ptr(), value.data_ptr(), kind, tokens, key.stride(0), key.stride(1),
                   value.stride(0), value.stride(1), slots.const_data_ptr<int64_t>(), c.key,
                   c.value, c.stride, c.blocks, c.heads, c.block, c.dim, stream);
  }));
  END_CALL
}

// read(key_pages, value_pages, slots, head_dim, dtype, key or None, value or None)
//   -> (status, key, value)
PyObject* py_read(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (!count(n, 7, "read")) return nullptr;
  BEGIN_CALL
  const at::Tensor& slots = tensor(args[2], "slots");
  const CacheView c = cache_of(tensor(args[0], "key_pages"), tensor(args[1], "value_pages"),
                               integer(args[3], "head_dim"));
  const int64_t tokens = check_slots(slots, c.device);
  at::Tensor key, value;
  if (args[5] == Py_None) {
    if (!THPDtype_Check(args[4])) type_error("dtype must be a torch dtype");
    const c10::ScalarType type = reinterpret_cast<THPDtype*>(args[4])->scalar_type;
    if (type_code(type) < 0) type_error("rows are read as bfloat16, float16 or float32");
    const int64_t size[3] = {tokens, c.heads, c.dim};
    const auto options = at::TensorOptions().dtype(type).device(c.device);
    key = at::empty(size, options);
    value = at::empty(size, options);
  } else {
    key = tensor(args[5], "out");
    value = tensor(args[6], "out");
  }
  const int kind = check_rows(key, value, tokens, c);
  if (args[5] != Py_None) {
    const at::Tensor &key_pages = THPVariable_Unpack(args[0]),
                     &value_pages = THPVariable_Unpack(args[1]);
    check_output(key, "the key rows of out",
                 {{&value, "its value rows"}, {&key_pages, "the key pages"},
                  {&value_pages, "the value pages"}, {&slots, "slots"}});
    check_output(value, "the value rows of out",
                 {{&key_pages, "the key pages"}, {&value_pages, "the value pages"},
                  {&slots, "slots"}});
    written(key), written(value);
  }
  int rc = 0;
  if (tokens)
    rc = on_device(c.device, [&](void* stream) {
      return g_read(c.key, c.value, c.stride, c.blocks, c.heads, c.block, c.dim,
                    slots.const_data_ptr<int64_t>(), tokens, key.data_ptr(), value.data_ptr(),
                    kind, key.stride(0), key.stride(1), value.stride(0), value.stride(1), stream);
    });
  return Py_BuildValue("(iNN)", rc, THPVariable_Wrap(key), THPVariable_Wrap(value));
  END_CALL
}

// attention(query, key_pages, value_pages, block_tables, seq_lens, query_starts or None,
//           scale or None, window or None, sinks, out or None, return_lse)
//   -> (status, out, lse or None)
PyObject* py_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (!count(n, 11, "attention")) return nullptr;
  BEGIN_CALL
  const at::Tensor& q = tensor(args[0], "query");
  const at::Tensor &tables = tensor(args[3], "block_tables"), &lens = tensor(args[4], "seq_lens");
  REQUIRE(q.dim() == 3, "query must be [tokens, heads, head_dim]");
  const int64_t tokens = q.size(0), heads = q.size(1);
  const CacheView c = cache_of(tensor(args[1], "key_pages"), tensor(args[2], "value_pages"),
                               q.size(2));
  const int kind = type_code(q.scalar_type());
  if (kind != KVX_DTYPE_BF16 && kind != KVX_DTYPE_FP16)
    type_error("query must be bfloat16 or float16");
  REQUIRE(heads > 0 && heads % c.heads == 0, std::to_string(heads) +
              " query heads are no multiple of " + std::to_string(c.heads) + " kv heads");
  REQUIRE(tables.scalar_type() == at::kInt && tables.dim() == 2,
          "block_tables must be an int32 tensor [batch, width]");
  REQUIRE(lens.scalar_type() == at::kInt && lens.dim() == 1 && lens.is_contiguous(),
          "seq_lens must be a contiguous int32 tensor [batch]");
  const int64_t batch = tables.size(0), width = tables.size(1);
  REQUIRE(lens.size(0) == batch, "block_tables has " + std::to_string(batch) +
              " sequences but seq_lens has " + std::to_string(lens.size(0)));
  REQUIRE(width <= 1 || tables.stride(1) == 1, "the entries of a block table must be contiguous");
  REQUIRE(q.stride(2) == 1, "the elements of a query row must be contiguous");
  REQUIRE(q.device() == c.device && tables.device() == c.device && lens.device() == c.device,
          "all tensors must be on the device of the cache");
  const int32_t* starts = nullptr;
  int64_t rows = tokens;  // query tokens of a sequence, at most
  if (args[5] == Py_None) {
    REQUIRE(tokens == 0 || (batch > 0 && tokens % batch == 0),
            std::to_string(tokens) + " query tokens cannot be shared by " +
                std::to_string(batch) + " sequences alike; pass query_starts");
    if (batch) rows = tokens / batch;
  } else {
    const at::Tensor& t = tensor(args[5], "query_starts");
    REQUIRE(t.scalar_type() == at::kInt && t.dim() == 1 && t.is_contiguous() &&
                t.size(0) == batch + 1,
            "query_starts must be a contiguous int32 tensor [batch + 1]");
    REQUIRE(t.device() == c.device, "all tensors must be on the device of the cache");
    starts = t.const_data_ptr<int32_t>();
  }
  double scale;
  if (args[6] == Py_None) {
    scale = 1.0 / std::sqrt(double(c.dim));
  } else {
    scale = PyFloat_AsDouble(args[6]);
    if (scale == -1.0 && PyErr_Occurred()) {
      PyErr_Clear();
      type_error("scale must be a number");
    }
    REQUIRE(std::isfinite(scale), "scale must be finite");
  }
  int64_t window = 0;
  if (args[7] != Py_None) {
    window = integer(args[7], "window");
    REQUIRE(window >= 1, "window must be at least 1 (None: no window)");
  }
  const int64_t sinks = integer(args[8], "sinks");
  REQUIRE(sinks >= 0, "sinks must not be negative");
  const auto options = q.options();
  at::Tensor out, lse;
  if (args[9] == Py_None) {
    out = at::empty(q.sizes(), options);
  } else {
    out = tensor(args[9], "out");
    REQUIRE(out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type() &&
                out.device() == c.device && out.stride(2) == 1,
            "out must have the shape, type and device of query and contiguous rows");
    // Other warps still read all of these when a first row is written.
    check_output(out, "out",
                 {{&q, "query"}, {&THPVariable_Unpack(args[1]), "the key pages"},
                  {&THPVariable_Unpack(args[2]), "the value pages"}, {&tables, "block_tables"},
                  {&lens, "seq_lens"}});
    if (args[5] != Py_None)
      check_output(out, "out", {{&THPVariable_Unpack(args[5]), "query_starts"}});
    written(out);
  }
  const int want_lse = PyObject_IsTrue(args[10]);
  if (want_lse < 0) return nullptr;
  if (want_lse) {
    const int64_t size[2] = {tokens, heads};
    lse = at::empty(size, options.dtype(at::kFloat));
  }
  int rc = 0;
  if (tokens && batch) {
    uint64_t bytes = 0;
    at::Tensor work;
    // The workspace is this call's own: the allocator keeps it from other
    // streams and graphs until the work queued here is done with it.
    {
      c10::cuda::OptionalCUDAGuard guard;
      if (c10::cuda::current_device() != c.device.index()) guard.set_device(c.device);
      rc = g_workspace(c.dim, rows * (heads / c.heads), &bytes);
    }
    if (rc == 0) {
      work = at::empty({int64_t(bytes)}, options.dtype(at::kByte));
      rc = on_device(c.device, [&](void* stream) {
        return g_attention(
            q.data_ptr(), q.stride(0), q.stride(1), out.data_ptr(), out.stride(0), out.stride(1),
            want_lse ? lse.data_ptr<float>() : nullptr, kind, tokens, heads, c.key, c.value,
            c.stride, c.blocks, c.heads, c.block, c.dim, tables.const_data_ptr<int32_t>(),
            tables.stride(0), width, lens.const_data_ptr<int32_t>(), starts, batch, scale, window,
            sinks, work.data_ptr(), bytes, stream);
      });
    }
  }
  if (want_lse)
    return Py_BuildValue("(iNN)", rc, THPVariable_Wrap(out), THPVariable_Wrap(lse));
  return Py_BuildValue("(iNO)", rc, THPVariable_Wrap(out), Py_None);
  END_CALL
}

// overlap(a, b): whether two tensors share memory, as the checks above see it
PyObject* py_overlap(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (!count(n, 2, "overlap")) return nullptr;
  BEGIN_CALL
  return PyBool_FromLong(overlap(tensor(args[0], "a"), tensor(args[1], "b")));
  END_CALL
}

#define METHOD(name, doc) \
  {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(py_##name)), \
   METH_FASTCALL, doc}
PyMethodDef kMethods[] = {
    METHOD(bind, "bind(write, read, attention, attention_workspace)"),
    METHOD(write, "kvx_q4_write on tensors; returns the status"),
    METHOD(read, "kvx_q4_read on tensors; returns (status, key, value)"),
    METHOD(overlap, "overlap(a, b): whether two tensors share memory"),
    METHOD(attention, "kvx_q4_attention on tensors; returns (status, out, lse)"),
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_kvxq4", "Tensor entry points of the 4-bit cache",
                       -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__kvxq4(void) { return PyModule_Create(&kModule); }
