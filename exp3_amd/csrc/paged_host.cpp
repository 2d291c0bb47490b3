// Host side of exp3_amd.paged, the extension module exp3_amd._C._paged: checks of the tensors,
// allocation of the outputs and the call of the C entry point. A decode step's kernels take 3 to
// 12 us; the same checks in Python and a ctypes call took 12 to 17 us of host time per call, these 6
// to 10.
//
// Functions take the tensors of a PagedCache one by one (None for the scales of a bf16 cache) and
// the raw stream of the current device; bad arguments raise ValueError.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <limits.h>
#include <stdarg.h>

#include <algorithm>
#include <sstream>
#include <stdexcept>
#include <utility>
#include <vector>

#include <ATen/TracerMode.h>
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/autograd/python_variable.h>

#include "sparse_prefill.h"

namespace {

constexpr int kScaleGroup = 32;          // dims per scale of a 4-bit page
constexpr int kTreeTokens = 256;         // nodes of a tree of drafted tokens

struct Invalid : std::runtime_error {
  using std::runtime_error::runtime_error;
};

template <typename... Parts>
[[noreturn]] void refuse(const Parts&... parts) {
  std::ostringstream text;
  (text << ... << parts);
  throw Invalid(text.str());
}

// Dispatch keys of tensors that are not what their storage holds: lazily zero ones, subclasses that
// compute by themselves, those of function transforms; and lazily negated ones.
constexpr c10::DispatchKeySet kNotPlain{
    c10::DispatchKey::ZeroTensor,       c10::DispatchKey::Python,
    c10::DispatchKey::Functionalize,    c10::DispatchKey::FuncTorchBatched,
    c10::DispatchKey::FuncTorchGradWrapper};
constexpr c10::DispatchKeySet kNegated{c10::DispatchKey::Negative};

const at::Tensor& tensor(PyObject* object, const char* name, bool may_be_negated = false) {
  if (!THPVariable_Check(object)) refuse(name, " must be a tensor, got ", Py_TYPE(object)->tp_name);
  const at::Tensor& x = THPVariable_Unpack(object);
  if (x.key_set().has_any(may_be_negated ? kNotPlain : kNotPlain | kNegated))
    refuse(name, " must be a plain tensor: the kernels read its storage (clone() makes one)");
  return x;
}

void* pointer(const at::Tensor& x) { return x.data_ptr(); }

void require_gpu(const at::Tensor& x) {
  if (!x.is_cuda())
    refuse("exp3_amd kernels run only on a ROCm GPU (MI355X); got a tensor on ", x.device());
}

void require_device(const at::Tensor& x, const c10::Device& device) {
  if (x.device() != device) refuse("tensors on different devices: ", device, " and ", x.device());
}

// No gradient would reach x, and no tangent of x the outputs.
void require_no_gradient(const at::Tensor& x, const char* name) {
  if (x.requires_grad() && c10::GradMode::is_enabled())
    refuse(name, " requires a gradient: the paged cache has no backward pass (torch.no_grad())");
  if (x._fw_grad(0).defined() && c10::AutogradState::get_tls_state().get_fw_grad_mode())
    refuse(name, " has a forward-mode tangent: the paged cache has no derivatives");
}

// Where torch records a graph, it records the allocation of the outputs and not the kernel that
// fills them. (Modes that only look on may be there.)
void require_eager() {
  using c10::impl::TorchDispatchModeKey;
  using c10::impl::TorchDispatchModeTLS;
  bool traced = at::tracer::impl::is_dispatch_enabled();
  if (!traced && TorchDispatchModeTLS::any_modes_set())
    for (auto key : {TorchDispatchModeKey::FAKE, TorchDispatchModeKey::PROXY,
                     TorchDispatchModeKey::FUNCTIONAL})
      traced = traced || TorchDispatchModeTLS::get_mode(key).has_value();
  if (traced) refuse("the paged cache's functions cannot be traced into a graph");
}

// x has been written in place: a backward pass that saved it has to find out. (Tensors made in
// inference mode have no version.)
void written(const at::Tensor& x) {
  if (!x.is_inference()) x.unsafeGetTensorImpl()->bump_version();
}

int small(int64_t x, const char* name) {
  if (x > INT_MAX) refuse(name, " of ", x, " is more than 2^31 - 1");
  return (int)x;
}

// Pages and page table of a call, as the C entry points take them; everything but the batch's
// sizes comes from the tensors.
struct Description {
  spx_paged_cache c{};
  c10::Device device;

  explicit Description(const c10::Device& d) : device(d) {}

  void pages(PyObject* const* args) {
    const at::Tensor& key = tensor(args[0], "key_pages");
    const at::Tensor& value = tensor(args[1], "value_pages");
    const bool four = args[2] != Py_None;
    if (four != (args[3] != Py_None))
      refuse("a 4-bit cache needs key_scales and value_scales, a bf16 cache neither");
    const auto type = four ? at::kByte : at::kBFloat16;
    if (key.dim() != 4 || value.sizes() != key.sizes() || key.scalar_type() != type ||
        value.scalar_type() != type || !key.is_contiguous() || !value.is_contiguous())
      refuse("pages must be contiguous ", type, " [pages, Hkv, page_size, D", four ? " // 2" : "",
             "] tensors of one shape, got ", key.sizes(), " ", key.scalar_type(), " and ",
             value.sizes(), " ", value.scalar_type());
    require_device(key, device);
    require_device(value, device);
    require_no_gradient(key, "key_pages");
    require_no_gradient(value, "value_pages");
    c.key_pages = pointer(key);
    c.value_pages = pointer(value);
    c.pages = small(key.size(0), "pages");
    c.kv_heads = small(key.size(1), "KV heads");
    c.page_size = small(key.size(2), "page_size");
    c.head_dim = small(key.size(3) * (four ? 2 : 1), "head_dim");
    if (!four) return;
    void** to[2] = {&c.key_scales, &c.value_scales};
    for (int i = 0; i < 2; ++i) {
      const at::Tensor& x = tensor(args[2 + i], "scales");
      if (x.dim() != 4 || x.size(0) != c.pages || x.size(1) != c.kv_heads ||
          x.size(2) != c.page_size || x.size(3) != c.head_dim / kScaleGroup ||
          x.scalar_type() != at::kByte || !x.is_contiguous())
        refuse("scales must be contiguous uint8 [pages, Hkv, page_size, D // 32] tensors, got ",
               x.sizes(), " ", x.scalar_type());
      require_device(x, device);
      *to[i] = pointer(x);
    }
  }

  const int32_t* lengths(PyObject* object, const char* name) {
    const at::Tensor& x = tensor(object, name);
    if (x.dim() != 1 || x.size(0) != c.batch || x.scalar_type() != at::kInt || !x.is_contiguous())
      refuse(name, " must be a contiguous int32 [", c.batch, "] tensor, got ", x.sizes(), " ",
             x.scalar_type());
    require_device(x, device);
    return static_cast<const int32_t*>(pointer(x));
  }

  // args: page_table, starts, counts or None
  void map(PyObject* const* args, int64_t batch, int64_t tokens) {
    const at::Tensor& table = tensor(args[0], "page_table");
    c.batch = small(batch, "batch");
    c.tokens = small(tokens, "tokens");
    if (table.dim() != 2 || table.size(0) != batch || table.scalar_type() != at::kInt)
      refuse("page_table must be an int32 [", batch, ", pages per sequence] tensor, got ",
             table.sizes(), " ", table.scalar_type());
    if (table.size(1) > 1 && table.stride(1) != 1)
      refuse("page_table must have unit stride within a row");
    require_device(table, device);
    c.page_table = static_cast<const int32_t*>(pointer(table));
    c.table_stride = table.stride(0);
    c.table_width = small(table.size(1), "table width");
    c.starts = lengths(args[1], "starts");
    c.counts = args[2] == Py_None ? nullptr : lengths(args[2], "counts");
  }
};

// A [B, T, H, D] bf16 tensor that the kernels read in place: unit dim stride, 16-byte rows, no
// lazy negation; any other layout is copied.
at::Tensor rows(const at::Tensor& x, const char* name) {
  require_no_gradient(x, name);
  if (x.scalar_type() != at::kBFloat16)
    refuse("expected a bfloat16 tensor, got ", x.scalar_type(), " (", name, ")");
  if (x.dim() != 4)
    refuse("expected a [batch, sequence, heads, dim] tensor, got ", x.sizes(), " (", name, ")");
  const auto s = x.strides();
  if (!x.is_neg() && s[3] == 1 && ((s[0] | s[1] | s[2]) & 7) == 0 &&
      (reinterpret_cast<uintptr_t>(x.data_ptr()) & 15) == 0)
    return x;
  c10::AutoGradMode no_grad(false);
  return (x.is_neg() ? x.resolve_neg() : x).contiguous().detach();
}

// A contiguous copy where the tensor is not contiguous or lazily negated.
at::Tensor plain(const at::Tensor& x, const char* name) {
  require_no_gradient(x, name);
  if (!x.is_neg() && x.is_contiguous()) return x;
  c10::AutoGradMode no_grad(false);
  return (x.is_neg() ? x.resolve_neg() : x).contiguous().detach();
}

// Whether two contiguous tensors have bytes in common.
bool overlap(const at::Tensor& x, const at::Tensor& y) {
  const auto a = reinterpret_cast<uintptr_t>(x.data_ptr()), b = reinterpret_cast<uintptr_t>(y.data_ptr());
  return x.numel() > 0 && y.numel() > 0 && a < b + y.nbytes() && b < a + x.nbytes();
}

at::Tensor empty(at::IntArrayRef shape, at::ScalarType type, const c10::Device& device) {
  return at::empty(shape, at::TensorOptions().dtype(type).device(device));
}

void check(int status, const char* name) {
  if (status == SPX_OK) return;
  const std::string text = std::string(name) + ": " + spx_last_error();
  if (status == SPX_EINVAL || status == SPX_EUNSUPPORTED) throw Invalid(text);
  throw std::runtime_error(text);
}

int64_t integer(PyObject* object) {
  const long long x = PyLong_AsLongLong(object);
  if (x == -1 && PyErr_Occurred()) throw std::bad_exception();
  return x;
}

bool truth(PyObject* object) {
  const int x = PyObject_IsTrue(object);
  if (x < 0) throw std::bad_exception();
  return x != 0;
}

PyObject* wrap(const at::Tensor& x) {
  if (!x.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(x);
}

PyObject* pair(const at::Tensor& x, const at::Tensor& y) {
  PyObject* a = wrap(x);
  PyObject* b = wrap(y);
  PyObject* out = a && b ? PyTuple_Pack(2, a, b) : nullptr;
  Py_XDECREF(a);
  Py_XDECREF(b);
  return out;
}

// Calls `body`, turning C++ exceptions into Python's.
template <typename Body>
PyObject* guarded(Py_ssize_t got, Py_ssize_t wanted, const Body& body) {
  if (got != wanted) {
    PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", wanted, got);
    return nullptr;
  }
  try {
    require_eager();
    return body();
  } catch (const Invalid& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
  } catch (const c10::OutOfMemoryError& e) {
    PyObject* torch = PyImport_ImportModule("torch");
    PyObject* type = torch ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
    PyErr_SetString(type ? type : PyExc_RuntimeError, e.what_without_backtrace());
    Py_XDECREF(type);
    Py_XDECREF(torch);
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

// A contiguous tensor of this type and shape on the call's device.
const at::Tensor& exactly(PyObject* object, const char* name, at::ScalarType type,
                          at::IntArrayRef shape, const c10::Device& device) {
  const at::Tensor& x = tensor(object, name);
  if (x.scalar_type() != type || x.sizes() != shape || !x.is_contiguous())
    refuse(name, " must be a contiguous ", type, " tensor of shape ", shape, ", got ", x.sizes(), " ",
           x.scalar_type());
  require_device(x, device);
  require_no_gradient(x, name);
  return x;
}

// pages x 4, page_table, starts, counts, k, v, q or None, cos or None, sin or None, interleaved,
// return_keys, stream, [positions] -> (rotated q or None, rotated k or None)
PyObject* append(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, n == 16 ? 16 : 15, [&]() -> PyObject* {
    const at::Tensor& k_in = tensor(args[7], "k", true);
    const at::Tensor& v_in = tensor(args[8], "v", true);
    require_gpu(k_in);
    require_gpu(v_in);
    Description d(k_in.device());
    require_device(v_in, d.device);
    const at::Tensor k = rows(k_in, "k"), v = rows(v_in, "v");
    if (k.sizes() != v.sizes()) refuse("k ", k.sizes(), " and v ", v.sizes(), " differ");
    d.pages(args);
    d.map(args + 4, k.size(0), k.size(1));
    if (k.size(2) != d.c.kv_heads || k.size(3) != d.c.head_dim)
      refuse("k ", k.sizes(), " does not fit a cache of ", d.c.kv_heads, " heads of ", d.c.head_dim);
    at::Tensor q, q_out, k_out;
    if (args[9] != Py_None) {
      const at::Tensor& q_in = tensor(args[9], "q", true);
      require_gpu(q_in);
      require_device(q_in, d.device);
      q = rows(q_in, "q");
      if (q.size(0) != k.size(0) || q.size(1) != k.size(1) || q.size(3) != k.size(3) ||
          q.size(2) == 0)
        refuse("q ", q.sizes(), " does not match k ", k.sizes());
      q_out = empty(q.sizes(), at::kBFloat16, d.device);
    }
    if (truth(args[13])) k_out = empty(k.sizes(), at::kBFloat16, d.device);
    const float* table[2] = {nullptr, nullptr};
    int64_t positions = 0, half = 0;
    if ((args[10] == Py_None) != (args[11] == Py_None)) refuse("rope needs cos and sin");
    if (args[10] != Py_None) {
      const at::Tensor& first = tensor(args[10], "rope");
      for (int i = 0; i < 2; ++i) {
        const at::Tensor& x = tensor(args[10 + i], "rope");
        if (x.dim() != 2 || x.sizes() != first.sizes() || x.scalar_type() != at::kFloat ||
            !x.is_contiguous())
          refuse("rope must be two contiguous float32 [positions, rotary_dim // 2] tensors of one "
                 "shape, got ", x.sizes(), " ", x.scalar_type());
        require_device(x, d.device);
        require_no_gradient(x, "rope");
        table[i] = static_cast<const float*>(pointer(x));
      }
      positions = first.size(0);
      half = first.size(1);
      // an empty table has no memory, and would pass for none
      if (positions == 0 || half == 0) refuse("rope tables are empty: ", first.sizes());
    }
    const bool interleaved = truth(args[12]);
    void* stream = reinterpret_cast<void*>(integer(args[14]));
    const int32_t* at_positions = nullptr;
    if (n == 16) {
      if (table[0] == nullptr) refuse("positions without a rope table");
      at_positions = static_cast<const int32_t*>(
          pointer(exactly(args[15], "positions", at::kInt, k.sizes().slice(0, 2), d.device)));
    }
    if (d.c.batch > 0 && d.c.tokens > 0) {
      void* q_ptr = q.defined() ? pointer(q) : nullptr;
      const int64_t* q_strides = q.defined() ? q.strides().data() : nullptr;
      const int q_heads = q.defined() ? small(q.size(2), "query heads") : 0;
      const int reach = small(positions, "rope positions"), rotary = small(2 * half, "rotary_dim");
      void* q_to = q_out.defined() ? pointer(q_out) : nullptr;
      void* k_to = k_out.defined() ? pointer(k_out) : nullptr;
      if (at_positions == nullptr)
        check(spx_paged_append(&d.c, q_ptr, q_strides, pointer(k), k.strides().data(), pointer(v),
                               v.strides().data(), q_heads, table[0], table[1], reach, rotary,
                               interleaved, q_to, k_to, stream),
              "spx_paged_append");
      else
        check(spx_paged_append_at(&d.c, q_ptr, q_strides, pointer(k), k.strides().data(), pointer(v),
                                  v.strides().data(), q_heads, table[0], table[1], reach, rotary,
                                  interleaved, at_positions, q_to, k_to, stream),
              "spx_paged_append_at");
      for (int i = 0; i < 4; ++i)
        if (args[i] != Py_None) written(tensor(args[i], "pages"));
    }
    return pair(q_out, k_out);
  });
}

// pages x 4, page_table, starts, counts, tokens, stream -> (k, v)
PyObject* gather(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 9, [&]() -> PyObject* {
    const at::Tensor& table = tensor(args[4], "page_table");
    require_gpu(tensor(args[0], "key_pages"));
    require_gpu(table);
    Description d(table.device());
    const int64_t tokens = integer(args[7]);
    if (tokens < 0) refuse("tokens must not be negative, got ", tokens);
    d.pages(args);
    d.map(args + 4, table.dim() > 0 ? table.size(0) : 0, tokens);
    const int64_t shape[4] = {d.c.batch, tokens, d.c.kv_heads, d.c.head_dim};
    const at::Tensor k = empty(shape, at::kBFloat16, d.device);
    const at::Tensor v = empty(shape, at::kBFloat16, d.device);
    void* stream = reinterpret_cast<void*>(integer(args[8]));
    if (d.c.batch > 0 && tokens > 0)
      check(spx_paged_gather(&d.c, pointer(k), pointer(v), stream), "spx_paged_gather");
    return pair(k, v);
  });
}

// pages x 4, page_table, starts, counts, q, scale, max_keys, return_lse, stream -> out or (out, lse)
PyObject* attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 12, [&]() -> PyObject* {
    const at::Tensor& q_in = tensor(args[7], "q", true);
    require_gpu(q_in);
    Description d(q_in.device());
    const at::Tensor q = rows(q_in, "q");
    d.pages(args);
    d.map(args + 4, q.size(0), q.size(1));
    if (q.size(3) != d.c.head_dim || q.size(2) == 0 || d.c.kv_heads == 0 ||
        q.size(2) % d.c.kv_heads != 0)
      refuse("q ", q.sizes(), " does not fit a cache of ", d.c.kv_heads, " heads of ", d.c.head_dim);
    const double scale = PyFloat_AsDouble(args[8]);
    if (scale == -1.0 && PyErr_Occurred()) throw std::bad_exception();
    const int64_t max_keys = integer(args[9]);
    if (max_keys < 0) refuse("max_keys must not be negative, got ", max_keys);
    const int bound = (int)std::min<int64_t>(max_keys, INT_MAX);
    const int q_heads = small(q.size(2), "query heads");
    const at::Tensor out = empty(q.sizes(), at::kBFloat16, d.device);
    at::Tensor lse, workspace;
    if (truth(args[10])) lse = empty(q.sizes().slice(0, 3), at::kFloat, d.device);
    void* stream = reinterpret_cast<void*>(integer(args[11]));
    if (d.c.batch > 0 && d.c.tokens > 0) {
      const int64_t bytes = spx_paged_attention_workspace_bytes(&d.c, q_heads, bound);
      if (bytes > 0) workspace = empty({bytes}, at::kByte, d.device);
      check(spx_paged_attention(&d.c, pointer(q), q.strides().data(), q_heads, bound, (float)scale,
                                workspace.defined() ? pointer(workspace) : nullptr, pointer(out),
                                lse.defined() ? static_cast<float*>(pointer(lse)) : nullptr, stream),
            "spx_paged_attention");
    }
    return lse.defined() ? pair(out, lse) : wrap(out);
  });
}

// parents, stream -> (depths, masks)
PyObject* draft_tree(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 2, [&]() -> PyObject* {
    const at::Tensor& parents = tensor(args[0], "parents");
    require_gpu(parents);
    if (parents.dim() != 2 || parents.scalar_type() != at::kInt || !parents.is_contiguous() ||
        parents.size(1) == 0 || parents.size(1) > kTreeTokens)
      refuse("parents must be a contiguous int32 [batch, tokens] tensor of 1 to ", kTreeTokens,
             " tokens, got ", parents.sizes(), " ", parents.scalar_type());
    const int64_t shape[3] = {parents.size(0), parents.size(1), (parents.size(1) + 63) / 64};
    const at::Tensor depths = empty(parents.sizes(), at::kInt, parents.device());
    const at::Tensor masks = empty(shape, at::kLong, parents.device());
    if (shape[0] > 0)
      check(spx_draft_tree(static_cast<const int32_t*>(pointer(parents)), small(shape[0], "batch"),
                           (int)shape[1], static_cast<int32_t*>(pointer(depths)),
                           static_cast<uint64_t*>(pointer(masks)),
                           reinterpret_cast<void*>(integer(args[1]))),
            "spx_draft_tree");
    return pair(depths, masks);
  });
}

// pages x 4, page_table, starts, counts, q, masks, scale, max_keys, return_lse, stream -> out or
// (out, lse)
PyObject* tree_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 13, [&]() -> PyObject* {
    const at::Tensor& q_in = tensor(args[7], "q", true);
    require_gpu(q_in);
    Description d(q_in.device());
    const at::Tensor q = rows(q_in, "q");
    d.pages(args);
    d.map(args + 4, q.size(0), q.size(1));
    if (q.size(3) != d.c.head_dim || q.size(2) == 0 || d.c.kv_heads == 0 ||
        q.size(2) % d.c.kv_heads != 0)
      refuse("q ", q.sizes(), " does not fit a cache of ", d.c.kv_heads, " heads of ", d.c.head_dim);
    if (q.size(1) > kTreeTokens) refuse(q.size(1), " drafted tokens are more than ", kTreeTokens);
    const int64_t shape[3] = {q.size(0), q.size(1), (q.size(1) + 63) / 64};
    const at::Tensor& masks = exactly(args[8], "masks", at::kLong, shape, d.device);
    const double scale = PyFloat_AsDouble(args[9]);
    if (scale == -1.0 && PyErr_Occurred()) throw std::bad_exception();
    const int64_t max_keys = integer(args[10]);
    if (max_keys < 0) refuse("max_keys must not be negative, got ", max_keys);
    const int bound = (int)std::min<int64_t>(max_keys, INT_MAX);
    const int q_heads = small(q.size(2), "query heads");
    const at::Tensor out = empty(q.sizes(), at::kBFloat16, d.device);
    at::Tensor lse;
    if (truth(args[11])) lse = empty(q.sizes().slice(0, 3), at::kFloat, d.device);
    void* stream = reinterpret_cast<void*>(integer(args[12]));
    if (d.c.batch > 0 && d.c.tokens > 0) {
      const int64_t bytes = spx_paged_tree_attention_workspace_bytes(&d.c, q_heads, bound);
      const at::Tensor workspace = empty({std::max<int64_t>(bytes, 16)}, at::kByte, d.device);
      check(spx_paged_tree_attention(&d.c, pointer(q), q.strides().data(), q_heads,
                                     static_cast<const uint64_t*>(pointer(masks)), bound, (float)scale,
                                     pointer(workspace), pointer(out),
                                     lse.defined() ? static_cast<float*>(pointer(lse)) : nullptr,
                                     stream),
            "spx_paged_tree_attention");
    }
    return lse.defined() ? pair(out, lse) : wrap(out);
  });
}

// The pages of one PagedCache object.
void cache_pages(PyObject* cache, PyObject* (&held)[4]) {
  static PyObject* names[4] = {
      PyUnicode_InternFromString("key_pages"), PyUnicode_InternFromString("value_pages"),
      PyUnicode_InternFromString("key_scales"), PyUnicode_InternFromString("value_scales")};
  for (int i = 0; i < 4; ++i) {
    held[i] = PyObject_GetAttr(cache, names[i]);
    if (held[i] == nullptr) throw std::bad_exception();
  }
}

// tuple of PagedCaches, page_table, starts, counts, then either parents, drafts, targets, stream ->
// (accepted, path, following), or path, stream -> None
PyObject* keep_path(PyObject*, PyObject* const* args, Py_ssize_t n) {
  const bool walk = n == 8;
  return guarded(n, walk ? 8 : 6, [&]() -> PyObject* {
    if (!PyTuple_Check(args[0]) || PyTuple_GET_SIZE(args[0]) == 0) refuse("no caches");
    const Py_ssize_t count = PyTuple_GET_SIZE(args[0]);
    const at::Tensor& first = tensor(args[4], walk ? "parents" : "path");
    require_gpu(first);
    if (first.dim() != 2 || first.size(1) > kTreeTokens)
      refuse(walk ? "parents" : "path", " must be an int32 [batch, tokens] tensor of at most ",
             kTreeTokens, " tokens, got ", first.sizes());
    Description d(first.device());
    const auto shape = first.sizes();
    exactly(args[4], walk ? "parents" : "path", at::kInt, shape, d.device);
    struct Pages {
      PyObject* held[4] = {};
      ~Pages() {
        for (PyObject* x : held) Py_XDECREF(x);
      }
    };
    std::vector<Pages> objects(count);
    std::vector<spx_paged_cache> caches(count);
    for (Py_ssize_t i = 0; i < count; ++i) {
      cache_pages(PyTuple_GET_ITEM(args[0], i), objects[i].held);
      d.pages(objects[i].held);
      if (i == 0) d.map(args + 1, shape[0], shape[1]);
      if (objects[i].held[2] == Py_None) d.c.key_scales = d.c.value_scales = nullptr;
      caches[i] = d.c;
    }
    // Rows would move twice, the second time from places that the first has filled.
    std::vector<std::pair<uintptr_t, size_t>> ranges;
    ranges.reserve(4 * count);
    for (const Pages& x : objects)
      for (PyObject* page : x.held)
        if (page != Py_None) {
          const at::Tensor& held = THPVariable_Unpack(page);
          ranges.emplace_back(reinterpret_cast<uintptr_t>(held.data_ptr()), held.nbytes());
        }
    std::sort(ranges.begin(), ranges.end());
    for (size_t i = 1; i < ranges.size(); ++i)
      if (ranges[i].first < ranges[i - 1].first + ranges[i - 1].second)
        refuse("the caches' pages overlap each other");
    at::Tensor accepted, path, following;
    const int64_t *drafts = nullptr, *targets = nullptr;
    if (walk) {
      drafts = static_cast<const int64_t*>(
          pointer(exactly(args[5], "drafts", at::kLong, shape, d.device)));
      targets = static_cast<const int64_t*>(
          pointer(exactly(args[6], "targets", at::kLong, shape, d.device)));
      accepted = empty({shape[0]}, at::kInt, d.device);
      path = empty(shape, at::kInt, d.device);
      following = empty({shape[0]}, at::kLong, d.device);
    }
    void* stream = reinterpret_cast<void*>(integer(args[walk ? 7 : 5]));
    if (shape[0] > 0 && shape[1] > 0) {
      const int32_t* nodes = static_cast<const int32_t*>(pointer(first));
      check(spx_paged_keep_path(caches.data(), small(count, "caches"), walk ? nodes : nullptr, drafts,
                                targets, walk ? nullptr : nodes,
                                walk ? static_cast<int32_t*>(pointer(accepted)) : nullptr,
                                walk ? static_cast<int32_t*>(pointer(path)) : nullptr,
                                walk ? static_cast<int64_t*>(pointer(following)) : nullptr, stream),
            "spx_paged_keep_path");
      for (const Pages& x : objects)
        for (PyObject* page : x.held)
          if (page != Py_None) written(tensor(page, "pages"));
    } else if (walk && shape[0] > 0) {
      refuse("trees without nodes");
    }
    if (!walk) Py_RETURN_NONE;
    PyObject *a = wrap(accepted), *b = wrap(path), *c = wrap(following);
    PyObject* out = a && b && c ? PyTuple_Pack(3, a, b, c) : nullptr;
    Py_XDECREF(a);
    Py_XDECREF(b);
    Py_XDECREF(c);
    return out;
  });
}

// A ledger tensor: [B, Hkv, slots] for all slots that the page table reaches.
const at::Tensor& ledger(const Description& d, PyObject* object, const char* name,
                         at::ScalarType type) {
  const at::Tensor& x = tensor(object, name);
  const int64_t reach = (int64_t)d.c.table_width * d.c.page_size;
  if (x.dim() != 3 || x.scalar_type() != type || x.size(0) != d.c.batch || x.size(1) != d.c.kv_heads ||
      x.size(2) < reach || !x.is_contiguous())
    refuse(name, " must be a contiguous ", type, " [", d.c.batch, ", ", d.c.kv_heads,
           ", slots] tensor of at least ", reach, " slots, got ", x.sizes(), " ", x.scalar_type());
  require_device(x, d.device);
  require_no_gradient(x, name);
  return x;
}

// pages x 4, page_table, starts, counts, weights, q, lse, scale, stream -> None
PyObject* accumulate(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 12, [&]() -> PyObject* {
    const at::Tensor& q_in = tensor(args[8], "q", true);
    require_gpu(q_in);
    Description d(q_in.device());
    const at::Tensor q = rows(q_in, "q");
    d.pages(args);
    d.map(args + 4, q.size(0), q.size(1));
    if (q.size(3) != d.c.head_dim || q.size(2) == 0 || d.c.kv_heads == 0 ||
        q.size(2) % d.c.kv_heads != 0)
      refuse("q ", q.sizes(), " does not fit a cache of ", d.c.kv_heads, " heads of ", d.c.head_dim);
    const at::Tensor& weights = ledger(d, args[7], "weights", at::kFloat);
    const at::Tensor& lse_in = tensor(args[9], "lse", true);
    if (lse_in.scalar_type() != at::kFloat || lse_in.sizes() != q.sizes().slice(0, 3))
      refuse("lse must be a float32 tensor of shape ", q.sizes().slice(0, 3), ", got ",
             lse_in.sizes(), " ", lse_in.scalar_type());
    require_device(lse_in, d.device);
    const at::Tensor lse = plain(lse_in, "lse");
    const double scale = PyFloat_AsDouble(args[10]);
    if (scale == -1.0 && PyErr_Occurred()) throw std::bad_exception();
    void* stream = reinterpret_cast<void*>(integer(args[11]));
    if (d.c.batch > 0 && d.c.tokens > 0) {
      const int q_heads = small(q.size(2), "query heads");
      const int64_t bytes = spx_paged_accumulate_weights_workspace_bytes(&d.c, q_heads);
      at::Tensor workspace;
      if (bytes > 0) workspace = empty({bytes}, at::kByte, d.device);
      check(spx_paged_accumulate_weights(&d.c, pointer(q), q.strides().data(), q_heads,
                                         static_cast<const float*>(pointer(lse)), (float)scale,
                                         workspace.defined() ? pointer(workspace) : nullptr,
                                         static_cast<float*>(pointer(weights)), weights.size(2), stream),
            "spx_paged_accumulate_weights");
      written(weights);
    }
    Py_RETURN_NONE;
  });
}

// pages x 4, page_table, lengths, weights, positions or None, seen or None, budget, recent, sinks,
// weights out or None, positions out or None, stream -> (lengths, weights, positions)
PyObject* evict(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 15, [&]() -> PyObject* {
    const at::Tensor& lengths = tensor(args[5], "lengths");
    require_gpu(lengths);
    Description d(lengths.device());
    d.pages(args);
    PyObject* const map[3] = {args[4], args[5], Py_None};
    d.map(map, lengths.dim() == 1 ? lengths.size(0) : 0, 1);
    const at::Tensor& weights = ledger(d, args[6], "weights", at::kFloat);
    const int32_t *positions = nullptr, *seen = nullptr;
    if (args[7] != Py_None) {
      const at::Tensor& x = ledger(d, args[7], "positions", at::kInt);
      if (x.sizes() != weights.sizes())
        refuse("positions ", x.sizes(), " and weights ", weights.sizes(), " differ");
      positions = static_cast<const int32_t*>(pointer(x));
    }
    if (args[8] != Py_None) seen = d.lengths(args[8], "seen");
    const int64_t budget = integer(args[9]), recent = integer(args[10]), sinks = integer(args[11]);
    if (budget <= 0 || recent < 0 || sinks < 0 || recent > budget || sinks > budget - recent)
      refuse("a budget of ", budget, " must be positive and hold the ", recent, " recent and ", sinks,
             " first tokens");
    if ((args[12] == Py_None) != (args[13] == Py_None)) refuse("out needs weights and positions");
    at::Tensor weights_out, positions_out;
    if (args[12] == Py_None) {
      weights_out = empty(weights.sizes(), at::kFloat, d.device);
      positions_out = empty(weights.sizes(), at::kInt, d.device);
    } else {
      weights_out = ledger(d, args[12], "out weights", at::kFloat);
      positions_out = ledger(d, args[13], "out positions", at::kInt);
      if (weights_out.sizes() != weights.sizes() || positions_out.sizes() != weights.sizes())
        refuse("out ", weights_out.sizes(), " and ", positions_out.sizes(), " differ from weights ",
               weights.sizes());
      // A row is written while others are read: only in its own place.
      bool shared = overlap(weights_out, positions_out) || overlap(positions_out, weights);
      shared = shared || (weights_out.data_ptr() != weights.data_ptr() && overlap(weights_out, weights));
      if (args[7] != Py_None) {
        const at::Tensor& x = tensor(args[7], "positions");
        shared = shared || overlap(weights_out, x) ||
                 (positions_out.data_ptr() != x.data_ptr() && overlap(positions_out, x));
      }
      for (PyObject* read : {args[5], args[8]})
        if (read != Py_None)
          shared = shared || overlap(weights_out, tensor(read, "lengths")) ||
                   overlap(positions_out, tensor(read, "lengths"));
      if (shared) refuse("out must be the weights and positions themselves or overlap no argument");
    }
    const at::Tensor left = empty(lengths.sizes(), at::kInt, d.device);
    void* stream = reinterpret_cast<void*>(integer(args[14]));
    if (d.c.batch > 0) {
      const int limit = (int)std::min<int64_t>(budget, INT_MAX);
      const int64_t bytes = spx_paged_evict_workspace_bytes(&d.c, limit);
      const at::Tensor workspace = empty({std::max<int64_t>(bytes, 16)}, at::kByte, d.device);
      check(spx_paged_evict(&d.c, static_cast<const float*>(pointer(weights)), positions,
                            weights.size(2), seen, limit, (int)std::min<int64_t>(recent, INT_MAX),
                            (int)std::min<int64_t>(sinks, INT_MAX), pointer(workspace),
                            static_cast<float*>(pointer(weights_out)),
                            static_cast<int32_t*>(pointer(positions_out)),
                            static_cast<int32_t*>(pointer(left)), stream),
            "spx_paged_evict");
      for (int i = 0; i < 4; ++i)
        if (args[i] != Py_None) written(tensor(args[i], "pages"));
      if (args[12] != Py_None) {
        written(weights_out);
        written(positions_out);
      }
    }
    PyObject *a = wrap(left), *b = wrap(weights_out), *c = wrap(positions_out);
    PyObject* out = a && b && c ? PyTuple_Pack(3, a, b, c) : nullptr;
    Py_XDECREF(a);
    Py_XDECREF(b);
    Py_XDECREF(c);
    return out;
  });
}

// pages x 4, page_table, starts, counts, batch, tokens -> (pages, page_size, Hkv, D, table width):
// the checks alone, on any device
PyObject* describe(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 9, [&]() -> PyObject* {
    Description d(tensor(args[0], "key_pages").device());
    d.pages(args);
    d.map(args + 4, integer(args[7]), integer(args[8]));
    return Py_BuildValue("iiiii", d.c.pages, d.c.page_size, d.c.kv_heads, d.c.head_dim,
                         d.c.table_width);
  });
}

PyMethodDef kMethods[] = {
    {"append", (PyCFunction)(void (*)(void))append, METH_FASTCALL, nullptr},
    {"gather", (PyCFunction)(void (*)(void))gather, METH_FASTCALL, nullptr},
    {"attention", (PyCFunction)(void (*)(void))attention, METH_FASTCALL, nullptr},
    {"draft_tree", (PyCFunction)(void (*)(void))draft_tree, METH_FASTCALL, nullptr},
    {"tree_attention", (PyCFunction)(void (*)(void))tree_attention, METH_FASTCALL, nullptr},
    {"keep_path", (PyCFunction)(void (*)(void))keep_path, METH_FASTCALL, nullptr},
    {"accumulate", (PyCFunction)(void (*)(void))accumulate, METH_FASTCALL, nullptr},
    {"evict", (PyCFunction)(void (*)(void))evict, METH_FASTCALL, nullptr},
    {"describe", (PyCFunction)(void (*)(void))describe, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_paged", nullptr, -1, kMethods,
                       nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__paged(void) { return PyModule_Create(&kModule); }
