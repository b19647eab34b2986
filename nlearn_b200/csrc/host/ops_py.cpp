// ops_py.cpp — the host side of the serving operators (nlearn_b200/paged.py,
// nlearn_b200/kernels/logits.py): checks of the tensors they are given, their
// outputs and workspaces, and the call of the C entry points of libnl_ops.so.
//
// The operators are a few microseconds of GPU work and take up to a dozen
// tensors.  The same checks written in Python read some sixty attributes and
// took longer than the kernels: 13.5 us a call for the attention of one short
// sequence (4.7 us on the GPU), 17.5 us for a step of the block tables (6.0 us).
//
// Every function takes its arguments by position (None where one is left out),
// raises ValueError for shapes, strides, places and values, TypeError for
// types, RuntimeError where a gradient is asked for or a call fails, and launches on the
// current stream of the tensors' device.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cstdarg>
#include <cstdio>
#include <string>
#include <utility>

#include "../../../include/nl_ops.h"

namespace {

struct Refusal {
  PyObject* type;
  std::string text;
};
[[noreturn]] void refuse(PyObject* type, const char* format, ...) {
  char buf[512];
  va_list args;
  va_start(args, format);
  vsnprintf(buf, sizeof(buf), format, args);
  va_end(args);
  throw Refusal{type, buf};
}
std::string list(c10::IntArrayRef x) {
  std::string s = "(";
  for (size_t i = 0; i < x.size(); ++i) s += (i ? ", " : "") + std::to_string(x[i]);
  return s + ")";
}
const char* type_name(const at::Tensor& t) { return c10::toString(t.scalar_type()); }

// ---------------------------------------------------------------- arguments
const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) refuse(PyExc_TypeError, "%s must be a torch.Tensor", name);
  return THPVariable_Unpack(o);
}
int place(const at::Tensor& t, const char* name) {
  if (!t.is_cuda())
    refuse(PyExc_ValueError, "%s: nlearn_b200 runs on CUDA tensors only (no CPU fallback)", name);
  return t.get_device();
}
void same_place(const at::Tensor& t, const char* name, int index) {
  if (place(t, name) != index)
    refuse(PyExc_ValueError, "%s is on cuda:%d, expected cuda:%d", name, static_cast<int>(t.get_device()), index);
}
void no_grad(const at::Tensor& t, const char* name) {
  if (t.requires_grad() && c10::GradMode::is_enabled())
    refuse(PyExc_RuntimeError, "%s: the serving operators have no backward, call them under torch.no_grad()", name);
}
int whole(PyObject* o, const char* name) {
  const long long x = PyLong_AsLongLong(o);
  if (x == -1 && PyErr_Occurred()) throw Refusal{nullptr, ""};
  if (x < INT32_MIN || x > INT32_MAX) refuse(PyExc_ValueError, "%s %lld: out of range", name, x);
  return static_cast<int>(x);
}
double number(PyObject* o) {
  const double x = PyFloat_AsDouble(o);
  if (x == -1.0 && PyErr_Occurred()) throw Refusal{nullptr, ""};
  return x;
}
int size32(int64_t n, const char* what) {
  if (n > INT32_MAX) refuse(PyExc_ValueError, "%s %lld: over the limit of 2**31 - 1", what, static_cast<long long>(n));
  return static_cast<int>(n);
}
uintptr_t address(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()); }

// A contiguous vector of n elements of a type.
template <typename E>
E* vector(const at::Tensor& t, const char* name, at::ScalarType type, int64_t n, int index) {
  same_place(t, name, index);
  if (t.scalar_type() != type) {
    // a wrong float type is a wrong value of a parameter, a wrong index type a wrong type
    refuse(type == at::kInt ? PyExc_TypeError : PyExc_ValueError, "%s must be %s, got %s", name, c10::toString(type),
           type_name(t));
  }
  if (type == at::kFloat) no_grad(t, name);
  if (t.dim() != 1 || t.size(0) != n || (n > 1 && t.stride(0) != 1))
    refuse(PyExc_ValueError, "%s must be a contiguous vector of %lld elements, got shape %s with strides %s", name,
           static_cast<long long>(n), list(t.sizes()).c_str(), list(t.strides()).c_str());
  return static_cast<E*>(t.data_ptr());
}
template <typename E>
E* vector_or_none(PyObject* o, const char* name, at::ScalarType type, int64_t n, int index) {
  return o == Py_None ? nullptr : vector<E>(tensor(o, name), name, type, n, index);
}

// An int32 matrix with contiguous rows that do not overlap; rows < 0: any number.
struct Matrix {
  int* p;
  int rows, cols;
  long long ld;
};
Matrix matrix(const at::Tensor& t, const char* name, int64_t rows, int index) {
  same_place(t, name, index);
  if (t.scalar_type() != at::kInt) refuse(PyExc_TypeError, "%s must be Int, got %s", name, type_name(t));
  if (t.dim() != 2 || (rows >= 0 && t.size(0) != rows) || (t.size(1) > 1 && t.stride(1) != 1) ||
      (t.size(0) > 1 && t.stride(0) < t.size(1)))
    refuse(PyExc_ValueError, "%s must be a matrix of %lld contiguous rows that do not overlap, got shape %s with strides %s",
           name, static_cast<long long>(rows), list(t.sizes()).c_str(), list(t.strides()).c_str());
  return {static_cast<int*>(t.data_ptr()), size32(t.size(0), name), size32(t.size(1), name),
          std::max<long long>(t.stride(0), t.size(1))};
}

// bf16 [n, heads, d] with contiguous 16-byte aligned rows: the tensor, or a copy where it is not so.
at::Tensor rows(const at::Tensor& t, const char* name, int64_t n, int64_t heads, int64_t d, int index) {
  same_place(t, name, index);
  if (t.scalar_type() != at::kBFloat16) refuse(PyExc_TypeError, "%s must be BFloat16, got %s", name, type_name(t));
  if (t.dim() != 3 || t.size(0) != n || t.size(1) != heads || t.size(2) != d)
    refuse(PyExc_ValueError, "%s must have shape (%lld, %lld, %lld), got %s", name, static_cast<long long>(n),
           static_cast<long long>(heads), static_cast<long long>(d), list(t.sizes()).c_str());
  // (expanded rows have stride 0: they are read as they are)
  if (t.stride(2) == 1 && !((t.stride(0) | t.stride(1)) & 7) && !(address(t) & 15)) return t;
  return t.clone(at::MemoryFormat::Contiguous);
}

// Whether a tensor that is written is free of elements that share memory: every stride steps over
// all that the smaller ones reach.
bool apart(const at::Tensor& t) {
  std::pair<int64_t, int64_t> dims[4];  // (stride, size); caches have the most dimensions
  int n = 0;
  for (int64_t i = 0; i < t.dim(); ++i)
    if (t.size(i) > 1) dims[n++] = {t.stride(i), t.size(i)};
  std::sort(dims, dims + n);
  int64_t span = 1;
  for (int i = 0; i < n; ++i) {
    if (dims[i].first < span) return false;
    span += (dims[i].second - 1) * dims[i].first;
  }
  return true;
}

struct Caches {
  void *k, *v;
  int dtype, n_pages, heads, page, d;
  long long page_s, head_s, tok_s;
};
Caches caches(const at::Tensor& k, const at::Tensor& v, int index) {
  same_place(k, "k_cache", index);
  same_place(v, "v_cache", index);
  no_grad(k, "k_cache");
  no_grad(v, "v_cache");
  const auto type = k.scalar_type();
  if ((type != at::kBFloat16 && type != at::kFloat8_e4m3fn) || v.scalar_type() != type)
    refuse(PyExc_TypeError, "caches must both be BFloat16 or Float8_e4m3fn, got %s and %s", type_name(k), type_name(v));
  if (k.dim() != 4 || v.sizes() != k.sizes())
    refuse(PyExc_ValueError, "caches must be [n_pages, kv_heads, page_size, head_dim], both of one shape, got %s and %s",
           list(k.sizes()).c_str(), list(v.sizes()).c_str());
  if (v.strides() != k.strides())
    refuse(PyExc_ValueError, "caches must have the same strides, got %s and %s", list(k.strides()).c_str(),
           list(v.strides()).c_str());
  const bool fp8 = type == at::kFloat8_e4m3fn;
  if ((k.size(3) > 1 && k.stride(3) != 1) || ((k.stride(0) | k.stride(1) | k.stride(2)) & (fp8 ? 15 : 7)) ||
      ((address(k) | address(v)) & 15))
    refuse(PyExc_ValueError, "cache rows must be contiguous and lie on 16-byte boundaries, got strides %s",
           list(k.strides()).c_str());
  size32(k.size(0) * k.size(2), "slots of a cache");
  return {k.data_ptr(), v.data_ptr(), fp8 ? NL_E4M3 : NL_BF16, size32(k.size(0), "pages"), size32(k.size(1), "heads"),
          size32(k.size(2), "page_size"), size32(k.size(3), "head_dim"), k.stride(0), k.stride(1), k.stride(2)};
}
// Caches that a call writes into.
void writable(const at::Tensor& k, const at::Tensor& v) {
  if (!apart(k)) refuse(PyExc_ValueError, "slots of the caches share memory, got strides %s", list(k.strides()).c_str());
  if (k.numel() > 0 && k.data_ptr() == v.data_ptr())
    refuse(PyExc_ValueError, "k_cache and v_cache are the same memory");
}
const float* cache_scale(PyObject* o, const char* name, const Caches& c, int index) {
  if (o == Py_None) return nullptr;
  if (c.dtype != NL_E4M3) refuse(PyExc_ValueError, "%s goes with a float8_e4m3fn cache", name);
  return vector<float>(tensor(o, name), name, at::kFloat, c.heads, index);
}

void call(int status, const char* what) {
  static const char* const names[] = {"NL_OK", "NL_ERR_SHAPE", "NL_ERR_ALIGN", "NL_ERR_LAUNCH", "NL_ERR_CUDA",
                                      "NL_ERR_DTYPE", "NL_ERR_WORKSPACE", "NL_ERR_TOO_LARGE"};
  if (status == 0) return;
  PyObject* module = PyImport_ImportModule("nlearn_b200._lib");
  PyObject* type = module ? PyObject_GetAttrString(module, "NlError") : nullptr;
  Py_XDECREF(module);
  if (!type) throw Refusal{nullptr, ""};
  const Refusal r{type, std::string(what) + " returned " +
                            (status < 0 && status > -8 ? names[-status] : std::to_string(status).c_str())};
  Py_DECREF(type);  // (the module keeps it)
  throw r;
}

// int32 vectors cut from one allocation, each on a 16-byte boundary (they share
// its storage: six allocations took two thirds of a call's host time).
class Cutter {
 public:
  Cutter(std::initializer_list<int64_t> sizes, const at::TensorOptions& options) {
    int64_t n = 0;
    for (const int64_t s : sizes) n += (s + 3) / 4 * 4;
    all_ = at::empty({n}, options);
  }
  at::Tensor next(int64_t n) {
    at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(all_.storage()), all_.key_set(), all_.dtype());
    t.unsafeGetTensorImpl()->set_sizes_contiguous(n);
    t.unsafeGetTensorImpl()->set_storage_offset(at_);
    at_ += (n + 3) / 4 * 4;
    return t;
  }

 private:
  at::Tensor all_;
  int64_t at_ = 0;
};

// ---------------------------------------------------------------- operators
// q, k_cache, v_cache, block_table, lens, k_new, v_new, k_scale, v_scale, scale, out, lse
PyObject* attention(PyObject* const* a) {
  const at::Tensor& q0 = tensor(a[0], "q");
  const int index = place(q0, "q");
  no_grad(q0, "q");
  if (q0.dim() != 3) refuse(PyExc_ValueError, "q must be [batch, heads, head_dim], got %s", list(q0.sizes()).c_str());
  const Caches c = caches(tensor(a[1], "k_cache"), tensor(a[2], "v_cache"), index);
  const int64_t B = q0.size(0), Hq = q0.size(1), d = q0.size(2);
  if (d != c.d || (d != 64 && d != 128))
    refuse(PyExc_ValueError, "head_dim must be 64 or 128 and the caches', got %lld and %d", static_cast<long long>(d), c.d);
  if (c.heads == 0 || Hq == 0 || Hq % c.heads)
    refuse(PyExc_ValueError, "%lld query heads do not share %d kv heads evenly", static_cast<long long>(Hq), c.heads);
  const at::Tensor q = rows(q0, "q", B, Hq, d, index);
  const Matrix table = matrix(tensor(a[3], "block_table"), "block_table", B, index);
  const int* lens = vector<int>(tensor(a[4], "lens"), "lens", at::kInt, B, index);
  at::Tensor kn, vn;
  if ((a[5] == Py_None) != (a[6] == Py_None)) refuse(PyExc_ValueError, "k_new and v_new come together");
  if (a[5] != Py_None) {
    const at::Tensor &k0 = tensor(a[5], "k_new"), &v0 = tensor(a[6], "v_new");
    writable(tensor(a[1], "k_cache"), tensor(a[2], "v_cache"));
    no_grad(k0, "k_new");
    no_grad(v0, "v_new");
    kn = rows(k0, "k_new", B, c.heads, d, index);
    vn = rows(v0, "v_new", B, c.heads, d, index);
    if (kn.strides() != vn.strides()) {
      kn = kn.contiguous();
      vn = vn.contiguous();
    }
  }
  const float* ks = cache_scale(a[7], "k_scale", c, index);
  const float* vs = cache_scale(a[8], "v_scale", c, index);
  const double scale = a[9] == Py_None ? (d == 64 ? 0.125 : 0.08838834764831845) : number(a[9]);
  at::Tensor out;
  if (a[10] == Py_None) {
    out = at::empty({B, Hq, d}, q.options());
  } else {
    out = tensor(a[10], "out");
    same_place(out, "out", index);
    no_grad(out, "out");
    if (out.sizes() != q0.sizes() || out.scalar_type() != at::kBFloat16 || out.stride(2) != 1 || !apart(out))
      refuse(PyExc_ValueError, "out must be bfloat16 %s with contiguous rows that do not overlap",
             list(q0.sizes()).c_str());
  }
  float* lse = nullptr;
  long long lse_b = 0;
  if (a[11] != Py_None) {
    const at::Tensor& t = tensor(a[11], "lse");
    same_place(t, "lse", index);
    no_grad(t, "lse");
    if (t.scalar_type() != at::kFloat || t.dim() != 2 || t.size(0) != B || t.size(1) != Hq ||
        (Hq > 1 && t.stride(1) != 1) || !apart(t))
      refuse(PyExc_ValueError, "lse must be float32 (%lld, %lld) with contiguous rows that do not overlap",
             static_cast<long long>(B), static_cast<long long>(Hq));
    lse = static_cast<float*>(t.data_ptr());
    lse_b = t.stride(0);
  }
  if (B > 0) {
    if (table.cols == 0 || c.n_pages == 0 || c.page == 0)
      refuse(PyExc_ValueError, "block_table and caches must hold at least one page");
    const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(index));
    const int b32 = size32(B, "batch"), h32 = size32(Hq, "heads");
    const size_t bytes = nl_paged_attention_workspace_bytes(b32, h32, c.heads, c.d, c.page, table.cols, c.dtype);
    at::Tensor ws;
    if (bytes) ws = at::empty({static_cast<int64_t>(bytes)}, q.options().dtype(at::kByte));
    const nl_paged_attention_args args{
        q.data_ptr(), c.k, c.v, table.p, lens, kn.defined() ? kn.data_ptr() : nullptr,
        vn.defined() ? vn.data_ptr() : nullptr, ks, vs, out.data_ptr(), lse, bytes ? ws.data_ptr() : nullptr,
        q.stride(0), q.stride(1), c.page_s, c.head_s, c.tok_s, table.ld, kn.defined() ? kn.stride(0) : 0,
        kn.defined() ? kn.stride(1) : 0, out.stride(0), out.stride(1), lse_b, bytes, b32, h32, c.heads, c.d, c.page,
        table.cols, c.n_pages, c.dtype, static_cast<float>(scale)};
    call(nl_paged_attention(&args, c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(index)).stream()),
         "nl_paged_attention");
  }
  if (a[10] != Py_None) return Py_NewRef(a[10]);
  return THPVariable_Wrap(out);
}

// k, v, k_cache, v_cache, slots, k_scale, v_scale
PyObject* kv_write(PyObject* const* a) {
  const at::Tensor &k0 = tensor(a[0], "k"), &v0 = tensor(a[1], "v");
  const int index = place(k0, "k");
  no_grad(k0, "k");
  no_grad(v0, "v");
  const Caches c = caches(tensor(a[2], "k_cache"), tensor(a[3], "v_cache"), index);
  writable(tensor(a[2], "k_cache"), tensor(a[3], "v_cache"));
  if (c.d & (c.dtype == NL_E4M3 ? 15 : 7))
    refuse(PyExc_ValueError, "head_dim %d: cache rows must be whole 16-byte pieces", c.d);
  const int64_t T = k0.dim() == 3 ? k0.size(0) : -1;
  at::Tensor k = rows(k0, "k", T, c.heads, c.d, index), v = rows(v0, "v", T, c.heads, c.d, index);
  if (k.strides() != v.strides()) {
    k = k.contiguous();
    v = v.contiguous();
  }
  const int* slots = vector<int>(tensor(a[4], "slots"), "slots", at::kInt, T, index);
  const float* ks = cache_scale(a[5], "k_scale", c, index);
  const float* vs = cache_scale(a[6], "v_scale", c, index);
  if (T > 0 && c.n_pages > 0 && c.page > 0 && c.heads > 0 && c.d > 0) {
    const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(index));
    const nl_paged_kv_write_args args{k.data_ptr(), v.data_ptr(), c.k, c.v, slots, ks, vs, k.stride(0), k.stride(1),
                                      c.page_s, c.head_s, c.tok_s, size32(T, "tokens"), c.heads, c.d, c.page,
                                      c.n_pages, c.dtype};
    call(nl_paged_kv_write(&args, c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(index)).stream()),
         "nl_paged_kv_write");
  }
  return Py_NewRef(Py_None);
}

// block_table, lens, new_lens, free_pages, n_free, page_size, n_tokens, done, lens_out, n_free_out
PyObject* update_tables(PyObject* const* a) {
  constexpr int kMaxRows = 8192;
  const at::Tensor& t0 = tensor(a[0], "block_table");
  const int index = place(t0, "block_table");
  const Matrix table = matrix(t0, "block_table", -1, index);
  const int page = whole(a[5], "page_size"), n_tokens = whole(a[6], "n_tokens");
  const at::Tensor& free0 = tensor(a[3], "free_pages");
  const int64_t n_pages = free0.dim() == 1 ? free0.size(0) : -1;
  int* free_pages = vector<int>(free0, "free_pages", at::kInt, n_pages, index);
  if (table.rows == 0 || table.rows > kMaxRows || table.cols == 0 || n_pages == 0)
    refuse(PyExc_ValueError, "block_table must have 1 to %d rows and at least one page a row, got (%d, %d) and %lld pages",
           kMaxRows, table.rows, table.cols, static_cast<long long>(n_pages));
  if (page < 1 || n_tokens < 0 || static_cast<int64_t>(table.cols) * page > INT32_MAX || n_pages * page > INT32_MAX)
    refuse(PyExc_ValueError, "page_size %d, n_tokens %d: out of range", page, n_tokens);
  const int64_t B = table.rows;
  const at::Tensor &lens0 = tensor(a[1], "lens"), &n_free0 = tensor(a[4], "n_free");
  const int* lens = vector<int>(lens0, "lens", at::kInt, B, index);
  const int* new_lens = vector<int>(tensor(a[2], "new_lens"), "new_lens", at::kInt, B, index);
  const int* n_free = vector<int>(n_free0, "n_free", at::kInt, 1, index);
  const int* done = vector_or_none<int>(a[7], "done", at::kInt, B, index);
  Cutter cut({n_tokens, n_tokens, B + 1, B, B, 1}, lens0.options());
  at::Tensor lens_out, n_free_out;
  if (a[8] == Py_None) lens_out = cut.next(B);
  else vector<int>(lens_out = tensor(a[8], "lens_out"), "lens_out", at::kInt, B, index);
  if (a[9] == Py_None) n_free_out = cut.next(1);
  else vector<int>(n_free_out = tensor(a[9], "n_free_out"), "n_free_out", at::kInt, 1, index);
  const at::Tensor slots = cut.next(n_tokens), positions = cut.next(n_tokens), cu = cut.next(B + 1);
  const at::Tensor status = cut.next(B);
  {
    const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(index));
    auto p = [](const at::Tensor& t) { return static_cast<int*>(t.data_ptr()); };
    const nl_update_block_tables_args args{table.p, lens, new_lens, done, free_pages, n_free, p(lens_out),
                                           p(n_free_out), p(slots), p(positions), p(cu), p(status), table.ld,
                                           table.rows, table.cols, page, static_cast<int>(n_pages), n_tokens};
    call(nl_update_block_tables(&args, c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(index)).stream()),
         "nl_update_block_tables");
  }
  PyObject* items[6] = {THPVariable_Wrap(slots), THPVariable_Wrap(positions), THPVariable_Wrap(cu),
                        a[8] == Py_None ? THPVariable_Wrap(lens_out) : Py_NewRef(a[8]),
                        a[9] == Py_None ? THPVariable_Wrap(n_free_out) : Py_NewRef(a[9]), THPVariable_Wrap(status)};
  PyObject* result = PyTuple_New(6);
  for (int i = 0; i < 6; ++i) {
    if (!items[i] || !result) {
      for (int k = i; k < 6; ++k) Py_XDECREF(items[k]);
      Py_XDECREF(result);
      throw Refusal{nullptr, ""};
    }
    PyTuple_SET_ITEM(result, i, items[i]);
  }
  return result;
}

// logits, tokens, lens, prompt_lens, repetition, frequency, presence, bias_ids, bias, mask, mask_rows, out
PyObject* logits(PyObject* const* a) {
  const at::Tensor& x = tensor(a[0], "logits");
  const int index = place(x, "logits");
  no_grad(x, "logits");
  const auto type = x.scalar_type();
  if (type != at::kFloat && type != at::kBFloat16)
    refuse(PyExc_TypeError, "logits must be float32 or bfloat16, got %s", type_name(x));
  const bool f32 = type == at::kFloat;
  constexpr int kMost = (1 << 30) - 1;
  if (x.dim() != 2) refuse(PyExc_ValueError, "logits must be [batch, vocab], got %s", list(x.sizes()).c_str());
  const int64_t B = x.size(0), V = x.size(1);
  auto good_rows = [&](const at::Tensor& t) { return (V <= 1 || t.stride(1) == 1) && (B <= 1 || t.stride(0) >= V); };
  if (!good_rows(x)) refuse(PyExc_ValueError, "rows of logits must be contiguous and not overlap");
  if (B > 65535 || V == 0 || V > kMost)
    refuse(PyExc_ValueError, "logits must have at most 65535 rows and 1 to 2**30 - 1 columns, got %s",
           list(x.sizes()).c_str());
  at::Tensor y;
  if (a[11] == Py_None) {
    // rows on 16-byte boundaries, whatever the vocabulary
    const int64_t per = f32 ? 4 : 8;
    y = at::empty_strided({B, V}, {(V + per - 1) / per * per, 1}, x.options());
  } else {
    y = tensor(a[11], "out");
    same_place(y, "out", index);
    no_grad(y, "out");
    if (y.sizes() != x.sizes() || y.scalar_type() != type)
      refuse(PyExc_ValueError, "out must have the shape and type of logits");
    if (!good_rows(y)) refuse(PyExc_ValueError, "rows of out must be contiguous and not overlap");
    const bool same = y.data_ptr() == x.data_ptr() && (B <= 1 || y.stride(0) == x.stride(0));
    auto end = [&](const at::Tensor& t) { return address(t) + ((B - 1) * t.stride(0) + V) * t.element_size(); };
    if (!same && B > 0 && address(y) < end(x) && address(x) < end(y))
      refuse(PyExc_ValueError, "out must be logits itself or not overlap it");
  }
  nl_process_logits_args args{};
  args.logits = x.data_ptr();
  args.out = y.data_ptr();
  args.ldx = std::max<long long>(x.stride(0), V);
  args.ldy = std::max<long long>(y.stride(0), V);
  args.dtype = f32 ? NL_F32 : NL_BF16;
  args.B = static_cast<int>(B);
  args.V = static_cast<int>(V);
  if (a[1] != Py_None) {
    if (a[2] == Py_None) refuse(PyExc_ValueError, "tokens come with lens");
    const Matrix t = matrix(tensor(a[1], "tokens"), "tokens", B, index);
    args.lens = vector<int>(tensor(a[2], "lens"), "lens", at::kInt, B, index);
    args.prompt_lens = vector_or_none<int>(a[3], "prompt_lens", at::kInt, B, index);
    args.repetition = vector_or_none<float>(a[4], "repetition", at::kFloat, B, index);
    args.frequency = vector_or_none<float>(a[5], "frequency", at::kFloat, B, index);
    args.presence = vector_or_none<float>(a[6], "presence", at::kFloat, B, index);
    if (t.cols > kMost) refuse(PyExc_ValueError, "tokens must have fewer than 2**30 columns, got %d", t.cols);
    if (t.cols > 0) {
      args.tokens = t.p;
      args.ldt = t.ld;
      args.L = t.cols;
    }
  } else {
    for (int i = 2; i <= 6; ++i)
      if (a[i] != Py_None) refuse(PyExc_ValueError, "penalties and lengths come with tokens");
  }
  at::Tensor bias_ids, bias;
  if ((a[7] == Py_None) != (a[8] == Py_None)) refuse(PyExc_ValueError, "bias and bias_ids come together");
  if (a[7] != Py_None) {
    bias_ids = tensor(a[7], "bias_ids");
    bias = tensor(a[8], "bias");
    no_grad(bias, "bias");
    same_place(bias, "bias", index);
    matrix(bias_ids, "bias_ids", B, index);
    if (bias.scalar_type() != at::kFloat || bias.sizes() != bias_ids.sizes())
      refuse(PyExc_ValueError, "bias must be float32 and of bias_ids' shape");
    if (bias.strides() != bias_ids.strides()) {
      bias = bias.contiguous();
      bias_ids = bias_ids.contiguous();
    }
    const Matrix m = matrix(bias_ids, "bias_ids", B, index);
    args.bias_ids = m.p;
    args.bias = static_cast<const float*>(bias.data_ptr());
    args.ldb = m.ld;
    args.n_bias = m.cols;
    if (m.cols > kMost) refuse(PyExc_ValueError, "bias must have fewer than 2**30 columns, got %d", m.cols);
  }
  if (a[9] != Py_None) {
    const Matrix m = matrix(tensor(a[9], "mask"), "mask", -1, index);
    if (m.cols < (V + 31) / 32)
      refuse(PyExc_ValueError, "mask must have %lld words a row, got %d", static_cast<long long>((V + 31) / 32), m.cols);
    if (a[10] == Py_None && m.rows != B)
      refuse(PyExc_ValueError, "mask must have %lld rows, or come with mask_rows", static_cast<long long>(B));
    args.mask_rows = vector_or_none<int>(a[10], "mask_rows", at::kInt, B, index);
    if (m.rows > 0) {
      args.mask = m.p;
      args.ldm = m.ld;
      args.n_masks = m.rows;
    }
  } else if (a[10] != Py_None) {
    refuse(PyExc_ValueError, "mask_rows come with mask");
  }
  if (B > 0) {
    const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(index));
    call(nl_process_logits(&args, c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(index)).stream()),
         "nl_process_logits");
  }
  if (a[11] != Py_None) return Py_NewRef(a[11]);
  return THPVariable_Wrap(y);
}

// Runs an operator; no C++ exception leaves it.
template <PyObject* (*F)(PyObject* const*), int N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "expected %d arguments, got %zd", N, n);
    return nullptr;
  }
  try {
    return F(args);
  } catch (const Refusal& r) {
    if (r.type) PyErr_SetString(r.type, r.text.c_str());
  } catch (const c10::OutOfMemoryError& e) {
    PyObject* module = PyImport_ImportModule("torch");
    PyObject* type = module ? PyObject_GetAttrString(module, "OutOfMemoryError") : nullptr;
    Py_XDECREF(module);
    if (type) PyErr_SetString(type, e.what_without_backtrace());
    Py_XDECREF(type);
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
  }
  return nullptr;
}

#define NL_ENTRY(name, f, n) \
  {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(entry<f, n>)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {NL_ENTRY("paged_decode_attention", attention, 12), NL_ENTRY("paged_kv_write", kv_write, 7),
                         NL_ENTRY("update_block_tables", update_tables, 10), NL_ENTRY("process_logits", logits, 12),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef definition = {PyModuleDef_HEAD_INIT, "_ops", "Host side of the serving operators.", -1, methods,
                          nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__ops() { return PyModule_Create(&definition); }
