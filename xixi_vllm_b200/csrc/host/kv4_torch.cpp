// Calls of the 4-bit cache kernels from Python without the interpreter's share of a launch: argument checks, output and
// workspace allocation, stream lookup and the C call of one operator are one C function. Driven from Python through ctypes
// the same work took 12 to 14 us a call, most of a small operator's time; here it takes about 5, of which the launch is 3.
//
// The kernels stay behind the C ABI of _xv_cuda.so: bind() receives its entry points' addresses, so this module links
// against torch and the Python C API only. No C++ exception leaves a function: each becomes the Python error it stands for.

#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <string>
#include <vector>

#include "xv_cuda.h"

namespace {

struct Entry {
  decltype(&xv_kv4_write) write;
  decltype(&xv_kv4_read) read;
  decltype(&xv_kv4_decode_splits) decode_splits;
  decltype(&xv_kv4_decode_workspace_bytes) decode_bytes;
  decltype(&xv_kv4_decode) decode;
  decltype(&xv_kv4_prefill_splits) prefill_splits;
  decltype(&xv_kv4_prefill_workspace_bytes) prefill_bytes;
  decltype(&xv_kv4_prefill) prefill;
} fn;
bool bound = false;

struct Refused {
  PyObject* type;
  std::string text;
};

[[noreturn]] void refuse(PyObject* type, const char* format, ...) {
  char text[512];
  va_list args;
  va_start(args, format);
  std::vsnprintf(text, sizeof text, format, args);
  va_end(args);
  throw Refused{type, text};
}

std::string shape_of(const at::Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + ")";
}

const at::Tensor& tensor(PyObject* o, const char* what) {
  if (!THPVariable_Check(o)) refuse(PyExc_TypeError, "%s must be a tensor, got %s", what, Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}

int integer(PyObject* o, const char* what) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Refused{nullptr, ""};
  if (v < INT32_MIN || v > INT32_MAX) refuse(PyExc_ValueError, "%s = %lld does not fit 32 bits", what, v);
  return static_cast<int>(v);
}

double real(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Refused{nullptr, ""};
  return v;
}

void bf16(const at::Tensor& t) {
  if (t.scalar_type() != at::kBFloat16) refuse(PyExc_TypeError, "GPU kernels take bfloat16 tensors, got %s", at::toString(t.scalar_type()));
}

// At least n contiguous elements of a type on the caches' device.
void* vector(const at::Tensor& t, int64_t n, at::ScalarType type, const at::Device& dev, const char* what) {
  if (t.scalar_type() != type || t.device() != dev || !t.is_contiguous() || t.numel() < n)
    refuse(PyExc_ValueError, "%s: needs %lld contiguous %s values on %s, got %s %s on %s", what, static_cast<long long>(n),
           at::toString(type), dev.str().c_str(), shape_of(t).c_str(), at::toString(t.scalar_type()), t.device().str().c_str());
  return t.data_ptr();
}

struct Caches {
  const at::Tensor &k, &v;
  at::Device dev;
  int blocks, heads, page;

  Caches(PyObject* k_, PyObject* v_, int head_dim, int heads_) : k(tensor(k_, "k_cache")), v(tensor(v_, "v_cache")), dev(k.device()) {
    if (k.scalar_type() != at::kByte || v.scalar_type() != at::kByte)
      refuse(PyExc_TypeError, "a 4-bit cache is a pair of uint8 tensors, got %s and %s", at::toString(k.scalar_type()),
             at::toString(v.scalar_type()));
    if (k.dim() != 4 || v.sizes() != k.sizes() || v.device() != dev)
      refuse(PyExc_ValueError, "4-bit caches need one 4-d shape and device, got %s on %s and %s on %s", shape_of(k).c_str(),
             dev.str().c_str(), shape_of(v).c_str(), v.device().str().c_str());
    if (!dev.is_cuda()) refuse(PyExc_ValueError, "4-bit caches are on %s", dev.str().c_str());
    if (head_dim != 128) refuse(PyExc_ValueError, "4-bit caches on the GPU need head_dim 128, got %d", head_dim);
    const int64_t page_ = k.size(2);
    if (page_ <= 0 || page_ % 16 || k.size(3) != head_dim / 2 + 8 || (heads_ >= 0 && k.size(1) != heads_) || k.size(1) < 1 ||
        k.size(0) * page_ > INT32_MAX || k.size(1) > INT32_MAX)
      refuse(PyExc_ValueError, "4-bit cache of shape %s: expected [blocks, %s, a multiple of 16, %d] for head_dim %d, below 2^31 tokens",
             shape_of(k).c_str(), heads_ >= 0 ? std::to_string(heads_).c_str() : "kv_heads", head_dim / 2 + 8, head_dim);
    if (!k.is_contiguous() || !v.is_contiguous()) refuse(PyExc_ValueError, "4-bit caches must be contiguous");
    blocks = static_cast<int>(k.size(0));
    heads = static_cast<int>(k.size(1));
    page = static_cast<int>(page_);
  }
};

void check(int rc, const char* what) {
  static const char* const reasons[] = {"bad shape", "misaligned pointer or stride", "workspace too small",
                                        "driver entry point missing", "tensor map encode failed", "launch failed",
                                        "unsupported configuration"};
  if (rc) refuse(PyExc_RuntimeError, "%s: %s", what, rc <= -1 && rc >= -7 ? reasons[-rc - 1] : std::to_string(rc).c_str());
}

template <typename F>
PyObject* guarded(Py_ssize_t n, Py_ssize_t want, F f) {
  try {
    if (n != want) refuse(PyExc_TypeError, "%zd arguments, expected %zd", n, want);
    if (!bound) refuse(PyExc_RuntimeError, "the kernel library's entry points are not bound");
    return f();
  } catch (const Refused& r) {
    if (r.type) PyErr_SetString(r.type, r.text.c_str());
  } catch (...) {
    torch::translate_exception_to_python(std::current_exception());      // out of memory keeps torch's own type
  }
  return nullptr;
}

// An uninitialised tensor, from torch's allocator without the dispatcher (0.3 us a tensor); the current device is `dev`.
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const at::Device& dev) {
  return at::Tensor(at::detail::empty_cuda(sizes, type, dev, std::nullopt));
}

// write(qkv | None, planes | None, splits, rows, q_w, k_w, eps, cos_sin, positions, slots, k_cache, v_cache, hq, hkv, d,
//       num_sms, status) -> q
PyObject* write(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 17, [&]() -> PyObject* {
    const int hq = integer(a[12], "num_q_heads"), hkv = integer(a[13], "num_kv_heads"), d = integer(a[14], "head_dim");
    const Caches c(a[10], a[11], d, hkv);
    if (hq < 0) refuse(PyExc_ValueError, "num_q_heads = %d", hq);
    const int64_t cols = (static_cast<int64_t>(hq) + 2ll * hkv) * d;
    const void* qkv = nullptr;
    const float* planes = nullptr;
    int64_t rows = integer(a[3], "rows");
    const int splits = integer(a[2], "splits");
    if (a[0] != Py_None) {
      const at::Tensor& x = tensor(a[0], "qkv");
      if (x.dim() != 2 || x.size(1) != cols || x.device() != c.dev)
        refuse(PyExc_ValueError, "qk_norm_rope_cache: qkv must be [T, %lld] on %s, got %s on %s", static_cast<long long>(cols),
               c.dev.str().c_str(), shape_of(x).c_str(), x.device().str().c_str());
      bf16(x);
      if (!x.is_contiguous()) refuse(PyExc_ValueError, "qk_norm_rope_cache needs contiguous qkv and cache tensors");
      rows = x.size(0);
      qkv = x.data_ptr();
    } else {
      planes = static_cast<const float*>(vector(tensor(a[1], "planes"), splits * rows * cols * 4, at::kByte, c.dev, "planes"));
    }
    if (rows > INT32_MAX) refuse(PyExc_ValueError, "%lld rows", static_cast<long long>(rows));
    const at::Tensor &qw = tensor(a[4], "q_w"), &kw = tensor(a[5], "k_w"), &cs = tensor(a[7], "cos_sin");
    bf16(qw);
    bf16(kw);
    const double eps = real(a[6]);
    const void* qwp = vector(qw, d, at::kBFloat16, c.dev, "q_w");
    const void* kwp = vector(kw, d, at::kBFloat16, c.dev, "k_w");
    const auto* csp = static_cast<const float*>(vector(cs, d, at::kFloat, c.dev, "cos_sin"));
    const auto* pos = static_cast<const int*>(vector(tensor(a[8], "positions"), rows, at::kInt, c.dev, "positions"));
    const auto* slots = static_cast<const int*>(vector(tensor(a[9], "slots"), rows, at::kInt, c.dev, "slots"));
    auto* status = static_cast<int*>(vector(tensor(a[16], "status"), 1, at::kInt, c.dev, "status"));
    const c10::cuda::OptionalCUDAGuard guard(c.dev);
    at::Tensor q = fresh({rows, static_cast<int64_t>(hq) * d}, at::kBFloat16, c.dev);
    if (rows > 0)
      check(fn.write(qkv, planes, splits, rows * cols, qwp, kwp, eps, csp, static_cast<int>(cs.numel() / d), pos, slots, q.data_ptr(),
                     c.k.data_ptr(), c.v.data_ptr(), static_cast<int>(rows), hq, hkv, d, c.page, c.blocks,
                     integer(a[15], "num_sms"), status, c10::cuda::getCurrentCUDAStream(c.dev.index()).stream()),
            "kv4_write");
    return THPVariable_Wrap(std::move(q));
  });
}

// read(k_cache, v_cache, slots, d, status) -> (k, v)
PyObject* read(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 5, [&]() -> PyObject* {
    const int d = integer(a[3], "head_dim");
    const Caches c(a[0], a[1], d, -1);
    const at::Tensor& s = tensor(a[2], "slots");
    const int64_t rows = s.numel();
    if (rows > INT32_MAX) refuse(PyExc_ValueError, "%lld slots", static_cast<long long>(rows));
    const auto* slots = static_cast<const int*>(vector(s, rows, at::kInt, c.dev, "slots"));
    auto* status = static_cast<int*>(vector(tensor(a[4], "status"), 1, at::kInt, c.dev, "status"));
    const c10::cuda::OptionalCUDAGuard guard(c.dev);
    at::Tensor k = fresh({rows, c.heads, d}, at::kBFloat16, c.dev), v = fresh({rows, c.heads, d}, at::kBFloat16, c.dev);
    if (rows > 0)
      check(fn.read(c.k.data_ptr(), c.v.data_ptr(), slots, k.data_ptr(), v.data_ptr(), static_cast<int>(rows), c.heads, d, c.page,
                    c.blocks, status, c10::cuda::getCurrentCUDAStream(c.dev.index()).stream()),
            "kv4_read");
    PyObject *ko = THPVariable_Wrap(std::move(k)), *vo = ko ? THPVariable_Wrap(std::move(v)) : nullptr;
    PyObject* pair = vo ? PyTuple_Pack(2, ko, vo) : nullptr;
    Py_XDECREF(ko);
    Py_XDECREF(vo);
    return pair;
  });
}

// attention(q, k_cache, v_cache, cu_q, kv_lens, block_tables, num_seqs, num_decode, max_q_len, scale, hq, hkv, d, num_sms,
//           status) -> out
PyObject* attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 15, [&]() -> PyObject* {
    const int hq = integer(a[10], "num_q_heads"), hkv = integer(a[11], "num_kv_heads"), d = integer(a[12], "head_dim");
    const Caches c(a[1], a[2], d, hkv);
    const at::Tensor &q = tensor(a[0], "q"), &bt = tensor(a[5], "block_tables"), &lens = tensor(a[4], "kv_lens");
    bf16(q);
    if (q.dim() != 2 || q.size(1) != static_cast<int64_t>(hq) * d || !q.is_contiguous() || q.device() != c.dev)
      refuse(PyExc_ValueError, "paged_attention: q must be a contiguous [T, %lld] tensor on %s, got %s on %s",
             static_cast<long long>(hq) * d, c.dev.str().c_str(), shape_of(q).c_str(), q.device().str().c_str());
    if (hq <= 0 || hq % hkv || hq / hkv > 16)
      refuse(PyExc_ValueError, "paged_attention: %d query heads over %d KV heads (at most 16 to one)", hq, hkv);
    const int B = integer(a[6], "num_seqs"), nd = integer(a[7], "num_decode"), most = integer(a[8], "max_q_len");
    const int np = B - nd;
    const int64_t T = q.size(0);
    if (most < 0) refuse(PyExc_ValueError, "paged_attention: max_q_len = %d", most);
    const int mq = static_cast<int>(std::min<int64_t>(most, T));       // no chunk has more rows than q
    if (nd < 0 || np < 0 || nd > T || T > INT32_MAX || bt.dim() != 2 || bt.size(0) < B || bt.size(1) > INT32_MAX)
      refuse(PyExc_ValueError, "paged_attention: %d decode rows and %d chunks for %lld query rows and a block table of %s", nd, np,
             static_cast<long long>(T), shape_of(bt).c_str());
    if (B > 65535) refuse(PyExc_ValueError, "paged_attention: at most 65535 sequences, got %d", B);
    const int maxb = static_cast<int>(bt.size(1));
    const int64_t reach = static_cast<int64_t>(maxb) * c.page;          // tokens that a block-table row can name
    if (reach > INT32_MAX)
      refuse(PyExc_ValueError, "paged_attention: block tables of %d pages name 2^31 tokens or more", maxb);
    const auto* tables = static_cast<const int*>(vector(bt, static_cast<int64_t>(B) * maxb, at::kInt, c.dev, "block_tables"));
    const auto* kv_lens = static_cast<const int*>(vector(lens, B, at::kInt, c.dev, "kv_lens"));
    const int* cu_q = np > 0 ? static_cast<const int*>(vector(tensor(a[3], "cu_q"), B + 1, at::kInt, c.dev, "cu_q")) : nullptr;
    const float scale = static_cast<float>(real(a[9]));
    if (!std::isfinite(scale)) refuse(PyExc_ValueError, "paged_attention: scale must be finite");
    const int sms = integer(a[13], "num_sms");
    auto* status = static_cast<int*>(vector(tensor(a[14], "status"), 1, at::kInt, c.dev, "status"));
    const c10::cuda::OptionalCUDAGuard guard(c.dev);
    at::Tensor out = fresh({T, q.size(1)}, at::kBFloat16, c.dev);
    if (T == 0 || maxb == 0 || c.blocks == 0) {                         // nothing is cached: every row is empty
      out.zero_();
      return THPVariable_Wrap(std::move(out));
    }
    // Rows that are behind the last sequence however long the chunks are; the chunk kernel clears what else there is.
    const int64_t used = std::min(T, nd + static_cast<int64_t>(np) * mq);
    if (used < T) out.narrow(0, used, T - used).zero_();
    const auto stream = c10::cuda::getCurrentCUDAStream(c.dev.index()).stream();
    // Workspaces come from torch's allocator, call by call: calls on two streams, or two captured graphs, never share one.
    if (nd > 0) {
      const int splits = fn.decode_splits(nd, hkv, sms, static_cast<int>(reach));
      const long long need = fn.decode_bytes(nd, hq, hkv, splits, sms);
      at::Tensor ws;
      if (need > 0) ws = fresh({need}, at::kByte, c.dev);
      check(fn.decode(q.data_ptr(), c.k.data_ptr(), c.v.data_ptr(), tables, kv_lens, out.data_ptr(), nd, hq, hkv, d, c.page, maxb,
                      c.blocks, scale, splits, sms, need > 0 ? ws.data_ptr() : nullptr, need, status, stream),
            "kv4_decode");
    }
    if (np > 0) {
      const int splits = fn.prefill_splits(np, mq, hq, hkv, static_cast<int>(reach), sms);
      const long long need = fn.prefill_bytes(np, mq, hq, hkv, splits);
      at::Tensor ws;
      if (need > 0) ws = fresh({need}, at::kByte, c.dev);
      check(fn.prefill(q.data_ptr(), c.k.data_ptr(), c.v.data_ptr(), tables, cu_q, kv_lens, out.data_ptr(), nd, np, mq,
                       static_cast<int>(T), static_cast<int>(used), hq, hkv, d, c.page, maxb, c.blocks, scale, splits, need > 0 ? ws.data_ptr() : nullptr, need,
                       status, stream),
            "kv4_prefill");
    }
    return THPVariable_Wrap(std::move(out));
  });
}

// bind(addresses of the eight entry points, in Entry's order)
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  void* at[8];
  if (n != 8) {
    PyErr_SetString(PyExc_TypeError, "eight addresses");
    return nullptr;
  }
  for (int i = 0; i < 8; ++i) {
    at[i] = PyLong_AsVoidPtr(a[i]);
    if (!at[i]) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "null address");
      return nullptr;
    }
  }
  fn.write = reinterpret_cast<decltype(fn.write)>(at[0]);
  fn.read = reinterpret_cast<decltype(fn.read)>(at[1]);
  fn.decode_splits = reinterpret_cast<decltype(fn.decode_splits)>(at[2]);
  fn.decode_bytes = reinterpret_cast<decltype(fn.decode_bytes)>(at[3]);
  fn.decode = reinterpret_cast<decltype(fn.decode)>(at[4]);
  fn.prefill_splits = reinterpret_cast<decltype(fn.prefill_splits)>(at[5]);
  fn.prefill_bytes = reinterpret_cast<decltype(fn.prefill_bytes)>(at[6]);
  fn.prefill = reinterpret_cast<decltype(fn.prefill)>(at[7]);
  bound = true;
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(bind)), METH_FASTCALL, nullptr},
    {"write", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(write)), METH_FASTCALL, nullptr},
    {"read", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(read)), METH_FASTCALL, nullptr},
    {"attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(attention)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_xv_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__xv_torch(void) {
  PyObject* m = PyModule_Create(&module);
  // The torch and Python that this was compiled against; ops/build.py looks for the text before it loads the file.
  if (m && PyModule_AddStringConstant(m, "built_for", XV_BUILT_FOR) < 0) Py_CLEAR(m);
  return m;
}
