// Host side of the small MXFP4, int8, rotary and per-head norm calls: argument
// checks, output allocation and the launch in one native call.  A product of one
// row or the rotation of one token takes the GPU 3-6 us; checking the tensors and
// making the call from Python takes 7-13, from here 4-6.
//
// Every function does the usual case only and returns None for anything else
// (an unusual stride, a type or size that does not fit, a refusal of the entry
// point), all of it before any launch; the caller's Python path then does the
// work or raises.  Once something may have been launched, a status other than OK
// comes back as an int, which the caller raises: the call is never made twice (in
// place it would be applied twice).  No state is kept.
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <ATen/EmptyTensor.h>
#include <Python.h>
#include <c10/core/impl/LocalDispatchKeySet.h>

#include "../../include/ltx_hip.h"

namespace {

struct Entry {
  decltype(&ltx_gemm_mxfp4_bf16) gemm;
  decltype(&ltx_gemm_mxfp4_workspace_bytes) gemm_ws;
  decltype(&ltx_gemm_mx4_bf16) mx4;
  decltype(&ltx_gemm_mx4_workspace_bytes) mx4_ws;
  decltype(&ltx_quantize_mxfp4) quantize;
  decltype(&ltx_dequantize_mxfp4_bf16) dequantize;
  decltype(&ltx_rotary) rotary;
  decltype(&ltx_quantize_int8) quantize8;
  decltype(&ltx_dequantize_w8_bf16) dequantize8;
  decltype(&ltx_gemm_i8_bf16) gemm8;
  decltype(&ltx_gemm_i8_workspace_bytes) gemm8_ws;
  decltype(&ltx_headnorm_rotary) headnorm;
  decltype(&ltx_headnorm_rotary_grad) headnorm_grad;
  decltype(&ltx_headnorm_rotary_grad_workspace_bytes) headnorm_ws;
} entry = {};

PyObject* general() { Py_RETURN_NONE; }

// the tensor of an argument that is exactly one; null otherwise
const at::Tensor* tensor(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }
// (device -1: host tensors, for entry points that are no GPU's)
bool on(const at::Tensor& t, int64_t device) { return t.get_device() == device && (t.is_cuda() || device < 0); }

// what a function returns for the entry point's status: `result` (a new
// reference, null with an error set) if OK, None after a refusal, else the status
PyObject* outcome(int status, PyObject* result) {
  if (status == LTX_OK || !result) return result;
  Py_DECREF(result);
  if (status == LTX_ERR_INVALID_ARG || status == LTX_ERR_UNSUPPORTED || status == LTX_ERR_ALIGNMENT) return general();
  return PyLong_FromLong(status);
}
PyObject* pair(at::Tensor a, at::Tensor b) {
  PyObject* pa = a.defined() ? THPVariable_Wrap(std::move(a)) : (Py_INCREF(Py_None), Py_None);
  PyObject* pb = b.defined() ? THPVariable_Wrap(std::move(b)) : (Py_INCREF(Py_None), Py_None);
  PyObject* r = pa && pb ? PyTuple_Pack(2, pa, pb) : nullptr;
  Py_XDECREF(pa);
  Py_XDECREF(pb);
  return r;
}

// A new tensor on the device of `like`, which is the current one: from its allocator,
// without the dispatcher's way there (0.4 us less), unless someone wants to see it there
// (a dispatch mode, a tracer, a function transform: keys that the thread includes beyond
// the usual ones) or uninitialised memory is to be filled.
at::Tensor empty(at::IntArrayRef size, at::ScalarType type, const at::Tensor& like) {
  const auto& context = at::globalContext();
  const bool fill = context.deterministicAlgorithms() && context.deterministicFillUninitializedMemory();
  if (!like.is_cuda() || fill ||
      !(c10::impl::tls_local_dispatch_key_set().included_ - c10::default_included_set).empty())
    return at::empty(size, like.options().dtype(type));
  static at::Allocator* const allocator = at::empty({0}, like.options()).storage().allocator();
  return at::detail::empty_generic(size, allocator, c10::DispatchKeySet(c10::DispatchKey::CUDA), type, std::nullopt);
}

// The axes of more than one entry, by ascending stride (in bytes).  A dense tensor
// is one axis, whatever its shape (a bias may have any); others have up to 4.
struct Axes {
  int n = 0;
  int64_t stride[4], size[4], unit;
  explicit Axes(const at::Tensor& t) : unit(t.element_size()) {
    if (t.is_contiguous()) {
      n = 1;
      stride[0] = unit;
      size[0] = t.numel();
      return;
    }
    TORCH_CHECK(t.dim() <= 4);
    for (int64_t d = 0; d < t.dim(); ++d) {
      if (t.size(d) == 1) continue;
      int i = n++;
      for (; i > 0 && stride[i - 1] > t.stride(d) * unit; --i) stride[i] = stride[i - 1], size[i] = size[i - 1];
      stride[i] = t.stride(d) * unit;
      size[i] = t.size(d);
    }
  }
  // bytes from the first element to the end of the last, along strides below `period`
  int64_t extent(int64_t period = INT64_MAX) const {
    int64_t e = unit;
    for (int i = 0; i < n && stride[i] < period; ++i) e += stride[i] * (size[i] - 1);
    return e;
  }
  bool whole_periods(int64_t period) const {
    for (int i = 0; i < n; ++i)
      if (stride[i] > period && stride[i] % period) return false;
    return true;
  }
};

// whether no two indices name the same element
bool distinct(const at::Tensor& t) {
  const Axes x(t);
  int64_t end = x.unit;
  for (int i = 0; i < x.n; ++i) {
    if (x.stride[i] < end) return false;
    end += x.stride[i] * (x.size[i] - 1);
  }
  return true;
}

// whether the two (not empty) share no memory: apart, or with a stride in common
// within which they are apart (column ranges of one buffer's rows)
bool apart(const at::Tensor& a, const at::Tensor& b) {
  const Axes xa(a), xb(b);
  const int64_t gap = static_cast<const char*>(b.const_data_ptr()) - static_cast<const char*>(a.const_data_ptr());
  if (gap >= xa.extent() || -gap >= xb.extent()) return true;
  for (int i = 0; i < xa.n; ++i)
    for (int j = 0; j < xb.n; ++j) {
      const int64_t period = xa.stride[i];
      if (period == 0 || xb.stride[j] != period || !xa.whole_periods(period) || !xb.whole_periods(period)) continue;
      const int64_t d = (gap % period + period) % period;
      if (xa.extent(period) <= d && d + xb.extent(period) <= period) return true;
    }
  return false;
}

// whether index for index the two (of one shape) are the same memory
bool same_view(const at::Tensor& a, const at::Tensor& b) {
  if (a.const_data_ptr() != b.const_data_ptr()) return false;
  for (int64_t d = 0; d < a.dim(); ++d)
    if (a.size(d) != 1 && a.stride(d) != b.stride(d)) return false;
  return true;
}

// dense-column (rows, K / 2) codes with scale words that cover them
// (`ld`: their row stride; that of an axis of one entry says nothing)
bool mxfp4(const at::Tensor* codes, const at::Tensor* words, int64_t device, int64_t* rows, int64_t* k, int64_t* ld) {
  if (!codes || !words || codes->scalar_type() != at::kByte || words->scalar_type() != at::kInt || codes->dim() != 2 ||
      words->dim() != 2 || !on(*codes, device) || !on(*words, device))
    return false;
  *rows = codes->size(0);
  *k = codes->size(1) * 2;
  *ld = words->size(0) > 1 ? words->stride(0) : (words->size(1) + 3) / 4 * 4;
  return codes->stride(1) == 1 && words->stride(1) == 1 && codes->stride(0) >= codes->size(1) &&
         *ld >= words->size(1) && words->size(0) * 128 >= *k && words->size(1) >= *rows;
}

// whether the words' memory goes on to a multiple of 4 rows, as products read them
bool whole_words(const at::Tensor& words, int64_t rows, int64_t k, int64_t ld) {
  return rows % 4 == 0 || (words.storage_offset() + (k - 1) / 128 * ld + (rows + 3) / 4 * 4) * 4 <=
                              static_cast<int64_t>(words.storage().nbytes());
}

// Row strides of a product's residual (0 without one) and of its output, new (M, N) or
// `given`; false for what needs the general path.
bool outputs(const at::Tensor* res, const at::Tensor* gate, const at::Tensor* given, bool resid, int64_t M, int64_t N,
             int64_t device, std::initializer_list<const at::Tensor*> operands, int64_t* ldr, int64_t* ldc) {
  *ldr = 0;
  *ldc = N;
  if (resid) {
    if (!res || !gate || res->dim() != 2 || res->scalar_type() != at::kBFloat16 || res->size(0) != M ||
        res->size(1) != N || res->stride(1) != 1 || !on(*res, device) || gate->scalar_type() != at::kFloat ||
        gate->numel() != N || !gate->is_contiguous() || !on(*gate, device))
      return false;
    *ldr = M > 1 ? res->stride(0) : N;
    if (*ldr < N) return false;
  }
  if (given) {
    if (given->dim() != 2 || given->scalar_type() != at::kBFloat16 || given->size(0) != M || given->size(1) != N ||
        given->stride(1) != 1 || !on(*given, device) || (resid && !same_view(*given, *res) && !apart(*given, *res)))
      return false;
    for (const at::Tensor* t : operands)
      if (t && !apart(*given, *t)) return false;
    if (resid && !apart(*given, *gate)) return false;
    if (M > 1) *ldc = given->stride(0);
    if (*ldc < N) return false;
  }
  return true;
}

// linear(x, x_words or None, codes, words, bias or None, flags, epilogue, residual or None, gate or None,
//        sigmoid_from or -1, out or None, device, stream)
PyObject* linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 13 || !entry.gemm) return general();
  const at::Tensor *x = tensor(a[0]), *xs = tensor(a[1]), *w = tensor(a[2]), *ws = tensor(a[3]), *bias = tensor(a[4]),
                   *res = tensor(a[7]), *gate = tensor(a[8]), *given = tensor(a[10]);
  const int64_t flags = PyLong_AsLongLong(a[5]), epi = PyLong_AsLongLong(a[6]), sig = PyLong_AsLongLong(a[9]),
                device = PyLong_AsLongLong(a[11]);
  void* stream = PyLong_AsVoidPtr(a[12]);
  if (PyErr_Occurred()) return nullptr;
  int64_t N, K, M, kx, ldws, ldxs = 0;
  if (!x || (!xs && a[1] != Py_None) || (!bias && a[4] != Py_None) || (!given && a[10] != Py_None) ||
      !mxfp4(w, ws, device, &N, &K, &ldws))
    return general();
  if (xs) {
    if (!mxfp4(x, xs, device, &M, &kx, &ldxs) || !whole_words(*xs, M, kx, ldxs)) return general();
  } else {
    if (x->dim() != 2 || x->scalar_type() != at::kBFloat16 || !on(*x, device) || x->stride(1) != 1) return general();
    M = x->size(0);
    kx = x->size(1);
  }
  if (kx != K || M < 1 || K < 1 || N < 1) return general();
  const int64_t width = x->size(1), lda = M > 1 ? x->stride(0) : width;
  if (lda < width) return general();
  if (bias && (bias->scalar_type() != at::kFloat || bias->numel() != N || !bias->is_contiguous() || !on(*bias, device)))
    return general();
  const bool resid = epi == LTX_GEMM_EPI_RESIDUAL || epi == LTX_GEMM_EPI_RESIDUAL_ROUND;
  int64_t ldr, ldc;
  if (!outputs(res, gate, given, resid, M, N, device, {x, xs, w, ws, bias}, &ldr, &ldc)) return general();
  at::Tensor out = given ? *given : empty({M, N}, at::kBFloat16, *x);
  const int64_t bytes = xs ? entry.mx4_ws(M, N, K) : entry.gemm_ws(M, N, K);
  at::Tensor work;
  if (bytes > 0) work = empty({bytes}, at::kByte, *x);
  float* wp = bytes > 0 ? static_cast<float*>(work.data_ptr()) : nullptr;
  const float* bp = bias ? bias->const_data_ptr<float>() : nullptr;
  const int64_t ldw = N > 1 ? w->stride(0) : K / 2;
  const void* rp = resid ? res->const_data_ptr() : nullptr;
  const float* gp = resid ? gate->const_data_ptr<float>() : nullptr;
  const int64_t from = sig < 0 ? N : sig;
  const auto* wc = static_cast<const uint8_t*>(w->const_data_ptr());
  const auto* wsp = static_cast<const uint32_t*>(ws->const_data_ptr());
  PyObject* result = THPVariable_Wrap(out);  // (before the launch: it may fail)
  if (!result) return nullptr;
  const int st = xs ? entry.mx4(static_cast<const uint8_t*>(x->const_data_ptr()), lda,
                                static_cast<const uint32_t*>(xs->const_data_ptr()), ldxs, wc, ldw, wsp, ldws, bp,
                                out.data_ptr(), ldc, M, N, K, (int)(epi | flags), rp, ldr, gp, from, wp, bytes, stream)
                    : entry.gemm(x->const_data_ptr(), lda, wc, ldw, wsp, ldws, bp, out.data_ptr(), ldc, M, N, K,
                                 (int)(epi | flags), rp, ldr, gp, from, wp, bytes, stream);
  return outcome(st, result);
}

// quantize(x, device, stream) -> (codes, words)
PyObject* quantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 3 || !entry.quantize) return general();
  const at::Tensor* x = tensor(a[0]);
  const int64_t device = PyLong_AsLongLong(a[1]);
  void* stream = PyLong_AsVoidPtr(a[2]);
  if (PyErr_Occurred()) return nullptr;
  if (!x || x->dim() != 2 || !on(*x, device) || x->stride(1) != 1) return general();
  const auto type = x->scalar_type();
  const int dtype = type == at::kBFloat16 ? 0 : (type == at::kHalf ? 1 : (type == at::kFloat ? 2 : -1));
  const int64_t rows = x->size(0), k = x->size(1), ldx = rows > 1 ? x->stride(0) : k;
  if (dtype < 0 || rows < 1 || k < 32 || k % 32 || ldx < k) return general();
  const int64_t ld = (rows + 3) / 4 * 4;
  at::Tensor codes = empty({rows, k / 2}, at::kByte, *x), words = empty({(k + 127) / 128, ld}, at::kInt, *x);
  PyObject* result = pair(codes, words);
  if (!result) return nullptr;
  return outcome(entry.quantize(x->const_data_ptr(), dtype, ldx, rows, k, static_cast<uint8_t*>(codes.data_ptr()), k / 2,
                                static_cast<uint32_t*>(words.data_ptr()), ld, stream),
                 result);
}

// dequantize(codes, words, device, stream)
PyObject* dequantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 4 || !entry.dequantize) return general();
  const at::Tensor *codes = tensor(a[0]), *words = tensor(a[1]);
  const int64_t device = PyLong_AsLongLong(a[2]);
  void* stream = PyLong_AsVoidPtr(a[3]);
  if (PyErr_Occurred()) return nullptr;
  int64_t rows, k, ld;
  if (!mxfp4(codes, words, device, &rows, &k, &ld) || rows < 1 || k < 1) return general();
  at::Tensor out = empty({rows, k}, at::kBFloat16, *codes);
  PyObject* result = THPVariable_Wrap(out);
  if (!result) return nullptr;
  return outcome(entry.dequantize(static_cast<const uint8_t*>(codes->const_data_ptr()),
                                  rows > 1 ? codes->stride(0) : k / 2,
                                  static_cast<const uint32_t*>(words->const_data_ptr()), ld, rows, k,
                                  out.data_ptr(), k, stream),
                 result);
}

int float_type(const at::Tensor& t) {
  const auto type = t.scalar_type();
  return type == at::kBFloat16 ? 0 : (type == at::kHalf ? 1 : (type == at::kFloat ? 2 : -1));
}

// dense-column (rows, k) int8 codes with a scale for each row
bool int8(const at::Tensor* codes, const at::Tensor* scales, int64_t device, int64_t* rows, int64_t* k, int64_t* ld) {
  if (!codes || !scales || codes->scalar_type() != at::kChar || scales->scalar_type() != at::kFloat ||
      codes->dim() != 2 || scales->dim() != 1 || !on(*codes, device) || !on(*scales, device))
    return false;
  *rows = codes->size(0);
  *k = codes->size(1);
  *ld = *rows > 1 ? codes->stride(0) : *k;
  return *rows > 0 && *k > 0 && codes->stride(1) == 1 && *ld >= *k && scales->size(0) == *rows && scales->is_contiguous();
}

// quantize8(x, device, stream) -> (codes, scales)
PyObject* quantize8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 3 || !entry.quantize8) return general();
  const at::Tensor* x = tensor(a[0]);
  const int64_t device = PyLong_AsLongLong(a[1]);
  void* stream = PyLong_AsVoidPtr(a[2]);
  if (PyErr_Occurred()) return nullptr;
  if (!x || x->dim() != 2 || !on(*x, device) || x->stride(1) != 1) return general();
  const int dtype = float_type(*x);
  const int64_t rows = x->size(0), k = x->size(1), ldx = rows > 1 ? x->stride(0) : k;
  if (dtype < 0 || rows < 1 || k < 16 || k % 16 || ldx < k) return general();
  at::Tensor codes = empty({rows, k}, at::kChar, *x), scales = empty({rows}, at::kFloat, *x);
  PyObject* result = pair(codes, scales);
  if (!result) return nullptr;
  return outcome(entry.quantize8(x->const_data_ptr(), dtype, ldx, rows, k, static_cast<int8_t*>(codes.data_ptr()), k,
                                 static_cast<float*>(scales.data_ptr()), stream),
                 result);
}

// dequantize8(codes, scales, device, stream)
PyObject* dequantize8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 4 || !entry.dequantize8) return general();
  const at::Tensor *codes = tensor(a[0]), *scales = tensor(a[1]);
  const int64_t device = PyLong_AsLongLong(a[2]);
  void* stream = PyLong_AsVoidPtr(a[3]);
  if (PyErr_Occurred()) return nullptr;
  int64_t rows, k, ld;
  if (!int8(codes, scales, device, &rows, &k, &ld)) return general();
  at::Tensor out = empty({rows, k}, at::kBFloat16, *codes);
  PyObject* result = THPVariable_Wrap(out);
  if (!result) return nullptr;
  return outcome(entry.dequantize8(static_cast<const int8_t*>(codes->const_data_ptr()), ld,
                                   scales->const_data_ptr<float>(), rows, k, out.data_ptr(), k, stream),
                 result);
}

// linear8(codes, scales, weight codes, weight scales, bias or None, flags, epilogue, residual or None, gate or None,
//         sigmoid_from or -1, out or None, device, stream)
PyObject* linear8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 13 || !entry.gemm8) return general();
  const at::Tensor *x = tensor(a[0]), *xs = tensor(a[1]), *w = tensor(a[2]), *ws = tensor(a[3]), *bias = tensor(a[4]),
                   *res = tensor(a[7]), *gate = tensor(a[8]), *given = tensor(a[10]);
  const int64_t flags = PyLong_AsLongLong(a[5]), epi = PyLong_AsLongLong(a[6]), sig = PyLong_AsLongLong(a[9]),
                device = PyLong_AsLongLong(a[11]);
  void* stream = PyLong_AsVoidPtr(a[12]);
  if (PyErr_Occurred()) return nullptr;
  int64_t M, N, K, kx, lda, ldw;
  if ((!bias && a[4] != Py_None) || (!given && a[10] != Py_None) || !int8(w, ws, device, &N, &K, &ldw) ||
      !int8(x, xs, device, &M, &kx, &lda) || kx != K)
    return general();
  if (bias && (bias->scalar_type() != at::kFloat || bias->numel() != N || !bias->is_contiguous() || !on(*bias, device)))
    return general();
  const bool resid = epi == LTX_GEMM_EPI_RESIDUAL || epi == LTX_GEMM_EPI_RESIDUAL_ROUND;
  int64_t ldr, ldc;
  if (!outputs(res, gate, given, resid, M, N, device, {x, xs, w, ws, bias}, &ldr, &ldc)) return general();
  at::Tensor out = given ? *given : empty({M, N}, at::kBFloat16, *x);
  const int64_t bytes = entry.gemm8_ws(M, N, K);
  at::Tensor work;
  if (bytes > 0) work = empty({bytes}, at::kByte, *x);
  PyObject* result = THPVariable_Wrap(out);  // (before the launch: it may fail)
  if (!result) return nullptr;
  return outcome(entry.gemm8(static_cast<const int8_t*>(x->const_data_ptr()), lda, xs->const_data_ptr<float>(),
                             static_cast<const int8_t*>(w->const_data_ptr()), ldw, ws->const_data_ptr<float>(),
                             bias ? bias->const_data_ptr<float>() : nullptr, out.data_ptr(), ldc, M, N, K,
                             (int)(epi | flags), resid ? res->const_data_ptr() : nullptr, ldr,
                             resid ? gate->const_data_ptr<float>() : nullptr, sig < 0 ? N : sig,
                             bytes > 0 ? work.data_ptr() : nullptr, bytes, stream),
                 result);
}

// one side of a rotation
bool side(const at::Tensor& x, const at::Tensor& out, ltx_rotary_rows* r) {
  const int b = x.dim() == 4 ? 1 : 0;
  if (x.stride(b + 2) != 1 || out.stride(b + 2) != 1) return false;
  *r = {x.const_data_ptr(), b ? x.stride(0) : 0, x.stride(b), x.stride(b + 1),
        out.data_ptr(),     b ? out.stride(0) : 0, out.stride(b), out.stride(b + 1), x.size(b + 1)};
  return true;
}

// an output that the caller gave for x
bool fits(const at::Tensor& out, const at::Tensor& x, const at::Tensor* other, const at::Tensor& pos,
          const at::Tensor& inv) {
  return out.scalar_type() == x.scalar_type() && out.sizes() == x.sizes() && out.device() == x.device() &&
         distinct(out) && (same_view(out, x) || apart(out, x)) && (!other || apart(out, *other)) &&
         apart(out, pos) && apart(out, inv);
}

// rotary(q, k or None, positions, inv_freq, flags, factor, q' or None, k' or None, device, stream) -> (q', k' or None)
PyObject* rotary(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 10 || !entry.rotary) return general();
  const at::Tensor *q = tensor(a[0]), *k = tensor(a[1]), *pos = tensor(a[2]), *inv = tensor(a[3]), *gq = tensor(a[6]),
                   *gk = tensor(a[7]);
  const int64_t flags = PyLong_AsLongLong(a[4]), device = PyLong_AsLongLong(a[8]);
  const double factor = PyFloat_AsDouble(a[5]);
  void* stream = PyLong_AsVoidPtr(a[9]);
  if (PyErr_Occurred()) return nullptr;
  if (!q || (!k && a[1] != Py_None) || !pos || !inv || (q->dim() != 3 && q->dim() != 4) ||
      (!gq && a[6] != Py_None) || (!gk && a[7] != Py_None) || (gk && !k))
    return general();
  const int64_t dims = q->dim(), batch = dims == 4 ? q->size(0) : 1, tokens = q->size(dims - 3), dh = q->size(dims - 1);
  const auto type = q->scalar_type(), ptype = pos->scalar_type();
  const int dtype = type == at::kBFloat16 ? 0 : (type == at::kHalf ? 1 : (type == at::kFloat ? 2 : -1));
  const int pos_type = ptype == at::kInt ? 0 : (ptype == at::kLong ? 1 : (ptype == at::kFloat ? 2 : (ptype == at::kDouble ? 3 : -1)));
  if (dtype < 0 || pos_type < 0 || batch < 1 || tokens < 1 || q->size(dims - 2) < 1 || !on(*q, device) ||
      !on(*pos, device) || !on(*inv, device) || inv->scalar_type() != at::kDouble || inv->dim() != 1 ||
      !inv->is_contiguous() || !pos->is_contiguous())
    return general();
  const bool own = pos->dim() == 2;
  if ((own && (pos->size(0) != batch || pos->size(1) != tokens)) || (!own && (pos->dim() != 1 || pos->size(0) != tokens)))
    return general();
  const int64_t d = 2 * inv->numel();
  if (d < 2 || d > dh) return general();
  if (k && (k->dim() != dims || k->scalar_type() != type || !on(*k, device) || k->size(dims - 1) != dh ||
            k->size(dims - 3) != tokens || (dims == 4 && k->size(0) != batch) || k->size(dims - 2) < 1))
    return general();
  if ((gq && !fits(*gq, *q, k, *pos, *inv)) || (gk && !fits(*gk, *k, q, *pos, *inv)) || (gq && gk && !apart(*gq, *gk)))
    return general();
  at::Tensor oq = gq ? *gq : empty(q->sizes(), type, *q), ok;
  if (k) ok = gk ? *gk : empty(k->sizes(), type, *k);
  ltx_rotary_rows rq, rk;
  if (!side(*q, oq, &rq) || (k && !side(*k, ok, &rk))) return general();
  PyObject* result = pair(oq, ok);
  if (!result) return nullptr;
  return outcome(entry.rotary(&rq, k ? &rk : nullptr, dtype, batch, tokens, dh, d, pos->const_data_ptr(), pos_type,
                              own ? tokens : 0, inv->const_data_ptr<double>(), factor, (int)flags, stream),
                 result);
}

// One side of the per-head norm (g, dw: of its gradient) and its output, new or `given`; false
// for what needs the general path.
bool head_side(const at::Tensor& x, const at::Tensor* g, const at::Tensor* w, const at::Tensor* given, int64_t device,
               at::Tensor* out, at::Tensor* dw, ltx_headnorm_rows* r) {
  const int b = x.dim() == 4 ? 1 : 0;
  const int64_t dh = x.size(b + 2);
  if (!on(x, device) || x.stride(b + 2) != 1 || x.size(b + 1) < 1) return false;
  if (w && (w->scalar_type() != at::kFloat || w->dim() != 1 || w->size(0) != dh || !w->is_contiguous() || !on(*w, device)))
    return false;
  if (g && (g->scalar_type() != x.scalar_type() || g->sizes() != x.sizes() || g->stride(b + 2) != 1 || !on(*g, device)))
    return false;
  if (given && (given->scalar_type() != x.scalar_type() || given->sizes() != x.sizes() || given->stride(b + 2) != 1 ||
                !on(*given, device) || !distinct(*given)))
    return false;
  *out = given ? *given : empty(x.sizes(), x.scalar_type(), x);
  if (g && w) *dw = empty({dh}, at::kFloat, x);
  auto batch = [&](const at::Tensor& t) { return b ? t.stride(0) : 0; };
  *r = {x.const_data_ptr(), batch(x), x.stride(b), x.stride(b + 1),
        out->data_ptr(), batch(*out), out->stride(b), out->stride(b + 1),
        g ? g->const_data_ptr() : nullptr, g ? batch(*g) : 0, g ? g->stride(b) : 0, g ? g->stride(b + 1) : 0,
        w ? w->const_data_ptr<float>() : nullptr, dw->defined() ? static_cast<float*>(dw->data_ptr()) : nullptr,
        x.size(b + 1)};
  return true;
}

// [gq, gk or None,] q, k or None, wq or None, wk or None, positions, inv_freq, flags, factor, eps, weight_offset,
// q' or None, k' or None, device, stream -> (q', k' or None) or (dq, dk or None, dwq or None, dwk or None)
template <bool GRAD>
PyObject* head_call(PyObject* const* a, Py_ssize_t n) {
  constexpr int G = GRAD ? 2 : 0;
  if (n != 14 + G || !(GRAD ? (void*)entry.headnorm_grad : (void*)entry.headnorm)) return general();
  const at::Tensor *gq = GRAD ? tensor(a[0]) : nullptr, *gk = GRAD ? tensor(a[1]) : nullptr;
  a += G;
  const at::Tensor *q = tensor(a[0]), *k = tensor(a[1]), *wq = tensor(a[2]), *wk = tensor(a[3]), *pos = tensor(a[4]),
                   *inv = tensor(a[5]), *oq = tensor(a[10]), *ok = tensor(a[11]);
  const int64_t flags = PyLong_AsLongLong(a[6]), device = PyLong_AsLongLong(a[12]);
  const double factor = PyFloat_AsDouble(a[7]), eps = PyFloat_AsDouble(a[8]), offset = PyFloat_AsDouble(a[9]);
  void* stream = PyLong_AsVoidPtr(a[13]);
  if (PyErr_Occurred()) return nullptr;
  auto odd = [&](int i, const at::Tensor* t) { return !t && a[i] != Py_None; };
  if (!q || odd(1, k) || odd(2, wq) || odd(3, wk) || odd(10, oq) || odd(11, ok) || !pos || !inv ||
      (q->dim() != 3 && q->dim() != 4) || (!k && (wk || gk || ok)) || (GRAD && (!gq || (k && !gk))))
    return general();
  const int64_t dims = q->dim(), batch = dims == 4 ? q->size(0) : 1, tokens = q->size(dims - 3), dh = q->size(dims - 1);
  const int dtype = float_type(*q);
  const auto ptype = pos->scalar_type();
  const int pos_type = ptype == at::kInt ? 0 : (ptype == at::kLong ? 1 : (ptype == at::kFloat ? 2 : (ptype == at::kDouble ? 3 : -1)));
  if (dtype < 0 || pos_type < 0 || batch < 1 || tokens < 1 || !on(*pos, device) || !on(*inv, device) ||
      inv->scalar_type() != at::kDouble || inv->dim() != 1 || !inv->is_contiguous() || !pos->is_contiguous())
    return general();
  const bool own = pos->dim() == 2;
  if ((own && (pos->size(0) != batch || pos->size(1) != tokens)) || (!own && (pos->dim() != 1 || pos->size(0) != tokens)))
    return general();
  const int64_t d = 2 * inv->numel();
  if (d < 2 || d > dh) return general();
  if (k && (k->dim() != dims || k->scalar_type() != q->scalar_type() || k->size(dims - 1) != dh ||
            k->size(dims - 3) != tokens || (dims == 4 && k->size(0) != batch)))
    return general();
  at::Tensor out[2], dw[2], work;
  ltx_headnorm_rows rows[2];
  if (!head_side(*q, gq, wq, oq, device, &out[0], &dw[0], &rows[0]) ||
      (k && !head_side(*k, gk, wk, ok, device, &out[1], &dw[1], &rows[1])))
    return general();
  // an output may be its own input (or gradient), and keeps off everything else
  auto fits8 = [&](const at::Tensor* mine, std::initializer_list<const at::Tensor*> own_ones,
                   std::initializer_list<const at::Tensor*> others) {
    if (!mine) return true;
    for (const at::Tensor* t : own_ones)
      if (t && !same_view(*mine, *t) && !apart(*mine, *t)) return false;
    for (const at::Tensor* t : others)
      if (t && !apart(*mine, *t)) return false;
    return true;
  };
  if (!fits8(oq, {q, gq}, {k, gk, ok, wq, wk, pos, inv}) || !fits8(ok, {k, gk}, {q, gq, oq, wq, wk, pos, inv}))
    return general();
  const bool sums = dw[0].defined() || dw[1].defined();
  const int64_t bytes = sums ? entry.headnorm_ws(dh) : 0;
  if (sums) work = empty({bytes}, at::kByte, *q);
  PyObject* result = pair(out[0], out[1]);
  if (result && GRAD) {
    PyObject* both = pair(dw[0], dw[1]);
    PyObject* four = both ? PySequence_Concat(result, both) : nullptr;
    Py_XDECREF(both);
    Py_DECREF(result);
    result = four;
  }
  if (!result) return nullptr;
  const int64_t pos_batch = own ? tokens : 0;
  const double* freq = inv->const_data_ptr<double>();
  if constexpr (GRAD)
    return outcome(entry.headnorm_grad(&rows[0], k ? &rows[1] : nullptr, dtype, batch, tokens, dh, d,
                                       pos->const_data_ptr(), pos_type, pos_batch, freq, factor, eps, offset, (int)flags,
                                       sums ? static_cast<float*>(work.data_ptr()) : nullptr, bytes, stream),
                   result);
  else
    return outcome(entry.headnorm(&rows[0], k ? &rows[1] : nullptr, dtype, batch, tokens, dh, d, pos->const_data_ptr(),
                                  pos_type, pos_batch, freq, factor, eps, offset, (int)flags, stream),
                   result);
}
PyObject* headnorm(PyObject*, PyObject* const* a, Py_ssize_t n) { return head_call<false>(a, n); }
PyObject* headnorm_grad(PyObject*, PyObject* const* a, Py_ssize_t n) { return head_call<true>(a, n); }

// a C++ exception (no memory for an output; nothing throws after a launch)
template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyObject* guarded(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  try {
    return F(self, a, n);
  } catch (...) {
    return general();  // the Python path meets the same condition and raises torch's error for it
  }
}

// bind(addresses of the entry points, in the order of Entry)
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  void** slots[] = {(void**)&entry.gemm,       (void**)&entry.gemm_ws,       (void**)&entry.mx4,
                    (void**)&entry.mx4_ws,     (void**)&entry.quantize,      (void**)&entry.dequantize,
                    (void**)&entry.rotary,     (void**)&entry.quantize8,     (void**)&entry.dequantize8,
                    (void**)&entry.gemm8,      (void**)&entry.gemm8_ws,      (void**)&entry.headnorm,
                    (void**)&entry.headnorm_grad, (void**)&entry.headnorm_ws};
  constexpr int kSlots = sizeof(slots) / sizeof(slots[0]);
  if (n != kSlots) {
    PyErr_Format(PyExc_TypeError, "bind takes %d addresses", kSlots);
    return nullptr;
  }
  for (int i = 0; i < kSlots; ++i) *slots[i] = PyLong_AsVoidPtr(a[i]);
  if (PyErr_Occurred()) return nullptr;
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"bind", (PyCFunction)(void (*)())bind, METH_FASTCALL, "entry point addresses"},
    {"linear", (PyCFunction)(void (*)())guarded<linear>, METH_FASTCALL, "an MXFP4 product, or None"},
    {"quantize", (PyCFunction)(void (*)())guarded<quantize>, METH_FASTCALL, "rows to MXFP4, or None"},
    {"dequantize", (PyCFunction)(void (*)())guarded<dequantize>, METH_FASTCALL, "MXFP4 rows to bf16, or None"},
    {"rotary", (PyCFunction)(void (*)())guarded<rotary>, METH_FASTCALL, "rotary positions, or None"},
    {"quantize8", (PyCFunction)(void (*)())guarded<quantize8>, METH_FASTCALL, "rows to int8, or None"},
    {"dequantize8", (PyCFunction)(void (*)())guarded<dequantize8>, METH_FASTCALL, "int8 rows to bf16, or None"},
    {"linear8", (PyCFunction)(void (*)())guarded<linear8>, METH_FASTCALL, "an int8 product, or None"},
    {"headnorm", (PyCFunction)(void (*)())guarded<headnorm>, METH_FASTCALL, "per-head norm and rotation, or None"},
    {"headnorm_grad", (PyCFunction)(void (*)())guarded<headnorm_grad>, METH_FASTCALL, "its gradients, or None"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// (BUILT_FOR: the build's torch and Python, whose ABI this is)
PyMODINIT_FUNC PyInit__calls() {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "BUILT_FOR", LTX_CALLS_BUILT_FOR) < 0) Py_CLEAR(m);
  return m;
}
