// Host side of the launches, native: a CPython module (`_b200_host.so`) that `ops/_lib.py` and `ops/kernels.py` use when it is there.
//
//   bind(table, last_error, fallback)   name -> (address, argument codes) of the launchers of the kernel library
//   call(name, *args)                   converts the arguments by their codes, calls the launcher with the GIL released and raises
//                                       RuntimeError on a code other than 0
//   gemm(...)                           ops.kernels.gemm for CUDA operands that need no copy: checks, output, split workspace, launch
//   quant_mxfp4, dequant_mx, norm_mx, gemm_mxfp4, gated_fwd, gated_down, gated_bwd   the same for ops.mxfp4, ops.norm_mx and the gated block
//
// ctypes converts twenty arguments through as many Python objects and calls: 5 of the 20 us a launch of a small model took.  With
// it, the native GEMM operator and no autograd nodes where no gradient is wanted: a step of a two-layer model of width 512 2020 ->
// 1625 us, sampling with one double and two single MMDiT blocks 1668 -> 1012 us.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <string>
#include <unordered_map>

namespace {

constexpr int MAX_INTS = 40, MAX_FLOATS = 8;

struct Entry {
  void* fn;
  std::string codes;             // P pointer, I int, L long long, U unsigned long long, F float
};
std::unordered_map<PyObject*, Entry> g_table;        // by interned name
const char* (*g_last_error)() = nullptr;
PyObject* g_fallback = nullptr;                      // the ctypes call, for arguments this module does not convert

// x86-64 System V: integer and pointer arguments fill their registers and then the stack in order, float arguments their own
// registers, independently of how the two mix; surplus arguments are ignored by the callee.  So one signature calls every launcher.
#if !defined(__x86_64__) || defined(_WIN32)
#error "the launcher trampoline is written for the x86-64 System V calling convention"
#endif
using Fn = int (*)(float, float, float, float, float, float, float, float,
                   long long, long long, long long, long long, long long, long long, long long, long long, long long, long long,
                   long long, long long, long long, long long, long long, long long, long long, long long, long long, long long,
                   long long, long long, long long, long long, long long, long long, long long, long long, long long, long long,
                   long long, long long, long long, long long, long long, long long, long long, long long, long long, long long);

int invoke(void* fn, const float* f, const long long* a) {
  return reinterpret_cast<Fn>(fn)(f[0], f[1], f[2], f[3], f[4], f[5], f[6], f[7],
      a[0], a[1], a[2], a[3], a[4], a[5], a[6], a[7], a[8], a[9], a[10], a[11], a[12], a[13], a[14], a[15], a[16], a[17], a[18], a[19],
      a[20], a[21], a[22], a[23], a[24], a[25], a[26], a[27], a[28], a[29], a[30], a[31], a[32], a[33], a[34], a[35], a[36], a[37],
      a[38], a[39]);
}

PyObject* raise_code(const char* name, int rc) {
  PyErr_Format(PyExc_RuntimeError, "%s failed with code %d: %s", name, rc, g_last_error ? g_last_error() : "");
  return nullptr;
}

const Entry* find(PyObject* name) {
  auto it = g_table.find(name);
  if (it != g_table.end()) return &it->second;
  if (!PyUnicode_Check(name)) return nullptr;
  PyObject* s = name;
  Py_INCREF(s);
  PyUnicode_InternInPlace(&s);
  it = g_table.find(s);
  Py_DECREF(s);
  return it == g_table.end() ? nullptr : &it->second;
}

PyObject* py_call(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs < 1) { PyErr_SetString(PyExc_TypeError, "call(name, *args)"); return nullptr; }
  const Entry* e = find(args[0]);
  if (e == nullptr || (Py_ssize_t)e->codes.size() != nargs - 1) return PyObject_Vectorcall(g_fallback, args, nargs, nullptr);
  float f[MAX_FLOATS] = {};
  long long a[MAX_INTS] = {};
  int nf = 0, na = 0;
  for (Py_ssize_t i = 1; i < nargs; ++i) {
    PyObject* o = args[i];
    const char c = e->codes[i - 1];
    if (c == 'F') {
      const double v = PyFloat_AsDouble(o);
      if (v == -1.0 && PyErr_Occurred()) return nullptr;
      f[nf++] = (float)v;
    } else if (o == Py_None && c == 'P') {
      a[na++] = 0;
    } else if (PyLong_Check(o)) {                    // (bool is one)
      a[na] = (long long)PyLong_AsUnsignedLongLongMask(o);           // wraps, as ctypes does
      if (c == 'I') a[na] = (int)a[na];
      if (a[na] == -1 && PyErr_Occurred()) return nullptr;
      ++na;
    } else {
      return PyObject_Vectorcall(g_fallback, args, nargs, nullptr);  // arrays of pointers and the like
    }
  }
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = invoke(e->fn, f, a);
  Py_END_ALLOW_THREADS
  if (rc != 0) return raise_code(PyUnicode_AsUTF8(args[0]), rc);
  Py_RETURN_NONE;
}

// the launchers of the micro-scaled operators, found by name when the table is bound
using Quant4Fn = int (*)(const void*, long long, int, int, const void*, int, void*, void*, int, void*, void*, int, void*);
using DequantFn = int (*)(const void*, const void*, void*, int, int, int, int, int, void*);
using NormMxFn = int (*)(const void*, const void*, const void*, void*, void*, int, int, float, void*, void*, int, void*, void*, int, void*);
using Gemm4Fn = int (*)(const void*, const void*, const void*, const void*, void*, int, int, int, long long, long long, long long, int, int,
                        const void*, const void*, long long, float, void*, long long, void*);
using GatedFn = int (*)(const void*, const void*, void*, void*, int, int, int, long long, long long, long long, long long, int, void*);
using GatedGradFn = int (*)(const void*, const void*, const void*, void*, void*, int, int, int, long long, long long, long long, long long, long long,
                            int, void*);
using DownFn = int (*)(const void*, const void*, const void*, void*, int, int, int, long long, long long, long long, long long, void*);
Quant4Fn g_quant4 = nullptr;
GatedFn g_gated = nullptr;
DownFn g_down = nullptr;
GatedGradFn g_gated_grad = nullptr;
DequantFn g_dequant = nullptr;
NormMxFn g_norm_mx = nullptr;
Gemm4Fn g_gemm4 = nullptr;

// bind({name: (address, codes)}, address of b200_last_error, fallback)
PyObject* py_bind(PyObject*, PyObject* args) {
  PyObject *table, *fallback;
  unsigned long long last;
  if (!PyArg_ParseTuple(args, "O!KO", &PyDict_Type, &table, &last, &fallback)) return nullptr;
  PyObject *key, *val;
  Py_ssize_t pos = 0;
  std::unordered_map<PyObject*, Entry> t;
  while (PyDict_Next(table, &pos, &key, &val)) {
    unsigned long long addr;
    const char* codes;
    if (!PyArg_ParseTuple(val, "Ks", &addr, &codes)) return nullptr;
    int nf = 0, na = 0;
    for (const char* c = codes; *c; ++c) (*c == 'F' ? nf : na)++;
    if (nf > MAX_FLOATS || na > MAX_INTS) continue;                  // left to the fallback
    Py_INCREF(key);
    PyUnicode_InternInPlace(&key);
    t[key] = Entry{reinterpret_cast<void*>(addr), codes};
    if (PyUnicode_CompareWithASCIIString(key, "b200_quant_mxfp4") == 0) g_quant4 = reinterpret_cast<Quant4Fn>(addr);
    if (PyUnicode_CompareWithASCIIString(key, "b200_gemm_gated") == 0) g_gated = reinterpret_cast<GatedFn>(addr);
    if (PyUnicode_CompareWithASCIIString(key, "b200_gated_down") == 0) g_down = reinterpret_cast<DownFn>(addr);
    if (PyUnicode_CompareWithASCIIString(key, "b200_gemm_gated_grad") == 0) g_gated_grad = reinterpret_cast<GatedGradFn>(addr);
    if (PyUnicode_CompareWithASCIIString(key, "b200_dequant_mx") == 0) g_dequant = reinterpret_cast<DequantFn>(addr);
    if (PyUnicode_CompareWithASCIIString(key, "b200_norm_mx") == 0) g_norm_mx = reinterpret_cast<NormMxFn>(addr);
    if (PyUnicode_CompareWithASCIIString(key, "b200_gemm_mxfp4") == 0) g_gemm4 = reinterpret_cast<Gemm4Fn>(addr);
  }
  g_table = std::move(t);
  g_last_error = reinterpret_cast<const char* (*)()>(last);
  Py_INCREF(fallback);
  Py_XDECREF(g_fallback);
  g_fallback = fallback;
  Py_RETURN_NONE;
}

using GemmFn = int (*)(const void*, const void*, void*, int, int, int, long long, long long, long long, int, int, int, int, const void*,
                       const void*, long long, float, void*, long long, void*);
using WorkFn = long long (*)(int, int, int);
GemmFn g_gemm = nullptr;
WorkFn g_gemm_ws = nullptr;
WorkFn g_gemm4_ws = nullptr;
thread_local std::unordered_map<unsigned long long, long long> t_ws, t_ws4;   // (device, M, N, K) -> bytes; bounded below

// bytes of the split workspace of a problem (the answer depends on the shape and the device alone)
long long workspace_bytes(std::unordered_map<unsigned long long, long long>& known, WorkFn ask, int dev, int64_t M, int64_t N, int64_t K) {
  if (M >= (1 << 20) || N >= (1 << 20) || K >= (1 << 20) || dev >= 16) return ask((int)M, (int)N, (int)K);
  const unsigned long long key = ((unsigned long long)dev << 60) | ((unsigned long long)M << 40) | ((unsigned long long)N << 20) | (unsigned long long)K;
  auto it = known.find(key);
  if (it == known.end()) {
    if (known.size() > 4096) known.clear();
    it = known.emplace(key, ask((int)M, (int)N, (int)K)).first;
  }
  return it->second;
}

// rows that the GEMM's tensor maps take as they are
bool plain(const at::Tensor& t) {
  return t.dim() == 2 && t.stride(1) == 1 && (t.stride(0) & 7) == 0 && t.stride(0) >= t.size(1) &&
         (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0;
}

// gemm(a, b, a_mn_major, b_mn_major, out, out_fp32, accumulate, bias, residual, alpha): the result, or None where the general
// path has to look at the operands (copies, errors).
PyObject* py_gemm(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 10 || g_gemm == nullptr) Py_RETURN_NONE;
  for (int i : {0, 1})
    if (!THPVariable_Check(args[i])) Py_RETURN_NONE;
  const at::Tensor &a = THPVariable_Unpack(args[0]), &b = THPVariable_Unpack(args[1]);
  const bool a_mn = PyObject_IsTrue(args[2]) == 1, b_mn = PyObject_IsTrue(args[3]) == 1, acc = PyObject_IsTrue(args[6]) == 1;
  bool f32 = PyObject_IsTrue(args[5]) == 1;
  if (PyErr_Occurred()) return nullptr;
  if (!a.is_cuda() || !b.is_cuda() || a.scalar_type() != at::kBFloat16 || b.scalar_type() != at::kBFloat16 || !plain(a) || !plain(b) ||
      a.device() != b.device())
    Py_RETURN_NONE;
  const int64_t M = a.size(a_mn ? 1 : 0), K = a.size(a_mn ? 0 : 1), N = b.size(b_mn ? 1 : 0);
  if (K != b.size(b_mn ? 0 : 1) || M <= 0 || N <= 0 || K <= 0 || M > 0x7fffffff || N > 0x7fffffff || K > 0x7fffffff) Py_RETURN_NONE;
  const int dev = a.device().index();
  if (c10::cuda::current_device() != dev) Py_RETURN_NONE;
  const bool has_out = args[4] != Py_None;
  at::Tensor out;
  if (has_out) {
    if (!THPVariable_Check(args[4])) Py_RETURN_NONE;
    out = THPVariable_Unpack(args[4]);
    const auto ty = out.scalar_type();
    if (!out.is_cuda() || out.dim() != 2 || out.size(0) != M || out.size(1) != N || out.stride(1) != 1 ||
        (ty != at::kBFloat16 && ty != at::kFloat) || (out.stride(0) * (int64_t)out.element_size()) % 16 != 0 ||
        (reinterpret_cast<uintptr_t>(out.data_ptr()) & 15) != 0)
      Py_RETURN_NONE;
    f32 = ty == at::kFloat;
  } else if (acc || N * (f32 ? 4 : 2) % 16 != 0) {
    Py_RETURN_NONE;
  }
  const void *bias = nullptr, *res = nullptr;
  long long ldr = 0;
  if (args[7] != Py_None) {
    if (!THPVariable_Check(args[7])) Py_RETURN_NONE;
    const at::Tensor& t = THPVariable_Unpack(args[7]);
    if (!t.is_cuda() || t.scalar_type() != at::kBFloat16 || !t.is_contiguous()) Py_RETURN_NONE;
    bias = t.data_ptr();
  }
  if (args[8] != Py_None) {
    if (!THPVariable_Check(args[8])) Py_RETURN_NONE;
    const at::Tensor& t = THPVariable_Unpack(args[8]);
    if (!t.is_cuda() || t.dim() != 2 || t.scalar_type() != at::kBFloat16 || t.stride(1) != 1) Py_RETURN_NONE;
    res = t.data_ptr();
    ldr = t.stride(0);
  }
  const double alpha = PyFloat_AsDouble(args[9]);
  if (alpha == -1.0 && PyErr_Occurred()) return nullptr;
  const long long ws_bytes = workspace_bytes(t_ws, g_gemm_ws, dev, M, N, K);
  int rc;
  {
    pybind11::gil_scoped_release nogil;
    if (!has_out) out = at::empty({M, N}, a.options().dtype(f32 ? at::kFloat : at::kBFloat16).requires_grad(false));
    at::Tensor ws;
    if (ws_bytes > 0) ws = at::empty({ws_bytes}, a.options().dtype(at::kByte).requires_grad(false));
    rc = g_gemm(a.data_ptr(), b.data_ptr(), out.data_ptr(), (int)M, (int)N, (int)K, a.stride(0), b.stride(0), out.stride(0), a_mn, b_mn,
                f32, acc, bias, res, ldr, (float)alpha, ws_bytes > 0 ? ws.data_ptr() : nullptr, ws_bytes,
                c10::cuda::getCurrentCUDAStream(dev).stream());
  }
  if (rc != 0) return raise_code("b200_gemm_bf16", rc);
  if (has_out) { Py_INCREF(args[4]); return args[4]; }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// ---- micro-scaled operators: None where the general path has to look at the operands ----
const at::Tensor* tensor_of(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }
bool int_of(PyObject* o, long long& v) {
  if (!PyLong_Check(o)) return false;
  v = PyLong_AsLongLong(o);
  return !(v == -1 && PyErr_Occurred());
}
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool tile_ok(long long t) { return t >= 0 && t % 16 == 0 && t < (1 << 20); }
int64_t sf_bytes(int64_t rows, int64_t k, int64_t tile) { return (rows + tile - 1) / tile * ((k + 127) / 128) * ((tile + 127) / 128) * 512; }
PyObject* wrap_or_none(at::Tensor& t) {
  if (t.defined()) return THPVariable_Wrap(std::move(t));
  Py_RETURN_NONE;
}
PyObject* wrap_all(at::Tensor* t, int n) {
  PyObject* out = PyTuple_New(n);
  if (out == nullptr) return nullptr;
  for (int i = 0; i < n; ++i) {
    PyObject* o = wrap_or_none(t[i]);
    if (o == nullptr) { Py_DECREF(out); return nullptr; }
    PyTuple_SET_ITEM(out, i, o);
  }
  return out;
}

// quant_mxfp4(x, row_tile or 0, col_tile or 0, noise, hadamard): (q_row, sf_row, q_col, sf_col)
PyObject* py_quant_mxfp4(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  const at::Tensor* x;
  long long rt, ct;
  if (nargs != 5 || g_quant4 == nullptr || (x = tensor_of(args[0])) == nullptr || !int_of(args[1], rt) || !int_of(args[2], ct)) {
    if (PyErr_Occurred()) return nullptr;
    Py_RETURN_NONE;
  }
  const int had = PyObject_IsTrue(args[4]);
  if (had < 0) return nullptr;
  if (!x->is_cuda() || x->scalar_type() != at::kBFloat16 || !plain(*x) || x->size(0) <= 0 || x->size(1) <= 0 || x->size(1) % 32 != 0 ||
      x->size(0) > 0x7fffffe0 || x->size(1) > 0x7fffffff || !tile_ok(rt) || !tile_ok(ct) || (rt == 0 && ct == 0))
    Py_RETURN_NONE;
  const int64_t R = x->size(0), C = x->size(1), Rp = (R + 31) / 32 * 32;
  const int dev = x->device().index();
  if (c10::cuda::current_device() != dev) Py_RETURN_NONE;
  const void* noise = nullptr;
  if (args[3] != Py_None) {
    const at::Tensor* n = tensor_of(args[3]);
    if (n == nullptr || n->device() != x->device() || n->scalar_type() != at::kByte || n->sizes() != x->sizes() || !n->is_contiguous() ||
        (reinterpret_cast<uintptr_t>(n->data_ptr()) & 7) != 0)
      Py_RETURN_NONE;
    noise = n->data_ptr();
  }
  at::Tensor t[4];
  int rc;
  {
    pybind11::gil_scoped_release nogil;
    const auto o = x->options().dtype(at::kByte).requires_grad(false);
    if (rt) { t[0] = at::empty({R, C / 2}, o); t[1] = at::empty({sf_bytes(R, C, rt)}, o); }
    if (ct) { t[2] = at::empty({C, Rp / 2}, o); t[3] = at::empty({sf_bytes(C, Rp, ct)}, o); }
    rc = g_quant4(x->data_ptr(), x->stride(0), (int)R, (int)C, noise, had, rt ? t[0].data_ptr() : nullptr, rt ? t[1].data_ptr() : nullptr,
                  (int)rt, ct ? t[2].data_ptr() : nullptr, ct ? t[3].data_ptr() : nullptr, (int)ct,
                  c10::cuda::getCurrentCUDAStream(dev).stream());
  }
  if (rc != 0) return raise_code("b200_quant_mxfp4", rc);
  return wrap_all(t, 4);
  END_HANDLE_TH_ERRORS
}

// dequant_mx(q, sf, rows, k, tile_rows, e2m1, fp32): [rows, k]
PyObject* py_dequant_mx(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  const at::Tensor *q, *sf;
  long long rows, k, tile;
  if (nargs != 7 || g_dequant == nullptr || (q = tensor_of(args[0])) == nullptr || (sf = tensor_of(args[1])) == nullptr ||
      !int_of(args[2], rows) || !int_of(args[3], k) || !int_of(args[4], tile)) {
    if (PyErr_Occurred()) return nullptr;
    Py_RETURN_NONE;
  }
  const int four = PyObject_IsTrue(args[5]), f32 = PyObject_IsTrue(args[6]);
  if (four < 0 || f32 < 0) return nullptr;
  const int dev = q->is_cuda() ? q->device().index() : -1;
  if (dev < 0 || sf->device() != q->device() || c10::cuda::current_device() != dev || rows <= 0 || k <= 0 || k % 32 != 0 || rows > 0x7fffffff ||
      k > 0x7fffffff || tile <= 0 || !tile_ok(tile) || q->scalar_type() != at::kByte || sf->scalar_type() != at::kByte || !q->is_contiguous() ||
      !sf->is_contiguous() || q->numel() != (four ? rows * (k / 2) : rows * k) || sf->numel() < sf_bytes(rows, k, tile) || !aligned16(q->data_ptr()))
    Py_RETURN_NONE;
  at::Tensor out;
  int rc;
  {
    pybind11::gil_scoped_release nogil;
    out = at::empty({rows, k}, q->options().dtype(f32 ? at::kFloat : at::kBFloat16).requires_grad(false));
    rc = g_dequant(q->data_ptr(), sf->data_ptr(), out.data_ptr(), (int)rows, (int)k, (int)tile, four, f32,
                   c10::cuda::getCurrentCUDAStream(dev).stream());
  }
  if (rc != 0) return raise_code("b200_dequant_mx", rc);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// norm_mx(x, weight, eps, residual, row_tile or 0, col_tile or 0): (q_row, sf_row, q_col, sf_col, h, rstd); h None without a residual
PyObject* py_norm_mx(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  const at::Tensor *x, *w, *res = nullptr;
  long long rt, ct;
  if (nargs != 6 || g_norm_mx == nullptr || (x = tensor_of(args[0])) == nullptr || (w = tensor_of(args[1])) == nullptr || !int_of(args[4], rt) ||
      !int_of(args[5], ct) || (args[3] != Py_None && (res = tensor_of(args[3])) == nullptr)) {
    if (PyErr_Occurred()) return nullptr;
    Py_RETURN_NONE;
  }
  const double eps = PyFloat_AsDouble(args[2]);
  if (eps == -1.0 && PyErr_Occurred()) return nullptr;
  if (!x->is_cuda() || x->scalar_type() != at::kBFloat16 || x->dim() != 2 || !x->is_contiguous() || x->size(0) <= 0 || x->size(1) <= 0 ||
      x->size(1) % 32 != 0 || x->size(1) > 8192 || x->size(0) > 0x7fffff00 || !aligned16(x->data_ptr()) || !tile_ok(rt) || !tile_ok(ct))
    Py_RETURN_NONE;
  const int64_t T = x->size(0), D = x->size(1), Tp = (T + 127) / 128 * 128;
  if (w->device() != x->device() || w->scalar_type() != at::kBFloat16 || w->dim() != 1 || w->size(0) != D || !w->is_contiguous() || !aligned16(w->data_ptr()))
    Py_RETURN_NONE;
  if (res != nullptr && (res->device() != x->device() || res->scalar_type() != at::kBFloat16 || res->sizes() != x->sizes() ||
                         !res->is_contiguous() || !aligned16(res->data_ptr())))
    Py_RETURN_NONE;
  const int dev = x->device().index();
  if (c10::cuda::current_device() != dev) Py_RETURN_NONE;
  at::Tensor t[6];
  int rc;
  {
    pybind11::gil_scoped_release nogil;
    const auto o = x->options().requires_grad(false), b = o.dtype(at::kByte);
    if (rt) { t[0] = at::empty({T, D}, b); t[1] = at::empty({sf_bytes(T, D, rt)}, b); }
    if (ct) { t[2] = at::empty({D, Tp}, b); t[3] = at::empty({sf_bytes(D, Tp, ct)}, b); }
    if (res != nullptr) t[4] = at::empty({T, D}, o);
    t[5] = at::empty({T}, o.dtype(at::kFloat));
    rc = g_norm_mx(x->data_ptr(), res != nullptr ? res->data_ptr() : nullptr, w->data_ptr(), res != nullptr ? t[4].data_ptr() : nullptr,
                   t[5].data_ptr(), (int)T, (int)D, (float)eps, rt ? t[0].data_ptr() : nullptr, rt ? t[1].data_ptr() : nullptr, (int)rt,
                   ct ? t[2].data_ptr() : nullptr, ct ? t[3].data_ptr() : nullptr, (int)ct, c10::cuda::getCurrentCUDAStream(dev).stream());
  }
  if (rc != 0) return raise_code("b200_norm_mx", rc);
  return wrap_all(t, 6);
  END_HANDLE_TH_ERRORS
}

// gemm_mxfp4(a_q, a_sf, a_tile, b_q, b_sf, b_tile, M, N, K, fp32, bias, residual, alpha): [M, N], a new tensor; the tiles have been checked to be
// the kernel's
PyObject* py_gemm_mxfp4(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 13 || g_gemm4 == nullptr || g_gemm4_ws == nullptr) Py_RETURN_NONE;
  const at::Tensor* t[4];
  for (int i = 0; i < 4; ++i)
    if ((t[i] = tensor_of(args[i < 2 ? i : i + 1])) == nullptr || !t[i]->is_cuda() || t[i]->scalar_type() != at::kByte || !t[i]->is_contiguous() ||
        t[i]->device() != t[0]->device() || !aligned16(t[i]->data_ptr()))
      Py_RETURN_NONE;
  long long M, N, K, a_tile, b_tile;
  if (!int_of(args[2], a_tile) || !int_of(args[5], b_tile) || !int_of(args[6], M) || !int_of(args[7], N) || !int_of(args[8], K)) {
    if (PyErr_Occurred()) return nullptr;
    Py_RETURN_NONE;
  }
  const int f32 = PyObject_IsTrue(args[9]);
  if (f32 < 0) return nullptr;
  const double alpha = PyFloat_AsDouble(args[12]);
  if (alpha == -1.0 && PyErr_Occurred()) return nullptr;
  const int dev = t[0]->device().index();
  if (c10::cuda::current_device() != dev || M <= 0 || N <= 0 || K <= 0 || K % 32 != 0 || M > 0x7fffffff || N > 0x7fffffff || K > 0x7fffffff ||
      N * (f32 ? 4 : 2) % 16 != 0 || a_tile <= 0 || b_tile <= 0 || !tile_ok(a_tile) || !tile_ok(b_tile) ||
      t[0]->numel() != M * (K / 2) || t[2]->numel() != N * (K / 2) || t[1]->numel() < sf_bytes(M, K, a_tile) || t[3]->numel() < sf_bytes(N, K, b_tile))
    Py_RETURN_NONE;
  const void *bias = nullptr, *res = nullptr;
  long long ldr = 0;
  if (args[10] != Py_None) {
    const at::Tensor* b = tensor_of(args[10]);
    if (b == nullptr || b->device() != t[0]->device() || b->scalar_type() != at::kBFloat16 || b->dim() != 1 || b->size(0) != N || !b->is_contiguous())
      Py_RETURN_NONE;
    bias = b->data_ptr();
  }
  if (args[11] != Py_None) {
    const at::Tensor* r = tensor_of(args[11]);
    if (r == nullptr || r->device() != t[0]->device() || r->scalar_type() != at::kBFloat16 || r->dim() != 2 || r->size(0) != M || r->size(1) != N ||
        r->stride(1) != 1)
      Py_RETURN_NONE;
    res = r->data_ptr();
    ldr = r->stride(0);
  }
  const long long ws_bytes = workspace_bytes(t_ws4, g_gemm4_ws, dev, M, N, K);
  at::Tensor out;
  int rc;
  {
    pybind11::gil_scoped_release nogil;
    const auto o = t[0]->options().requires_grad(false);
    out = at::empty({M, N}, o.dtype(f32 ? at::kFloat : at::kBFloat16));
    at::Tensor ws;
    if (ws_bytes > 0) ws = at::empty({ws_bytes}, o);
    rc = g_gemm4(t[0]->data_ptr(), t[1]->data_ptr(), t[2]->data_ptr(), t[3]->data_ptr(), out.data_ptr(), (int)M, (int)N, (int)K, K / 2, K / 2, N, f32, 0,
                 bias, res, ldr, (float)alpha, ws_bytes > 0 ? ws.data_ptr() : nullptr, ws_bytes, c10::cuda::getCurrentCUDAStream(dev).stream());
  }
  if (rc != 0) return raise_code("b200_gemm_mxfp4", rc);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

bool bf16_plain(const at::Tensor* t, c10::Device dev) {
  return t != nullptr && t->is_cuda() && t->device() == dev && t->scalar_type() == at::kBFloat16 && plain(*t) && t->size(0) <= 0x7fffffff &&
         t->size(1) <= 0x7fffffff;
}

// gated_fwd(x [T, D], w [2F, D], act, gu: 0 none, 1 bf16, 2 fp32): (a [T, F], gu [T, 2F] or None)
PyObject* py_gated_fwd(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  const at::Tensor *x, *w;
  long long act, want;
  if (nargs != 4 || g_gated == nullptr || (x = tensor_of(args[0])) == nullptr || (w = tensor_of(args[1])) == nullptr || !int_of(args[2], act) ||
      !int_of(args[3], want)) {
    if (PyErr_Occurred()) return nullptr;
    Py_RETURN_NONE;
  }
  if (!x->is_cuda() || !bf16_plain(x, x->device()) || !bf16_plain(w, x->device())) Py_RETURN_NONE;
  const int64_t T = x->size(0), D = x->size(1), F = w->size(0) / 2;
  const int dev = x->device().index();
  if (c10::cuda::current_device() != dev || T <= 0 || D <= 0 || F <= 0 || D % 8 != 0 || F % 8 != 0 || w->size(0) != 2 * F || w->size(1) != D) Py_RETURN_NONE;
  at::Tensor t[2];
  int rc;
  {
    pybind11::gil_scoped_release nogil;
    const auto o = x->options().requires_grad(false);
    t[0] = at::empty({T, F}, o);
    if (want) t[1] = at::empty({T, 2 * F}, want == 2 ? o.dtype(at::kFloat) : o);
    rc = g_gated(x->data_ptr(), w->data_ptr(), t[0].data_ptr(), want ? t[1].data_ptr() : nullptr, (int)T, (int)F, (int)D, x->stride(0), w->stride(0),
                 F, 2 * F, (int)act + (want == 2 ? 2 : 0), c10::cuda::getCurrentCUDAStream(dev).stream());
  }
  if (rc != 0) return raise_code("b200_gemm_gated", rc);
  return wrap_all(t, 2);
  END_HANDLE_TH_ERRORS
}

// gated_down(a [T, F], w [D, F], residual [T, D] or None): y [T, D], T up to 64
PyObject* py_gated_down(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  const at::Tensor *a, *w, *res = nullptr;
  if (nargs != 3 || g_down == nullptr || (a = tensor_of(args[0])) == nullptr || (w = tensor_of(args[1])) == nullptr ||
      (args[2] != Py_None && (res = tensor_of(args[2])) == nullptr)) {
    if (PyErr_Occurred()) return nullptr;
    Py_RETURN_NONE;
  }
  if (!a->is_cuda() || !bf16_plain(a, a->device()) || !bf16_plain(w, a->device()) || (res != nullptr && !bf16_plain(res, a->device()))) Py_RETURN_NONE;
  const int64_t T = a->size(0), F = a->size(1), D = w->size(0);
  const int dev = a->device().index();
  if (c10::cuda::current_device() != dev || T <= 0 || T > 64 || D <= 0 || F <= 0 || D % 8 != 0 || F % 8 != 0 || w->size(1) != F ||
      (res != nullptr && (res->size(0) != T || res->size(1) != D)))
    Py_RETURN_NONE;
  at::Tensor t[1];
  int rc;
  {
    pybind11::gil_scoped_release nogil;
    t[0] = at::empty({T, D}, a->options().requires_grad(false));
    rc = g_down(a->data_ptr(), w->data_ptr(), res != nullptr ? res->data_ptr() : nullptr, t[0].data_ptr(), (int)T, (int)D, (int)F, a->stride(0), w->stride(0),
                res != nullptr ? res->stride(0) : 0, D, c10::cuda::getCurrentCUDAStream(dev).stream());
  }
  if (rc != 0) return raise_code("b200_gated_down", rc);
  return THPVariable_Wrap(t[0]);
  END_HANDLE_TH_ERRORS
}

// gated_bwd(dy [T, D], w_down [D, F], gu [T, 2F] (bf16 or fp32), act, want_a): (dgu [T, 2F], a [T, F] or None)
PyObject* py_gated_bwd(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  const at::Tensor *dy, *w, *gu;
  long long act;
  if (nargs != 5 || g_gated_grad == nullptr || (dy = tensor_of(args[0])) == nullptr || (w = tensor_of(args[1])) == nullptr ||
      (gu = tensor_of(args[2])) == nullptr || !int_of(args[3], act)) {
    if (PyErr_Occurred()) return nullptr;
    Py_RETURN_NONE;
  }
  const int want = PyObject_IsTrue(args[4]);
  if (want < 0) return nullptr;
  if (!dy->is_cuda() || !bf16_plain(dy, dy->device()) || !bf16_plain(w, dy->device())) Py_RETURN_NONE;
  const bool f32 = gu->scalar_type() == at::kFloat;
  if (f32 ? !(gu->device() == dy->device() && plain(*gu)) : !bf16_plain(gu, dy->device())) Py_RETURN_NONE;
  const int64_t T = dy->size(0), D = dy->size(1), F = w->size(1);
  const int dev = dy->device().index();
  if (c10::cuda::current_device() != dev || T <= 0 || D <= 0 || F <= 0 || D % 8 != 0 || F % 8 != 0 || w->size(0) != D || gu->size(0) != T ||
      gu->size(1) != 2 * F)
    Py_RETURN_NONE;
  at::Tensor t[2];
  int rc;
  {
    pybind11::gil_scoped_release nogil;
    const auto o = dy->options().requires_grad(false);
    t[0] = at::empty({T, 2 * F}, o);
    if (want) t[1] = at::empty({T, F}, o);
    rc = g_gated_grad(dy->data_ptr(), w->data_ptr(), gu->data_ptr(), t[0].data_ptr(), want ? t[1].data_ptr() : nullptr, (int)T, (int)F, (int)D,
                      dy->stride(0), w->stride(0), gu->stride(0), 2 * F, F, (int)act + (f32 ? 2 : 0), c10::cuda::getCurrentCUDAStream(dev).stream());
  }
  if (rc != 0) return raise_code("b200_gemm_gated_grad", rc);
  return wrap_all(t, 2);
  END_HANDLE_TH_ERRORS
}

// bind_mx(address of b200_gemm_mxfp4_workspace)
PyObject* py_bind_mx(PyObject*, PyObject* args) {
  unsigned long long w;
  if (!PyArg_ParseTuple(args, "K", &w)) return nullptr;
  g_gemm4_ws = reinterpret_cast<WorkFn>(w);
  Py_RETURN_NONE;
}

// bind_gemm(address of b200_gemm_bf16, address of b200_gemm_bf16_workspace)
PyObject* py_bind_gemm(PyObject*, PyObject* args) {
  unsigned long long g, w;
  if (!PyArg_ParseTuple(args, "KK", &g, &w)) return nullptr;
  g_gemm = reinterpret_cast<GemmFn>(g);
  g_gemm_ws = reinterpret_cast<WorkFn>(w);
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"bind", py_bind, METH_VARARGS, nullptr},
    {"bind_gemm", py_bind_gemm, METH_VARARGS, nullptr},
    {"call", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_call)), METH_FASTCALL, nullptr},
    {"bind_mx", py_bind_mx, METH_VARARGS, nullptr},
    {"quant_mxfp4", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_quant_mxfp4)), METH_FASTCALL, nullptr},
    {"gated_fwd", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_gated_fwd)), METH_FASTCALL, nullptr},
    {"gated_down", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_gated_down)), METH_FASTCALL, nullptr},
    {"gated_bwd", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_gated_bwd)), METH_FASTCALL, nullptr},
    {"dequant_mx", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_dequant_mx)), METH_FASTCALL, nullptr},
    {"norm_mx", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_norm_mx)), METH_FASTCALL, nullptr},
    {"gemm_mxfp4", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_gemm_mxfp4)), METH_FASTCALL, nullptr},
    {"gemm", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_gemm)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_b200_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__b200_host(void) { return PyModule_Create(&module); }
