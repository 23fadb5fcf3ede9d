// Host side of the launches, native: a CPython module (`_b200_host.so`) that `ops/_lib.py` and `ops/kernels.py` use when it is there.
//
//   bind(table, last_error, fallback)   name -> (address, argument codes) of the launchers of the kernel library
//   call(name, *args)                   converts the arguments by their codes, calls the launcher with the GIL released and raises
//                                       RuntimeError on a code other than 0
//   gemm(...)                           ops.kernels.gemm for CUDA operands that need no copy: checks, output, split workspace, launch
//   quant_mxfp4, dequant_mx, norm_mx, gemm_mxfp4, gated_fwd, gated_down, gated_bwd   the same for ops.mxfp4, ops.norm_mx and the gated block
//   attention_mask                      the tables of ops.masked_attention.attention_mask
//   route, distill_loss, masked_attention   ops.moe_ops.route, ops.functional.distill_loss and masked_attention with their autograd nodes: a backward
//                                       pass then runs in autograd's thread without Python (seven tokens' distillation and its gradient
//                                       101 us of host time, now 53; of which 42 are autograd's own)
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
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>

#include <mutex>
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

// the launchers of the operators with autograd nodes
using RouteFn = int (*)(const void*, int, long long, const float*, int, int, int, int, int, int, int, float, int*, float*, int*, void*);
using RouteBwdFn = int (*)(const void*, int, long long, const int*, const float*, int, int, int, int, int, float, void*, void*);
using DistillFn = int (*)(const void*, int, long long, const long long*, const void*, int, const void*, int, int, int, int, int, float, float, long long,
                          float*, float*, double*, void*);
using DistillBwdFn = int (*)(const void*, int, long long, const long long*, const void*, int, const void*, int, int, int, int, int, float, float,
                             long long, const float*, const double*, const float*, void*, long long, void*);
using MaskedFn = int (*)(const void*, const void*, const void*, void*, void*, float*, const float*, const float*, const int*, int, int, int, int, int, int,
                         long long, long long, long long, long long, long long, long long, float, float, void*, long long, void*);
using MaskedRowsFn = int (*)(const void*, const void*, const void*, void*, float*, const float*, const float*, const int*, int, int, int, int, int, int,
                             long long, long long, long long, long long, long long, long long, float, float, void*, long long, void*);
using MaskedBwdFn = int (*)(const void*, const void*, const void*, const void*, const void*, const void*, const float*, float*, float*, void*, void*,
                            const float*, const int*, int, int, int, int, int, int, long long, long long, long long, long long, long long, long long,
                            long long, long long, long long, long long, float, float, void*, long long, void*);
RouteFn g_route = nullptr;
RouteBwdFn g_route_bwd = nullptr;
DistillFn g_distill = nullptr;
DistillBwdFn g_distill_bwd = nullptr;
MaskedFn g_masked = nullptr;
MaskedRowsFn g_masked_rows = nullptr;
MaskedBwdFn g_masked_bwd = nullptr;
int (*g_few_rows)(int, int, int, int) = nullptr;
long long (*g_rows_ws)(int, int, int, int, int, int) = nullptr;
long long (*g_masked_bwd_ws)(int, int, int, int, int, int) = nullptr;
long long (*g_masked_fwd_ws)(int, int, int, int, int) = nullptr;
long long (*g_mask_ints)(int, int, int) = nullptr;
int (*g_mask)(const void*, int, const uint8_t*, int, int, int, int, int, int*, void*) = nullptr;

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
    auto take = [&](const char* name, auto& fn) {
      if (PyUnicode_CompareWithASCIIString(key, name) == 0) fn = reinterpret_cast<std::decay_t<decltype(fn)>>(addr);
    };
    take("b200_route", g_route);
    take("b200_route_bwd", g_route_bwd);
    take("b200_distill_fwd", g_distill);
    take("b200_distill_bwd", g_distill_bwd);
    take("b200_attn_masked_fwd", g_masked);
    take("b200_attn_mask", g_mask);
    take("b200_attn_masked_rows", g_masked_rows);
    take("b200_attn_masked_bwd", g_masked_bwd);
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

// ---- operators with autograd nodes of their own: None where the general path has to look at the operands (copies, other types, errors) ----
namespace ag = torch::autograd;

void check_rc(const char* name, int rc) {
  TORCH_CHECK(rc == 0, name, " failed with code ", rc, ": ", g_last_error ? g_last_error() : "");
}
cudaStream_t stream_of(const at::Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }
at::Tensor plain_grad(const at::Tensor& g, at::ScalarType type) {     // contiguous, aligned, of a type
  at::Tensor r = g.to(type).contiguous();
  return aligned16(r.data_ptr()) ? r : r.clone();
}
// A CUDA tensor of the current device; its rows (dim 2) contiguous and apart.
bool here(const at::Tensor& t) { return t.is_cuda() && c10::cuda::current_device() == t.device().index(); }
bool rows_ok(const at::Tensor& t) { return t.dim() == 2 && t.stride(1) == 1 && t.stride(0) >= t.size(1); }
bool float_or_bf16(const at::Tensor& t) { return t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16; }
// None: `t` stays undefined; false where it is neither that nor a tensor
bool optional_tensor(PyObject* o, at::Tensor& t) {
  if (o == Py_None) return true;
  const at::Tensor* p = tensor_of(o);
  if (p == nullptr) return false;
  t = *p;
  return true;
}
bool float_of(PyObject* o, double& v) {
  v = PyFloat_AsDouble(o);
  return !(v == -1.0 && PyErr_Occurred());
}
template <typename N>
void set_node(const std::shared_ptr<N>& node, at::Tensor& out, ag::edge_list&& edges) {
  node->set_next_edges(std::move(edges));
  ag::set_history(out, node);
}

struct RouteBackward : public ag::Node {
  ag::SavedVariable logits, idx;
  int sigmoid, renorm;
  float scale;
  std::string name() const override { return "RouteBackward"; }
  void release_variables() override { logits.reset_data(); idx.reset_data(); }
  ag::variable_list apply(ag::variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    if (!grads[0].defined()) return {at::Tensor()};
    const at::Tensor x = logits.unpack(), i = idx.unpack(), g = plain_grad(grads[0], at::kFloat);
    at::Tensor dx = at::empty(x.sizes(), x.options().requires_grad(false));
    check_rc("b200_route_bwd", g_route_bwd(x.data_ptr(), x.scalar_type() == at::kBFloat16, x.stride(0), i.data_ptr<int>(), g.data_ptr<float>(),
                                           (int)x.size(0), (int)x.size(1), (int)i.size(1), sigmoid, renorm, scale, dx.data_ptr(), stream_of(x)));
    return {dx};
  }
};

// route(logits, k, sigmoid, bias or None, groups, top_groups, renormalize, scale): (idx, w, counts)
PyObject* py_route(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  const at::Tensor* x;
  at::Tensor bias;
  long long k, sigmoid, groups, top, renorm;
  double scale;
  if (nargs != 8 || g_route == nullptr || g_route_bwd == nullptr || (x = tensor_of(args[0])) == nullptr || !int_of(args[1], k) ||
      !int_of(args[2], sigmoid) || !optional_tensor(args[3], bias) || !int_of(args[4], groups) || !int_of(args[5], top) ||
      !int_of(args[6], renorm) || !float_of(args[7], scale)) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
  if (!here(*x) || !rows_ok(*x) || !float_or_bf16(*x)) Py_RETURN_NONE;
  const int64_t T = x->size(0), E = x->size(1);
  if (T < 1 || T > 0x7fffffff || E < 1 || E > 256 || k < 1 || k > 32 || k > E || groups < 1 || groups > 32 || E % groups != 0 || top < 1 ||
      top > groups || top * (E / groups) < k)
    Py_RETURN_NONE;
  if (bias.defined() && (bias.device() != x->device() || bias.scalar_type() != at::kFloat || bias.dim() != 1 || bias.size(0) != E || !bias.is_contiguous()))
    Py_RETURN_NONE;
  at::Tensor t[3];
  {
    pybind11::gil_scoped_release nogil;
    const auto o = x->options().requires_grad(false);
    t[0] = at::empty({T, k}, o.dtype(at::kInt));
    t[1] = at::empty({T, k}, o.dtype(at::kFloat));
    t[2] = at::empty({E}, o.dtype(at::kInt));
    check_rc("b200_route", g_route(x->data_ptr(), x->scalar_type() == at::kBFloat16, x->stride(0), bias.defined() ? bias.data_ptr<float>() : nullptr,
                                   (int)T, (int)E, (int)k, (int)sigmoid, (int)groups, (int)top, (int)renorm, (float)scale, t[0].data_ptr<int>(),
                                   t[1].data_ptr<float>(), t[2].data_ptr<int>(), stream_of(*x)));
    if (ag::compute_requires_grad(*x)) {
      auto node = std::shared_ptr<RouteBackward>(new RouteBackward(), ag::deleteNode);
      node->logits = ag::SavedVariable(*x, false);
      node->idx = ag::SavedVariable(t[0], false);
      node->sigmoid = (int)sigmoid;
      node->renorm = (int)renorm;
      node->scale = (float)scale;
      set_node(node, t[1], ag::collect_next_edges(*x));
    }
  }
  return wrap_all(t, 3);
  END_HANDLE_TH_ERRORS
}

struct DistillArgs {
  int K, rest;
  float alpha, tau;
  long long ignore;
};
const long long* labels_of(const at::Tensor& t) { return t.defined() ? reinterpret_cast<const long long*>(t.data_ptr<int64_t>()) : nullptr; }

struct DistillLossBackward : public ag::Node {
  ag::SavedVariable logits, labels, ids, values, stats, teacher;
  DistillArgs a;
  std::string name() const override { return "DistillLossBackward"; }
  void release_variables() override {
    for (auto* v : {&logits, &labels, &ids, &values, &stats, &teacher}) v->reset_data();
  }
  ag::variable_list apply(ag::variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    if (!grads[0].defined()) return {at::Tensor()};
    const at::Tensor x = logits.unpack(), l = labels.unpack(), i = ids.unpack(), v = values.unpack(), s = stats.unpack(), te = teacher.unpack(),
                     g = plain_grad(grads[0], at::kFloat);
    at::Tensor dx = at::empty(x.sizes(), x.options().requires_grad(false));
    check_rc("b200_distill_bwd",
             g_distill_bwd(x.data_ptr(), x.scalar_type() == at::kBFloat16, x.stride(0), labels_of(l), i.data_ptr(), i.scalar_type() == at::kLong,
                           v.data_ptr(), v.scalar_type() == at::kBFloat16, (int)x.size(0), a.K, (int)x.size(1), a.rest, a.alpha, a.tau, a.ignore,
                           s.data_ptr<float>(), te.data_ptr<double>(), g.data_ptr<float>(), dx.data_ptr(), dx.stride(0), stream_of(x)));
    return {dx};
  }
};

// distill_loss(logits, labels or None, ids, values, alpha, temperature, rest, ignore_index): loss
PyObject* py_distill_loss(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  const at::Tensor *x, *i, *v;
  at::Tensor l;
  double alpha, tau;
  long long rest, ignore;
  if (nargs != 8 || g_distill == nullptr || g_distill_bwd == nullptr || (x = tensor_of(args[0])) == nullptr || !optional_tensor(args[1], l) ||
      (i = tensor_of(args[2])) == nullptr || (v = tensor_of(args[3])) == nullptr || !float_of(args[4], alpha) || !float_of(args[5], tau) ||
      !int_of(args[6], rest) || !int_of(args[7], ignore)) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
  if (!here(*x) || !rows_ok(*x) || !float_or_bf16(*x)) Py_RETURN_NONE;
  const int64_t T = x->size(0), V = x->size(1);
  if (T < 1 || T > 0x7fff0000 || V < 1 || V > (rest ? 900000 : 1 << 30) || !(alpha >= 0.0 && alpha <= 1.0) || !((float)tau > 0.f && (float)tau < INFINITY) ||
      (!l.defined() && alpha < 1.0))
    Py_RETURN_NONE;
  if (i->device() != x->device() || v->device() != x->device() || i->dim() != 2 || i->sizes() != v->sizes() || i->size(0) != T || i->size(1) < 1 ||
      i->size(1) > 1024 || (i->scalar_type() != at::kLong && i->scalar_type() != at::kInt) || !float_or_bf16(*v) || !i->is_contiguous() ||
      !v->is_contiguous())
    Py_RETURN_NONE;
  if (l.defined() && (l.device() != x->device() || l.scalar_type() != at::kLong || l.dim() != 1 || l.size(0) != T || !l.is_contiguous())) Py_RETURN_NONE;
  at::Tensor loss;
  {
    pybind11::gil_scoped_release nogil;
    const auto o = x->options().requires_grad(false);
    const DistillArgs a = {(int)i->size(1), rest != 0, (float)alpha, (float)tau, ignore};
    loss = at::empty({T}, o.dtype(at::kFloat));
    at::Tensor stats = at::empty({T, 4}, o.dtype(at::kFloat)), teacher = at::empty({T}, o.dtype(at::kDouble));
    check_rc("b200_distill_fwd",
             g_distill(x->data_ptr(), x->scalar_type() == at::kBFloat16, x->stride(0), labels_of(l), i->data_ptr(), i->scalar_type() == at::kLong,
                       v->data_ptr(), v->scalar_type() == at::kBFloat16, (int)T, a.K, (int)V, a.rest, a.alpha, a.tau, a.ignore, loss.data_ptr<float>(),
                       stats.data_ptr<float>(), teacher.data_ptr<double>(), stream_of(*x)));
    if (ag::compute_requires_grad(*x)) {
      auto node = std::shared_ptr<DistillLossBackward>(new DistillLossBackward(), ag::deleteNode);
      node->logits = ag::SavedVariable(*x, false);
      node->labels = ag::SavedVariable(l, false);
      node->ids = ag::SavedVariable(*i, false);
      node->values = ag::SavedVariable(v->detach(), false);
      node->stats = ag::SavedVariable(stats, false);
      node->teacher = ag::SavedVariable(teacher, false);
      node->a = a;
      set_node(node, loss, ag::collect_next_edges(*x));
    }
  }
  return THPVariable_Wrap(std::move(loss));
  END_HANDLE_TH_ERRORS
}

// [B, S, H, D] as the kernels read it without a copy (ops.masked_attention._bshd)
struct Pitch { long long row, batch; };
bool bshd(const at::Tensor& t, Pitch& p) {
  const int64_t B = t.size(0), S = t.size(1), H = t.size(2), D = t.size(3), w = H * D;
  p.row = S > 1 ? t.stride(1) : w;
  p.batch = B > 1 ? t.stride(0) : S * p.row;
  return t.stride(3) == 1 && (H == 1 || t.stride(2) == D) && p.row >= w && p.batch >= w && p.row % 8 == 0 && p.batch % 8 == 0 && aligned16(t.data_ptr());
}
const float* floats_of(const at::Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }
at::Tensor workspace(long long bytes, const at::Tensor& like) {
  return bytes > 0 ? at::empty({bytes}, like.options().dtype(at::kByte).requires_grad(false)) : at::Tensor();
}

struct MaskedAttentionBackward : public ag::Node {
  ag::SavedVariable q, k, v, out, low, lse, slopes, mask;
  float softcap, scale;
  std::string name() const override { return "MaskedAttentionBackward"; }
  void release_variables() override {
    for (auto* s : {&q, &k, &v, &out, &low, &lse, &slopes, &mask}) s->reset_data();
  }
  ag::variable_list apply(ag::variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    if (!grads[0].defined()) return {at::Tensor(), at::Tensor(), at::Tensor()};
    const at::Tensor a = q.unpack(), b = k.unpack(), c = v.unpack(), o = out.unpack(shared_from_this()), lo = low.unpack(), ls = lse.unpack(),
                     sl = slopes.unpack(), m = mask.unpack(), g = plain_grad(grads[0], at::kBFloat16);
    Pitch pq, pk, pv;
    TORCH_CHECK(bshd(a, pq) && bshd(b, pk) && bshd(c, pv), "masked_attention: saved operands");
    const int64_t B = a.size(0), Sq = a.size(1), Hq = a.size(2), D = a.size(3), Skv = b.size(1), Hkv = b.size(2);
    const auto f32 = a.options().dtype(at::kFloat).requires_grad(false);
    at::Tensor dq = at::empty({B, Sq, Hq, D}, f32), dk = at::empty({B, Skv, Hkv, D}, a.options().requires_grad(false)), dv = at::empty_like(dk),
               delta = at::empty({B, Hq, Sq}, f32);
    const long long n = g_masked_bwd_ws((int)B, (int)Sq, (int)Skv, (int)Hq, (int)Hkv, (int)D), w = Hkv * D;
    at::Tensor ws = workspace(n, a);
    check_rc("b200_attn_masked_bwd",
             g_masked_bwd(a.data_ptr(), b.data_ptr(), c.data_ptr(), o.data_ptr(), lo.data_ptr(), g.data_ptr(), ls.data_ptr<float>(),
                          delta.data_ptr<float>(), dq.data_ptr<float>(), dk.data_ptr(), dv.data_ptr(), floats_of(sl), m.data_ptr<int>(), (int)B, (int)Sq,
                          (int)Skv, (int)Hq, (int)Hkv, (int)D, pq.row, pk.row, pv.row, w, w, pq.batch, pk.batch, pv.batch, Skv * w, Skv * w, scale,
                          softcap, n > 0 ? ws.data_ptr() : nullptr, n, stream_of(a)));
    return {dq.to(at::kBFloat16), dk, dv};
  }
};

// masked_attention(q, k, v, the mask's buffer, B, Sq, Skv, slopes or None, softcap, scale): out.  (Sink logits take the general path.)
PyObject* py_masked_attention(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  const at::Tensor *q, *k, *v, *m;
  at::Tensor sl;
  long long mb, mq, mk;
  double softcap, scale;
  if (nargs != 10 || g_masked == nullptr || g_masked_fwd_ws == nullptr || g_masked_rows == nullptr || g_masked_bwd == nullptr || g_few_rows == nullptr ||
      (q = tensor_of(args[0])) == nullptr || (k = tensor_of(args[1])) == nullptr || (v = tensor_of(args[2])) == nullptr ||
      (m = tensor_of(args[3])) == nullptr || !int_of(args[4], mb) || !int_of(args[5], mq) || !int_of(args[6], mk) || !optional_tensor(args[7], sl) ||
      !float_of(args[8], softcap) || !float_of(args[9], scale)) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
  if (!here(*q) || q->dim() != 4 || k->dim() != 4 || k->sizes() != v->sizes() || q->scalar_type() != at::kBFloat16 || k->scalar_type() != at::kBFloat16 ||
      v->scalar_type() != at::kBFloat16 || k->device() != q->device() || v->device() != q->device() || m->device() != q->device())
    Py_RETURN_NONE;
  const int64_t B = q->size(0), Sq = q->size(1), Hq = q->size(2), D = q->size(3), Skv = k->size(1), Hkv = k->size(2);
  Pitch pq, pk, pv;
  if (B != mb || Sq != mq || Skv != mk || k->size(0) != B || k->size(3) != D || (D != 64 && D != 128) || Hkv < 1 || Hq < 1 || Hq % Hkv != 0 ||
      !bshd(*q, pq) || !bshd(*k, pk) || !bshd(*v, pv) || !((float)scale > 0.f && (float)scale < INFINITY) ||
      !(softcap == 0.0 || (softcap >= 1e-12 && softcap <= 1e18)) || m->scalar_type() != at::kInt || !m->is_contiguous())
    Py_RETURN_NONE;
  if (sl.defined() && (sl.device() != q->device() || sl.scalar_type() != at::kFloat || sl.dim() != 1 || sl.size(0) != Hq || !sl.is_contiguous()))
    Py_RETURN_NONE;
  at::Tensor out;
  {
    pybind11::gil_scoped_release nogil;
    const bool grad = ag::compute_requires_grad(*q, *k, *v);
    const auto o = q->options().requires_grad(false);
    out = at::empty({B, Sq, Hq, D}, o);
    at::Tensor lse = at::empty({B, Hq, Sq}, o.dtype(at::kFloat)), low;
    if (!grad && g_few_rows((int)B, (int)Sq, (int)Hq, (int)Hkv)) {
      const long long n = g_rows_ws((int)B, (int)Sq, (int)Skv, (int)Hq, (int)Hkv, (int)D);
      at::Tensor ws = workspace(n, *q);
      check_rc("b200_attn_masked_rows",
               g_masked_rows(q->data_ptr(), k->data_ptr(), v->data_ptr(), out.data_ptr(), lse.data_ptr<float>(), nullptr, floats_of(sl), m->data_ptr<int>(),
                             (int)B, (int)Sq, (int)Skv, (int)Hq, (int)Hkv, (int)D, pq.row, pk.row, pv.row, pq.batch, pk.batch, pv.batch, (float)scale,
                             (float)softcap, n > 0 ? ws.data_ptr() : nullptr, n, stream_of(*q)));
    } else {
      if (grad) low = at::empty({B, Sq, Hq, D}, o);
      const long long n = g_masked_fwd_ws((int)B, (int)Sq, (int)Skv, (int)Hq, (int)D);
      at::Tensor ws = workspace(n, *q);
      check_rc("b200_attn_masked_fwd",
               g_masked(q->data_ptr(), k->data_ptr(), v->data_ptr(), out.data_ptr(), grad ? low.data_ptr() : nullptr, lse.data_ptr<float>(), nullptr,
                        floats_of(sl), m->data_ptr<int>(), (int)B, (int)Sq, (int)Skv, (int)Hq, (int)Hkv, (int)D, pq.row, pk.row, pv.row, pq.batch, pk.batch,
                        pv.batch, (float)scale, (float)softcap, n > 0 ? ws.data_ptr() : nullptr, n, stream_of(*q)));
    }
    if (grad) {
      auto node = std::shared_ptr<MaskedAttentionBackward>(new MaskedAttentionBackward(), ag::deleteNode);
      node->softcap = (float)softcap;
      node->scale = (float)scale;
      set_node(node, out, ag::collect_next_edges(*q, *k, *v));
      node->q = ag::SavedVariable(*q, false);
      node->k = ag::SavedVariable(*k, false);
      node->v = ag::SavedVariable(*v, false);
      node->out = ag::SavedVariable(out, true);
      node->low = ag::SavedVariable(low, false);
      node->lse = ag::SavedVariable(lse, false);
      node->slopes = ag::SavedVariable(sl.defined() ? sl.detach() : sl, false);
      node->mask = ag::SavedVariable(*m, false);
    }
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// attention_mask(documents or None, prefix or None, B, Sq, Skv, causal, window, index of the device): the mask's buffer
PyObject* py_attention_mask(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  at::Tensor ids, flags;
  long long B, Sq, Skv, causal, window, dev;
  if (nargs != 8 || g_mask == nullptr || g_mask_ints == nullptr || !optional_tensor(args[0], ids) || !optional_tensor(args[1], flags) ||
      !int_of(args[2], B) || !int_of(args[3], Sq) || !int_of(args[4], Skv) || !int_of(args[5], causal) || !int_of(args[6], window) ||
      !int_of(args[7], dev)) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
  if (B < 1 || Sq < 1 || Skv < Sq || Skv > (1 << 30) || B > 0x7fffffff || window < 0 || window >= (1 << 30) || dev != c10::cuda::current_device())
    Py_RETURN_NONE;
  for (const at::Tensor* t : {&ids, &flags})
    if (t->defined() && (!here(*t) || t->dim() != 2 || t->size(0) != B || t->size(1) != Skv || !t->is_contiguous())) Py_RETURN_NONE;
  if ((ids.defined() && ids.scalar_type() != at::kInt && ids.scalar_type() != at::kLong) || (flags.defined() && (flags.scalar_type() != at::kBool || !causal)))
    Py_RETURN_NONE;
  at::Tensor buf;
  {
    pybind11::gil_scoped_release nogil;
    const long long n = g_mask_ints((int)B, (int)Sq, (int)Skv);
    TORCH_CHECK(n > 0, "attention_mask: ", B, " x ", Sq, " x ", Skv);
    buf = at::empty({n}, at::TensorOptions().dtype(at::kInt).device(at::kCUDA, (c10::DeviceIndex)dev));
    check_rc("b200_attn_mask", g_mask(ids.defined() ? ids.data_ptr() : nullptr, ids.defined() && ids.scalar_type() == at::kLong,
                                      flags.defined() ? reinterpret_cast<const uint8_t*>(flags.data_ptr()) : nullptr, (int)B, (int)Sq, (int)Skv,
                                      (int)causal, (int)window, buf.data_ptr<int>(), stream_of(buf)));
  }
  return THPVariable_Wrap(std::move(buf));
  END_HANDLE_TH_ERRORS
}

// bind_masked(addresses of b200_attn_masked_few_rows, _rows_workspace, _bwd_workspace, b200_attn_mask_ints, b200_attn_masked_fwd_workspace)
PyObject* py_bind_masked(PyObject*, PyObject* args) {
  unsigned long long a, b, c, d, e;
  if (!PyArg_ParseTuple(args, "KKKKK", &a, &b, &c, &d, &e)) return nullptr;
  g_masked_fwd_ws = reinterpret_cast<long long (*)(int, int, int, int, int)>(e);
  g_mask_ints = reinterpret_cast<long long (*)(int, int, int)>(d);
  g_few_rows = reinterpret_cast<int (*)(int, int, int, int)>(a);
  g_rows_ws = reinterpret_cast<long long (*)(int, int, int, int, int, int)>(b);
  g_masked_bwd_ws = reinterpret_cast<long long (*)(int, int, int, int, int, int)>(c);
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"bind_masked", py_bind_masked, METH_VARARGS, nullptr},
    {"attention_mask", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_attention_mask)), METH_FASTCALL, nullptr},
    {"route", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_route)), METH_FASTCALL, nullptr},
    {"distill_loss", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_distill_loss)), METH_FASTCALL, nullptr},
    {"masked_attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_masked_attention)), METH_FASTCALL, nullptr},
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
