// The operators of beam/_C.py for the ordinary call: plain torch tensors, no tile named, nothing to report.
//
// A call of a small product is bound by the host: through ctypes, 5.1 us for gemmrc at 64^3, of which the launch takes 3.3 and
// the rest is attribute look-ups on three tensors and the conversion of ten arguments.  Here the tensors' fields are read
// where they lie.  Same machine, us for a call returning, through ctypes -> here: gemmrc and matmul 5.1 -> 3.1, split-K 6.0 ->
// 3.6, GEMM+LayerNorm 7.1 -> 3.8 (checked, with the wait for the result, 19.3 -> 15.4), GEMM and SiLU 9.1 (two launches) -> 4.4,
// MXFP4 quantising and reading back 14.6 -> 7.6 (both).
//
// Every function returns the library's status (0: done), or kNotHandled before anything is launched: beam/_C.py then takes its
// general path, which also words the errors.  So nothing here has to be complete, and nothing here may differ from there.
// The interpreter's lock is released around the library's calls, as ctypes does.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <c10/hip/HIPCachingAllocator.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <climits>
#include <cstdint>

#include "../../include/beam_hip.h"

namespace {

constexpr long kNotHandled = -1;
constexpr long kFellBack = -2;  // gemmrc_ln: the call repeated itself as two passes

struct View {
  void* ptr;
  const int64_t* size;
  int64_t numel;
  int dims;
  int dtype;
};

// What _C._describe tells of a torch tensor; false: not an ordinary one.  (Subclasses, and wrappers without memory of their
// own, whose pointer throws, are the general path's.)
bool describe(PyObject* o, View* v) {
  if (!THPVariable_CheckExact(o)) return false;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || !t.is_contiguous()) return false;
  const at::ScalarType s = t.scalar_type();
  if (s == at::kHalf) v->dtype = BEAM_F16;
  else if (s == at::kBFloat16) v->dtype = BEAM_BF16;
  else return false;
  v->ptr = t.data_ptr();
  v->size = t.sizes().data();
  v->dims = (int)t.dim();
  v->numel = t.numel();
  return true;
}

struct Problem {
  View a, b, c;
  int M, N, K;
  void* stream;
};

// [M, K] x [N, K] (or [K, N]) -> [M, N] of one type, and where a launch goes: the current device's current stream.
bool problem(PyObject* const* args, bool b_kmajor, Problem* q) {
  if (!describe(args[0], &q->a) || !describe(args[1], &q->b) || !describe(args[2], &q->c)) return false;
  if (q->a.dims != 2 || q->b.dims != 2 || q->c.dims != 2 || q->a.dtype != q->b.dtype || q->a.dtype != q->c.dtype) return false;
  const int64_t M = q->a.size[0], K = q->a.size[1], N = q->b.size[b_kmajor ? 1 : 0];
  if (q->b.size[b_kmajor ? 0 : 1] != K || q->c.size[0] != M || q->c.size[1] != N || M > INT_MAX || N > INT_MAX || K > INT_MAX) return false;
  q->M = (int)M;
  q->N = (int)N;
  q->K = (int)K;
  q->stream = c10::hip::getCurrentHIPStream().stream();
  return true;
}

// Runs f, which returns a status or kNotHandled, and hands its value on.  Whatever a tensor throws is left to the general path.
template <typename F>
PyObject* status_of(F f) {
  long s = kNotHandled;
  try {
    s = f();
  } catch (...) {
  }
  if (PyErr_Occurred()) PyErr_Clear();
  return PyLong_FromLong(s);
}

PyObject* gemmrc(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return status_of([&]() -> long {
    Problem q;
    if (n != 3 || !problem(args, false, &q)) return kNotHandled;
    int rc;
    Py_BEGIN_ALLOW_THREADS;
    rc = beam_gemmrc(q.a.ptr, q.b.ptr, q.c.ptr, q.M, q.N, q.K, q.a.dtype, nullptr, q.stream);
    Py_END_ALLOW_THREADS;
    return rc;
  });
}

PyObject* matmul(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return status_of([&]() -> long {
    Problem q;
    if (n != 3 || !problem(args, true, &q)) return kNotHandled;
    int rc;
    Py_BEGIN_ALLOW_THREADS;
    rc = beam_matmul_nn(q.a.ptr, q.b.ptr, q.c.ptr, q.M, q.N, q.K, q.a.dtype, nullptr, q.stream);
    Py_END_ALLOW_THREADS;
    return rc;
  });
}

// (a, b, c, workspace, its bytes): the library's choice of tile and slices
PyObject* gemmrc_splitk(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return status_of([&]() -> long {
    Problem q;
    if (n != 5 || !problem(args, false, &q)) return kNotHandled;
    void* const ws = PyLong_AsVoidPtr(args[3]);
    const size_t ws_bytes = PyLong_AsSize_t(args[4]);
    if (PyErr_Occurred()) return kNotHandled;
    const int s = beam_splitk_effective(q.M, q.N, q.K, nullptr, 0);
    if (s < 0 || (s > 1 && beam_splitk_workspace_bytes(q.M, q.N, s) > ws_bytes)) return kNotHandled;
    int rc;
    Py_BEGIN_ALLOW_THREADS;
    rc = beam_gemmrc_splitk(q.a.ptr, q.b.ptr, q.c.ptr, q.M, q.N, q.K, q.a.dtype, nullptr, 0, s > 1 ? ws : nullptr, s > 1 ? ws_bytes : 0, q.stream);
    Py_END_ALLOW_THREADS;
    return rc;
  });
}

// (a, b, c, gamma, beta, eps, check, workspace, its bytes): BEAM_LN_AUTO
PyObject* gemmrc_ln(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return status_of([&]() -> long {
    Problem q;
    View g, bt;
    if (n != 9 || !problem(args, false, &q) || !describe(args[3], &g) || !describe(args[4], &bt)) return kNotHandled;
    if (g.dims != 1 || bt.dims != 1 || g.size[0] != q.N || bt.size[0] != q.N || g.dtype != q.a.dtype || bt.dtype != q.a.dtype) return kNotHandled;
    const double eps = PyFloat_AsDouble(args[5]);
    const int check = PyObject_IsTrue(args[6]);
    void* const ws = PyLong_AsVoidPtr(args[7]);
    const size_t ws_bytes = PyLong_AsSize_t(args[8]);
    if (PyErr_Occurred()) return kNotHandled;
    const bool aligned = (((uintptr_t)q.a.ptr | (uintptr_t)q.b.ptr | (uintptr_t)q.c.ptr) & 15) == 0 && (((uintptr_t)g.ptr | (uintptr_t)bt.ptr) & 7) == 0;
    int rc, fell_back = 0;
    bool room;
    Py_BEGIN_ALLOW_THREADS;
    // (the query may be the first call of the process and set the device up)
    room = ws && ws_bytes >= (aligned ? beam_gemmrc_ln_workspace_bytes_for(q.M, q.N, q.K, nullptr, BEAM_LN_AUTO)
                                      : beam_gemmrc_ln_workspace_bytes_ex(q.M, q.N, nullptr, BEAM_LN_AUTO));
    rc = !room ? 0
         : check ? beam_gemmrc_ln_checked(q.a.ptr, q.b.ptr, g.ptr, bt.ptr, (float)eps, q.c.ptr, q.M, q.N, q.K, q.a.dtype, nullptr, ws, ws_bytes,
                                          q.stream, &fell_back)
                 : beam_gemmrc_ln_ex(q.a.ptr, q.b.ptr, g.ptr, bt.ptr, (float)eps, q.c.ptr, q.M, q.N, q.K, q.a.dtype, nullptr, BEAM_LN_AUTO, ws,
                                     ws_bytes, q.stream);
    Py_END_ALLOW_THREADS;
    return !room ? kNotHandled : rc == 0 && fell_back ? kFellBack : rc;
  });
}

// (a, b, c, x, y)
PyObject* parallel_gemmrc_silu(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return status_of([&]() -> long {
    Problem q;
    View x, y;
    if (n != 5 || !problem(args, false, &q) || !describe(args[3], &x) || !describe(args[4], &y)) return kNotHandled;
    if (x.numel != y.numel || x.dtype != q.a.dtype || y.dtype != q.a.dtype) return kNotHandled;
    int rc;
    Py_BEGIN_ALLOW_THREADS;
    rc = beam_parallel_gemmrc_silu(q.a.ptr, q.b.ptr, q.c.ptr, q.M, q.N, q.K, x.ptr, y.ptr, x.numel, q.a.dtype, nullptr, q.stream);
    Py_END_ALLOW_THREADS;
    return rc;
  });
}

// ---- feed-forward operators.  They run on whatever GPU their tensors lie on; here only where that is the current one.

int current_device() {
  int d = -1;
  return hipGetDevice(&d) == hipSuccess ? d : -1;
}

bool on_device(PyObject* o, int device) { return THPVariable_Unpack(o).device().index() == device; }

// A 16-bit matrix on `device`.
bool matrix(PyObject* o, int device, View* v) { return describe(o, v) && v->dims == 2 && v->size[0] <= INT_MAX && v->size[1] <= INT_MAX && on_device(o, device); }

bool is_matrix(PyObject* o, int device, int dtype, int64_t rows, int64_t cols, View* v) {
  return matrix(o, device, v) && v->dtype == dtype && v->size[0] == rows && v->size[1] == cols;
}

// Elements and scales in MXFP4 on `device`, and what they stand for.
struct Held {
  void* elements;
  void* scales;
  int64_t rows, cols;
};
bool held(PyObject* q, PyObject* s, int device, Held* h) {
  if (!THPVariable_CheckExact(q) || !THPVariable_CheckExact(s)) return false;
  const at::Tensor& e = THPVariable_Unpack(q);
  const at::Tensor& t = THPVariable_Unpack(s);
  for (const at::Tensor* x : {&e, &t})
    if (!x->defined() || !x->is_cuda() || x->layout() != at::kStrided || !x->is_contiguous() || x->scalar_type() != at::kByte || x->device().index() != device) return false;
  if (e.dim() != 2 || t.dim() != 3 || e.size(0) > INT_MAX / 4 || e.size(1) > INT_MAX / 4) return false;
  h->rows = e.size(0);
  h->cols = 2 * e.size(1);
  h->elements = e.data_ptr();
  h->scales = t.data_ptr();
  return h->cols % 32 == 0 && t.size(0) == (h->cols + 255) / 256 && t.size(1) == h->rows && t.size(2) == 8;
}

// Workspace of one call, from torch's allocator: it goes back when the call returns, to calls behind it on its stream.
c10::DataPtr call_workspace(size_t bytes) { return bytes ? c10::hip::HIPCachingAllocator::get()->allocate(bytes) : c10::DataPtr(); }

// (a, b, h, gu or None)
PyObject* gemmrc_gated(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return status_of([&]() -> long {
    View a, b, h, gu;
    const int dev = current_device();
    if (n != 4 || !matrix(args[0], dev, &a) || !matrix(args[1], dev, &b)) return kNotHandled;
    const int64_t M = a.size[0], K = a.size[1], N2 = b.size[0];
    if (b.dtype != a.dtype || b.size[1] != K || N2 % 2 != 0 || !is_matrix(args[2], dev, a.dtype, M, N2 / 2, &h)) return kNotHandled;
    const bool train = args[3] != Py_None;
    if (train && !is_matrix(args[3], dev, a.dtype, M, N2, &gu)) return kNotHandled;
    void* const stream = c10::hip::getCurrentHIPStream().stream();
    int rc;
    Py_BEGIN_ALLOW_THREADS;
    rc = beam_gemmrc_gated(a.ptr, b.ptr, h.ptr, train ? gu.ptr : nullptr, (int)M, (int)(N2 / 2), (int)K, a.dtype, stream);
    Py_END_ALLOW_THREADS;
    return rc;
  });
}

// (dh, gu, a, b, da or None, db or None)
PyObject* gemmrc_gated_backward(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return status_of([&]() -> long {
    View dh, gu, a, b, da, db;
    const int dev = current_device();
    if (n != 6 || !matrix(args[2], dev, &a) || !matrix(args[3], dev, &b)) return kNotHandled;
    const int64_t M = a.size[0], K = a.size[1], N2 = b.size[0];
    if (b.dtype != a.dtype || b.size[1] != K || N2 % 2 != 0) return kNotHandled;
    if (!is_matrix(args[0], dev, a.dtype, M, N2 / 2, &dh) || !is_matrix(args[1], dev, a.dtype, M, N2, &gu)) return kNotHandled;
    const bool want_a = args[4] != Py_None, want_b = args[5] != Py_None;
    if ((want_a && !is_matrix(args[4], dev, a.dtype, M, K, &da)) || (want_b && !is_matrix(args[5], dev, a.dtype, N2, K, &db))) return kNotHandled;
    void* const stream = c10::hip::getCurrentHIPStream().stream();
    const size_t bytes = beam_gemmrc_gated_backward_workspace_bytes((int)M, (int)(N2 / 2), (int)K, want_a, want_b);
    const c10::DataPtr ws = call_workspace(bytes);
    int rc;
    Py_BEGIN_ALLOW_THREADS;
    rc = beam_gemmrc_gated_backward(dh.ptr, gu.ptr, a.ptr, b.ptr, want_a ? da.ptr : nullptr, want_b ? db.ptr : nullptr, (int)M, (int)(N2 / 2), (int)K,
                                    a.dtype, ws.get(), bytes, stream);
    Py_END_ALLOW_THREADS;
    return rc;
  });
}

// (x, q, scales)
PyObject* mxfp4_quantize(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return status_of([&]() -> long {
    View x;
    Held h;
    const int dev = current_device();
    if (n != 3 || !matrix(args[0], dev, &x) || !held(args[1], args[2], dev, &h) || x.size[0] != h.rows || x.size[1] != h.cols) return kNotHandled;
    void* const stream = c10::hip::getCurrentHIPStream().stream();
    int rc;
    Py_BEGIN_ALLOW_THREADS;
    rc = beam_mxfp4_quantize(x.ptr, h.elements, h.scales, (int)h.rows, (int)h.cols, x.dtype, stream);
    Py_END_ALLOW_THREADS;
    return rc;
  });
}

// (q, scales, x)
PyObject* mxfp4_dequantize(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return status_of([&]() -> long {
    View x;
    Held h;
    const int dev = current_device();
    if (n != 3 || !matrix(args[2], dev, &x) || !held(args[0], args[1], dev, &h) || x.size[0] != h.rows || x.size[1] != h.cols) return kNotHandled;
    void* const stream = c10::hip::getCurrentHIPStream().stream();
    int rc;
    Py_BEGIN_ALLOW_THREADS;
    rc = beam_mxfp4_dequantize(h.elements, h.scales, x.ptr, (int)h.rows, (int)h.cols, x.dtype, stream);
    Py_END_ALLOW_THREADS;
    return rc;
  });
}

// (a, a_scales, b, b_scales, c)
PyObject* gemmrc_mxfp4(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return status_of([&]() -> long {
    View c;
    Held a, b;
    const int dev = current_device();
    if (n != 5 || !held(args[0], args[1], dev, &a) || !held(args[2], args[3], dev, &b) || a.cols != b.cols || !matrix(args[4], dev, &c)) return kNotHandled;
    if (c.size[0] != a.rows || c.size[1] != b.rows) return kNotHandled;
    void* const stream = c10::hip::getCurrentHIPStream().stream();
    int rc;
    Py_BEGIN_ALLOW_THREADS;
    rc = beam_gemmrc_mxfp4(a.elements, a.scales, b.elements, b.scales, c.ptr, (int)a.rows, (int)b.rows, (int)a.cols, c.dtype, stream);
    Py_END_ALLOW_THREADS;
    return rc;
  });
}

// (a, b, b_scales, c)
PyObject* linear_mxfp4(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return status_of([&]() -> long {
    View a, c;
    Held b;
    const int dev = current_device();
    if (n != 4 || !matrix(args[0], dev, &a) || !held(args[1], args[2], dev, &b) || a.size[1] != b.cols) return kNotHandled;
    if (!is_matrix(args[3], dev, a.dtype, a.size[0], b.rows, &c)) return kNotHandled;
    void* const stream = c10::hip::getCurrentHIPStream().stream();
    const size_t bytes = beam_linear_mxfp4_workspace_bytes((int)a.size[0], (int)b.cols);
    const c10::DataPtr ws = call_workspace(bytes);
    int rc;
    Py_BEGIN_ALLOW_THREADS;
    rc = beam_linear_mxfp4(a.ptr, b.elements, b.scales, c.ptr, (int)a.size[0], (int)b.rows, (int)b.cols, a.dtype, ws.get(), bytes, stream);
    Py_END_ALLOW_THREADS;
    return rc;
  });
}

#define BEAM_METHOD(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, nullptr}
PyMethodDef kMethods[] = {BEAM_METHOD(gemmrc),    BEAM_METHOD(matmul),
                          BEAM_METHOD(gemmrc_splitk), BEAM_METHOD(gemmrc_ln),
                          BEAM_METHOD(parallel_gemmrc_silu),
                          BEAM_METHOD(gemmrc_gated), BEAM_METHOD(gemmrc_gated_backward),
                          BEAM_METHOD(mxfp4_quantize), BEAM_METHOD(mxfp4_dequantize),
                          BEAM_METHOD(gemmrc_mxfp4), BEAM_METHOD(linear_mxfp4), {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_torch_binding", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_binding() { return PyModule_Create(&kModule); }
