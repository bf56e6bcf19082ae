// The eager call of the 4-bit and group-norm operators as CPython functions over the C ABI.
//
// A call through ctypes costs 13 to 19 us on the host (operand checks, one to three allocations, twenty argument
// conversions), a multiple of what these kernels take for few rows.  The functions here do the same for the usual case --
// CUDA tensors of a supported type whose rows the kernels take as they are -- and return None for every other: the
// Python layer then does it step by step, with its copies, its other cases and its errors.  No kernel and no arithmetic
// here.
#include <Python.h>

#include <ATen/ops/empty.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/pq_b200.h"

namespace {

using at::Tensor;

// the tensor behind a Python object, or nullptr for anything else
const Tensor* tensor_of(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

bool aligned(const Tensor& t, uintptr_t a) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % a == 0; }
int dtype_code(at::ScalarType t) { return t == at::kBFloat16 ? PQ_DTYPE_BF16 : (t == at::kHalf ? PQ_DTYPE_FP16 : -1); }
bool plain(const Tensor& t, at::ScalarType type, c10::Device device) {
  return t.scalar_type() == type && t.device() == device && t.layout() == at::kStrided && t.is_contiguous();
}
Tensor make(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) { return at::empty(sizes, like.options().dtype(type)); }
void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

PyObject* none() { Py_RETURN_NONE; }
PyObject* fail(const char* what, int rc) {
  if (rc == PQ_ERR_CUDA) PyErr_Format(PyExc_RuntimeError, "%s: %s (cudaError %d)", what, pq_status_str(rc), pq_last_cuda_error());
  else PyErr_Format(PyExc_RuntimeError, "%s: %s", what, pq_status_str(rc));
  return nullptr;
}
// a tuple of new references; an undefined tensor becomes None
PyObject* tuple_of(std::initializer_list<const Tensor*> v) {
  PyObject* t = PyTuple_New(static_cast<Py_ssize_t>(v.size()));
  if (t == nullptr) return nullptr;
  Py_ssize_t i = 0;
  for (const Tensor* e : v) {
    PyObject* o = e->defined() ? THPVariable_Wrap(*e) : Py_NewRef(Py_None);
    if (o == nullptr) { Py_DECREF(t); return nullptr; }
    PyTuple_SET_ITEM(t, i++, o);
  }
  return t;
}
PyObject* tuple2(const Tensor& a, const Tensor& b) { return tuple_of({&a, &b}); }
PyObject* tuple3(const Tensor& a, const Tensor& b, const Tensor& c) { return tuple_of({&a, &b, &c}); }

// C++ exceptions (allocation failures, a bad device) become Python's
template <typename F>
PyObject* guarded(F&& f) {
  try {
    return f();
  } catch (const c10::OutOfMemoryError& e) {
    PyObject* torch = PyImport_ImportModule("torch");
    PyObject* type = torch != nullptr ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
    PyErr_SetString(type != nullptr ? type : PyExc_RuntimeError, e.what_without_backtrace());
    Py_XDECREF(type);
    Py_XDECREF(torch);
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

// Allocation and launch run without the interpreter lock, like a call through ctypes: a launch waits while the queue is full, and
// what it waits for may need another Python thread.
struct Unlocked {
  PyThreadState* state = PyEval_SaveThread();
  Unlocked() = default;
  Unlocked(const Unlocked&) = delete;
  Unlocked& operator=(const Unlocked&) = delete;
  ~Unlocked() { PyEval_RestoreThread(state); }
};

Tensor scale_tensor(int64_t M, int64_t K, int fmt, const Tensor& like) {
  const int64_t per = fmt == PQ_FP4_MX ? 128 : 64;
  return make({(M + 127) / 128, (K + per - 1) / per, 512}, at::kByte, like);
}
// packed rows as the quantising operators return them; `row` nullptr: mx
bool plain_rows(const Tensor* codes, const Tensor* scales, const Tensor* row) {
  if (codes == nullptr || scales == nullptr || !codes->is_cuda() || codes->dim() != 2) return false;
  const int64_t M = codes->size(0), K2 = codes->size(1), per = row == nullptr ? 64 : 32;
  return plain(*codes, at::kByte, codes->device()) && aligned(*codes, 16) && K2 > 0 && K2 % 16 == 0 && plain(*scales, at::kByte, codes->device()) &&
         scales->dim() == 3 && scales->size(0) == (M + 127) / 128 && scales->size(1) == (K2 + per - 1) / per && scales->size(2) == 512 &&
         (row == nullptr || (plain(*row, at::kFloat, codes->device()) && row->dim() == 1 && row->size(0) == M));
}
// a rank-32 factor of the product in fp32
bool plain_low(const Tensor& t, int64_t rows, c10::Device device) {
  return plain(t, at::kFloat, device) && t.dim() == 2 && t.size(0) == rows && t.size(1) == 32 && aligned(t, 16);
}
// an argument that is a tensor or None; false for anything else
bool optional_tensor(PyObject* o, const Tensor** t) {
  *t = o == Py_None ? nullptr : tensor_of(o);
  return o == Py_None || *t != nullptr;
}

// quant_rows_fp4(x [M,K], fmt) -> (codes, scales, row scales or None), or None
PyObject* quant_rows_fp4(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    const Tensor* xp = n == 2 ? tensor_of(a[0]) : nullptr;
    if (xp == nullptr || !xp->is_cuda() || xp->dim() != 2 || xp->layout() != at::kStrided) return none();
    const Tensor& x = *xp;
    const int code = dtype_code(x.scalar_type()), fmt = static_cast<int>(PyLong_AsLong(a[1]));
    const int64_t M = x.size(0), K = x.size(1);
    if (code < 0 || K <= 0 || K % 32 != 0 || x.stride(1) != 1 || (M > 1 && (x.stride(0) % 16 != 0 || x.stride(0) < K)) || !aligned(x, 32)) return none();
    Tensor codes, scales, row;
    int rc;
    {
      Unlocked unlocked;
      c10::cuda::CUDAGuard guard(x.device());
      codes = make({M, K / 2}, at::kByte, x);
      scales = scale_tensor(M, K, fmt, x);
      if (fmt == PQ_FP4_NV) row = make({M}, at::kFloat, x);
      rc = pq_quant_rows_fp4(x.data_ptr(), code, M, K, M > 1 ? x.stride(0) : K, fmt, codes.data_ptr<uint8_t>(), scales.data_ptr<uint8_t>(),
                             row.defined() ? row.data_ptr<float>() : nullptr, stream_of(x));
    }
    return rc == PQ_OK ? tuple3(codes, scales, row) : fail("pq_quant_rows_fp4", rc);
  });
}

// dequant_rows_fp4(codes, scales, row scales or None, bf16?) -> [M,K], or None
PyObject* dequant_rows_fp4(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    const Tensor* row;
    if (n != 4 || !optional_tensor(a[2], &row)) return none();
    const Tensor *codes = tensor_of(a[0]), *scales = tensor_of(a[1]);
    if (!plain_rows(codes, scales, row)) return none();
    const bool bf16 = a[3] == Py_True;
    const int64_t M = codes->size(0), K = codes->size(1) * 2;
    Tensor out;
    int rc;
    {
      Unlocked unlocked;
      c10::cuda::CUDAGuard guard(codes->device());
      out = make({M, K}, bf16 ? at::kBFloat16 : at::kHalf, *codes);
      rc = pq_dequant_rows_fp4(codes->data_ptr<uint8_t>(), K / 2, scales->data_ptr<uint8_t>(), row != nullptr ? row->data_ptr<float>() : nullptr,
                               row != nullptr ? PQ_FP4_NV : PQ_FP4_MX, out.data_ptr(), bf16 ? PQ_DTYPE_BF16 : PQ_DTYPE_FP16, K, M, K,
                               stream_of(*codes));
    }
    return rc == PQ_OK ? THPVariable_Wrap(out) : fail("pq_dequant_rows_fp4", rc);
  });
}

// fp4_gemm(codes, scales, rows or None of x, the same of w, bias or None, bf16?, workspace, its bytes, low-rank rows t and lb or
// None) -> [M,N], or None
PyObject* fp4_gemm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    const Tensor *x_row, *w_row, *bias, *t, *lb;
    if (n != 12 || !optional_tensor(a[2], &x_row) || !optional_tensor(a[5], &w_row) || !optional_tensor(a[6], &bias) ||
        !optional_tensor(a[10], &t) || !optional_tensor(a[11], &lb) || (t == nullptr) != (lb == nullptr))
      return none();
    const Tensor *xq = tensor_of(a[0]), *xs = tensor_of(a[1]), *wq = tensor_of(a[3]), *ws = tensor_of(a[4]);
    if (!plain_rows(xq, xs, x_row) || !plain_rows(wq, ws, w_row) || (x_row == nullptr) != (w_row == nullptr) ||
        wq->device() != xq->device() || wq->size(1) != xq->size(1) || wq->size(0) == 0)
      return none();
    const int64_t M = xq->size(0), N = wq->size(0), K = xq->size(1) * 2;
    if (bias != nullptr && (!plain(*bias, at::kFloat, xq->device()) || bias->numel() != N)) return none();
    if (t != nullptr && !(plain_low(*t, M, xq->device()) && plain_low(*lb, N, xq->device()))) return none();
    const bool bf16 = a[7] == Py_True;
    void* const workspace = PyLong_AsVoidPtr(a[8]);
    const size_t ws_bytes = PyLong_AsSize_t(a[9]);
    Tensor out;
    int rc;
    {
      Unlocked unlocked;
      c10::cuda::CUDAGuard guard(xq->device());
      out = make({M, N}, bf16 ? at::kBFloat16 : at::kHalf, *xq);
      auto floats = [](const Tensor* v) { return v != nullptr ? v->data_ptr<float>() : nullptr; };
      rc = pq_fp4_gemm_lowrank(xq->data_ptr<uint8_t>(), K / 2, xs->data_ptr<uint8_t>(), floats(x_row), wq->data_ptr<uint8_t>(), K / 2,
                               ws->data_ptr<uint8_t>(), floats(w_row), floats(bias), floats(t), floats(lb),
                               x_row != nullptr ? PQ_FP4_NV : PQ_FP4_MX, out.data_ptr(), bf16 ? PQ_DTYPE_BF16 : PQ_DTYPE_FP16, N, M, N, K,
                               workspace, ws_bytes, stream_of(*xq));
    }
    return rc == PQ_OK ? THPVariable_Wrap(out) : fail("pq_fp4_gemm", rc);
  });
}

// fp4_lowrank_rows(t [M,32], row scales or None) -> fp32 [M,32], or None
PyObject* fp4_lowrank_rows(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    const Tensor *t = n == 2 ? tensor_of(a[0]) : nullptr, *row;
    if (t == nullptr || !optional_tensor(a[1], &row) || !t->is_cuda() || t->dim() != 2 || t->size(1) != 32) return none();
    const int code = dtype_code(t->scalar_type());
    const int64_t M = t->size(0);
    if (code < 0 || !plain(*t, t->scalar_type(), t->device()) || !aligned(*t, 16)) return none();
    if (row != nullptr && !(plain(*row, at::kFloat, t->device()) && row->dim() == 1 && row->size(0) == M)) return none();
    Tensor out;
    int rc;
    {
      Unlocked unlocked;
      c10::cuda::CUDAGuard guard(t->device());
      out = make({M, 32}, at::kFloat, *t);
      rc = pq_fp4_lowrank_rows(t->data_ptr(), code, row != nullptr ? row->data_ptr<float>() : nullptr, out.data_ptr<float>(), M, stream_of(*t));
    }
    return rc == PQ_OK ? THPVariable_Wrap(out) : fail("pq_fp4_lowrank_rows", rc);
  });
}

// fp4_lowrank_factors(t [M,32], row scales or None, B [32,N], column scales or None) -> (fp32 [M,32], fp32 [N,32]), or None
PyObject* fp4_lowrank_factors(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    const Tensor *t = n == 4 ? tensor_of(a[0]) : nullptr, *b = n == 4 ? tensor_of(a[2]) : nullptr, *row, *col;
    if (t == nullptr || b == nullptr || !optional_tensor(a[1], &row) || !optional_tensor(a[3], &col) || !t->is_cuda() || t->dim() != 2 ||
        t->size(1) != 32 || b->dim() != 2 || b->size(0) != 32)
      return none();
    const int tc = dtype_code(t->scalar_type()), bc = dtype_code(b->scalar_type());
    const int64_t M = t->size(0), N = b->size(1);
    if (tc < 0 || bc < 0 || !plain(*t, t->scalar_type(), t->device()) || !aligned(*t, 16) || !plain(*b, b->scalar_type(), t->device())) return none();
    if (row != nullptr && !(plain(*row, at::kFloat, t->device()) && row->dim() == 1 && row->size(0) == M)) return none();
    if (col != nullptr && !(plain(*col, at::kFloat, t->device()) && col->dim() == 1 && col->size(0) == N)) return none();
    Tensor t_out, b_out;
    int rc;
    {
      Unlocked unlocked;
      c10::cuda::CUDAGuard guard(t->device());
      t_out = make({M, 32}, at::kFloat, *t);
      b_out = make({N, 32}, at::kFloat, *t);
      rc = pq_fp4_lowrank_factors(t->data_ptr(), tc, row != nullptr ? row->data_ptr<float>() : nullptr, t_out.data_ptr<float>(), M, b->data_ptr(),
                                  bc, N, col != nullptr ? col->data_ptr<float>() : nullptr, b_out.data_ptr<float>(), N, stream_of(*t));
    }
    return rc == PQ_OK ? tuple2(t_out, b_out) : fail("pq_fp4_lowrank_factors", rc);
  });
}

// lowrank_layout(A [K,32] or None, B [32,N] or None) -> (A^T or None, B^T or None), contiguous; or None
PyObject* lowrank_layout(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    const Tensor *A, *B;
    if (n != 2 || !optional_tensor(a[0], &A) || !optional_tensor(a[1], &B) || (A == nullptr && B == nullptr)) return none();
    const Tensor& like = A != nullptr ? *A : *B;
    for (const Tensor* v : {A, B})
      if (v != nullptr && (!v->is_cuda() || v->dim() != 2 || dtype_code(v->scalar_type()) < 0 || !plain(*v, v->scalar_type(), like.device()))) return none();
    if ((A != nullptr && (A->size(1) != 32 || !aligned(*A, 16))) || (B != nullptr && B->size(0) != 32)) return none();
    const int64_t K = A != nullptr ? A->size(0) : 0, N = B != nullptr ? B->size(1) : 0;
    Tensor at, bt;
    int rc;
    {
      Unlocked unlocked;
      c10::cuda::CUDAGuard guard(like.device());
      if (A != nullptr) at = make({32, K}, A->scalar_type(), *A);
      if (B != nullptr) bt = make({N, 32}, B->scalar_type(), *B);
      rc = pq_lowrank_layout(A != nullptr ? A->data_ptr() : nullptr, 32, at.defined() ? at.data_ptr() : nullptr, K, B != nullptr ? B->data_ptr() : nullptr,
                             N, bt.defined() ? bt.data_ptr() : nullptr, N, stream_of(like));
    }
    return rc == PQ_OK ? tuple2(at, bt) : fail("pq_lowrank_layout", rc);
  });
}

// group_norm(x [B,T,C], groups, weight or None, bias or None, eps, act, mode, z wanted?, status word) with mode 0: z, 1: INT8, 2: mx, 3: nv
// -> z, (q, s, z or None), (codes, scales, row scales or None); None where the Python layer has to look; False for a size
// that the quantising forms do not take
PyObject* group_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    const Tensor *w, *b;
    const Tensor* xp = n == 9 ? tensor_of(a[0]) : nullptr;
    if (xp == nullptr || !optional_tensor(a[2], &w) || !optional_tensor(a[3], &b)) return none();
    const Tensor& x = *xp;
    if (!x.is_cuda() || x.dim() != 3 || !PyLong_Check(a[1])) return none();
    const int code = dtype_code(x.scalar_type());
    const int64_t B = x.size(0), T = x.size(1), C = x.size(2);
    const long groups = PyLong_AsLong(a[1]);
    const double eps = PyFloat_AsDouble(a[4]);
    const int act = static_cast<int>(PyLong_AsLong(a[5])), mode = static_cast<int>(PyLong_AsLong(a[6]));
    if (PyErr_Occurred() != nullptr) { PyErr_Clear(); return none(); }
    if (code < 0 || !plain(x, x.scalar_type(), x.device()) || !aligned(x, 16) || B * T == 0 || B > 65535 || groups <= 0 || groups > C || C % groups != 0 ||
        C % 8 != 0 || C > 8192 || (mode == 1 && C % 16 != 0) || (mode >= 2 && C % 32 != 0))
      return none();
    const bool grad = c10::GradMode::is_enabled();
    if (grad && x.requires_grad()) return none();
    for (const Tensor* v : {w, b})
      if (v != nullptr && (!plain(*v, x.scalar_type(), x.device()) || v->dim() != 1 || v->size(0) != C || !aligned(*v, 16) || (grad && v->requires_grad())))
        return none();
    void* const status = PyLong_AsVoidPtr(a[8]);
    const bool want_z = mode == 0 || a[7] == Py_True;
    Tensor z, q, scales, row;
    int rc;
    {
      Unlocked unlocked;
      c10::cuda::CUDAGuard guard(x.device());
      const void* wp = w != nullptr ? w->data_ptr() : nullptr;
      const void* bp = b != nullptr ? b->data_ptr() : nullptr;
      const int64_t bytes = pq_group_norm_workspace_bytes(B, T, C, static_cast<int>(groups));
      Tensor ws = make({bytes}, at::kByte, x);
      void* st = stream_of(x);
      const float e = static_cast<float>(eps);
      const int g = static_cast<int>(groups);
      if (mode < 2 && want_z) z = make({B, T, C}, x.scalar_type(), x);
      void* zp = z.defined() ? z.data_ptr() : nullptr;
      if (mode == 0) {
        rc = pq_group_norm(x.data_ptr(), code, B, T, C, C, T * C, g, wp, bp, 0, e, act, zp, C, T * C, ws.data_ptr(), bytes, status, st);
      } else if (mode == 1) {
        q = make({B * T, C}, at::kChar, x);
        row = make({B * T}, at::kFloat, x);
        rc = pq_group_norm_quant_rows(x.data_ptr(), code, B, T, C, C, T * C, g, wp, bp, 0, e, act, zp, C, T * C, q.data_ptr<int8_t>(),
                                      row.data_ptr<float>(), ws.data_ptr(), bytes, status, st);
      } else {
        const int fmt = mode == 2 ? PQ_FP4_MX : PQ_FP4_NV;
        q = make({B * T, C / 2}, at::kByte, x);
        scales = scale_tensor(B * T, C, fmt, x);
        if (fmt == PQ_FP4_NV) row = make({B * T}, at::kFloat, x);
        rc = pq_group_norm_quant_fp4(x.data_ptr(), code, B, T, C, C, T * C, g, wp, bp, 0, e, act, fmt, q.data_ptr<uint8_t>(), scales.data_ptr<uint8_t>(),
                                     row.defined() ? row.data_ptr<float>() : nullptr, ws.data_ptr(), bytes, status, st);
      }
    }
    if (rc == PQ_ERR_UNSUPPORTED) {
      if (mode == 0) return none();
      Py_RETURN_FALSE;
    }
    if (rc != PQ_OK) return fail(mode == 0 ? "pq_group_norm" : "pq_group_norm_quant", rc);
    return mode == 0 ? THPVariable_Wrap(z) : (mode == 1 ? tuple3(q, row, z) : tuple3(q, scales, row));
  });
}

#define PQ_FAST(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef kMethods[] = {PQ_FAST(quant_rows_fp4), PQ_FAST(dequant_rows_fp4), PQ_FAST(fp4_gemm), PQ_FAST(fp4_lowrank_rows), PQ_FAST(fp4_lowrank_factors), PQ_FAST(lowrank_layout),
                           PQ_FAST(group_norm), {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_bind", "eager calls of the 4-bit and group-norm operators", -1, kMethods,
                       nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__bind() { return PyModule_Create(&kModule); }
