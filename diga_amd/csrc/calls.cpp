// The short way from Python to the 8-bit row and matrix product entry points (diga_amd/matmul.py).
//
// A call from Python costs about 6 us of checks, allocations and argument conversion before the launch, two or three times what the
// kernels of a single token take.  Here the ordinary call -- plain tensors on the current GPU, of the documented types, shapes and
// layouts, none that needs a gradient -- is recognised, allocated for and launched in C++.  Anything else returns None, launches
// nothing, and the Python function goes on with its own checks: it alone says what is wrong, and takes the rarer layouts.  A launch
// that fails raises here: a second one of a norm in place would add the residual twice.
#include <Python.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_strided.h>

#include "../../include/diga_hip.h"

namespace {

decltype(&diga_rms_norm_fp8) f_rms_norm = nullptr;
decltype(&diga_silu_mul_fp8) f_silu_mul = nullptr;
decltype(&diga_quantize_fp8) f_quantize = nullptr;
decltype(&diga_matmul_fp8) f_matmul = nullptr;
decltype(&diga_grouped_matmul_fp8) f_grouped_fp8 = nullptr;
decltype(&diga_grouped_matmul) f_grouped = nullptr;
decltype(&diga_last_error_string) f_last_error = nullptr;
PyObject* error_type = nullptr;

using at::ScalarType;
constexpr ScalarType E4M3 = at::kFloat8_e4m3fn;

int type_code(ScalarType t) { return t == at::kBFloat16 ? DIGA_BF16 : t == at::kHalf ? DIGA_FP16 : t == at::kFloat ? DIGA_FP32 : -1; }

// the GPU that obj, the call's first tensor, is on, if that is the current one; -1 otherwise
int gpu_of(PyObject* obj) {
  if (!THPVariable_CheckExact(obj)) return -1;
  const at::Tensor& t = THPVariable_Unpack(obj);
  if (!t.is_cuda()) return -1;
  const int index = t.get_device();
  return index == c10::hip::current_device() ? index : -1;
}
// whether forward-mode differentiation would take t's tangent through the call
bool has_tangent(const at::Tensor& t) { return t._fw_grad(0).defined() && c10::AutogradState::get_tls_state().get_fw_grad_mode(); }
// obj as a plain tensor on GPU `index` that no derivative is asked of; NULL otherwise
const at::Tensor* plain(PyObject* obj, int index) {
  if (!THPVariable_CheckExact(obj)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(obj);
  if (!t.is_cuda() || t.get_device() != index || t.layout() != at::kStrided || t.is_neg()) return nullptr;
  return (t.requires_grad() && c10::GradMode::is_enabled()) || has_tangent(t) ? nullptr : &t;
}
// a matrix with adjacent columns
bool matrix(const at::Tensor& t, ScalarType type) { return t.dim() == 2 && t.scalar_type() == type && t.size(1) > 0 && t.stride(1) == 1; }
bool sizes_are(const at::Tensor& t, std::initializer_list<int64_t> s) { return t.sizes() == at::IntArrayRef(s); }

int64_t up16(int64_t n) { return (n + 15) / 16 * 16; }
int64_t blocks(int64_t n) { return (n + 127) / 128; }

struct Rows {
  at::Tensor q, scale;
  int64_t ldq;
  Rows(int64_t m, int64_t n, const at::Tensor& like) : ldq(up16(n)) {
    q = at::empty({m, ldq}, like.options().dtype(E4M3));
    if (ldq != n) q = q.narrow(1, 0, n);
    scale = at::empty_strided({m, blocks(n)}, {1, m}, like.options().dtype(at::kFloat));
  }
};

void* stream(int index) { return c10::hip::getCurrentHIPStream(index).stream(); }

// t was written in place: a later backward that saved it has to notice (inference tensors count no versions)
void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

PyObject* none() { Py_RETURN_NONE; }

// an entry point returned rc < 0: arguments it refuses are left to Python
PyObject* failed(const char* name, int rc) {
  if (rc == DIGA_EINVAL) return none();
  return PyErr_Format(error_type, "%s: error %d: %s", name, rc, f_last_error());
}

// rms_norm(x, weight, residual or None, eps, residual_out or None) -> (q, scale, h or None)
PyObject* rms_norm(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  if (n_args != 5 || !f_rms_norm || !PyFloat_Check(a[3])) return none();
  const int index = gpu_of(a[0]);
  if (index < 0) return none();
  const at::Tensor *x = plain(a[0], index), *w = plain(a[1], index), *r = nullptr, *given = nullptr;
  if (!x || !w || x->dim() != 2 || x->size(0) == 0) return none();
  const ScalarType type = x->scalar_type();
  const int code = type_code(type), wcode = type_code(w->scalar_type());
  const int64_t m = x->size(0), n = x->size(1);
  if (code < 0 || wcode < 0 || !matrix(*x, type) || n > DIGA_RMS_NORM_MAX_N || !sizes_are(*w, {n}) || !w->is_contiguous()) return none();
  at::Tensor h;
  if (a[2] != Py_None) {
    if (!(r = plain(a[2], index)) || !matrix(*r, type) || !sizes_are(*r, {m, n})) return none();
    if (a[4] != Py_None) {
      if (!(given = plain(a[4], index)) || !matrix(*given, type) || !sizes_are(*given, {m, n})) return none();
      h = *given;
    } else {
      h = at::empty({m, n}, x->options());
    }
  } else if (a[4] != Py_None) {
    return none();
  }
  Rows out(m, n, *x);
  const int rc = f_rms_norm(x->const_data_ptr(), x->stride(0), r ? r->const_data_ptr() : nullptr, r ? r->stride(0) : 0, code, w->const_data_ptr(), wcode,
                            (float)PyFloat_AS_DOUBLE(a[3]), m, (int)n, out.q.mutable_data_ptr(), out.ldq, out.scale.mutable_data_ptr<float>(), 1, m,
                            r ? h.mutable_data_ptr() : nullptr, r ? h.stride(0) : 0, stream(index));
  if (rc < 0) return failed("diga_rms_norm_fp8", rc);
  PyObject* hobj = Py_None;
  if (given) written(*given), hobj = a[4];
  if (!r || given) Py_INCREF(hobj);
  else hobj = THPVariable_Wrap(std::move(h));
  return Py_BuildValue("(NNN)", THPVariable_Wrap(std::move(out.q)), THPVariable_Wrap(std::move(out.scale)), hobj);
  END_HANDLE_TH_ERRORS
}

PyObject* act(PyObject* obj, decltype(f_silu_mul) f, bool gated) {
  const int index = gpu_of(obj);
  const at::Tensor* x = index >= 0 ? plain(obj, index) : nullptr;
  if (!f || !x || x->dim() != 2 || x->size(0) == 0) return none();
  const int code = type_code(x->scalar_type());
  const int64_t m = x->size(0), n = gated ? x->size(1) / 2 : x->size(1);
  if (code < 0 || !matrix(*x, x->scalar_type()) || n > (1 << 24) || (gated && x->size(1) % 2)) return none();
  Rows out(m, n, *x);
  const int rc = f(x->const_data_ptr(), x->stride(0), code, m, (int)n, out.q.mutable_data_ptr(), out.ldq, out.scale.mutable_data_ptr<float>(), 1, m, stream(index));
  if (rc < 0) return failed(gated ? "diga_silu_mul_fp8" : "diga_quantize_fp8", rc);
  return Py_BuildValue("(NN)", THPVariable_Wrap(std::move(out.q)), THPVariable_Wrap(std::move(out.scale)));
}
PyObject* silu_mul(PyObject*, PyObject* x) {
  HANDLE_TH_ERRORS
  return act(x, f_silu_mul, true);
  END_HANDLE_TH_ERRORS
}
PyObject* quantize(PyObject*, PyObject* x) {
  HANDLE_TH_ERRORS
  return act(x, f_quantize, false);
  END_HANDLE_TH_ERRORS
}

// The result of a product: `given` (None: a new one) of `type`, [m, n]; its tensor object with a reference of its own, or NULL
bool output(PyObject* given, int index, int64_t m, int64_t n, ScalarType type, const at::Tensor& like, at::Tensor& out) {
  if (given == Py_None) {
    out = at::empty({m, n}, like.options().dtype(type));
    return true;
  }
  const at::Tensor* t = plain(given, index);
  if (!t || !matrix(*t, type) || !sizes_are(*t, {m, n})) return false;
  out = *t;
  return true;
}
PyObject* returned(PyObject* given, at::Tensor&& out) {
  if (given == Py_None) return THPVariable_Wrap(std::move(out));
  written(out);
  Py_INCREF(given);
  return given;
}

// matmul(xq, xs, wq, ws, out_dtype, out or None)
PyObject* matmul(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  if (n_args != 6 || !f_matmul || !THPDtype_Check(a[4])) return none();
  const int index = gpu_of(a[0]);
  if (index < 0) return none();
  const at::Tensor *x = plain(a[0], index), *xs = plain(a[1], index), *w = plain(a[2], index), *ws = plain(a[3], index);
  const ScalarType type = reinterpret_cast<THPDtype*>(a[4])->scalar_type;
  if (!x || !xs || !w || !ws || (type != at::kBFloat16 && type != at::kHalf) || !matrix(*x, E4M3) || !matrix(*w, E4M3)) return none();
  const int64_t m = x->size(0), k = x->size(1), n = w->size(0);
  if (m == 0 || n == 0 || n > (1 << 24) || k > (1 << 23) || w->size(1) != k || k % 16 != 0) return none();
  if (xs->scalar_type() != at::kFloat || !sizes_are(*xs, {m, blocks(k)}) || ws->scalar_type() != at::kFloat || !sizes_are(*ws, {blocks(n), blocks(k)}) || !ws->is_contiguous())
    return none();
  at::Tensor out;
  if (!output(a[5], index, m, n, type, *x, out)) return none();
  const int rc = f_matmul(x->const_data_ptr(), m > 1 ? x->stride(0) : k, xs->const_data_ptr<float>(), xs->stride(0), xs->stride(1), w->const_data_ptr(),
                          n > 1 ? w->stride(0) : k, ws->const_data_ptr<float>(), out.mutable_data_ptr(), type_code(type), out.stride(0), m, (int)n, (int)k,
                          stream(index));
  return rc < 0 ? failed("diga_matmul_fp8", rc) : returned(a[5], std::move(out));
  END_HANDLE_TH_ERRORS
}

// grouped(x, xs or None, w, ws or None, offsets, rows or None, out_dtype, out or None): with scales e4m3, without bf16 / fp16
PyObject* grouped(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  if (n_args != 8 || !f_grouped || !f_grouped_fp8 || !THPDtype_Check(a[6])) return none();
  const int index = gpu_of(a[0]);
  if (index < 0) return none();
  const bool fp8 = a[1] != Py_None;
  const at::Tensor *x = plain(a[0], index), *w = plain(a[2], index), *off = plain(a[4], index), *rows = nullptr, *xs = nullptr, *ws = nullptr;
  if (!x || !w || !off || (a[5] != Py_None && !(rows = plain(a[5], index)))) return none();
  if (fp8 && (!(xs = plain(a[1], index)) || !(ws = plain(a[3], index)))) return none();
  const ScalarType type = x->scalar_type(), out_type = reinterpret_cast<THPDtype*>(a[6])->scalar_type;
  if (fp8 ? type != E4M3 || (out_type != at::kBFloat16 && out_type != at::kHalf) : (type != at::kBFloat16 && type != at::kHalf) || type_code(out_type) < 0) return none();
  if (!matrix(*x, type) || w->dim() != 3 || w->scalar_type() != type || w->numel() == 0 || w->stride(2) != 1) return none();
  const int64_t xr = x->size(0), k = x->size(1), e = w->size(0), n = w->size(1);
  if (xr == 0 || w->size(2) != k || n > (1 << 24) || k > (1 << 23) || e > 4096 || k % (fp8 ? 16 : 8) != 0) return none();
  if (off->scalar_type() != at::kInt || !sizes_are(*off, {e + 1}) || !off->is_contiguous()) return none();
  if (rows && (rows->scalar_type() != at::kInt || rows->dim() != 1 || !rows->is_contiguous())) return none();
  if (fp8 && (xs->scalar_type() != at::kFloat || !sizes_are(*xs, {xr, blocks(k)}) || ws->scalar_type() != at::kFloat || !sizes_are(*ws, {e, blocks(n), blocks(k)}) || !ws->is_contiguous()))
    return none();
  const int64_t t = rows ? rows->size(0) : xr, ldx = xr > 1 ? x->stride(0) : k, ldw = n > 1 ? w->stride(1) : k;
  if (t == 0) return none();
  at::Tensor out;
  if (!output(a[7], index, t, n, out_type, *x, out)) return none();
  const int32_t* r = rows ? rows->const_data_ptr<int32_t>() : nullptr;
  const int rc = fp8 ? f_grouped_fp8(x->const_data_ptr(), ldx, xr, xs->const_data_ptr<float>(), xs->stride(0), xs->stride(1), r, w->const_data_ptr(), ldw, w->stride(0),
                                     ws->const_data_ptr<float>(), off->const_data_ptr<int32_t>(), (int)e, out.mutable_data_ptr(), type_code(out_type), out.stride(0), t,
                                     (int)n, (int)k, stream(index))
                     : f_grouped(x->const_data_ptr(), ldx, xr, type_code(type), r, w->const_data_ptr(), ldw, w->stride(0), off->const_data_ptr<int32_t>(), (int)e,
                                 out.mutable_data_ptr(), type_code(out_type), out.stride(0), t, (int)n, (int)k, stream(index));
  return rc < 0 ? failed(fp8 ? "diga_grouped_matmul_fp8" : "diga_grouped_matmul", rc) : returned(a[7], std::move(out));
  END_HANDLE_TH_ERRORS
}

// bind(addresses of diga_rms_norm_fp8, diga_silu_mul_fp8, diga_quantize_fp8, diga_matmul_fp8, diga_grouped_matmul_fp8, diga_grouped_matmul,
// diga_last_error_string, the type of errors)
PyObject* bind(PyObject*, PyObject* args) {
  unsigned long long p[7];
  PyObject* type;
  if (!PyArg_ParseTuple(args, "KKKKKKKO", p, p + 1, p + 2, p + 3, p + 4, p + 5, p + 6, &type)) return nullptr;
  Py_INCREF(type);
  Py_XSETREF(error_type, type);
  f_last_error = reinterpret_cast<decltype(f_last_error)>(p[6]);
  f_rms_norm = reinterpret_cast<decltype(f_rms_norm)>(p[0]);
  f_silu_mul = reinterpret_cast<decltype(f_silu_mul)>(p[1]);
  f_quantize = reinterpret_cast<decltype(f_quantize)>(p[2]);
  f_matmul = reinterpret_cast<decltype(f_matmul)>(p[3]);
  f_grouped_fp8 = reinterpret_cast<decltype(f_grouped_fp8)>(p[4]);
  f_grouped = reinterpret_cast<decltype(f_grouped)>(p[5]);
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"bind", bind, METH_VARARGS, "addresses of the library's entry points"},
    {"rms_norm", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(rms_norm)), METH_FASTCALL, nullptr},
    {"silu_mul", silu_mul, METH_O, nullptr},
    {"quantize", quantize, METH_O, nullptr},
    {"matmul", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(matmul)), METH_FASTCALL, nullptr},
    {"grouped", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(grouped)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", "ordinary calls of diga_amd.matmul, recognised and launched in C++", -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__calls() { return PyModule_Create(&module); }
