// call.cpp — the Python module blackhole_b200._call: the calls of experts.py for
// arguments that need no second look.
//
// A small product or activation is over on the GPU in 2 to 10 us; reading a dozen
// tensor attributes, allocating the result and passing the arguments through
// ctypes takes Python 4 to 8 us more than this module does, and a list of 40
// gradients with their copies 35 us more.  Each function here looks at its
// arguments, allocates what the call needs, makes it on the current stream and
// returns the result; or it returns None, having done nothing, where anything is
// out of the ordinary (another device than the current one, a stride that wants a
// copy, a type or shape that does not fit, inputs that autograd follows, arguments that the call refuses), and
// experts.py takes the call from there, with its checks and messages.  A call that
// failed on the way, with some of its work perhaps done, raises.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <exception>
#include <optional>
#include <stdexcept>
#include <string>
#include <vector>

#include "hexmoe.h"

namespace {

// A plain tensor argument; nullptr where it is none.
const at::Tensor* tensor(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

int code_of(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return HEXMOE_F32;
    case at::kBFloat16: return HEXMOE_BF16;
    case at::kHalf: return HEXMOE_F16;
    default: return -1;
  }
}

// On the current CUDA device, strided.
bool here(const at::Tensor& t) {
  return t.is_cuda() && t.layout() == at::kStrided && t.get_device() == c10::cuda::current_device();
}
// Autograd is to see a call with this input.
bool recorded(const at::Tensor& t) { return c10::GradMode::is_enabled() && t.requires_grad(); }
void* stream_of(const at::Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }
bool matrix(const at::Tensor& t) { return t.dim() == 2 && t.stride(1) == 1 && t.stride(0) >= t.size(1); }

// int32 or int64 [experts + 1], contiguous: its code, or -1.
int offsets_code(const at::Tensor& o, int64_t experts) {
  if (!here(o) || o.dim() != 1 || o.size(0) != experts + 1 || o.stride(0) != 1) return -1;
  return o.scalar_type() == at::kInt ? HEXMOE_I32 : o.scalar_type() == at::kLong ? HEXMOE_I64 : -1;
}

at::Tensor workspace(size_t bytes, const at::Tensor& like) {
  return at::empty({static_cast<int64_t>(bytes)}, like.options().dtype(at::kByte));
}

// Whether a call refused its arguments, before any work.  Any other failure may have come after a launch: made once
// more, the call could scale what it has scaled already.
bool refused(int rc, const char* what) {
  if (rc == HEXMOE_OK) return false;
  if (rc == HEXMOE_E_ARG || rc == HEXMOE_E_DTYPE) return true;
  throw std::runtime_error(std::string(what) + ": " + hexmoe_last_error());
}

// C++ exceptions (an allocation or a launch that fails) become Python's.
template <typename F>
PyObject* guarded(F&& f) {
  try {
    return f();
  } catch (const c10::OutOfMemoryError&) {
    Py_RETURN_NONE;   // the Python path meets it again and raises torch's own exception
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// (x, w, offsets, transpose)
PyObject* grouped_mm(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    const at::Tensor *x = n_args == 4 ? tensor(a[0]) : nullptr, *w = x ? tensor(a[1]) : nullptr,
                     *off = w ? tensor(a[2]) : nullptr;
    if (!off || !here(*x) || !here(*w) || x->scalar_type() != w->scalar_type() || !matrix(*x) || w->dim() != 3 ||
        recorded(*x) || recorded(*w))
      Py_RETURN_NONE;
    const int code = code_of(x->scalar_type()), transpose = a[3] == Py_True;
    const int64_t E = w->size(0), N = w->size(1), K = w->size(2), R = x->size(0);
    const int index = offsets_code(*off, E);
    if (code <= HEXMOE_F32 || index < 0 || (a[3] != Py_True && a[3] != Py_False) || w->stride(2) != 1 ||
        w->stride(1) < K || N >= (1 << 24) || K >= (1 << 24) || x->size(1) != (transpose ? N : K))
      Py_RETURN_NONE;
    const int64_t width = transpose ? K : N;
    at::Tensor out = at::empty({R, width}, x->options());
    const size_t bytes = hexmoe_grouped_mm_workspace_bytes(R, E, N, K, transpose);
    at::Tensor ws;
    if (bytes) ws = workspace(bytes, *x);
    const int rc = hexmoe_grouped_mm(x->data_ptr(), x->stride(0), w->data_ptr(), w->stride(1), w->stride(0), code, R,
                                     E, N, K, transpose, off->data_ptr(), index, out.data_ptr(), width, code,
                                     bytes ? ws.data_ptr() : nullptr, bytes, stream_of(*x));
    if (refused(rc, "hexmoe_grouped_mm")) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(out));
  });
}

// (dy, x, offsets, f32): f32 asks for a float32 result
PyObject* grouped_wgrad(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    const at::Tensor *dy = n_args == 4 ? tensor(a[0]) : nullptr, *x = dy ? tensor(a[1]) : nullptr,
                     *off = x ? tensor(a[2]) : nullptr;
    if (!off || !here(*dy) || !here(*x) || dy->scalar_type() != x->scalar_type() || !matrix(*dy) || !matrix(*x) ||
        off->dim() != 1 || off->size(0) < 2 || recorded(*dy) || recorded(*x))
      Py_RETURN_NONE;
    const int code = code_of(x->scalar_type());
    const int64_t E = off->size(0) - 1, N = dy->size(1), K = x->size(1), R = x->size(0);
    const int index = offsets_code(*off, E);
    if (code <= HEXMOE_F32 || index < 0 || dy->size(0) != R || N >= (1 << 24) || K >= (1 << 24)) Py_RETURN_NONE;
    const bool f32 = a[3] == Py_True;
    at::Tensor out = at::empty({E, N, K}, f32 ? x->options().dtype(at::kFloat) : x->options());
    const size_t bytes = hexmoe_grouped_wgrad_workspace_bytes(R, E, N, K);
    at::Tensor ws;
    if (bytes) ws = workspace(bytes, *x);
    const int rc = hexmoe_grouped_wgrad(dy->data_ptr(), dy->stride(0), x->data_ptr(), x->stride(0), code, R, E, N, K,
                                        off->data_ptr(), index, out.data_ptr(), K, N * K, f32 ? HEXMOE_F32 : code, 0,
                                        bytes ? ws.data_ptr() : nullptr, bytes, stream_of(*x));
    if (refused(rc, "hexmoe_grouped_wgrad")) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(out));
  });
}

// float32 [rows] or None: false where it is neither
bool row_weights(PyObject* o, int64_t rows, const float** p) {
  *p = nullptr;
  if (o == Py_None) return true;
  const at::Tensor* t = tensor(o);
  if (!t || !here(*t) || t->scalar_type() != at::kFloat || t->dim() != 1 || t->size(0) != rows ||
      (rows > 1 && t->stride(0) != 1))
    return false;
  *p = t->data_ptr<float>();
  return true;
}

// (h, row_weights)
PyObject* swiglu(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    const at::Tensor* h = n_args == 2 ? tensor(a[0]) : nullptr;
    const float* weights = nullptr;
    if (!h || !here(*h) || code_of(h->scalar_type()) < 0 || !matrix(*h) || h->size(1) % 2 || !h->size(1) ||
        h->size(1) > (1 << 30) || !row_weights(a[1], h->size(0), &weights) || recorded(*h) ||
        (weights && recorded(*tensor(a[1]))))
      Py_RETURN_NONE;
    const int64_t rows = h->size(0), inter = h->size(1) / 2;
    at::Tensor act = at::empty({rows, inter}, h->options());
    const int rc = hexmoe_swiglu(h->data_ptr(), code_of(h->scalar_type()), rows, inter, h->stride(0), weights,
                                 act.data_ptr(), inter, stream_of(*h));
    if (refused(rc, "hexmoe_swiglu")) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(act));
  });
}

// (dact, h, row_weights): (dh, drow_weights or None)
PyObject* swiglu_backward(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    const at::Tensor *dact = n_args == 3 ? tensor(a[0]) : nullptr, *h = dact ? tensor(a[1]) : nullptr;
    const float* weights = nullptr;
    if (!h || !here(*h) || !here(*dact) || code_of(h->scalar_type()) < 0 || dact->scalar_type() != h->scalar_type() ||
        !matrix(*h) || !matrix(*dact) || h->size(1) % 2 || !h->size(1) || h->size(1) > (1 << 30) ||
        dact->size(0) != h->size(0) || dact->size(1) * 2 != h->size(1) || !row_weights(a[2], h->size(0), &weights))
      Py_RETURN_NONE;
    const int64_t rows = dact->size(0), inter = dact->size(1);
    at::Tensor dh = at::empty({rows, 2 * inter}, h->options()), dw;
    if (weights || a[2] != Py_None) dw = at::empty({rows}, h->options().dtype(at::kFloat));
    const int rc = hexmoe_swiglu_backward(dact->data_ptr(), dact->stride(0), h->data_ptr(), h->stride(0),
                                          code_of(h->scalar_type()), rows, inter, weights, dh.data_ptr(), 2 * inter,
                                          dw.defined() ? dw.data_ptr<float>() : nullptr, stream_of(*h));
    if (refused(rc, "hexmoe_swiglu_backward")) Py_RETURN_NONE;
    PyObject* first = THPVariable_Wrap(std::move(dh));
    if (!first) return nullptr;
    PyObject* second = Py_None;
    if (dw.defined()) {
      second = THPVariable_Wrap(std::move(dw));
      if (!second) {
        Py_DECREF(first);
        return nullptr;
      }
    } else {
      Py_INCREF(Py_None);
    }
    PyObject* both = PyTuple_Pack(2, first, second);
    Py_DECREF(first);
    Py_DECREF(second);
    return both;
  });
}

// (grads, out or None, max_norm, inf): grads and out are lists
PyObject* clip_grad_norm(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    if (n_args != 4 || !PyList_Check(a[0]) || (a[1] != Py_None && !PyList_Check(a[1])) || !PyFloat_Check(a[2]))
      Py_RETURN_NONE;
    const Py_ssize_t n = PyList_GET_SIZE(a[0]);
    const bool copies = a[1] != Py_None;
    if (n == 0 || n > (1 << 16) || (copies && PyList_GET_SIZE(a[1]) != n)) Py_RETURN_NONE;
    std::vector<const void*> src(n);
    std::vector<void*> dst(copies ? n : 0);
    std::vector<int64_t> counts(n);
    std::vector<int32_t> types(n), dst_types(copies ? n : 0);
    int device = -1;
    auto dense_here = [&](const at::Tensor* t, int32_t* type) {
      if (!t || !t->is_cuda() || t->layout() != at::kStrided || !t->is_contiguous()) return false;
      if (device < 0) device = c10::cuda::current_device();
      if (t->get_device() != device) return false;
      return (*type = code_of(t->scalar_type())) >= 0;
    };
    const at::Tensor* first = nullptr;
    for (Py_ssize_t i = 0; i < n; ++i) {
      const at::Tensor* g = tensor(PyList_GET_ITEM(a[0], i));
      if (!dense_here(g, &types[i])) Py_RETURN_NONE;
      src[i] = g->data_ptr();
      counts[i] = g->numel();
      if (!first) first = g;
      if (copies) {
        const at::Tensor* o = tensor(PyList_GET_ITEM(a[1], i));
        if (!dense_here(o, &dst_types[i]) || o->sizes() != g->sizes()) Py_RETURN_NONE;
        dst[i] = o->data_ptr();
      }
    }
    const double max_norm = PyFloat_AS_DOUBLE(a[2]);
    const size_t bytes = hexmoe_clip_grad_norm_workspace_bytes(static_cast<int32_t>(n));
    at::Tensor norm = at::empty({}, first->options().dtype(at::kFloat)), ws = workspace(bytes, *first);
    const int rc = hexmoe_clip_grad_norm(static_cast<int32_t>(n), src.data(), counts.data(), types.data(),
                                         copies ? dst.data() : nullptr, copies ? dst_types.data() : nullptr,
                                         static_cast<float>(max_norm), a[3] == Py_True, norm.data_ptr<float>(),
                                         ws.data_ptr(), bytes, stream_of(*first));
    if (refused(rc, "hexmoe_clip_grad_norm")) Py_RETURN_NONE;
    for (Py_ssize_t i = 0; i < n; ++i) {   // autograd, which may hold what was written, looks at its version
      const at::Tensor& written = *tensor(PyList_GET_ITEM(a[copies], i));
      if (!written.is_inference()) written.unsafeGetTensorImpl()->bump_version();
    }
    return THPVariable_Wrap(std::move(norm));
  });
}

PyMethodDef methods[] = {
    {"grouped_mm", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(grouped_mm)), METH_FASTCALL, nullptr},
    {"grouped_wgrad", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(grouped_wgrad)), METH_FASTCALL, nullptr},
    {"swiglu", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(swiglu)), METH_FASTCALL, nullptr},
    {"swiglu_backward", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(swiglu_backward)), METH_FASTCALL, nullptr},
    {"clip_grad_norm", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(clip_grad_norm)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_call", "Calls of blackhole_b200.experts for ordinary arguments.", -1, methods};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__call(void) { return PyModule_Create(&module_def); }
