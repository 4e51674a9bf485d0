// call.cpp — the Python module blackhole_b200._call: the calls of experts.py, router.py
// and int8.py for arguments that need no second look.
//
// A small product or activation is over on the GPU in 2 to 10 us; reading a dozen
// tensor attributes, allocating the result and passing the arguments through
// ctypes takes Python 4 to 8 us more than this module does, and a list of 40
// gradients with their copies 35 us more.  Each function here looks at its
// arguments, allocates what the call needs, makes it on the current stream and
// returns the result; or it returns None, having done nothing, where anything is
// out of the ordinary (another device than the current one, a stride that wants a
// copy, a type or shape that does not fit, inputs that autograd follows, arguments that the call refuses), and
// the Python function takes the call from there, with its checks and messages.  A call that
// failed on the way, with some of its work perhaps done, raises.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/AutogradState.h>
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
// Autograd is to see a call with this input: it requires a gradient, or has a tangent of forward-mode differentiation.
bool recorded(const at::Tensor& t) {
  return (c10::GradMode::is_enabled() && t.requires_grad()) ||
         (c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(0).defined());
}
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

// A plain int argument that fits; false where it is something else.
bool integer(PyObject* o, int32_t* v) {
  if (!PyLong_CheckExact(o)) return false;
  int overflow = 0;
  const long long n = PyLong_AsLongLongAndOverflow(o, &overflow);
  if (overflow || n < INT32_MIN || n > INT32_MAX) return false;
  *v = static_cast<int32_t>(n);
  return true;
}
bool truth(PyObject* o, int32_t* v) {
  *v = o == Py_True;
  return o == Py_True || o == Py_False;
}
// float32 of these sizes, contiguous, here
bool scales(const at::Tensor* t, at::IntArrayRef sizes) {
  return t && here(*t) && t->scalar_type() == at::kFloat && t->sizes() == sizes && t->is_contiguous();
}
// int8 matrices whose rows begin and repeat on multiples of 16 bytes, here
bool int8_stack(const at::Tensor& t) {
  return here(t) && t.scalar_type() == at::kChar && t.dim() == 3 && t.stride(2) == 1 && t.stride(1) >= t.size(2) &&
         t.stride(1) % 16 == 0 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 &&
         (t.size(0) == 1 || (t.stride(0) >= t.stride(1) && t.stride(0) % 16 == 0)) && t.size(0) <= INT32_MAX &&
         t.size(1) <= INT32_MAX && t.size(2) <= INT32_MAX;
}

// (logits, k, scoring, bias or None, groups, topk_groups or None, group_top, renormalize, scale): (weights, ids)
PyObject* route(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    const at::Tensor* l = n_args == 9 ? tensor(a[0]) : nullptr;
    int32_t k, scoring, groups, open_groups, group_top, renorm;
    if (!l || !here(*l) || code_of(l->scalar_type()) < 0 || !matrix(*l) || recorded(*l) || !integer(a[1], &k) ||
        !integer(a[2], &scoring) || !integer(a[4], &groups) || !integer(a[6], &group_top) || !truth(a[7], &renorm) ||
        !PyFloat_CheckExact(a[8]))
      Py_RETURN_NONE;
    if (a[5] == Py_None) open_groups = groups;
    else if (!integer(a[5], &open_groups)) Py_RETURN_NONE;
    const int64_t T = l->size(0), E = l->size(1);
    const at::Tensor* bias = a[3] == Py_None ? nullptr : tensor(a[3]);
    if ((a[3] != Py_None && !scales(bias, {E})) || E > INT32_MAX || k < 1 || k > 32) Py_RETURN_NONE;
    const auto f32 = l->options().dtype(at::kFloat);
    at::Tensor weights = at::empty({T, k}, f32), ids = at::empty({T, k}, f32.dtype(at::kInt));
    const int rc = hexmoe_route(l->data_ptr(), code_of(l->scalar_type()), l->stride(0), T, static_cast<int32_t>(E), k, scoring,
                                bias ? bias->data_ptr<float>() : nullptr, groups, open_groups, group_top, renorm,
                                static_cast<float>(PyFloat_AS_DOUBLE(a[8])), weights.data_ptr<float>(), ids.data_ptr<int32_t>(),
                                stream_of(*l));
    if (refused(rc, "hexmoe_route")) Py_RETURN_NONE;
    PyObject* first = THPVariable_Wrap(std::move(weights));
    if (!first) return nullptr;
    PyObject* second = THPVariable_Wrap(std::move(ids));
    if (!second) {
      Py_DECREF(first);
      return nullptr;
    }
    PyObject* both = PyTuple_Pack(2, first, second);
    Py_DECREF(first);
    Py_DECREF(second);
    return both;
  });
}

// (dweights, logits, ids, scoring, renormalize, scale)
PyObject* route_backward(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    const at::Tensor *d = n_args == 6 ? tensor(a[0]) : nullptr, *l = d ? tensor(a[1]) : nullptr, *ids = l ? tensor(a[2]) : nullptr;
    int32_t scoring, renorm;
    if (!ids || !here(*l) || !here(*ids) || code_of(l->scalar_type()) < 0 || !matrix(*l) || ids->dim() != 2 ||
        ids->size(0) != l->size(0) || ids->size(1) > INT32_MAX || !ids->is_contiguous() || !scales(d, ids->sizes()) ||
        (ids->scalar_type() != at::kInt && ids->scalar_type() != at::kLong) || !integer(a[3], &scoring) || !truth(a[4], &renorm) ||
        !PyFloat_CheckExact(a[5]) || l->size(1) > INT32_MAX)
      Py_RETURN_NONE;
    const int64_t T = l->size(0), E = l->size(1);
    at::Tensor out = at::empty({T, E}, l->options());
    const int rc = hexmoe_route_backward(d->data_ptr<float>(), l->data_ptr(), code_of(l->scalar_type()), l->stride(0), T,
                                         static_cast<int32_t>(E), static_cast<int32_t>(ids->size(1)), ids->data_ptr(),
                                         ids->scalar_type() == at::kLong ? HEXMOE_I64 : HEXMOE_I32, scoring, renorm,
                                         static_cast<float>(PyFloat_AS_DOUBLE(a[5])), out.data_ptr(), E, stream_of(*l));
    if (refused(rc, "hexmoe_route_backward")) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(out));
  });
}

// (x, w, w_scale, offsets): x of f32, bf16 or fp16, the result in its type
PyObject* grouped_mm_int8(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    const at::Tensor *x = n_args == 4 ? tensor(a[0]) : nullptr, *w = x ? tensor(a[1]) : nullptr, *s = w ? tensor(a[2]) : nullptr,
                     *off = s ? tensor(a[3]) : nullptr;
    if (!off || !here(*x) || code_of(x->scalar_type()) < 0 || !matrix(*x) || recorded(*x) || !int8_stack(*w) ||
        !scales(s, w->sizes().slice(0, 2)) || recorded(*s) || x->size(1) != w->size(2) || w->size(2) > 131071)
      Py_RETURN_NONE;
    const int64_t E = w->size(0), N = w->size(1), K = w->size(2), R = x->size(0);
    const int code = code_of(x->scalar_type()), index = offsets_code(*off, E);
    if (index < 0) Py_RETURN_NONE;
    at::Tensor out = at::empty({R, N}, x->options()), ws;
    const size_t bytes = hexmoe_grouped_mm_int8_workspace_bytes(R, E, N, K, code);
    if (bytes) ws = workspace(bytes, *x);
    const int rc = hexmoe_grouped_mm_int8(x->data_ptr(), code, x->stride(0), nullptr, w->data_ptr<int8_t>(), w->stride(1), w->stride(0),
                                          s->data_ptr<float>(), R, E, N, K, off->data_ptr(), index, out.data_ptr(), N, code,
                                          bytes ? ws.data_ptr() : nullptr, bytes, stream_of(*x));
    if (refused(rc, "hexmoe_grouped_mm_int8")) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(out));
  });
}

// (x, topk_weights, topk_ids, w13, w13_scale, w2, w2_scale)
PyObject* int8_moe(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    const at::Tensor* t[7] = {};
    for (int i = 0; i < 7; ++i)
      if (n_args != 7 || !(t[i] = tensor(a[i]))) Py_RETURN_NONE;
    const at::Tensor &x = *t[0], &weights = *t[1], &ids = *t[2], &w13 = *t[3], &s13 = *t[4], &w2 = *t[5], &s2 = *t[6];
    if (!here(x) || code_of(x.scalar_type()) < 0 || !matrix(x) || !here(ids) || ids.dim() != 2 || !ids.is_contiguous() ||
        (ids.scalar_type() != at::kInt && ids.scalar_type() != at::kLong) || !scales(&weights, ids.sizes()) ||
        !int8_stack(w13) || !int8_stack(w2) || !scales(&s13, w13.sizes().slice(0, 2)) || !scales(&s2, w2.sizes().slice(0, 2)) ||
        recorded(x) || recorded(weights) || recorded(s13) || recorded(s2))
      Py_RETURN_NONE;
    const int64_t T = ids.size(0), k = ids.size(1), E = w2.size(0), H = w2.size(1), I = w2.size(2);
    if (x.size(0) != T || x.size(1) != H || w13.size(0) != E || w13.size(1) != 2 * I || w13.size(2) != H || T == 0 || k == 0 || k > 1024)
      Py_RETURN_NONE;
    at::Tensor out = at::empty({T, H}, x.options());
    const int code = code_of(x.scalar_type());
    const size_t bytes = hexmoe_int8_forward_workspace_bytes(T, k, E, H, I);
    at::Tensor ws = workspace(bytes, x);
    const int rc = hexmoe_int8_forward(x.data_ptr(), code, x.stride(0), T, H, I, k, weights.data_ptr<float>(), ids.data_ptr(),
                                       ids.scalar_type() == at::kLong ? HEXMOE_I64 : HEXMOE_I32, E, w13.data_ptr<int8_t>(), w13.stride(1),
                                       w13.stride(0), s13.data_ptr<float>(), w2.data_ptr<int8_t>(), w2.stride(1), w2.stride(0),
                                       s2.data_ptr<float>(), out.data_ptr(), code, ws.data_ptr(), bytes, stream_of(x));
    if (refused(rc, "hexmoe_int8_forward")) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(out));
  });
}

PyMethodDef methods[] = {
    {"grouped_mm", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(grouped_mm)), METH_FASTCALL, nullptr},
    {"grouped_wgrad", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(grouped_wgrad)), METH_FASTCALL, nullptr},
    {"swiglu", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(swiglu)), METH_FASTCALL, nullptr},
    {"swiglu_backward", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(swiglu_backward)), METH_FASTCALL, nullptr},
    {"clip_grad_norm", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(clip_grad_norm)), METH_FASTCALL, nullptr},
    {"route", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(route)), METH_FASTCALL, nullptr},
    {"route_backward", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(route_backward)), METH_FASTCALL, nullptr},
    {"grouped_mm_int8", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(grouped_mm_int8)), METH_FASTCALL, nullptr},
    {"int8_moe", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(int8_moe)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_call", "Calls of blackhole_b200.experts, router and int8 for ordinary arguments.", -1, methods};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__call(void) { return PyModule_Create(&module_def); }
