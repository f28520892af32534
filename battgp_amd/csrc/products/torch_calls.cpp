// The calls of battgp_amd/products.py that need no second look, from torch tensors to the C entries without the time that
// reading a tensor's properties and filling in arguments takes from Python (7.3 us a call, of which the launch is 2.5).
// Every function answers None where anything is out of the ordinary - a type, a shape, a stride, a device, a gradient that
// is asked for, an error - and products.py then goes through its own checks, which say what is wrong.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <string>

#include "../../../include/battgp_products.h"

namespace {

using at::Tensor;

// What else than the numbers in its memory a tensor stands for: nothing, other tensors (inside vmap, jvp and grad, and
// wrappers, whose pointer may read as NULL), or a dual number.
enum Stands { FOR_ITSELF, FOR_OTHERS, WITH_TANGENT };
Stands stands(const Tensor& t) {
  if (!t.has_storage() || (t.numel() > 0 && !t.const_data_ptr())) return FOR_OTHERS;
  return t._fw_grad(0).defined() ? WITH_TANGENT : FOR_ITSELF;
}

// a dense tensor on the GPU that no gradient is recorded for, in neither mode; NULL if it is anything else
const Tensor* gpu_tensor(PyObject* o, int dim, int device = -1) {
  if (!THPVariable_Check(o)) return nullptr;
  const Tensor& t = THPVariable_Unpack(o);
  if (t.layout() != at::kStrided || !t.is_cuda() || t.dim() != dim || (device >= 0 && t.get_device() != device)) return nullptr;
  if (t.is_neg() || (t.requires_grad() && c10::GradMode::is_enabled()) || stands(t) != FOR_ITSELF) return nullptr;
  return &t;
}

int code_of(at::ScalarType t) {
  switch (t) {
    case at::kDouble: return BGP_F64;
    case at::kFloat: return BGP_F32;
    case at::kBFloat16: return BGP_BF16;
    case at::kHalf: return BGP_F16;
    default: return -1;
  }
}

// leading dimension of a matrix with contiguous rows, 0 if they are not
int64_t rows(const Tensor& t) {
  const int64_t m = t.size(0), n = t.size(1);
  if (n > 1 && t.stride(1) != 1) return 0;
  if (m <= 1) return n > 1 ? n : 1;
  if (t.stride(0) < n) return 0;
  return t.stride(0) > 0 ? t.stride(0) : 1;
}

struct Weights {
  int64_t stride, ld;
  int trans;
};
// of w[G, N, K]; turned: of its groups' transposes; ld 0 if neither axis of a group is contiguous
Weights weights(const Tensor& w, bool turned) {
  const int64_t n = turned ? w.size(2) : w.size(1), k = turned ? w.size(1) : w.size(2), g = w.size(0) > 1 ? w.stride(0) : 0;
  const int64_t sn = turned ? w.stride(2) : w.stride(1), sk = turned ? w.stride(1) : w.stride(2), one = 1;
  if ((sk == 1 || k <= 1) && (n <= 1 || sn >= std::max(k, one))) return Weights{g, n > 1 ? sn : std::max(k, one), 0};
  if ((sn == 1 || n <= 1) && (k <= 1 || sk >= std::max(n, one))) return Weights{g, k > 1 ? sk : std::max(n, one), 1};
  return Weights{0, 0, 0};
}

void* stream_of(int device) { return c10::hip::getCurrentHIPStream(static_cast<c10::DeviceIndex>(device)).stream(); }

// a C entry that may ask for a workspace; true if it did its work
template <class F> bool done(const Tensor& like, F&& call) {
  int64_t rc = call(nullptr, 0);
  if (rc > 0) {
    const Tensor work = at::empty({rc}, like.options().dtype(at::kByte));
    rc = call(work.data_ptr(), rc);
  }
  return rc == 0;
}

bool offsets_fit(const Tensor* off, int64_t groups) {
  return off && off->scalar_type() == at::kLong && off->size(0) == groups + 1 && groups <= BGP_MAX_GROUPS && (groups == 0 || off->stride(0) == 1);
}

// out[t, :] = x[t, :] w_g^T (turned: x[t, :] w_g)
bool rows_product(const Tensor& x, const Tensor& w, bool turned, const Tensor& off, int device, Tensor* out) {
  const int64_t t = x.size(0), k = x.size(1), g = w.size(0), n = turned ? w.size(2) : w.size(1), ldx = rows(x);
  const Weights l = weights(w, turned);
  if (!ldx || !l.ld) return false;
  *out = at::empty({t, n}, x.options());
  return done(x, [&](void* work, int64_t bytes) {
    return bgp_grouped_gemm(device, stream_of(device), code_of(x.scalar_type()), t, n, k, g, x.data_ptr(), ldx, w.data_ptr(), l.stride, l.ld, l.trans,
                            off.data_ptr<int64_t>(), out->data_ptr(), n > 1 ? n : 1, 1, work, bytes);
  });
}

template <class F> PyObject* guarded(F&& body) {
  try {
    if (PyObject* r = body()) return r;
  } catch (...) {  // e.g. no memory: the call is repeated from Python, where the error is raised
  }
  PyErr_Clear();
  Py_RETURN_NONE;
}

PyObject* grouped(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    const Tensor* x = n == 3 ? gpu_tensor(a[0], 2) : nullptr;
    if (!x || code_of(x->scalar_type()) < 0) return nullptr;
    const int device = x->get_device();
    const Tensor *w = gpu_tensor(a[1], 3, device), *off = gpu_tensor(a[2], 1, device);
    if (!w || w->scalar_type() != x->scalar_type() || w->size(2) != x->size(1) || !offsets_fit(off, w->size(0))) return nullptr;
    Tensor y;
    return rows_product(*x, *w, false, *off, device, &y) ? THPVariable_Wrap(y) : nullptr;
  });
}

PyObject* grouped_grad(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    const Tensor* x = n == 4 ? gpu_tensor(a[1], 2) : nullptr;
    if (!x || code_of(x->scalar_type()) < 0) return nullptr;
    const int device = x->get_device();
    const Tensor *dy = gpu_tensor(a[0], 2, device), *w = gpu_tensor(a[2], 3, device), *off = gpu_tensor(a[3], 1, device);
    if (!dy || !w || dy->scalar_type() != x->scalar_type() || w->scalar_type() != x->scalar_type() || w->size(2) != x->size(1) ||
        dy->size(0) != x->size(0) || dy->size(1) != w->size(1) || !offsets_fit(off, w->size(0)))
      return nullptr;
    const int64_t lddy = rows(*dy), ldx = rows(*x), g = w->size(0), nn = w->size(1), k = w->size(2), ldw = k > 1 ? k : 1;
    Tensor dx;
    if (!lddy || !ldx || !rows_product(*dy, *w, true, *off, device, &dx)) return nullptr;
    const Tensor dw = at::empty({g, nn, k}, x->options());
    if (!done(*x, [&](void* work, int64_t bytes) {
          return bgp_grouped_gemm_dw(device, stream_of(device), code_of(x->scalar_type()), x->size(0), nn, k, g, dy->data_ptr(), lddy, x->data_ptr(), ldx,
                                     off->data_ptr<int64_t>(), dw.data_ptr(), nn * ldw, ldw, work, bytes);
        }))
      return nullptr;
    PyObject* r = PyTuple_New(2);
    PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(dx));
    PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(dw));
    return r;
  });
}

PyObject* quantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    const Tensor* x = n == 3 ? gpu_tensor(a[0], 2) : nullptr;
    if (!x || code_of(x->scalar_type()) < 0) return nullptr;
    const int pow2 = PyObject_IsTrue(a[1]), residual = PyObject_IsTrue(a[2]);
    const int64_t ldx = rows(*x), m = x->size(0), k = x->size(1), ld = k > 1 ? k : 1;
    if (pow2 < 0 || residual < 0 || !ldx) return nullptr;
    const int device = x->get_device();
    const Tensor q = at::empty({m, k}, x->options().dtype(at::kChar));
    const Tensor scale = at::empty({m}, x->options().dtype(x->scalar_type() == at::kDouble ? at::kDouble : at::kFloat));
    const Tensor rest = residual ? at::empty({m, k}, x->options()) : Tensor();
    if (bgp_quantize_rows(device, stream_of(device), code_of(x->scalar_type()), m, k, x->data_ptr(), ldx, q.data_ptr<int8_t>(), ld, scale.data_ptr(), pow2,
                          residual ? rest.data_ptr() : nullptr, ld) != 0)
      return nullptr;
    PyObject* r = PyTuple_New(residual ? 3 : 2);
    PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(q));
    PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(scale));
    if (residual) PyTuple_SET_ITEM(r, 2, THPVariable_Wrap(rest));
    return r;
  });
}

// a, b, a_scale, b_scale, c or None, the result's type as one of the header's codes
PyObject* int8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    const Tensor* x = n == 6 ? gpu_tensor(a[0], 2) : nullptr;
    if (!x) return nullptr;
    const int device = x->get_device();
    const Tensor *b = gpu_tensor(a[1], 2, device), *sa = gpu_tensor(a[2], 1, device), *sb = gpu_tensor(a[3], 1, device);
    const Tensor* c = a[4] == Py_None ? nullptr : gpu_tensor(a[4], 2, device);
    const long code = PyLong_AsLong(a[5]);
    if (!b || !sa || !sb || (a[4] != Py_None && !c) || code < BGP_F64 || code > BGP_F16) return nullptr;
    static const at::ScalarType types[] = {at::kDouble, at::kFloat, at::kBFloat16, at::kHalf};
    const at::ScalarType type = types[code], stype = code == BGP_F64 ? at::kDouble : at::kFloat;
    const int64_t m = x->size(0), k = x->size(1), nn = b->size(0), lda = rows(*x), ldb = rows(*b);
    auto scales = [&](const Tensor& s, int64_t count) { return s.scalar_type() == stype && s.size(0) == count && (count <= 1 || s.stride(0) == 1); };
    if (x->scalar_type() != at::kChar || b->scalar_type() != at::kChar || b->size(1) != k || k > BGP_INT8_MAX_K || !lda || !ldb || !scales(*sa, m) || !scales(*sb, nn))
      return nullptr;
    int64_t ldc = 0;
    if (c && (c->scalar_type() != type || c->size(0) != m || c->size(1) != nn || !(ldc = rows(*c)))) return nullptr;
    const Tensor y = at::empty({m, nn}, x->options().dtype(type));
    return done(*x, [&](void* work, int64_t bytes) {
             return bgp_int8_gemm(device, stream_of(device), (int)code, m, nn, k, x->data_ptr<int8_t>(), lda, b->data_ptr<int8_t>(), ldb, sa->data_ptr(),
                                  sb->data_ptr(), c ? c->data_ptr() : nullptr, ldc, y.data_ptr(), nn > 1 ? nn : 1, work, bytes);
           })
               ? THPVariable_Wrap(y)
               : nullptr;
  });
}

// of any tensor: one of Stands
PyObject* stands_for(PyObject*, PyObject* o) {
  int r = FOR_OTHERS;
  try {
    if (THPVariable_Check(o)) r = stands(THPVariable_Unpack(o));
  } catch (...) {  // a pointer that is not to be asked for
  }
  return PyLong_FromLong(r);
}

PyMethodDef methods[] = {{"stands_for", (PyCFunction)stands_for, METH_O, nullptr},
                         {"grouped", (PyCFunction)(void*)grouped, METH_FASTCALL, nullptr},
                         {"grouped_grad", (PyCFunction)(void*)grouped_grad, METH_FASTCALL, nullptr},
                         {"quantize", (PyCFunction)(void*)quantize, METH_FASTCALL, nullptr},
                         {"int8", (PyCFunction)(void*)int8, METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_products_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__products_torch() { return PyModule_Create(&module); }
