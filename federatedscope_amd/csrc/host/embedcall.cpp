// Whole embedding calls of the plain form (include/fsagg.h), checked, allocated
// and launched in one C++ walk.
//
// A call of a few tokens is bound by the host: the Python way of a lookup
// takes 8.8 us a call in a run of calls, here 4.7 (its kernel 2.6), a gradient
// of 48 tokens 10.1 and 6.8 (5.6).  A round's row-sparse uploads are one
// (tokens, rows) pair per client, whose Python checks (device, types, shapes,
// strides, overlap) cost about 3 us, 100 clients' more than the kernels they
// launch; here they are a few TensorImpl reads each.
//
// embed_lookup(table, ids, scale, device, stream, fn) -> tensor or None
// embed_grad(ids, grads, coefs, num_rows, out, accumulate, device, stream,
//            size_fn, fn) -> tensor or None
//     ids, grads      equally long, non-empty lists of tensors
//     coefs           list of float, one per part
//     out             a tensor that no part may overlap, or None
//     device, stream  the current ones
//     fn, size_fn     addresses of fsagg_embed_lookup, fsagg_embed_grad and
//                     fsagg_embed_grad_workspace_bytes
// None is not an error: some tensor is not of the plain form (contiguous int64
// or int32 tokens; strided float32, float16 or bfloat16 rows of one type and
// width; all on the current device), or the library refused the call, and the
// caller's own checks say why.
//
// has_sparse(dict) -> bool: whether a value is a sparse COO tensor (asked of
// every upload, most of which have none: 161 keys 2 us, 19 us in Python).
// sparse_dicts(list) -> list of int: the places of the dicts for which it is
// (100 dicts of 161 keys 60 us).
#define PY_SSIZE_T_CLEAN
#include <ATen/ATen.h>
#include <Python.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <string>

namespace {

// struct fsagg_embed_part
struct EmbedPart {
  const void *ids;
  const void *rows;
  int64_t tokens, row_stride;
  float coef;
  int32_t ids64;
};

const c10::TensorImpl *tensor_of(PyObject *o) {
  return o && THPVariable_Check(o)
             ? THPVariable_Unpack(o).unsafeGetTensorImpl()
             : nullptr;
}

// the first element's address; false for a tensor that is not plain memory
// (nor for a view whose memory holds the negative of its values)
bool address(const c10::TensorImpl *t, uintptr_t &p) {
  if (t->layout() != c10::kStrided || !t->has_storage() ||
      t->key_set().has(c10::DispatchKey::Negative))
    return false;
  const void *d = t->storage().data();
  p = d ? reinterpret_cast<uintptr_t>(d) +
              uintptr_t(t->storage_offset()) * t->dtype().itemsize()
        : 0;
  return p != 0 || t->numel() == 0;
}

// FSAGG_F32, _F16, _BF16; -1 for other types
int code_of(const caffe2::TypeMeta &t) {
  return t == caffe2::TypeMeta::Make<float>()          ? 0
         : t == caffe2::TypeMeta::Make<at::Half>()     ? 1
         : t == caffe2::TypeMeta::Make<at::BFloat16>() ? 2
                                                       : -1;
}

struct Table {
  std::string buf;
  int64_t tokens = 0, dim = -1;
  int code = -1;
  caffe2::TypeMeta dtype;
  c10::Device dev{c10::kCPU};
};

// false: not of the plain form (or, with an error set, a factor that is no
// number)
bool walk(PyObject *ids, PyObject *grads, PyObject *coefs, uintptr_t lo,
          uintptr_t hi, Table &T) {
  const Py_ssize_t n = PyList_GET_SIZE(ids);
  if (n < 1 || PyList_GET_SIZE(grads) != n || PyList_GET_SIZE(coefs) != n)
    return false;
  T.buf.assign(size_t(n) * sizeof(EmbedPart), '\0');
  auto *part = reinterpret_cast<EmbedPart *>(&T.buf[0]);
  int64_t &tokens = T.tokens, &dim = T.dim;
  caffe2::TypeMeta &dtype = T.dtype;
  c10::Device &dev = T.dev;
  for (Py_ssize_t i = 0; i < n; ++i) {
    const c10::TensorImpl *t = tensor_of(PyList_GET_ITEM(ids, i));
    const c10::TensorImpl *g = tensor_of(PyList_GET_ITEM(grads, i));
    if (!t || !g) return false;
    uintptr_t pt, pg;
    if (!address(t, pt) || !address(g, pg)) return false;
    if (i == 0) {
      dev = g->device();
      dtype = g->dtype();
      T.code = code_of(dtype);
      if (T.code < 0 || !dev.is_cuda() || g->dim() < 1) return false;
      dim = g->sizes().back();
    }
    const bool i64 = t->dtype() == caffe2::TypeMeta::Make<int64_t>();
    if (g->device() != dev || t->device() != dev || g->dtype() != dtype ||
        (!i64 && t->dtype() != caffe2::TypeMeta::Make<int32_t>()) ||
        !t->is_contiguous() || g->dim() != t->dim() + 1 ||
        g->sizes().back() != dim)
      return false;
    for (int64_t d = 0; d < t->dim(); ++d)
      if (g->sizes()[d] != t->sizes()[d]) return false;
    const int64_t rows = t->numel();
    int64_t stride = dim;
    if (g->dim() == 2 && (dim <= 1 || g->strides()[1] == 1))
      stride = g->strides()[0];
    else if (!g->is_contiguous())
      return false;
    if (stride < 0 || rows > (int64_t(1) << 28)) return false;
    const uintptr_t size = dtype.itemsize();
    const uintptr_t gend =
        rows > 0 ? pg + (uintptr_t(rows - 1) * uintptr_t(stride) +
                         uintptr_t(dim)) * size
                 : pg;
    const uintptr_t tend = pt + uintptr_t(rows) * t->dtype().itemsize();
    if ((pg < hi && lo < gend) || (pt < hi && lo < tend)) return false;
    const double c = PyFloat_AsDouble(PyList_GET_ITEM(coefs, i));
    if (c == -1.0 && PyErr_Occurred()) return false;
    part[i] = {reinterpret_cast<const void *>(pt),
               reinterpret_cast<const void *>(pg), rows, stride, float(c),
               i64 ? 1 : 0};
    tokens += rows;
  }
  return true;
}

using LookupFn = int (*)(const void *, int64_t, int64_t, int64_t, int,
                         const void *, int, int64_t, float, void *, void *);
using SizeFn = size_t (*)(int64_t, int64_t, int64_t);
using GradFn = int (*)(const EmbedPart *, int, int, int64_t, int64_t, void *,
                       int, int64_t, int, void *, size_t, void *);

PyObject *lookup(PyObject *table, PyObject *ids, float scale, int device,
                 void *stream, LookupFn fn) {
  const c10::TensorImpl *t = tensor_of(table), *x = tensor_of(ids);
  uintptr_t pt, px;
  if (!t || !x || !address(t, pt) || !address(x, px)) Py_RETURN_NONE;
  const int code = code_of(t->dtype());
  const bool i64 = x->dtype() == caffe2::TypeMeta::Make<int64_t>();
  if (code < 0 || !t->device().is_cuda() || x->device() != t->device() ||
      (!i64 && x->dtype() != caffe2::TypeMeta::Make<int32_t>()) ||
      !x->is_contiguous() || t->dim() != 2 ||
      (t->sizes()[1] > 1 && t->strides()[1] != 1) ||
      t->device().index() != device)
    Py_RETURN_NONE;
  const int64_t dim = t->sizes()[1];
  c10::SmallVector<int64_t, 5> shape(x->sizes().begin(), x->sizes().end());
  shape.push_back(dim);
  at::Tensor out = at::empty(
      shape, at::TensorOptions().dtype(t->dtype()).device(t->device()));
  if (fn(reinterpret_cast<const void *>(pt), t->sizes()[0], dim,
         t->strides()[0], code, reinterpret_cast<const void *>(px), i64,
         x->numel(), scale, out.data_ptr(), stream) != 0)
    Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(out));
}

PyObject *grad(PyObject *ids, PyObject *grads, PyObject *coefs, int64_t rows,
               PyObject *out_obj, int accumulate, int device, void *stream,
               SizeFn size_fn, GradFn fn) {
  const bool given = out_obj != Py_None;
  const c10::TensorImpl *o = tensor_of(out_obj);
  if ((given && !o) || (accumulate && !given) || rows < 0) Py_RETURN_NONE;
  uintptr_t po = 0, hi = 0;
  int64_t stride = 0;
  if (given) {
    if (!address(o, po) || code_of(o->dtype()) < 0 || o->dim() != 2 ||
        o->sizes()[0] != rows)
      Py_RETURN_NONE;
    const int64_t dim = o->sizes()[1];
    stride = o->strides()[0];
    if ((dim > 1 && o->strides()[1] != 1) || (rows > 1 && stride < dim))
      Py_RETURN_NONE;
    if (o->numel() > 0)
      hi = po + (uintptr_t(rows - 1) * uintptr_t(stride) + uintptr_t(dim)) *
                    o->dtype().itemsize();
  }
  Table T;
  if (!walk(ids, grads, coefs, hi ? po : 0, hi, T)) {
    if (PyErr_Occurred()) return nullptr;
    Py_RETURN_NONE;
  }
  if (T.dev.index() != device ||
      (given && (o->sizes()[1] != T.dim || o->device() != T.dev)))
    Py_RETURN_NONE;
  const auto options = at::TensorOptions().device(T.dev);
  at::Tensor out =
      given ? THPVariable_Unpack(out_obj)
            : at::empty({rows, T.dim}, options.dtype(T.dtype));
  if (!given) stride = T.dim;
  const size_t need = size_fn(T.tokens, T.dim, rows);
  at::Tensor ws = at::empty({int64_t(need)}, options.dtype(at::kByte));
  if (fn(reinterpret_cast<const EmbedPart *>(T.buf.data()),
         int(PyList_GET_SIZE(ids)), T.code, rows, T.dim, out.data_ptr(),
         given ? code_of(o->dtype()) : T.code, stride, accumulate,
         need ? ws.data_ptr() : nullptr, need, stream) != 0)
    Py_RETURN_NONE;
  if (given) {
    Py_INCREF(out_obj);
    return out_obj;
  }
  return THPVariable_Wrap(std::move(out));
}


}  // namespace

PyObject *embed_lookup(PyObject *, PyObject *args) {
  PyObject *table, *ids;
  float scale;
  int device;
  unsigned long long stream, fn;
  if (!PyArg_ParseTuple(args, "OOfiKK", &table, &ids, &scale, &device,
                        &stream, &fn))
    return nullptr;
  try {
    return lookup(table, ids, scale, device, reinterpret_cast<void *>(stream),
                  reinterpret_cast<LookupFn>(fn));
  } catch (...) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
}

PyObject *embed_grad(PyObject *, PyObject *args) {
  PyObject *ids, *grads, *coefs, *out;
  long long rows;
  int accumulate, device;
  unsigned long long stream, size_fn, fn;
  if (!PyArg_ParseTuple(args, "O!O!O!LOpiKKK", &PyList_Type, &ids,
                        &PyList_Type, &grads, &PyList_Type, &coefs, &rows,
                        &out, &accumulate, &device, &stream, &size_fn, &fn))
    return nullptr;
  try {
    return grad(ids, grads, coefs, rows, out, accumulate, device,
                reinterpret_cast<void *>(stream),
                reinterpret_cast<SizeFn>(size_fn),
                reinterpret_cast<GradFn>(fn));
  } catch (...) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
}

namespace {

// after an exception of torch's: its Python error, or one of ours
PyObject *failed() {
  if (!PyErr_Occurred())
    PyErr_SetString(PyExc_RuntimeError, "a value could not be looked at");
  return nullptr;
}

bool any_sparse(PyObject *dict) {
  PyObject *key, *value;
  Py_ssize_t pos = 0;
  // (nearly all values are of one type, which is asked about once)
  PyTypeObject *last = nullptr;
  bool tensor = false;
  while (PyDict_Next(dict, &pos, &key, &value)) {
    if (Py_TYPE(value) != last) {
      last = Py_TYPE(value);
      tensor = THPVariable_Check(value);
    }
    if (tensor && THPVariable_Unpack(value).unsafeGetTensorImpl()->is_sparse())
      return true;
  }
  return false;
}

}  // namespace

PyObject *has_sparse(PyObject *, PyObject *dict) {
  try {
    return PyBool_FromLong(PyDict_Check(dict) && any_sparse(dict));
  } catch (...) {
    return failed();
  }
}

PyObject *sparse_dicts(PyObject *, PyObject *dicts) {
  if (!PyList_Check(dicts)) {
    PyErr_SetString(PyExc_TypeError, "a list of dicts is expected");
    return nullptr;
  }
  PyObject *found = PyList_New(0);
  if (!found) return nullptr;
  try {
    for (Py_ssize_t i = 0; i < PyList_GET_SIZE(dicts); ++i) {
      PyObject *d = PyList_GET_ITEM(dicts, i);
      if (!PyDict_Check(d) || !any_sparse(d)) continue;
      PyObject *at = PyLong_FromSsize_t(i);
      if (!at || PyList_Append(found, at) != 0) {
        Py_XDECREF(at);
        Py_DECREF(found);
        return nullptr;
      }
      Py_DECREF(at);
    }
  } catch (...) {
    Py_DECREF(found);
    return failed();
  }
  return found;
}
