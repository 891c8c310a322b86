// embed_parts: the parts table of fsagg_embed_grad (include/fsagg.h) from
// lists of token and gradient tensors, in one C++ walk.
//
// A round's row-sparse uploads are one (tokens, rows) pair per client; the
// Python checks of a pair (device, types, shapes, strides, overlap) cost
// about 3 us, 100 clients' more than the kernels they launch.  Here they are
// a few TensorImpl reads each.
//
// embed_parts(ids, grads, coefs, out_lo, out_hi) -> (bytes table, int tokens,
//   int dim, int dtype_code) or None
//     ids, grads  equally long, non-empty lists of tensors
//     coefs       list of float, one per part
//     out_lo/hi   addresses that no part may touch (0, 0: none)
// None is not an error: some pair is not of the plain form (contiguous int64
// or int32 tokens; strided float32, float16 or bfloat16 rows of one type and
// width on the tokens' GPU), and the caller's own checks say why.
//
// has_sparse(dict) -> bool: whether a value is a sparse COO tensor (asked of
// every upload, most of which have none: 161 keys 2 us, 19 us in Python).
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
bool address(const c10::TensorImpl *t, uintptr_t &p) {
  if (t->layout() != c10::kStrided || !t->has_storage()) return false;
  const void *d = t->storage().data();
  p = d ? reinterpret_cast<uintptr_t>(d) +
              uintptr_t(t->storage_offset()) * t->dtype().itemsize()
        : 0;
  return p != 0 || t->numel() == 0;
}

PyObject *walk(PyObject *ids, PyObject *grads, PyObject *coefs, uintptr_t lo,
               uintptr_t hi) {
  const Py_ssize_t n = PyList_GET_SIZE(ids);
  if (n < 1 || PyList_GET_SIZE(grads) != n || PyList_GET_SIZE(coefs) != n)
    Py_RETURN_NONE;
  std::string buf(size_t(n) * sizeof(EmbedPart), '\0');
  auto *part = reinterpret_cast<EmbedPart *>(&buf[0]);
  int64_t tokens = 0, dim = -1;
  caffe2::TypeMeta dtype;
  c10::Device dev(c10::kCPU);
  int code = -1;
  for (Py_ssize_t i = 0; i < n; ++i) {
    const c10::TensorImpl *t = tensor_of(PyList_GET_ITEM(ids, i));
    const c10::TensorImpl *g = tensor_of(PyList_GET_ITEM(grads, i));
    if (!t || !g) Py_RETURN_NONE;
    uintptr_t pt, pg;
    if (!address(t, pt) || !address(g, pg)) Py_RETURN_NONE;
    if (i == 0) {
      dev = g->device();
      dtype = g->dtype();
      if (dtype == caffe2::TypeMeta::Make<float>()) code = 0;
      else if (dtype == caffe2::TypeMeta::Make<at::Half>()) code = 1;
      else if (dtype == caffe2::TypeMeta::Make<at::BFloat16>()) code = 2;
      else Py_RETURN_NONE;
      if (!dev.is_cuda() || g->dim() < 1) Py_RETURN_NONE;
      dim = g->sizes().back();
    }
    const bool i64 = t->dtype() == caffe2::TypeMeta::Make<int64_t>();
    if (g->device() != dev || t->device() != dev || g->dtype() != dtype ||
        (!i64 && t->dtype() != caffe2::TypeMeta::Make<int32_t>()) ||
        !t->is_contiguous() || g->dim() != t->dim() + 1 ||
        g->sizes().back() != dim)
      Py_RETURN_NONE;
    for (int64_t d = 0; d < t->dim(); ++d)
      if (g->sizes()[d] != t->sizes()[d]) Py_RETURN_NONE;
    const int64_t rows = t->numel();
    int64_t stride = dim;
    if (g->dim() == 2 && (dim <= 1 || g->strides()[1] == 1))
      stride = g->strides()[0];
    else if (!g->is_contiguous())
      Py_RETURN_NONE;
    if (stride < 0 || rows > (int64_t(1) << 28)) Py_RETURN_NONE;
    const uintptr_t size = dtype.itemsize();
    const uintptr_t gend =
        rows > 0 ? pg + (uintptr_t(rows - 1) * uintptr_t(stride) +
                         uintptr_t(dim)) * size
                 : pg;
    const uintptr_t tend = pt + uintptr_t(rows) * t->dtype().itemsize();
    if ((pg < hi && lo < gend) || (pt < hi && lo < tend)) Py_RETURN_NONE;
    const double c = PyFloat_AsDouble(PyList_GET_ITEM(coefs, i));
    if (c == -1.0 && PyErr_Occurred()) return nullptr;
    part[i] = {reinterpret_cast<const void *>(pt),
               reinterpret_cast<const void *>(pg), rows, stride, float(c),
               i64 ? 1 : 0};
    tokens += rows;
  }
  return Py_BuildValue("(y#LLi)", buf.data(), Py_ssize_t(buf.size()),
                       (long long)tokens, (long long)dim, code);
}

}  // namespace

PyObject *embed_parts(PyObject *, PyObject *args) {
  PyObject *ids, *grads, *coefs;
  unsigned long long lo, hi;
  if (!PyArg_ParseTuple(args, "O!O!O!KK", &PyList_Type, &ids, &PyList_Type,
                        &grads, &PyList_Type, &coefs, &lo, &hi))
    return nullptr;
  try {
    return walk(ids, grads, coefs, uintptr_t(lo), uintptr_t(hi));
  } catch (...) {
    Py_RETURN_NONE;
  }
}

PyObject *has_sparse(PyObject *, PyObject *dict) {
  if (!PyDict_Check(dict)) Py_RETURN_FALSE;
  PyObject *key, *value;
  Py_ssize_t pos = 0;
  while (PyDict_Next(dict, &pos, &key, &value)) {
    const c10::TensorImpl *t = tensor_of(value);
    if (t && t->is_sparse()) Py_RETURN_TRUE;
  }
  Py_RETURN_FALSE;
}
