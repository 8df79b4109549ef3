// Checked pointers of torch tensors for paged.py, in one call: a check in
// Python costs half a microsecond a tensor, more than some of the operators
// take on the GPU.
//
//   pointers(names, kinds, tensor, count, tensor, count, ...) -> tuple of ints
//
// Each tensor is on torch's current CUDA device and, by its letter in `kinds`,
//   i  int32, f  fp32, h  bf16: contiguous, at least `count` elements -> address
//   F  fp32, H  bf16: 2-D rows of `count` dense elements -> address, row stride
//   K  bf16: 4-D pool, dense in its last two axes -> address, strides 0 and 1
// (None gives 0 for i, f, h.) The tuple ends with the current stream. A tensor
// that does not fit raises ValueError with its name.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <string>

namespace {

PyObject* refuse(PyObject* names, Py_ssize_t i, const char* wanted, PyObject* got) {
  PyObject* name = PyTuple_GetItem(names, i);
  if (name == nullptr) return nullptr;
  std::string what = Py_TYPE(got)->tp_name;
  if (THPVariable_Check(got)) {
    const at::Tensor& t = THPVariable_Unpack(got);
    what = std::string(c10::toString(t.scalar_type())) + " [";
    for (int64_t d = 0; d < t.dim(); ++d) what += (d ? ", " : "") + std::to_string(t.size(d));
    what += "] with strides [";
    for (int64_t d = 0; d < t.dim(); ++d) what += (d ? ", " : "") + std::to_string(t.stride(d));
    what += "] on " + t.device().str();
  }
  PyErr_Format(PyExc_ValueError, "%U: %s on the current device, got %s", name, wanted, what.c_str());
  return nullptr;
}

PyObject* pointers_of(PyObject* const* args, Py_ssize_t nargs) {
  if (nargs < 2 || !PyTuple_Check(args[0]) || !PyUnicode_Check(args[1])) {
    PyErr_SetString(PyExc_TypeError, "pointers(names, kinds, tensor, count, ...)");
    return nullptr;
  }
  Py_ssize_t n = 0;
  const char* kinds = PyUnicode_AsUTF8AndSize(args[1], &n);
  if (kinds == nullptr) return nullptr;
  if (nargs != 2 + 2 * n) {
    PyErr_SetString(PyExc_TypeError, "pointers: a tensor and a count for each kind");
    return nullptr;
  }
  long long out[64];
  int k = 0;
  int device = -1;  // asked for with the first CUDA tensor
  for (Py_ssize_t i = 0; i < n; ++i) {
    if (k + 4 >= 64) {
      PyErr_SetString(PyExc_TypeError, "pointers: too many tensors");
      return nullptr;
    }
    PyObject* obj = args[2 + 2 * i];
    const long long count = PyLong_AsLongLong(args[3 + 2 * i]);
    if (count == -1 && PyErr_Occurred()) return nullptr;
    const char kind = kinds[i];
    if (obj == Py_None && (kind == 'i' || kind == 'f' || kind == 'h')) {
      out[k++] = 0;
      continue;
    }
    const at::ScalarType type = kind == 'i'                  ? at::kInt
                                : kind == 'f' || kind == 'F' ? at::kFloat
                                                             : at::kBFloat16;
    const char* wanted = kind == 'i'   ? "a contiguous int32 tensor with an element for each"
                         : kind == 'f' ? "a contiguous fp32 tensor with an element for each"
                         : kind == 'h' ? "a contiguous bf16 tensor with an element for each"
                         : kind == 'F' ? "dense fp32 rows"
                         : kind == 'H' ? "dense bf16 rows"
                                       : "a bf16 pool [pages, kv_heads, page_size, head_dim] with dense slots";
    if (!THPVariable_Check(obj)) return refuse(args[0], i, wanted, obj);
    const at::Tensor& t = THPVariable_Unpack(obj);
    if (t.is_cuda() && device < 0) device = c10::cuda::current_device();
    if (t.scalar_type() != type || !t.is_cuda() || t.get_device() != device) return refuse(args[0], i, wanted, obj);
    if (kind == 'i' || kind == 'f' || kind == 'h') {
      if (!t.is_contiguous() || t.numel() < count) return refuse(args[0], i, wanted, obj);
    } else if (kind == 'F' || kind == 'H') {
      if (t.dim() != 2 || t.size(1) != count || (count > 1 && t.stride(1) != 1)) return refuse(args[0], i, wanted, obj);
    } else if (t.dim() != 4 || t.stride(3) != 1 || t.stride(2) != t.size(3)) {
      return refuse(args[0], i, wanted, obj);
    }
    out[k++] = reinterpret_cast<long long>(t.data_ptr());
    if (kind == 'F' || kind == 'H') {
      out[k++] = t.stride(0);
    } else if (kind == 'K') {
      out[k++] = t.stride(0);
      out[k++] = t.stride(1);
    }
  }
  if (device < 0) device = c10::cuda::current_device();
  out[k++] = reinterpret_cast<long long>(c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream());
  PyObject* result = PyTuple_New(k);
  if (result == nullptr) return nullptr;
  for (int i = 0; i < k; ++i) {
    PyObject* v = PyLong_FromLongLong(out[i]);
    if (v == nullptr) {
      Py_DECREF(result);
      return nullptr;
    }
    PyTuple_SET_ITEM(result, i, v);
  }
  return result;
}

PyObject* pointers(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  try {
    return pointers_of(args, nargs);
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

PyMethodDef methods[] = {
    {"pointers", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(pointers)), METH_FASTCALL,
     "pointers(names, kinds, tensor, count, ...) -> addresses (and strides), and the current stream"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensors", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensors(void) { return PyModule_Create(&module); }
