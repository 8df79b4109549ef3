// The operators of lcr_b200/paged.py on torch tensors: each function checks its
// tensors, takes torch's current stream and calls the C ABI -- in one step from
// Python, where the checks alone, at half a microsecond a tensor, took longer
// than some of the operators do on the GPU. They return the lcr_status; a
// tensor that does not fit raises ValueError with its name.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <dlfcn.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <string>

#include "lcr_b200.h"

namespace {

decltype(&lcr_plan_step) plan_step_c = nullptr;
decltype(&lcr_qk_norm_rope_kv) qk_norm_rope_kv_c = nullptr;
decltype(&lcr_chunk_attention) chunk_attention_c = nullptr;
decltype(&lcr_token_probs) token_probs_c = nullptr;
decltype(&lcr_verify_drafts_bounded) verify_drafts_c = nullptr;

// A Python error is set.
struct Refused {};

// The tensors of one call.
class Call {
 public:
  Call(PyObject* const* args, Py_ssize_t nargs, Py_ssize_t wanted, bool bound) : args_(args) {
    if (nargs != wanted) raise(PyExc_TypeError, "expected " + std::to_string(wanted) + " arguments");
    if (!bound) raise(PyExc_RuntimeError, "_tensors.open(path of liblcr_b200.so) comes first");
  }

  [[noreturn]] static void raise(PyObject* type, const std::string& text) {
    PyErr_SetString(type, text.c_str());
    throw Refused();
  }

  static std::string shape(const at::Tensor& t) {
    std::string s = std::string(c10::toString(t.scalar_type())) + " [";
    for (int64_t d = 0; d < t.dim(); ++d) s += (d ? ", " : "") + std::to_string(t.size(d));
    s += "] with strides [";
    for (int64_t d = 0; d < t.dim(); ++d) s += (d ? ", " : "") + std::to_string(t.stride(d));
    return s + "] on " + t.device().str();
  }

  [[noreturn]] void refuse(int i, const char* name, const std::string& wanted) {
    raise(PyExc_ValueError, std::string(name) + ": " + wanted + " on the current device, got " +
                                (THPVariable_Check(args_[i]) ? shape(THPVariable_Unpack(args_[i])) : Py_TYPE(args_[i])->tp_name));
  }

  // A CUDA tensor of the current device.
  const at::Tensor& tensor(int i, const char* name, at::ScalarType type, const char* wanted) {
    if (!THPVariable_Check(args_[i])) refuse(i, name, wanted);
    const at::Tensor& t = THPVariable_Unpack(args_[i]);
    if (!t.is_cuda() || t.scalar_type() != type) refuse(i, name, wanted);
    if (device_ < 0) device_ = c10::cuda::current_device();
    if (t.get_device() != device_) refuse(i, name, wanted);
    return t;
  }
  // Contiguous, at least n elements.
  template <class T>
  T* flat(int i, const char* name, at::ScalarType type, int64_t n) {
    const at::Tensor& t = tensor(i, name, type, "a contiguous tensor of its type");
    if (!t.is_contiguous() || t.numel() < n) {
      refuse(i, name, std::string("a contiguous ") + c10::toString(type) + " tensor of " + std::to_string(n) + " elements");
    }
    return static_cast<T*>(t.data_ptr());
  }
  bool absent(int i) const { return args_[i] == Py_None; }
  template <class T>
  T* maybe(int i, const char* name, at::ScalarType type, int64_t n) {
    return absent(i) ? nullptr : flat<T>(i, name, type, n);
  }
  // Contiguous, at least n elements, and `steps` (the elements from one index to
  // the next of the layout that is read) has those of its own dimensions: a
  // padded or a transposed one would be misread.
  template <class T>
  T* dense(int i, const char* name, at::ScalarType type, int64_t n, at::IntArrayRef steps, const char* wanted) {
    T* p = flat<T>(i, name, type, n);
    const at::Tensor& t = THPVariable_Unpack(args_[i]);
    int64_t step = 1;
    for (int64_t d = t.dim() - 1; d > 0; --d) {
      step *= t.size(d);
      if (step != 1 && std::find(steps.begin(), steps.end(), step) == steps.end()) refuse(i, name, wanted);
    }
    return p;
  }
  // The gain of a norm, for the elements of one head (of every head the same).
  void* gain(int i, const char* name, int64_t d) {
    void* p = maybe<void>(i, name, at::kBFloat16, d);
    if (p != nullptr && numel(i) != d) refuse(i, name, std::to_string(d) + " elements, for every head the same");
    return p;
  }
  int64_t numel(int i) { return THPVariable_Unpack(args_[i]).numel(); }
  int32_t* ints(int i, const char* name, int64_t n) { return flat<int32_t>(i, name, at::kInt, n); }
  // Rows of dense elements.
  const at::Tensor& rows(int i, const char* name, at::ScalarType type) {
    const at::Tensor& t = tensor(i, name, type, "rows of its type");
    if (t.dim() != 2 || (t.size(1) > 1 && t.stride(1) != 1)) {
      refuse(i, name, std::string("dense ") + c10::toString(type) + " rows");
    }
    return t;
  }
  const at::Tensor& table(int i, const char* name) {
    const at::Tensor& t = tensor(i, name, at::kInt, "an int32 matrix");
    if (t.dim() != 2 || !t.is_contiguous()) refuse(i, name, "a contiguous int32 matrix");
    return t;
  }
  // A pair of pools [pages, kv_heads, page_size, head_dim].
  lcr_kv_view view(int ik, int iv, int* pages) {
    const char* wanted = "a bf16 pool [pages, kv_heads, page_size, head_dim] with dense slots";
    const at::Tensor &k = tensor(ik, "keys", at::kBFloat16, wanted), &v = tensor(iv, "values", at::kBFloat16, wanted);
    if (k.dim() != 4 || k.stride(3) != 1 || k.stride(2) != k.size(3)) refuse(ik, "keys", wanted);
    if (v.sizes() != k.sizes() || v.strides() != k.strides()) refuse(iv, "values", "a pool like keys");
    if (k.stride(0) > INT32_MAX || k.stride(1) > INT32_MAX || k.size(0) > INT32_MAX) {
      refuse(ik, "keys", "a pool with strides of 31 bits");
    }
    *pages = static_cast<int>(k.size(0));
    return {k.data_ptr(),
            v.data_ptr(),
            nullptr,
            static_cast<int>(k.size(2)),
            static_cast<int>(k.stride(0)),
            static_cast<int>(k.stride(1)),
            static_cast<int>(k.size(1)),
            static_cast<int>(k.size(3))};
  }
  double number(int i) {
    const double x = PyFloat_AsDouble(args_[i]);
    if (x == -1.0 && PyErr_Occurred()) throw Refused();
    return x;
  }
  int integer(int i) {
    const long x = PyLong_AsLong(args_[i]);
    if (x == -1 && PyErr_Occurred()) throw Refused();
    if (x < INT32_MIN || x > INT32_MAX) raise(PyExc_ValueError, "a number past 32 bits");
    return static_cast<int>(x);
  }
  static void fits(bool ok, const char* text) {
    if (!ok) raise(PyExc_ValueError, text);
  }
  static int small(int64_t n) {
    if (n > INT32_MAX) raise(PyExc_ValueError, "a size past 31 bits");
    return static_cast<int>(n);
  }
  lcr_stream_t stream() {
    if (device_ < 0) device_ = c10::cuda::current_device();
    return reinterpret_cast<lcr_stream_t>(c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device_)).stream());
  }

 private:
  PyObject* const* args_;
  int device_ = -1;
};

// (block_tables, held, free_pages, free_count, cached, new_tokens, finished,
//  page_size, held_out, free_count_out, row_starts, kv_lengths, positions,
//  slots, row_sequence)
int plan_step(PyObject* const* args, Py_ssize_t nargs) {
  Call c(args, nargs, 15, plan_step_c != nullptr);
  const at::Tensor& t = c.table(0, "block_tables");
  const int n = c.small(t.size(0)), width = c.small(t.size(1));
  const at::Tensor& stack = c.tensor(2, "free_pages", at::kInt, "an int32 tensor");
  const at::Tensor& pos = c.tensor(12, "positions", at::kInt, "an int32 tensor");
  const int rows = c.small(pos.numel());
  return plan_step_c(static_cast<int32_t*>(t.data_ptr()), width, c.ints(1, "held", n), c.ints(8, "held_out", n),
                     c.ints(2, "free_pages", 1), c.ints(3, "free_count", 1), c.ints(9, "free_count_out", 1),
                     c.small(stack.numel()), c.ints(4, "cached", n), c.ints(5, "new_tokens", n),
                     c.maybe<int32_t>(6, "finished", at::kInt, n), n, c.integer(7), rows, c.ints(10, "row_starts", n + 1),
                     c.ints(11, "kv_lengths", n), c.ints(12, "positions", rows), c.ints(13, "slots", rows),
                     c.ints(14, "row_sequence", rows), c.stream());
}

// (q_out, keys, values, qkv, positions, slots, inv_freq, q_gain, k_gain, eps)
int qk_norm_rope_kv(PyObject* const* args, Py_ssize_t nargs) {
  Call c(args, nargs, 10, qk_norm_rope_kv_c != nullptr);
  int pages = 0;
  const lcr_kv_view view = c.view(1, 2, &pages);
  const at::Tensor &q = c.rows(0, "q_out", at::kBFloat16), &x = c.rows(3, "qkv", at::kBFloat16);
  const int d = view.head_dim, rows = c.small(x.size(0));
  const int64_t heads = d > 0 ? x.size(1) / d - 2 * static_cast<int64_t>(view.num_kv_heads) : 0;
  Call::fits(heads > 0 && x.size(1) == (heads + 2 * view.num_kv_heads) * d && q.size(0) == rows && q.size(1) == heads * d,
             "qkv and q_out do not fit the pools' heads");
  return qk_norm_rope_kv_c(q.data_ptr(), q.stride(0), &view, pages, x.data_ptr(), x.stride(0), rows, c.small(heads),
                           c.gain(7, "q_gain", d), c.gain(8, "k_gain", d),
                           static_cast<float>(c.number(9)), c.flat<float>(6, "inv_freq", at::kFloat, d / 2),
                           c.ints(4, "positions", rows), c.ints(5, "slots", rows), c.stream());
}

// (out, q, keys, values, block_tables, row_starts, kv_lengths, scale, workspace)
int chunk_attention(PyObject* const* args, Py_ssize_t nargs) {
  Call c(args, nargs, 9, chunk_attention_c != nullptr);
  int pages = 0;
  lcr_kv_view view = c.view(2, 3, &pages);
  const at::Tensor &o = c.rows(0, "out", at::kBFloat16), &q = c.rows(1, "q", at::kBFloat16);
  const at::Tensor& t = c.table(4, "block_tables");
  const at::Tensor& kv = c.tensor(6, "kv_lengths", at::kInt, "an int32 tensor");
  const at::Tensor& w = c.tensor(8, "workspace", at::kByte, "bytes");
  const int n = c.small(kv.numel()), rows = c.small(q.size(0)), d = view.head_dim;
  const int heads = d > 0 ? c.small(q.size(1) / d) : 0;
  Call::fits(heads > 0 && q.size(1) == static_cast<int64_t>(heads) * d && o.sizes() == q.sizes() && t.size(0) >= n,
             "q, out, block_tables and kv_lengths do not fit one another and the pools' heads");
  view.page_table = static_cast<const int32_t*>(t.data_ptr());
  return chunk_attention_c(o.data_ptr(), o.stride(0), q.data_ptr(), q.stride(0), &view, c.small(t.size(1)), pages,
                           c.ints(5, "row_starts", n + 1), c.ints(6, "kv_lengths", n), n, rows, heads,
                           static_cast<float>(c.number(7)), c.flat<void>(8, "workspace", at::kByte, 0),
                           static_cast<size_t>(w.numel()), c.stream());
}

// (probs, logits, temperature, row_sequence)
int token_probs(PyObject* const* args, Py_ssize_t nargs) {
  Call c(args, nargs, 4, token_probs_c != nullptr);
  const at::Tensor &p = c.rows(0, "probs", at::kFloat), &x = c.rows(1, "logits", at::kFloat);
  Call::fits(p.sizes() == x.sizes(), "probs and logits have the same shape");
  const int rows = c.small(x.size(0));
  const int32_t* seq = c.maybe<int32_t>(3, "row_sequence", at::kInt, rows);
  const float* t = c.maybe<float>(2, "temperature", at::kFloat, seq != nullptr ? 1 : rows);
  const int temperatures = t != nullptr ? c.small(c.numel(2)) : 0;
  return token_probs_c(static_cast<float*>(p.data_ptr()), p.stride(0), static_cast<const float*>(x.data_ptr()), x.stride(0),
                       rows, c.small(x.size(1)), t, temperatures, seq, c.stream());
}

// (tokens, accepted, target_probs, target_starts, drafts, draft_counts,
//  draft_probs, uniforms)
int verify_drafts(PyObject* const* args, Py_ssize_t nargs) {
  Call c(args, nargs, 8, verify_drafts_c != nullptr);
  const at::Tensor &t = c.table(0, "tokens"), &d = c.table(4, "drafts");
  const at::Tensor& p = c.rows(2, "target_probs", at::kFloat);
  const int n = c.small(d.size(0)), k = c.small(d.size(1)), vocab = c.small(p.size(1));
  Call::fits(t.size(0) == n && t.size(1) == k + 1, "tokens: [requests, max_drafts + 1]");
  const int64_t most = k, ids = vocab;
  float* q = c.absent(6) ? nullptr
                         : c.dense<float>(6, "draft_probs", at::kFloat, n * most * ids, {ids, most * ids},
                                          "contiguous Float [requests, max_drafts, vocab]");
  float* u = c.dense<float>(7, "uniforms", at::kFloat, n * (most + 1), {most + 1}, "contiguous Float [requests, max_drafts + 1]");
  return verify_drafts_c(static_cast<int32_t*>(t.data_ptr()), c.ints(1, "accepted", n), static_cast<const float*>(p.data_ptr()),
                         p.stride(0), c.small(p.size(0)), c.ints(3, "target_starts", n + 1), c.ints(4, "drafts", 0),
                         c.ints(5, "draft_counts", n), q, u, n, k, vocab, c.stream());
}

template <int (*F)(PyObject* const*, Py_ssize_t)>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  try {
    return PyLong_FromLong(F(args, nargs));
  } catch (const Refused&) {
    return nullptr;
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

PyObject* open_library(PyObject*, PyObject* path) {
  const char* p = PyUnicode_AsUTF8(path);
  if (p == nullptr) return nullptr;
  void* lib = dlopen(p, RTLD_NOW);
  if (lib == nullptr) {
    PyErr_SetString(PyExc_RuntimeError, dlerror());
    return nullptr;
  }
  auto bind = [&](auto& f, const char* name) {
    f = reinterpret_cast<std::remove_reference_t<decltype(f)>>(dlsym(lib, name));
    return f != nullptr;
  };
  if (!(bind(plan_step_c, "lcr_plan_step") && bind(qk_norm_rope_kv_c, "lcr_qk_norm_rope_kv") &&
        bind(chunk_attention_c, "lcr_chunk_attention") && bind(token_probs_c, "lcr_token_probs") &&
        bind(verify_drafts_c, "lcr_verify_drafts_bounded"))) {
    PyErr_SetString(PyExc_RuntimeError, "the library lacks an operator");
    return nullptr;
  }
  Py_RETURN_NONE;
}

// The current stream's handle (cudaStream_t) and device.
PyObject* current(PyObject*, PyObject*) {
  try {
    const int device = c10::cuda::current_device();
    const auto s = c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream();
    return Py_BuildValue("(Li)", static_cast<long long>(reinterpret_cast<intptr_t>(s)), device);
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

#define LCR_FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(entry<f>)), METH_FASTCALL
PyMethodDef methods[] = {{"open", open_library, METH_O, "binds the operators of the library at a path"},
                         {"current", current, METH_NOARGS, "(stream handle, device) of torch"},
                         {"plan_step", LCR_FAST(plan_step), "lcr_plan_step"},
                         {"qk_norm_rope_kv", LCR_FAST(qk_norm_rope_kv), "lcr_qk_norm_rope_kv"},
                         {"chunk_attention", LCR_FAST(chunk_attention), "lcr_chunk_attention"},
                         {"token_probs", LCR_FAST(token_probs), "lcr_token_probs"},
                         {"verify_drafts", LCR_FAST(verify_drafts), "lcr_verify_drafts"},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensors", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensors(void) { return PyModule_Create(&module); }
