// Short way from Python to the serving operators' C entry points, for requests that
// need nothing but the launch: tensors of the right types, shapes, strides and
// device on a stream that is not being captured.  Each function returns None for
// any other request, and the Python function that called it goes on to say what is
// wrong with it, to copy what the kernels cannot read, or to change the device
// (kernels/paged_cache.py, kernels/spec_verify.py: the same launch through ctypes).
// Tests of a request, allocation of its results and the call take about 5 us less
// here than there.
//
// The library stays loaded by kernels/_lib.py alone: bind() takes its functions'
// addresses.  Scratch and error words are _lib's too, asked for once per stream
// and device; forget() drops what is remembered of them.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContextLight.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <climits>
#include <cmath>
#include <map>
#include <utility>

#include "simsd_b200.h"

namespace {

struct {
  decltype(&simsd_paged_append) append = nullptr;
  decltype(&simsd_paged_attention) attention = nullptr;
  decltype(&simsd_paged_attention_workspace_size) attention_bytes = nullptr;
  decltype(&simsd_speculative_verify) verify = nullptr;
  decltype(&simsd_speculative_verify_workspace_size) verify_bytes = nullptr;
  PyObject* error_ptr = nullptr;        // _lib.error_ptr
  PyObject* stream_scratch = nullptr;   // _lib.stream_scratch
} g;

// Scratch of a stream; holds its owner
struct Scratch {
  char* at = nullptr;
  size_t bytes = 0;
  PyObject* owner = nullptr;
  Scratch() = default;
  Scratch(char* a, size_t n, PyObject* o) : at(a), bytes(n), owner(o) { Py_XINCREF(owner); }
  Scratch(const Scratch& s) : Scratch(s.at, s.bytes, s.owner) {}
  Scratch& operator=(Scratch s) {
    std::swap(at, s.at);
    std::swap(bytes, s.bytes);
    std::swap(owner, s.owner);
    return *this;
  }
  ~Scratch() { Py_XDECREF(owner); }
};
using ScratchMap = std::map<std::pair<int, cudaStream_t>, Scratch>;
ScratchMap& g_scratch = *new ScratchMap;   // never destroyed: the interpreter may be gone by then
int* g_error[64];

void forget_all() {
  ScratchMap old;                          // owners go once nothing refers to them
  old.swap(g_scratch);
  for (auto& e : g_error) e = nullptr;
}

// The error word of device `dev`; nullptr with a Python error set
int* error_word(int dev) {
  if (dev >= 64) return nullptr;
  if (g_error[dev] == nullptr) {
    PyObject* r = PyObject_CallFunction(g.error_ptr, "i", dev);
    if (r == nullptr) return nullptr;
    g_error[dev] = reinterpret_cast<int*>(PyLong_AsVoidPtr(r));
    Py_DECREF(r);
  }
  return g_error[dev];
}

// Scratch of the stream; without an address, and with a Python error set, where there is
// none.  The Python function may let other threads in, and they ask for scratch or forget
// it: nothing of the map is kept over the call.
Scratch scratch(int dev, cudaStream_t stream, size_t bytes) {
  const auto it = g_scratch.find({dev, stream});
  if (it != g_scratch.end() && it->second.bytes >= bytes) return it->second;
  PyObject* r = PyObject_CallFunction(g.stream_scratch, "iKni", dev, (unsigned long long)(uintptr_t)stream,
                                      (Py_ssize_t)bytes, SIMSD_PAGED_COUNTER_BYTES);
  if (r == nullptr) return {};
  const Scratch s(reinterpret_cast<char*>(PyLong_AsVoidPtr(PyTuple_GetItem(r, 0))), PyLong_AsSize_t(PyTuple_GetItem(r, 1)), r);
  Py_DECREF(r);
  g_scratch[{dev, stream}] = s;
  return s;
}

// A request's tensors and numbers, and whether all of them are what is wanted
struct Request {
  PyObject* const* args;
  int dev = -1;
  bool good = true;

  const at::Tensor* tensor(int i, at::ScalarType type, bool optional = false) {
    if (!good) return nullptr;
    if (optional && args[i] == Py_None) return nullptr;
    if (!THPVariable_Check(args[i])) {
      good = false;
      return nullptr;
    }
    const at::Tensor& t = THPVariable_Unpack(args[i]);
    good = t.is_cuda() && t.layout() == at::kStrided && (dev < 0 || t.get_device() == dev) &&
           (type == at::ScalarType::Undefined || t.scalar_type() == type) && !(c10::GradMode::is_enabled() && t.requires_grad());
    if (!good) return nullptr;
    dev = (int)t.get_device();
    return &t;
  }
  long long number(int i) {
    if (!good) return 0;
    const long long v = PyLong_AsLongLong(args[i]);
    if (v == -1 && PyErr_Occurred()) {
      PyErr_Clear();
      good = false;
    }
    return v;
  }
  double real(int i) {
    if (!good) return 0;
    const double v = PyFloat_AsDouble(args[i]);
    if (v == -1.0 && PyErr_Occurred()) {
      PyErr_Clear();
      good = false;
    }
    return v;
  }
  // the device is current (and its stream's handle)
  bool here(cudaStream_t& stream) {
    if (!good || at::cuda::current_device() != dev) return false;
    stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream();
    return true;
  }
};

int half_code(const at::Tensor& t) {
  return t.scalar_type() == at::kBFloat16 ? SIMSD_BF16 : t.scalar_type() == at::kHalf ? SIMSD_F16 : -1;
}
template <typename T = void>
T* ptr(const at::Tensor* t) {
  return t == nullptr ? nullptr : reinterpret_cast<T*>(t->data_ptr());
}
bool is_shape(const at::Tensor& t, std::initializer_list<int64_t> s) { return t.sizes() == at::IntArrayRef(s); }
bool cache_good(const at::Tensor& k, const at::Tensor& v, at::ScalarType type) {
  return k.dim() == 4 && k.scalar_type() == type && v.scalar_type() == type && k.sizes() == v.sizes() &&
         k.strides() == v.strides() && k.stride(3) == 1 && k.size(0) <= INT_MAX && k.size(2) <= INT_MAX;
}

PyObject* none() { Py_RETURN_NONE; }

// (qkv, heads, kv_heads, k_cache, v_cache, slots, positions, cos, sin, q_weight, k_weight, eps) -> q
PyObject* append(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 12 || g.append == nullptr) return none();
  Request r{args};
  const auto any = at::ScalarType::Undefined;
  const at::Tensor* qkv = r.tensor(0, any);
  if (!r.good) return none();
  const auto type = qkv->scalar_type();
  const int code = half_code(*qkv);
  const long long heads = r.number(1), kv_heads = r.number(2);
  const at::Tensor *k = r.tensor(3, type), *v = r.tensor(4, type), *slots = r.tensor(5, at::kLong),
                   *pos = r.tensor(6, at::kLong), *cos = r.tensor(7, at::kFloat), *sin = r.tensor(8, at::kFloat),
                   *qw = r.tensor(9, type, true), *kw = r.tensor(10, type, true);
  const double eps = r.real(11);
  if (!r.good || code < 0 || !cache_good(*k, *v, type) || heads < 1 || heads > 65536 || kv_heads != k->size(1)) return none();
  const int64_t D = k->size(3);
  if (qkv->dim() != 2 || qkv->size(1) != (heads + 2 * kv_heads) * D || qkv->stride(1) != 1) return none();
  const int64_t T = qkv->size(0);
  if (T > INT_MAX || !is_shape(*slots, {T}) || !is_shape(*pos, {T}) || !slots->is_contiguous() || !pos->is_contiguous() ||
      cos->dim() != 2 || cos->sizes() != sin->sizes() || !cos->is_contiguous() || !sin->is_contiguous() ||
      cos->size(1) > D || (qw && (!is_shape(*qw, {D}) || !qw->is_contiguous())) ||
      (kw && (!is_shape(*kw, {D}) || !kw->is_contiguous())))
    return none();
  cudaStream_t stream;
  if (!r.here(stream)) return none();
  int* err = error_word(r.dev);
  if (err == nullptr) return PyErr_Occurred() ? nullptr : none();
  at::Tensor q = at::empty({T, heads, D}, qkv->options());
  const int rc = g.append(ptr(qkv), qkv->stride(0), (int)T, (int)heads, (int)kv_heads, (int)D, 2 * (int)cos->size(1), ptr(qw),
                          ptr(kw), (float)eps, ptr<float>(cos), ptr<float>(sin), cos->size(0), ptr<int64_t>(pos),
                          ptr<int64_t>(slots), q.data_ptr(), ptr(k), ptr(v), (int)k->size(0), (int)k->size(2), k->stride(0),
                          k->stride(1), k->stride(2), code, err, stream);
  return rc == SIMSD_OK ? THPVariable_Wrap(std::move(q)) : none();
  END_HANDLE_TH_ERRORS
}

// (q, k_cache, v_cache, page_table, seq_lens, scale, tail_mask, return_lse) -> o or (o, lse)
PyObject* attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 8 || g.attention == nullptr) return none();
  Request r{args};
  const at::Tensor* q = r.tensor(0, at::ScalarType::Undefined);
  if (!r.good) return none();
  const auto type = q->scalar_type();
  const int code = half_code(*q);
  const at::Tensor *k = r.tensor(1, type), *v = r.tensor(2, type), *table = r.tensor(3, at::kInt),
                   *lens = r.tensor(4, at::kInt), *tail = r.tensor(6, at::kBool, true);
  if (!r.good || code < 0 || (q->dim() != 3 && q->dim() != 4) || !q->is_contiguous() || !cache_good(*k, *v, type))
    return none();
  const int64_t B = q->size(0), L = q->dim() == 4 ? q->size(1) : 1, Hq = q->size(-2), D = q->size(-1), Hk = k->size(1);
  if (B > INT_MAX || L > INT_MAX || Hq > INT_MAX || Hk < 1 || Hq < 1 || Hq % Hk || k->size(3) != D || table->dim() != 2 ||
      table->size(0) != B || table->stride(1) != 1 || table->size(1) > INT_MAX || !is_shape(*lens, {B}) ||
      !lens->is_contiguous())
    return none();
  int64_t ldm_b = 0, ldm_t = 0;
  if (tail) {
    if (!is_shape(*tail, {L, L}) && !is_shape(*tail, {B, L, L})) return none();
    if (tail->stride(-1) != 1) return none();
    ldm_t = tail->stride(-2);
    ldm_b = tail->dim() == 3 ? tail->stride(0) : 0;
  }
  const double scale = args[5] == Py_None ? 1.0 / std::sqrt((double)D) : r.real(5);
  const int with_lse = PyObject_IsTrue(args[7]);
  cudaStream_t stream;
  if (with_lse < 0) return nullptr;
  if (!r.here(stream) || c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None) return none();
  int* err = error_word(r.dev);
  if (err == nullptr) return PyErr_Occurred() ? nullptr : none();
  const Scratch ws = scratch(r.dev, stream, g.attention_bytes((int)L, (int)Hq, (int)Hk, (int)D));
  if (ws.at == nullptr) return nullptr;
  at::Tensor o = at::empty(q->sizes(), q->options()), lse;
  if (with_lse) lse = at::empty(q->sizes().slice(0, q->dim() - 1), q->options().dtype(at::kFloat));
  const int rc = g.attention(ptr(q), ptr(k), ptr(v), (int)k->size(0), (int)k->size(2), k->stride(0), k->stride(1), k->stride(2),
                             ptr<int32_t>(table), table->stride(0), (int)table->size(1), ptr<int32_t>(lens),
                             ptr<uint8_t>(tail), ldm_b, ldm_t, (int)B, (int)L, (int)Hq, (int)Hk, (int)D, (float)scale,
                             o.data_ptr(), with_lse ? lse.data_ptr<float>() : nullptr, code, ws.at, ws.bytes, err, stream);
  if (rc != SIMSD_OK) return none();
  if (!with_lse) return THPVariable_Wrap(std::move(o));
  PyObject* out = PyTuple_New(2);
  if (out == nullptr) return nullptr;
  PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(std::move(o)));
  PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(std::move(lse)));
  return out;
  END_HANDLE_TH_ERRORS
}

// (target_logits, draft_tokens, uniform, noise, draft_logits, temperature, n_draft) -> (tokens, accepted, logprobs)
PyObject* verify(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 7 || g.verify == nullptr) return none();
  Request r{args};
  const at::Tensor* target = r.tensor(0, at::ScalarType::Undefined);
  if (!r.good || target->dim() != 3) return none();
  const auto type = target->scalar_type();
  const int code = type == at::kFloat ? SIMSD_F32 : half_code(*target);
  const int64_t B = target->size(0), R = target->size(1), K = R - 1, V = target->size(2);
  const at::Tensor *x = r.tensor(1, at::kLong), *u = r.tensor(2, at::kFloat), *e = r.tensor(3, at::kFloat),
                   *draft = r.tensor(4, type, true), *temp = r.tensor(5, at::kFloat, true), *count = r.tensor(6, at::kInt, true);
  if (!r.good || code < 0 || R < 1 || V < 1 || B > INT_MAX || R > INT_MAX || V > INT_MAX || target->stride(2) != 1 ||
      !is_shape(*x, {B, K}) || !is_shape(*u, {B, K}) || !is_shape(*e, {B, V}) || x->stride(1) != 1 || u->stride(1) != 1 ||
      e->stride(1) != 1 || (draft && (!is_shape(*draft, {B, K, V}) || draft->stride(2) != 1)) ||
      (temp && (!is_shape(*temp, {B}) || !temp->is_contiguous())) || (count && (!is_shape(*count, {B}) || !count->is_contiguous())))
    return none();
  cudaStream_t stream;
  if (!r.here(stream) || c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None) return none();
  int* err = error_word(r.dev);
  if (err == nullptr) return PyErr_Occurred() ? nullptr : none();
  const size_t skip = SIMSD_PAGED_COUNTER_BYTES;       // the attention's counters
  const Scratch ws = scratch(r.dev, stream, g.verify_bytes((int)B, (int)K, (int)V) + skip);
  if (ws.at == nullptr) return nullptr;
  if (K == 0) draft = nullptr;
  at::Tensor tokens = at::empty({B, R}, target->options().dtype(at::kLong)),
             accepted = at::empty({B}, target->options().dtype(at::kLong)),
             logprobs = at::empty({B, R}, target->options().dtype(at::kFloat));
  const int rc = g.verify(ptr(target), target->stride(0), target->stride(1), ptr(draft), draft ? draft->stride(0) : 0,
                          draft ? draft->stride(1) : 0, ptr<int64_t>(x), x->stride(0), ptr<float>(u), u->stride(0),
                          ptr<float>(e), e->stride(0), ptr<float>(temp), ptr<int32_t>(count), (int)B, (int)K, (int)V, code,
                          tokens.data_ptr<int64_t>(), accepted.data_ptr<int64_t>(), logprobs.data_ptr<float>(), ws.at + skip,
                          ws.bytes - skip, err, stream);
  if (rc != SIMSD_OK) return none();
  PyObject* out = PyTuple_New(3);
  if (out == nullptr) return nullptr;
  PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(std::move(tokens)));
  PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(std::move(accepted)));
  PyTuple_SET_ITEM(out, 2, THPVariable_Wrap(std::move(logprobs)));
  return out;
  END_HANDLE_TH_ERRORS
}

// bind({name: address of the library's function}, error_ptr, stream_scratch)
PyObject* bind(PyObject*, PyObject* args) {
  PyObject *fns, *error_ptr, *stream_scratch;
  if (!PyArg_ParseTuple(args, "O!OO", &PyDict_Type, &fns, &error_ptr, &stream_scratch)) return nullptr;
  auto address = [&](const char* name) -> void* {
    PyObject* a = PyDict_GetItemString(fns, name);
    return a ? PyLong_AsVoidPtr(a) : nullptr;
  };
  g.append = reinterpret_cast<decltype(g.append)>(address("simsd_paged_append"));
  g.attention = reinterpret_cast<decltype(g.attention)>(address("simsd_paged_attention"));
  g.attention_bytes = reinterpret_cast<decltype(g.attention_bytes)>(address("simsd_paged_attention_workspace_size"));
  g.verify = reinterpret_cast<decltype(g.verify)>(address("simsd_speculative_verify"));
  g.verify_bytes = reinterpret_cast<decltype(g.verify_bytes)>(address("simsd_speculative_verify_workspace_size"));
  Py_XINCREF(error_ptr);
  Py_XINCREF(stream_scratch);
  Py_XDECREF(g.error_ptr);
  Py_XDECREF(g.stream_scratch);
  g.error_ptr = error_ptr;
  g.stream_scratch = stream_scratch;
  forget_all();
  Py_RETURN_NONE;
}

PyObject* forget(PyObject*, PyObject*) {
  forget_all();
  Py_RETURN_NONE;
}

// scratch(device, stream, bytes) -> (address, bytes) that the operators would get
PyObject* scratch_of(PyObject*, PyObject* args) {
  int dev;
  unsigned long long stream;
  Py_ssize_t bytes;
  if (!PyArg_ParseTuple(args, "iKn", &dev, &stream, &bytes)) return nullptr;
  const Scratch s = scratch(dev, reinterpret_cast<cudaStream_t>((uintptr_t)stream), (size_t)bytes);
  if (s.at == nullptr) return nullptr;
  return Py_BuildValue("Kn", (unsigned long long)reinterpret_cast<uintptr_t>(s.at), (Py_ssize_t)s.bytes);
}

PyMethodDef methods[] = {
    {"bind", bind, METH_VARARGS, nullptr},
    {"forget", forget, METH_NOARGS, nullptr},
    {"scratch", scratch_of, METH_VARARGS, nullptr},
    {"paged_append", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(append)), METH_FASTCALL, nullptr},
    {"paged_attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(attention)), METH_FASTCALL, nullptr},
    {"speculative_verify", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(verify)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

#ifndef SIMSD_BUILT_FOR
#define SIMSD_BUILT_FOR "an unknown version"
#endif
// built_for: the torch and Python whose headers this was compiled against (build.py)
PyMODINIT_FUNC PyInit__binding(void) {
  PyObject* m = PyModule_Create(&module);
  if (m != nullptr && PyModule_AddStringConstant(m, "built_for", SIMSD_BUILT_FOR) != 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
