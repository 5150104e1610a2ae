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
  decltype(&simsd_paged_attention_window) attention = nullptr;
  decltype(&simsd_paged_attention_workspace_size) attention_bytes = nullptr;
  decltype(&simsd_speculative_verify) verify = nullptr;
  decltype(&simsd_speculative_verify_workspace_size) verify_bytes = nullptr;
  decltype(&simsd_paged_append8) append8 = nullptr;
  decltype(&simsd_paged_attention8) attention8 = nullptr;
  decltype(&simsd_paged_attention8_workspace_size) attention8_bytes = nullptr;
  decltype(&simsd_paged_reserve) reserve = nullptr;
  decltype(&simsd_paged_release) release = nullptr;
  decltype(&simsd_adjust_logits) adjust = nullptr;
  decltype(&simsd_count_tokens) count = nullptr;
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

// What the two forms of attention have in common: queries, tables, mask, window
struct Attention {
  const at::Tensor *q, *k, *v, *table, *lens, *tail;
  int64_t B, L, Hq, D, Hk, ldm_b = 0, ldm_t = 0;
  double scale;
  int code, with_lse, window = 0, sinks;

  // args[at ...]: page_table, seq_lens, scale, tail_mask, return_lse, window, sinks
  bool read(Request& r, at::ScalarType cache, int at) {
    if (!r.good) return false;
    code = half_code(*q);
    const auto type = cache == at::ScalarType::Undefined ? q->scalar_type() : cache;
    k = r.tensor(1, type), v = r.tensor(2, type);
    table = r.tensor(at, at::kInt), lens = r.tensor(at + 1, at::kInt), tail = r.tensor(at + 3, at::kBool, true);
    if (!r.good || code < 0 || (q->dim() != 3 && q->dim() != 4) || !q->is_contiguous() || !cache_good(*k, *v, type)) return false;
    B = q->size(0), L = q->dim() == 4 ? q->size(1) : 1, Hq = q->size(-2), D = q->size(-1), Hk = k->size(1);
    if (B > INT_MAX || L > INT_MAX || Hq > INT_MAX || Hk < 1 || Hq < 1 || Hq % Hk || k->size(3) != D || table->dim() != 2 ||
        table->size(0) != B || table->stride(1) != 1 || table->size(1) > INT_MAX || !is_shape(*lens, {B}) ||
        !lens->is_contiguous())
      return false;
    if (tail) {
      if (!is_shape(*tail, {L, L}) && !is_shape(*tail, {B, L, L})) return false;
      if (tail->stride(-1) != 1) return false;
      ldm_t = tail->stride(-2);
      ldm_b = tail->dim() == 3 ? tail->stride(0) : 0;
    }
    scale = r.args[at + 2] == Py_None ? 1.0 / std::sqrt((double)D) : r.real(at + 2);
    with_lse = r.args[at + 4] == Py_True ? 1 : r.args[at + 4] == Py_False ? 0 : -1;
    if (r.args[at + 5] != Py_None) {
      const long long w = r.number(at + 5);
      if (w < 1 || w > INT_MAX) return false;
      window = (int)w;
    }
    const long long s = r.number(at + 6);
    if (!r.good || s < 0 || s > INT_MAX || with_lse < 0) return false;
    sinks = (int)s;
    return true;
  }
};

// Runs `call(scratch, error word, stream, o, lse)` of a request that is good; o or (o, lse)
template <typename Size, typename Call>
PyObject* attend(Request& r, const Attention& a, Size bytes, Call call) {
  cudaStream_t stream;
  if (!r.here(stream) || c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None) return none();
  int* err = error_word(r.dev);
  if (err == nullptr) return PyErr_Occurred() ? nullptr : none();
  const Scratch ws = scratch(r.dev, stream, bytes((int)a.L, (int)a.Hq, (int)a.Hk, (int)a.D));
  if (ws.at == nullptr) return nullptr;
  at::Tensor o = at::empty(a.q->sizes(), a.q->options()), lse;
  if (a.with_lse) lse = at::empty(a.q->sizes().slice(0, a.q->dim() - 1), a.q->options().dtype(at::kFloat));
  if (call(ws, err, stream, o.data_ptr(), a.with_lse ? lse.data_ptr<float>() : nullptr) != SIMSD_OK) return none();
  if (!a.with_lse) return THPVariable_Wrap(std::move(o));
  PyObject* out = PyTuple_New(2);
  if (out == nullptr) return nullptr;
  PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(std::move(o)));
  PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(std::move(lse)));
  return out;
}

// (q, k_cache, v_cache, page_table, seq_lens, scale, tail_mask, return_lse, window, sinks) -> o or (o, lse)
PyObject* attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 10 || g.attention == nullptr) return none();
  Request r{args};
  Attention a;
  a.q = r.tensor(0, at::ScalarType::Undefined);
  if (!a.read(r, at::ScalarType::Undefined, 3)) return none();
  return attend(r, a, g.attention_bytes, [&](const Scratch& ws, int* err, cudaStream_t stream, void* o, float* lse) {
    return g.attention(ptr(a.q), ptr(a.k), ptr(a.v), (int)a.k->size(0), (int)a.k->size(2), a.k->stride(0), a.k->stride(1),
                       a.k->stride(2), ptr<int32_t>(a.table), a.table->stride(0), (int)a.table->size(1), ptr<int32_t>(a.lens),
                       ptr<uint8_t>(a.tail), a.ldm_b, a.ldm_t, (int)a.B, (int)a.L, (int)a.Hq, (int)a.Hk, (int)a.D,
                       (float)a.scale, a.window, a.sinks, o, lse, a.code, ws.at, ws.bytes, err, stream);
  });
  END_HANDLE_TH_ERRORS
}

// scales of an 8-bit cache [pages, heads, page_size / block]
bool scales_good(const at::Tensor& cache, const at::Tensor& k, const at::Tensor& v) {
  return k.dim() == 3 && k.sizes() == v.sizes() && k.strides() == v.strides() && k.size(0) == cache.size(0) &&
         k.size(1) == cache.size(1) && k.size(2) > 0 && cache.size(2) % k.size(2) == 0;
}

// (q, k_cache, v_cache, k_scale, v_scale, page_table, seq_lens, scale, tail_mask, return_lse, window, sinks) -> o or (o, lse)
PyObject* attention8(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 12 || g.attention8 == nullptr) return none();
  Request r{args};
  Attention a;
  a.q = r.tensor(0, at::ScalarType::Undefined);
  const at::Tensor *ks = r.tensor(3, at::kFloat), *vs = r.tensor(4, at::kFloat);
  if (!a.read(r, at::kFloat8_e4m3fn, 5) || !scales_good(*a.k, *ks, *vs)) return none();
  return attend(r, a, g.attention8_bytes, [&](const Scratch& ws, int* err, cudaStream_t stream, void* o, float* lse) {
    return g.attention8(ptr(a.q), ptr(a.k), ptr(a.v), ptr<float>(ks), ptr<float>(vs), (int)a.k->size(0), (int)a.k->size(2),
                        (int)(a.k->size(2) / ks->size(2)), a.k->stride(0), a.k->stride(1), a.k->stride(2), ks->stride(0),
                        ks->stride(1), ks->stride(2), ptr<int32_t>(a.table), a.table->stride(0), (int)a.table->size(1),
                        ptr<int32_t>(a.lens), ptr<uint8_t>(a.tail), a.ldm_b, a.ldm_t, (int)a.B, (int)a.L, (int)a.Hq, (int)a.Hk,
                        (int)a.D, (float)a.scale, a.window, a.sinks, o, lse, a.code, ws.at, ws.bytes, err, stream);
  });
  END_HANDLE_TH_ERRORS
}

// (qkv, heads, kv_heads, k_cache, v_cache, k_scale, v_scale, page_table, seq_lens, cos, sin, q_weight, k_weight, eps, count) -> q
PyObject* append8(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 15 || g.append8 == nullptr) return none();
  Request r{args};
  const at::Tensor* qkv = r.tensor(0, at::ScalarType::Undefined);
  if (!r.good) return none();
  const auto type = qkv->scalar_type();
  const int code = half_code(*qkv);
  const long long heads = r.number(1), kv_heads = r.number(2);
  const at::Tensor *k = r.tensor(3, at::kFloat8_e4m3fn), *v = r.tensor(4, at::kFloat8_e4m3fn), *ks = r.tensor(5, at::kFloat),
                   *vs = r.tensor(6, at::kFloat), *table = r.tensor(7, at::kInt), *lens = r.tensor(8, at::kInt),
                   *cos = r.tensor(9, at::kFloat), *sin = r.tensor(10, at::kFloat), *qw = r.tensor(11, type, true),
                   *kw = r.tensor(12, type, true), *count = r.tensor(14, at::kInt, true);
  const double eps = r.real(13);
  if (!r.good || code < 0 || !cache_good(*k, *v, at::kFloat8_e4m3fn) || heads < 1 || heads > 65536 || kv_heads != k->size(1) ||
      !scales_good(*k, *ks, *vs))
    return none();
  if (qkv->dim() != 3) return none();
  const int64_t D = k->size(3), B = qkv->size(0);
  if (qkv->size(2) != (heads + 2 * kv_heads) * D || qkv->stride(2) != 1) return none();
  const int64_t L = qkv->size(1);
  if (B > INT_MAX || L > INT_MAX || table->dim() != 2 || table->size(0) != B || table->stride(1) != 1 ||
      table->size(1) > INT_MAX || !is_shape(*lens, {B}) || !lens->is_contiguous() || cos->dim() != 2 ||
      cos->sizes() != sin->sizes() || !cos->is_contiguous() || !sin->is_contiguous() || cos->size(1) > D ||
      (qw && (!is_shape(*qw, {D}) || !qw->is_contiguous())) || (kw && (!is_shape(*kw, {D}) || !kw->is_contiguous())) ||
      (count && (!is_shape(*count, {B}) || !count->is_contiguous())))
    return none();
  cudaStream_t stream;
  if (!r.here(stream)) return none();
  int* err = error_word(r.dev);
  if (err == nullptr) return PyErr_Occurred() ? nullptr : none();
  at::Tensor q = at::empty({B, L, heads, D}, qkv->options());
  const int rc = g.append8(ptr(qkv), qkv->stride(0), qkv->stride(1), (int)B, (int)L, (int)heads, (int)kv_heads, (int)D,
                           2 * (int)cos->size(1), ptr(qw), ptr(kw), (float)eps, ptr<float>(cos), ptr<float>(sin), cos->size(0),
                           ptr<int32_t>(table), table->stride(0), (int)table->size(1), ptr<int32_t>(lens), ptr<int32_t>(count),
                           q.data_ptr(), ptr(k), ptr(v), ptr<float>(ks), ptr<float>(vs), (int)k->size(0), (int)k->size(2),
                           (int)(k->size(2) / ks->size(2)), k->stride(0), k->stride(1), k->stride(2), ks->stride(0),
                           ks->stride(1), ks->stride(2), code, err, stream);
  return rc == SIMSD_OK ? THPVariable_Wrap(std::move(q)) : none();
  END_HANDLE_TH_ERRORS
}

// counters of a stream (its scratch), or nothing where the call has to go another way
bool counters(Request& r, cudaStream_t& stream, int*& err, Scratch& ws) {
  if (!r.here(stream) || c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None) return false;
  err = error_word(r.dev);
  if (err == nullptr) return false;
  ws = scratch(r.dev, stream, SIMSD_PAGED_COUNTER_BYTES);
  return ws.at != nullptr;
}
bool row_good(const at::Tensor& t, int64_t B) { return is_shape(t, {B}) && t.is_contiguous(); }
bool pool_good(const at::Tensor& table, const at::Tensor& pages, const at::Tensor& free) {
  return table.dim() == 2 && (table.size(1) < 2 || table.stride(1) == 1) && table.size(0) <= INT_MAX && table.size(1) <= INT_MAX &&
         pages.dim() == 1 && pages.is_contiguous() && pages.size(0) <= INT_MAX && free.numel() == 1;
}

// (page_table, lens, held, free_pages, free_count, L, page_size, count) -> (slots, positions, total)
PyObject* reserve(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 8 || g.reserve == nullptr) return none();
  Request r{args};
  const at::Tensor *table = r.tensor(0, at::kInt), *lens = r.tensor(1, at::kInt), *held = r.tensor(2, at::kInt),
                   *pages = r.tensor(3, at::kInt), *free = r.tensor(4, at::kInt), *count = r.tensor(7, at::kInt, true);
  const long long L = r.number(5), page_size = r.number(6);
  if (!r.good || !pool_good(*table, *pages, *free)) return none();
  const int64_t B = table->size(0);
  if (!row_good(*lens, B) || !row_good(*held, B) || (count && !row_good(*count, B)) || L < 0 || L > INT_MAX || page_size < 1 ||
      page_size > INT_MAX)
    return none();
  cudaStream_t stream;
  int* err;
  Scratch ws;
  if (!counters(r, stream, err, ws)) return PyErr_Occurred() ? nullptr : none();
  at::Tensor slots = at::empty({B, L}, table->options().dtype(at::kLong)), positions = at::empty_like(slots),
             total = at::empty({B}, table->options());
  const int rc = g.reserve(ptr<int32_t>(table), table->stride(0), (int)table->size(1), ptr<int32_t>(lens), ptr<int32_t>(count),
                           ptr<int32_t>(held), ptr<int32_t>(pages), (int)pages->size(0), ptr<int32_t>(free), (int)B, (int)L,
                           (int)page_size, slots.data_ptr<int64_t>(), positions.data_ptr<int64_t>(), total.data_ptr<int32_t>(),
                           ws.at, ws.bytes, err, stream);
  if (rc != SIMSD_OK) return none();
  PyObject* out = PyTuple_New(3);
  if (out == nullptr) return nullptr;
  PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(std::move(slots)));
  PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(std::move(positions)));
  PyTuple_SET_ITEM(out, 2, THPVariable_Wrap(std::move(total)));
  return out;
  END_HANDLE_TH_ERRORS
}

// (page_table, held, free_pages, free_count, keep, page_size) -> True
PyObject* release(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 6 || g.release == nullptr) return none();
  Request r{args};
  const at::Tensor *table = r.tensor(0, at::kInt), *held = r.tensor(1, at::kInt), *pages = r.tensor(2, at::kInt),
                   *free = r.tensor(3, at::kInt), *keep = r.tensor(4, at::kInt);
  const long long page_size = r.number(5);
  if (!r.good || !pool_good(*table, *pages, *free)) return none();
  const int64_t B = table->size(0);
  if (!row_good(*held, B) || !row_good(*keep, B) || page_size < 1 || page_size > INT_MAX) return none();
  cudaStream_t stream;
  int* err;
  Scratch ws;
  if (!counters(r, stream, err, ws)) return PyErr_Occurred() ? nullptr : none();
  const int rc = g.release(ptr<int32_t>(table), table->stride(0), (int)table->size(1), ptr<int32_t>(held), ptr<int32_t>(pages),
                           (int)pages->size(0), ptr<int32_t>(free), ptr<int32_t>(keep), (int)B, (int)page_size, ws.at, ws.bytes,
                           err, stream);
  if (rc != SIMSD_OK) return none();
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// (logits, counts, drafts, repetition, presence, frequency, seen, bias_ids, bias_values, allowed, out) -> out
PyObject* adjust(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 11 || g.adjust == nullptr) return none();
  Request r{args};
  const at::Tensor* x = r.tensor(0, at::ScalarType::Undefined);
  if (!r.good || x->dim() != 3) return none();
  const auto type = x->scalar_type();
  const int code = type == at::kFloat ? SIMSD_F32 : half_code(*x);
  const int64_t B = x->size(0), R = x->size(1), V = x->size(2), W = (V + 31) / 32;
  const at::Tensor *counts = r.tensor(1, at::kInt, true), *drafts = r.tensor(2, at::kLong, true),
                   *rep = r.tensor(3, at::kFloat, true), *pres = r.tensor(4, at::kFloat, true),
                   *freq = r.tensor(5, at::kFloat, true), *seen = r.tensor(6, at::kInt, true), *ids = r.tensor(7, at::kInt, true),
                   *vals = r.tensor(8, at::kFloat, true), *allowed = r.tensor(9, at::kInt, true), *out = r.tensor(10, type, true);
  auto rows = [](const at::Tensor* t, std::initializer_list<int64_t> s) {
    return t == nullptr || (is_shape(*t, s) && (t->size(-1) < 2 || t->stride(-1) == 1));
  };
  if (!r.good || code < 0 || V < 1 || R < 1 || B > INT_MAX || R > INT_MAX || V > INT_MAX || (V > 1 && x->stride(2) != 1) ||
      !rows(counts, {B, V}) || !rows(drafts, {B, R - 1}) || !rows(rep, {B}) || !rows(pres, {B}) || !rows(freq, {B}) ||
      !rows(seen, {B, W}) || (ids == nullptr) != (vals == nullptr) || !rows(out, {B, R, V}))
    return none();
  if (ids && (ids->dim() != 2 || ids->size(1) > INT_MAX || !rows(ids, {B, ids->size(1)}) || !rows(vals, {B, ids->size(1)}))) return none();
  if (allowed && !(allowed->dim() == 3 ? rows(allowed, {B, R, W}) : rows(allowed, {B, W}))) return none();
  cudaStream_t stream;
  if (!r.here(stream)) return none();
  int* err = error_word(r.dev);
  if (err == nullptr) return PyErr_Occurred() ? nullptr : none();
  at::Tensor y = out ? *out : at::empty({B, R, V}, x->options());
  auto ld = [](const at::Tensor* t) { return t ? t->stride(0) : 0; };
  const int rc = g.adjust(ptr(x), x->stride(0), x->stride(1), y.data_ptr(), y.stride(0), y.stride(1), (int)B, (int)R, (int)V, code,
                          ptr<int32_t>(counts), ld(counts), ptr<int64_t>(drafts), ld(drafts), ptr<uint32_t>(seen), ld(seen),
                          ptr<float>(rep), ptr<float>(pres), ptr<float>(freq), ptr<int32_t>(ids), ld(ids), ptr<float>(vals),
                          ld(vals), ids ? (int)ids->size(1) : 0, ptr<uint32_t>(allowed), ld(allowed),
                          allowed && allowed->dim() == 3 ? allowed->stride(1) : 0, err, stream);
  return rc == SIMSD_OK ? THPVariable_Wrap(std::move(y)) : none();
  END_HANDLE_TH_ERRORS
}

// (counts, tokens) -> True
PyObject* count(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 2 || g.count == nullptr) return none();
  Request r{args};
  const at::Tensor *counts = r.tensor(0, at::kInt), *tokens = r.tensor(1, at::kLong);
  if (!r.good || counts->dim() != 2 || tokens->dim() != 2 || counts->size(1) < 1 || counts->size(1) > INT_MAX ||
      counts->size(0) > INT_MAX || tokens->size(0) != counts->size(0) || tokens->size(1) > INT_MAX ||
      (counts->size(1) > 1 && counts->stride(1) != 1) || (tokens->size(1) > 1 && tokens->stride(1) != 1))
    return none();
  cudaStream_t stream;
  if (!r.here(stream)) return none();
  int* err = error_word(r.dev);
  if (err == nullptr) return PyErr_Occurred() ? nullptr : none();
  const int rc = g.count(ptr<int32_t>(counts), counts->stride(0), ptr<int64_t>(tokens), tokens->stride(0), (int)counts->size(0),
                         (int)tokens->size(1), (int)counts->size(1), err, stream);
  if (rc != SIMSD_OK) return none();
  Py_RETURN_TRUE;
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
  g.attention = reinterpret_cast<decltype(g.attention)>(address("simsd_paged_attention_window"));
  g.attention_bytes = reinterpret_cast<decltype(g.attention_bytes)>(address("simsd_paged_attention_workspace_size"));
  g.verify = reinterpret_cast<decltype(g.verify)>(address("simsd_speculative_verify"));
  g.verify_bytes = reinterpret_cast<decltype(g.verify_bytes)>(address("simsd_speculative_verify_workspace_size"));
  g.append8 = reinterpret_cast<decltype(g.append8)>(address("simsd_paged_append8"));
  g.attention8 = reinterpret_cast<decltype(g.attention8)>(address("simsd_paged_attention8"));
  g.attention8_bytes = reinterpret_cast<decltype(g.attention8_bytes)>(address("simsd_paged_attention8_workspace_size"));
  g.reserve = reinterpret_cast<decltype(g.reserve)>(address("simsd_paged_reserve"));
  g.release = reinterpret_cast<decltype(g.release)>(address("simsd_paged_release"));
  g.adjust = reinterpret_cast<decltype(g.adjust)>(address("simsd_adjust_logits"));
  g.count = reinterpret_cast<decltype(g.count)>(address("simsd_count_tokens"));
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
    {"paged_append8", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(append8)), METH_FASTCALL, nullptr},
    {"paged_attention8", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(attention8)), METH_FASTCALL, nullptr},
    {"paged_reserve", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(reserve)), METH_FASTCALL, nullptr},
    {"paged_release", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(release)), METH_FASTCALL, nullptr},
    {"adjust_logits", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(adjust)), METH_FASTCALL, nullptr},
    {"count_tokens", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(count)), METH_FASTCALL, nullptr},
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
