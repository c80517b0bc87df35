// The entry points over 4-bit caches and on logits as Python functions of torch tensors: the argument checks in C++,
// because in Python they take longer than the launch (a lone call 8.6 us of host time; here 4, what a launch alone takes)
// and these calls are made once per layer and step. Bound to the C ABI's functions by address (bind), so that the
// library is the one that kernels/cuda_ext.py loaded. A refused call raises RuntimeError.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <torch/csrc/autograd/python_variable.h>

#include <stdexcept>
#include <string>

#include "cohere_hip.h"

namespace {

using at::Tensor;

decltype(&cohere_dec_attention_q4) f_attention;
decltype(&cohere_dec_scatter_kv_q4) f_scatter;
decltype(&cohere_dec_gather_kv_q4) f_gather;
decltype(&cohere_gemm_kv_q4) f_gemm_kv;
decltype(&cohere_dec_logits) f_logits;
decltype(&cohere_last_error) f_error;
PyObject *get_device, *get_stream;  // torch._C's

struct Refused : std::runtime_error {
  using std::runtime_error::runtime_error;
};

// one call's arguments
struct Call {
  const char* name;
  PyObject* const* args;
  Py_ssize_t n;

  [[noreturn]] void refuse(const char* why) const { throw Refused(std::string(name) + ": " + why); }
  void need(bool ok, const char* why) const {
    if (__builtin_expect(!ok, 0)) refuse(why);
  }
  const Tensor* maybe(int i) const {
    if (args[i] == Py_None) return nullptr;
    need(THPVariable_Check(args[i]), "a tensor expected");
    const Tensor& t = THPVariable_Unpack(args[i]);
    need(t.defined() && t.layout() == at::kStrided, "a dense tensor expected");
    return &t;
  }
  const Tensor& tensor(int i) const {
    const Tensor* t = maybe(i);
    need(t != nullptr, "a tensor is missing");
    return *t;
  }
  int64_t whole(int i) const {
    const long long v = PyLong_AsLongLong(args[i]);
    if (v == -1 && PyErr_Occurred()) {
      PyErr_Clear();
      refuse("a whole number expected");
    }
    return v;
  }
  double number(int i) const {
    const double v = PyFloat_AsDouble(args[i]);
    if (v == -1. && PyErr_Occurred()) {
      PyErr_Clear();
      refuse("a number expected");
    }
    return v;
  }
  bool truth(int i) const {
    const int v = PyObject_IsTrue(args[i]);
    if (v < 0) {
      PyErr_Clear();
      refuse("a truth value expected");
    }
    return v != 0;
  }
  // the stream to launch on: every tensor (null: absent) has to be on the current GPU
  template <class... T>
  void* stream(const Tensor& first, const T*... rest) const {
    const int dev = first.is_cuda() ? first.get_device() : -1;
    need(dev >= 0 && ((!rest || (rest->is_cuda() && rest->get_device() == dev)) && ...),
         "tensors on the current GPU expected");
    PyObject* cur = PyObject_CallNoArgs(get_device);
    const long now = cur ? PyLong_AsLong(cur) : -1;
    Py_XDECREF(cur);
    PyErr_Clear();
    need(now == dev, "tensors on the current GPU expected");
    PyObject* d = PyLong_FromLong(dev);
    PyObject* s = d ? PyObject_CallOneArg(get_stream, d) : nullptr;
    Py_XDECREF(d);
    void* raw = s ? PyLong_AsVoidPtr(s) : nullptr;
    Py_XDECREF(s);
    const bool bad = PyErr_Occurred() != nullptr;
    PyErr_Clear();
    need(!bad, "no stream");
    return raw;
  }
  // at least n int32 values one after the other
  bool index(const Tensor& t, int64_t n) const {
    return t.scalar_type() == at::kInt && t.numel() >= n && t.is_contiguous();
  }
};

template <class T>
T* ptr(const Tensor& t) {
  return static_cast<T*>(t.data_ptr());
}
template <class T>
T* ptr(const Tensor* t) {
  return t ? static_cast<T*>(t->data_ptr()) : nullptr;
}

// the launch, with the interpreter free for other threads meanwhile
template <class F>
void launch(F f) {
  int rc;
  Py_BEGIN_ALLOW_THREADS;
  rc = f();
  Py_END_ALLOW_THREADS;
  if (rc) throw Refused(f_error());
}

// codes uint8 (..., 64) and maxima bf16 (..., 4), keys and values alike, `dims` sizes before them
struct Caches {
  const Tensor &k4, &v4, &ks, &vs;
  Caches(const Call& c, int at, int dims)
      : k4(c.tensor(at)), v4(c.tensor(at + 1)), ks(c.tensor(at + 2)), vs(c.tensor(at + 3)) {
    c.need(k4.dim() == dims + 1 && k4.size(dims) == 64 && v4.sizes() == k4.sizes() && k4.scalar_type() == at::kByte &&
               v4.scalar_type() == at::kByte && k4.is_contiguous() && v4.is_contiguous(),
           "contiguous uint8 caches of 64 bytes a vector");
    c.need(ks.dim() == dims + 1 && ks.size(dims) == 4 && ks.sizes().slice(0, dims) == k4.sizes().slice(0, dims) &&
               vs.sizes() == ks.sizes() && ks.scalar_type() == at::kBFloat16 && vs.scalar_type() == at::kBFloat16 &&
               ks.is_contiguous() && vs.is_contiguous(),
           "contiguous bf16 maxima, 4 a vector");
    c.need(k4.numel() > 0, "empty caches");
  }
};

void attention(const Call& c) {
  const bool self = c.truth(0);
  const Tensor &active = c.tensor(1), &q = c.tensor(2), &n = c.tensor(7), &out = c.tensor(11);
  const Caches kv(c, 3, 3);
  const double scale = c.number(8);
  const int64_t splits = c.whole(9);
  const Tensor* part = c.maybe(10);
  const int64_t S = kv.k4.size(0), KV = kv.k4.size(1), T = kv.k4.size(2);
  c.need(q.dim() == 2 && out.dim() == 2 && q.scalar_type() == at::kBFloat16 && out.scalar_type() == at::kBFloat16 &&
             q.stride(1) == 1 && out.is_contiguous(),
         "bf16 q (rows, ...) with unit column stride, contiguous out");
  const int64_t rows = q.size(0), H = out.size(1) / 128;
  c.need(out.size(0) == rows && H > 0 && out.size(1) % 128 == 0 && H % KV == 0 &&
             q.size(1) >= (H + (self ? 2 * KV : 0)) * 128,
         "out (rows, H * 128), H a multiple of the key heads, q as wide as its heads");
  c.need(c.index(active, rows) && c.index(n, S), "int32 active per row, n per slot");
  c.need(splits >= 1 && splits <= 64 && (splits == 1 || (part && part->scalar_type() == at::kFloat &&
                                                        part->is_contiguous() &&
                                                        part->numel() / 130 / splits >= rows * H)),
         "1 to 64 splits, more than 1 need part");
  if (rows == 0) return;
  void* st = c.stream(q, &active, &kv.k4, &kv.v4, &kv.ks, &kv.vs, &n, part, &out);
  launch([&] {
    return f_attention(self, ptr<int32_t>(active), rows, ptr<uint16_t>(q), q.stride(0), ptr<uint8_t>(kv.k4),
                       ptr<uint8_t>(kv.v4), ptr<uint16_t>(kv.ks), ptr<uint16_t>(kv.vs), ptr<int32_t>(n), S, H, KV, T,
                       (float)scale, splits, ptr<float>(part), part ? part->numel() : 0, ptr<uint16_t>(out), st);
  });
}

// kv, slot_of, frame_of and the caches of a scatter or gather
struct Rows {
  const Caches caches;
  const Tensor &kv, &slot_of, &frame_of;
  int64_t rows, L, S, H, T;
  void* stream = nullptr;
  Rows(const Call& c, int kv_at, int slot_at, int cache_at)
      : caches(c, cache_at, 4), kv(c.tensor(kv_at)), slot_of(c.tensor(slot_at)), frame_of(c.tensor(slot_at + 1)) {
    L = caches.k4.size(0); S = caches.k4.size(1); H = caches.k4.size(2); T = caches.k4.size(3);
    c.need(kv.dim() == 2 && kv.scalar_type() == at::kBFloat16 && kv.size(1) == L * 2 * H * 128 && kv.stride(1) == 1,
           "bf16 kv (rows, L * 2 * H * 128) with unit column stride");
    rows = kv.size(0);
    c.need(c.index(slot_of, rows) && c.index(frame_of, rows), "int32 slot and position per row");
    if (rows) stream = c.stream(kv, &slot_of, &frame_of, &caches.k4, &caches.v4, &caches.ks, &caches.vs);
  }
};

void scatter(const Call& c) {
  const Rows r(c, 0, 1, 3);
  if (r.rows == 0) return;
  launch([&] {
    return f_scatter(ptr<uint16_t>(r.kv), r.kv.stride(0), r.rows, ptr<int32_t>(r.slot_of), ptr<int32_t>(r.frame_of),
                     ptr<uint8_t>(r.caches.k4), ptr<uint8_t>(r.caches.v4), ptr<uint16_t>(r.caches.ks),
                     ptr<uint16_t>(r.caches.vs), r.L, r.S, r.H, r.T, r.stream);
  });
}

void gather(const Call& c) {
  const Rows r(c, 6, 0, 2);
  if (r.rows == 0) return;
  launch([&] {
    return f_gather(ptr<int32_t>(r.slot_of), ptr<int32_t>(r.frame_of), r.rows, ptr<uint8_t>(r.caches.k4),
                    ptr<uint8_t>(r.caches.v4), ptr<uint16_t>(r.caches.ks), ptr<uint16_t>(r.caches.vs), r.L, r.S, r.H, r.T,
                    ptr<uint16_t>(r.kv), r.kv.stride(0), r.stream);
  });
}

void gemm_kv(const Call& c) {
  const Tensor &a = c.tensor(0), &w = c.tensor(1), &slot_of = c.tensor(3), &frame_of = c.tensor(4);
  const Tensor* bias = c.maybe(2);
  const Caches kv(c, 5, 4);
  const int64_t L = kv.k4.size(0), S = kv.k4.size(1), H = kv.k4.size(2), T = kv.k4.size(3);
  c.need(a.dim() == 2 && w.dim() == 2 && a.scalar_type() == at::kBFloat16 && w.scalar_type() == at::kBFloat16 &&
             a.stride(1) == 1 && w.is_contiguous() && w.size(0) == L * 2 * H * 128 && w.size(1) == a.size(1) &&
             a.size(1) % 32 == 0 && (!bias || (bias->scalar_type() == at::kBFloat16 && bias->is_contiguous() &&
                                               bias->numel() == w.size(0))),
         "bf16 a (rows, K), w (L * 2 * H * 128, K), bias, K % 32 == 0");
  const int64_t rows = a.size(0);
  c.need(c.index(slot_of, rows) && c.index(frame_of, rows), "int32 slot and position per row");
  if (rows == 0) return;
  void* st = c.stream(a, &w, bias, &slot_of, &frame_of, &kv.k4, &kv.v4, &kv.ks, &kv.vs);
  launch([&] {
    return f_gemm_kv(ptr<uint16_t>(a), a.stride(0), ptr<uint16_t>(w), ptr<uint16_t>(bias), rows, a.size(1),
                     ptr<int32_t>(slot_of), ptr<int32_t>(frame_of), ptr<uint8_t>(kv.k4), ptr<uint8_t>(kv.v4),
                     ptr<uint16_t>(kv.ks), ptr<uint16_t>(kv.vs), L, S, H, T, st);
  });
}

void logits(const Call& c) {
  const Tensor &x = c.tensor(0), &y = c.tensor(1), &active = c.tensor(2), &pos = c.tensor(3);
  const Tensor *tokens = c.maybe(4), *first = c.maybe(5), *plen = c.maybe(6), *pen = c.maybe(7), *bias = c.maybe(8),
               *bias_of = c.maybe(9), *mask = c.maybe(10), *classes = c.maybe(11), *trans = c.maybe(12),
               *start = c.maybe(13), *state = c.maybe(14);
  c.need(x.dim() == 2 && x.size(1) > 0 && x.size(1) % 8 == 0 && y.sizes() == x.sizes() &&
             x.scalar_type() == at::kBFloat16 && y.scalar_type() == at::kBFloat16 && x.stride(1) == 1 && y.stride(1) == 1,
         "bf16 logits and y (rows, V), unit column stride, V % 8 == 0");
  const int64_t rows = x.size(0), V = x.size(1), S = pos.numel();
  c.need(c.index(active, rows) && c.index(pos, 1) && (!first || c.index(*first, S)) && (!plen || c.index(*plen, S)),
         "int32 active per row, pos, first, plen per slot");
  c.need(!tokens || (tokens->dim() == 2 && tokens->scalar_type() == at::kLong && tokens->is_contiguous() &&
                     tokens->size(0) >= S && tokens->size(1) > 0),
         "contiguous int64 tokens (slots, positions)");
  c.need(!pen || (pen->dim() == 2 && pen->size(0) == S && pen->size(1) == 3 && pen->scalar_type() == at::kFloat &&
                  pen->is_contiguous() && tokens && first),
         "penalties fp32 (slots, 3) need tokens and first");
  c.need(!bias || (bias->dim() == 2 && bias->size(0) > 0 && bias->size(1) == V && bias->scalar_type() == at::kBFloat16 &&
                   bias->is_contiguous() && bias_of && c.index(*bias_of, S)),
         "bias bf16 (B, V) needs int32 bias_of per slot");
  c.need(!mask || (mask->dim() == 2 && mask->size(0) > 0 && mask->size(1) == (V + 31) / 32 && c.index(*mask, 1) && start &&
                   c.index(*start, S)),
         "mask int32 (M, ceil(V / 32)) needs int32 start per slot");
  c.need((!classes && !trans) ||
             (classes && trans && mask && classes->numel() == V && c.index(*classes, V) && trans->dim() == 2 &&
              trans->size(0) == mask->size(0) && trans->size(1) > 0 && c.index(*trans, 1) && state && state->dim() == 2 &&
              state->size(0) == S && state->size(1) == 2 && c.index(*state, 1) && tokens && plen),
         "a grammar needs mask, classes (V), trans (M, C), state (slots, 2), tokens and plen");
  if (rows == 0) return;
  void* st = c.stream(x, &y, &active, &pos, tokens, first, plen, pen, bias, bias_of, mask, classes, trans, start, state);
  launch([&] {
    return f_logits(ptr<uint16_t>(x), x.stride(0), ptr<uint16_t>(y), y.stride(0), rows, V, ptr<int32_t>(active),
                    ptr<int32_t>(pos), S, ptr<int64_t>(tokens), tokens ? tokens->size(1) : 1, ptr<int32_t>(first),
                    ptr<int32_t>(plen), ptr<float>(pen), ptr<uint16_t>(bias), bias ? bias->size(0) : 0,
                    ptr<int32_t>(bias_of), ptr<int32_t>(mask), mask ? mask->size(0) : 0, ptr<int32_t>(classes),
                    ptr<int32_t>(trans), trans ? trans->size(1) : 0, ptr<int32_t>(start), ptr<int32_t>(state), st);
  });
}

// no C++ exception leaves a function that Python calls
template <void (*F)(const Call&), int N>
PyObject* entry(const char* name, PyObject* const* args, Py_ssize_t n) {
  if (n != N) return PyErr_Format(PyExc_TypeError, "%s takes %d arguments", name, N);
  try {
    if (!f_error) throw Refused("the library is not bound");
    F(Call{name, args, n});
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  } catch (...) {
    PyErr_Format(PyExc_RuntimeError, "%s failed", name);
    return nullptr;
  }
  Py_RETURN_NONE;
}
#define ENTRY(NAME, F, N)                                                             \
  PyObject* py_##F(PyObject*, PyObject* const* args, Py_ssize_t n) {                  \
    return entry<F, N>(NAME, args, n);                                                \
  }
ENTRY("dec_attention_q4", attention, 12)
ENTRY("dec_scatter_kv_q4", scatter, 7)
ENTRY("dec_gather_kv_q4", gather, 7)
ENTRY("gemm_kv_q4", gemm_kv, 9)
ENTRY("dec_logits", logits, 15)

// bind(addresses): the C ABI's functions by name
PyObject* bind(PyObject*, PyObject* addresses) {
  if (!PyDict_Check(addresses)) return PyErr_Format(PyExc_TypeError, "bind takes the functions' addresses by name");
  bool ok = true;
  const auto at = [&](const char* name, auto& f) {
    PyObject* v = PyDict_GetItemString(addresses, name);
    void* p = v ? PyLong_AsVoidPtr(v) : nullptr;
    if (!p) ok = false;
    else f = reinterpret_cast<std::remove_reference_t<decltype(f)>>(p);
  };
  at("cohere_dec_attention_q4", f_attention);
  at("cohere_dec_scatter_kv_q4", f_scatter);
  at("cohere_dec_gather_kv_q4", f_gather);
  at("cohere_gemm_kv_q4", f_gemm_kv);
  at("cohere_dec_logits", f_logits);
  PyObject* c = PyImport_ImportModule("torch._C");
  if (c) {
    get_device = PyObject_GetAttrString(c, "_cuda_getDevice");
    get_stream = PyObject_GetAttrString(c, "_cuda_getCurrentRawStream");
    Py_DECREF(c);
  }
  if (PyErr_Occurred()) return nullptr;
  if (ok) at("cohere_last_error", f_error);
  if (!ok) return PyErr_Format(PyExc_ImportError, "bind: a function is missing");
  Py_RETURN_NONE;
}

#define METHOD(NAME, F) {NAME, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_##F)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD("dec_attention_q4", attention),
                         METHOD("dec_scatter_kv_q4", scatter),
                         METHOD("dec_gather_kv_q4", gather),
                         METHOD("gemm_kv_q4", gemm_kv),
                         METHOD("dec_logits", logits),
                         {"bind", bind, METH_O, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "cohere_calls", "Calls of the C ABI with torch tensors.", -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit_cohere_calls(void) { return PyModule_Create(&module); }
