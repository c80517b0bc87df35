// The entry points over 4-bit caches and pages, on logits and of beam search as Python functions of torch tensors: the
// argument checks in C++, because in Python they take longer than the launch (a lone call 8.6 us of host time; here 4,
// what a launch alone takes) and these calls are made once per layer and step. Bound to the C ABI's functions by address
// (bind), so that the library is the one that kernels/cuda_ext.py loaded. A refused call raises RuntimeError.
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
decltype(&cohere_dec_attention_paged) f_paged;
decltype(&cohere_dec_attention_paged_q8) f_paged_q8;
decltype(&cohere_dec_gather_paged) f_gather_paged;
decltype(&cohere_dec_gather_paged_q8) f_gather_paged_q8;
decltype(&cohere_dec_beam_select_eos) f_select;
decltype(&cohere_dec_beam_reorder) f_reorder;
decltype(&cohere_dec_beam_advance) f_advance;
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

// pages (.., pages, KV, P, 128) with `lead` sizes before them, in 8 bits with scales
struct Pages {
  const Tensor &k, &v;
  const Tensor *ks = nullptr, *vs = nullptr;
  int64_t L, pages, KV, P;
  Pages(const Call& c, int at, int lead, bool q8) : k(c.tensor(at)), v(c.tensor(at + 1)) {
    c.need(k.dim() == lead + 4 && k.size(lead + 3) == 128 && v.sizes() == k.sizes() && k.is_contiguous() &&
               v.is_contiguous() && k.scalar_type() == (q8 ? at::kChar : at::kBFloat16) &&
               v.scalar_type() == k.scalar_type(),
           q8 ? "contiguous int8 pages (.., pages, KV, P, 128)" : "contiguous bf16 pages (.., pages, KV, P, 128)");
    c.need(k.numel() > 0, "no pages");
    L = lead ? k.size(0) : 1; pages = k.size(lead); KV = k.size(lead + 1); P = k.size(lead + 2);
    if (q8) {
      ks = &c.tensor(at + 2);
      vs = &c.tensor(at + 3);
      c.need(ks->sizes() == k.sizes().slice(0, lead + 3) && vs->sizes() == ks->sizes() &&
                 ks->scalar_type() == at::kFloat && vs->scalar_type() == at::kFloat && ks->is_contiguous() &&
                 vs->is_contiguous(),
             "contiguous fp32 scales, one a vector");
    }
  }
};

bool table_ok(const Call& c, const Tensor& t) { return t.dim() == 2 && t.size(0) > 0 && t.size(1) > 0 && c.index(t, 1); }

template <bool Q8>
void attention_paged(const Call& c) {
  constexpr int Z = Q8 ? 2 : 0;
  const Tensor &active = c.tensor(0), &q = c.tensor(2), &table = c.tensor(5 + Z), &n = c.tensor(6 + Z),
               &out = c.tensor(10 + Z);
  const Tensor *starts = c.maybe(1), *part = c.maybe(9 + Z);
  const Pages kv(c, 3, 0, Q8);
  const double scale = c.number(7 + Z);
  const int64_t splits = c.whole(8 + Z);
  c.need(q.dim() == 2 && out.dim() == 2 && q.scalar_type() == at::kBFloat16 && out.scalar_type() == at::kBFloat16 &&
             q.stride(1) == 1 && out.is_contiguous(),
         "bf16 q (rows, ...) with unit column stride, contiguous out");
  const int64_t rows = q.size(0), H = out.size(1) / 128, seqs = active.numel();
  c.need(out.size(0) == rows && H > 0 && out.size(1) % 128 == 0 && H % kv.KV == 0 && q.size(1) >= (H + 2 * kv.KV) * 128,
         "out (rows, H * 128), H a multiple of the key heads, q as wide as its heads");
  c.need(table_ok(c, table) && c.index(active, seqs) && c.index(n, table.size(0)),
         "int32 table (slots, pages), active per sequence, n per slot");
  c.need(starts ? c.index(*starts, seqs + 1) : rows == seqs, "int32 starts (sequences + 1), or a row per sequence");
  c.need(splits >= 1 && splits <= 64 && (splits == 1 || (part && part->scalar_type() == at::kFloat &&
                                                        part->is_contiguous() &&
                                                        part->numel() / 130 / splits >= rows * H)),
         "1 to 64 splits, more than 1 need part");
  if (rows == 0 || seqs == 0) return;
  void* st = c.stream(q, &active, starts, &kv.k, &kv.v, kv.ks, kv.vs, &table, &n, part, &out);
  launch([&] {
    if constexpr (Q8)
      return f_paged_q8(ptr<int32_t>(active), ptr<int32_t>(starts), seqs, ptr<uint16_t>(q), q.stride(0), rows,
                        ptr<int8_t>(kv.k), ptr<int8_t>(kv.v), ptr<float>(kv.ks), ptr<float>(kv.vs), kv.pages, kv.P,
                        ptr<int32_t>(table), table.size(1), ptr<int32_t>(n), table.size(0), H, kv.KV, (float)scale,
                        splits, ptr<float>(part), part ? part->numel() : 0, ptr<uint16_t>(out), st);
    else
      return f_paged(ptr<int32_t>(active), ptr<int32_t>(starts), seqs, ptr<uint16_t>(q), q.stride(0), rows,
                     ptr<uint16_t>(kv.k), ptr<uint16_t>(kv.v), kv.pages, kv.P, ptr<int32_t>(table), table.size(1),
                     ptr<int32_t>(n), table.size(0), H, kv.KV, (float)scale, splits, ptr<float>(part),
                     part ? part->numel() : 0, ptr<uint16_t>(out), st);
  });
}

template <bool Q8>
void gather_paged(const Call& c) {
  const Tensor &slot_of = c.tensor(0), &pos_of = c.tensor(1), &table = c.tensor(2), &kv = c.tensor(Q8 ? 7 : 5);
  const Pages p(c, 3, 1, Q8);
  c.need(kv.dim() == 2 && kv.scalar_type() == at::kBFloat16 && kv.size(1) == p.L * 2 * p.KV * 128 && kv.stride(1) == 1,
         "bf16 kv (rows, L * 2 * KV * 128) with unit column stride");
  const int64_t rows = kv.size(0);
  c.need(table_ok(c, table) && c.index(slot_of, rows) && c.index(pos_of, rows),
         "int32 table (slots, pages), slot and position per row");
  if (rows == 0) return;
  void* st = c.stream(kv, &slot_of, &pos_of, &table, &p.k, &p.v, p.ks, p.vs);
  launch([&] {
    if constexpr (Q8)
      return f_gather_paged_q8(ptr<int32_t>(slot_of), ptr<int32_t>(pos_of), rows, ptr<int32_t>(table), table.size(0),
                               table.size(1), ptr<int8_t>(p.k), ptr<int8_t>(p.v), ptr<float>(p.ks), ptr<float>(p.vs), p.L,
                               p.pages, p.KV, p.P, ptr<uint16_t>(kv), kv.stride(0), st);
    else
      return f_gather_paged(ptr<int32_t>(slot_of), ptr<int32_t>(pos_of), rows, ptr<int32_t>(table), table.size(0),
                            table.size(1), ptr<uint16_t>(p.k), ptr<uint16_t>(p.v), p.L, p.pages, p.KV, p.P,
                            ptr<uint16_t>(kv), kv.stride(0), st);
  });
}

// a contiguous matrix (or vector, w < 0) of at least `rows` rows of one type
bool matrix(const Tensor& t, at::ScalarType type, int64_t rows, int64_t w) {
  return t.scalar_type() == type && t.is_contiguous() &&
         (w < 0 ? t.dim() == 1 && t.size(0) >= rows : t.dim() == 2 && t.size(0) >= rows && t.size(1) == w);
}

void beam_select(const Call& c) {
  const Tensor &logits = c.tensor(0), &groups = c.tensor(1), &score = c.tensor(2), &finished = c.tensor(3),
               &parent = c.tensor(7), &token = c.tensor(8), &total = c.tensor(9), &work = c.tensor(10);
  const Tensor *made = c.maybe(4), *norm = c.maybe(5);
  const int64_t pad = c.whole(6), eos = c.whole(11), n = groups.numel();
  c.need(score.dim() == 2 && score.size(0) > 0 && score.size(1) >= 1 && score.size(1) <= 16, "score (groups, 1 to 16 beams)");
  const int64_t G = score.size(0), B = score.size(1);
  c.need(logits.dim() == 2 && logits.scalar_type() == at::kBFloat16 && logits.size(0) == n * B && logits.stride(1) == 1,
         "bf16 logits (groups * beams, V) with unit column stride");
  c.need(c.index(groups, n) && matrix(score, at::kFloat, G, B) && matrix(finished, at::kByte, G, B),
         "int32 groups, contiguous fp32 score and uint8 finished (groups, beams)");
  c.need(!norm || (made && matrix(*made, at::kInt, G, B) && matrix(*norm, at::kFloat, 1, -1)),
         "fp32 norm needs int32 made (groups, beams)");
  c.need(matrix(parent, at::kInt, n, B) && matrix(token, at::kLong, n, B) && matrix(total, at::kFloat, n, B),
         "int32 parent, int64 token, fp32 total (groups, beams)");
  c.need(work.scalar_type() == at::kByte && work.is_contiguous(), "contiguous uint8 work");
  if (n == 0) return;
  void* st = c.stream(logits, &groups, &score, &finished, made, norm, &parent, &token, &total, &work);
  launch([&] {
    return f_select(ptr<uint16_t>(logits), logits.stride(0), n, B, logits.size(1), ptr<int32_t>(groups), G,
                    ptr<float>(score), ptr<uint8_t>(finished), ptr<int32_t>(made), ptr<float>(norm),
                    norm ? norm->numel() : 0, pad, eos, ptr<int32_t>(parent), ptr<int64_t>(token), ptr<float>(total),
                    work.data_ptr(), work.numel(), st);
  });
}

void beam_reorder(const Call& c) {
  const Tensor &groups = c.tensor(0), &parent = c.tensor(1), &n = c.tensor(2);
  const Tensor *done = c.maybe(3), *table = c.maybe(4), *tokens = c.maybe(5), *states = c.maybe(6), *k = c.maybe(7),
               *ks = c.maybe(9);
  const int64_t m = groups.numel();
  c.need(parent.dim() == 2 && parent.size(1) >= 1 && parent.size(1) <= 16, "parent (groups, 1 to 16 beams)");
  const int64_t B = parent.size(1), slots = n.numel(), G = slots / B;
  c.need(c.index(groups, m) && matrix(parent, at::kInt, m, B) && c.index(n, 1) && slots % B == 0,
         "int32 groups, parent (groups, beams), n per slot (groups * beams)");
  c.need(!done || matrix(*done, at::kByte, G, -1), "uint8 done per group");
  c.need(!table || (table_ok(c, *table) && table->size(0) >= slots), "int32 table (slots, pages)");
  c.need(!tokens || (tokens->dim() == 2 && tokens->size(1) > 0 && matrix(*tokens, at::kLong, slots, tokens->size(1))),
         "contiguous int64 tokens (slots, positions)");
  c.need(!states || (states->dim() == 2 && states->size(1) > 0 && matrix(*states, at::kInt, slots, states->size(1))),
         "contiguous int32 states (slots, ..)");
  c.need(!k || table, "pages need a table");
  const Tensor* v = c.maybe(8);
  const Tensor* vs = c.maybe(10);
  c.need(!k == !v && !ks == !vs && (k || !ks), "keys and values, or neither");
  int64_t L = 0, pages = 0, KV = 0, P = 1;
  if (k) {
    const Pages p(c, 7, 1, ks != nullptr);
    L = p.L; pages = p.pages; KV = p.KV; P = p.P;
  }
  if (m == 0) return;
  void* st = c.stream(groups, &parent, &n, done, table, tokens, states, k, v, ks, vs);
  launch([&] {
    return f_reorder(ptr<int32_t>(groups), m, B, ptr<int32_t>(parent), ptr<int32_t>(n), ptr<uint8_t>(done), G,
                     ptr<int32_t>(table), table ? table->size(1) : 0, ptr<int64_t>(tokens), tokens ? tokens->size(1) : 0,
                     ptr<int32_t>(states), states ? states->size(1) : 0, k ? k->data_ptr() : nullptr,
                     v ? v->data_ptr() : nullptr, ptr<float>(ks), ptr<float>(vs), L, pages, KV, P, ks ? 8 : 16, st);
  });
}

void beam_advance(const Call& c) {
  const Tensor &groups = c.tensor(0), &parent = c.tensor(1), &token = c.tensor(2), &total = c.tensor(3), &tok = c.tensor(5),
               &pos = c.tensor(6), &score = c.tensor(8), &finished = c.tensor(9), &made = c.tensor(10), &done = c.tensor(11),
               &limit = c.tensor(12), &out = c.tensor(13), &emb = c.tensor(16), &ptab = c.tensor(17), &w0 = c.tensor(18),
               &b0 = c.tensor(19), &w1 = c.tensor(21), &b1 = c.tensor(22), &x = c.tensor(24), &h = c.tensor(25);
  const Tensor *held = c.maybe(7), *flags = c.maybe(26);
  const int64_t dummy = c.whole(4), eos = c.whole(14), n = groups.numel();
  const bool by_length = c.truth(15);
  const double eps0 = c.number(20), eps1 = c.number(23);
  c.need(score.dim() == 2 && score.size(0) > 0 && score.size(1) >= 1 && score.size(1) <= 16, "score (groups, 1 to 16 beams)");
  const int64_t G = score.size(0), B = score.size(1);
  c.need(c.index(groups, n) && matrix(parent, at::kInt, n, B) && matrix(token, at::kLong, n, B) &&
             matrix(total, at::kFloat, n, B),
         "int32 groups and parent, int64 token, fp32 total (groups, beams)");
  c.need(matrix(tok, at::kLong, G * B, -1) && matrix(pos, at::kInt, G * B, -1) &&
             (!held || matrix(*held, at::kInt, G * B, -1)) && matrix(score, at::kFloat, G, B) &&
             matrix(finished, at::kByte, G, B) && matrix(made, at::kInt, G, B) && matrix(done, at::kByte, G, -1) &&
             matrix(limit, at::kInt, G, -1) && out.dim() == 2 && out.size(1) > 0 &&
             matrix(out, at::kLong, G * B, out.size(1)),
         "the groups' state: tok, pos, out per slot, score, finished, made (groups, beams), done, limit per group");
  c.need(emb.dim() == 2 && ptab.dim() == 2 && emb.size(1) == ptab.size(1) && emb.size(0) > 0 && ptab.size(0) > 0, "emb, ptab");
  const int64_t w = emb.size(1);
  c.need(matrix(emb, at::kBFloat16, 1, w) && matrix(ptab, at::kBFloat16, 1, w) && matrix(w0, at::kBFloat16, w, -1) &&
             matrix(b0, at::kBFloat16, w, -1) && matrix(w1, at::kBFloat16, w, -1) && matrix(b1, at::kBFloat16, w, -1) &&
             matrix(x, at::kBFloat16, n * B, w) && matrix(h, at::kBFloat16, n * B, w),
         "contiguous bf16 emb, ptab, norms, x, h of one width");
  c.need(!flags || (flags->scalar_type() == at::kByte && flags->is_contiguous() && flags->numel() >= G && flags->is_cpu()),
         "flags: pinned uint8 per group");
  if (n == 0) return;
  void* st = c.stream(groups, &parent, &token, &total, &tok, &pos, held, &score, &finished, &made, &done, &limit, &out, &emb,
                      &ptab, &w0, &b0, &w1, &b1, &x, &h);
  launch([&] {
    return f_advance(ptr<int32_t>(groups), n, B, ptr<int32_t>(parent), ptr<int64_t>(token), ptr<float>(total), G, dummy,
                     ptr<int64_t>(tok), ptr<int32_t>(pos), ptr<int32_t>(held), ptr<float>(score), ptr<uint8_t>(finished),
                     ptr<int32_t>(made), ptr<uint8_t>(done), ptr<int32_t>(limit), ptr<int64_t>(out), out.size(1), eos,
                     by_length,
                     ptr<uint16_t>(emb), emb.size(0), ptr<uint16_t>(ptab), ptab.size(0), ptr<uint16_t>(w0),
                     ptr<uint16_t>(b0), (float)eps0, ptr<uint16_t>(w1), ptr<uint16_t>(b1), (float)eps1, ptr<uint16_t>(x),
                     ptr<uint16_t>(h), w, ptr<uint8_t>(flags), st);
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
constexpr auto paged = attention_paged<false>, paged_q8 = attention_paged<true>, gather_pages = gather_paged<false>,
               gather_pages_q8 = gather_paged<true>;
ENTRY("dec_attention_paged", paged, 11)
ENTRY("dec_attention_paged_q8", paged_q8, 13)
ENTRY("dec_gather_paged", gather_pages, 6)
ENTRY("dec_gather_paged_q8", gather_pages_q8, 8)
ENTRY("dec_beam_select", beam_select, 12)
ENTRY("dec_beam_reorder", beam_reorder, 11)
ENTRY("dec_beam_advance", beam_advance, 27)

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
  at("cohere_dec_attention_paged", f_paged);
  at("cohere_dec_attention_paged_q8", f_paged_q8);
  at("cohere_dec_gather_paged", f_gather_paged);
  at("cohere_dec_gather_paged_q8", f_gather_paged_q8);
  at("cohere_dec_beam_select_eos", f_select);
  at("cohere_dec_beam_reorder", f_reorder);
  at("cohere_dec_beam_advance", f_advance);
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
                         METHOD("dec_attention_paged", paged),
                         METHOD("dec_attention_paged_q8", paged_q8),
                         METHOD("dec_gather_paged", gather_pages),
                         METHOD("dec_gather_paged_q8", gather_pages_q8),
                         METHOD("dec_beam_select", beam_select),
                         METHOD("dec_beam_reorder", beam_reorder),
                         METHOD("dec_beam_advance", beam_advance),
                         {"bind", bind, METH_O, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "cohere_calls", "Calls of the C ABI with torch tensors.", -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit_cohere_calls(void) { return PyModule_Create(&module); }
