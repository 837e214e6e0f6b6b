// ops_torch.cpp -- the batched decode operators on torch tensors: a CPython
// module (_ops) that takes shapes, strides, types and addresses from the
// tensors, checks that they fit together, and calls libchpe.so on the current
// stream of the tensors' device.
//
// A decode step calls the operators hundreds of times (three per layer), each
// for a few microseconds of GPU work: the same checks written in Python took
// 10 to 14 us a call, here they take under one.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstdint>
#include <stdexcept>
#include <string>

#include "../../include/chpe.h"

namespace {

using at::Tensor;

struct Unfit : std::runtime_error {  // becomes ValueError
  using std::runtime_error::runtime_error;
};
struct Misuse : std::runtime_error {  // becomes TypeError
  using std::runtime_error::runtime_error;
};
void want(bool ok, const char* what) {
  if (!ok) throw Unfit(what);
}
[[noreturn]] void unfit(const std::string& what) { throw Unfit(what); }

const char* type_name(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return "float32";
    case at::kInt: return "int32";
    case at::kLong: return "int64";
    case at::kByte: return "uint8";
    case at::kHalf: return "float16";
    case at::kBFloat16: return "bfloat16";
    default: return c10::toString(t);
  }
}
int dtype_of(const Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kFloat: return CHPE_F32;
    case at::kHalf: return CHPE_F16;
    case at::kBFloat16: return CHPE_BF16;
    default: unfit(std::string(name) + " must be float32, float16 or bfloat16, not " + type_name(t.scalar_type()));
  }
}

// The operators have no gradient: one that autograd would expect must not get lost.
void no_gradient(const Tensor& t, const char* name) {
  if (t.requires_grad() && c10::GradMode::is_enabled())
    unfit(std::string(name) + " requires a gradient, which this operator does not have: call it under torch.no_grad()");
}

// ---- arguments: positional and by name -----------------------------------------
template <int N>
struct Args {
  PyObject* at[N] = {};

  // names[0..positional) may be given by position, all of them by name
  void parse(PyObject* const* names, int positional, PyObject* const* args, Py_ssize_t n, PyObject* kw, const char* fn) {
    if (n > positional) throw Misuse(std::string(fn) + " takes " + std::to_string(positional) + " arguments by position");
    for (Py_ssize_t i = 0; i < n; i++) at[i] = args[i];
    const Py_ssize_t k = kw ? PyTuple_GET_SIZE(kw) : 0;
    for (Py_ssize_t j = 0; j < k; j++) {
      PyObject* key = PyTuple_GET_ITEM(kw, j);
      int i = 0;
      while (i < N && names[i] != key) i++;
      if (i == N)  // not the interned name: compare the letters
        for (i = 0; i < N && PyUnicode_Compare(names[i], key) != 0;) i++;
      if (i == N || (i < n)) {
        const char* s = PyUnicode_AsUTF8(key);
        if (!s) PyErr_Clear();
        throw Misuse(std::string(fn) + (i == N ? ": unknown argument " : ": given twice: ") + (s ? s : "?"));
      }
      at[i] = args[n + j];
    }
    for (int i = 0; i < N; i++)
      if (at[i] == Py_None) at[i] = nullptr;
  }
  const Tensor* tensor(int i, const char* name, bool needed = false) const {
    if (!at[i]) {
      if (needed) throw Misuse(std::string(name) + " is missing");
      return nullptr;
    }
    if (!THPVariable_Check(at[i])) throw Misuse(std::string(name) + " must be a tensor");
    const Tensor& t = THPVariable_Unpack(at[i]);
    no_gradient(t, name);
    return &t;
  }
  double number(int i, const char* name, double def) const {
    if (!at[i]) return def;
    const double v = PyFloat_AsDouble(at[i]);
    if (v == -1.0 && PyErr_Occurred()) {
      PyErr_Clear();
      throw Misuse(std::string(name) + " must be a number");
    }
    return v;
  }
};

// ---- tensors ---------------------------------------------------------------------
void on(const Tensor& t, const char* name, at::ScalarType type, int dev) {
  if (!t.is_cuda() || t.get_device() != dev || t.scalar_type() != type)
    unfit(std::string(name) + " must be a " + type_name(type) + " tensor on cuda:" + std::to_string(dev));
}
int cuda_of(const Tensor& t, const char* name) {
  if (!t.is_cuda()) unfit(std::string(name) + " must be a CUDA tensor");
  return t.get_device();
}
// Address of a contiguous 1-D tensor of n values (nullptr: none given).
template <typename T>
T* vec(const Tensor* t, const char* name, at::ScalarType type, int64_t n, int dev) {
  if (!t) return nullptr;
  on(*t, name, type, dev);
  if (t->dim() != 1 || t->size(0) != n || !t->is_contiguous())
    unfit(std::string(name) + " must be a contiguous tensor of " + std::to_string(n) + " values");
  return static_cast<T*>(t->data_ptr());
}
// Stride between the tokens of [n, heads, d] whose heads are contiguous.
int64_t heads_of(const Tensor& t, const char* name, at::ScalarType type, int dev, int64_t n, int64_t heads, int64_t d) {
  on(t, name, type, dev);
  if (t.dim() != 3 || t.size(0) != n || t.size(1) != heads || t.size(2) != d)
    unfit(std::string(name) + " must have the shape [" + std::to_string(n) + ", " + std::to_string(heads) + ", " +
          std::to_string(d) + "]");
  if (t.numel() && ((d > 1 && t.stride(2) != 1) || (heads > 1 && t.stride(1) != d)))
    unfit(std::string(name) + ": the heads of a token must be contiguous");
  return t.stride(0);
}
// Stride between the rows of [n, width] (width < 0: any) with contiguous rows.
int64_t rows_of(const Tensor& t, const char* name, at::ScalarType type, int dev, int64_t n, int64_t width) {
  on(t, name, type, dev);
  if (t.dim() != 2 || t.size(0) != n || (width >= 0 && t.size(1) != width))
    unfit(std::string(name) + " must have the shape [" + std::to_string(n) + ", " +
          (width < 0 ? "any" : std::to_string(width)) + "]");
  if (t.size(1) > 1 && t.stride(1) != 1) unfit(std::string(name) + ": rows must be contiguous");
  return t.stride(0);
}
int cache_of(const Tensor& k, const Tensor& v, int64_t kv, int64_t d, int dev) {
  if (!k.is_cuda() || !v.is_cuda() || k.get_device() != dev || v.get_device() != dev || k.dim() != 4 ||
      k.sizes() != v.sizes() || k.scalar_type() != v.scalar_type() || k.size(2) != kv || k.size(3) != d ||
      !k.is_contiguous() || !v.is_contiguous())
    unfit("the caches must be two contiguous tensors [pages, page size, " + std::to_string(kv) + ", " +
          std::to_string(d) + "] of one type on q's device");
  return dtype_of(k, "the cache");
}
uint32_t u32(int64_t v, const char* what) {
  if (v < 0 || v > UINT32_MAX) unfit(std::string(what) + " is too large");
  return (uint32_t)v;
}
void* stream_of(int dev) { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream(); }
Tensor make(at::IntArrayRef shape, at::ScalarType type, int dev) {
  return at::empty(shape, at::TensorOptions().dtype(type).device(at::Device(at::kCUDA, (c10::DeviceIndex)dev)));
}

// Autograd's record that t was written in place (as torch's own in-place operators leave it;
// inference tensors have none).
void written(const Tensor* t) {
  if (t && !t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}

// ---- errors ------------------------------------------------------------------------
struct Refused {};  // the library's own message becomes ChpeError
void check(int rc) {
  if (rc != 0) throw Refused();
}
template <typename F>
PyObject* guarded(F f) {
  try {
    return f();
  } catch (const Unfit& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
  } catch (const Misuse& e) {
    PyErr_SetString(PyExc_TypeError, e.what());
  } catch (const Refused&) {
    PyObject* pkg = PyImport_ImportModule("chpe_qwen_engine_b200");
    PyObject* type = pkg ? PyObject_GetAttrString(pkg, "ChpeError") : nullptr;
    if (type) PyErr_SetString(type, chpe_last_error(nullptr));
    Py_XDECREF(type);
    Py_XDECREF(pkg);
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}
PyObject* pair(PyObject* a, PyObject* b) {
  PyObject* t = a && b ? PyTuple_New(2) : nullptr;
  if (!t) {
    Py_XDECREF(a);
    Py_XDECREF(b);
    return nullptr;
  }
  PyTuple_SET_ITEM(t, 0, a);
  PyTuple_SET_ITEM(t, 1, b);
  return t;
}
PyObject* again(PyObject* o) {
  Py_INCREF(o);
  return o;
}
template <int N>
void intern(PyObject* (&names)[N], const char* const (&text)[N]) {
  if (!names[0])
    for (int i = 0; i < N; i++) names[i] = PyUnicode_InternFromString(text[i]);
}

// inv_freq: a CPU tensor or anything with a buffer of contiguous doubles.
struct Frequencies {
  Py_buffer view{};
  const double* data = nullptr;
  int64_t n = 0;
  bool held = false;
  explicit Frequencies(PyObject* o) {
    static const char* const what = "inv_freq must be a contiguous array of 64-bit values on the host";
    if (!o) return;
    if (THPVariable_Check(o)) {
      const Tensor& t = THPVariable_Unpack(o);
      no_gradient(t, "inv_freq");
      want(t.is_cpu() && t.scalar_type() == at::kDouble && t.dim() == 1 && t.is_contiguous(), what);
      data = static_cast<const double*>(t.data_ptr());
      n = t.size(0);
      return;
    }
    if (PyObject_GetBuffer(o, &view, PyBUF_C_CONTIGUOUS | PyBUF_FORMAT) != 0) {
      PyErr_Clear();
      unfit(what);
    }
    held = true;
    if (view.ndim != 1 || view.itemsize != 8 || !view.format || std::string(view.format) != "d") {
      PyBuffer_Release(&view);
      held = false;
      unfit(what);
    }
    data = static_cast<const double*>(view.buf);
    n = view.shape[0];
  }
  ~Frequencies() {
    if (held) PyBuffer_Release(&view);
  }
  Frequencies(const Frequencies&) = delete;
  Frequencies& operator=(const Frequencies&) = delete;
};

// ---- the operators -------------------------------------------------------------------
PyObject* qk_norm_rope(PyObject*, PyObject* const* args, Py_ssize_t n, PyObject* kw) {
  enum { Q, K, V, POS, FREQ, QW, KW, EPS, OFF, KC, VC, SLOTS, QO, KO, N };
  static const char* const text[N] = {"q", "k", "v", "positions", "inv_freq", "q_weight", "k_weight", "eps",
                                      "weight_offset", "k_cache", "v_cache", "slots", "q_out", "k_out"};
  static PyObject* names[N];
  return guarded([&]() -> PyObject* {
    intern(names, text);
    Args<N> a;
    a.parse(names, 5, args, n, kw, "qk_norm_rope");
    const Tensor& q = *a.tensor(Q, "q", true);
    const int dev = cuda_of(q, "q"), dt = dtype_of(q, "q");
    const Tensor& k = *a.tensor(K, "k", true);
    const at::ScalarType type = q.scalar_type();
    want(q.dim() == 3 && k.dim() == 3, "q and k must be [tokens, heads, head dim]");
    const int64_t T = q.size(0), H = q.size(1), D = q.size(2), KVH = k.size(1);
    const int64_t qs = heads_of(q, "q", type, dev, T, H, D), ks = heads_of(k, "k", type, dev, T, KVH, D);
    const Tensor *kc = a.tensor(KC, "k_cache"), *vc = a.tensor(VC, "v_cache"), *v = a.tensor(V, "v");
    const Tensor *slots = a.tensor(SLOTS, "slots"), *pos = a.tensor(POS, "positions");
    Tensor q_made, k_made;
    const Tensor *qo = a.tensor(QO, "q_out"), *ko = a.tensor(KO, "k_out");
    if (!qo) qo = &(q_made = make({T, H, D}, type, dev));
    if (!ko && !kc) ko = &(k_made = make({T, KVH, D}, type, dev));
    const int64_t qos = heads_of(*qo, "q_out", type, dev, T, H, D);
    const int64_t kos = ko ? heads_of(*ko, "k_out", type, dev, T, KVH, D) : 0;
    int64_t vs = 0, rows = 0;
    int ct = dt;
    want(!vc == !kc, "k_cache and v_cache go together");
    if (kc) {
      want(v && slots, "a cache needs v and slots");
      vs = heads_of(*v, "v", type, dev, T, KVH, D);
      ct = cache_of(*kc, *vc, KVH, D, dev);
      rows = kc->size(0) * kc->size(1);
    }
    const Frequencies f(a.at[FREQ]);
    want(!f.n || pos, "a rotation needs positions");
    check(chpe_qk_norm_rope(
        q.data_ptr(), k.data_ptr(), kc ? v->data_ptr() : nullptr, dt, qs, ks, vs, u32(T, "q"), u32(H, "q"),
        u32(KVH, "k"), u32(D, "q"), vec<float>(a.tensor(QW, "q_weight"), "q_weight", at::kFloat, D, dev),
        vec<float>(a.tensor(KW, "k_weight"), "k_weight", at::kFloat, D, dev), (float)a.number(OFF, "weight_offset", 0.0),
        (float)a.number(EPS, "eps", 1e-6), f.n ? vec<int32_t>(pos, "positions", at::kInt, T, dev) : nullptr, f.data,
        u32(2 * f.n, "inv_freq"), qo->data_ptr(), qos, ko ? ko->data_ptr() : nullptr, kos,
        kc ? kc->data_ptr() : nullptr, kc ? vc->data_ptr() : nullptr, ct, (uint64_t)rows,
        kc ? vec<int64_t>(slots, "slots", at::kLong, T, dev) : nullptr, stream_of(dev)));
    for (const Tensor* t : {qo, ko, kc, vc}) written(t);
    return pair(a.at[QO] ? again(a.at[QO]) : THPVariable_Wrap(q_made),
                a.at[KO] ? again(a.at[KO]) : kc ? again(Py_None) : THPVariable_Wrap(k_made));
  });
}

PyObject* attention_decode_paged(PyObject*, PyObject* const* args, Py_ssize_t n, PyObject* kw) {
  enum { Q, KC, VC, TABLE, LENS, SCALE, OUT, LSE, WS, N };
  static const char* const text[N] = {"q", "k_cache", "v_cache", "page_table", "seq_lens", "scale", "out", "lse", "workspace"};
  static PyObject* names[N];
  return guarded([&]() -> PyObject* {
    intern(names, text);
    Args<N> a;
    a.parse(names, 5, args, n, kw, "attention_decode_paged");
    const Tensor& q = *a.tensor(Q, "q", true);
    const int dev = cuda_of(q, "q"), dt = dtype_of(q, "q");
    const Tensor &kc = *a.tensor(KC, "k_cache", true), &vc = *a.tensor(VC, "v_cache", true);
    const Tensor &table = *a.tensor(TABLE, "page_table", true), &lens = *a.tensor(LENS, "seq_lens", true);
    want(q.dim() == 3, "q must be [batch, heads, head dim]");
    want(kc.dim() == 4, "the caches must be [pages, page size, kv heads, head dim]");
    const int64_t B = q.size(0), H = q.size(1), D = q.size(2), KVH = kc.size(2);
    const int ct = cache_of(kc, vc, KVH, D, dev);
    const int64_t qs = heads_of(q, "q", q.scalar_type(), dev, B, H, D);
    Tensor made, scratch;
    const Tensor *out = a.tensor(OUT, "out"), *lse = a.tensor(LSE, "lse"), *ws = a.tensor(WS, "workspace");
    if (!out) out = &(made = make({B, H, D}, q.scalar_type(), dev));
    const int64_t os = heads_of(*out, "out", q.scalar_type(), dev, B, H, D);
    const int64_t ts = rows_of(table, "page_table", at::kInt, dev, B, -1);
    if (lse) {
      on(*lse, "lse", at::kFloat, dev);
      want(lse->dim() == 2 && lse->size(0) == B && lse->size(1) == H && lse->is_contiguous(),
           "lse must be a contiguous float32 tensor [batch, heads]");
    }
    if (!ws) ws = &(scratch = make({(int64_t)chpe_attention_decode_paged_workspace((uint32_t)D)}, at::kByte, dev));
    on(*ws, "workspace", at::kByte, dev);
    want(ws->is_contiguous(), "workspace must be contiguous");
    check(chpe_attention_decode_paged(
        q.data_ptr(), dt, qs, kc.data_ptr(), vc.data_ptr(), ct, u32(kc.size(0), "the cache"), u32(kc.size(1), "the page"),
        static_cast<const int32_t*>(table.data_ptr()), ts, u32(table.size(1), "page_table"),
        vec<int32_t>(&lens, "seq_lens", at::kInt, B, dev), u32(B, "the batch"), u32(H, "q"), u32(KVH, "the cache"),
        u32(D, "q"), (float)a.number(SCALE, "scale", 1.0 / std::sqrt((double)D)), out->data_ptr(), os,
        lse ? static_cast<float*>(lse->data_ptr()) : nullptr, ws->data_ptr(), (size_t)ws->numel(), stream_of(dev)));
    written(out);
    written(lse);
    return a.at[OUT] ? again(a.at[OUT]) : THPVariable_Wrap(made);
  });
}

PyObject* logits_process(PyObject*, PyObject* const* args, Py_ssize_t n, PyObject* kw) {
  enum { X, HIST, PLEN, TLEN, REP, FREQ, PRES, IDS, VALS, MASK, OUT, ARGMAX, WANT, N };
  static const char* const text[N] = {"logits", "history", "prompt_lens", "total_lens", "repetition", "frequency", "presence",
                                      "bias_ids", "bias_values", "mask", "out", "argmax", "want_logits"};
  static PyObject* names[N];
  return guarded([&]() -> PyObject* {
    intern(names, text);
    Args<N> a;
    a.parse(names, 1, args, n, kw, "logits_process");
    const Tensor& x = *a.tensor(X, "logits", true);
    const int dev = cuda_of(x, "logits"), dt = dtype_of(x, "logits");
    want(x.dim() == 2, "logits must be [batch, vocab]");
    const int64_t B = x.size(0), V = x.size(1);
    const int64_t xs = rows_of(x, "logits", x.scalar_type(), dev, B, V);
    const int full = a.at[WANT] ? PyObject_IsTrue(a.at[WANT]) : 1;
    if (full < 0) return nullptr;
    Tensor made, best;
    const Tensor *out = a.tensor(OUT, "out"), *am = a.tensor(ARGMAX, "argmax");
    if (!out && full) out = &(made = make({B, V}, at::kFloat, dev));
    if (!am) am = &(best = make({B}, at::kInt, dev));
    const int64_t os = out ? rows_of(*out, "out", at::kFloat, dev, B, V) : 0;
    const Tensor *hist = a.tensor(HIST, "history"), *ids = a.tensor(IDS, "bias_ids"), *vals = a.tensor(VALS, "bias_values"),
                 *mask = a.tensor(MASK, "mask");
    const int64_t hs = hist ? rows_of(*hist, "history", at::kInt, dev, B, -1) : 0;
    want(!ids == !vals, "bias_ids and bias_values go together");
    int64_t bs = 0;
    if (ids) {
      bs = rows_of(*ids, "bias_ids", at::kInt, dev, B, -1);
      want(rows_of(*vals, "bias_values", at::kFloat, dev, B, ids->size(1)) == bs || B <= 1,
           "bias_ids and bias_values must have one stride");
    }
    const int64_t ms = mask ? rows_of(*mask, "mask", at::kInt, dev, B, (V + 31) / 32) : 0;
    check(chpe_logits_process(
        x.data_ptr(), dt, xs, u32(B, "the batch"), u32(V, "the vocabulary"),
        // (an empty history has no address of its own, but is one)
        !hist ? nullptr : static_cast<const int32_t*>(hist->numel() ? hist->data_ptr() : x.data_ptr()), hs,
        hist ? u32(hist->size(1), "history") : 0,
        vec<int32_t>(a.tensor(PLEN, "prompt_lens"), "prompt_lens", at::kInt, B, dev),
        vec<int32_t>(a.tensor(TLEN, "total_lens"), "total_lens", at::kInt, B, dev),
        vec<float>(a.tensor(REP, "repetition"), "repetition", at::kFloat, B, dev),
        vec<float>(a.tensor(FREQ, "frequency"), "frequency", at::kFloat, B, dev),
        vec<float>(a.tensor(PRES, "presence"), "presence", at::kFloat, B, dev),
        ids ? static_cast<const int32_t*>(ids->data_ptr()) : nullptr,
        ids ? static_cast<const float*>(vals->data_ptr()) : nullptr, bs, ids ? u32(ids->size(1), "bias_ids") : 0,
        mask ? static_cast<const uint32_t*>(mask->data_ptr()) : nullptr, ms,
        out ? static_cast<float*>(out->data_ptr()) : nullptr, os, vec<int32_t>(am, "argmax", at::kInt, B, dev),
        stream_of(dev)));
    written(out);
    written(am);
    return pair(a.at[OUT] ? again(a.at[OUT]) : out ? THPVariable_Wrap(made) : again(Py_None),
                a.at[ARGMAX] ? again(a.at[ARGMAX]) : THPVariable_Wrap(best));
  });
}

PyMethodDef kMethods[] = {
    {"qk_norm_rope", (PyCFunction)(void (*)(void))qk_norm_rope, METH_FASTCALL | METH_KEYWORDS,
     "qk_norm_rope(q, k, v, positions, inv_freq, *, q_weight=None, k_weight=None, eps=1e-6, weight_offset=0.0,\n"
     "             k_cache=None, v_cache=None, slots=None, q_out=None, k_out=None) -> (q_out, k_out)\n\n"
     "chpe_qk_norm_rope.  q [T, H, D], k and v [T, KV, D] (v may be None without a\n"
     "cache); positions [T] int32; inv_freq: 64-bit values on the host (numpy array or\n"
     "CPU tensor) or None for no rotation; slots [T] int64.  k_out is made when there\n"
     "is no cache; with one it is the tensor passed, or None."},
    {"attention_decode_paged", (PyCFunction)(void (*)(void))attention_decode_paged, METH_FASTCALL | METH_KEYWORDS,
     "attention_decode_paged(q, k_cache, v_cache, page_table, seq_lens, *, scale=None, out=None, lse=None,\n"
     "                       workspace=None) -> out\n\n"
     "chpe_attention_decode_paged.  q [B, H, D]; page_table [B, pages] int32; seq_lens\n"
     "[B] int32; scale 1/sqrt(D) unless given; lse: a float32 tensor [B, H] to fill."},
    {"logits_process", (PyCFunction)(void (*)(void))logits_process, METH_FASTCALL | METH_KEYWORDS,
     "logits_process(logits, *, history=None, prompt_lens=None, total_lens=None, repetition=None, frequency=None,\n"
     "               presence=None, bias_ids=None, bias_values=None, mask=None, out=None, argmax=None,\n"
     "               want_logits=True) -> (processed logits or None, winning tokens)\n\n"
     "chpe_logits_process.  logits [B, V]; history [B, L] int32; lengths [B] int32;\n"
     "penalties [B] float32; bias_ids [B, n] int32 with bias_values [B, n] float32;\n"
     "mask [B, ceil(V/32)] int32 words.  A bias list or mask expanded over the rows\n"
     "(stride 0) is shared.  The logits come as float32, the tokens as int32."},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_ops", "The batched decode operators on torch tensors.", -1, kMethods,
                       nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__ops(void) { return PyModule_Create(&kModule); }
