// Host side of the operators of packed batches and of layer norm: argument checks, allocation of results and the call of the kernel library's C
// entry, in one C++ call.  For a small problem the host's time is the operator's: the same in Python took 22 us for an attention's backward
// pass, 20 for a layer norm's and 9 for a rotation.
//
// The module has no kernels and no fallback; `bind` gives it the entries of the library that torchft_b200.ops._native has loaded.  Wrong
// arguments raise ValueError before anything is launched, an entry's error code goes to the `check` that `bind` was given.
#include <Python.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>

#include <cmath>
#include <cstdint>
#include <string>
#include <vector>

namespace {

using at::Tensor;
using Stream = cudaStream_t;

struct Entries {
  int (*spans)(const int*, const unsigned char*, void*, int*, void*, int*, int, int, int, int, Stream);
  int (*masked_fwd)(const void*, const void*, const void*, void*, float*, const void*, const void*, const int*, const float*, int, int, int, int, int,
                    long long, long long, long long, long long, float, float, int, int*, Stream);
  int (*masked_bwd)(const void*, const void*, const void*, const void*, const void*, const float*, void*, void*, void*, void*, const void*,
                    const void*, const int*, const float*, int, int, int, int, int, long long, long long, long long, long long, long long, long long,
                    long long, long long, float, float, int, const float*, int*, Stream);
  long long (*bwd_scratch)(int, int, int, int);
  int (*rope_axes)(void*, const int*, const double*, const int*, long long, int, int, int, long long, int, int, int, Stream);
  int (*layernorm_fwd)(const void*, const void*, void*, const void*, const void*, void*, float*, float*, long long, int, float, int, Stream);
  int (*layernorm_bwd)(const void*, const void*, const void*, const float*, const float*, const void*, void*, void*, void*, float*, long long, int,
                       int, int, int*, Stream);
  long long (*layernorm_scratch)(int);
};
Entries entries;
PyObject* check = nullptr;  // check(code, name) raises

struct Args {
  PyObject* const* a;
  Py_ssize_t n;
  Py_ssize_t at = 0;
  PyObject* next() {
    TORCH_CHECK_TYPE(at < n, "too few arguments");
    return a[at++];
  }
  const Tensor& tensor() {
    PyObject* o = next();
    TORCH_CHECK_TYPE(THPVariable_Check(o), "argument ", at, " must be a tensor");
    return with_memory(THPVariable_Unpack(o));
  }
  const Tensor* maybe() {
    PyObject* o = next();
    if (o == Py_None) return nullptr;
    TORCH_CHECK_TYPE(THPVariable_Check(o), "argument ", at, " must be a tensor or None");
    return &with_memory(THPVariable_Unpack(o));
  }
  const Tensor& with_memory(const Tensor& t) const {
    TORCH_CHECK_TYPE(!t.unsafeGetTensorImpl()->is_python_dispatch(), "argument ", at, " must be a plain tensor, not one whose operators are Python's");
    return t;
  }
  long long integer() {
    const long long v = PyLong_AsLongLong(next());
    if (v == -1 && PyErr_Occurred()) throw python_error();
    return v;
  }
  int size(const char* name) {
    const long long v = integer();
    TORCH_CHECK_VALUE(v >= 0 && v <= INT32_MAX, name, " is out of range");
    return static_cast<int>(v);
  }
  double real() {
    const double v = PyFloat_AsDouble(next());
    if (v == -1.0 && PyErr_Occurred()) throw python_error();
    return v;
  }
  bool truth() {
    const int v = PyObject_IsTrue(next());
    if (v < 0) throw python_error();
    return v != 0;
  }
};

// Calls without the interpreter's lock: an allocation or a launch may wait for the GPU, and other threads answer heartbeats meanwhile.
struct Unlocked {
  PyThreadState* state = PyEval_SaveThread();
  ~Unlocked() { PyEval_RestoreThread(state); }
  Unlocked() = default;
  Unlocked(const Unlocked&) = delete;
};

// On a device that has been checked: straight from the allocator (at::empty's way there takes as long again).
Tensor empty(at::IntArrayRef shape, at::ScalarType type, at::Device device) {
  Unlocked unlocked;
  return Tensor(at::detail::empty_cuda(shape, type, device, std::nullopt));
}

template <typename F, typename... A>
void launch(const char* name, F entry, A... args) {
  int rc;
  {
    Unlocked unlocked;
    rc = entry(args...);
  }
  if (rc == 0) return;
  PyObject* r = PyObject_CallFunction(check, "is", rc, name);
  Py_XDECREF(r);
  if (r == nullptr) throw python_error();
}

// The tensors' device (`t` is one of them) is the current one, on whose stream the kernel is launched.
Stream here(const Tensor& t) {
  TORCH_CHECK_VALUE(t.is_cuda(), "the tensors must be on a GPU");
  TORCH_CHECK_VALUE(t.get_device() == c10::cuda::current_device(), "the tensors are on ", t.device(), ", which is not the current device");
  return c10::cuda::getCurrentCUDAStream(t.get_device()).stream();
}

// Contiguous, of the type and shape, and on the device.
void like(const Tensor* t, const char* name, at::ScalarType type, at::IntArrayRef shape, at::Device device) {
  if (t == nullptr) return;
  TORCH_CHECK_VALUE(t->scalar_type() == type && t->sizes() == shape && t->device() == device && t->is_contiguous(), name, " must be contiguous ", type,
                    " of shape ", shape, " on ", device, ", got ", t->scalar_type(), " of ", t->sizes(), " on ", t->device());
}

// Of contiguous tensors: whether they share memory.
bool overlap(const Tensor* a, const Tensor* b) {
  if (a == nullptr || b == nullptr || a->numel() == 0 || b->numel() == 0) return false;
  const auto from = [](const Tensor* t) { return reinterpret_cast<uintptr_t>(t->data_ptr()); };
  return from(a) < from(b) + b->nbytes() && from(b) < from(a) + a->nbytes();
}

struct Named {
  const Tensor* t;
  const char* name;
};

// A result is no part of what is read at other times than it is written, and of no other result.  `place`: what it may be written over, as a whole.
void result_apart(Named r, std::initializer_list<Named> place, std::initializer_list<Named> others) {
  if (r.t == nullptr) return;
  for (const Named& o : place)
    TORCH_CHECK_VALUE(!overlap(r.t, o.t) || r.t->data_ptr() == o.t->data_ptr(), r.name, " may be ", o.name, " as a whole, but no part of its memory");
  for (const Named& o : others) TORCH_CHECK_VALUE(!overlap(r.t, o.t), r.name, " and ", o.name, " share memory");
}

void* at_of(const Tensor* t) { return t == nullptr ? nullptr : t->data_ptr(); }

// ------------------------------------------------------------------ spans

// Where the parts of a span buffer begin, in 32-bit words: rows, tiles, positions, padded, end.
struct SpanParts {
  long long tiles, positions, padded, end;
  SpanParts(long long batch, long long seq) {
    tiles = 4 * batch * seq;
    positions = tiles + 8 * batch * ((seq + 127) / 128);
    padded = positions + batch * seq;
    end = padded + batch * ((seq + 1023) / 1024);
  }
};

// (documents, prefix or None, causal, window) -> the span buffer
PyObject* attention_spans(PyObject*, PyObject* const* argv, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a{argv, n};
  const Tensor& documents = a.tensor();
  const Tensor* prefix = a.maybe();
  const bool causal = a.truth();
  const long long window = a.integer();
  TORCH_CHECK_VALUE(documents.dim() == 2 && documents.scalar_type() == at::kInt && documents.is_contiguous(),
                    "documents must be contiguous int32 [batch, seq]");
  if (prefix != nullptr) {
    TORCH_CHECK_VALUE(prefix->scalar_type() == at::kBool || prefix->scalar_type() == at::kByte, "prefix must be bool or uint8");
    like(prefix, "prefix", prefix->scalar_type(), documents.sizes(), documents.device());
  }
  TORCH_CHECK_VALUE(window >= 0 && window <= INT32_MAX, "window must be 0 or a number of keys");
  TORCH_CHECK_VALUE(causal || (window == 0 && prefix == nullptr), "a window or a prefix goes with a causal mask");
  const Stream stream = here(documents);
  const long long B = documents.size(0), S = documents.size(1);
  const SpanParts parts(B, S);
  Tensor buf = empty({parts.end}, at::kInt, documents.device());
  if (B > 0 && S > 0) {
    TORCH_CHECK_VALUE(B <= INT32_MAX && S <= INT32_MAX, "too many documents");
    int* base = buf.data_ptr<int>();
    launch("attention_spans", entries.spans, documents.data_ptr<int>(), static_cast<const unsigned char*>(at_of(prefix)), base,
           base + parts.positions, base + parts.tiles, base + parts.padded, static_cast<int>(B), static_cast<int>(S), causal,
           static_cast<int>(window), stream);
  }
  return THPVariable_Wrap(std::move(buf));
  END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------------------ attention

struct Mask {
  const Tensor *spans, *slopes;
  int batch, seq, heads, kv_heads, dim;
  float cap;
  bool causal;
  const int *rows = nullptr, *tiles = nullptr, *padded = nullptr;

  explicit Mask(Args& a) {
    spans = a.maybe();
    slopes = a.maybe();
    batch = a.size("batch");
    seq = a.size("seq_len");
    heads = a.size("n_heads");
    kv_heads = a.size("n_kv_heads");
    dim = a.size("head_dim");
    const double c = a.real();
    causal = a.truth();
    TORCH_CHECK_VALUE((dim == 64 || dim == 128) && heads > 0 && kv_heads > 0 && heads % kv_heads == 0,
                      "masked attention takes head dims 64 and 128 and groups of equally many query heads");
    cap = static_cast<float>(c);
    TORCH_CHECK_VALUE(c == 0.0 || (cap >= 1e-9f && cap <= 1e30f), "softcap must be 0 or a cap from 1e-9 to 1e30");
  }
  // a [batch * seq, n * dim] view of bf16
  void view(const Tensor& t, const char* name, int n, at::Device device) const {
    TORCH_CHECK_VALUE(t.dim() == 2 && t.size(0) == static_cast<long long>(batch) * seq && t.size(1) == static_cast<long long>(n) * dim &&
                          t.scalar_type() == at::kBFloat16 && t.stride(1) == 1 && t.device() == device &&
                          (t.size(0) <= 1 || t.stride(0) >= t.size(1)),
                      name, " must be bf16 [", static_cast<long long>(batch) * seq, ", ", n * dim, "] with unit inner stride, its rows apart, on ", device,
                      ", got ", t.scalar_type(), " of ", t.sizes(), ", strides ", t.strides(), ", on ", t.device());
  }
  // Between rows; of one there is none.
  static long long ld(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }
  void rest(const Tensor* lse, at::Device device) {
    like(slopes, "slopes", at::kFloat, {heads}, device);
    like(lse, "lse", at::kFloat, {batch, heads, seq}, device);
    if (spans != nullptr) {
      const SpanParts parts(batch, seq);
      like(spans, "spans", at::kInt, {parts.end}, device);
      rows = spans->data_ptr<int>();
      tiles = rows + parts.tiles;
      padded = rows + parts.padded;
    }
  }
  const float* slopes_at() const { return static_cast<const float*>(at_of(slopes)); }
  float scale() const { return static_cast<float>(1.0 / std::sqrt(static_cast<double>(dim))); }
};

// (q, k, v, out, lse or None, spans or None, slopes or None, batch, seq, heads, kv_heads, dim, softcap, causal, status word's address) -> the
// number of kernels launched
PyObject* attention_masked_fwd(PyObject*, PyObject* const* argv, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a{argv, n};
  const Tensor &q = a.tensor(), &k = a.tensor(), &v = a.tensor(), &out = a.tensor();
  const Tensor* lse = a.maybe();
  Mask m(a);
  int* status = reinterpret_cast<int*>(a.integer());
  const at::Device device = q.device();
  m.view(q, "q", m.heads, device);
  m.view(k, "k", m.kv_heads, device);
  m.view(v, "v", m.kv_heads, device);
  m.view(out, "out", m.heads, device);
  m.rest(lse, device);
  const Stream stream = here(q);
  if (m.batch == 0 || m.seq == 0) return PyLong_FromLong(0);
  launch("attention_masked_fwd", entries.masked_fwd, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), static_cast<float*>(at_of(lse)),
         m.rows, m.tiles, m.padded, m.slopes_at(), m.batch, m.seq, m.heads, m.kv_heads, m.dim, m.ld(q), m.ld(k), m.ld(v), m.ld(out),
         m.scale(), m.cap, m.causal, status, stream);
  return PyLong_FromLong(1);
  END_HANDLE_TH_ERRORS
}

// (q, k, v, o, d_o, lse, dq, dk, dv, scratch or None, rope or None, spans or None, ..., causal, status word's address) as above
PyObject* attention_masked_bwd(PyObject*, PyObject* const* argv, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a{argv, n};
  const Tensor &q = a.tensor(), &k = a.tensor(), &v = a.tensor(), &o = a.tensor(), &d_o = a.tensor(), &lse = a.tensor(), &dq = a.tensor(),
               &dk = a.tensor(), &dv = a.tensor();
  const Tensor *scratch = a.maybe(), *rope = a.maybe();
  Mask m(a);
  int* status = reinterpret_cast<int*>(a.integer());
  const at::Device device = q.device();
  m.view(q, "q", m.heads, device);
  m.view(k, "k", m.kv_heads, device);
  m.view(v, "v", m.kv_heads, device);
  m.view(o, "o", m.heads, device);
  m.view(d_o, "d_o", m.heads, device);
  m.view(dq, "dq", m.heads, device);
  m.view(dk, "dk", m.kv_heads, device);
  m.view(dv, "dv", m.kv_heads, device);
  m.rest(&lse, device);
  if (rope != nullptr)
    TORCH_CHECK_VALUE(rope->scalar_type() == at::kFloat && rope->is_contiguous() && rope->device() == device && rope->dim() == 3 &&
                          rope->size(0) >= m.seq && rope->size(1) == m.dim / 2 && rope->size(2) == 2,
                      "rope must be the table of the sequence and head dim on the device of q");
  const Stream stream = here(q);
  if (m.batch == 0 || m.seq == 0) return PyLong_FromLong(0);
  const long long need = entries.bwd_scratch(m.batch, m.seq, m.heads, m.kv_heads);
  Tensor own;
  if (scratch == nullptr) {
    own = empty({need}, at::kByte, device);
    scratch = &own;
  }
  TORCH_CHECK_VALUE(scratch->device() == device && scratch->scalar_type() == at::kByte && scratch->numel() >= need && scratch->is_contiguous(),
                    "scratch must be ", need, " contiguous bytes on ", device);
  launch("attention_masked_bwd", entries.masked_bwd, q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), d_o.data_ptr(), lse.data_ptr<float>(),
         dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), scratch->data_ptr(), m.rows, m.tiles, m.padded, m.slopes_at(), m.batch, m.seq, m.heads,
         m.kv_heads, m.dim, m.ld(q), m.ld(k), m.ld(v), m.ld(o), m.ld(d_o), m.ld(dq), m.ld(dk), m.ld(dv), m.scale(),
         m.cap, m.causal, static_cast<const float*>(at_of(rope)), status, stream);
  return PyLong_FromLong(3);
  END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------------------ rotation

// (buf, positions, inv_freq, axis, n_heads, head_dim, half, backward) -> the number of kernels launched
PyObject* rope_axes(PyObject*, PyObject* const* argv, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a{argv, n};
  const Tensor &buf = a.tensor(), &positions = a.tensor(), &inv_freq = a.tensor(), &axis = a.tensor();
  const int heads = a.size("n_heads"), dim = a.size("head_dim");
  const bool half = a.truth(), backward = a.truth();
  const at::ScalarType type = buf.scalar_type();
  TORCH_CHECK_VALUE(buf.dim() == 2 && (type == at::kBFloat16 || type == at::kFloat) && (buf.size(1) <= 1 || buf.stride(1) == 1),
                    "buf must be a 2-D bf16 or fp32 tensor with unit inner stride");
  const long long T = buf.size(0), width = buf.size(1);
  const int vector = type == at::kFloat ? 4 : 8;
  TORCH_CHECK_VALUE(dim > 0 && dim % (half ? 2 * vector : vector) == 0 && dim <= 1024, "head_dim must be a multiple of ", half ? 2 * vector : vector,
                    " up to 1024 in ", type, half ? ", half-split" : "");
  const long long ld = T > 1 ? buf.stride(0) : static_cast<long long>(heads) * dim;  // of one row there is none
  TORCH_CHECK_VALUE(heads >= 1 && heads <= 1 << 20 && width >= static_cast<long long>(heads) * dim && ld >= static_cast<long long>(heads) * dim,
                    "buf of shape ", buf.sizes(), " does not hold ", heads, " heads of ", dim);
  TORCH_CHECK_VALUE(ld % vector == 0, "the rows of buf must start a multiple of ", vector, " elements apart");
  TORCH_CHECK_VALUE(positions.dim() == 2 && positions.size(0) >= 1 && positions.size(0) <= INT32_MAX, "positions must be contiguous int32 [axes, rows]");
  const at::Device device = buf.device();
  like(&positions, "positions", at::kInt, {positions.size(0), T}, device);
  like(&inv_freq, "inv_freq", at::kDouble, {dim / 2}, device);
  like(&axis, "axis", at::kInt, {dim / 2}, device);
  const Stream stream = here(buf);
  if (T > 0)
    launch("rope_axes", entries.rope_axes, buf.data_ptr(), positions.data_ptr<int>(), inv_freq.data_ptr<double>(), axis.data_ptr<int>(), T,
           static_cast<int>(positions.size(0)), heads, dim, ld, type == at::kFloat, half, backward, stream);
  return PyLong_FromLong(T > 0);
  END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------------------ layer norm

void norm_rows(const Tensor& x) {
  TORCH_CHECK_VALUE(x.dim() == 2 && (x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kFloat) && x.size(1) % 8 == 0 && x.size(1) > 0 &&
                        x.size(1) <= 16384,
                    "x must be [rows, width] in bf16 or fp32 with a width that is a multiple of 8 up to 16384");
}

PyObject* pack(std::initializer_list<Tensor> ts) {
  PyObject* r = PyTuple_New(static_cast<Py_ssize_t>(ts.size()));
  if (r == nullptr) throw python_error();
  Py_ssize_t i = 0;
  for (const Tensor& t : ts) {
    if (t.defined()) {
      PyTuple_SET_ITEM(r, i++, THPVariable_Wrap(t));
    } else {
      Py_INCREF(Py_None);
      PyTuple_SET_ITEM(r, i++, Py_None);
    }
  }
  return r;
}

// The caller's result or a new one.
Tensor result(const Tensor* given, at::IntArrayRef shape, at::ScalarType type, at::Device device) {
  return given != nullptr ? *given : empty(shape, type, device);
}

// (x, w, b or None, eps, then res, h_out, out, mean, rstd or None each) -> (out, mean, rstd, h or None)
PyObject* layernorm_fwd(PyObject*, PyObject* const* argv, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a{argv, n};
  const Tensor &x = a.tensor(), &w = a.tensor();
  const Tensor* b = a.maybe();
  const double eps = a.real();
  const Tensor *res = a.maybe(), *h_given = a.maybe(), *out_given = a.maybe(), *mean_given = a.maybe(), *rstd_given = a.maybe();
  norm_rows(x);
  const at::Device device = x.device();
  const at::ScalarType type = x.scalar_type();
  const long long T = x.size(0), D = x.size(1);
  like(&x, "x", type, {T, D}, device);
  like(res, "res", type, {T, D}, device);
  like(h_given, "h_out", type, {T, D}, device);
  like(out_given, "out", type, {T, D}, device);
  like(&w, "w", type, {D}, device);
  like(b, "b", type, {D}, device);
  like(mean_given, "mean", at::kFloat, {T}, device);
  like(rstd_given, "rstd", at::kFloat, {T}, device);
  if (res == nullptr) h_given = nullptr;
  result_apart({out_given, "out"}, {{&x, "x"}, {res, "res"}}, {{h_given, "h_out"}, {&w, "w"}, {b, "b"}, {mean_given, "mean"}, {rstd_given, "rstd"}});
  result_apart({h_given, "h_out"}, {{&x, "x"}, {res, "res"}}, {{&w, "w"}, {b, "b"}, {mean_given, "mean"}, {rstd_given, "rstd"}});
  result_apart({mean_given, "mean"}, {}, {{&x, "x"}, {res, "res"}, {&w, "w"}, {b, "b"}, {rstd_given, "rstd"}});
  result_apart({rstd_given, "rstd"}, {}, {{&x, "x"}, {res, "res"}, {&w, "w"}, {b, "b"}});
  const Stream stream = here(x);
  Tensor out = result(out_given, {T, D}, type, device);
  Tensor mean = result(mean_given, {T}, at::kFloat, device), rstd = result(rstd_given, {T}, at::kFloat, device);
  Tensor h = res != nullptr ? result(h_given, {T, D}, type, device) : overlap(&out, &x) ? Tensor() : x;  // not where out took its place
  if (T > 0)
    launch("layernorm_fwd", entries.layernorm_fwd, x.data_ptr(), at_of(res), res == nullptr ? nullptr : h.data_ptr(), w.data_ptr(), at_of(b),
           out.data_ptr(), mean.data_ptr<float>(), rstd.data_ptr<float>(), T, static_cast<int>(D), static_cast<float>(eps), type == at::kFloat,
           stream);
  return pack({out, mean, rstd, h});
  END_HANDLE_TH_ERRORS
}

// (dy, x, w, mean, rstd, then dres, dx, dw, db or None each, bias, accumulate, scratch or None, status word's address) -> (dx, dw, db)
PyObject* layernorm_bwd(PyObject*, PyObject* const* argv, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a{argv, n};
  const Tensor &dy = a.tensor(), &x = a.tensor(), &w = a.tensor(), &mean = a.tensor(), &rstd = a.tensor();
  const Tensor *dres = a.maybe(), *dx_given = a.maybe(), *dw_given = a.maybe(), *db_given = a.maybe();
  const bool bias = a.truth(), accumulate = a.truth();
  const Tensor* scratch = a.maybe();
  int* status = reinterpret_cast<int*>(a.integer());
  norm_rows(x);
  TORCH_CHECK_VALUE(!accumulate || (dw_given != nullptr && (!bias || db_given != nullptr)), "accumulate needs dw and db");
  const at::Device device = x.device();
  const at::ScalarType type = x.scalar_type();
  const long long T = x.size(0), D = x.size(1);
  like(&x, "x", type, {T, D}, device);
  like(&dy, "dy", type, {T, D}, device);
  like(dres, "dres", type, {T, D}, device);
  like(dx_given, "dx", type, {T, D}, device);
  like(&w, "w", type, {D}, device);
  like(dw_given, "dw", type, {D}, device);
  if (bias) like(db_given, "db", type, {D}, device);
  like(&mean, "mean", at::kFloat, {T}, device);
  like(&rstd, "rstd", at::kFloat, {T}, device);
  if (!bias) db_given = nullptr;
  result_apart({dx_given, "dx"}, {{&dy, "dy"}, {&x, "x"}, {dres, "dres"}}, {{&w, "w"}, {&mean, "mean"}, {&rstd, "rstd"}, {dw_given, "dw"}, {db_given, "db"}});
  for (const Named& sums : {Named{dw_given, "dw"}, Named{db_given, "db"}})
    result_apart(sums, {}, {{&dy, "dy"}, {&x, "x"}, {dres, "dres"}, {&w, "w"}, {&mean, "mean"}, {&rstd, "rstd"}});
  result_apart({dw_given, "dw"}, {}, {{db_given, "db"}});
  const Stream stream = here(x);
  Tensor dx = result(dx_given, {T, D}, type, device), dw = result(dw_given, {D}, type, device), db;
  if (bias) db = result(db_given, {D}, type, device);
  if (T == 0) {
    if (!accumulate) {
      dw.zero_();
      if (bias) db.zero_();
    }
    return pack({dx, dw, db});
  }
  const long long need = entries.layernorm_scratch(static_cast<int>(D));
  Tensor own;
  if (scratch == nullptr) {
    own = empty({need}, at::kFloat, device);
    scratch = &own;
  }
  TORCH_CHECK_VALUE(scratch->device() == device && scratch->scalar_type() == at::kFloat && scratch->is_contiguous() && scratch->numel() >= need &&
                        reinterpret_cast<uintptr_t>(scratch->data_ptr()) % 16 == 0,
                    "scratch must be ", need, " contiguous fp32 on ", device);
  result_apart({scratch, "scratch"}, {}, {{&dy, "dy"}, {&x, "x"}, {dres, "dres"}, {&w, "w"}, {&mean, "mean"}, {&rstd, "rstd"}, {&dx, "dx"}, {&dw, "dw"},
                                          {bias ? &db : nullptr, "db"}});
  launch("layernorm_bwd", entries.layernorm_bwd, dy.data_ptr(), x.data_ptr(), w.data_ptr(), mean.data_ptr<float>(), rstd.data_ptr<float>(),
         at_of(dres), dx.data_ptr(), dw.data_ptr(), bias ? db.data_ptr() : nullptr, scratch->data_ptr<float>(), T,
         static_cast<int>(D), accumulate, type == at::kFloat, status, stream);
  return pack({dx, dw, db});
  END_HANDLE_TH_ERRORS
}

// (check, addresses of the entries in the order of Entries)
PyObject* bind(PyObject*, PyObject* const* argv, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a{argv, n};
  PyObject* c = a.next();
  std::vector<void*> at;
  while (a.at < a.n) at.push_back(reinterpret_cast<void*>(a.integer()));
  TORCH_CHECK_VALUE(at.size() == sizeof(Entries) / sizeof(void*), "bind takes the address of every entry");
  for (size_t i = 0; i < at.size(); ++i) reinterpret_cast<void**>(&entries)[i] = at[i];
  Py_INCREF(c);
  Py_XDECREF(check);
  check = c;
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

#define FTB200_METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FTB200_METHOD(bind),
                         FTB200_METHOD(attention_spans),
                         FTB200_METHOD(attention_masked_fwd),
                         FTB200_METHOD(attention_masked_bwd),
                         FTB200_METHOD(rope_axes),
                         FTB200_METHOD(layernorm_fwd),
                         FTB200_METHOD(layernorm_bwd),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_ops_host", "Host side of the packed-batch operators.", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__ops_host() { return PyModule_Create(&module); }
