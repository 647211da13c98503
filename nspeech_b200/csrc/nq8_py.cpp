// nq8_py.cpp -- the decoding operators' argument checks and calls for Python.
//
// A decoder's step is many small calls; read through Python attributes and
// ctypes, a call's tensors cost more time than its kernels (10 to 45 us a
// call).  This module does the same on the tensors themselves: it checks them,
// allocates outputs and workspaces with torch's allocator, and calls the C ABI
// (include/nq8.h) on the current stream of the tensors' device.  The public
// functions are those of attention.py, cache.py and beam.py.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <string>
#include <vector>

#include "../../include/nq8.h"
#include "nq8_overlap.h"

namespace {

PyObject *g_misfit = nullptr;  // fast_matmul.MatMulError(message)
PyObject *g_failed = nullptr;  // lib.NqError(code, message)
uint64_t g_ready = 0;          // devices that nq_init has seen

struct Failed {};  // a Python error is set

[[noreturn]] void misfit(const std::string &msg) {
  PyErr_SetString(g_misfit, msg.c_str());
  throw Failed();
}
void check(int64_t rc) {
  if (rc >= 0) return;
  char buf[512];
  nq_last_error(buf, sizeof(buf));
  PyObject *e = PyObject_CallFunction(g_failed, "is", static_cast<int>(rc), buf);
  if (e) {
    PyErr_SetObject(g_failed, e);
    Py_DECREF(e);
  }
  throw Failed();
}

struct Ref {  // owned reference
  PyObject *p;
  ~Ref() { Py_XDECREF(p); }
};

std::string text(at::IntArrayRef s) {
  std::string r = "(";
  for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
  return r + ")";
}
std::string where(int dev) { return "cuda:" + std::to_string(dev); }

// A tensor whose memory is what it stands for; the operators have no gradients.
const at::Tensor &tensor(PyObject *o, const char *name) {
  if (!THPVariable_Check(o)) misfit(std::string(name) + " must be a tensor");
  const at::Tensor &t = THPVariable_Unpack(o);
  if (t.is_neg() || t.is_conj()) misfit(std::string(name) + " is a negated or conjugated view (resolve_neg, resolve_conj)");
  if (t.requires_grad() && c10::GradMode::is_enabled())
    misfit(std::string(name) + " requires a gradient, which this operator does not have (torch.no_grad, detach)");
  return t;
}
// A given output is written: autograd's saved uses of it are out of date.
void written(const at::Tensor &t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
int64_t integer(PyObject *o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Failed();
  return v;
}
int small(PyObject *o, const char *name) {
  const int64_t v = integer(o);
  if (v > INT32_MAX || v < INT32_MIN) misfit(std::string(name) + " is out of range");
  return static_cast<int>(v);
}
int code_of(const at::Tensor &t, const char *name) {
  const auto d = t.scalar_type();
  if (d == at::kFloat) return NQ_F32;
  if (d == at::kBFloat16) return NQ_BF16;
  misfit(std::string(name) + " has dtype " + c10::toString(d) + " (f32 or bf16)");
}

// The device of a call as the current one, made ready by nq_init.
class Device {
 public:
  Device(const at::Tensor &t, const char *name) {
    if (!t.is_cuda()) misfit(std::string(name) + " must live on a CUDA device");
    enter(t.get_device());
  }
  explicit Device(int index) { enter(index); }
  ~Device() {
    if (was != index) c10::cuda::set_device(static_cast<c10::DeviceIndex>(was));
  }
  int index, was;
  void *stream() const { return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(index)).stream(); }
  c10::Device device() const { return {c10::kCUDA, static_cast<c10::DeviceIndex>(index)}; }

 private:
  void enter(int i) {
    index = i;
    was = c10::cuda::current_device();
    if (was != index) c10::cuda::set_device(static_cast<c10::DeviceIndex>(index));
    if (index < 64 && !(g_ready >> index & 1)) {
      // nq_init allocates: allowed while this thread captures another stream
      cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
      cudaThreadExchangeStreamCaptureMode(&mode);
      const int rc = nq_init(index);
      cudaThreadExchangeStreamCaptureMode(&mode);
      if (rc < 0 && was != index) c10::cuda::set_device(static_cast<c10::DeviceIndex>(was));  // no object, no destructor
      check(rc);
      g_ready |= uint64_t{1} << index;
    }
  }
};

at::Tensor empty(at::IntArrayRef size, at::ScalarType type, const Device &dev) {
  return at::detail::empty_cuda(size, type, dev.device(), std::nullopt);
}

nq_rows rows_of(const at::Tensor &t, const char *name, at::ScalarType type, int dev) {
  if (t.dim() != 3 || t.scalar_type() != type || !t.is_cuda() || t.get_device() != dev ||
      (t.stride(2) != 1 && t.size(2) > 1 && t.numel() > 0))
    misfit(std::string(name) + " must be [rows, heads, head_dim] of " + c10::toString(type) + " on " + where(dev) + " with unit last stride");
  return nq_rows{t.data_ptr(), t.stride(0), t.stride(1)};
}
// Contiguous int32 [n] (n < 0: any length), or None.
const int32_t *ints(PyObject *o, const char *name, int64_t n, int dev) {
  if (o == Py_None) return nullptr;
  const at::Tensor &t = tensor(o, name);
  if (t.scalar_type() != at::kInt || t.dim() != 1 || !t.is_cuda() || t.get_device() != dev || !t.is_contiguous() ||
      (n >= 0 && t.numel() != n))
    misfit(std::string(name) + " must be contiguous int32" + (n >= 0 ? " [" + std::to_string(n) + "]" : "") + " on " + where(dev));
  return static_cast<const int32_t *>(t.data_ptr());
}
float scale_of(PyObject *o, int64_t dim) {
  if (o == Py_None) return static_cast<float>(1.0 / std::sqrt(static_cast<double>(dim)));
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Failed();
  return static_cast<float>(v);
}
// An output that shares memory with itself or with `other` (which it may be,
// where `same`) as far as torch can say.
void apart(const at::Tensor &out, const at::Tensor &other, bool same, const std::string &what) {
  if (at::has_internal_overlap(out) == at::MemOverlap::Yes) misfit("an output overlaps itself");
  const auto how = at::get_overlap_status(out, other);
  if (how == at::MemOverlapStatus::Partial || (how == at::MemOverlapStatus::Full && !same)) misfit("an output overlaps " + what);
}
// out, if given.
void check_output(PyObject *o, const at::Tensor &q, const at::Tensor *k, const at::Tensor *v) {
  if (o == Py_None) return;
  const at::Tensor &out = tensor(o, "out");
  apart(out, q, true, "q");
  if (k) apart(out, *k, false, "k");
  if (v) apart(out, *v, false, "v");
}
at::Tensor output(PyObject *o, const at::Tensor &q, const Device &dev) {
  if (o == Py_None) return empty(q.sizes(), q.scalar_type(), dev);
  const at::Tensor &out = THPVariable_Unpack(o);
  if (out.sizes() != q.sizes()) misfit("out has shape " + text(out.sizes()) + ", q " + text(q.sizes()));
  return out;
}

// q, k, v, left, right, sinks, scale, q_offsets, k_offsets, q_lens, k_lens, seqs, out
PyObject *window_attention(PyObject *const *a) {
  const at::Tensor &q = tensor(a[0], "q"), &k = tensor(a[1], "k"), &v = tensor(a[2], "v");
  if (q.dim() != 3 || k.dim() != 3) misfit("q, k and v must be [rows, heads, head_dim]");
  if (v.sizes() != k.sizes() || k.size(2) != q.size(2) || k.size(1) == 0 || q.size(1) % k.size(1))
    misfit("q " + text(q.sizes()) + ", k " + text(k.sizes()) + " and v " + text(v.sizes()) + " do not fit together");
  const int code = code_of(q, "q");
  check_output(a[12], q, &k, &v);
  const Device dev(q, "q");
  int64_t seqs = 1;
  if (a[11] != Py_None)
    seqs = integer(a[11]);
  else
    for (int i = 7; i < 11; ++i)
      if (a[i] != Py_None) {
        seqs = tensor(a[i], "offsets").numel() - (i < 9);
        break;
      }
  if (seqs < 0 || seqs > (1 << 24)) misfit("no such number of sequences");
  const at::Tensor out = output(a[12], q, dev);
  const auto type = q.scalar_type();
  const nq_rows r[4] = {rows_of(q, "q", type, dev.index), rows_of(k, "k", type, dev.index), rows_of(v, "v", type, dev.index),
                        rows_of(out, "out", type, dev.index)};
  const int32_t *qo = ints(a[7], "q_offsets", seqs + 1, dev.index), *ko = ints(a[8], "k_offsets", seqs + 1, dev.index),
                *ql = ints(a[9], "q_lens", seqs, dev.index), *kl = ints(a[10], "k_lens", seqs, dev.index);
  const int left = small(a[3], "left"), right = small(a[4], "right"), sinks = small(a[5], "sinks");
  const int hq = static_cast<int>(q.size(1)), hk = static_cast<int>(k.size(1)), d = static_cast<int>(q.size(2)), n = static_cast<int>(seqs);
  const int64_t need = nq_window_attention_workspace(code, n, q.size(0), k.size(0), hq, hk, d, left, right, sinks);
  check(need);
  at::Tensor ws;
  if (need) ws = empty({need}, at::kByte, dev);
  check(nq_window_attention(r, r + 1, r + 2, r + 3, code, n, q.size(0), k.size(0), qo, ko, ql, kl, hq, hk, d, left, right, sinks,
                            scale_of(a[6], d), need ? ws.data_ptr() : nullptr, need, dev.stream()));
  if (a[12] == Py_None) return THPVariable_Wrap(out);
  written(out);
  return Py_INCREF(a[12]), a[12];
}

const nq_cache *cache_of(PyObject *o) { return reinterpret_cast<const nq_cache *>(integer(o)); }
at::ScalarType type_of(const nq_cache *c) { return c->dtype == NQ_F32 ? at::kFloat : at::kBFloat16; }

// cache, device, q, layer, offsets, first, n, left, right, sinks, scale, out
PyObject *cache_attention(PyObject *const *a) {
  const nq_cache *c = cache_of(a[0]);
  const Device dev(small(a[1], "device"));
  const at::Tensor &q = tensor(a[2], "q");
  if (q.dim() != 3 || q.size(2) != c->head_dim || q.size(1) % c->kv_heads)
    misfit("q must be [rows, a multiple of " + std::to_string(c->kv_heads) + " heads, " + std::to_string(c->head_dim) + "]");
  check_output(a[11], q, nullptr, nullptr);
  const int first = small(a[5], "first");
  const int n = a[6] != Py_None ? small(a[6], "n") : a[4] != Py_None ? static_cast<int>(tensor(a[4], "offsets").numel()) - 1 : c->slots - first;
  const nq_rows rq = rows_of(q, "q", type_of(c), dev.index);
  const at::Tensor out = output(a[11], q, dev);
  const nq_rows ro = rows_of(out, "out", type_of(c), dev.index);
  const int32_t *off = ints(a[4], "offsets", static_cast<int64_t>(n) + 1, dev.index);
  const int left = small(a[7], "left"), right = small(a[8], "right"), sinks = small(a[9], "sinks"), hq = static_cast<int>(q.size(1));
  const int64_t need = nq_cache_attention_workspace(c, n, q.size(0), hq, left, right, sinks);
  check(need);
  at::Tensor ws;
  if (need) ws = empty({need}, at::kByte, dev);
  check(nq_cache_attention(c, small(a[3], "layer"), &rq, &ro, first, n, q.size(0), off, hq, left, right, sinks,
                           scale_of(a[10], q.size(2)), need ? ws.data_ptr() : nullptr, need, dev.stream()));
  if (a[11] == Py_None) return THPVariable_Wrap(out);
  written(out);
  return Py_INCREF(a[11]), a[11];
}

// New tokens of a range of slots: offsets, or the same number each.
struct Range {
  const int32_t *offsets = nullptr;
  int tokens = 0, first, n;
  Range(const nq_cache *c, PyObject *new_tokens, PyObject *f, PyObject *count, int dev) {
    first = small(f, "first");
    if (THPVariable_Check(new_tokens)) {
      n = count == Py_None ? static_cast<int>(THPVariable_Unpack(new_tokens).numel()) - 1 : small(count, "n");
      offsets = ints(new_tokens, "offsets", static_cast<int64_t>(n) + 1, dev);
    } else {
      tokens = small(new_tokens, "tokens");
      n = count == Py_None ? c->slots - first : small(count, "n");
    }
  }
};

// cache, device, tokens, first, n
PyObject *cache_reserve(PyObject *const *a) {
  const nq_cache *c = cache_of(a[0]);
  const Device dev(small(a[1], "device"));
  const Range r(c, a[2], a[3], a[4], dev.index);
  check(nq_cache_reserve(c, r.first, r.n, r.offsets, r.tokens, dev.stream()));
  Py_RETURN_NONE;
}

// cache, device, k, v, tokens, first, n, layer
PyObject *cache_write(PyObject *const *a) {
  const nq_cache *c = cache_of(a[0]);
  const Device dev(small(a[1], "device"));
  const at::Tensor &k = tensor(a[2], "k"), &v = tensor(a[3], "v");
  const Range r(c, a[4], a[5], a[6], dev.index);
  const int64_t d = k.dim();
  if (k.sizes() != v.sizes() || (d != 3 && d != 4) || k.size(d - 2) != c->kv_heads || k.size(d - 1) != c->head_dim)
    misfit("k and v must be [(layers,) rows, " + std::to_string(c->kv_heads) + ", " + std::to_string(c->head_dim) + "]");
  const int64_t layers = d == 4 ? k.size(0) : 1;
  nq_rows side[2];
  int64_t by[2] = {0, 0};
  const at::Tensor *t[2] = {&k, &v};
  for (int i = 0; i < 2; ++i) {
    if (t[i]->scalar_type() != type_of(c) || !t[i]->is_cuda() || t[i]->get_device() != dev.index ||
        (t[i]->stride(d - 1) != 1 && c->head_dim > 1 && t[i]->numel() > 0))
      misfit(std::string(i ? "v" : "k") + " must be " + c10::toString(type_of(c)) + " on " + where(dev.index) + " with unit last stride");
    side[i] = nq_rows{t[i]->data_ptr(), t[i]->stride(d - 3), t[i]->stride(d - 2)};
    if (d == 4) by[i] = t[i]->stride(0);
  }
  check(nq_cache_write(c, side, side + 1, by[0], by[1], small(a[7], "layer"), static_cast<int>(layers), k.size(d - 3), r.first, r.n,
                       r.offsets, r.tokens, dev.stream()));
  Py_RETURN_NONE;
}

// cache, device, src (None: free), first, n (for None)
PyObject *cache_fork(PyObject *const *a) {
  const nq_cache *c = cache_of(a[0]);
  const Device dev(small(a[1], "device"));
  const int first = small(a[3], "first");
  const int32_t *src = ints(a[2], "src", -1, dev.index);
  const int n = a[2] != Py_None ? static_cast<int>(THPVariable_Unpack(a[2]).numel()) : a[4] != Py_None ? small(a[4], "n") : c->slots - first;
  check(nq_cache_fork(c, first, n, src, dev.stream()));
  Py_RETURN_NONE;
}

// cache, device, window, sinks, first, n
PyObject *cache_trim(PyObject *const *a) {
  const nq_cache *c = cache_of(a[0]);
  const Device dev(small(a[1], "device"));
  const int first = small(a[4], "first"), n = a[5] != Py_None ? small(a[5], "n") : c->slots - first;
  check(nq_cache_trim(c, first, n, small(a[3], "sinks"), small(a[2], "window"), dev.stream()));
  Py_RETURN_NONE;
}

// cache, device
PyObject *cache_compact(PyObject *const *a) {
  const Device dev(small(a[1], "device"));
  check(nq_cache_compact(cache_of(a[0]), dev.stream()));
  Py_RETURN_NONE;
}
PyObject *cache_check(PyObject *const *a) {
  const Device dev(small(a[1], "device"));
  const nq_cache *c = cache_of(a[0]);
  int rc;
  Py_BEGIN_ALLOW_THREADS rc = nq_cache_status(c, nullptr, dev.stream());
  Py_END_ALLOW_THREADS check(rc);
  Py_RETURN_NONE;
}

void *pair(const at::Tensor &t, const char *name, int64_t items, int64_t beams, bool flag, at::ScalarType type, int dev) {
  const bool is = flag ? t.scalar_type() == at::kBool || t.scalar_type() == at::kByte : t.scalar_type() == type;
  if (t.dim() != 2 || t.size(0) != items || t.size(1) != beams || !is || !t.is_cuda() || t.get_device() != dev || !t.is_contiguous())
    misfit(std::string(name) + " must be contiguous [" + std::to_string(items) + ", " + std::to_string(beams) + "] of " +
           (flag ? "bool or uint8" : c10::toString(type)) + " on " + where(dev));
  return t.data_ptr();
}

// logits, scores, finished, eos, out
PyObject *beam_select(PyObject *const *a) {
  const at::Tensor &x = tensor(a[0], "logits"), &s = tensor(a[1], "scores");
  if (x.dim() != 3) misfit("logits must be [items, beams, vocab]");
  const int64_t items = x.size(0), beams = x.size(1), vocab = x.size(2);
  if ((vocab > 1 && x.stride(2) != 1) || (items > 1 && beams > 1 && x.stride(0) != beams * x.stride(1)))
    misfit("logits must have unit stride along the vocabulary and evenly spaced rows");
  const int code = code_of(x, "logits");
  at::Tensor o[4];
  if (a[4] != Py_None) {
    const Ref seq{PySequence_Fast(a[4], "out must be (scores, parents, tokens, finished)")};
    if (!seq.p) throw Failed();
    if (PySequence_Fast_GET_SIZE(seq.p) != 4) misfit("out must be (scores, parents, tokens, finished)");
    for (int i = 0; i < 4; ++i) {
      o[i] = tensor(PySequence_Fast_GET_ITEM(seq.p, i), "each of out");
      apart(o[i], x, false, "the logits");
      apart(o[i], s, i == 0, "the scores");
      if (a[2] != Py_None) apart(o[i], tensor(a[2], "finished"), i == 3, "finished");
      for (int j = 0; j < i; ++j) apart(o[i], o[j], false, "another output");
    }
  }
  const Device dev(x, "logits");
  if (items > 65535 || beams > 65535) misfit("too many items or beams");
  const int64_t need = nq_beam_workspace(static_cast<int>(items), static_cast<int>(beams), vocab);
  check(need);
  const void *scores = pair(s, "scores", items, beams, false, at::kFloat, dev.index);
  const void *finished = a[2] == Py_None ? nullptr : pair(tensor(a[2], "finished"), "finished", items, beams, true, at::kBool, dev.index);
  if (a[4] == Py_None) {
    o[0] = empty({items, beams}, at::kFloat, dev);
    o[1] = empty({items, beams}, at::kInt, dev);
    o[2] = empty({items, beams}, at::kInt, dev);
    o[3] = empty({items, beams}, at::kBool, dev);
  }
  const at::ScalarType types[4] = {at::kFloat, at::kInt, at::kInt, at::kBool};
  void *po[4];
  for (int i = 0; i < 4; ++i) po[i] = pair(o[i], "out", items, beams, i == 3, types[i], dev.index);
  const at::Tensor ws = empty({need}, at::kByte, dev);
  const int64_t ld = beams > 1 ? x.stride(1) : items > 1 ? x.stride(0) : vocab;
  check(nq_beam_select(x.data_ptr(), code, ld, static_cast<int>(items), static_cast<int>(beams), vocab, static_cast<const float *>(scores),
                       static_cast<const uint8_t *>(finished), small(a[3], "eos"), static_cast<float *>(po[0]),
                       static_cast<int32_t *>(po[1]), static_cast<int32_t *>(po[2]), static_cast<uint8_t *>(po[3]), ws.data_ptr(), need,
                       dev.stream()));
  if (a[4] != Py_None) {
    for (const at::Tensor &t : o) written(t);
    return Py_INCREF(a[4]), a[4];
  }
  PyObject *r = PyTuple_New(4);
  if (!r) throw Failed();
  for (int i = 0; i < 4; ++i) PyTuple_SET_ITEM(r, i, THPVariable_Wrap(o[i]));
  return r;
}

// Bytes between the rows of a state whose rows are contiguous.
int64_t row_stride(const at::Tensor &t, int64_t rows, int64_t row_bytes) {
  if (t.is_contiguous()) return row_bytes;
  int64_t want = 1;
  for (int64_t i = t.dim() - 1; i > 0; --i) {
    if (t.size(i) > 1 && t.stride(i) != want) misfit("a state's rows must be contiguous");
    want *= t.size(i);
  }
  return rows > 1 ? t.stride(0) * static_cast<int64_t>(t.element_size()) : row_bytes;
}

// states, parents, out
PyObject *beam_reorder(PyObject *const *a) {
  const at::Tensor &parents = tensor(a[1], "parents");
  const Device dev(parents, "parents");
  if (parents.scalar_type() != at::kInt || !parents.is_contiguous()) misfit("parents must be contiguous int32 on " + where(dev.index));
  const int64_t rows = parents.numel();
  if (rows > INT32_MAX) misfit("too many rows");
  const Ref in{PySequence_Fast(a[0], "states must be a sequence of tensors")};
  if (!in.p) throw Failed();
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(in.p);
  const Ref given{a[2] == Py_None ? nullptr : PySequence_Fast(a[2], "out must be a sequence of tensors")};
  if (a[2] != Py_None && !given.p) throw Failed();
  if (given.p && PySequence_Fast_GET_SIZE(given.p) != n)
    misfit(std::to_string(PySequence_Fast_GET_SIZE(given.p)) + " outputs for " + std::to_string(n) + " states");
  Ref result{PyList_New(n)};
  if (!result.p) throw Failed();
  std::vector<const void *> src;
  std::vector<void *> dst;
  std::vector<int64_t> bytes, src_by, dst_by;
  std::vector<at::Tensor> outs;  // given ones
  for (Py_ssize_t i = 0; i < n; ++i) {
    const at::Tensor &t = tensor(PySequence_Fast_GET_ITEM(in.p, i), "a state");
    const std::string want = "a state must be [" + std::to_string(rows) + ", ...] on " + where(dev.index) + ", like its output";
    if (t.dim() < 1 || t.size(0) != rows || !t.is_cuda() || t.get_device() != dev.index) misfit(want);
    at::Tensor o;
    if (given.p) {
      PyObject *e = PySequence_Fast_GET_ITEM(given.p, i);
      o = tensor(e, "an output");
      if (o.sizes() != t.sizes() || o.scalar_type() != t.scalar_type() || !o.is_cuda() || o.get_device() != dev.index) misfit(want);
      Py_INCREF(e);
      PyList_SET_ITEM(result.p, i, e);
      outs.push_back(o);
    } else {
      o = empty(t.sizes(), t.scalar_type(), dev);
      PyList_SET_ITEM(result.p, i, THPVariable_Wrap(o));
    }
    if (t.numel() == 0) continue;
    const int64_t row = t.numel() / rows * static_cast<int64_t>(t.element_size());
    src.push_back(t.data_ptr());
    dst.push_back(o.data_ptr());
    bytes.push_back(row);
    src_by.push_back(row_stride(t, rows, row));
    dst_by.push_back(row_stride(o, rows, row));
  }
  constexpr size_t kMost = 16;  // states of one launch, which checks its own
  if (src.size() > kMost &&
      nq::reorder_overlaps(src.data(), dst.data(), bytes.data(), src_by.data(), dst_by.data(), static_cast<int>(src.size()), rows))
    misfit("an output overlaps another state");
  for (size_t i = 0; i < dst.size(); ++i)
    if (nq::overlap({dst[i], bytes[i], dst_by[i]}, {parents.data_ptr(), 4, 4}, rows)) misfit("an output overlaps the parents");
  for (size_t i = 0; i < src.size(); i += kMost)
    check(nq_beam_reorder(&src[i], &dst[i], &bytes[i], &src_by[i], &dst_by[i], static_cast<int>(std::min(kMost, src.size() - i)),
                          static_cast<int>(rows), static_cast<const int32_t *>(parents.data_ptr()), dev.stream()));
  for (const at::Tensor &t : outs) written(t);
  PyObject *r = result.p;
  result.p = nullptr;
  return r;
}

PyObject *errors(PyObject *const *a) {
  Py_INCREF(a[0]);
  Py_INCREF(a[1]);
  g_misfit = a[0];
  g_failed = a[1];
  Py_RETURN_NONE;
}

// No C++ exception leaves a function: torch's become its Python errors.
template <PyObject *(*F)(PyObject *const *), int N>
PyObject *call(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "%d arguments expected, %zd given", N, n);
    return nullptr;
  }
  try {
    return F(args);
  } catch (const Failed &) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

#define NQ_FN(name, n) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(call<name, n>)), METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {NQ_FN(window_attention, 13), NQ_FN(cache_attention, 12), NQ_FN(cache_reserve, 5), NQ_FN(cache_write, 8),
                           NQ_FN(cache_fork, 5),        NQ_FN(cache_trim, 6),       NQ_FN(cache_compact, 2), NQ_FN(cache_check, 2),
                           NQ_FN(beam_select, 5),       NQ_FN(beam_reorder, 3),     NQ_FN(errors, 2),        {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "nq8_py", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject *PyInit_nq8_py() { return PyModule_Create(&g_module); }
