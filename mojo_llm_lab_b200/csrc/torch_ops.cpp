// Python extension behind the paged-cache functions of ops.py: checks of the
// tensors, result allocation, the current stream, and the C ABI call.
//
// ops.py does this in Python for the other operators.  The single-token forms
// here take 3-17 us on the GPU, with ten or more tensors each to check: a call
// took 20-32 us from Python in that form, in this one 4-10, launches and
// allocations included.
//
// Every function takes the positional arguments of its namesake in ops.py.
// Errors are those of ops.py: ValueError for shapes, types and alignment,
// MllbError for CUDA failures; no C++ exception leaves a function.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <exception>
#include <string>

#include "mllb200.h"

namespace {

PyObject* g_error = nullptr;  // _lib.MllbError

struct ValueFailure {
  std::string text;
};
struct CallFailure {
  int code;
  std::string text;
};
struct PythonFailure {};  // a Python error is set

[[noreturn]] void refuse(const char* fmt, ...) {
  char text[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(text, sizeof(text), fmt, ap);
  va_end(ap);
  throw ValueFailure{text};
}

void check(int64_t rc, const char* what) {
  if (rc >= 0) return;
  const std::string text = std::string(what) + ": " + mllb_last_error();
  if (rc == MLLB_EINVAL || rc == MLLB_EALIGN) throw ValueFailure{text + " (code " + std::to_string(rc) + ")"};
  throw CallFailure{static_cast<int>(rc), text};
}

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) refuse("%s must be a torch.Tensor", name);
  return THPVariable_Unpack(o);
}

// None gives an undefined tensor.
at::Tensor maybe(PyObject* o, const char* name) { return o == Py_None ? at::Tensor() : tensor(o, name); }

int64_t integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw PythonFailure{};
  return v;
}
double real(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw PythonFailure{};
  return v;
}
bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw PythonFailure{};
  return v != 0;
}

int type_of(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return MLLB_TYPE_F32;
    case at::kHalf: return MLLB_TYPE_F16;
    case at::kBFloat16: return MLLB_TYPE_BF16;
    default: return -1;
  }
}

// Last dimension contiguous, the others of any stride.
void need_view(const at::Tensor& t, const char* name, int64_t dims) {
  if (t.dim() != dims) refuse("%s must have %d dimensions, got %d", name, static_cast<int>(dims), static_cast<int>(t.dim()));
  if (t.numel() == 0) refuse("%s is empty", name);
  if (t.size(-1) > 1 && t.stride(-1) != 1) refuse("%s must be contiguous in its last dimension", name);
}

void need_ints(const at::Tensor& t, const char* name, std::initializer_list<int64_t> shape) {
  if (t.scalar_type() != at::kInt || t.sizes() != at::IntArrayRef(shape) || !t.is_contiguous()) {
    std::string text;
    for (const int64_t n : shape) text += (text.empty() ? "" : ", ") + std::to_string(n);
    refuse("%s must be a contiguous torch.int32 tensor of shape [%s]", name, text.c_str());
  }
}

void need_table(const at::Tensor& t, const char* name) {
  if (t.dim() != 2) refuse("%s must be a table of pages [lines, pages]", name);
  need_ints(t, name, {t.size(0), t.size(1)});
}

// All defined tensors on one CUDA device.
c10::Device one_device(std::initializer_list<const at::Tensor*> ts) {
  const c10::Device dev = (*ts.begin())->device();
  for (const at::Tensor* t : ts)
    if (t->defined() && t->device() != dev)
      refuse("tensors on different devices: %s, %s", dev.str().c_str(), t->device().str().c_str());
  if (!dev.is_cuda()) refuse("the tensors must be CUDA tensors");
  return dev;
}

template <typename T = void>
T* ptr(const at::Tensor& t) {
  return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr;
}

at::Tensor empty(at::IntArrayRef shape, at::ScalarType type, c10::Device dev) {
  return at::empty(shape, at::TensorOptions().dtype(type).device(dev));
}

mllb_paged_cache paged_cache(const at::Tensor& k, const at::Tensor& v, bool layers) {
  const int64_t lead = layers && k.dim() == 5 ? 1 : 0;
  if (type_of(k) != MLLB_TYPE_F16 && type_of(k) != MLLB_TYPE_BF16) refuse("k_cache must be torch.float16 or torch.bfloat16");
  need_view(k, "k_cache", 4 + lead);
  bool match = v.scalar_type() == k.scalar_type() && v.sizes() == k.sizes();
  for (int64_t i = 0; match && i < k.dim(); ++i) match = k.size(i) == 1 || v.stride(i) == k.stride(i);
  if (!match) refuse("v_cache must match k_cache in type, shape and strides");
  const int64_t d = k.size(3 + lead);
  // A dimension of one element may carry any stride: it gets one that the kernels take.
  auto step = [&](int64_t dim) { return k.size(dim) > 1 ? k.stride(dim) : d * 8; };
  mllb_paged_cache c = {};
  c.k = k.data_ptr();
  c.v = v.data_ptr();
  c.pages = k.size(lead);
  c.kv_heads = k.size(lead + 1);
  c.page_size = k.size(lead + 2);
  c.head_dim = d;
  c.page_stride = step(lead);
  c.head_stride = step(lead + 1);
  c.row_stride = step(lead + 2);
  c.layers = lead ? k.size(0) : 1;
  c.layer_stride = lead ? step(0) : 0;
  c.type = type_of(k);
  return c;
}

// A C ABI call without the interpreter lock (a full launch queue makes it wait).
template <typename F>
int64_t unlocked(F call) {
  PyThreadState* state = PyEval_SaveThread();
  const int64_t rc = call();
  PyEval_RestoreThread(state);
  return rc;
}

void* stream_of(c10::Device dev) { return c10::cuda::getCurrentCUDAStream(dev.index()).stream(); }

using Args = PyObject* const*;

PyObject* paged_qkv_append(Args o) {
  const at::Tensor &qkv = tensor(o[0], "qkv"), &positions = tensor(o[1], "positions"), &rows = tensor(o[2], "rows"),
                   &table = tensor(o[3], "page_table"), &k = tensor(o[4], "k_cache"), &v = tensor(o[5], "v_cache"),
                   &freqs = tensor(o[7], "freqs");
  const int64_t q_heads = integer(o[6]);
  const at::Tensor seq = maybe(o[8], "seq"), q_gamma = maybe(o[9], "q_gamma"), k_gamma = maybe(o[10], "k_gamma");
  at::Tensor q_out = maybe(o[14], "q_out");
  const mllb_paged_cache cache = paged_cache(k, v, false);
  if (type_of(qkv) < 0) refuse("qkv must be torch.float32, torch.float16 or torch.bfloat16");
  need_view(qkv, "qkv", 2);
  const int64_t tokens = qkv.size(0), d = cache.head_dim;
  if (q_heads <= 0 || qkv.size(1) != (q_heads + 2 * cache.kv_heads) * d)
    refuse("qkv must hold (q_heads + 2 kv_heads) x head_dim values a token");
  need_ints(positions, "positions", {tokens});
  need_ints(rows, "rows", {tokens});
  need_table(table, "page_table");
  if (seq.defined())
    need_ints(seq, "seq", {tokens});
  else if (tokens > table.size(0))
    refuse("without seq, token t is sequence t's: more tokens than sequences");
  for (const at::Tensor* g : {&q_gamma, &k_gamma})
    if (g->defined() && (g->scalar_type() != at::kFloat || g->numel() != d || !g->is_contiguous()))
      refuse("%s must be %d contiguous fp32 values", g == &q_gamma ? "q_gamma" : "k_gamma", static_cast<int>(d));
  if (freqs.scalar_type() != at::kDouble || freqs.dim() != 1 || !freqs.is_contiguous() || freqs.numel() < 1 ||
      freqs.numel() > d / 2)
    refuse("freqs must be 1 to %d contiguous fp64 values", static_cast<int>(d / 2));
  if (q_out.defined() && (q_out.scalar_type() != k.scalar_type() || q_out.sizes() != at::IntArrayRef({tokens, q_heads, d}) ||
                          !q_out.is_contiguous()))
    refuse("q_out must be contiguous [tokens, q_heads, head_dim] of the caches' type");
  const c10::Device dev = one_device({&qkv, &positions, &rows, &table, &k, &v, &freqs, &seq, &q_gamma, &k_gamma, &q_out});
  const c10::cuda::CUDAGuard guard(dev);
  if (!q_out.defined()) q_out = empty({tokens, q_heads, d}, k.scalar_type(), dev);
  mllb_paged_append a = {};
  a.qkv = ptr(qkv);
  a.tokens = tokens;
  a.qkv_stride = tokens > 1 ? qkv.stride(0) : qkv.size(1);
  a.positions = ptr<const int32_t>(positions);
  a.rows = ptr<const int32_t>(rows);
  a.seq = ptr<const int32_t>(seq);
  a.page_table = ptr<const int32_t>(table);
  a.seqs = table.size(0);
  a.table_width = table.size(1);
  a.q_gamma = ptr<const float>(q_gamma);
  a.k_gamma = ptr<const float>(k_gamma);
  a.freqs = ptr<const double>(freqs);
  a.rot_dim = 2 * freqs.numel();
  a.q_heads = q_heads;
  a.interleaved = truth(o[11]);
  a.magnitude = real(o[12]);
  a.eps = real(o[13]);
  a.q_out = ptr(q_out);
  a.qkv_type = type_of(qkv);
  const unsigned flags = truth(o[15]) ? MLLB_LAUNCH_PDL : 0;
  void* stream = stream_of(dev);
  check(unlocked([&] { return mllb_paged_qkv_append(&a, &cache, flags, stream); }), "paged_qkv_append");
  return THPVariable_Wrap(q_out);
}

PyObject* paged_attention(Args o) {
  const at::Tensor &q = tensor(o[0], "q"), &k = tensor(o[1], "k_cache"), &v = tensor(o[2], "v_cache"),
                   &table = tensor(o[3], "page_table"), &lens = tensor(o[4], "seq_lens");
  const at::Tensor prefix_table = maybe(o[5], "prefix_table"), prefix_lens = maybe(o[6], "prefix_lens"),
                   group_start = maybe(o[7], "group_start"), q_start = maybe(o[8], "q_start");
  at::Tensor out = maybe(o[10], "out"), workspace = maybe(o[11], "workspace");
  const mllb_paged_cache cache = paged_cache(k, v, false);
  if (q.scalar_type() != k.scalar_type()) refuse("q must be of the caches' type");
  need_view(q, "q", 3);
  const int64_t tokens = q.size(0), q_heads = q.size(1), d = q.size(2);
  if (d != cache.head_dim) refuse("q has heads of %d, the caches of %d", static_cast<int>(d), static_cast<int>(cache.head_dim));
  if (q_heads % cache.kv_heads) refuse("q_heads must be a multiple of kv_heads");
  need_table(table, "page_table");
  const int64_t seqs = table.size(0);
  need_ints(lens, "seq_lens", {seqs});
  int64_t groups = 0, prefix_width = 0;
  if (prefix_table.defined()) {
    need_table(prefix_table, "prefix_table");
    groups = prefix_table.size(0);
    prefix_width = prefix_table.size(1);
    if (!prefix_lens.defined()) refuse("prefix_table needs prefix_lens");
    need_ints(prefix_lens, "prefix_lens", {groups});
    if (group_start.defined())
      need_ints(group_start, "group_start", {groups + 1});
    else if (groups > 1)
      refuse("several groups need group_start");
  } else if (prefix_lens.defined() || group_start.defined()) {
    refuse("prefix_lens and group_start need prefix_table");
  }
  if (q_start.defined())
    need_ints(q_start, "q_start", {seqs + 1});
  else if (tokens != seqs)
    refuse("without q_start every sequence has one token");
  if (out.defined()) {
    if (out.scalar_type() != q.scalar_type()) refuse("out must be of the type of q");
    if (out.sizes() != q.sizes()) refuse("out must have the shape of q");
    need_view(out, "out", 3);
  }
  if (workspace.defined() && (workspace.scalar_type() != at::kByte || !workspace.is_contiguous()))
    refuse("workspace must be contiguous torch.uint8");
  const c10::Device dev = one_device({&q, &k, &v, &table, &lens, &prefix_table, &prefix_lens, &group_start, &q_start, &out,
                                      &workspace});
  const c10::cuda::CUDAGuard guard(dev);
  if (!out.defined()) out = empty({tokens, q_heads, d}, q.scalar_type(), dev);
  // The stride of a dimension of one element counts as whole heads.
  auto step = [d](const at::Tensor& t, int64_t dim) { return t.size(dim) > 1 ? t.stride(dim) : d; };
  mllb_paged_attn a = {};
  a.q = ptr(q);
  a.out = ptr(out);
  a.tokens = tokens;
  a.q_heads = q_heads;
  a.q_token_stride = step(q, 0);
  a.q_head_stride = step(q, 1);
  a.out_token_stride = step(out, 0);
  a.out_head_stride = step(out, 1);
  a.page_table = ptr<const int32_t>(table);
  a.seq_lens = ptr<const int32_t>(lens);
  a.seqs = seqs;
  a.table_width = table.size(1);
  a.prefix_table = ptr<const int32_t>(prefix_table);
  a.prefix_lens = ptr<const int32_t>(prefix_lens);
  a.group_start = ptr<const int32_t>(group_start);
  a.groups = groups;
  a.prefix_width = prefix_width;
  a.q_start = ptr<const int32_t>(q_start);
  a.scale = o[9] == Py_None ? 1.0 / std::sqrt(static_cast<double>(d)) : real(o[9]);
  if (!workspace.defined()) {
    const int64_t need = mllb_paged_attention_call_workspace(&a, &cache);
    check(need, "paged_attention");
    workspace = empty({need}, at::kByte, dev);
  }
  const unsigned flags = truth(o[12]) ? MLLB_LAUNCH_PDL : 0;
  void* stream = stream_of(dev);
  check(unlocked([&] { return mllb_paged_attention(&a, &cache, workspace.data_ptr(), workspace.numel(), flags, stream); }),
        "paged_attention");
  return THPVariable_Wrap(out);
}

// Three result tensors from `out` (a sequence of three, or None for new ones).
void take_three(PyObject* o, at::Tensor (&t)[3]) {
  if (o == Py_None) return;
  if (!PySequence_Check(o) || PySequence_Size(o) != 3) refuse("out must hold three tensors");
  for (int i = 0; i < 3; ++i) {
    PyObject* item = PySequence_GetItem(o, i);
    if (!item) throw PythonFailure{};
    const bool fine = THPVariable_Check(item);
    if (fine) t[i] = THPVariable_Unpack(item);
    Py_DECREF(item);
    if (!fine) refuse("out must hold three tensors");
  }
}

PyObject* three(const at::Tensor (&t)[3]) {
  PyObject* r = PyTuple_New(3);
  if (!r) throw PythonFailure{};
  for (int i = 0; i < 3; ++i) PyTuple_SET_ITEM(r, i, THPVariable_Wrap(t[i]));
  return r;
}

PyObject* beam_select(Args o) {
  const at::Tensor &logits = tensor(o[0], "logits"), &scores = tensor(o[1], "scores");
  const at::Tensor done = maybe(o[3], "done");
  at::Tensor workspace = maybe(o[6], "workspace");
  if (type_of(logits) < 0) refuse("logits must be torch.float32, torch.float16 or torch.bfloat16");
  need_view(logits, "logits", 3);
  const int64_t batch = logits.size(0), beams = logits.size(1), vocab = logits.size(2);
  const int64_t n = o[2] == Py_None ? beams : integer(o[2]), end_token = integer(o[4]);
  if (scores.scalar_type() != at::kFloat || scores.sizes() != at::IntArrayRef({batch, beams}) || !scores.is_contiguous())
    refuse("scores must be contiguous fp32 [batch, beams]");
  if (done.defined()) {
    if ((done.scalar_type() != at::kBool && done.scalar_type() != at::kByte) ||
        done.sizes() != at::IntArrayRef({batch, beams}) || !done.is_contiguous())
      refuse("done must be contiguous bool or uint8 [batch, beams]");
    if (end_token < 0 || end_token >= vocab) refuse("done beams need an end_token of the vocabulary");
  }
  const int64_t need = mllb_beam_select_workspace(batch, beams, vocab, n);
  check(need, "beam_select");
  at::Tensor out[3];
  take_three(o[5], out);
  if (out[0].defined()) {
    if (out[0].scalar_type() != at::kFloat || out[0].sizes() != at::IntArrayRef({batch, n}) || !out[0].is_contiguous())
      refuse("out scores must be contiguous fp32 [batch, n]");
    need_ints(out[1], "out tokens", {batch, n});
    need_ints(out[2], "out parents", {batch, n});
  }
  if (workspace.defined() && (workspace.scalar_type() != at::kByte || !workspace.is_contiguous()))
    refuse("workspace must be contiguous torch.uint8");
  const c10::Device dev = one_device({&logits, &scores, &done, &out[0], &out[1], &out[2], &workspace});
  const c10::cuda::CUDAGuard guard(dev);
  if (!out[0].defined()) {
    out[0] = empty({batch, n}, at::kFloat, dev);
    out[1] = empty({batch, n}, at::kInt, dev);
    out[2] = empty({batch, n}, at::kInt, dev);
  }
  if (!workspace.defined()) workspace = empty({need}, at::kByte, dev);
  mllb_beam_scores a = {};
  a.logits = ptr(logits);
  a.batch = batch;
  a.beams = beams;
  a.vocab = vocab;
  a.n = n;
  a.batch_stride = batch > 1 ? logits.stride(0) : 0;
  a.beam_stride = beams > 1 ? logits.stride(1) : 0;
  a.scores = ptr<const float>(scores);
  a.done = ptr<const uint8_t>(done);
  a.end_token = end_token;
  a.type = type_of(logits);
  const unsigned flags = truth(o[7]) ? MLLB_LAUNCH_PDL : 0;
  void* stream = stream_of(dev);
  check(unlocked([&] {
          return mllb_beam_select(&a, ptr<float>(out[0]), ptr<int32_t>(out[1]), ptr<int32_t>(out[2]), workspace.data_ptr(),
                                  workspace.numel(), flags, stream);
        }),
        "beam_select");
  return three(out);
}

PyObject* beam_reorder(Args o) {
  const at::Tensor &parents = tensor(o[0], "parents"), &table = tensor(o[1], "page_table"), &lens = tensor(o[2], "seq_lens"),
                   &fresh = tensor(o[3], "fresh"), &k = tensor(o[4], "k_cache"), &v = tensor(o[5], "v_cache");
  const mllb_paged_cache cache = paged_cache(k, v, true);
  need_table(table, "page_table");
  const int64_t rows = table.size(0), width = table.size(1);
  if (parents.dim() != 2 || parents.numel() != rows || rows == 0)
    refuse("parents must be [batch, beams] and page_table [batch * beams, pages]");
  need_ints(parents, "parents", {parents.size(0), parents.size(1)});
  need_ints(lens, "seq_lens", {rows});
  need_ints(fresh, "fresh", {rows});
  at::Tensor out[3];
  take_three(o[6], out);
  if (out[0].defined()) {
    need_ints(out[0], "out table", {rows, width});
    need_ints(out[1], "out lens", {rows});
    need_ints(out[2], "out used", {rows});
  }
  const c10::Device dev = one_device({&parents, &table, &lens, &fresh, &k, &v, &out[0], &out[1], &out[2]});
  const c10::cuda::CUDAGuard guard(dev);
  if (!out[0].defined()) {
    out[0] = empty({rows, width}, at::kInt, dev);
    out[1] = empty({rows}, at::kInt, dev);
    out[2] = empty({rows}, at::kInt, dev);
  }
  mllb_beam_rows a = {};
  a.parents = ptr<const int32_t>(parents);
  a.page_table = ptr<const int32_t>(table);
  a.seq_lens = ptr<const int32_t>(lens);
  a.fresh = ptr<const int32_t>(fresh);
  a.batch = parents.size(0);
  a.beams = parents.size(1);
  a.table_width = width;
  const unsigned flags = truth(o[7]) ? MLLB_LAUNCH_PDL : 0;
  void* stream = stream_of(dev);
  check(unlocked([&] {
          return mllb_beam_reorder(&a, &cache, ptr<int32_t>(out[0]), ptr<int32_t>(out[1]), ptr<int32_t>(out[2]), flags, stream);
        }),
        "beam_reorder");
  return three(out);
}

// The boundary: counts the arguments, turns every exception into a Python error.
template <PyObject* (*kCall)(Args), int kArgs>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != kArgs) {
    PyErr_Format(PyExc_TypeError, "expected %d arguments, got %zd", kArgs, n);
    return nullptr;
  }
  try {
    return kCall(args);
  } catch (const PythonFailure&) {
  } catch (const ValueFailure& e) {
    PyErr_SetString(PyExc_ValueError, e.text.c_str());
  } catch (const CallFailure& e) {
    PyObject* error = PyObject_CallFunction(g_error ? g_error : PyExc_RuntimeError, "is", e.code, e.text.c_str());
    if (error) {
      PyErr_SetObject(g_error ? g_error : PyExc_RuntimeError, error);
      Py_DECREF(error);
    }
  } catch (const std::bad_alloc&) {
    PyErr_NoMemory();
  } catch (const std::exception& e) {  // out of memory on the device among them
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
  }
  return nullptr;
}

PyObject* set_error(PyObject*, PyObject* type) {
  Py_INCREF(type);
  Py_XDECREF(g_error);
  g_error = type;
  Py_RETURN_NONE;
}

template <PyObject* (*kCall)(Args), int kArgs>
PyMethodDef method(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<kCall, kArgs>)), METH_FASTCALL, nullptr};
}

PyMethodDef g_methods[] = {method<paged_qkv_append, 16>("paged_qkv_append"),
                           method<paged_attention, 13>("paged_attention"),
                           method<beam_select, 8>("beam_select"),
                           method<beam_reorder, 8>("beam_reorder"),
                           {"set_error", set_error, METH_O, nullptr},
                           {nullptr, nullptr, 0, nullptr}};

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "mllb200_torch", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_mllb200_torch(void) { return PyModule_Create(&g_module); }
