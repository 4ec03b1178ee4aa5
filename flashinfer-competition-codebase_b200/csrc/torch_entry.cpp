// torch_entry.cpp — the serving operators' calls from Python without the interpreter's cost.
//
// A call of a small size is bound by host work: checking a dozen tensors, allocating the
// outputs and passing 27 values through ctypes took 14 to 20 us where the launch takes 3.
// Each function here checks its tensors, allocates its outputs and makes the one library
// call of its namesake in serving.py.  It returns
//   the result              the call is made
//   None                    some check did not hold: serving.py checks again in Python, and
//                           raises, or makes the rarer call itself (int64 indices, other forms)
//   an int                  the library's error code
// It owns no rule of its own: what it accepts, serving.py accepts with the same result.

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <optional>
#include <vector>

#include "gdn_b200.h"

namespace {

using at::Tensor;

// An argument that is no tensor, or a tensor that fails a check, ends the fast path.
struct NotHere {};

const Tensor& tensor(PyObject* o) {
  if (!THPVariable_Check(o)) throw NotHere{};
  return THPVariable_Unpack(o);
}

std::optional<Tensor> maybe(PyObject* o) {
  if (o == Py_None) return std::nullopt;
  return tensor(o);
}

void need(bool ok) {
  if (!ok) throw NotHere{};
}

void need(const Tensor& t, at::ScalarType type, at::IntArrayRef sizes, const at::Device& dev) {
  need(t.scalar_type() == type && t.device() == dev && t.sizes() == sizes && t.is_contiguous());
}

long long integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    throw NotHere{};
  }
  return v;
}

int int32(PyObject* o) {
  const long long v = integer(o);
  need(v >= INT32_MIN && v <= INT32_MAX);
  return static_cast<int>(v);
}

double number_or_zero(PyObject* o) {
  if (o == Py_None) return 0.0;
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    throw NotHere{};
  }
  return v;
}

Tensor empty(at::IntArrayRef sizes, at::ScalarType type, const at::Device& dev) {
  return at::detail::empty_cuda(sizes, type, dev, std::nullopt);
}

template <typename T = void> T* ptr(const Tensor& t) { return static_cast<T*>(t.data_ptr()); }
template <typename T = void> T* ptr(const std::optional<Tensor>& t) {
  return t ? static_cast<T*>(t->data_ptr()) : nullptr;
}

int32_t* counter(PyObject* o, const at::Device& dev, std::optional<Tensor>& hold) {
  hold = maybe(o);
  if (hold) need(*hold, at::kInt, {1}, dev);
  return ptr<int32_t>(hold);
}

// The device is current while this lives, and `stream` is its current stream.
struct On {
  c10::cuda::OptionalCUDAGuard guard;
  void* stream;
  explicit On(const at::Device& dev) {
    if (c10::cuda::current_device() != dev.index()) guard.set_device(dev);
    stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  }
};

PyObject* wrap(int code) {
  if (code != GDN_OK) return PyLong_FromLong(code);
  Py_RETURN_TRUE;
}
PyObject* wrap(int code, std::initializer_list<Tensor> results) {
  if (code != GDN_OK) return PyLong_FromLong(code);
  PyObject* out = PyTuple_New(static_cast<Py_ssize_t>(results.size()));
  if (!out) return nullptr;
  Py_ssize_t i = 0;
  for (const Tensor& t : results) PyTuple_SET_ITEM(out, i++, THPVariable_Wrap(t));
  return out;
}

int dtype_code(at::ScalarType t) {
  if (t == at::kBFloat16) return GDN_DTYPE_BF16;
  if (t == at::kHalf) return GDN_DTYPE_FP16;
  need(t == at::kFloat);
  return GDN_DTYPE_FP32;
}

// ------------------------------------------------------------------ paged_attention_decode

void cache(const Tensor& t, at::ScalarType type, const at::Device& dev, int64_t HKV, int64_t D,
           int64_t (&strides)[3]) {
  need(t.dim() == 4 && t.scalar_type() == type && t.device() == dev && t.size(2) == HKV &&
       t.size(3) == D && t.stride(3) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0);
  for (int i = 0; i < 3; ++i) {
    strides[i] = t.size(i) > 1 ? t.stride(i) : 0;
    need((t.size(i) <= 1 || strides[i] > 0) && strides[i] % 8 == 0);
  }
}

PyObject* attend(PyObject* const* a) {
  const Tensor &q = tensor(a[0]), &kc = tensor(a[1]), &vc = tensor(a[2]), &tables = tensor(a[3]),
               &lens = tensor(a[4]);
  const auto k = maybe(a[5]), v = maybe(a[6]), given = maybe(a[10]);
  const int window = int32(a[8]), sinks = int32(a[9]);
  need(q.dim() == 4 && q.size(1) == 1 && q.is_cuda() && q.is_contiguous());
  const int64_t B = q.size(0), HQ = q.size(2), D = q.size(3);
  const at::Device dev = q.device();
  const at::ScalarType type = q.scalar_type();
  need((type == at::kBFloat16 || type == at::kHalf) && (D == 64 || D == 128 || D == 256));
  need(kc.dim() == 4 && kc.sizes() == vc.sizes());
  const int64_t pages = kc.size(0), page_size = kc.size(1), HKV = kc.size(2);
  need(HKV > 0 && HQ > 0 && HQ % HKV == 0 && pages > 0 && page_size > 0 && pages <= INT32_MAX);
  int64_t ks[3], vs[3];
  cache(kc, type, dev, HKV, D, ks);
  cache(vc, type, dev, HKV, D, vs);
  need(tables.dim() == 2 && tables.scalar_type() == at::kInt && tables.device() == dev &&
       tables.size(0) == B);
  const int64_t width = tables.size(1);
  need(width <= 1 || tables.stride(1) == 1);
  need(width <= (int64_t{1} << 31) && width * page_size <= (int64_t{1} << 31) - 2048);
  need(lens, at::kInt, {B}, dev);
  need(k.has_value() == v.has_value());
  if (k) {
    need(*k, type, {B, 1, HKV, D}, dev);
    need(*v, type, {B, 1, HKV, D}, dev);
  }
  constexpr int most = (1 << 30) - 1;
  need(window >= 0 && window <= most && sinks >= 0 && sinks <= most);
  if (given) need(*given, type, {B, 1, HQ, D}, dev);
  std::optional<Tensor> hold;
  int32_t* bad = counter(a[11], dev, hold);
  const double scale = number_or_zero(a[7]);
  const Tensor output = given ? *given : empty({B, 1, HQ, D}, type, dev);
  const Tensor lse = empty({B, HQ}, at::kFloat, dev);
  const int64_t held = width * page_size, seen = int64_t{window} + sinks;
  const size_t bytes = gdn_paged_attention_workspace_bytes(
      static_cast<int>(B), static_cast<int>(HQ), static_cast<int>(HKV), static_cast<int>(D),
      static_cast<int>(window > 0 && seen < held ? seen : held));
  Tensor ws;
  if (bytes) ws = empty({static_cast<int64_t>(bytes)}, at::kByte, dev);
  const On on(dev);
  const int code = gdn_paged_attention_decode(
      ptr(q), ptr(kc), ptr(vc), ptr<int32_t>(tables), ptr<int32_t>(lens), ptr(k), ptr(v), scale,
      window, sinks, ptr(output), ptr<float>(lse), bytes ? ptr(ws) : nullptr, bytes,
      dtype_code(type), static_cast<int>(B), static_cast<int>(HQ), static_cast<int>(HKV),
      static_cast<int>(D), static_cast<int>(pages), static_cast<int>(page_size),
      static_cast<int>(width), B > 1 ? tables.stride(0) : width, ks, vs, bad, on.stream);
  return wrap(code, {output, lse});
}

// ------------------------------------------------------------------ beam_select

PyObject* select(PyObject* const* a) {
  const Tensor &logits = tensor(a[0]), &scores = tensor(a[1]);
  const auto finished = maybe(a[3]);
  const int eos = int32(a[4]);
  need(logits.dim() == 3 && logits.is_cuda());
  const int64_t B = logits.size(0), K = logits.size(1), V = logits.size(2);
  const int64_t n = a[2] == Py_None ? K : integer(a[2]);
  const at::Device dev = logits.device();
  need(K >= 1 && K <= 64 && V >= 1 && V <= INT32_MAX && B <= INT32_MAX && n >= 1 && n <= 64);
  need(V == 1 || logits.stride(2) == 1);
  need(scores, at::kFloat, {B, K}, dev);
  if (finished) {
    need(*finished, at::kBool, {B, K}, dev);
    need(eos >= 0 && eos < V);
  }
  const int type = dtype_code(logits.scalar_type());
  const Tensor tokens = empty({B, n}, at::kInt, dev), parents = empty({B, n}, at::kInt, dev);
  const Tensor out = empty({B, n}, at::kFloat, dev);
  const size_t bytes = gdn_beam_select_workspace_bytes(static_cast<int>(B), static_cast<int>(K),
                                                       static_cast<int>(V), static_cast<int>(n));
  const Tensor ws = empty({static_cast<int64_t>(bytes)}, at::kByte, dev);
  const On on(dev);
  const int code = gdn_beam_select(
      ptr(logits), type, logits.stride(0), logits.stride(1), ptr<float>(scores),
      ptr<uint8_t>(finished), eos, static_cast<int>(B), static_cast<int>(K), static_cast<int>(V),
      static_cast<int>(n), ptr<int32_t>(tokens), ptr<int32_t>(parents), ptr<float>(out), ptr(ws),
      bytes, on.stream);
  return wrap(code, {tokens, parents, out});
}

// ------------------------------------------------------------------ cache pages

struct PoolList {
  void* base[32];
  int64_t bytes[32], pitch[32];
  int count = 0;
  int64_t pages = -1;
  std::optional<at::Device> dev;

  void add(PyObject* o) {
    const Tensor& t = tensor(o);
    need(count < 32 && t.dim() >= 2 && t.is_cuda() && t.numel() > 0 && t.is_contiguous());
    if (pages < 0) pages = t.size(0);
    if (!dev) dev = t.device();
    need(t.size(0) == pages && t.device() == *dev && pages <= (1 << 30));
    base[count] = t.data_ptr();
    bytes[count] = pitch[count] = t.numel() / pages * static_cast<int64_t>(t.element_size());
    ++count;
  }
  PoolList(PyObject* o, std::optional<at::Device> device = std::nullopt, int64_t num_pages = -1)
      : pages(num_pages), dev(device) {
    if (THPVariable_Check(o)) {
      add(o);
    } else {
      need(PyList_Check(o) || PyTuple_Check(o));
      const Py_ssize_t n = PySequence_Fast_GET_SIZE(o);
      for (Py_ssize_t i = 0; i < n; ++i) add(PySequence_Fast_GET_ITEM(o, i));
    }
  }
};

const Tensor& indices(PyObject* o, const at::Device& dev) {
  const Tensor& t = tensor(o);
  need(t.dim() == 1 && t.scalar_type() == at::kInt && t.device() == dev && t.is_contiguous() &&
       t.size(0) <= INT32_MAX);
  return t;
}

const Tensor& references(PyObject* o) {
  const Tensor& t = tensor(o);
  need(t.is_cuda() && t.size(0) >= 1);
  return indices(o, t.device());
}

PyObject* copy(PyObject* const* a) {
  PoolList p(a[0]);
  need(p.count > 0);
  const Tensor &src = indices(a[1], *p.dev), &dst = indices(a[2], *p.dev);
  need(src.size(0) == dst.size(0) && src.size(0) <= 4096);
  std::optional<Tensor> hold;
  int32_t* bad = counter(a[3], *p.dev, hold);
  const On on(*p.dev);
  return wrap(gdn_copy_pages(p.base, p.bytes, p.pitch, p.count, static_cast<int>(p.pages),
                             ptr<int32_t>(src), ptr<int32_t>(dst), static_cast<int>(src.size(0)),
                             bad, on.stream));
}

PyObject* alloc(PyObject* const* a) {
  const Tensor &refs = references(a[0]), &flags = tensor(a[1]);
  const at::Device dev = refs.device();
  need(flags.dim() == 1 && flags.scalar_type() == at::kBool && flags.device() == dev &&
       flags.is_contiguous() && flags.size(0) <= INT32_MAX);
  const int64_t n = flags.size(0);
  const Tensor pages = empty({n}, at::kInt, dev), ws = empty({n}, at::kInt, dev);
  const On on(dev);
  return wrap(gdn_alloc_pages(ptr<int32_t>(refs), static_cast<int>(refs.size(0)),
                              ptr<uint8_t>(flags), static_cast<int>(n), ptr<int32_t>(pages),
                              ptr(ws), static_cast<size_t>(4 * n), on.stream),
              {pages});
}

PyObject* release(PyObject* const* a) {
  const Tensor &refs = references(a[0]), &pages = tensor(a[1]);
  const at::Device dev = refs.device();
  need(pages.scalar_type() == at::kInt && pages.device() == dev && pages.is_contiguous());
  std::optional<Tensor> hold;
  int32_t* bad = counter(a[2], dev, hold);
  const On on(dev);
  return wrap(gdn_free_pages(ptr<int32_t>(refs), static_cast<int>(refs.size(0)),
                             ptr<int32_t>(pages), pages.numel(), bad, on.stream));
}

PyObject* fork(PyObject* const* a) {
  const Tensor &tables = tensor(a[0]), &lens = tensor(a[1]), &refs = references(a[3]);
  const at::Device dev = refs.device();
  const Tensor& parents = indices(a[2], dev);
  const int page_size = int32(a[4]);
  need(tables.dim() == 2 && tables.scalar_type() == at::kInt && tables.device() == dev &&
       tables.is_contiguous());
  const int64_t rows = tables.size(0), width = tables.size(1), n = parents.size(0);
  need(rows <= INT32_MAX && width <= INT32_MAX && page_size >= 1 &&
       width * page_size <= (int64_t{1} << 31) - 1);
  need(lens, at::kInt, {rows}, dev);
  PoolList p(a[5], dev, refs.size(0));
  std::optional<Tensor> hold;
  int32_t* bad = counter(a[6], dev, hold);
  const Tensor new_tables = empty({n, width}, at::kInt, dev), new_lens = empty({n}, at::kInt, dev);
  const Tensor ws = empty({3 * n}, at::kInt, dev);
  const On on(dev);
  return wrap(
      gdn_fork_pages(ptr<int32_t>(tables), width, ptr<int32_t>(lens), ptr<int32_t>(parents),
                     ptr<int32_t>(refs), ptr<int32_t>(new_tables), ptr<int32_t>(new_lens),
                     static_cast<int>(rows), static_cast<int>(n), static_cast<int>(width),
                     static_cast<int>(refs.size(0)), page_size, p.base, p.bytes, p.pitch, p.count,
                     ptr(ws), static_cast<size_t>(12 * n), bad, on.stream),
      {new_tables, new_lens});
}

PyObject* compact(PyObject* const* a) {
  const Tensor& refs = references(a[0]);
  const at::Device dev = refs.device();
  const auto tables = maybe(a[1]);
  if (tables)
    need(tables->scalar_type() == at::kInt && tables->device() == dev && tables->is_contiguous());
  const int64_t P = refs.size(0), entries = tables ? tables->numel() : 0;
  PoolList p(a[2], dev, P);
  const int64_t words = 2 * (P / 2 + 1) + 1;
  const Tensor remap = empty({P}, at::kInt, dev), live = empty({1}, at::kInt, dev);
  const Tensor ws = empty({words}, at::kInt, dev);
  const On on(dev);
  return wrap(gdn_compact_pages(ptr<int32_t>(refs), static_cast<int>(P),
                                entries ? ptr<int32_t>(tables) : nullptr, entries,
                                ptr<int32_t>(remap), ptr<int32_t>(live), p.base, p.bytes, p.pitch,
                                p.count, ptr(ws), static_cast<size_t>(4 * words), on.stream),
              {remap, live});
}

template <PyObject* (*kCall)(PyObject* const*), int kArgs>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != kArgs) Py_RETURN_NONE;
  try {
    return kCall(args);
  } catch (...) {      // a check, or an allocation (before the library call): Python raises
    PyErr_Clear();
    Py_RETURN_NONE;
  }
}

#define GDN_ENTRY(name, args) \
  {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(&entry<name, args>)), METH_FASTCALL, nullptr}

PyMethodDef kMethods[] = {
    GDN_ENTRY(attend, 12), GDN_ENTRY(select, 5), GDN_ENTRY(copy, 4),    GDN_ENTRY(alloc, 2),
    GDN_ENTRY(release, 3), GDN_ENTRY(fork, 7),   GDN_ENTRY(compact, 3), {nullptr, nullptr, 0, nullptr}};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "gdn_b200_torch", nullptr, -1, kMethods,
                       nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_gdn_b200_torch(void) { return PyModule_Create(&kModule); }
