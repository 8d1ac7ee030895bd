/* Host-side call path of the paged operators and token_logprobs, as a CPython
 * extension over torch's tensors.
 *
 * A serving step makes these calls once a layer with kernels of 3 to 10 µs.
 * Written in Python, one call's checks, packed arguments, allocations and launch
 * take 10 to 13 µs of the host; here they take 4. Each function takes a call
 * whose arguments are as the kernels want them, and otherwise does nothing and
 * returns None: the Python function then reports what is wrong, or copies what
 * only needs another layout. So every refusal and its text lives in Python, and
 * whatever this file takes, Python would have passed on unchanged.
 *
 * A returned int is the C ABI's status. bind() gives the entry points' addresses;
 * nothing here links to the HIP library.
 */
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <torch/csrc/autograd/python_variable.h>

#include "ssalaad_amd.h"

namespace {

using at::Tensor;

struct {
  decltype(&ssl_paged_append) append;
  decltype(&ssl_paged_attention_workspace_size) attention_bytes;
  decltype(&ssl_paged_attention) attention;
  decltype(&ssl_pages_free) free;
  decltype(&ssl_pages_fork_workspace_size) fork_bytes;
  decltype(&ssl_pages_fork) fork;
  decltype(&ssl_pages_compact_workspace_size) compact_bytes;
  decltype(&ssl_pages_compact) compact;
  decltype(&ssl_token_logprobs) logprobs;
} entry;
PyObject* raw_stream;  // torch._C._cuda_getCurrentRawStream

// A plain strided GPU tensor, or null.
const Tensor* tensor(PyObject* o) {
  if (!THPVariable_Check(o)) return nullptr;
  const Tensor& t = THPVariable_Unpack(o);
  if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || t.is_neg() ||
      t.key_set().has(c10::DispatchKey::Python))
    return nullptr;
  return &t;
}

bool dtype_of(const Tensor& t, int64_t* code, int64_t* align) {
  const auto s = t.scalar_type();
  *code = s == at::kFloat ? SSL_F32 : s == at::kBFloat16 ? SSL_BF16 : SSL_F16;
  *align = s == at::kFloat ? 4 : 8;
  return s == at::kFloat || s == at::kBFloat16 || s == at::kHalf;
}

bool aligned(const Tensor& t) { return ((uintptr_t)t.data_ptr() & 15) == 0; }

struct Call {
  at::Device device{at::kCUDA, 0};
  at::ScalarType dtype;
  int64_t align;
  ssl_paged_cache cache{};

  // The pools of one layer (4-D), or of several where `layers`.
  bool pools(PyObject* ko, PyObject* vo, bool layers) {
    const Tensor *k = tensor(ko), *v = tensor(vo);
    if (!k || !v || !dtype_of(*k, &cache.dtype, &align)) return false;
    dtype = k->scalar_type();
    device = k->device();
    const int64_t n = k->dim();
    if (v->scalar_type() != dtype || v->device() != device || (n != 4 && !(n == 5 && layers)) ||
        k->sizes() != v->sizes() || k->strides() != v->strides() || k->numel() == 0 ||
        !aligned(*k) || !aligned(*v) || k->stride(n - 1) != 1)
      return false;
    for (int64_t i = 0; i < n - 1; ++i)
      if (k->stride(i) % align) return false;
    cache.k = k->data_ptr();
    cache.v = v->data_ptr();
    cache.layer_stride = n == 5 ? k->stride(0) : 0;
    cache.layers = n == 5 ? k->size(0) : 1;
    cache.page_stride = k->stride(n - 4);
    cache.head_stride = k->stride(n - 3);
    cache.slot_stride = k->stride(n - 2);
    cache.pages = k->size(n - 4);
    cache.kv_heads = k->size(n - 3);
    cache.page = k->size(n - 2);
    cache.head_dim = k->size(n - 1);
    return true;
  }
  bool table(PyObject* o) {
    const Tensor* t = tensor(o);
    if (!t || t->scalar_type() != at::kInt || t->device() != device || t->dim() != 2 ||
        (t->stride(1) != 1 && t->size(1) > 1) || t->stride(0) < t->size(1))
      return false;
    cache.table = (const int32_t*)t->data_ptr();
    cache.seqs = t->size(0);
    cache.cols = t->size(1);
    cache.table_stride = cache.seqs > 1 ? t->stride(0) : cache.cols;
    return true;
  }
  // n contiguous int32, or null
  const int32_t* ints(PyObject* o, int64_t n) const {
    const Tensor* t = tensor(o);
    if (!t || t->scalar_type() != at::kInt || t->device() != device || t->dim() != 1 ||
        t->size(0) != n || !t->is_contiguous())
      return nullptr;
    return (const int32_t*)t->data_ptr();
  }
  // [n, heads, head_dim] in the pools' type with 16-byte rows
  bool rows(const Tensor* t, int64_t n, int64_t heads, const void** p, int64_t* token,
            int64_t* head) const {
    if (!t || t->scalar_type() != dtype || t->device() != device || t->dim() != 3 ||
        t->size(0) != n || t->size(1) != heads || t->size(2) != cache.head_dim ||
        t->stride(2) != 1 || t->stride(0) % align || t->stride(1) % align || !aligned(*t))
      return false;
    *p = t->data_ptr();
    *token = t->stride(0);
    *head = t->stride(1);
    return true;
  }
  Tensor empty(at::IntArrayRef size, at::ScalarType type) const {
    return at::empty(size, at::TensorOptions().dtype(type).device(device));
  }
  // Whether launches go to `device` as it is, with its current stream.
  bool stream(void** st) const {
    const c10::impl::VirtualGuardImpl guard(at::kCUDA);
    if (guard.getDevice().index() != device.index()) return false;
    PyObject* i = PyLong_FromLong(device.index());
    PyObject* r = i ? PyObject_CallOneArg(raw_stream, i) : nullptr;
    Py_XDECREF(i);
    if (!r) return false;
    *st = PyLong_AsVoidPtr(r);
    Py_DECREF(r);
    return !PyErr_Occurred();
  }
};

// None, after dropping an error met on the way: the Python function meets it too.
PyObject* not_taken() {
  PyErr_Clear();
  Py_RETURN_NONE;
}

bool integer(PyObject* o, int64_t* v) {
  if (!PyLong_Check(o)) return false;
  *v = PyLong_AsLongLong(o);
  return !(*v == -1 && PyErr_Occurred());
}

template <typename F, typename A>
int launch(F fn, const A& args, void* stream) {
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = fn(&args, stream);
  Py_END_ALLOW_THREADS
  return rc;
}

// C++ exceptions (an allocation that failed, say) end here; Python's own path
// raises them in torch's terms.
template <typename F>
PyObject* guarded(F f) {
  try {
    return f();
  } catch (...) {
    return not_taken();
  }
}

/* append(q, k, v, cos, sin, k_pool, v_pool, table, seqs, positions, q_norm, k_norm, eps) */
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    Call c;
    ssl_paged_append_args x{};
    const Tensor* q = n_args == 13 ? tensor(a[0]) : nullptr;
    if (!q || q->dim() != 3 || !c.pools(a[5], a[6], false) || !c.table(a[7])) return not_taken();
    const int64_t n = q->size(0), heads = q->size(1), kv = c.cache.kv_heads;
    if (n == 0 || !c.rows(q, n, heads, &x.q, &x.q_token, &x.q_head) ||
        !c.rows(tensor(a[1]), n, kv, &x.k, &x.k_token, &x.k_head) ||
        !c.rows(tensor(a[2]), n, kv, &x.v, &x.v_token, &x.v_head))
      return not_taken();
    const Tensor *cos = tensor(a[3]), *sin = tensor(a[4]);
    for (const Tensor* t : {cos, sin})
      if (!t || t->scalar_type() != at::kFloat || t->device() != c.device || t->dim() != 2 ||
          t->size(1) * 2 != c.cache.head_dim || t->stride(1) != 1 || t->stride(0) % 4 || !aligned(*t))
        return not_taken();
    if (cos->size(0) != sin->size(0)) return not_taken();
    x.cos = (const float*)cos->data_ptr();
    x.sin = (const float*)sin->data_ptr();
    x.cos_stride = cos->stride(0);
    x.sin_stride = sin->stride(0);
    x.angles = cos->size(0);
    const void** norms[2] = {&x.q_norm, &x.k_norm};
    for (int i = 0; i < 2; ++i) {
      if (a[10 + i] == Py_None) continue;
      const Tensor* w = tensor(a[10 + i]);
      if (!w || w->scalar_type() != c.dtype || w->device() != c.device || w->dim() != 1 ||
          w->size(0) != c.cache.head_dim || w->stride(0) != 1 || !aligned(*w))
        return not_taken();
      *norms[i] = w->data_ptr();
    }
    if (!PyFloat_Check(a[12])) return not_taken();
    x.eps = PyFloat_AS_DOUBLE(a[12]);
    x.seq_ids = c.ints(a[8], n);
    x.positions = c.ints(a[9], n);
    void* st;
    if (!x.seq_ids || !x.positions || !c.stream(&st)) return not_taken();
    Tensor out = c.empty({n, heads, c.cache.head_dim}, c.dtype);
    x.q_out = out.data_ptr();
    x.tokens = n;
    x.heads = heads;
    x.cache = c.cache;
    x.cache.bytes = sizeof x;
    if (int rc = launch(entry.append, x, st)) return PyLong_FromLong(rc);
    return THPVariable_Wrap(std::move(out));
  });
}

/* attention(q, k_pool, v_pool, table, lengths, cu, window, sinks, scale, max_tokens, max_length) */
PyObject* attention(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    Call c;
    ssl_paged_attention_args x{};
    const Tensor* q = n_args == 11 ? tensor(a[0]) : nullptr;
    if (!q || q->dim() != 3 || !c.pools(a[1], a[2], false) || !c.table(a[3])) return not_taken();
    const int64_t n = q->size(0), heads = q->size(1);
    if (n == 0 || heads == 0 || heads % c.cache.kv_heads ||
        !c.rows(q, n, heads, &x.q, &x.q_token, &x.q_head))
      return not_taken();
    x.lengths = c.ints(a[4], c.cache.seqs);
    if (!x.lengths) return not_taken();
    if (a[5] != Py_None) {
      x.cu = c.ints(a[5], c.cache.seqs + 1);
      if (!x.cu) return not_taken();
    } else if (n != c.cache.seqs) {
      return not_taken();
    }
    if (!integer(a[6], &x.window) || !integer(a[7], &x.sinks) || x.window < 0 || x.sinks < 0)
      return not_taken();
    if (a[8] == Py_None) x.scale = 1 / std::sqrt((double)c.cache.head_dim);
    else if (PyFloat_Check(a[8])) x.scale = PyFloat_AS_DOUBLE(a[8]);
    else return not_taken();
    const int64_t reach = c.cache.cols * c.cache.page;
    x.max_tokens = n;
    x.max_length = reach;
    if (a[9] != Py_None && !integer(a[9], &x.max_tokens)) return not_taken();
    if (a[10] != Py_None && !integer(a[10], &x.max_length)) return not_taken();
    if (x.max_tokens < 0 || x.max_length < 0) return not_taken();
    x.max_tokens = std::min(x.max_tokens, n);
    x.max_length = std::min(x.max_length, reach);
    void* st;
    if (!c.stream(&st)) return not_taken();
    Tensor out = c.empty({n, heads, c.cache.head_dim}, c.dtype), work;
    x.out = out.data_ptr();
    x.tokens = n;
    x.heads = heads;
    x.cache = c.cache;
    x.cache.bytes = sizeof x;
    x.workspace_bytes = entry.attention_bytes(&x);
    if (x.workspace_bytes) {
      work = c.empty({x.workspace_bytes}, at::kByte);
      x.workspace = work.data_ptr();
    }
    if (int rc = launch(entry.attention, x, st)) return PyLong_FromLong(rc);
    return THPVariable_Wrap(std::move(out));
  });
}

// Several outputs and a scratch in one allocation, each 256-byte aligned: four
// allocations take 2 µs of a call that takes 6. (One output kept keeps all of
// them.) allocate() takes the sum of their room()s; piece() and scratch() hand
// them out.
class Pieces {
 public:
  explicit Pieces(const Call& c) : call(c) {}
  static int64_t room(int64_t bytes) { return (bytes + 255) / 256 * 256; }
  void allocate(int64_t bytes) { block = call.empty({std::max<int64_t>(bytes, 1)}, at::kByte); }
  Tensor piece(at::IntArrayRef size, at::ScalarType type) {
    const int64_t item = (int64_t)c10::elementSize(type);
    Tensor t = at::detail::make_tensor<c10::TensorImpl>(
        c10::Storage(block.storage()), c10::DispatchKeySet(c10::DispatchKey::CUDA),
        c10::scalarTypeToTypeMeta(type));
    c10::TensorImpl* impl = t.unsafeGetTensorImpl();
    impl->set_sizes_contiguous(size);
    impl->set_storage_offset(at / item);
    at += room(t.numel() * item);
    return t;
  }
  void* scratch(int64_t bytes) {
    void* p = (char*)block.data_ptr() + at;
    at += room(bytes);
    return p;
  }

 private:
  const Call& call;
  Tensor block;
  int64_t at = 0;
};

PyObject* tuple_of(std::initializer_list<Tensor> ts) {
  PyObject* r = PyTuple_New((Py_ssize_t)ts.size());
  Py_ssize_t i = 0;
  for (const Tensor& t : ts) {
    PyObject* o = r ? THPVariable_Wrap(t) : nullptr;
    if (!o) {
      Py_XDECREF(r);
      return nullptr;
    }
    PyTuple_SET_ITEM(r, i++, o);
  }
  return r;
}

// The reference counts [pages], or null.
const Tensor* counts(PyObject* o, const Call& c) {
  const Tensor* t = tensor(o);
  if (!t || t->scalar_type() != at::kInt || t->device() != c.device || t->dim() != 1 ||
      t->size(0) == 0 || !t->is_contiguous())
    return nullptr;
  return t;
}

/* free(table, lengths, refs, seqs) */
PyObject* free_pages(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    Call c;
    ssl_pages_args x{};
    const Tensor *t = n_args == 4 ? tensor(a[0]) : nullptr, *s = t ? tensor(a[3]) : nullptr;
    if (!t || !s || s->dim() != 1) return not_taken();
    c.device = t->device();
    const Tensor* refs = counts(a[2], c);
    if (!refs || !c.table(a[0])) return not_taken();
    x.lengths = c.ints(a[1], c.cache.seqs);
    x.n = s->size(0);
    x.dst = c.ints(a[3], x.n);
    void* st;
    if (!x.lengths || !x.dst || !c.stream(&st)) return not_taken();
    Pieces out(c);
    out.allocate(Pieces::room(4 * c.cache.seqs * c.cache.cols) + Pieces::room(4 * c.cache.seqs) +
                 Pieces::room(4 * refs->size(0)));
    Tensor table = out.piece({c.cache.seqs, c.cache.cols}, at::kInt);
    Tensor lengths = out.piece({c.cache.seqs}, at::kInt);
    Tensor refs_out = out.piece({refs->size(0)}, at::kInt);
    x.refs = (const int32_t*)refs->data_ptr();
    x.table_out = (int32_t*)table.data_ptr();
    x.lengths_out = (int32_t*)lengths.data_ptr();
    x.refs_out = (int32_t*)refs_out.data_ptr();
    x.cache = c.cache;
    x.cache.bytes = sizeof x;
    x.cache.pages = refs->size(0);
    x.cache.layers = x.cache.kv_heads = 1;
    x.cache.page = 16;
    x.cache.head_dim = 64;
    if (int rc = launch(entry.free, x, st)) return PyLong_FromLong(rc);
    return tuple_of({table, lengths, refs_out});
  });
}

/* fork(table, lengths, refs, k_pool, v_pool, src, dst) */
PyObject* fork_pages(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    Call c;
    ssl_pages_args x{};
    if (n_args != 7 || !c.pools(a[3], a[4], true) || !c.table(a[0])) return not_taken();
    const Tensor *refs = counts(a[2], c), *s = tensor(a[5]);
    if (!refs || refs->size(0) != c.cache.pages || !s || s->dim() != 1) return not_taken();
    x.n = s->size(0);
    x.lengths = c.ints(a[1], c.cache.seqs);
    x.src = c.ints(a[5], x.n);
    x.dst = c.ints(a[6], x.n);
    void* st;
    if (!x.lengths || !x.src || !x.dst || !c.stream(&st)) return not_taken();
    x.workspace_bytes = entry.fork_bytes(x.n);
    Pieces out(c);
    out.allocate(Pieces::room(4 * c.cache.seqs * c.cache.cols) + Pieces::room(4 * c.cache.seqs) +
                 Pieces::room(4 * c.cache.pages) + Pieces::room(x.n) +
                 Pieces::room(x.workspace_bytes));
    Tensor table = out.piece({c.cache.seqs, c.cache.cols}, at::kInt);
    Tensor lengths = out.piece({c.cache.seqs}, at::kInt);
    Tensor refs_out = out.piece({c.cache.pages}, at::kInt);
    Tensor ok = out.piece({x.n}, at::kBool);
    x.refs = (const int32_t*)refs->data_ptr();
    x.table_out = (int32_t*)table.data_ptr();
    x.lengths_out = (int32_t*)lengths.data_ptr();
    x.refs_out = (int32_t*)refs_out.data_ptr();
    x.ok = (uint8_t*)ok.data_ptr();
    x.workspace = out.scratch(x.workspace_bytes);
    x.cache = c.cache;
    x.cache.bytes = sizeof x;
    if (int rc = launch(entry.fork, x, st)) return PyLong_FromLong(rc);
    return tuple_of({table, lengths, refs_out, ok});
  });
}

/* compact(table, refs, k_pool, v_pool) */
PyObject* compact_pages(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    Call c;
    ssl_pages_args x{};
    if (n_args != 4 || !c.pools(a[2], a[3], true) || !c.table(a[0])) return not_taken();
    const Tensor* refs = counts(a[1], c);
    void* st;
    if (!refs || refs->size(0) != c.cache.pages || !c.stream(&st)) return not_taken();
    x.workspace_bytes = entry.compact_bytes(c.cache.pages);
    Pieces out(c);
    out.allocate(Pieces::room(4 * c.cache.seqs * c.cache.cols) + Pieces::room(4 * c.cache.pages) +
                 Pieces::room(4) + Pieces::room(x.workspace_bytes));
    Tensor table = out.piece({c.cache.seqs, c.cache.cols}, at::kInt);
    Tensor refs_out = out.piece({c.cache.pages}, at::kInt), live = out.piece({}, at::kInt);
    x.refs = (const int32_t*)refs->data_ptr();
    x.table_out = (int32_t*)table.data_ptr();
    x.refs_out = (int32_t*)refs_out.data_ptr();
    x.live_out = (int32_t*)live.data_ptr();
    x.workspace = out.scratch(x.workspace_bytes);
    x.cache = c.cache;
    x.cache.bytes = sizeof x;
    if (int rc = launch(entry.compact, x, st)) return PyLong_FromLong(rc);
    return tuple_of({table, refs_out, live});
  });
}

/* logprobs(logits, tokens, top) */
PyObject* logprobs(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    Call c;
    ssl_token_logprobs_args x{};
    const Tensor *t = n_args == 3 ? tensor(a[0]) : nullptr, *tok = t ? tensor(a[1]) : nullptr;
    int64_t align;
    if (!t || !tok || t->dim() != 2 || !dtype_of(*t, &x.dtype, &align) || !integer(a[2], &x.top))
      return not_taken();
    x.rows = t->size(0);
    x.vocab = t->size(1);
    c.device = t->device();
    if (x.rows == 0 || x.vocab == 0 || t->stride(1) != 1 || (x.rows > 1 && t->stride(0) < x.vocab) ||
        tok->scalar_type() != at::kLong || tok->device() != c.device || tok->dim() != 1 ||
        tok->size(0) != x.rows || !tok->is_contiguous() || x.top < 0 ||
        x.top > std::min<int64_t>(x.vocab, 64))
      return not_taken();
    void* st;
    if (!c.stream(&st)) return not_taken();
    Pieces out(c);
    out.allocate(2 * Pieces::room(4 * x.rows) + Pieces::room(8 * x.rows * x.top) +
                 Pieces::room(4 * x.rows * x.top));
    Tensor logprob = out.piece({x.rows}, at::kFloat), entropy = out.piece({x.rows}, at::kFloat);
    Tensor ids = out.piece({x.rows, x.top}, at::kLong), top = out.piece({x.rows, x.top}, at::kFloat);
    x.bytes = sizeof x;
    x.logits = t->data_ptr();
    x.ld = x.rows > 1 ? t->stride(0) : x.vocab;
    x.tokens = (const int64_t*)tok->data_ptr();
    x.logprob = (float*)logprob.data_ptr();
    x.entropy = (float*)entropy.data_ptr();
    x.top_ids = (int64_t*)ids.data_ptr();
    x.top_logprobs = (float*)top.data_ptr();
    if (int rc = launch(entry.logprobs, x, st)) return PyLong_FromLong(rc);
    return tuple_of({logprob, entropy, ids, top});
  });
}

/* bind(raw_stream, nine addresses in the order of `entry`) */
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  if (n_args != 10) {
    PyErr_SetString(PyExc_TypeError, "bind takes the raw stream function and nine addresses");
    return nullptr;
  }
  void* p[9];
  for (int i = 0; i < 9; ++i) {
    p[i] = PyLong_AsVoidPtr(a[i + 1]);
    if (PyErr_Occurred()) return nullptr;
    if (!p[i]) {
      PyErr_SetString(PyExc_ValueError, "bind: a null address");
      return nullptr;
    }
  }
  static_assert(sizeof entry == sizeof p, "one address an entry point");
  memcpy(&entry, p, sizeof p);
  Py_INCREF(a[0]);
  Py_XSETREF(raw_stream, a[0]);
  Py_RETURN_NONE;
}

#define SSL_METHOD(name, fn) \
  {name, (PyCFunction)(void (*)(void))fn, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {
    SSL_METHOD("bind", bind),           SSL_METHOD("append", append),
    SSL_METHOD("attention", attention), SSL_METHOD("free", free_pages),
    SSL_METHOD("fork", fork_pages),     SSL_METHOD("compact", compact_pages),
    SSL_METHOD("logprobs", logprobs),   {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "tensorcall", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit_tensorcall(void) { return PyModule_Create(&module); }
