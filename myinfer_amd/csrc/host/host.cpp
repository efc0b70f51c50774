// The host path of one attention layer's step, over torch tensors: the checks, the descriptors, the output
// and the foreign call of kernels.prepare_attention and AppendCall for the forms a model's layers use, and
// the views QuantizedKVCache.fetch returns; and of a drafted step's calls: the tree, its attention, the append at
// positions, reading rows back and keeping the accepted ones.
//
// In Python the two calls of a decode step cost about 45 us of host time, three times their kernels' time
// on a 4096-token cache of 8 heads; here about 10. A drafted step's calls, in Python and here,
// us: a tree of 10 nodes and its attention 40.6 / 18.4, sixteen tokens written at positions and read back 45.1 / 15.2, the
// accepted rows of 32 layers 216 / 24, one token's queries rotated 8.8 / 5.4. Every function returns None for anything but those
// forms (other types, devices, strides, a call the library refuses): the Python path then serves the call
// or raises, so that what is accepted and what is refused has one definition. A launch that failed is not
// tried again: the Python side gets its (negative) status to raise. The interpreter lock is released
// around the library's calls, which may wait for room in a full queue.

#include <ATen/ATen.h>
#include <string.h>

#include <algorithm>
#include <initializer_list>
#include <type_traits>
#include <vector>

#include <torch/csrc/autograd/python_variable.h>
#include <torch/version.h>

#include "../../../include/kvq.h"

namespace {

using AttnFn = int (*)(const kvq_rows*, const kvq_qtensor*, const kvq_qtensor*, const int32_t*, const kvq_rows*, int, int,
                       int, int, int, int, int, int, int, float, int, int, void*, size_t, void*);
using SizeFn = size_t (*)(int, int, int, int, int, int, int);
using AppendFn = int (*)(const kvq_rows*, const kvq_qtensor*, const kvq_rows*, const kvq_qtensor*, int64_t, int, int, int,
                         int, int, int, int, void*);
using RopeAppendFn = int (*)(const kvq_rows*, const kvq_qtensor*, const kvq_rows*, const kvq_qtensor*,
                             const kvq_rope_params*, int64_t, int, int, int, int, int, int, int, void*);

struct {
  AttnFn decode = nullptr, prefill = nullptr;
  SizeFn decode_ws = nullptr, prefill_ws = nullptr;
} g;

// The entry points of a drafted step (bind_draft).
struct {
  decltype(&kvq_draft_tree) draft_tree = nullptr;
  decltype(&kvq_tree_attn) tree = nullptr;
  decltype(&kvq_tree_attn_dense) tree_dense = nullptr;
  decltype(&kvq_paged_tree_attn) tree_paged = nullptr;
  decltype(&kvq_tree_workspace_size) tree_ws = nullptr;
  decltype(&kvq_tree_kernel) tree_kernel = nullptr;
  decltype(&kvq_rope_axes) rope_axes = nullptr;
  decltype(&kvq_rope_axes_append) axes_append = nullptr;
  decltype(&kvq_dequantize) dequantize = nullptr;
  decltype(&kvq_paged_dequantize) paged_dequantize = nullptr;
  decltype(&kvq_keep_rows) keep_rows = nullptr;
} d;

// The destination of an AppendCall (myinfer_amd/_lib.py, AppendState).
struct AppendState {
  void* fn;
  const kvq_qtensor *kq, *vq;
  const void* rope;  // kvq_rope_params, kvq_axes (of an AxesAppendCall, whose fn and stream are not read) or NULL
  int64_t B, H, rows, code_words, groups;
  int32_t bits, group, code, device;
  void* stream;
};

PyObject* none() { Py_RETURN_NONE; }

// What a library call that did not return KVQ_OK becomes: see above. (Nothing was launched by a refused one.)
PyObject* failed(int rc) {
  if (rc == KVQ_ERR_HIP) return PyLong_FromLong(rc);
  return none();
}

// Releases the interpreter lock while it lives.
struct Unlocked {
  PyThreadState* st = PyEval_SaveThread();
  ~Unlocked() { PyEval_RestoreThread(st); }
};

int dtype_code(at::ScalarType t) {
  return t == at::kHalf ? KVQ_DTYPE_F16 : t == at::kBFloat16 ? KVQ_DTYPE_BF16 : -1;
}

// Rows that the kernels read in place: 4-D, unit stride along D, 16-byte aligned, strides of 8 elements.
bool rows_of(const at::Tensor& t, kvq_rows* r) {
  if (t.dim() != 4 || t.stride(3) != 1) return false;
  *r = {t.data_ptr(), t.stride(0), t.stride(1), t.stride(2)};
  return !(((uintptr_t)r->data | 2 * (uintptr_t)(r->stride_b | r->stride_h | r->stride_l)) % 16);
}

struct Triple {
  at::Tensor c, s, b;
};
bool triple_of(PyObject* o, Triple* t) {
  if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 3) return false;
  PyObject* const* x = &PyTuple_GET_ITEM(o, 0);
  if (!THPVariable_Check(x[0]) || !THPVariable_Check(x[1]) || !THPVariable_Check(x[2])) return false;
  t->c = THPVariable_Unpack(x[0]);
  t->s = THPVariable_Unpack(x[1]);
  t->b = THPVariable_Unpack(x[2]);
  return true;
}
bool qtensor_of(const Triple& t, int64_t B, int64_t Hkv, int64_t S, int64_t D, int bits, int group, at::ScalarType dt,
                const at::Device& dev, int32_t* range_exp, kvq_qtensor* q) {
  const auto& c = t.c;
  if (c.dim() != 4 || t.s.dim() != 4 || t.b.dim() != 4) return false;
  if ((c.scalar_type() != at::kUInt32 && c.scalar_type() != at::kInt) || t.s.scalar_type() != dt ||
      t.b.scalar_type() != dt)
    return false;
  if (c.device() != dev || t.s.device() != dev || t.b.device() != dev) return false;
  if (c.size(0) != B || c.size(1) != Hkv || c.size(2) != S || c.size(3) * 32 != D * bits) return false;
  if (t.s.size(0) != B || t.s.size(1) != Hkv || t.s.size(2) != S || t.s.size(3) * group != D) return false;
  if (t.s.sizes() != t.b.sizes() || t.s.strides() != t.b.strides()) return false;
  if (c.stride(3) != 1 || t.s.stride(3) != 1) return false;
  *q = {(uint32_t*)c.data_ptr(), t.s.data_ptr(), t.b.data_ptr(), c.stride(0), c.stride(1), c.stride(2),
        t.s.stride(0), t.s.stride(1), t.s.stride(2), range_exp};
  return true;
}

// attention(queries, keys, values, scale, causal, window, seq_lens, group_size, bits, prefill, k_range, v_range,
//           workspace, stream) -> the output, the workspace bytes needed if the given ones are too few, the negative
//           status of a failed launch, or None
PyObject* attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 14 || !g.decode || !THPVariable_Check(a[0])) return none();
  try {
    const at::Tensor& q = THPVariable_Unpack(a[0]);
    Triple k, v;
    if (!triple_of(a[1], &k) || !triple_of(a[2], &v)) return none();
    const double scale = PyFloat_AsDouble(a[3]);
    const long causal = PyLong_AsLong(a[4]), window = PyLong_AsLong(a[5]);
    const long group = PyLong_AsLong(a[7]), bits = PyLong_AsLong(a[8]), prefill = PyLong_AsLong(a[9]);
    void* kw = PyLong_AsVoidPtr(a[10]);
    void* vw = PyLong_AsVoidPtr(a[11]);
    void* stream = PyLong_AsVoidPtr(a[13]);
    if (PyErr_Occurred()) {
      PyErr_Clear();
      return none();
    }
    kvq_rows qr;
    const int code = dtype_code(q.scalar_type());
    if (code < 0 || !q.is_cuda() || !rows_of(q, &qr) || (bits != 4 && bits != 8) || group <= 0 || window < 0) return none();
    const int64_t B = q.size(0), Hq = q.size(1), L = q.size(2), D = q.size(3);
    if (k.c.dim() != 4) return none();
    const int64_t Hkv = k.c.size(1), S = k.c.size(2);
    if (B <= 0 || Hkv <= 0 || L <= 0 || S <= 0 || Hq % Hkv || Hq <= 0) return none();
    if (B > INT32_MAX || Hq > INT32_MAX || L > INT32_MAX || S > INT32_MAX || window > INT32_MAX) return none();
    kvq_qtensor kq, vq;
    const at::Device dev = q.device();
    if (!qtensor_of(k, B, Hkv, S, D, bits, group, q.scalar_type(), dev, (int32_t*)kw, &kq) ||
        !qtensor_of(v, B, Hkv, S, D, bits, group, q.scalar_type(), dev, (int32_t*)vw, &vq))
      return none();
    const int32_t* lens = nullptr;
    if (a[6] != Py_None) {
      if (!THPVariable_Check(a[6])) return none();
      const at::Tensor& t = THPVariable_Unpack(a[6]);
      if (t.scalar_type() != at::kInt || t.device() != dev || t.numel() != B || !t.is_contiguous()) return none();
      lens = (const int32_t*)t.data_ptr();
    }
    const size_t need = (prefill ? g.prefill_ws : g.decode_ws)((int)B, (int)Hq, (int)Hkv, (int)L, (int)D, (int)S, (int)window);
    if (need == 0) return none();
    if (!THPVariable_Check(a[12])) return PyLong_FromSize_t(need);
    const at::Tensor& ws = THPVariable_Unpack(a[12]);
    if (ws.nbytes() < need) return PyLong_FromSize_t(need);
    at::Tensor out = at::empty({B, Hq, L, D}, q.options().requires_grad(false));
    const kvq_rows orr = {out.data_ptr(), Hq * L * D, L * D, D};
    void* const wp = ws.data_ptr();
    const size_t wn = ws.nbytes();
    int rc;
    {
      Unlocked u;
      rc = (prefill ? g.prefill : g.decode)(&qr, &kq, &vq, lens, &orr, (int)B, (int)Hq, (int)Hkv, (int)L, (int)D, (int)S,
                                            (int)bits, (int)group, code, (float)scale, (int)causal, (int)window, wp, wn,
                                            stream);
    }
    if (rc != KVQ_OK) return failed(rc);
    return THPVariable_Wrap(std::move(out));
  } catch (...) {
    return none();
  }
}

// append(state address, keys, values, row_offset, rope_offset) -> True, the negative status of a failed launch, or None
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 5 || !THPVariable_Check(a[1]) || !THPVariable_Check(a[2])) return none();
  try {
    const AppendState* st = (const AppendState*)PyLong_AsVoidPtr(a[0]);
    const long long row = PyLong_AsLongLong(a[3]), pos = PyLong_AsLongLong(a[4]);
    if (PyErr_Occurred() || !st) {
      PyErr_Clear();
      return none();
    }
    const at::Tensor &k = THPVariable_Unpack(a[1]), &v = THPVariable_Unpack(a[2]);
    if (!k.is_cuda() || !v.is_cuda() || k.get_device() != st->device || v.get_device() != st->device) return none();
    if (dtype_code(k.scalar_type()) != st->code || v.scalar_type() != k.scalar_type() || !st->vq) return none();
    kvq_rows kr, vr;
    if (!rows_of(k, &kr) || !rows_of(v, &vr) || k.sizes() != v.sizes()) return none();
    const int64_t L = k.size(2), D = k.size(3);
    if (k.size(0) != st->B || k.size(1) != st->H || row < 0 || row + L > st->rows || L > INT32_MAX) return none();
    if (D * st->bits / 32 != st->code_words || D / st->group != st->groups) return none();
    int rc;
    {
      Unlocked u;
      if (st->rope) {
        kvq_rope_params rp = *(const kvq_rope_params*)st->rope;
        rp.offset = pos;
        rc = ((RopeAppendFn)st->fn)(&kr, st->kq, &vr, st->vq, &rp, row, (int)st->B, (int)st->H, (int)L, (int)D, st->bits,
                                    st->group, st->code, st->stream);
      } else {
        rc = ((AppendFn)st->fn)(&kr, st->kq, &vr, st->vq, row, (int)st->B, (int)st->H, (int)L, (int)D, st->bits, st->group,
                                st->code, st->stream);
      }
    }
    if (rc != KVQ_OK) return failed(rc);
    Py_RETURN_TRUE;
  } catch (...) {
    return none();
  }
}

// views(keys, values, rows) -> the triples' first `rows` rows, as x[..., :rows, :] of each, or None
PyObject* views(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 3) return none();
  try {
    const long long rows = PyLong_AsLongLong(a[2]);
    if (PyErr_Occurred()) {
      PyErr_Clear();
      return none();
    }
    Triple t[2];
    if (!triple_of(a[0], &t[0]) || !triple_of(a[1], &t[1])) return none();
    PyObject* both = PyTuple_New(2);
    for (int i = 0; i < 2; ++i) {
      PyObject* tr = PyTuple_New(3);
      PyTuple_SET_ITEM(both, i, tr);
      const at::Tensor* x[3] = {&t[i].c, &t[i].s, &t[i].b};
      for (int j = 0; j < 3; ++j) {
        if (x[j]->dim() < 2 || rows < 0 || rows > x[j]->size(-2)) {
          Py_DECREF(both);
          return none();
        }
        c10::SmallVector<int64_t, 8> size(x[j]->sizes().begin(), x[j]->sizes().end());
        size[size.size() - 2] = rows;
        PyTuple_SET_ITEM(tr, j, THPVariable_Wrap(x[j]->as_strided(size, x[j]->strides(), x[j]->storage_offset())));
      }
    }
    return both;
  } catch (...) {
    return none();
  }
}

// ---- a drafted step

// An int32 tensor of `n` contiguous entries on `dev`: its data, or NULL.
const int32_t* ints_of(PyObject* o, int64_t n, const at::Device& dev) {
  if (!THPVariable_Check(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (t.scalar_type() != at::kInt || t.device() != dev || t.dim() != 1 || t.numel() != n || !t.is_contiguous()) return nullptr;
  return (const int32_t*)t.data_ptr();
}

// A block table [B, pages] on `dev` whose rows follow each other.
bool table_of(PyObject* o, int64_t B, const at::Device& dev, const int32_t** data, int64_t* stride, int64_t* pages) {
  if (!THPVariable_Check(o)) return false;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (t.scalar_type() != at::kInt || t.device() != dev || t.dim() != 2 || t.size(0) != B || !t.is_contiguous()) return false;
  *data = (const int32_t*)t.data_ptr();
  *stride = *pages = t.size(1);
  return true;
}

// int32 positions [axes, B, L] or [axes, L] into a descriptor.
bool positions_of(PyObject* o, int64_t B, int64_t L, const at::Device& dev, kvq_axes* ax) {
  if (!THPVariable_Check(o)) return false;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (t.scalar_type() != at::kInt || t.device() != dev || t.dim() < 2 || t.dim() > 3) return false;
  const bool shared = t.dim() == 2;
  if (t.size(0) != ax->axes || t.size(-1) != L || (!shared && t.size(1) != B)) return false;
  ax->positions = (const int32_t*)t.data_ptr();
  ax->pos_stride_a = t.stride(0);
  ax->pos_stride_b = shared ? 0 : t.stride(1);
  ax->pos_stride_l = t.stride(-1);
  return true;
}

// The range word registered for a codes buffer (kernels._range_words: storage address -> (weak reference to the buffer,
// word)), or NULL.
int32_t* word_of(PyObject* words, const at::Tensor& codes) {
  const void* at = codes.storage().data();
  PyObject* key = PyLong_FromVoidPtr((void*)at);
  PyObject* hit = key ? PyDict_GetItem(words, key) : nullptr;
  Py_XDECREF(key);
  if (!hit || !PyTuple_Check(hit) || PyTuple_GET_SIZE(hit) != 2) return nullptr;
  PyObject* buf = PyWeakref_GetObject(PyTuple_GET_ITEM(hit, 0));
  PyObject* word = PyTuple_GET_ITEM(hit, 1);
  if (!buf || !THPVariable_Check(buf) || !THPVariable_Check(word)) return nullptr;
  if (THPVariable_Unpack(buf).storage().data() != at) return nullptr;
  return (int32_t*)THPVariable_Unpack(word).data_ptr();
}

bool fits_int(std::initializer_list<int64_t> v) {
  for (int64_t x : v)
    if (x < 0 || x > INT32_MAX) return false;
  return true;
}

// draft_tree(parents, starts: None, int or tensor, stream) -> int32 buffer: the bits [B][L][words], the depths [B][L] and,
// with starts, the positions [B][L]; the negative status of a failed launch, or None
PyObject* draft_tree(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 3 || !d.draft_tree || !THPVariable_Check(a[0])) return none();
  try {
    const at::Tensor& p = THPVariable_Unpack(a[0]);
    void* stream = PyLong_AsVoidPtr(a[2]);
    int64_t start = 0;
    const int32_t* starts = nullptr;
    if (!p.is_cuda() || p.scalar_type() != at::kInt || p.dim() < 1 || p.dim() > 2) return none();
    const bool shared = p.dim() == 1;
    const int64_t B = shared ? 1 : p.size(0), L = p.size(-1);
    if (L < 1 || L > KVQ_TREE_MAX_NODES || !fits_int({B}) || (p.stride(-1) != 1 && L > 1)) return none();
    if (PyLong_Check(a[1])) {
      start = PyLong_AsLongLong(a[1]);
      if (start < INT32_MIN || start >= (int64_t)INT32_MAX + 1 - L) return none();
    } else if (a[1] != Py_None && !(starts = ints_of(a[1], B, p.device()))) {
      return none();
    }
    if (PyErr_Occurred()) {
      PyErr_Clear();
      return none();
    }
    const int64_t words = (L + 31) / 32, nodes = B * L;
    at::Tensor buf = at::empty({nodes * (words + (a[1] == Py_None ? 1 : 2))}, p.options().requires_grad(false));
    uint32_t* bits = (uint32_t*)buf.data_ptr();
    int32_t* depths = (int32_t*)bits + nodes * words;
    int rc;
    {
      Unlocked u;
      rc = d.draft_tree((const int32_t*)p.data_ptr(), shared ? 0 : p.stride(0), (int)B, (int)L, bits, depths, starts, start,
                        a[1] == Py_None ? nullptr : depths + nodes, stream);
    }
    if (rc != KVQ_OK) return failed(rc);
    return THPVariable_Wrap(std::move(buf));
  } catch (...) {
    PyErr_Clear();
    return none();
  }
}

// tree_attention(queries, keys, values, scale, window, seq_lens, group_size, bits, range words, workspace, stream, tree
//                buffer, trees (0: one for the batch), nodes, block table or None, max_len) -> as attention()
PyObject* tree_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 16 || !d.tree || !THPVariable_Check(a[0]) || !THPVariable_Check(a[11]) || !PyDict_Check(a[8])) return none();
  try {
    const at::Tensor& q = THPVariable_Unpack(a[0]);
    const double scale = PyFloat_AsDouble(a[3]);
    const long window = PyLong_AsLong(a[4]), group = PyLong_AsLong(a[6]), bits = PyLong_AsLong(a[7]);
    void* stream = PyLong_AsVoidPtr(a[10]);
    const long trees = PyLong_AsLong(a[12]), nodes = PyLong_AsLong(a[13]), max_len = PyLong_AsLong(a[15]);
    if (PyErr_Occurred()) {
      PyErr_Clear();
      return none();
    }
    kvq_rows qr;
    const int code = dtype_code(q.scalar_type());
    if (code < 0 || !q.is_cuda() || !rows_of(q, &qr)) return none();
    const int64_t B = q.size(0), Hq = q.size(1), L = q.size(2), D = q.size(3);
    const at::Device dev = q.device();
    const at::Tensor& tb = THPVariable_Unpack(a[11]);
    const int64_t words = (L + 31) / 32;
    if (B <= 0 || Hq <= 0 || L != nodes || (trees && trees != B) || tb.device() != dev || window < 0 || window > INT32_MAX)
      return none();
    kvq_tree tree;
    tree.bits = (const uint32_t*)tb.data_ptr();
    tree.depths = (const int32_t*)tree.bits + (trees ? B : 1) * L * words;
    tree.bits_stride_b = trees ? L * words : 0;
    tree.depths_stride_b = trees ? L : 0;
    const bool dense = THPVariable_Check(a[1]), paged = a[14] != Py_None;
    int64_t Hkv, S, table_stride = 0, pages = 0, num_pages = 0;
    const int32_t *lens = nullptr, *table = nullptr;
    kvq_rows kr, vr;
    kvq_qtensor kq, vq;
    if (dense) {
      if (paged || !THPVariable_Check(a[2])) return none();
      const at::Tensor &k = THPVariable_Unpack(a[1]), &v = THPVariable_Unpack(a[2]);
      if (!rows_of(k, &kr) || !rows_of(v, &vr) || k.sizes() != v.sizes()) return none();
      if (k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type() || k.device() != dev || v.device() != dev)
        return none();
      Hkv = k.size(1), S = k.size(2);
      if (k.size(0) != B || k.size(3) != D) return none();
    } else {
      Triple k, v;
      if (!triple_of(a[1], &k) || !triple_of(a[2], &v) || k.c.dim() != 4) return none();
      if ((bits != 4 && bits != 8) || (group != 32 && group != 64 && group != 128)) return none();
      Hkv = k.c.size(1), S = k.c.size(2);
      int64_t lead = B, rows = S;
      if (paged) {
        if (S != KVQ_PAGE_ROWS || !table_of(a[14], B, dev, &table, &table_stride, &pages)) return none();
        num_pages = lead = k.c.size(0);
        S = max_len >= 0 ? max_len : pages * KVQ_PAGE_ROWS;
      }
      const bool bf = code == KVQ_DTYPE_BF16;  // (the range words, which only bf16 caches need)
      int32_t* kw = bf ? word_of(a[8], k.c) : nullptr;
      int32_t* vw = bf ? word_of(a[8], v.c) : nullptr;
      if (!qtensor_of(k, lead, Hkv, rows, D, (int)bits, (int)group, q.scalar_type(), dev, kw, &kq) ||
          !qtensor_of(v, lead, Hkv, rows, D, (int)bits, (int)group, q.scalar_type(), dev, vw, &vq))
        return none();
    }
    if (Hkv <= 0 || Hq % Hkv || S < L || !fits_int({B, Hq, S, num_pages})) return none();
    if (a[5] != Py_None && !(lens = ints_of(a[5], B, dev))) return none();
    if (paged && !lens) return none();
    const int b = (int)B, hq = (int)Hq, hk = (int)Hkv, l = (int)L, dd = (int)D, s = (int)S, w = (int)window;
    if (!dense && !paged && code == KVQ_DTYPE_BF16 && (!kq.range_exp || !vq.range_exp) &&
        d.tree_kernel(b, hq, hk, l, dd, s, (int)bits, (int)group, w) == KVQ_TREE_PREFILL)
      return none();  // (its exponents are computed)
    const size_t need = d.tree_ws(b, hq, hk, l, dd, s, w);
    if (need == 0) return none();
    if (!THPVariable_Check(a[9])) return PyLong_FromSize_t(need);
    const at::Tensor& ws = THPVariable_Unpack(a[9]);
    if (ws.nbytes() < need) return PyLong_FromSize_t(need);
    at::Tensor out = at::empty({B, Hq, L, D}, q.options().requires_grad(false));
    const kvq_rows orr = {out.data_ptr(), Hq * L * D, L * D, D};
    void* const wp = ws.data_ptr();
    const size_t wn = ws.nbytes();
    const float sc = (float)scale;
    int rc;
    {
      Unlocked u;
      if (dense) {
        rc = d.tree_dense(&qr, &kr, &vr, lens, &orr, b, hq, hk, l, dd, s, code, sc, &tree, w, wp, wn, stream);
      } else if (paged) {
        rc = d.tree_paged(&qr, &kq, &vq, (int)num_pages, table, table_stride, lens, &orr, b, hq, hk, l, dd, s, (int)bits,
                          (int)group, code, sc, &tree, w, wp, wn, stream);
      } else {
        rc = d.tree(&qr, &kq, &vq, lens, &orr, b, hq, hk, l, dd, s, (int)bits, (int)group, code, sc, &tree, w, wp, wn, stream);
      }
    }
    if (rc != KVQ_OK) return failed(rc);
    return THPVariable_Wrap(std::move(out));
  } catch (...) {
    PyErr_Clear();
    return none();
  }
}

// rope_axes(descriptor address, x, positions, stream) -> True, the negative status of a failed launch, or None
PyObject* rope_axes(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 4 || !d.rope_axes || !THPVariable_Check(a[1])) return none();
  try {
    const kvq_axes* desc = (const kvq_axes*)PyLong_AsVoidPtr(a[0]);
    void* stream = PyLong_AsVoidPtr(a[3]);
    if (PyErr_Occurred() || !desc) {
      PyErr_Clear();
      return none();
    }
    const at::Tensor& x = THPVariable_Unpack(a[1]);
    const int code = dtype_code(x.scalar_type());
    kvq_rows xr;
    if (code < 0 || !x.is_cuda() || x.numel() == 0 || !rows_of(x, &xr)) return none();
    kvq_axes ax = *desc;
    const int64_t B = x.size(0), H = x.size(1), L = x.size(2), D = x.size(3);
    if (!fits_int({B, H, L, D}) || !positions_of(a[2], B, L, x.device(), &ax)) return none();
    int rc;
    {
      Unlocked u;
      rc = d.rope_axes(&xr, &ax, (int)B, (int)H, (int)L, (int)D, code, stream);
    }
    if (rc != KVQ_OK) return failed(rc);
    Py_RETURN_TRUE;
  } catch (...) {
    PyErr_Clear();
    return none();
  }
}

// axes_append(state address, keys, values, positions, row_offset, queries or None, stream, block table or None, starts or
// None) -> as append(); with a block table the state's destination is a pool (B: its pages, rows: a page's)
PyObject* axes_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 9 || !d.axes_append || !THPVariable_Check(a[1]) || !THPVariable_Check(a[2])) return none();
  try {
    const AppendState* st = (const AppendState*)PyLong_AsVoidPtr(a[0]);
    const long long row = PyLong_AsLongLong(a[4]);
    void* stream = PyLong_AsVoidPtr(a[6]);
    if (PyErr_Occurred() || !st) {
      PyErr_Clear();
      return none();
    }
    const at::Tensor &k = THPVariable_Unpack(a[1]), &v = THPVariable_Unpack(a[2]);
    if (!k.is_cuda() || !v.is_cuda() || k.get_device() != st->device || v.get_device() != st->device) return none();
    if (dtype_code(k.scalar_type()) != st->code || v.scalar_type() != k.scalar_type() || !st->vq) return none();
    kvq_rows kr, vr, qr;
    if (k.numel() == 0 || !rows_of(k, &kr) || !rows_of(v, &vr) || k.sizes() != v.sizes()) return none();
    const int64_t B = k.size(0), L = k.size(2), D = k.size(3);
    const bool paged = a[7] != Py_None;
    int64_t table_stride = 0, pages = 0;
    const int32_t *table = nullptr, *starts = nullptr;
    if (k.size(1) != st->H || row < 0 || !fits_int({B, L}) || (!paged && (B != st->B || row + L > st->rows))) return none();
    if (paged) {
      if (st->rows != KVQ_PAGE_ROWS || !table_of(a[7], B, k.device(), &table, &table_stride, &pages)) return none();
      if (a[8] != Py_None && !(starts = ints_of(a[8], B, k.device()))) return none();
    } else if (a[8] != Py_None) {
      return none();
    }
    if (D * st->bits / 32 != st->code_words || D / st->group != st->groups) return none();
    int64_t Hq = 0;
    if (a[5] != Py_None) {
      if (!THPVariable_Check(a[5])) return none();
      const at::Tensor& q = THPVariable_Unpack(a[5]);
      if (q.numel() == 0 || q.scalar_type() != k.scalar_type() || q.device() != k.device() || !rows_of(q, &qr)) return none();
      if (q.size(0) != B || q.size(2) != L || q.size(3) != D || !fits_int({q.size(1)})) return none();
      Hq = q.size(1);
    }
    kvq_axes ax = *(const kvq_axes*)st->rope;
    if (!positions_of(a[3], B, L, k.device(), &ax)) return none();
    int rc;
    {
      Unlocked u;
      rc = d.axes_append(&kr, st->kq, &vr, st->vq, Hq ? &qr : nullptr, (int)Hq, &ax, table ? (int)st->B : 0, table,
                         table_stride, starts, row, (int)B, (int)st->H, (int)L, (int)D, st->bits, st->group, st->code, stream);
    }
    if (rc != KVQ_OK) return failed(rc);
    Py_RETURN_TRUE;
  } catch (...) {
    PyErr_Clear();
    return none();
  }
}

// dequantize(keys, values, start, stop, group_size, bits, out pair or None, block table or None, seq_lens, stream) -> the
// pair of values [B, H, stop - start, D] (of pages: rows [0, stop), with out), the negative status of a failed launch, or None
PyObject* dequantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 10 || !d.dequantize) return none();
  try {
    Triple k, v;
    if (!triple_of(a[0], &k) || !triple_of(a[1], &v)) return none();
    const long long start = PyLong_AsLongLong(a[2]), stop = PyLong_AsLongLong(a[3]);
    const long group = PyLong_AsLong(a[4]), bits = PyLong_AsLong(a[5]);
    void* stream = PyLong_AsVoidPtr(a[9]);
    if (PyErr_Occurred()) {
      PyErr_Clear();
      return none();
    }
    const int code = dtype_code(k.s.scalar_type());
    if (code < 0 || !k.s.is_cuda() || k.c.dim() != 4 || k.s.dim() != 4 || (bits != 4 && bits != 8) || group <= 0) return none();
    const at::Device dev = k.s.device();
    const int64_t lead = k.c.size(0), H = k.c.size(1), S = k.c.size(2), D = k.s.size(3) * group, rows = stop - start;
    kvq_qtensor kq, vq;
    if (!qtensor_of(k, lead, H, S, D, (int)bits, (int)group, k.s.scalar_type(), dev, nullptr, &kq) ||
        !qtensor_of(v, lead, H, S, D, (int)bits, (int)group, k.s.scalar_type(), dev, nullptr, &vq))
      return none();
    int64_t B = lead, table_stride = 0, pages = 0;
    const int32_t *table = nullptr, *lens = nullptr;
    if (a[7] != Py_None) {
      if (!THPVariable_Check(a[7]) || THPVariable_Unpack(a[7]).dim() != 2 || S != KVQ_PAGE_ROWS || start != 0) return none();
      B = THPVariable_Unpack(a[7]).size(0);
      if (!table_of(a[7], B, dev, &table, &table_stride, &pages) || !(lens = ints_of(a[8], B, dev)) || a[6] == Py_None)
        return none();
    } else if (start < 0 || stop > S) {
      return none();
    }
    if (rows <= 0 || B <= 0 || H <= 0 || !fits_int({lead, B, H, rows, D})) return none();
    at::Tensor out[2];
    kvq_rows o[2];
    const bool given = a[6] != Py_None;
    if (given && (!PyTuple_Check(a[6]) || PyTuple_GET_SIZE(a[6]) != 2)) return none();
    for (int i = 0; i < 2; ++i) {
      if (given) {
        PyObject* x = PyTuple_GET_ITEM(a[6], i);
        if (!THPVariable_Check(x)) return none();
        out[i] = THPVariable_Unpack(x);
        if (out[i].scalar_type() != k.s.scalar_type() || out[i].device() != dev || out[i].dim() != 4 || out[i].size(0) != B ||
            out[i].size(1) != H || out[i].size(2) != rows || out[i].size(3) != D)
          return none();
      } else {
        out[i] = at::empty({B, H, rows, D}, k.s.options().requires_grad(false));
      }
      if (!rows_of(out[i], &o[i])) return none();
    }
    int rc;
    {
      Unlocked u;
      if (table) {
        rc = d.paged_dequantize(&kq, &o[0], &vq, &o[1], (int)lead, table, table_stride, lens, (int)B, (int)H, (int)rows, (int)D,
                                (int)bits, (int)group, code, stream);
      } else {
        rc = d.dequantize(&kq, &o[0], &vq, &o[1], start, (int)B, (int)H, (int)rows, (int)D, (int)bits, (int)group, code, stream);
      }
    }
    if (rc != KVQ_OK) return failed(rc);
    if (given) {
      Py_INCREF(a[6]);
      return a[6];
    }
    PyObject* both = PyTuple_New(2);
    for (int i = 0; i < 2; ++i) PyTuple_SET_ITEM(both, i, THPVariable_Wrap(std::move(out[i])));
    return both;
  } catch (...) {
    PyErr_Clear();
    return none();
  }
}

// The tensors of nested tuples and lists, as arrays of rows [lead][H][rows][width] on `dev`.
struct RowArrays {
  std::vector<kvq_row_array> arrays;
  int64_t lead = 0, H = 0, rows = INT64_MAX;  // rows: the fewest of an array
  bool add(PyObject* o, const at::Device& dev, int depth) {
    if (THPVariable_Check(o)) {
      const at::Tensor& t = THPVariable_Unpack(o);
      if (t.dim() != 4 || t.device() != dev || t.stride(3) != 1) return false;
      if (arrays.empty()) lead = t.size(0), H = t.size(1);
      if (t.size(0) != lead || t.size(1) != H) return false;
      const int64_t n = t.element_size();
      arrays.push_back({t.data_ptr(), n * t.stride(0), n * t.stride(1), n * t.stride(2), n * t.size(3)});
      rows = std::min(rows, t.size(2));
      most = std::max(most, t.size(2));
      return true;
    }
    const bool list = PyList_Check(o);
    if (depth == 0 || (!list && !PyTuple_Check(o))) return false;
    const Py_ssize_t m = list ? PyList_GET_SIZE(o) : PyTuple_GET_SIZE(o);
    for (Py_ssize_t i = 0; i < m; ++i)
      if (!add(list ? PyList_GET_ITEM(o, i) : PyTuple_GET_ITEM(o, i), dev, depth - 1)) return false;
    return true;
  }
  int64_t most = 0;
};

// keep_rows(tensors in nested tuples and lists, rows, start, n, block table or None, starts or None, stream) -> True, the
// negative status of a failed launch, or None
PyObject* keep_rows(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 7 || !d.keep_rows || !THPVariable_Check(a[1])) return none();
  try {
    const at::Tensor& rows = THPVariable_Unpack(a[1]);
    const long long start = PyLong_AsLongLong(a[2]), drafted = PyLong_AsLongLong(a[3]);
    void* stream = PyLong_AsVoidPtr(a[6]);
    if (PyErr_Occurred()) {
      PyErr_Clear();
      return none();
    }
    if (!rows.is_cuda() || rows.scalar_type() != at::kInt || rows.dim() < 1 || rows.dim() > 2 || rows.size(-1) < 1 ||
        (rows.size(-1) > 1 && rows.stride(-1) != 1))
      return none();
    const at::Device dev = rows.device();
    RowArrays arr;
    arr.arrays.reserve(256);
    if (!arr.add(a[0], dev, 3) || arr.arrays.empty() || arr.lead <= 0 || arr.H <= 0) return none();
    int64_t B = arr.lead, table_stride = 0, pages = 0;
    const int32_t *table = nullptr, *starts = nullptr;
    if (a[4] != Py_None) {
      if (!THPVariable_Check(a[4]) || THPVariable_Unpack(a[4]).dim() != 2) return none();
      B = THPVariable_Unpack(a[4]).size(0);
      if (!table_of(a[4], B, dev, &table, &table_stride, &pages) || arr.rows != KVQ_PAGE_ROWS || arr.most != KVQ_PAGE_ROWS)
        return none();
      if (a[5] != Py_None && !(starts = ints_of(a[5], B, dev))) return none();
    } else if (a[5] != Py_None || start < 0 || drafted < 0 || start + drafted > arr.rows) {
      return none();
    }
    if (B <= 0 || (rows.dim() == 2 && rows.size(0) != B)) return none();
    if (!fits_int({arr.lead, B, arr.H, rows.size(-1), drafted, (int64_t)arr.arrays.size()})) return none();
    int rc;
    {
      Unlocked u;
      rc = d.keep_rows(arr.arrays.data(), (int)arr.arrays.size(), table ? (int)arr.lead : 0, table, table_stride,
                       (const int32_t*)rows.data_ptr(), rows.dim() == 2 ? rows.stride(0) : 0, starts, start, (int)drafted,
                       (int)rows.size(-1), (int)B, (int)arr.H, stream);
    }
    if (rc != KVQ_OK) return failed(rc);
    Py_RETURN_TRUE;
  } catch (...) {
    PyErr_Clear();
    return none();
  }
}

// bind_draft(the entry points of a drafted step, in d's order)
PyObject* bind_draft(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 11) {
    PyErr_SetString(PyExc_TypeError, "bind_draft takes 11 addresses");
    return nullptr;
  }
  void* at[11];
  for (int i = 0; i < 11; ++i) at[i] = PyLong_AsVoidPtr(a[i]);
  if (PyErr_Occurred()) return nullptr;
  auto set = [&, i = 0](auto& fn) mutable { fn = (std::decay_t<decltype(fn)>)at[i++]; };
  set(d.draft_tree), set(d.tree), set(d.tree_dense), set(d.tree_paged), set(d.tree_ws), set(d.tree_kernel);
  set(d.rope_axes), set(d.axes_append), set(d.dequantize), set(d.paged_dequantize), set(d.keep_rows);
  return none();
}

// bind(decode, prefill, decode_workspace_size, prefill_workspace_size, abi, state_bytes, torch): the library's
// entry points; raises where this module was built against another ABI, AppendState or torch.
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 7) {
    PyErr_SetString(PyExc_TypeError, "bind takes 4 addresses, the ABI version, AppendState's size and torch's version");
    return nullptr;
  }
  const long abi = PyLong_AsLong(a[4]), state = PyLong_AsLong(a[5]);
  const char* torch = PyUnicode_AsUTF8(a[6]);
  if (PyErr_Occurred() || !torch) return nullptr;
  const size_t m = strlen(TORCH_VERSION);
  if (abi != KVQ_ABI_VERSION || state != (long)sizeof(AppendState) || strncmp(torch, TORCH_VERSION, m) ||
      (torch[m] >= '0' && torch[m] <= '9')) {
    PyErr_Format(PyExc_ImportError,
                 "_kvqhost.so was built for ABI version %d, an AppendState of %zu bytes and torch %s; here they are %ld, %ld "
                 "and %s: rebuild it",
                 KVQ_ABI_VERSION, sizeof(AppendState), TORCH_VERSION, abi, state, torch);
    return nullptr;
  }
  g.decode = (AttnFn)PyLong_AsVoidPtr(a[0]);
  g.prefill = (AttnFn)PyLong_AsVoidPtr(a[1]);
  g.decode_ws = (SizeFn)PyLong_AsVoidPtr(a[2]);
  g.prefill_ws = (SizeFn)PyLong_AsVoidPtr(a[3]);
  if (PyErr_Occurred()) return nullptr;
  return none();
}

PyMethodDef methods[] = {
    {"attention", (PyCFunction)(void*)attention, METH_FASTCALL, "one quantized attention call"},
    {"append", (PyCFunction)(void*)append, METH_FASTCALL, "one quantize-append"},
    {"views", (PyCFunction)(void*)views, METH_FASTCALL, "the first rows of two triples"},
    {"draft_tree", (PyCFunction)(void*)draft_tree, METH_FASTCALL, "the bits and depths of trees"},
    {"tree_attention", (PyCFunction)(void*)tree_attention, METH_FASTCALL, "one attention call over a tree"},
    {"rope_axes", (PyCFunction)(void*)rope_axes, METH_FASTCALL, "one rotation at positions"},
    {"axes_append", (PyCFunction)(void*)axes_append, METH_FASTCALL, "one quantize-append at positions"},
    {"dequantize", (PyCFunction)(void*)dequantize, METH_FASTCALL, "rows of two triples read back"},
    {"keep_rows", (PyCFunction)(void*)keep_rows, METH_FASTCALL, "accepted rows moved up"},
    {"bind_draft", (PyCFunction)(void*)bind_draft, METH_FASTCALL, "set the entry points of a drafted step"},
    {"bind", (PyCFunction)(void*)bind, METH_FASTCALL, "set the library's entry points"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_kvqhost", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__kvqhost() { return PyModule_Create(&module); }
