// Host path of the operators around a cache with scales per (page, kv head), for ordinary calls.
//
// A small call costs its caller more time in fetching shapes, strides and addresses through Python than it
// takes on the GPU.  These functions do the same in C++: they check everything the Python functions check,
// fill the parameter block of the C ABI and launch on torch's current stream.  A call that is in
// any way out of the ordinary -- an argument of another type or shape, a layout that needs a copy, a
// device that is not the current one -- is left to the Python function (the answer is None), which
// copies, switches devices or raises with the reason.  So nothing here raises, and a check that fails here is
// never the last word.
//
// Answers: None (not taken), an int (a PaStatus that is not PA_OK), or a tuple of new tensors.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstring>

#include "../../include/pa_decode_sm100.h"
#include "pa_places.h"

namespace {

// Entry points of the CUDA library, handed over once by the Python side (which has loaded it).
int (*g_decode_tables)(const PaDecodeParams*, int64_t, void*) = nullptr;
int (*g_append)(const PaCacheAppendParams*, void*) = nullptr;
int (*g_scores)(const PaBlockScoreParams*, void*) = nullptr;
int (*g_select)(const PaBlockSelectParams*, void*) = nullptr;

constexpr int64_t kD = 128;
constexpr int64_t kPartition = 256;

// The tensor behind a Python object, or null.
const at::Tensor* tensor(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

bool is(const at::Tensor& t, at::ScalarType type, int64_t dims) { return t.scalar_type() == type && t.dim() == dims; }
bool sized(const at::Tensor& t, std::initializer_list<int64_t> want) {
  if (t.dim() != (int64_t)want.size()) return false;
  int64_t d = 0;
  for (int64_t w : want)
    if (t.size(d++) != w) return false;
  return true;
}
bool aligned16(const at::Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }
bool block_size_ok(int64_t bs) { return bs == 16 || bs == 64 || bs == 1024; }

// All tensors on one CUDA device, which is the current one; its index, or -1.
int common_device(std::initializer_list<const at::Tensor*> ts) {
  int index = -1;
  for (const at::Tensor* t : ts) {
    if (!t->is_cuda()) return -1;
    const int i = t->get_device();
    if (index >= 0 && i != index) return -1;
    index = i;
  }
  return index >= 0 && index == c10::cuda::current_device() ? index : -1;
}
void* stream_of(int device) { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream(); }

// Key and value cache of one pool in a layout that needs no second look: [NB, Hkv, 8, bs, 16] and
// [NB, Hkv, 128, bs] or [NB, Hkv, bs/16, 128, 16] (bs > 16), dense pages of one head.
bool caches_ok(const at::Tensor& k, const at::Tensor& v, bool* transposed) {
  if (!is(k, at::kFloat8_e4m3fn, 5) || v.scalar_type() != at::kFloat8_e4m3fn) return false;
  const int64_t nb = k.size(0), h = k.size(1), bs = k.size(3);
  if (nb < 1 || h < 1 || !block_size_ok(bs) || k.size(2) != kD / 16 || k.size(4) != 16) return false;
  if (k.stride(4) != 1 || k.stride(3) != 16 || k.stride(2) != 16 * bs) return false;
  if (v.dim() == 4) {
    *transposed = false;
    return sized(v, {nb, h, kD, bs}) && v.stride(3) == 1 && v.stride(2) == bs;
  }
  *transposed = true;
  return bs > 16 && sized(v, {nb, h, bs / 16, kD, 16}) && v.stride(4) == 1 && v.stride(3) == 16 && v.stride(2) == 16 * kD;
}
// Scales [NB, Hkv, 1, 1] that share strides, or one value each (0-dim).  -2: neither.
int scale_mode(const at::Tensor& k, const at::Tensor& v, int64_t nb, int64_t h) {
  if (k.scalar_type() != at::kFloat || v.scalar_type() != at::kFloat) return -2;
  if (k.dim() == 0 && v.dim() == 0) return PA_QUANT_PER_TENSOR;
  if (nb * h > 1 && sized(k, {nb, h, 1, 1}) && sized(v, {nb, h, 1, 1}) && k.stride(0) == v.stride(0) && k.stride(1) == v.stride(1))
    return PA_QUANT_PER_BLOCK;
  return -2;
}
// An optional int32 status tensor; false where it is something else.
bool status_of(PyObject* o, int device, int32_t** out) {
  *out = nullptr;
  if (o == Py_None) return true;
  const at::Tensor* t = tensor(o);
  if (!t || t->scalar_type() != at::kInt || !t->is_cuda() || t->get_device() != device || t->numel() < 1) return false;
  *out = t->data_ptr<int32_t>();
  return true;
}
bool to_int(PyObject* o, int64_t* out) {
  if (!PyLong_Check(o)) return false;
  int overflow = 0;
  *out = PyLong_AsLongLongAndOverflow(o, &overflow);
  return overflow == 0 && *out >= 0 && *out <= 0x7fffffff;
}
bool to_float(PyObject* o, float* out) {
  if (!PyFloat_Check(o)) return false;
  *out = (float)PyFloat_AS_DOUBLE(o);
  return true;
}
PyObject* wrap(std::initializer_list<at::Tensor> ts) {
  PyObject* tuple = PyTuple_New((Py_ssize_t)ts.size());
  if (!tuple) return nullptr;
  Py_ssize_t i = 0;
  for (const at::Tensor& t : ts) {
    PyObject* o = THPVariable_Wrap(t);
    if (!o) {
      Py_DECREF(tuple);
      return nullptr;
    }
    PyTuple_SET_ITEM(tuple, i++, o);
  }
  return tuple;
}

// An exception of torch (no memory, say) becomes "not taken": the Python path meets it again and raises it.
template <typename F>
PyObject* guarded(F&& body) {
  try {
    PyObject* r = body();
    if (r == nullptr && !PyErr_Occurred()) Py_RETURN_NONE;
    return r;
  } catch (const std::exception&) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
}

// decode(output, query, key_cache, value_cache, lengths, tables, softmax_scale, query_len, max_len, key_scale, value_scale, status)
//   -> (exp_sums, max_logits, tmp_output)
PyObject* decode(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 12 || !g_decode_tables) return nullptr;
    const at::Tensor *out = tensor(a[0]), *q = tensor(a[1]), *k = tensor(a[2]), *v = tensor(a[3]), *len = tensor(a[4]), *bt = tensor(a[5]),
                     *ks = tensor(a[9]), *vs = tensor(a[10]);
    float scale;
    int64_t ql, longest;
    if (!out || !q || !k || !v || !len || !bt || !ks || !vs || !to_float(a[6], &scale) || !to_int(a[7], &ql) || !to_int(a[8], &longest))
      return nullptr;
    bool transposed;
    if (!is(*out, at::kBFloat16, 3) || !is(*q, at::kBFloat16, 3) || !q->sizes().equals(out->sizes()) || !caches_ok(*k, *v, &transposed)) return nullptr;
    const int64_t s = q->size(0), heads = q->size(1), nb = k->size(0), h = k->size(1), bs = k->size(3);
    if (s < 1 || q->size(2) != kD || ql < 1 || ql > 4 || heads % (ql * h) || heads == 0) return nullptr;
    const int64_t rows = heads / h, group = rows / ql;
    if (rows > 64) return nullptr;
    if (out->stride(2) != 1 || q->stride(2) != 1 || q->stride(1) != kD || (q->stride(0) & 15) || !aligned16(*q)) return nullptr;
    if (!is(*len, at::kInt, 1) || len->size(0) != s || len->stride(0) != 1) return nullptr;
    const bool per_head = bt->dim() == 3;
    if (bt->scalar_type() != at::kInt || (bt->dim() != 2 && !per_head) || bt->size(0) != s || (per_head && bt->size(1) != h) ||
        bt->size(-1) < 1 || bt->stride(-1) != 1 || (per_head && h > 1 && bt->stride(1) <= 0))
      return nullptr;
    const int mode = scale_mode(*ks, *vs, nb, h);
    if (mode < 0) return nullptr;
    const int device = common_device({out, q, k, v, len, bt, ks, vs});
    int32_t* status;
    if (device < 0 || !status_of(a[11], device, &status)) return nullptr;

    const int64_t parts = longest <= kPartition ? 1 : (longest + kPartition - 1) / kPartition;
    const at::TensorOptions fp32 = out->options().dtype(at::kFloat);
    at::Tensor sums = at::empty({s, h, parts, rows}, fp32), tops = at::empty({s, h, parts, rows}, fp32);
    at::Tensor tmp = at::empty({s, h, parts, rows, kD}, fp32);   // (bf16 would round every partition once more)
    PaDecodeParams p;
    std::memset(&p, 0, sizeof(p));
    p.struct_size = sizeof(p);
    p.abi_version = PA_ABI_VERSION;
    p.out = out->data_ptr();
    p.query = q->data_ptr();
    p.key_cache = k->data_ptr();
    p.value_cache = v->data_ptr();
    p.block_tables = bt->data_ptr<int32_t>();
    p.context_lens = len->data_ptr<int32_t>();
    p.key_scale = ks->data_ptr<float>();
    p.value_scale = vs->data_ptr<float>();
    p.exp_sums = sums.data_ptr<float>();
    p.max_logits = tops.data_ptr<float>();
    p.tmp_out = tmp.data_ptr();
    p.status = status;
    p.num_seqs = (int32_t)s;
    p.num_kv_heads = (int32_t)h;
    p.query_group_size = (int32_t)group;
    p.query_len = (int32_t)ql;
    p.head_size = (int32_t)kD;
    p.block_size = (int32_t)bs;
    p.num_blocks = (int32_t)nb;
    p.max_blocks_per_seq = (int32_t)bt->size(-1);
    p.partition_size = (int32_t)kPartition;
    p.max_partitions = (int32_t)parts;
    p.out_stride_seq = out->stride(0);
    p.out_stride_head = out->stride(1);
    p.q_stride_seq = q->stride(0);
    p.q_stride_head = q->stride(1);
    p.k_stride_block = k->stride(0);
    p.k_stride_head = k->stride(1);
    p.v_stride_block = v->stride(0);
    p.v_stride_head = v->stride(1);
    p.bt_stride_seq = bt->stride(0);
    if (mode == PA_QUANT_PER_BLOCK) {
      p.kv_scale_stride_block = ks->stride(0);
      p.kv_scale_stride_head = ks->stride(1);
    }
    p.ws_stride_part = rows;
    p.ws_stride_head = parts * rows;
    p.ws_stride_seq = h * p.ws_stride_head;
    p.tmp_stride_row = kD;
    p.tmp_stride_part = rows * kD;
    p.tmp_stride_head = parts * p.tmp_stride_part;
    p.tmp_stride_seq = h * p.tmp_stride_head;
    p.q_dtype = PA_DT_BF16;
    p.kv_dtype = PA_DT_E4M3FN;
    p.out_dtype = PA_DT_BF16;
    p.tmp_dtype = PA_DT_F32;
    p.q_quant_mode = PA_QUANT_NONE;
    p.kv_quant_mode = mode;
    p.v_layout = transposed ? PA_V_TRANSPOSED : PA_V_NORMAL;
    p.softmax_scale = scale;
    const int rc = g_decode_tables(&p, per_head && h > 1 ? bt->stride(1) : 0, stream_of(device));
    return rc != PA_OK ? PyLong_FromLong(rc) : wrap({sums, tops, tmp});
  });
}

// append(key, value, key_cache, value_cache, key_scale, value_scale, tables, lengths, start, key_bounds, status) -> ()
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 11 || !g_append) return nullptr;
    const at::Tensor *key = tensor(a[0]), *val = tensor(a[1]), *k = tensor(a[2]), *v = tensor(a[3]), *ks = tensor(a[4]), *vs = tensor(a[5]),
                     *bt = tensor(a[6]), *len = tensor(a[7]), *start = tensor(a[8]), *bounds = a[9] == Py_None ? nullptr : tensor(a[9]);
    if (!key || !val || !k || !v || !ks || !vs || !bt || !len || !start || (a[9] != Py_None && !bounds)) return nullptr;
    bool transposed;
    if (!is(*key, at::kBFloat16, 3) || !is(*val, at::kBFloat16, 3) || !val->sizes().equals(key->sizes()) || !caches_ok(*k, *v, &transposed)) return nullptr;
    const int64_t t = key->size(0), nb = k->size(0), h = k->size(1), bs = k->size(3);
    if (key->size(1) != h || key->size(2) != kD) return nullptr;
    for (const at::Tensor* x : {key, val})
      if (x->stride(2) != 1 || (x->stride(0) & 7) || (x->stride(1) & 7) || !aligned16(*x)) return nullptr;
    const int mode = scale_mode(*ks, *vs, nb, h);
    if (mode < 0) return nullptr;
    auto distinct = [&](const at::Tensor& x) { return pa_places::distinct(nb, h, x.stride(0), x.stride(1)); };
    if (!distinct(*k) || !distinct(*v)) return nullptr;
    if (mode == PA_QUANT_PER_BLOCK &&
        (!distinct(*ks) || pa_places::meet(vs->data_ptr<float>() - ks->data_ptr<float>(), nb, h, ks->stride(0), ks->stride(1))))
      return nullptr;
    if (!is(*bt, at::kInt, 2) || bt->size(1) < 1 || bt->stride(1) != 1) return nullptr;
    const int64_t s = bt->size(0);
    if (!is(*len, at::kInt, 1) || len->size(0) != s || !is(*start, at::kInt, 1) || start->size(0) != s + 1 ||
        (s > 1 && len->stride(0) != 1) || start->stride(0) != 1)
      return nullptr;
    if (bounds && (bounds->scalar_type() != at::kFloat8_e4m3fn || !sized(*bounds, {nb, h, 2, kD}) || bounds->stride(3) != 1 ||
                   bounds->stride(2) != kD || !distinct(*bounds)))
      return nullptr;
    const int device = common_device({key, val, k, v, ks, vs, bt, len, start, bounds ? bounds : key});
    int32_t* status;
    if (device < 0 || !status_of(a[10], device, &status)) return nullptr;
    PaCacheAppendParams p;
    std::memset(&p, 0, sizeof(p));
    p.struct_size = sizeof(p);
    p.abi_version = PA_ABI_VERSION;
    p.key = key->data_ptr();
    p.value = val->data_ptr();
    p.key_cache = k->data_ptr();
    p.value_cache = v->data_ptr();
    p.key_scale = ks->data_ptr<float>();
    p.value_scale = vs->data_ptr<float>();
    p.key_bounds = bounds ? bounds->data_ptr() : nullptr;
    p.block_tables = bt->data_ptr<int32_t>();
    p.context_lens = len->data_ptr<int32_t>();
    p.row_start = start->data_ptr<int32_t>();
    p.status = status;
    p.num_tokens = (int32_t)t;
    p.num_seqs = (int32_t)s;
    p.num_kv_heads = (int32_t)h;
    p.head_size = (int32_t)kD;
    p.block_size = (int32_t)bs;
    p.num_blocks = (int32_t)nb;
    p.max_blocks_per_seq = (int32_t)bt->size(1);
    p.kv_quant_mode = mode;
    p.v_layout = transposed ? PA_V_TRANSPOSED : PA_V_NORMAL;
    p.key_stride_token = key->stride(0);
    p.key_stride_head = key->stride(1);
    p.value_stride_token = val->stride(0);
    p.value_stride_head = val->stride(1);
    p.k_stride_block = k->stride(0);
    p.k_stride_head = k->stride(1);
    p.v_stride_block = v->stride(0);
    p.v_stride_head = v->stride(1);
    if (mode == PA_QUANT_PER_BLOCK) {
      p.kv_scale_stride_block = ks->stride(0);
      p.kv_scale_stride_head = ks->stride(1);
    }
    if (bounds) {
      p.bounds_stride_block = bounds->stride(0);
      p.bounds_stride_head = bounds->stride(1);
    }
    p.bt_stride_seq = bt->stride(0);
    const int rc = g_append(&p, stream_of(device));
    return rc != PA_OK ? PyLong_FromLong(rc) : PyTuple_New(0);
  });
}

// scores(query, key_bounds, lengths, tables, softmax_scale, query_len, block_size, key_scale, status) -> (scores,)
PyObject* scores(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 9 || !g_scores) return nullptr;
    const at::Tensor *q = tensor(a[0]), *b = tensor(a[1]), *len = tensor(a[2]), *bt = tensor(a[3]), *ks = a[7] == Py_None ? nullptr : tensor(a[7]);
    float scale;
    int64_t ql, bs;
    if (!q || !b || !len || !bt || (a[7] != Py_None && !ks) || !to_float(a[4], &scale) || !to_int(a[5], &ql) || !to_int(a[6], &bs)) return nullptr;
    if (!is(*q, at::kBFloat16, 3) || !is(*b, at::kFloat8_e4m3fn, 4) || !(scale > 0.f) || !block_size_ok(bs)) return nullptr;
    const int64_t s = q->size(0), heads = q->size(1), nb = b->size(0), h = b->size(1);
    if (s < 1 || nb < 1 || h < 1 || q->size(2) != kD || b->size(2) != 2 || b->size(3) != kD || ql < 1 || ql > 4 || heads == 0 || heads % (ql * h) ||
        heads / h > 64)
      return nullptr;
    if (b->stride(3) != 1 || b->stride(2) != kD || q->stride(2) != 1 || q->stride(1) != kD || (q->stride(0) & 7) || !aligned16(*q)) return nullptr;
    if (!is(*bt, at::kInt, 2) || bt->size(0) != s || bt->size(1) < 1 || bt->stride(1) != 1 || !is(*len, at::kInt, 1) || len->size(0) != s ||
        (s > 1 && len->stride(0) != 1))
      return nullptr;
    int mode = PA_QUANT_NONE;
    if (ks && (mode = scale_mode(*ks, *ks, nb, h)) < 0) return nullptr;
    const int device = common_device({q, b, len, bt, ks ? ks : q});
    int32_t* status;
    if (device < 0 || !status_of(a[8], device, &status)) return nullptr;
    const int64_t width = bt->size(1);
    at::Tensor out = at::empty({s, h, width}, q->options().dtype(at::kFloat));
    PaBlockScoreParams p;
    std::memset(&p, 0, sizeof(p));
    p.struct_size = sizeof(p);
    p.abi_version = PA_ABI_VERSION;
    p.query = q->data_ptr();
    p.key_bounds = b->data_ptr();
    p.block_tables = bt->data_ptr<int32_t>();
    p.context_lens = len->data_ptr<int32_t>();
    p.key_scale = ks ? ks->data_ptr<float>() : nullptr;
    p.scores = out.data_ptr<float>();
    p.status = status;
    p.num_seqs = (int32_t)s;
    p.num_kv_heads = (int32_t)h;
    p.rows = (int32_t)(heads / h);
    p.head_size = (int32_t)kD;
    p.block_size = (int32_t)bs;
    p.num_blocks = (int32_t)nb;
    p.max_blocks_per_seq = (int32_t)width;
    p.q_dtype = PA_DT_BF16;
    p.q_quant_mode = PA_QUANT_NONE;
    p.kv_quant_mode = mode;
    p.q_stride_seq = q->stride(0);
    p.bounds_stride_block = b->stride(0);
    p.bounds_stride_head = b->stride(1);
    p.bt_stride_seq = bt->stride(0);
    if (mode == PA_QUANT_PER_BLOCK) {
      p.kv_scale_stride_block = ks->stride(0);
      p.kv_scale_stride_head = ks->stride(1);
    }
    p.scores_stride_seq = h * width;
    p.scores_stride_head = width;
    p.softmax_scale = scale;
    const int rc = g_scores(&p, stream_of(device));
    return rc != PA_OK ? PyLong_FromLong(rc) : wrap({out});
  });
}

// select(scores, lengths, tables, block_size, top_k, keep_first, keep_last, status) -> (tables, lengths)
PyObject* select(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 8 || !g_select) return nullptr;
    const at::Tensor *sc = tensor(a[0]), *len = tensor(a[1]), *bt = tensor(a[2]);
    int64_t bs, top_k, first, last;
    if (!sc || !len || !bt || !to_int(a[3], &bs) || !to_int(a[4], &top_k) || !to_int(a[5], &first) || !to_int(a[6], &last)) return nullptr;
    if (!is(*sc, at::kFloat, 3) || !block_size_ok(bs) || last < 1 || top_k < 1 || top_k < first + last) return nullptr;
    const int64_t s = sc->size(0), h = sc->size(1);
    if (s < 1 || h < 1 || sc->stride(2) != 1 || !is(*bt, at::kInt, 2) || bt->size(0) != s || bt->size(1) < 1 || bt->size(1) > sc->size(2) ||
        bt->stride(1) != 1 || !is(*len, at::kInt, 1) || len->size(0) != s || (s > 1 && len->stride(0) != 1))
      return nullptr;
    const int device = common_device({sc, len, bt});
    int32_t* status;
    if (device < 0 || !status_of(a[7], device, &status)) return nullptr;
    at::Tensor tables = at::empty({s, h, top_k}, len->options()), lengths = at::empty({s}, len->options());
    PaBlockSelectParams p;
    std::memset(&p, 0, sizeof(p));
    p.struct_size = sizeof(p);
    p.abi_version = PA_ABI_VERSION;
    p.scores = sc->data_ptr<float>();
    p.block_tables = bt->data_ptr<int32_t>();
    p.context_lens = len->data_ptr<int32_t>();
    p.tables = tables.data_ptr<int32_t>();
    p.lengths = lengths.data_ptr<int32_t>();
    p.status = status;
    p.num_seqs = (int32_t)s;
    p.num_kv_heads = (int32_t)h;
    p.block_size = (int32_t)bs;
    p.max_blocks_per_seq = (int32_t)bt->size(1);
    p.top_k = (int32_t)top_k;
    p.keep_first = (int32_t)first;
    p.keep_last = (int32_t)last;
    p.scores_stride_seq = sc->stride(0);
    p.scores_stride_head = sc->stride(1);
    p.bt_stride_seq = bt->stride(0);
    p.tables_stride_seq = h * top_k;
    p.tables_stride_head = top_k;
    const int rc = g_select(&p, stream_of(device));
    return rc != PA_OK ? PyLong_FromLong(rc) : wrap({tables, lengths});
  });
}

// bind(decode_tables, append, scores, select, abi_version): addresses in the loaded CUDA library
PyObject* bind(PyObject*, PyObject* args) {
  unsigned long long f[4];
  int version;
  if (!PyArg_ParseTuple(args, "KKKKi", &f[0], &f[1], &f[2], &f[3], &version)) return nullptr;
  if (version != PA_ABI_VERSION) {
    PyErr_SetString(PyExc_ImportError, "the host calls were built for another ABI version; rebuild");
    return nullptr;
  }
  g_decode_tables = reinterpret_cast<decltype(g_decode_tables)>(f[0]);
  g_append = reinterpret_cast<decltype(g_append)>(f[1]);
  g_scores = reinterpret_cast<decltype(g_scores)>(f[2]);
  g_select = reinterpret_cast<decltype(g_select)>(f[3]);
  Py_RETURN_NONE;
}

PyMethodDef kMethods[] = {
    {"bind", bind, METH_VARARGS, nullptr},
    {"decode", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(decode)), METH_FASTCALL, nullptr},
    {"append", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(append)), METH_FASTCALL, nullptr},
    {"scores", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(scores)), METH_FASTCALL, nullptr},
    {"select", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(select)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "pa_calls", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_pa_calls(void) { return PyModule_Create(&kModule); }
