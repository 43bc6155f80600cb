// CPython binding of the speculative-decoding operators (8-bit KV cache,
// drafted-tree attention, logits processing): argument checks, output
// allocation and the call of one C entry point. Small calls are bounded by the
// host: the same checks in Python and the call through ctypes took 12 to 20 us a
// call on the GPU host, of which the launch is 3. litevllm_b200/ops.py documents
// the functions and is their only caller; errors are the ones its other functions
// raise.
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include "litekern.h"

namespace {

PyTypeObject* g_cache_type = nullptr;  // ops.QuantizedCache
PyObject* g_error = nullptr;           // _lib.LiteKernError

struct PyRaised {};  // a Python exception is set

[[noreturn]] void raise(PyObject* type, const char* text) {
  PyErr_SetString(type, text);
  throw PyRaised();
}
[[noreturn]] void type_error(const char* text) { raise(PyExc_TypeError, text); }
[[noreturn]] void value_error(const char* text) { raise(PyExc_ValueError, text); }

using T = const at::Tensor*;

T tensor(PyObject* o, bool optional = false) {
  if (optional && o == Py_None) return nullptr;
  if (!THPVariable_Check(o)) type_error("expected a torch.Tensor");
  return &THPVariable_Unpack(o);
}

int32_t n32(int64_t n) {
  if (n > INT32_MAX) value_error("a size does not fit 32 bits");
  return static_cast<int32_t>(n);
}

int64_t integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw PyRaised();
  return v;
}

// All on one CUDA device: its index.
template <size_t N> int device_of(const T (&ts)[N]) {
  int dev = -1;
  for (T t : ts) {
    if (!t) continue;
    if (!t->is_cuda())
      raise(PyExc_RuntimeError, "litevllm_b200 kernels run on CUDA tensors only (no CPU fallback)");
    const int d = t->get_device();
    if (dev < 0) dev = d;
    else if (d != dev) raise(PyExc_RuntimeError, "tensors on different devices");
  }
  return dev;
}

int dtype_code(at::ScalarType t, bool fp32) {
  switch (t) {
    case at::kHalf: return LK_DTYPE_F16;
    case at::kBFloat16: return LK_DTYPE_BF16;
    case at::kFloat:
      if (fp32) return LK_DTYPE_F32;
      [[fallthrough]];
    default: type_error(fp32 ? "dtype not supported here (allowed: float32, float16, bfloat16)"
                             : "dtype not supported here (allowed: float16, bfloat16)");
  }
}

// Runs a C entry point without the interpreter lock (a launch may wait for room in
// the queue) and raises its error.
template <typename... P, typename... A> void call(int (*entry)(P...), A... a) {
  PyThreadState* state = PyEval_SaveThread();
  const int rc = entry(a...);
  PyEval_RestoreThread(state);
  if (rc == LK_OK) return;
  PyErr_Format(g_error, "%s (code %d)", lk_status_string(rc), rc);
  throw PyRaised();
}

template <typename P = void> P* ptr(T t) { return t ? static_cast<P*>(t->data_ptr()) : nullptr; }

void* stream_of(int dev) { return c10::cuda::getCurrentCUDAStream(dev).stream(); }

void check_status(T s) {
  if (s && (s->scalar_type() != at::kInt || s->numel() < 1)) type_error("status must be an int32 tensor");
}

// A contiguous int32 [n] tensor; `keep` holds a copy if one was needed.
T int32_row(T t, int64_t n, const char* text, at::Tensor& keep) {
  if (t->scalar_type() != at::kInt || t->numel() != n) type_error(text);
  if (t->is_contiguous()) return t;
  keep = t->contiguous();
  return &keep;
}

struct Caches {
  T kd, ks, vd, vs;  // ks == nullptr: 16-bit
  int fmt;
  int64_t nb, bs, H_kv, D;
};

bool is_quantised(PyObject* o) {
  return PyObject_TypeCheck(o, g_cache_type) && PyTuple_GET_SIZE(o) == 2;
}

Caches caches(PyObject* k, PyObject* v, bool allow_16bit) {
  Caches c = {};
  if (is_quantised(k) && is_quantised(v)) {
    c.kd = tensor(PyTuple_GET_ITEM(k, 0));
    c.ks = tensor(PyTuple_GET_ITEM(k, 1));
    c.vd = tensor(PyTuple_GET_ITEM(v, 0));
    c.vs = tensor(PyTuple_GET_ITEM(v, 1));
    const at::ScalarType t = c.kd->scalar_type();
    if ((t != at::kChar && t != at::kFloat8_e4m3fn) || c.vd->scalar_type() != t)
      type_error("8-bit caches are both torch.int8 or both torch.float8_e4m3fn");
    if (c.ks->scalar_type() != at::kFloat || c.vs->scalar_type() != at::kFloat)
      type_error("scales must be fp32");
    c.fmt = t == at::kChar ? LK_KV_INT8 : LK_KV_E4M3;
    if (c.kd->dim() != 4 || c.vd->sizes() != c.kd->sizes())
      value_error("cache data must be [num_blocks, block_size, H_kv, D] of equal shapes");
  } else if (allow_16bit && !is_quantised(k) && !is_quantised(v)) {
    c.kd = tensor(k);
    c.vd = tensor(v);
    c.fmt = LK_KV_16BIT;
    if (c.kd->dim() != 4 || c.vd->sizes() != c.kd->sizes()) value_error("cache shape mismatch");
  } else {
    type_error("key_cache and value_cache must both be QuantizedCache");
  }
  c.nb = c.kd->size(0);
  c.bs = c.kd->size(1);
  c.H_kv = c.kd->size(2);
  c.D = c.kd->size(3);
  if (c.ks) {
    auto shape_ok = [&](T s) {
      return s->dim() == 3 && s->size(0) == c.nb && s->size(1) == c.H_kv && s->size(2) == c.bs;
    };
    if (!shape_ok(c.ks) || !shape_ok(c.vs)) value_error("scales must be [num_blocks, H_kv, block_size]");
    if (!c.ks->is_contiguous() || !c.vs->is_contiguous() || !c.kd->is_contiguous() ||
        !c.vd->is_contiguous())
      value_error("caches and scales must be contiguous");
  } else if (!c.kd->is_contiguous() || !c.vd->is_contiguous()) {
    value_error("caches must be contiguous");
  }
  return c;
}

void heads_contiguous(T t, const char* text) {
  if (t->stride(2) != 1 || t->stride(1) != t->size(2)) value_error(text);
}

// Rows in memory: n of `bytes` bytes, `stride` bytes from one to the next.
struct Rows {
  const char* at;
  int64_t n, bytes, stride;
};

// Whether two sets of rows share a byte. Rows that lie between each other's do not.
bool meet(const Rows& a, const Rows& b) {
  auto row = [](const Rows& r, int64_t i) { return r.at + i * r.stride; };
  if (a.n == 0 || b.n == 0 || a.bytes == 0 || b.bytes == 0 || row(a, a.n - 1) + a.bytes <= b.at ||
      row(b, b.n - 1) + b.bytes <= a.at)
    return false;
  for (int64_t i = 0, j = 0; i < a.n && j < b.n;) {
    if (row(a, i) + a.bytes <= row(b, j)) ++i;
    else if (row(b, j) + b.bytes <= row(a, i)) ++j;
    else return true;
  }
  return false;
}

template <typename F> PyObject* guarded(F&& f) {
  HANDLE_TH_ERRORS
  try {
    return f();
  } catch (const PyRaised&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// store(key, value, key_cache, value_cache, slot_mapping, status)
PyObject* store(PyObject*, PyObject* const* a, Py_ssize_t) {
  return guarded([&]() -> PyObject* {
    const Caches c = caches(a[2], a[3], false);
    const T key = tensor(a[0]), value = tensor(a[1]), slots = tensor(a[4]), status = tensor(a[5], true);
    const int dev = device_of({key, value, c.kd, c.ks, c.vd, c.vs, slots, status});
    if (key->dim() != 3 || value->sizes() != key->sizes())
      value_error("key/value must be [T, H_kv, D] with equal shapes");
    if (key->size(1) != c.H_kv || key->size(2) != c.D)
      value_error("caches must be [num_blocks, block_size, H_kv, D]");
    heads_contiguous(key, "key/value must have unit d-stride and head stride D");
    heads_contiguous(value, "key/value must have unit d-stride and head stride D");
    const int code = dtype_code(key->scalar_type(), false);
    if (value->scalar_type() != key->scalar_type()) type_error("key and value must share a dtype");
    if (slots->scalar_type() != at::kLong || slots->numel() != key->size(0))
      type_error("slot_mapping must be int64 [T]");
    check_status(status);
    const at::Tensor s = slots->is_contiguous() ? *slots : slots->contiguous();
    const c10::cuda::CUDAGuard guard(dev);
    call(lk_store_kv_q8, ptr(key), ptr(value), ptr(c.kd), ptr<float>(c.ks), ptr(c.vd),
         ptr<float>(c.vs), static_cast<const int64_t*>(s.data_ptr()), n32(key->size(0)), n32(c.H_kv),
         n32(c.D), key->stride(0), value->stride(0), c.nb, n32(c.bs), code, c.fmt,
         ptr<int32_t>(status), stream_of(dev));
    Py_RETURN_NONE;
  });
}

// load(key_cache, value_cache, block_tables, context_lens, cu_rows, num_rows, dtype, key_out,
//      value_out, status)
PyObject* load(PyObject*, PyObject* const* a, Py_ssize_t) {
  return guarded([&]() -> PyObject* {
    const Caches c = caches(a[0], a[1], false);
    T bt = tensor(a[2]), ctx = tensor(a[3]), cu = tensor(a[4]);
    const T ko = tensor(a[7], true), vo = tensor(a[8], true), status = tensor(a[9], true);
    const int dev = device_of({c.kd, c.ks, c.vd, c.vs, bt, ctx, cu, ko, vo, status});
    if (bt->scalar_type() != at::kInt || bt->dim() != 2) type_error("block_tables must be int32 [B, max_blocks]");
    const int64_t B = bt->size(0), max_blocks = bt->size(1), rows = integer(a[5]);
    at::Tensor bt_keep, ctx_keep, cu_keep;
    if (max_blocks > 0 && bt->stride(1) != 1) {
      bt_keep = bt->contiguous();
      bt = &bt_keep;
    }
    ctx = int32_row(ctx, B, "context_lens must be int32 [B]", ctx_keep);
    cu = int32_row(cu, B + 1, "cu_rows must be int32 [B + 1]", cu_keep);
    check_status(status);
    if (rows < 0) value_error("num_rows must not be negative");
    if (!THPDtype_Check(a[6])) type_error("dtype must be a torch.dtype");
    const at::ScalarType type = reinterpret_cast<THPDtype*>(a[6])->scalar_type;
    const int code = dtype_code(type, true);
    const c10::cuda::CUDAGuard guard(dev);
    at::Tensor outs[2];
    const T given[2] = {ko, vo};
    for (int i = 0; i < 2; ++i) {
      if (!given[i]) {
        outs[i] = at::empty({rows, c.H_kv, c.D}, c.kd->options().dtype(type));
      } else {
        outs[i] = *given[i];
        if (outs[i].dim() != 3 || outs[i].size(0) != rows || outs[i].size(1) != c.H_kv ||
            outs[i].size(2) != c.D || outs[i].scalar_type() != type || !outs[i].is_contiguous())
          value_error("key_out/value_out must be contiguous [num_rows, H_kv, D] of dtype");
      }
    }
    auto whole = [](const at::Tensor& t) {
      return Rows{static_cast<const char*>(t.data_ptr()), 1, static_cast<int64_t>(t.nbytes()), 0};
    };
    if (meet(whole(outs[0]), whole(outs[1])))
      value_error("key_out and value_out must be different tensors that do not overlap");
    call(lk_load_kv_q8, outs[0].data_ptr(), outs[1].data_ptr(), ptr(c.kd), ptr<float>(c.ks),
         ptr(c.vd), ptr<float>(c.vs), ptr<int32_t>(bt), bt->stride(0), ptr<int32_t>(ctx),
         ptr<int32_t>(cu), n32(B), rows, n32(c.H_kv), n32(c.D), c.nb, n32(c.bs), n32(max_blocks),
         code, c.fmt, ptr<int32_t>(status), stream_of(dev));
    PyObject* t = PyTuple_New(2);
    if (!t) throw PyRaised();
    for (int i = 0; i < 2; ++i) {
      PyObject* o = given[i] ? Py_NewRef(a[7 + i]) : THPVariable_Wrap(outs[i]);
      PyTuple_SET_ITEM(t, i, o);
    }
    return t;
  });
}

// load_blocks(key_cache, value_cache, block_tables, context_lens, dtype, status)
PyObject* load_blocks(PyObject*, PyObject* const* a, Py_ssize_t) {
  return guarded([&]() -> PyObject* {
    const Caches c = caches(a[0], a[1], false);
    T bt = tensor(a[2]), ctx = tensor(a[3]);
    const T status = tensor(a[5], true);
    const int dev = device_of({c.kd, c.ks, c.vd, c.vs, bt, ctx, status});
    if (bt->scalar_type() != at::kInt || bt->dim() != 2) type_error("block_tables must be int32 [B, max_blocks]");
    const int64_t B = bt->size(0), max_blocks = bt->size(1);
    at::Tensor bt_keep, ctx_keep;
    if (max_blocks > 0 && bt->stride(1) != 1) {
      bt_keep = bt->contiguous();
      bt = &bt_keep;
    }
    ctx = int32_row(ctx, B, "context_lens must be int32 [B]", ctx_keep);
    check_status(status);
    if (!THPDtype_Check(a[4])) type_error("dtype must be a torch.dtype");
    const at::ScalarType type = reinterpret_cast<THPDtype*>(a[4])->scalar_type;
    const int code = dtype_code(type, true);
    const c10::cuda::CUDAGuard guard(dev);
    const at::Tensor outs[3] = {at::empty({B * max_blocks, c.bs, c.H_kv, c.D}, c.kd->options().dtype(type)),
                                at::empty({B * max_blocks, c.bs, c.H_kv, c.D}, c.kd->options().dtype(type)),
                                at::empty({B, max_blocks}, c.kd->options().dtype(at::kInt))};
    call(lk_load_kv_q8_blocks, outs[0].data_ptr(), outs[1].data_ptr(), ptr<int32_t>(&outs[2]), ptr(c.kd),
         ptr<float>(c.ks), ptr(c.vd), ptr<float>(c.vs), ptr<int32_t>(bt), bt->stride(0), ptr<int32_t>(ctx),
         n32(B), n32(c.H_kv), n32(c.D), c.nb, n32(c.bs), n32(max_blocks), code, c.fmt,
         ptr<int32_t>(status), stream_of(dev));
    PyObject* t = PyTuple_New(3);
    if (!t) throw PyRaised();
    for (int i = 0; i < 3; ++i) PyTuple_SET_ITEM(t, i, THPVariable_Wrap(outs[i]));
    return t;
  });
}

// tree(query, key_cache, value_cache, block_tables, context_lens, cu_seqlens_q, max_q_len, scale,
//      tree_mask, out, workspace, status); max_q_len None: decode over an 8-bit cache
PyObject* tree(PyObject*, PyObject* const* a, Py_ssize_t) {
  return guarded([&]() -> PyObject* {
    const bool decode = a[6] == Py_None;
    if (decode && a[5] != Py_None) type_error("max_q_len must be an integer");
    const Caches c = caches(a[1], a[2], !decode);
    const T query = tensor(a[0]), mask_in = tensor(a[8], true), out_in = tensor(a[9], true);
    T bt = tensor(a[3]), ctx = tensor(a[4]), cu = tensor(a[5], decode);
    const T ws_in = tensor(a[10], true), status = tensor(a[11], true);
    const int dev =
        device_of({query, c.kd, c.ks, c.vd, c.vs, bt, ctx, cu, mask_in, out_in, ws_in, status});
    if (query->dim() != 3) value_error("query must be [T, H, D]");
    if (c.fmt == LK_KV_16BIT && (c.kd->scalar_type() != query->scalar_type() ||
                                 c.vd->scalar_type() != query->scalar_type()))
      type_error("query dtype must match the cache dtype");
    const int64_t n = query->size(0), H = query->size(1), D = query->size(2);
    if (c.D != D) value_error("cache shape mismatch");
    heads_contiguous(query, "query must have unit d-stride and head stride D");
    if (bt->scalar_type() != at::kInt || bt->dim() != 2) type_error("block_tables must be int32 [B, max_blocks]");
    const int64_t B = bt->size(0), max_blocks = bt->size(1), max_q = decode ? 1 : integer(a[6]);
    if (max_q < 0) value_error("max_q_len must not be negative");
    if (decode && B != n) value_error("decode takes one query per row of block_tables");
    at::Tensor bt_keep, ctx_keep, cu_keep, mask_keep;
    if (max_blocks > 0 && bt->stride(1) != 1) {
      bt_keep = bt->contiguous();
      bt = &bt_keep;
    }
    ctx = int32_row(ctx, B, "context_lens must be int32 [B]", ctx_keep);
    if (cu) cu = int32_row(cu, B + 1, "cu_seqlens_q must be int32 [B + 1]", cu_keep);
    T mask = mask_in;
    if (mask) {
      if (mask->scalar_type() != at::kLong || mask->dim() != 2 || mask->size(0) != n)
        type_error("tree_mask must be int64 [T, words]");
      if (mask->size(1) * 64 < max_q) value_error("tree_mask must have a bit for each of max_q_len tokens");
      if (mask->stride(1) != 1) {
        mask_keep = mask->contiguous();
        mask = &mask_keep;
      }
    }
    const int code = dtype_code(query->scalar_type(), false);
    check_status(status);
    const double scale = PyFloat_AsDouble(a[7]);
    if (scale == -1.0 && PyErr_Occurred()) throw PyRaised();
    const c10::cuda::CUDAGuard guard(dev);
    at::Tensor out;
    if (!out_in) {
      out = at::empty({n, H, D}, query->options());
    } else {
      out = *out_in;
      if (out.dim() != 3 || out.sizes() != query->sizes() || out.scalar_type() != query->scalar_type() ||
          out.stride(2) != 1 || out.stride(1) != D || (n > 1 && out.stride(0) < H * D))
        value_error("bad out tensor");
      const int64_t esz = query->element_size();
      const Rows from = {static_cast<const char*>(query->data_ptr()), n, H * D * esz, query->stride(0) * esz},
                 to = {static_cast<const char*>(out.data_ptr()), n, H * D * esz, out.stride(0) * esz};
      if ((from.at != to.at || (n > 1 && from.stride != to.stride)) && meet(from, to))
        value_error("out must be the query itself or not overlap it");
    }
    auto result = [&]() { return out_in ? Py_NewRef(a[9]) : THPVariable_Wrap(out); };
    if (n == 0 || B == 0 || max_q == 0) return result();
    // The partials of split contexts live in a buffer of this call's own unless the
    // caller gives one: calls on other streams and captured graphs never share it.
    const size_t need = lk_paged_tree_workspace_bytes(n32(n), n32(B), n32(max_q), n32(H), n32(c.H_kv),
                                                      n32(D), n32(c.bs), n32(max_blocks), c.fmt);
    at::Tensor ws;
    void* ws_ptr = nullptr;
    size_t ws_bytes = 0;
    if (ws_in) {
      if (!ws_in->is_contiguous()) value_error("workspace must be contiguous");
      ws_ptr = ws_in->data_ptr();
      ws_bytes = ws_in->nbytes();
      if (ws_bytes < need) {
        PyErr_Format(PyExc_ValueError, "workspace too small: need %zu bytes", need);
        throw PyRaised();
      }
    } else if (need > 0) {
      ws = at::empty({static_cast<int64_t>(need)}, query->options().dtype(at::kByte));
      ws_ptr = ws.data_ptr();
      ws_bytes = need;
    }
    call(lk_paged_tree_attention, out.data_ptr(), out.stride(0), ptr(query), query->stride(0),
         ptr(c.kd), ptr<float>(c.ks), ptr(c.vd), ptr<float>(c.vs), c.nb, ptr<int32_t>(bt),
         bt->stride(0), ptr<int32_t>(cu), ptr<int32_t>(ctx), ptr<int64_t>(mask),
         mask ? mask->stride(0) : 0, mask ? n32(mask->size(1)) : 0, n32(n), n32(B), n32(max_q), n32(H),
         n32(c.H_kv), n32(D), n32(c.bs), n32(max_blocks), static_cast<float>(scale), code, c.fmt,
         ws_ptr, ws_bytes, ptr<int32_t>(status), stream_of(dev));
    return result();
  });
}

// logits(logits, prompt_ids, prompt_lens, output_ids, output_lens, repetition, presence, frequency,
//        bias_ids, bias, allowed, out, status)
PyObject* logits(PyObject*, PyObject* const* a, Py_ssize_t) {
  return guarded([&]() -> PyObject* {
    T x = tensor(a[0]);
    const T prompt = tensor(a[1], true), plens = tensor(a[2], true), output = tensor(a[3], true),
            olens = tensor(a[4], true), bias_ids = tensor(a[8], true), bias = tensor(a[9], true),
            allowed = tensor(a[10], true), out_in = tensor(a[11], true), status = tensor(a[12], true);
    const T row_terms[3] = {tensor(a[5], true), tensor(a[6], true), tensor(a[7], true)};
    const int dev = device_of({x, prompt, plens, output, olens, row_terms[0], row_terms[1], row_terms[2],
                               bias_ids, bias, allowed, out_in, status});
    if (x->dim() != 2 || x->size(1) == 0) value_error("logits must be [B, V]");
    const int64_t B = x->size(0), V = x->size(1);
    const int code = dtype_code(x->scalar_type(), true);
    at::Tensor keep[12];
    // rows of their own, unit column stride: a copy if need be
    auto rows = [&](T t, int slot) -> T {
      if (t->size(1) == 0 || (t->stride(1) == 1 && (B <= 1 || t->stride(0) >= t->size(1)))) return t;
      keep[slot] = t->contiguous();
      return &keep[slot];
    };
    auto ld = [](T t) { return t ? std::max(t->stride(0), t->size(1)) : int64_t{0}; };
    const T x_rows = rows(x, 0);
    if (x_rows != x && out_in && out_in->data_ptr() == x->data_ptr())
      value_error("in place, logits must have unit column stride and rows of their own");
    x = x_rows;
    auto ids = [&](T t, T lens, const char* text, const char* lens_text, int slot) -> std::pair<T, T> {
      if (!t) return {nullptr, nullptr};
      if (t->scalar_type() != at::kLong || t->dim() != 2 || t->size(0) != B) type_error(text);
      return {rows(t, slot), lens ? int32_row(lens, B, lens_text, keep[slot + 1]) : nullptr};
    };
    const auto [p, pl] = ids(prompt, plens, "prompt_ids must be int64 [B, L]", "prompt_lens must be int32 [B]", 1);
    const auto [o, ol] = ids(output, olens, "output_ids must be int64 [B, L]", "output_lens must be int32 [B]", 3);
    static const char* const names[3] = {"repetition must be fp32 [B]", "presence must be fp32 [B]",
                                         "frequency must be fp32 [B]"};
    T term[3];
    for (int i = 0; i < 3; ++i) {
      term[i] = row_terms[i];
      if (!term[i]) continue;
      if (term[i]->scalar_type() != at::kFloat || term[i]->numel() != B) type_error(names[i]);
      if (!term[i]->is_contiguous()) {
        keep[5 + i] = term[i]->contiguous();
        term[i] = &keep[5 + i];
      }
    }
    T bi = bias_ids, bv = bias;
    if (!bi != !bv) value_error("bias_ids and bias go together");
    if (bi) {
      if (bi->scalar_type() != at::kLong || bi->dim() != 2 || bi->size(0) != B) type_error("bias_ids must be int64 [B, n]");
      if (bv->scalar_type() != at::kFloat || bv->sizes() != bi->sizes()) type_error("bias must be fp32 [B, n]");
      if (!bi->is_contiguous()) bi = &(keep[8] = bi->contiguous());
      if (!bv->is_contiguous()) bv = &(keep[9] = bv->contiguous());
    }
    T al = allowed;
    if (al) {
      if (al->scalar_type() != at::kInt || al->dim() != 2 || al->size(0) != B || al->size(1) * 32 < V)
        type_error("allowed must be int32 [B, >= ceil(V / 32)]");
      al = rows(al, 10);
    }
    check_status(status);
    const c10::cuda::CUDAGuard guard(dev);
    at::Tensor out;
    if (!out_in) {
      out = at::empty({B, V}, x->options());
    } else {
      out = *out_in;
      if (out.dim() != 2 || out.size(0) != B || out.size(1) != V || out.scalar_type() != x->scalar_type() ||
          out.stride(1) != 1 || (B > 1 && out.stride(0) < V))
        value_error("out must be [B, V] of the logits' dtype with unit column stride");
      const int64_t esz = x->element_size(), out_ld = std::max(out.stride(0), V);
      const Rows from = {static_cast<const char*>(x->data_ptr()), B, V * esz, ld(x) * esz},
                 to = {static_cast<const char*>(out.data_ptr()), B, V * esz, out_ld * esz};
      if ((from.at != to.at || from.stride != to.stride) && meet(from, to))
        value_error("out must be the logits themselves or not overlap them");
    }
    if (B > 0)
      call(lk_process_logits, out.data_ptr(), std::max(out.stride(0), V), ptr(x), n32(B), n32(V),
           ld(x), ptr<int64_t>(p), ld(p), ptr<int32_t>(pl), p ? n32(p->size(1)) : 0, ptr<int64_t>(o),
           ld(o), ptr<int32_t>(ol), o ? n32(o->size(1)) : 0, ptr<float>(term[0]), ptr<float>(term[1]),
           ptr<float>(term[2]), ptr<int64_t>(bi), ptr<float>(bv), bi ? n32(bi->size(1)) : 0,
           ptr<int32_t>(al), ld(al), code, ptr<int32_t>(status), stream_of(dev));
    return out_in ? Py_NewRef(a[11]) : THPVariable_Wrap(out);
  });
}

// init(QuantizedCache, LiteKernError)
PyObject* init(PyObject*, PyObject* const* a, Py_ssize_t) {
  g_cache_type = reinterpret_cast<PyTypeObject*>(Py_NewRef(a[0]));
  g_error = Py_NewRef(a[1]);
  Py_RETURN_NONE;
}

// Arguments are positional and complete; the count is checked here for all.
template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t), int N>
PyObject* exactly(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "expected %d arguments, got %zd", N, n);
    return nullptr;
  }
  return F(self, a, n);
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t), int N>
PyMethodDef method(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(exactly<F, N>)), METH_FASTCALL,
          nullptr};
}

PyMethodDef g_methods[] = {method<init, 2>("init"),   method<store, 6>("store"), method<load, 10>("load"),
                           method<load_blocks, 6>("load_blocks"), method<tree, 12>("tree"),
                           method<logits, 13>("logits"), {nullptr, nullptr, 0, nullptr}};

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_spec", nullptr, -1, g_methods};

}  // namespace

PyMODINIT_FUNC PyInit__spec() {
  PyObject* m = PyModule_Create(&g_module);
  // the loader compares it with the torch it is loaded beside
  if (m && PyModule_AddStringConstant(m, "torch_version", LK_TORCH_VERSION) < 0) Py_CLEAR(m);
  return m;
}
