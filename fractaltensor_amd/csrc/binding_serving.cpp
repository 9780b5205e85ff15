// _serving: the entry points on a paged cache of keys and values and the verification of drafted tokens, for callers that hold torch
// tensors, as a CPython module in the manner of _fast (binding.cpp): checked, allocated and launched in one native call, and
// None, with nothing done, for whatever is not plainly right.  A call runs on the device of its tensors, on that device's current stream.
#include <c10/core/DeviceGuard.h>

#include "binding_common.h"

namespace {

// FTK_* of include/ftk.h, -1 for what it does not name
int type_code(at::ScalarType t) {
  switch (t) {
    case at::kHalf: return FTK_F16;
    case at::kBFloat16: return FTK_BF16;
    case at::ScalarType::Float8_e4m3fn: return FTK_E4M3;
    case at::kChar: return FTK_INT8;
    case at::kFloat: return FTK_F32;
    default: return -1;
  }
}

bool on(PyObject* o, const at::Tensor& with) { return is_tensor(o) && tensor_of(o).device() == with.device(); }
bool plain_on(PyObject* o, at::ScalarType type, const at::Tensor& with) { return plain(o, type) && on(o, with); }
bool small(int64_t n) { return n >= 0 && n <= INT_MAX; }

bool number(PyObject* o, int* out) {
  if (!PyLong_Check(o)) return false;
  const long long v = PyLong_AsLongLong(o);
  if (v < 0 || v > INT_MAX) {
    PyErr_Clear();
    return false;
  }
  *out = (int)v;
  return true;
}

// The cache and the batch out of k_pages, v_pages, table, lens, starts, k_exps, v_exps.
struct Cache {
  ftk_kv_pages pages;
  ftk_kv_batch batch;
};
bool cache_of(PyObject* const* a, int64_t tokens, Cache* c) {
  if (!is_tensor(a[0]) || !is_tensor(a[1])) return false;
  const at::Tensor &k = tensor_of(a[0]), &v = tensor_of(a[1]);
  const int type = type_code(k.scalar_type());
  if (type < 0 || type == FTK_F32 || !plain(a[0], k.scalar_type()) || !plain_on(a[1], k.scalar_type(), k) || k.dim() != 4 || k.sizes() != v.sizes()) return false;
  for (int i = 0; i < 4; ++i)
    if (!small(k.size(i))) return false;
  if (!plain_on(a[2], at::kInt, k) || !plain_on(a[3], at::kInt, k) || !plain_on(a[4], at::kInt, k)) return false;
  const at::Tensor &table = tensor_of(a[2]), &lens = tensor_of(a[3]), &starts = tensor_of(a[4]);
  if (table.dim() != 2 || lens.dim() != 1 || starts.dim() != 1 || table.size(0) != lens.size(0) || starts.size(0) != lens.size(0) + 1) return false;
  if (!small(table.size(0)) || !small(table.size(1)) || !small(tokens)) return false;
  c->pages = {k.data_ptr(), v.data_ptr(), nullptr, nullptr, type, dim(k, 0), dim(k, 1), dim(k, 2), dim(k, 3)};
  if (type == FTK_E4M3 || type == FTK_INT8) {
    for (int i = 5; i < 7; ++i) {
      if (!plain_on(a[i], at::kChar, k)) return false;
      const at::Tensor& e = tensor_of(a[i]);
      if (e.dim() != 3 || e.size(0) != k.size(0) || e.size(1) != k.size(1) || e.size(2) != k.size(2)) return false;
      (i == 5 ? c->pages.k_exps : c->pages.v_exps) = e.data_ptr();
    }
  } else if (a[5] != Py_None || a[6] != Py_None) {
    return false;
  }
  c->batch = {(const int*)table.data_ptr(), (const int*)lens.data_ptr(), (const int*)starts.data_ptr(), dim(table, 0), dim(table, 1), (int)tokens};
  return true;
}

// Rows [tokens, heads, D] whose elements of a head are neighbours; strides of dimensions of one are nobody's.
struct Strided {
  void* data;
  long long token, head;
};
bool strided(PyObject* o, at::ScalarType type, const at::Tensor& with, int64_t heads, int64_t D, Strided* s) {
  if (!on(o, with)) return false;
  const at::Tensor& t = tensor_of(o);
  if (t.scalar_type() != type || t.dim() != 3 || (heads > 0 && t.size(1) != heads) || t.size(2) != D || t.stride(2) != 1) return false;
  s->data = t.data_ptr();
  s->token = t.size(0) > 1 ? t.stride(0) : 0;
  s->head = t.size(1) > 1 ? t.stride(1) : 0;
  return s->token % 8 == 0 && s->head % 8 == 0;
}

// kv_cache_write(keys, values, k_pages, v_pages, table, lens, starts, k_exps, v_exps) -> True
PyObject* kv_cache_write(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 9 || !is_tensor(a[0]) || !is_tensor(a[1])) Py_RETURN_NONE;
    const at::Tensor &keys = tensor_of(a[0]), &values = tensor_of(a[1]);
    if (!keys.is_cuda() || keys.dim() != 3 || values.dim() != 3 || keys.size(0) != values.size(0)) Py_RETURN_NONE;
    const int type = type_code(keys.scalar_type());
    Cache c;
    if ((type != FTK_F16 && type != FTK_BF16) || !cache_of(a + 2, keys.size(0), &c) || !on(a[2], keys)) Py_RETURN_NONE;
    if ((c.pages.type == FTK_F16 || c.pages.type == FTK_BF16) && c.pages.type != type) Py_RETURN_NONE;
    Strided k, v;
    if (!strided(a[0], keys.scalar_type(), keys, c.pages.heads, c.pages.head_size, &k) ||
        !strided(a[1], keys.scalar_type(), keys, c.pages.heads, c.pages.head_size, &v))
      Py_RETURN_NONE;
    if (!count("kv_cache_write")) return nullptr;
    const c10::DeviceGuard guard(keys.device());
    void* const s = stream();
    const int rc = in_library([&] { return ftk_kv_cache_write(k.data, v.data, type, k.token, k.head, v.token, v.head, &c.pages, &c.batch, s); });
    if (rc) return raise(rc);
    Py_RETURN_TRUE;
  });
}

// kv_cache_read(dtype tensor, k_pages, v_pages, table, lens, starts, k_exps, v_exps, tokens, out keys or None, out values or None)
//   -> (keys, values).  The first argument is a tensor of the type that is asked for.
PyObject* kv_cache_read(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    int tokens;
    if (n != 11 || !is_tensor(a[0]) || !number(a[8], &tokens)) Py_RETURN_NONE;
    const auto out_type = tensor_of(a[0]).scalar_type();
    const int type = type_code(out_type);
    Cache c;
    if (!cache_of(a + 1, tokens, &c)) Py_RETURN_NONE;
    if (type != FTK_F16 && type != FTK_BF16 && type != FTK_F32) Py_RETURN_NONE;
    const at::Tensor& pages = tensor_of(a[1]);
    at::Tensor out[2];
    for (int i = 0; i < 2; ++i) {
      if (a[9 + i] == Py_None) {
        out[i] = empty({tokens, c.pages.heads, c.pages.head_size}, out_type, pages);
      } else {
        if (!plain_on(a[9 + i], out_type, pages)) Py_RETURN_NONE;
        out[i] = tensor_of(a[9 + i]);
        if (out[i].dim() != 3 || out[i].size(0) != tokens || out[i].size(1) != c.pages.heads || out[i].size(2) != c.pages.head_size) Py_RETURN_NONE;
      }
    }
    if (!count("kv_cache_read")) return nullptr;
    const c10::DeviceGuard guard(pages.device());
    void *const k = out[0].data_ptr(), *const v = out[1].data_ptr(), *const s = stream();
    const int rc = in_library([&] { return ftk_kv_cache_read(&c.pages, &c.batch, type, k, v, s); });
    if (rc) return raise(rc);
    PyObject* both = PyTuple_New(2);
    if (!both) return nullptr;
    for (int i = 0; i < 2; ++i) PyTuple_SET_ITEM(both, i, THPVariable_Wrap(std::move(out[i])));
    return both;
  });
}

// paged_attention(q, k_pages, v_pages, table, lens, starts, k_exps, v_exps, scale or None, causal, window, max_queries, max_keys, out or None,
//                 lse (True: allocated, False: none, or a tensor), workspace or None) -> (o, lse or None)
PyObject* paged_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 16 || !is_tensor(a[0])) Py_RETURN_NONE;
    const at::Tensor& q = tensor_of(a[0]);
    if (!q.is_cuda() || q.dim() != 3 || !small(q.size(1))) Py_RETURN_NONE;
    const int type = type_code(q.scalar_type());
    Cache c;
    Strided st;
    if ((type != FTK_F16 && type != FTK_BF16) || !cache_of(a + 1, q.size(0), &c) || !on(a[1], q)) Py_RETURN_NONE;
    if ((c.pages.type == FTK_F16 || c.pages.type == FTK_BF16) && c.pages.type != type) Py_RETURN_NONE;
    if (!strided(a[0], q.scalar_type(), q, 0, c.pages.head_size, &st)) Py_RETURN_NONE;
    double scale = 1.0 / std::sqrt((double)c.pages.head_size);
    if (a[8] != Py_None) {
      if (!PyFloat_Check(a[8]) && !PyLong_Check(a[8])) Py_RETURN_NONE;
      scale = PyFloat_AsDouble(a[8]);
      if (PyErr_Occurred()) return nullptr;
    }
    int window, max_queries, max_keys;
    if ((a[9] != Py_True && a[9] != Py_False) || !number(a[10], &window) || !number(a[11], &max_queries) || !number(a[12], &max_keys)) Py_RETURN_NONE;
    at::Tensor o, lse, ws;
    if (a[13] == Py_None) {
      o = empty(q.sizes(), q.scalar_type(), q);
    } else {
      if (!plain_on(a[13], q.scalar_type(), q) || tensor_of(a[13]).sizes() != q.sizes()) Py_RETURN_NONE;
      o = tensor_of(a[13]);
    }
    if (a[14] == Py_True) {
      lse = empty({q.size(0), q.size(1)}, at::kFloat, q);
    } else if (a[14] != Py_False) {
      if (!plain_on(a[14], at::kFloat, q)) Py_RETURN_NONE;
      lse = tensor_of(a[14]);
      if (lse.dim() != 2 || lse.size(0) != q.size(0) || lse.size(1) != q.size(1)) Py_RETURN_NONE;
    }
    const c10::DeviceGuard guard(q.device());
    const int heads = dim(q, 1);
    if (a[15] != Py_None) {
      if (!on(a[15], q) || !tensor_of(a[15]).is_contiguous()) Py_RETURN_NONE;
      ws = tensor_of(a[15]);
    } else if (const size_t need = ftk_paged_attn_workspace_bytes(&c.pages, &c.batch, heads, window, max_queries, max_keys)) {
      ws = empty({(int64_t)need}, at::kByte, q);
    }
    if (!count("paged_attention")) return nullptr;
    void *const op = o.data_ptr(), *const wp = ws.defined() && ws.nbytes() ? ws.data_ptr() : nullptr, *const s = stream();
    float* const lp = lse.defined() ? (float*)lse.data_ptr() : nullptr;
    const size_t bytes = wp ? ws.nbytes() : 0;
    const bool causal = a[9] == Py_True;
    const int rc = in_library([&] {
      return ftk_paged_attn(st.data, type, st.token, st.head, &c.pages, &c.batch, op, lp, heads, (float)scale, causal, window, max_queries, max_keys, wp, bytes, s);
    });
    if (rc) return raise(rc);
    PyObject* both = PyTuple_New(2);
    if (!both) return nullptr;
    PyTuple_SET_ITEM(both, 0, THPVariable_Wrap(std::move(o)));
    if (lse.defined()) {
      PyTuple_SET_ITEM(both, 1, THPVariable_Wrap(std::move(lse)));
    } else {
      Py_INCREF(Py_None);
      PyTuple_SET_ITEM(both, 1, Py_None);
    }
    return both;
  });
}

// verify_drafts(target [B,K+1,V], draft [B,K,V] or None, drafts [B,K], accept [B,K], sample [B], lens [B] or None, workspace or None)
//   -> (tokens, accepted)
PyObject* verify_drafts(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 7 || !is_tensor(a[0]) || !is_tensor(a[2])) Py_RETURN_NONE;
    const at::Tensor &target = tensor_of(a[0]), &drafts = tensor_of(a[2]);
    const int type = type_code(target.scalar_type());
    const auto ids = drafts.scalar_type();
    if ((type != FTK_F16 && type != FTK_BF16 && type != FTK_F32) || !plain(a[0], target.scalar_type()) || target.dim() != 3) Py_RETURN_NONE;
    if ((ids != at::kInt && ids != at::kLong) || !plain_on(a[2], ids, target) || drafts.dim() != 2) Py_RETURN_NONE;
    const int64_t B = target.size(0), K = drafts.size(1), V = target.size(2);
    if (target.size(1) != K + 1 || drafts.size(0) != B || !small(B) || !small(K) || !small(V)) Py_RETURN_NONE;
    const void* draft = nullptr;
    if (a[1] != Py_None) {
      if (!plain_on(a[1], target.scalar_type(), target)) Py_RETURN_NONE;
      const at::Tensor& d = tensor_of(a[1]);
      if (d.dim() != 3 || d.size(0) != B || d.size(1) != K || d.size(2) != V) Py_RETURN_NONE;
      draft = d.data_ptr();
    }
    if (!plain_on(a[3], at::kFloat, target) || !plain_on(a[4], at::kFloat, target)) Py_RETURN_NONE;
    const at::Tensor &accept = tensor_of(a[3]), &sample = tensor_of(a[4]);
    if (accept.dim() != 2 || accept.size(0) != B || accept.size(1) != K || sample.dim() != 1 || sample.size(0) != B) Py_RETURN_NONE;
    const int* lens = nullptr;
    if (a[5] != Py_None) {
      if (!plain_on(a[5], at::kInt, target) || tensor_of(a[5]).dim() != 1 || tensor_of(a[5]).size(0) != B) Py_RETURN_NONE;
      lens = (const int*)tensor_of(a[5]).data_ptr();
    }
    at::Tensor ws;
    if (a[6] != Py_None) {
      if (!on(a[6], target) || !tensor_of(a[6]).is_contiguous()) Py_RETURN_NONE;
      ws = tensor_of(a[6]);
    } else {
      ws = empty({(int64_t)ftk_verify_drafts_workspace_bytes((int)B, (int)V)}, at::kByte, target);
    }
    at::Tensor tokens = empty({B, K + 1}, ids, target), accepted = empty({B}, at::kInt, target);
    if (!count("verify_drafts")) return nullptr;
    const c10::DeviceGuard guard(target.device());
    void *const tp = target.data_ptr(), *const ip = drafts.data_ptr(), *const op = tokens.data_ptr(), *const wp = ws.data_ptr(), *const s = stream();
    const float *const ap = (const float*)accept.data_ptr(), *const sp = (const float*)sample.data_ptr();
    int* const np = (int*)accepted.data_ptr();
    const size_t bytes = ws.nbytes();
    const int rc = in_library(
        [&] { return ftk_verify_drafts(tp, draft, type, ip, ids == at::kLong, ap, sp, lens, op, np, (int)B, (int)K, (int)V, wp, bytes, s); });
    if (rc) return raise(rc);
    PyObject* both = PyTuple_New(2);
    if (!both) return nullptr;
    PyTuple_SET_ITEM(both, 0, THPVariable_Wrap(std::move(tokens)));
    PyTuple_SET_ITEM(both, 1, THPVariable_Wrap(std::move(accepted)));
    return both;
  });
}

PyMethodDef methods[] = {
    {"init", (PyCFunction)(void*)init, METH_FASTCALL, "init(counts, raise)"},
    {"kv_cache_write", (PyCFunction)(void*)kv_cache_write, METH_FASTCALL, "kv_cache_write(keys, values, k_pages, v_pages, table, lens, starts, k_exps, v_exps)"},
    {"kv_cache_read", (PyCFunction)(void*)kv_cache_read, METH_FASTCALL,
     "kv_cache_read(like, k_pages, v_pages, table, lens, starts, k_exps, v_exps, tokens, keys, values)"},
    {"paged_attention", (PyCFunction)(void*)paged_attention, METH_FASTCALL,
     "paged_attention(q, k_pages, v_pages, table, lens, starts, k_exps, v_exps, scale, causal, window, max_queries, max_keys, out, lse, workspace)"},
    {"verify_drafts", (PyCFunction)(void*)verify_drafts, METH_FASTCALL, "verify_drafts(target, draft, drafts, accept, sample, lens, workspace)"},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_serving", "the serving entry points on torch tensors", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__serving(void) { return PyModule_Create(&module); }
