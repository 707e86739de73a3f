// Host fast paths of the Python layer: one call from the interpreter checks the
// tensors, allocates the outputs and launches through the C ABI.
//
// A denoising step of one short request is bound by the host: per layer the
// Python form of Attention.forward and RotaryEmbedding.forward spent 11 and 14
// us (attribute reads, views, 20-odd ctypes conversions) on launches whose
// kernels take 9 and 3 us; these forms take 7 and 5.  The step of one 384-token
// request over 32 layers, whose kernels sum to about 400 us: 1047 -> 522 us, which
// still varies with the host.  Every function here takes the ordinary case only
// and returns None for anything else -- another type, layout, device or tensor
// class, and what the C ABI refuses before it launches anything -- and the Python
// form, which raises what is to be raised, runs then.  A failure of the HIP
// runtime raises here: the launch may be on the stream already, and a second run
// would rotate in place, or unmask, twice.  Nothing is kept between calls.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cstring>
#include <utility>

#include "dllm_attn.h"

namespace {

// The tensor behind `o` when it is a plain strided device tensor of type `ty`.
const at::Tensor* plain(PyObject* o, at::ScalarType ty) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || t.scalar_type() != ty || !t.has_storage())
    return nullptr;
  return &t;
}

// [n, heads * D] or [n, heads, D] with contiguous heads inside a row.
bool token_rows(const at::Tensor& t, int64_t heads, int64_t D) {
  if (t.dim() == 2) return t.size(1) == heads * D && t.stride(1) == 1;
  return t.dim() == 3 && t.size(1) == heads && t.size(2) == D && t.stride(2) == 1 && t.stride(1) == D;
}

template <typename T>
T* ptr(const at::Tensor& t) {
  return reinterpret_cast<T*>(t.data_ptr());
}

void* stream_of(int device) { return c10::hip::getCurrentHIPStream((c10::DeviceIndex)device).stream(); }

// Runs f without the GIL: a launch may wait for a full queue.  (The GIL is taken
// back also when f throws: data_ptr() may, where it has to copy first.)
template <typename F>
int no_gil(F f) {
  struct Released {
    PyThreadState* s = PyEval_SaveThread();
    ~Released() { PyEval_RestoreThread(s); }
  } released;
  return f();
}

template <typename F>
PyObject* guarded(F f) {
  try {
    return f();
  } catch (...) {  // the Python form meets the same condition and reports it
    Py_RETURN_NONE;
  }
}

// What a call returns for a code other than DLLM_OK.
PyObject* refused(const char* what, int rc) {
  if (rc == DLLM_ERR_INVALID_ARG || rc == DLLM_ERR_UNSUPPORTED || rc == DLLM_ERR_WORKSPACE) Py_RETURN_NONE;
  return PyErr_Format(PyExc_RuntimeError, "%s failed (code %d): %s", what, rc, dllm_last_error());
}

// attn(q, k, v, k_cache, v_cache, plan: bytes, scale) -> output or None.
// `plan` is the packed launch description of one step and head shape.
struct PlanArgs {
  int64_t device, rows, Hq, Hkv, D;
  int64_t n_dense, max_q_dense, cu, dense_ids;
  int64_t n_cached, max_q_cached, max_keys_cached, cached_ids, slots, slot_off, ws, ws_bytes;
};
// Behind it where the cached rows are in 8-bit pages.
struct PageArgs {
  int64_t max_keep, rows, keeps, table, max_pages, lens;
};

// An 8-bit cache (uint8 [pages, heads, bytes of a page]), or null.
const at::Tensor* pages_of(PyObject* o, int64_t heads, int device) {
  const at::Tensor* t = plain(o, at::kByte);
  if (!t || t->get_device() != device || t->dim() != 3 || t->size(1) != heads ||
      t->size(2) != (int64_t)dllm_quant_page_bytes(128) || !t->is_contiguous())
    return nullptr;
  return t;
}

PyObject* attn(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 7 || !PyBytes_CheckExact(a[5]) || !PyFloat_CheckExact(a[6])) Py_RETURN_NONE;
  const bool paged = PyBytes_GET_SIZE(a[5]) == (Py_ssize_t)(sizeof(PlanArgs) + sizeof(PageArgs));
  if (!paged && PyBytes_GET_SIZE(a[5]) != (Py_ssize_t)sizeof(PlanArgs)) Py_RETURN_NONE;
  return guarded([&]() -> PyObject* {
    PlanArgs p;
    PageArgs pg = {};
    std::memcpy(&p, PyBytes_AS_STRING(a[5]), sizeof(p));
    if (paged) std::memcpy(&pg, PyBytes_AS_STRING(a[5]) + sizeof(p), sizeof(pg));
    const at::Tensor *q = plain(a[0], at::kBFloat16), *k = plain(a[1], at::kBFloat16), *v = plain(a[2], at::kBFloat16);
    if (!q || !k || !v || q->get_device() != p.device || k->get_device() != p.device || v->get_device() != p.device ||
        !token_rows(*q, p.Hq, p.D) || !token_rows(*k, p.Hkv, p.D) || !token_rows(*v, p.Hkv, p.D) ||
        q->size(0) != p.rows || k->size(0) != p.rows || v->size(0) != p.rows)
      Py_RETURN_NONE;
    const at::Tensor *kc = nullptr, *vc = nullptr;
    int64_t cache_slots = 0;
    if (paged) {
      kc = pages_of(a[3], p.Hkv, (int)p.device);
      vc = pages_of(a[4], p.Hkv, (int)p.device);
      if (!kc || !vc || kc->numel() == 0 || vc->numel() == 0 || p.D != 128) Py_RETURN_NONE;
      if (std::min(kc->size(0), vc->size(0)) > INT32_MAX) Py_RETURN_NONE;
    } else if (p.n_cached) {
      kc = plain(a[3], at::kBFloat16);
      vc = plain(a[4], at::kBFloat16);
      for (const at::Tensor* t : {kc, vc})
        if (!t || t->get_device() != p.device || t->numel() == 0 || t->dim() < 2 || !t->is_contiguous() ||
            t->size(-1) != p.D || t->size(-2) != p.Hkv)
          Py_RETURN_NONE;
      cache_slots = std::min(kc->numel(), vc->numel()) / (p.Hkv * p.D);
    }
    at::Tensor o = at::empty_like(*q);
    const float scale = (float)PyFloat_AS_DOUBLE(a[6]);
    void* st = stream_of((int)p.device);
    auto dev_i32 = [](int64_t x) { return reinterpret_cast<const int32_t*>(x); };
    const char* what = "dllm_attn_varlen_fwd";
    const int rc = no_gil([&] {
      int r = DLLM_OK;
      if (p.n_dense)
        r = dllm_attn_varlen_fwd(ptr<dllm_bf16>(*q), ptr<dllm_bf16>(*k), ptr<dllm_bf16>(*v), ptr<dllm_bf16>(o),
                                 dev_i32(p.cu), dev_i32(p.cu), dev_i32(p.dense_ids), (int)p.n_dense,
                                 (int)p.max_q_dense, (int)p.max_q_dense, (int)p.Hq, (int)p.Hkv, (int)p.D, q->stride(0),
                                 k->stride(0), v->stride(0), o.stride(0), scale, st);
      if (r == DLLM_OK && paged) {
        what = "dllm_attn_chunk_paged_fwd";
        r = dllm_attn_chunk_paged_fwd(ptr<dllm_bf16>(*q), ptr<dllm_bf16>(*k), ptr<dllm_bf16>(*v), ptr<dllm_bf16>(o),
                                      dev_i32(p.cu), dev_i32(p.cached_ids), (int)p.n_cached, (int)p.max_q_cached,
                                      (int)pg.max_keep, pg.rows, pg.keeps, kc->data_ptr(), vc->data_ptr(), DLLM_CACHE_FP8,
                                      (int)std::min(kc->size(0), vc->size(0)), dev_i32(pg.table), (int)pg.max_pages,
                                      dev_i32(pg.lens), 0, (int)p.Hq, (int)p.Hkv, (int)p.D, q->stride(0), k->stride(0),
                                      v->stride(0), o.stride(0), scale, reinterpret_cast<void*>(p.ws), (size_t)p.ws_bytes,
                                      st);
      } else if (r == DLLM_OK && p.n_cached) {
        what = "dllm_attn_block_cached_fwd";
        r = dllm_attn_block_cached_fwd(ptr<dllm_bf16>(*q), ptr<dllm_bf16>(*k), ptr<dllm_bf16>(*v), ptr<dllm_bf16>(o),
                                       dev_i32(p.cu), dev_i32(p.cached_ids), (int)p.n_cached, (int)p.max_q_cached,
                                       (int)p.max_keys_cached, ptr<dllm_bf16>(*kc), ptr<dllm_bf16>(*vc), cache_slots,
                                       dev_i32(p.slots), dev_i32(p.slot_off), (int)p.Hq, (int)p.Hkv, (int)p.D,
                                       q->stride(0), k->stride(0), v->stride(0), o.stride(0), scale,
                                       reinterpret_cast<void*>(p.ws), (size_t)p.ws_bytes, st);
      }
      return r;
    });
    if (rc != DLLM_OK) return refused(what, rc);
    return THPVariable_Wrap(o.dim() == 2 ? std::move(o) : o.view({-1, p.Hq * p.D}));
  });
}

// quant_copy(key, value, k_cache, v_cache, slot_mapping, store) -> True or None
PyObject* quant_copy(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 6 || !PyBool_Check(a[5])) Py_RETURN_NONE;
  const bool store = a[5] == Py_True;
  return guarded([&]() -> PyObject* {
    const at::Tensor *k = plain(a[0], at::kBFloat16), *v = plain(a[1], at::kBFloat16), *slot = plain(a[4], at::kInt);
    if (!k || !v || !slot || k->dim() != 3 || !token_rows(*k, k->size(1), 128) || k->size(0) > INT32_MAX ||
        v->dim() != 3 || !token_rows(*v, k->size(1), 128) || v->size(0) != k->size(0) || slot->numel() != k->size(0) ||
        !slot->is_contiguous())
      Py_RETURN_NONE;
    const int dev = k->get_device();
    const at::Tensor *kp = pages_of(a[2], k->size(1), dev), *vp = pages_of(a[3], k->size(1), dev);
    if (!kp || !vp || v->get_device() != dev || slot->get_device() != dev || c10::hip::current_device() != dev)
      Py_RETURN_NONE;
    void* st = stream_of(dev);
    const int rc = no_gil([&] {
      return (store ? dllm_store_kvcache_fp8(ptr<dllm_bf16>(*k), k->stride(0), ptr<dllm_bf16>(*v), v->stride(0),
                                             ptr<uint8_t>(*kp), ptr<uint8_t>(*vp), std::min(kp->size(0), vp->size(0)),
                                             ptr<int32_t>(*slot), (int)k->size(0), (int)k->size(1), 128, st)
                    : dllm_load_kvcache_fp8(ptr<dllm_bf16>(*k), k->stride(0), ptr<dllm_bf16>(*v), v->stride(0),
                                            ptr<uint8_t>(*kp), ptr<uint8_t>(*vp), std::min(kp->size(0), vp->size(0)),
                                            ptr<int32_t>(*slot), (int)k->size(0), (int)k->size(1), 128, st));
    });
    if (rc != DLLM_OK) return refused(store ? "dllm_store_kvcache_fp8" : "dllm_load_kvcache_fp8", rc);
    Py_RETURN_TRUE;
  });
}

// chunk(q, k, v, k_cache, v_cache, plan: bytes, scale) -> output or None.
// `plan` is this description, n_groups launches and then the streams that are behind the
// tables' upload: on any other the Python form runs, which makes it wait.
struct ChunkTables {
  int64_t device, rows, n_groups, max_pages, max_page, mask_block, cu, lens, tables, seg_ids;
};
struct ChunkGroup {
  int64_t first, n_seg, max_q, max_cached, total_q, total_cached;
};
ChunkGroup chunk_group(PyObject* plan, int64_t i) {
  ChunkGroup g;
  std::memcpy(&g, PyBytes_AS_STRING(plan) + sizeof(ChunkTables) + i * sizeof(g), sizeof(g));
  return g;
}
bool behind_upload(PyObject* plan, int64_t n_groups, void* stream) {
  const char* at = PyBytes_AS_STRING(plan) + sizeof(ChunkTables) + n_groups * sizeof(ChunkGroup);
  const char* const end = PyBytes_AS_STRING(plan) + PyBytes_GET_SIZE(plan);
  for (int64_t s; at < end; at += sizeof(s)) {
    std::memcpy(&s, at, sizeof(s));
    if (s == (int64_t)reinterpret_cast<intptr_t>(stream)) return true;
  }
  return false;
}

PyObject* chunk(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 7 || !PyBytes_CheckExact(a[5]) || PyBytes_GET_SIZE(a[5]) < (Py_ssize_t)sizeof(ChunkTables) ||
      PyBytes_GET_SIZE(a[5]) % (Py_ssize_t)sizeof(int64_t) || !PyFloat_CheckExact(a[6]))
    Py_RETURN_NONE;
  return guarded([&]() -> PyObject* {
    ChunkTables p;
    std::memcpy(&p, PyBytes_AS_STRING(a[5]), sizeof(p));
    const at::Tensor* t[3];
    int64_t heads[3];
    for (int i = 0; i < 3; ++i) {
      t[i] = plain(a[i], at::kBFloat16);
      if (!t[i] || t[i]->get_device() != p.device || t[i]->dim() < 2 || t[i]->size(0) != p.rows) Py_RETURN_NONE;
      heads[i] = t[i]->dim() == 2 ? t[i]->size(1) / 128 : t[i]->size(1);
      if (heads[i] <= 0 || !token_rows(*t[i], heads[i], 128)) Py_RETURN_NONE;
    }
    const int64_t Hq = heads[0], Hkv = heads[1];
    if (heads[2] != Hkv || Hq % Hkv || p.rows == 0 || c10::hip::current_device() != p.device) Py_RETURN_NONE;
    void* const st = stream_of((int)p.device);
    const int64_t room = (PyBytes_GET_SIZE(a[5]) - (int64_t)sizeof(p)) / (int64_t)sizeof(ChunkGroup);
    if (p.n_groups < 0 || p.n_groups > room || !behind_upload(a[5], p.n_groups, st)) Py_RETURN_NONE;
    const at::Tensor *kc = pages_of(a[3], Hkv, (int)p.device), *vc = pages_of(a[4], Hkv, (int)p.device);
    const int kind = kc ? DLLM_CACHE_FP8 : DLLM_CACHE_BF16;
    if (!kc) {
      kc = plain(a[3], at::kBFloat16);
      vc = plain(a[4], at::kBFloat16);
      for (const at::Tensor* c : {kc, vc})
        if (!c || c->get_device() != p.device || c->dim() != 4 || c->size(1) != 256 || c->size(2) != Hkv ||
            c->size(3) != 128 || !c->is_contiguous())
          Py_RETURN_NONE;
    }
    if (!vc) Py_RETURN_NONE;
    const int64_t pages = std::min(kc->size(0), vc->size(0));
    if (p.max_page >= pages || pages > INT32_MAX) Py_RETURN_NONE;
    at::Tensor o = at::empty({p.rows, Hq * 128}, t[0]->options());
    size_t nb = 0;  // the launches follow one another, so they share it
    for (int64_t i = 0; i < p.n_groups; ++i) {
      const ChunkGroup g = chunk_group(a[5], i);
      nb = std::max(nb, dllm_attn_chunk_workspace_size((int)g.n_seg, (int)g.max_q, (int)g.max_cached, g.total_q,
                                                       g.total_cached, (int)Hq, (int)Hkv, 128));
    }
    at::Tensor ws;
    if (nb) ws = at::empty({(int64_t)nb}, t[0]->options().dtype(at::kByte));
    const float scale = (float)PyFloat_AS_DOUBLE(a[6]);
    auto dev_i32 = [](int64_t x) { return reinterpret_cast<const int32_t*>(x); };
    const int rc = no_gil([&] {
      int r = DLLM_OK;
      for (int64_t i = 0; i < p.n_groups && r == DLLM_OK; ++i) {
        const ChunkGroup g = chunk_group(a[5], i);
        r = dllm_attn_chunk_paged_fwd(
            ptr<dllm_bf16>(*t[0]), ptr<dllm_bf16>(*t[1]), ptr<dllm_bf16>(*t[2]), ptr<dllm_bf16>(o),
            dev_i32(p.cu) + (p.seg_ids ? 0 : g.first), p.seg_ids ? dev_i32(p.seg_ids) + g.first : nullptr, (int)g.n_seg,
            (int)g.max_q, (int)g.max_cached, g.total_q, g.total_cached, kc->data_ptr(), vc->data_ptr(), kind, (int)pages,
            dev_i32(p.tables) + g.first * p.max_pages, (int)p.max_pages, dev_i32(p.lens) + g.first, (int)p.mask_block,
            (int)Hq, (int)Hkv, 128, t[0]->stride(0), t[1]->stride(0), t[2]->stride(0), o.stride(0), scale,
            nb ? ws.data_ptr() : nullptr, nb, st);
      }
      return r;
    });
    if (rc != DLLM_OK) return refused("dllm_attn_chunk_paged_fwd", rc);
    return THPVariable_Wrap(std::move(o));
  });
}

// rope(positions, query, key, cos_sin_cache, head_size, inplace) -> (query, key) or None
PyObject* rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 6 || !PyLong_CheckExact(a[4]) || !PyBool_Check(a[5])) Py_RETURN_NONE;
  int overflow = 0;
  const int64_t D = PyLong_AsLongLongAndOverflow(a[4], &overflow);
  const bool inplace = a[5] == Py_True;
  return guarded([&]() -> PyObject* {
    const at::Tensor *pos = plain(a[0], at::kLong), *q = plain(a[1], at::kBFloat16), *k = plain(a[2], at::kBFloat16),
                     *cs = plain(a[3], at::kFloat);
    if (!pos || !q || !k || !cs || overflow || D <= 0 || D > 1024) Py_RETURN_NONE;
    const int dev = q->get_device();
    if (k->get_device() != dev || pos->get_device() != dev || cs->get_device() != dev || pos->dim() != 1 ||
        !pos->is_contiguous() || cs->dim() != 2 || cs->size(1) != D || !cs->is_contiguous())
      Py_RETURN_NONE;
    const int64_t rows = pos->size(0);
    int64_t heads[2];
    const at::Tensor* t[2] = {q, k};
    for (int i = 0; i < 2; ++i) {
      const int64_t width = t[i]->dim() == 2 ? t[i]->size(1) : t[i]->dim() == 3 ? t[i]->size(1) * D : 0;
      heads[i] = width / D;
      if (rows == 0 || width <= 0 || width % D || t[i]->size(0) != rows || !token_rows(*t[i], heads[i], D))
        Py_RETURN_NONE;
    }
    at::Tensor qo = *q, ko = *k;
    if (!inplace) {
      qo = at::empty(q->sizes(), q->options());
      ko = at::empty(k->sizes(), k->options());
    }
    void* st = stream_of(dev);
    const int rc = no_gil([&] {
      return dllm_rope_neox(ptr<dllm_bf16>(*q), q->stride(0), ptr<dllm_bf16>(qo), qo.stride(0), ptr<dllm_bf16>(*k),
                            k->stride(0), ptr<dllm_bf16>(ko), ko.stride(0), ptr<int64_t>(*pos), ptr<float>(*cs),
                            cs->size(0), (int)rows, (int)heads[0], (int)heads[1], (int)D, st);
    });
    if (rc != DLLM_OK) return refused("dllm_rope_neox", rc);
    PyObject* x = inplace ? Py_NewRef(a[1]) : THPVariable_Wrap(std::move(qo));
    PyObject* y = inplace ? Py_NewRef(a[2]) : THPVariable_Wrap(std::move(ko));
    PyObject* r = x && y ? PyTuple_Pack(2, x, y) : nullptr;
    Py_XDECREF(x);
    Py_XDECREF(y);
    return r;
  });
}

// softmax_max(logits) -> (x0, x0_p) or None
PyObject* softmax_max(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 1) Py_RETURN_NONE;
  return guarded([&]() -> PyObject* {
    const at::Tensor* l = plain(a[0], at::kBFloat16);
    if (!l || l->dim() != 2 || l->stride(1) != 1 || l->size(0) <= 0 || l->size(0) > INT32_MAX ||
        l->size(1) > INT32_MAX)
      Py_RETURN_NONE;
    const int M = (int)l->size(0), V = (int)l->size(1);
    at::Tensor x0 = at::empty({M}, l->options().dtype(at::kLong));
    at::Tensor xp = at::empty({M}, l->options());
    const size_t nb = dllm_softmax_max_split_workspace_size(M, V);
    at::Tensor ws;
    if (nb) ws = at::empty({(int64_t)nb}, l->options().dtype(at::kByte));
    void* st = stream_of(l->get_device());
    const int rc = no_gil([&] {
      return dllm_softmax_max(ptr<dllm_bf16>(*l), l->stride(0), M, V, ptr<int64_t>(x0), ptr<dllm_bf16>(xp),
                              nb ? ws.data_ptr() : nullptr, nb, st);
    });
    if (rc != DLLM_OK) return refused("dllm_softmax_max", rc);
    PyObject* x = THPVariable_Wrap(std::move(x0));
    PyObject* y = THPVariable_Wrap(std::move(xp));
    PyObject* r = x && y ? PyTuple_Pack(2, x, y) : nullptr;
    Py_XDECREF(x);
    Py_XDECREF(y);
    return r;
  });
}

// unmask(tokens, seq_params, max_win, x0, conf, mask_id) -> unmasked positions per sequence (int32) or None
PyObject* unmask(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 6 || !PyLong_CheckExact(a[2]) || !PyLong_CheckExact(a[5])) Py_RETURN_NONE;
  const long long win = PyLong_AsLongLong(a[2]), mask = PyLong_AsLongLong(a[5]);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
  return guarded([&]() -> PyObject* {
    const at::Tensor *tok = plain(a[0], at::kLong), *prm = plain(a[1], at::kInt), *x0 = plain(a[3], at::kLong),
                     *conf = plain(a[4], at::kBFloat16);
    if (!tok || !prm || !x0 || !conf || !tok->is_contiguous() || !prm->is_contiguous() || !x0->is_contiguous() ||
        !conf->is_contiguous() || prm->dim() != 2 || prm->size(1) != 5 || prm->size(0) == 0 || win < 0 ||
        win > INT32_MAX || prm->size(0) > INT32_MAX || conf->numel() < x0->numel())
      Py_RETURN_NONE;
    const int dev = tok->get_device();
    if (prm->get_device() != dev || x0->get_device() != dev || conf->get_device() != dev) Py_RETURN_NONE;
    const int n_seq = (int)prm->size(0);
    at::Tensor out = at::empty({n_seq}, prm->options());  // the kernel writes every entry
    void* st = stream_of(dev);
    const int rc = no_gil([&] {
      return dllm_lowconf_unmask(ptr<int64_t>(*tok), tok->numel(), ptr<int32_t>(*prm), n_seq, (int)win,
                                 ptr<int64_t>(*x0), ptr<dllm_bf16>(*conf), x0->numel(), mask, ptr<int32_t>(out), st);
    });
    if (rc != DLLM_OK) return refused("dllm_lowconf_unmask", rc);
    return THPVariable_Wrap(std::move(out));
  });
}

#define FN(name, doc) \
  { #name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, doc }
PyMethodDef methods[] = {
    FN(attn, "attn(q, k, v, k_cache, v_cache, plan, scale) -> output or None"),
    FN(quant_copy, "quant_copy(key, value, k_cache, v_cache, slot_mapping, store) -> True or None"),
    FN(chunk, "chunk(q, k, v, k_cache, v_cache, plan, scale) -> output or None"),
    FN(rope, "rope(positions, query, key, cos_sin_cache, head_size, inplace) -> (query, key) or None"),
    FN(softmax_max, "softmax_max(logits) -> (x0, x0_p) or None"),
    FN(unmask, "unmask(tokens, seq_params, max_win, x0, conf, mask_id) -> counts or None"),
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_native", "Host fast paths over the C ABI", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__native(void) { return PyModule_Create(&module); }
