// front.cpp -- call path of the position and paged-cache operators for torch tensors (ops.py).
//
// These run once or twice per layer and token, and at decode sizes the checks of a dozen tensors from
// Python and ctypes' conversion of some thirty arguments (17-21 us a call) exceed the kernels' time.
// Each function here checks its operands, makes the outputs and calls the C entry point, whose address
// bind() was given.  It returns the result, or the entry's status where that is not zero, or None
// for operands that it does not take: ops.py then goes through its own checks, which name the
// reason.  No device code and no link to libbeacon_cuda.so.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/beacon_cuda.h"

namespace {

decltype(&beacon_qk_norm_rope_fwd) g_fwd = nullptr;
decltype(&beacon_qk_norm_rope_bwd) g_bwd = nullptr;
decltype(&beacon_qk_norm_rope_append) g_append = nullptr;
decltype(&beacon_paged_attention_fwd) g_attn = nullptr;
decltype(&beacon_qk_norm_rope_bwd_workspace_size) g_bwd_ws = nullptr;
decltype(&beacon_paged_attention_workspace_size) g_attn_ws = nullptr;

using at::Tensor;

// A tensor argument; `none`: None may stand for it (null).
bool arg(PyObject* o, const Tensor** t, bool none = false) {
  if (o == Py_None) {
    *t = nullptr;
    return none;
  }
  if (!THPVariable_Check(o)) return false;
  *t = &THPVariable_Unpack(o);
  return true;
}
bool integer(PyObject* o, int64_t* v) {
  if (!PyLong_Check(o)) return false;
  *v = PyLong_AsLongLong(o);
  if (*v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return true;
}
bool real(PyObject* o, float* v) {
  if (!PyFloat_Check(o)) return false;
  *v = (float)PyFloat_AS_DOUBLE(o);
  return true;
}
void* ptr(const Tensor* t) { return t == nullptr ? nullptr : t->data_ptr(); }

int dtype_code(at::ScalarType t) {
  return t == at::kFloat ? BEACON_F32 : t == at::kBFloat16 ? BEACON_BF16 : -1;
}
bool is(const Tensor& t, at::ScalarType dt) { return t.is_cuda() && t.scalar_type() == dt; }
bool dense(const Tensor& t, at::ScalarType dt) { return is(t, dt) && t.is_contiguous(); }
bool ints(const Tensor* t, int64_t n) { return t == nullptr || (dense(*t, at::kInt) && t->numel() == n); }
bool gain(const Tensor* t, at::ScalarType dt, int64_t dim) { return t == nullptr || (dense(*t, dt) && t->numel() == dim); }

struct Rope {
  const Tensor *qkv, *q_gain, *k_gain, *table, *positions;
  int64_t ld, rot, rows;
  int interleaved;
  float eps;
};
// The operands that the three rotation entries share; width: heads' elements of a token row.
bool rope(Rope& r, int64_t width, int64_t dim) {
  const Tensor& x = *r.qkv;
  const at::ScalarType dt = x.scalar_type();
  if (dtype_code(dt) < 0 || !x.is_cuda() || x.dim() != 2 || x.size(1) != width || x.stride(1) != 1) return false;
  if (!gain(r.q_gain, dt, dim) || !gain(r.k_gain, dt, dim) || !ints(r.positions, x.size(0))) return false;
  if (r.table != nullptr && (!dense(*r.table, at::kFloat) || r.table->dim() != 2)) return false;
  r.ld = x.size(0) > 1 ? x.stride(0) : std::max(x.stride(0), width);
  r.rot = r.table == nullptr ? 0 : r.table->size(1);
  r.rows = r.table == nullptr ? 0 : r.table->size(0);
  return true;
}

struct Paging {
  const Tensor *k, *v, *table, *cu_q, *kv_lens;
  int64_t seqs, width, stride, pages, page, heads, dim;
};
bool paging(Paging& g) {
  const Tensor &k = *g.k, &v = *g.v, &t = *g.table;
  const at::ScalarType dt = k.scalar_type();
  if (k.dim() != 4 || k.sizes() != v.sizes() || k.strides() != v.strides() || dtype_code(dt) < 0 || !k.is_cuda() ||
      !is(v, dt) || k.stride(3) != 1)
    return false;
  g.seqs = g.kv_lens->numel();
  if (!ints(g.kv_lens, g.seqs) || !ints(g.cu_q, g.seqs + 1) || !is(t, at::kInt) || t.dim() != 2 ||
      t.size(0) != g.seqs || (t.stride(1) != 1 && t.size(1) > 1))
    return false;
  g.width = t.size(1);
  g.stride = g.seqs > 1 ? t.stride(0) : std::max(t.stride(0), g.width);
  g.pages = k.size(0);
  g.heads = k.size(1);
  g.page = k.size(2);
  g.dim = k.size(3);
  return true;
}
int64_t token_stride(const Paging& g) { return g.page > 1 ? g.k->stride(2) : std::max(g.k->stride(2), g.dim); }

void* stream() { return c10::cuda::getCurrentCUDAStream().stream(); }

Tensor make(at::IntArrayRef sizes, const Tensor& like) { return at::empty(sizes, like.options()); }

// A call's scratch from the caching allocator: ordered on the call's stream, and kept by a graph that captures it.
Tensor scratch(size_t bytes, const Tensor& like) {
  return at::empty({(int64_t)bytes}, like.options().dtype(at::kByte));
}

PyObject* status(int rc) { return PyLong_FromLong(rc); }

// A call's body: C++ exceptions (an allocation that fails) become Python ones.
template <typename F>
PyObject* guarded(F&& f) {
  try {
    at::AutoDispatchBelowADInplaceOrView below;  // outputs carry no autograd state
    return f();
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

PyObject* pack3(const Tensor& a, const Tensor& b, const Tensor& c) {
  return Py_BuildValue("(NNN)", THPVariable_Wrap(a), THPVariable_Wrap(b), THPVariable_Wrap(c));
}

// (qkv, q_gain, k_gain, table, batch, seq, heads, kv_heads, positions, interleaved, eps)
PyObject* front_fwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Rope r;
    int64_t B, S, H, K;
    if (n != 11 || !g_fwd || !arg(a[0], &r.qkv) || !arg(a[1], &r.q_gain, true) || !arg(a[2], &r.k_gain, true) ||
        !arg(a[3], &r.table, true) || !integer(a[4], &B) || !integer(a[5], &S) || !integer(a[6], &H) ||
        !integer(a[7], &K) || !arg(a[8], &r.positions, true) || !real(a[10], &r.eps))
      Py_RETURN_NONE;
    r.interleaved = PyObject_IsTrue(a[9]);
    const int64_t heads = H + 2 * K;
    if (H <= 0 || K <= 0 || H > 65536 || K > 65536 || B < 0 || S < 0 || r.qkv->dim() != 2 ||
        r.qkv->size(1) % heads != 0 || (S > 0 && B > INT32_MAX / S) || r.qkv->size(0) != B * S)
      Py_RETURN_NONE;
    const int64_t D = r.qkv->size(1) / heads;
    if (!rope(r, heads * D, D)) Py_RETURN_NONE;
    Tensor q = make({B, H, S, D}, *r.qkv), k = make({B, K, S, D}, *r.qkv), v = make({B, K, S, D}, *r.qkv);
    const int rc = g_fwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), r.qkv->data_ptr(), r.ld, ptr(r.q_gain), ptr(r.k_gain),
                         (const float*)ptr(r.table), r.rows, (const int32_t*)ptr(r.positions), B, S, H, K, D, r.rot,
                         r.interleaved, r.eps, dtype_code(r.qkv->scalar_type()), stream());
    return rc != BEACON_OK ? status(rc) : pack3(q, k, v);
  });
}

// (dq, dk, dv, qkv, q_gain, k_gain, table, positions, interleaved, eps)
PyObject* front_bwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Rope r;
    const Tensor *dq, *dk, *dv;
    if (n != 10 || !g_bwd || !arg(a[0], &dq) || !arg(a[1], &dk) || !arg(a[2], &dv) || !arg(a[3], &r.qkv) ||
        !arg(a[4], &r.q_gain) || !arg(a[5], &r.k_gain) || !arg(a[6], &r.table, true) ||
        !arg(a[7], &r.positions, true) || !real(a[9], &r.eps))
      Py_RETURN_NONE;
    r.interleaved = PyObject_IsTrue(a[8]);
    const at::ScalarType dt = r.qkv->scalar_type();
    if (dq->dim() != 4 || dk->dim() != 4 || dk->sizes() != dv->sizes() || !dense(*dq, dt) || !dense(*dk, dt) ||
        !dense(*dv, dt))
      Py_RETURN_NONE;
    const int64_t B = dq->size(0), H = dq->size(1), S = dq->size(2), D = dq->size(3), K = dk->size(1);
    const int64_t width = (H + 2 * K) * D;
    if (dk->size(0) != B || dk->size(2) != S || dk->size(3) != D || r.qkv->dim() != 2 || r.qkv->size(0) != B * S ||
        !rope(r, width, D))
      Py_RETURN_NONE;
    Tensor dx = make({B * S, width}, *dq), dqg = make({D}, *dq), dkg = make({D}, *dq);
    const size_t need = g_bwd_ws(D);
    Tensor ws = scratch(need, *dq);
    const int rc = g_bwd(dx.data_ptr(), width, dqg.data_ptr(), dkg.data_ptr(), dq->data_ptr(), dk->data_ptr(),
                         dv->data_ptr(), r.qkv->data_ptr(), r.ld, ptr(r.q_gain), ptr(r.k_gain),
                         (const float*)ptr(r.table), r.rows, (const int32_t*)ptr(r.positions), B, S, H, K, D, r.rot,
                         r.interleaved, r.eps, dtype_code(dt), ws.data_ptr(), need, stream());
    return rc != BEACON_OK ? status(rc) : pack3(dx, dqg, dkg);
  });
}

// (qkv, q_gain, k_gain, table, k_cache, v_cache, page_table, cu_q, kv_lens, heads, positions, interleaved, eps)
PyObject* front_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Rope r;
    Paging g;
    int64_t H;
    if (n != 13 || !g_append || !arg(a[0], &r.qkv) || !arg(a[1], &r.q_gain, true) || !arg(a[2], &r.k_gain, true) ||
        !arg(a[3], &r.table, true) || !arg(a[4], &g.k) || !arg(a[5], &g.v) || !arg(a[6], &g.table) ||
        !arg(a[7], &g.cu_q) || !arg(a[8], &g.kv_lens) || !integer(a[9], &H) || !arg(a[10], &r.positions, true) ||
        !real(a[12], &r.eps))
      Py_RETURN_NONE;
    r.interleaved = PyObject_IsTrue(a[11]);
    if (!paging(g) || H <= 0 || H > 65536 || r.qkv->scalar_type() != g.k->scalar_type() ||
        !rope(r, (H + 2 * g.heads) * g.dim, g.dim))
      Py_RETURN_NONE;
    const int64_t T = r.qkv->size(0);
    Tensor q = make({T, H, g.dim}, *r.qkv);
    const int rc =
        g_append(q.data_ptr(), g.k->data_ptr(), g.v->data_ptr(), r.qkv->data_ptr(), r.ld, ptr(r.q_gain), ptr(r.k_gain),
                 (const float*)ptr(r.table), r.rows, (const int32_t*)ptr(r.positions), (const int32_t*)ptr(g.cu_q),
                 (const int32_t*)ptr(g.kv_lens), (const int32_t*)ptr(g.table), T, g.seqs, g.width, g.stride, g.pages,
                 g.page, g.k->stride(0), g.k->stride(1), token_stride(g), H, g.heads, g.dim, r.rot, r.interleaved, r.eps,
                 dtype_code(r.qkv->scalar_type()), stream());
    return rc != BEACON_OK ? status(rc) : THPVariable_Wrap(q);
  });
}

// (q, k_cache, v_cache, page_table, cu_q, kv_lens, max_q, causal)
PyObject* front_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Paging g;
    const Tensor* q;
    int64_t max_q;
    if (n != 8 || !g_attn || !arg(a[0], &q) || !arg(a[1], &g.k) || !arg(a[2], &g.v) || !arg(a[3], &g.table) ||
        !arg(a[4], &g.cu_q) || !arg(a[5], &g.kv_lens) || !integer(a[6], &max_q))
      Py_RETURN_NONE;
    if (!paging(g) || q->dim() != 3 || q->size(2) != g.dim || !is(*q, g.k->scalar_type()) || q->stride(2) != 1 ||
        (q->stride(1) != g.dim && q->size(1) > 1))
      Py_RETURN_NONE;
    const int64_t T = q->size(0), H = q->size(1);
    Tensor out = make({T, H, g.dim}, *q), lse = at::empty({T, H}, q->options().dtype(at::kFloat));
    const size_t need = g_attn_ws(g.dim, dtype_code(q->scalar_type()));
    Tensor ws = scratch(need, *q);
    const int rc = g_attn(out.data_ptr(), (float*)lse.data_ptr(), q->data_ptr(),
                          T > 1 ? q->stride(0) : std::max(q->stride(0), H * g.dim), g.k->data_ptr(), g.v->data_ptr(),
                          (const int32_t*)ptr(g.cu_q), (const int32_t*)ptr(g.kv_lens), (const int32_t*)ptr(g.table), T,
                          g.seqs, max_q, g.width, g.stride, g.pages, g.page, g.k->stride(0), g.k->stride(1),
                          token_stride(g), H, g.heads, g.dim, PyObject_IsTrue(a[7]), dtype_code(q->scalar_type()),
                          ws.data_ptr(), need, stream());
    return rc != BEACON_OK ? status(rc) : Py_BuildValue("(NN)", THPVariable_Wrap(out), THPVariable_Wrap(lse));
  });
}

// bind(fwd, bwd, append, attention, bwd_workspace_size, attention_workspace_size): addresses of the C entry points
PyObject* front_bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  void* p[6];
  for (int i = 0; i < 6; ++i) {
    p[i] = n == 6 ? PyLong_AsVoidPtr(a[i]) : nullptr;
    if (p[i] == nullptr) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "bind: six addresses");
      return nullptr;
    }
  }
  g_fwd = reinterpret_cast<decltype(g_fwd)>(p[0]);
  g_bwd = reinterpret_cast<decltype(g_bwd)>(p[1]);
  g_append = reinterpret_cast<decltype(g_append)>(p[2]);
  g_attn = reinterpret_cast<decltype(g_attn)>(p[3]);
  g_bwd_ws = reinterpret_cast<decltype(g_bwd_ws)>(p[4]);
  g_attn_ws = reinterpret_cast<decltype(g_attn_ws)>(p[5]);
  Py_RETURN_NONE;
}

#define FRONT(name, fn) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(fn)), METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {FRONT("bind", front_bind),
                           FRONT("qk_norm_rope_fwd", front_fwd),
                           FRONT("qk_norm_rope_bwd", front_bwd),
                           FRONT("qk_norm_rope_append", front_append),
                           FRONT("paged_attention", front_attention),
                           {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "beacon_front", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_beacon_front(void) { return PyModule_Create(&g_module); }
