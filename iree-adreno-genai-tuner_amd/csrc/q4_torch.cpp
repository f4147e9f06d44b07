// CPython module _q4torch: the ordinary calls of the tensor-level wrappers (q4llm/ops.py, QLinear.forward)
// in native code.
//
// A decode projection or a decode attention call takes 4 to 8 us on the GPU, and the Python wrapper took 11
// to 17 us of host time: checks, attribute reads, torch.empty, the current stream and the ctypes
// conversions. Each function here does the same for the usual operands (plain contiguous device tensors of
// the documented types and shapes) in one step and returns the result. For anything else, and whenever
// the library returns a status other than Q4_OK, it returns None without having launched anything, and
// the Python wrapper runs its own checks and raises its own error. Nothing is kept between calls.
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/TensorSubclassLikeUtils.h>
#include <ATen/ops/empty.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <algorithm>

#include "q4llm.h"

namespace {

using at::Tensor;

// A plain strided device tensor that the library may read through its address.
bool plain(const Tensor& t) {
  return t.defined() && t.is_cuda() && t.layout() == at::kStrided && !t.is_neg() && !t.is_conj() &&
         !at::isTensorSubclassLike(t);
}
bool plain_as(const Tensor& t, at::ScalarType dt) { return plain(t) && t.scalar_type() == dt && t.is_contiguous(); }
bool same_device(const Tensor& a, const Tensor& b) { return a.get_device() == b.get_device(); }

// A tensor argument: false when it is neither a tensor nor (if `optional`) None.
bool arg(PyObject* o, Tensor* t, bool optional = false) {
  if (optional && o == Py_None) return true;
  if (!THPVariable_Check(o)) return false;
  *t = THPVariable_Unpack(o);
  return t->defined();
}

bool arg(PyObject* o, int64_t* v) {
  if (!PyLong_Check(o)) return false;
  *v = PyLong_AsLongLong(o);
  if (*v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return true;
}

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

// An int4 weight pair [N, K/8] int32, [N, K/group] fp16 on one device.
bool weights(const Tensor& qw, const Tensor& sc, int64_t group, int64_t* n, int64_t* k) {
  if (group <= 0 || group > INT32_MAX || !plain_as(qw, at::kInt) || !plain_as(sc, at::kHalf) || qw.dim() != 2 ||
      sc.dim() != 2 || !same_device(qw, sc))
    return false;
  *n = qw.size(0);
  *k = qw.size(1) * 8;
  return *n > 0 && *k > 0 && *k % group == 0 && sc.size(0) == *n && sc.size(1) == *k / group;
}

template <typename T>
T* data(const Tensor& t) {
  return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr;
}

// Runs `f` without the interpreter lock, as ctypes does.
template <typename F>
int unlocked(F f) {
  PyThreadState* s = PyEval_SaveThread();
  const int st = f();
  PyEval_RestoreThread(s);
  return st;
}

// Every entry: a C++ exception (an allocation that fails, say) means "not here".
template <typename F>
PyObject* guarded(F f) {
  try {
    return f();
  } catch (...) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
}

// gemv(qweight, scales, x, group, out dtype code or -1, residual, out): y [N]
PyObject* gemv(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  return guarded([&]() -> PyObject* {
    Tensor qw, sc, x, res, out;
    int64_t group, code, n, k;
    if (nargs != 7 || !arg(a[0], &qw) || !arg(a[1], &sc) || !arg(a[2], &x) || !arg(a[3], &group) || !arg(a[4], &code) ||
        !arg(a[5], &res, true) || !arg(a[6], &out, true) || !weights(qw, sc, group, &n, &k))
      Py_RETURN_NONE;
    const bool f16x = x.scalar_type() == at::kHalf;
    if (!plain_as(x, f16x ? at::kHalf : at::kFloat) || x.numel() != k || !same_device(x, qw)) Py_RETURN_NONE;
    if (res.defined() && (!plain_as(res, at::kFloat) || res.dim() != 1 || res.size(0) != n || !same_device(res, qw)))
      Py_RETURN_NONE;
    if (out.defined()) {
      const bool f16 = out.scalar_type() == at::kHalf;
      if (!plain_as(out, f16 ? at::kHalf : at::kFloat) || out.dim() != 1 || out.size(0) != n || !same_device(out, qw) ||
          (f16 && res.defined()))
        Py_RETURN_NONE;
      code = f16 ? Q4_F16 : Q4_F32;
    } else {
      if ((code != Q4_F16 && code != Q4_F32) || (code == Q4_F16 && res.defined())) Py_RETURN_NONE;
      out = at::empty({n}, x.options().dtype(code == Q4_F16 ? at::kHalf : at::kFloat));
    }
    void* st = stream_of(x);
    const int rc = unlocked([&] {
      return q4_gemv(data<int32_t>(qw), data<uint16_t>(sc), x.data_ptr(), f16x ? Q4_F16 : Q4_F32, out.data_ptr(),
                     static_cast<int>(code), data<float>(res), n, k, static_cast<int>(group), st);
    });
    if (rc != Q4_OK) Py_RETURN_NONE;
    return a[6] != Py_None ? (Py_INCREF(a[6]), a[6]) : THPVariable_Wrap(out);
  });
}

// y [M, N] = residual + x [M, K] W^T; M == 1 with `gemv_row` set: the decode GEMV
PyObject* linear_impl(const Tensor& qw, const Tensor& sc, const Tensor& x, int64_t group, const Tensor& res,
                      bool gemv_row) {
  int64_t n, k;
  if (!weights(qw, sc, group, &n, &k) || !plain_as(x, at::kFloat) || x.dim() != 2 || x.size(1) != k || x.size(0) < 1 ||
      !same_device(x, qw))
    Py_RETURN_NONE;
  const int64_t m = x.size(0);
  if (res.defined() && (!plain_as(res, at::kFloat) || !same_device(res, qw) || res.dim() != 2 || res.size(0) != m ||
                        res.size(1) != n))
    Py_RETURN_NONE;
  const bool one = m == 1 && gemv_row;
  // the sizes q4_linear's tiled path takes through a workspace (ops._linear_workspace)
  const bool ws_path = !one && m > 16 && k % 64 == 0 && group % 32 == 0 && (group & (group - 1)) == 0 &&
                       m * k < (int64_t{1} << 29);
  Tensor out = at::empty({m, n}, x.options()), ws;
  size_t ws_bytes = 0;
  if (ws_path) {
    if (q4_linear_ws_split_bytes(m, n, k, static_cast<int>(group), &ws_bytes) != Q4_OK) Py_RETURN_NONE;
    ws = at::empty({static_cast<int64_t>(ws_bytes)}, x.options().dtype(at::kByte));
  }
  void* st = stream_of(x);
  const int rc = unlocked([&] {
    const int g = static_cast<int>(group);
    if (one)
      return q4_gemv(data<int32_t>(qw), data<uint16_t>(sc), x.data_ptr(), Q4_F32, out.data_ptr(), Q4_F32,
                     data<float>(res), n, k, g, st);
    if (ws_path)
      return q4_linear_ws(data<float>(x), m, data<int32_t>(qw), data<uint16_t>(sc), data<float>(out), data<float>(res),
                          n, k, g, ws.data_ptr(), ws_bytes, st);
    return q4_linear(data<float>(x), m, data<int32_t>(qw), data<uint16_t>(sc), data<float>(out), data<float>(res), n, k,
                     g, st);
  });
  if (rc != Q4_OK) Py_RETURN_NONE;
  return THPVariable_Wrap(out);
}

// linear(qweight, scales, x, group, residual, decode row as GEMV: bool)
PyObject* linear(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  return guarded([&]() -> PyObject* {
    Tensor qw, sc, x, res;
    int64_t group;
    if (nargs != 6 || !arg(a[0], &qw) || !arg(a[1], &sc) || !arg(a[2], &x) || !arg(a[3], &group) ||
        !arg(a[4], &res, true))
      Py_RETURN_NONE;
    return linear_impl(qw, sc, x, group, res, a[5] == Py_True);
  });
}

// attn_bucket(q, k_cache, v_cache, L, start, scale, workspace): out [C, n_q * hd]
PyObject* attn(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  return guarded([&]() -> PyObject* {
    Tensor q, kc, vc, start, ws;
    int64_t L;
    if (nargs != 7 || !arg(a[0], &q) || !arg(a[1], &kc) || !arg(a[2], &vc) || !arg(a[3], &L) || !arg(a[4], &start) ||
        !PyFloat_Check(a[5]) || !arg(a[6], &ws, true))
      Py_RETURN_NONE;
    if (!plain(q) || q.scalar_type() != at::kFloat || q.dim() != 3 || q.stride(2) != 1 || q.stride(1) != q.size(2) ||
        !plain_as(kc, at::kHalf) || !plain_as(vc, at::kHalf) || kc.dim() != 3 || !plain_as(start, at::kInt) ||
        start.numel() < 1 || !same_device(kc, q) || !same_device(vc, q) || !same_device(start, q))
      Py_RETURN_NONE;
    const int64_t c = q.size(0), nq = q.size(1), hd = q.size(2), nkv = kc.size(1);
    if (c > INT32_MAX || nq > INT32_MAX || L > INT32_MAX || L < INT32_MIN || q.stride(0) > INT32_MAX || c < 1)
      Py_RETURN_NONE;
    if (ws.defined()) {
      if (!plain_as(ws, at::kByte) || !same_device(ws, q)) Py_RETURN_NONE;
    } else {
      size_t b = 0;
      if (attn_workspace_bytes(c, nq, nkv, hd, L, &b) != Q4_OK) Py_RETURN_NONE;
      ws = at::empty({static_cast<int64_t>(b > 0 ? b : 1)}, q.options().dtype(at::kByte));
    }
    Tensor out = at::empty({c, nq * hd}, q.options());
    void* st = stream_of(q);
    const float scale = static_cast<float>(PyFloat_AS_DOUBLE(a[5]));
    const int rc = unlocked([&] {
      return attn_bucket(data<float>(q), static_cast<int>(q.stride(0)), data<uint16_t>(kc), data<uint16_t>(vc),
                         data<float>(out), c, nq, nkv, hd, L, data<int32_t>(start), scale, ws.data_ptr(), ws.numel(), st);
    });
    if (rc != Q4_OK) Py_RETURN_NONE;
    return THPVariable_Wrap(out);
  });
}

// gemm(a, b, workspace): C [M, N] fp16 (gemm_f16_nt_ws with a workspace, gemm_f16_nt with None)
PyObject* gemm(PyObject*, PyObject* const* o, Py_ssize_t nargs) {
  return guarded([&]() -> PyObject* {
    Tensor a, b, ws;
    if (nargs != 3 || !arg(o[0], &a) || !arg(o[1], &b) || !arg(o[2], &ws, true) || !plain(a) || !plain(b) ||
        a.scalar_type() != at::kHalf || b.scalar_type() != at::kHalf || a.dim() != 2 || b.dim() != 2 ||
        a.stride(1) != 1 || b.stride(1) != 1 || a.size(1) != b.size(1) || !same_device(a, b))
      Py_RETURN_NONE;
    if (ws.defined() && (!plain_as(ws, at::kByte) || !same_device(ws, a))) Py_RETURN_NONE;
    const int64_t m = a.size(0), n = b.size(0), k = a.size(1);
    if (m < 1 || n < 1 || k < 1) Py_RETURN_NONE;
    Tensor c = at::empty({m, n}, a.options());
    void* st = stream_of(a);
    const int rc = unlocked([&] {
      if (ws.defined())
        return gemm_f16_nt_ws(data<uint16_t>(a), data<uint16_t>(b), data<uint16_t>(c), m, n, k, a.stride(0), b.stride(0),
                              n, ws.data_ptr(), ws.numel(), st);
      return gemm_f16_nt(data<uint16_t>(a), data<uint16_t>(b), data<uint16_t>(c), m, n, k, a.stride(0), b.stride(0), n,
                         st);
    });
    if (rc != Q4_OK) Py_RETURN_NONE;
    return THPVariable_Wrap(c);
  });
}

// ---- batched serving over a paged cache ----

bool code_of(at::ScalarType s, int* code) {
  *code = s == at::kFloat ? Q4_F32 : s == at::kHalf ? Q4_F16 : s == at::kBFloat16 ? Q4_BF16 : -1;
  return *code >= 0;
}
bool arg(PyObject* o, float* v) {
  if (!PyFloat_Check(o)) return false;
  *v = static_cast<float>(PyFloat_AS_DOUBLE(o));
  return true;
}

// A [tokens, heads, head_dim] operand whose dims of a head lie next to each other, on the device of `on`.
bool heads(const Tensor& t, at::ScalarType dt, int64_t tokens, int64_t n, int64_t hd, const Tensor& on) {
  return plain(t) && t.scalar_type() == dt && t.dim() == 3 && t.size(0) == tokens && t.size(1) == n && t.size(2) == hd &&
         (hd == 1 || t.stride(2) == 1) && same_device(t, on);
}
bool indices(const Tensor& t, int64_t n, const Tensor& on) {
  return plain_as(t, at::kInt) && t.dim() == 1 && t.size(0) == n && same_device(t, on);
}

// inv_freq, interleaved and mscale of a Rope for heads of hd dims.
bool rope_arg(PyObject* const* a, int64_t hd, const Tensor& on, Tensor* inv_freq, q4_rope* r) {
  if (!arg(a[0], inv_freq) || !PyBool_Check(a[1]) || !arg(a[2], &r->mscale) || !plain_as(*inv_freq, at::kFloat) ||
      inv_freq->dim() != 1 || 2 * inv_freq->size(0) > hd || !same_device(*inv_freq, on))
    return false;
  r->inv_freq = data<float>(*inv_freq);
  r->rot_dim = static_cast<int>(2 * inv_freq->size(0));
  r->layout = a[1] == Py_True ? Q4_ROPE_INTERLEAVED : Q4_ROPE_HALF;
  return true;
}

// Cache, page table, lengths and cu_q (None) of a paged call of `tokens` tokens of type dt.
struct Paged {
  Tensor kc, vc, table, lens, cu;
  q4_paged_kv kv;
};
bool paged_arg(PyObject* const* a, PyObject* cu, at::ScalarType dt, int64_t tokens, const Tensor& on, Paged* p) {
  if (!arg(a[0], &p->kc) || !arg(a[1], &p->vc) || !arg(a[2], &p->table) || !arg(a[3], &p->lens) || !arg(cu, &p->cu, true))
    return false;
  const at::ScalarType ct = dt == at::kFloat ? at::kHalf : dt;
  if (!plain_as(p->kc, ct) || !plain_as(p->vc, ct) || p->kc.dim() != 4 || p->vc.sizes() != p->kc.sizes() ||
      !same_device(p->kc, on) || !same_device(p->vc, on))
    return false;
  if (!plain(p->table) || p->table.scalar_type() != at::kInt || p->table.dim() != 2 || p->table.size(0) < 1 ||
      p->table.size(1) < 1 || (p->table.size(1) > 1 && p->table.stride(1) != 1) || !same_device(p->table, on))
    return false;
  const int64_t batch = p->table.size(0), most = p->table.size(1);
  if (batch > INT32_MAX || most > INT32_MAX || !indices(p->lens, batch, on) ||
      (p->cu.defined() && !indices(p->cu, batch + 1, on)) || (!p->cu.defined() && tokens % batch))
    return false;
  for (int i = 1; i < 4; ++i)
    if (p->kc.size(i) > INT32_MAX) return false;
  int code = 0;
  code_of(ct, &code);
  p->kv = q4_paged_kv{p->kc.data_ptr(), p->vc.data_ptr(), data<int32_t>(p->table), data<int32_t>(p->lens),
                      data<int32_t>(p->cu), p->kc.size(0), batch > 1 ? p->table.stride(0) : most, code,
                      static_cast<int>(p->kc.size(1)), static_cast<int>(p->kc.size(2)), static_cast<int>(p->kc.size(3)),
                      static_cast<int>(batch), static_cast<int>(most)};
  return true;
}

// rope(x, positions, inv_freq, interleaved, mscale, inverse, out)
PyObject* rope(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  return guarded([&]() -> PyObject* {
    Tensor x, pos, freq, out;
    q4_rope r{};
    int code;
    if (nargs != 7 || !arg(a[0], &x) || !arg(a[1], &pos) || !arg(a[6], &out, true) || !PyBool_Check(a[5]) || !plain(x) ||
        x.dim() != 3 || !code_of(x.scalar_type(), &code))
      Py_RETURN_NONE;
    const int64_t t = x.size(0), h = x.size(1), hd = x.size(2);
    if (t < 1 || h > INT32_MAX || hd > INT32_MAX || !heads(x, x.scalar_type(), t, h, hd, x) || !indices(pos, t, x) ||
        !rope_arg(a + 2, hd, x, &freq, &r) || (out.defined() && !heads(out, x.scalar_type(), t, h, hd, x)))
      Py_RETURN_NONE;
    const c10::DeviceGuard on(x.device());
    if (!out.defined()) out = at::empty({t, h, hd}, x.options());
    void* st = stream_of(x);
    const int rc = unlocked([&] {
      return rope_rotate(x.data_ptr(), x.stride(0), x.stride(1), out.data_ptr(), out.stride(0), out.stride(1), code, t,
                         static_cast<int>(h), static_cast<int>(hd), data<int32_t>(pos), &r, a[5] == Py_True, st);
    });
    if (rc != Q4_OK) Py_RETURN_NONE;
    return a[6] != Py_None ? (Py_INCREF(a[6]), a[6]) : THPVariable_Wrap(out);
  });
}

// append(k, v, k_cache, v_cache, page_table, seq_lens, cu_q, inv_freq or None, interleaved, mscale, q, q_out): q_out, or
// True without q
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  return guarded([&]() -> PyObject* {
    Tensor k, v, q, qo, freq;
    Paged p;
    q4_rope r{};
    int code;
    if (nargs != 12 || !arg(a[0], &k) || !arg(a[1], &v) || !arg(a[10], &q, true) || !arg(a[11], &qo, true) || !plain(k) ||
        k.dim() != 3 || k.size(0) < 1 || !code_of(k.scalar_type(), &code) || (qo.defined() && !q.defined()))
      Py_RETURN_NONE;
    const at::ScalarType dt = k.scalar_type();
    const int64_t t = k.size(0), n_kv = k.size(1), hd = k.size(2);
    if (!paged_arg(a + 2, a[6], dt, t, k, &p) || p.kc.size(2) != n_kv || p.kc.size(3) != hd || !heads(k, dt, t, n_kv, hd, k) ||
        !heads(v, dt, t, n_kv, hd, k) || (a[7] != Py_None && !rope_arg(a + 7, hd, k, &freq, &r)))
      Py_RETURN_NONE;
    int64_t n_q = 0;
    if (q.defined()) {
      if (q.dim() != 3) Py_RETURN_NONE;
      n_q = q.size(1);
      if (n_q < 1 || n_q > INT32_MAX || !heads(q, dt, t, n_q, hd, k) || (qo.defined() && !heads(qo, dt, t, n_q, hd, k)))
        Py_RETURN_NONE;
    }
    const c10::DeviceGuard on(k.device());
    if (q.defined() && !qo.defined()) qo = at::empty({t, n_q, hd}, q.options());
    void* st = stream_of(k);
    const int rc = unlocked([&] {
      const bool w = q.defined();
      return paged_kv_append(&p.kv, k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), code, t,
                             a[7] == Py_None ? nullptr : &r, w ? q.data_ptr() : nullptr, w ? q.stride(0) : 0,
                             w ? q.stride(1) : 0, w ? qo.data_ptr() : nullptr, w ? qo.stride(0) : 0, w ? qo.stride(1) : 0,
                             static_cast<int>(n_q), st);
    });
    if (rc != Q4_OK) Py_RETURN_NONE;
    if (!q.defined()) Py_RETURN_TRUE;
    return a[11] != Py_None ? (Py_INCREF(a[11]), a[11]) : THPVariable_Wrap(qo);
  });
}

// paged(q, k_cache, v_cache, page_table, seq_lens, scale, cu_q, shared_pages, shared_len, L or None, workspace, out)
PyObject* paged(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  return guarded([&]() -> PyObject* {
    Tensor q, sp, ws, out;
    Paged p;
    int64_t shared, L;
    float scale;
    int code;
    if (nargs != 12 || !arg(a[0], &q) || !arg(a[5], &scale) || !arg(a[7], &sp, true) || !arg(a[8], &shared) ||
        !arg(a[10], &ws, true) || !arg(a[11], &out, true) || !plain(q) || q.dim() != 3 || q.size(0) < 1 ||
        !code_of(q.scalar_type(), &code))
      Py_RETURN_NONE;
    const at::ScalarType dt = q.scalar_type();
    const int64_t t = q.size(0), n_q = q.size(1), hd = q.size(2), align = 16 / q.element_size();
    if (t > INT32_MAX || n_q > INT32_MAX || !paged_arg(a + 1, a[6], dt, t, q, &p) || p.kc.size(3) != hd ||
        !heads(q, dt, t, n_q, hd, q) || q.stride(0) % align || q.stride(1) % align ||
        reinterpret_cast<uintptr_t>(q.data_ptr()) % 16)
      Py_RETURN_NONE;
    if (shared < 0 || shared > INT32_MAX || (shared > 0 && (!sp.defined() || sp.dim() != 1 || !indices(sp, sp.size(0), q) ||
                                                            sp.size(0) * p.kv.page_size < shared)))
      Py_RETURN_NONE;
    if (a[9] == Py_None) L = std::min<int64_t>(std::max<int64_t>(int64_t{p.kv.max_pages} * p.kv.page_size, shared), int64_t{1} << 30);
    else if (!arg(a[9], &L) || L < 1 || L > INT32_MAX) Py_RETURN_NONE;
    if (out.defined() && (!plain_as(out, dt) || out.dim() != 2 || out.size(0) != t || out.size(1) != n_q * hd || !same_device(out, q)))
      Py_RETURN_NONE;
    if (ws.defined() && (!plain_as(ws, at::kByte) || !same_device(ws, q))) Py_RETURN_NONE;
    const c10::DeviceGuard on(q.device());
    if (!ws.defined()) {
      size_t need = 0;
      if (paged_attn_workspace_bytes_for(t, static_cast<int>(n_q), p.kv.n_kv, static_cast<int>(hd), p.kv.batch,
                                         static_cast<int>(L), static_cast<int>(shared), p.cu.defined(), &need) != Q4_OK)
        Py_RETURN_NONE;
      ws = at::empty({static_cast<int64_t>(std::max<size_t>(need, 16))}, q.options().dtype(at::kByte));
    }
    if (!out.defined()) out = at::empty({t, n_q * hd}, q.options());
    void* st = stream_of(q);
    const int rc = unlocked([&] {
      return paged_attn(&p.kv, q.data_ptr(), q.stride(0), q.stride(1), out.data_ptr(), code, t, static_cast<int>(n_q),
                        static_cast<int>(L), shared ? data<int32_t>(sp) : nullptr, static_cast<int>(shared), scale,
                        ws.data_ptr(), ws.numel(), st);
    });
    if (rc != Q4_OK) Py_RETURN_NONE;
    return a[11] != Py_None ? (Py_INCREF(a[11]), a[11]) : THPVariable_Wrap(out);
  });
}

// Rows of `n` fp32 or int32 values next to each other, on the device of `on`.
bool rows_of(const Tensor& t, at::ScalarType dt, at::IntArrayRef sizes, const Tensor& on) {
  return plain(t) && t.scalar_type() == dt && t.sizes() == sizes && (sizes.back() <= 1 || t.stride(-1) == 1) && same_device(t, on);
}

// verify(tokens, draft_probs, target_probs, uniforms, n_draft, workspace): (tokens, accepted)
PyObject* verify(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  return guarded([&]() -> PyObject* {
    Tensor tok, draft, target, u, nd, ws;
    if (nargs != 6 || !arg(a[0], &tok) || !arg(a[1], &draft, true) || !arg(a[2], &target) || !arg(a[3], &u) ||
        !arg(a[4], &nd, true) || !arg(a[5], &ws, true) || !plain(tok) || tok.dim() != 2 || !plain(target) || target.dim() != 3)
      Py_RETURN_NONE;
    const int64_t b = tok.size(0), k = tok.size(1), v = target.size(2);
    if (b < 1 || b > INT32_MAX || k > INT32_MAX || !rows_of(tok, at::kInt, {b, k}, target) ||
        !rows_of(target, at::kFloat, {b, k + 1, v}, target) || !rows_of(u, at::kFloat, {b, k + 1}, target) ||
        (draft.defined() && !rows_of(draft, at::kFloat, {b, k, v}, target)) || (nd.defined() && !indices(nd, b, target)) ||
        (ws.defined() && (!plain_as(ws, at::kByte) || !same_device(ws, target))))
      Py_RETURN_NONE;
    const c10::DeviceGuard on(target.device());
    if (!ws.defined()) {
      size_t need = 0;
      if (spec_verify_workspace_bytes(static_cast<int>(b), static_cast<int>(k), v, &need) != Q4_OK) Py_RETURN_NONE;
      ws = at::empty({static_cast<int64_t>(need)}, target.options().dtype(at::kByte));
    }
    Tensor out = at::empty({b, k + 1}, tok.options()), acc = at::empty({b}, tok.options());
    void* st = stream_of(target);
    const int rc = unlocked([&] {
      const bool d = draft.defined();
      return spec_verify(data<int32_t>(tok), tok.stride(0), data<float>(draft), d ? draft.stride(0) : 0, d ? draft.stride(1) : 0,
                         data<float>(target), target.stride(0), target.stride(1), data<float>(u), u.stride(0),
                         data<int32_t>(nd), static_cast<int>(b), static_cast<int>(k), v, data<int32_t>(out),
                         data<int32_t>(acc), ws.data_ptr(), ws.numel(), st);
    });
    if (rc != Q4_OK) Py_RETURN_NONE;
    return Py_BuildValue("(NN)", THPVariable_Wrap(out), THPVariable_Wrap(acc));
  });
}

PyMethodDef kMethods[] = {
    {"gemv", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(gemv)), METH_FASTCALL, nullptr},
    {"linear", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(linear)), METH_FASTCALL, nullptr},
    {"attn", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(attn)), METH_FASTCALL, nullptr},
    {"gemm", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(gemm)), METH_FASTCALL, nullptr},
    {"rope", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(rope)), METH_FASTCALL, nullptr},
    {"append", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(append)), METH_FASTCALL, nullptr},
    {"paged", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(paged)), METH_FASTCALL, nullptr},
    {"verify", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(verify)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_q4torch", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__q4torch() { return PyModule_Create(&kModule); }
