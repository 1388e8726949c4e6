// The tensor front ends of hipkittens_b200 in native code: argument checks, output allocation and the C-ABI call for the
// entry points that a serving loop calls once per layer and token. In Python the checks of one call (about sixty
// attribute reads), the stream lookup and the ctypes conversions took 9 to 11 us; here they take under 2.
//
// Every function returns None when an argument is anything but a plain CUDA tensor that the call accepts as it is. The
// Python front end then runs its own checks, which raise what there is to raise (or accept, for instance, a tensor
// subclass); nothing is decided here that is not decided there. Otherwise: an int (an HK_E* code) when the
// library refused the call, else the outputs.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAStream.h>
#include <cuda_runtime_api.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>

#include <optional>

#include "../../include/hk_attn.h"

namespace {

using at::Tensor;

// A plain strided CUDA tensor, or null. The wrappers of torch.func's transforms are of the exact class too, but have no
// storage, and so no pointer to read.
const Tensor* plain(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const Tensor& t = THPVariable_Unpack(o);
  return t.defined() && t.is_cuda() && t.layout() == at::kStrided && t.has_storage() ? &t : nullptr;
}
bool is(const Tensor* t, at::ScalarType type, int64_t dim) { return t && t->scalar_type() == type && t->dim() == dim; }
bool dense(const Tensor* t, at::ScalarType type, int64_t dim) { return is(t, type, dim) && t->is_contiguous(); }
bool same_device(const Tensor& ref, std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    if (t->device() != ref.device()) return false;
  return true;
}
// An output: the caller's, or a new one. False: the Python front end is to look at it.
bool output(PyObject* o, const Tensor& ref, at::IntArrayRef shape, at::ScalarType type, Tensor& out) {
  if (o == Py_None) {
    out = at::empty(shape, ref.options().dtype(type).requires_grad(false));
    return out.has_storage();  // under a transform a new tensor is a wrapper as well
  }
  const Tensor* t = plain(o);
  if (!dense(t, type, int64_t(shape.size())) || t->sizes() != shape || t->device() != ref.device()) return false;
  out = *t;
  return true;
}
void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }
int i32(int64_t v) { return static_cast<int>(v); }
bool fits(std::initializer_list<int64_t> vs) {  // ctypes would refuse what an int does not hold
  for (int64_t v : vs)
    if (v > 0x7fffffffll) return false;
  return true;
}
bool number(PyObject* o, float& v) {
  if (o == Py_None) {
    v = 0.f;
    return true;
  }
  if (!PyFloat_CheckExact(o)) return false;
  v = static_cast<float>(PyFloat_AS_DOUBLE(o));
  return true;
}

// The device pointer of a tensor. data_ptr() can throw and must not race with a resize_ or set_ of another thread, so it
// is read while the interpreter lock is held.
template <typename T = void>
T* ptr(const Tensor& t) { return static_cast<T*>(t.data_ptr()); }

// The library call without the interpreter lock, as ctypes makes it. `call` must not throw: it holds pointers and numbers
// that were read before, and touches no tensor.
template <typename Call>
int unlocked(const Call& call) {
  int rc;
  Py_BEGIN_ALLOW_THREADS rc = call();
  Py_END_ALLOW_THREADS return rc;
}
PyObject* result(int rc, const Tensor& a, const Tensor& b) {
  if (rc != HK_OK) return PyLong_FromLong(rc);
  return Py_BuildValue("(NN)", THPVariable_Wrap(a), THPVariable_Wrap(b));
}

bool tma_strides(const Tensor& t, long long* st) {
  bool good = t.stride(3) == 1;
  for (int i = 0; i < 3; ++i) {
    st[i] = t.stride(i);
    good = good && st[i] > 0 && st[i] % 8 == 0;
  }
  return good;
}

// A window and its sinks, as the last two arguments; without them, none.
bool window_args(PyObject* const* a, Py_ssize_t n_args, Py_ssize_t without, int& window, int& sinks) {
  window = sinks = 0;
  if (n_args == without) return true;
  if (n_args != without + 2 || !PyLong_CheckExact(a[without]) || !PyLong_CheckExact(a[without + 1])) return false;
  int over_w = 0, over_s = 0;
  const long w = PyLong_AsLongAndOverflow(a[without], &over_w), s = PyLong_AsLongAndOverflow(a[without + 1], &over_s);
  if (over_w || over_s || w < 1 || s < 0 || !fits({w, s})) return false;
  window = i32(w), sinks = i32(s);
  return true;
}

// attn_fwd(q, k, v, causal, softmax_scale, out, lse, kv_lens[, window, sinks])
PyObject* attn_fwd(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  float scale;
  int window, sinks;
  if (!window_args(a, n_args, 8, window, sinks) || !PyBool_Check(a[3]) || !number(a[4], scale)) Py_RETURN_NONE;
  if (window && a[3] != Py_True) Py_RETURN_NONE;
  const Tensor *q = plain(a[0]), *k = plain(a[1]), *v = plain(a[2]);
  for (const Tensor* t : {q, k, v})
    if (!is(t, at::kBFloat16, 4)) Py_RETURN_NONE;
  const int64_t b = q->size(0), n = q->size(1), h = q->size(2), d = q->size(3), nk = k->size(1), hkv = k->size(2);
  if (k->sizes() != v->sizes() || k->size(0) != b || k->size(3) != d || !same_device(*q, {k, v}) ||
      !fits({b, n, nk, h, hkv}))
    Py_RETURN_NONE;
  const bool strided = !(q->is_contiguous() && k->is_contiguous() && v->is_contiguous());
  long long qs[3], ks[3], vs[3];
  const bool q_ok = tma_strides(*q, qs), k_ok = tma_strides(*k, ks), v_ok = tma_strides(*v, vs);
  if ((strided || window) && !(q_ok && k_ok && v_ok)) Py_RETURN_NONE;
  const Tensor* lens = nullptr;
  if (a[7] != Py_None) {
    lens = plain(a[7]);
    if (!dense(lens, at::kInt, 1) || lens->size(0) != b || lens->device() != q->device()) Py_RETURN_NONE;
  }
  Tensor out, lse;
  if (!output(a[5], *q, q->sizes(), at::kBFloat16, out) || !output(a[6], *q, {b, h, 1, n}, at::kFloat, lse))
    Py_RETURN_NONE;
  void* st = stream_of(*q);
  const int causal = a[3] == Py_True, dev = q->device().index();
  const void *qp = ptr(*q), *kp = ptr(*k), *vp = ptr(*v);
  void* outp = ptr(out);
  float* lsep = ptr<float>(lse);
  const int32_t* lensp = lens ? ptr<int32_t>(*lens) : nullptr;
  const int rc = unlocked([&] {
    if (window)
      return hk_attn_fwd_window(qp, kp, vp, outp, lsep, i32(b), i32(n), i32(nk), i32(h), i32(hkv), i32(d), qs, ks, vs, lensp,
                                window, sinks, scale, dev, st);
    if (lens || nk != n || strided)
      return hk_attn_fwd_cross(qp, kp, vp, outp, lsep, i32(b), i32(n), i32(nk), i32(h), i32(hkv), i32(d), qs, ks, vs, lensp,
                               causal, scale, dev, st);
    return hk_attn_fwd(qp, kp, vp, outp, lsep, i32(b), i32(n), i32(h), i32(hkv), i32(d), causal, scale, dev, st);
  });
  return result(rc, out, lse);
  END_HANDLE_TH_ERRORS
}

// attn_bwd_strided(q, k, v, o, d_o, lse, dq, dk, dv, causal, softmax_scale, kv_lens[, window, sinks]): 0 when launched
PyObject* attn_bwd_strided(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  float scale;
  int window, sinks;
  if (!window_args(a, n_args, 12, window, sinks) || !PyBool_Check(a[9]) || !number(a[10], scale)) Py_RETURN_NONE;
  if (window && a[9] != Py_True) Py_RETURN_NONE;
  const Tensor *q = plain(a[0]), *k = plain(a[1]), *v = plain(a[2]), *o = plain(a[3]), *d_o = plain(a[4]),
               *lse = plain(a[5]), *dq = plain(a[6]), *dk = plain(a[7]), *dv = plain(a[8]);
  for (const Tensor* t : {q, k, v, dq, dk, dv})
    if (!is(t, at::kBFloat16, 4)) Py_RETURN_NONE;
  if (!dense(o, at::kBFloat16, 4) || !dense(d_o, at::kBFloat16, 4) || !dense(lse, at::kFloat, 4)) Py_RETURN_NONE;
  const int64_t b = q->size(0), n = q->size(1), h = q->size(2), d = q->size(3), nk = k->size(1), hkv = k->size(2);
  for (const Tensor* t : {o, d_o, dq})
    if (t->sizes() != q->sizes()) Py_RETURN_NONE;
  for (const Tensor* t : {v, dk, dv})
    if (t->sizes() != k->sizes()) Py_RETURN_NONE;
  if (k->size(0) != b || k->size(3) != d || lse->sizes() != at::IntArrayRef({b, h, 1, n}) ||
      !same_device(*q, {k, v, o, d_o, lse, dq, dk, dv}) || !fits({b, n, nk, h, hkv}))
    Py_RETURN_NONE;
  long long st[6][3];
  int i = 0;
  for (const Tensor* t : {q, k, v, dq, dk, dv})
    if (!tma_strides(*t, st[i++])) Py_RETURN_NONE;
  const Tensor* lens = nullptr;
  if (a[11] != Py_None) {
    lens = plain(a[11]);
    if (!dense(lens, at::kInt, 1) || lens->size(0) != b || lens->device() != q->device()) Py_RETURN_NONE;
  }
  const Tensor delta = at::empty({b, h, 1, n}, lse->options().requires_grad(false));
  if (!delta.has_storage()) Py_RETURN_NONE;
  Tensor ws;
  const size_t need =
      window ? hk_attn_bwd_window_workspace_bytes(i32(b), i32(n), i32(nk), i32(h), i32(hkv), i32(d), window, sinks) : 0;
  if (need && !output(Py_None, *q, {int64_t(need)}, at::kByte, ws)) Py_RETURN_NONE;
  void* stream = stream_of(*q);
  const int causal = a[9] == Py_True, dev = q->device().index();
  const void *qp = ptr(*q), *kp = ptr(*k), *vp = ptr(*v), *op = ptr(*o), *dop = ptr(*d_o);
  const float* lsep = ptr<float>(*lse);
  float* deltap = ptr<float>(delta);
  void *dqp = ptr(*dq), *dkp = ptr(*dk), *dvp = ptr(*dv);
  const int32_t* lensp = lens ? ptr<int32_t>(*lens) : nullptr;
  void* wsp = need ? ptr(ws) : nullptr;
  const int rc = unlocked([&] {
    if (window)
      return hk_attn_bwd_window(qp, kp, vp, op, dop, lsep, deltap, dqp, dkp, dvp, i32(b), i32(n), i32(nk), i32(h), i32(hkv),
                                i32(d), st[0], st[1], st[2], st[3], st[4], st[5], lensp, window, sinks, scale, wsp, need, dev,
                                stream);
    return hk_attn_bwd_strided(qp, kp, vp, op, dop, lsep, deltap, dqp, dkp, dvp, i32(b), i32(n), i32(nk), i32(h),
                               i32(hkv), i32(d), st[0], st[1], st[2], st[3], st[4], st[5], lensp, causal, scale, dev,
                               stream);
  });
  return PyLong_FromLong(rc);
  END_HANDLE_TH_ERRORS
}

// rotary_bnhd(x, cos, sin, out, pos_offset)
PyObject* rotary_bnhd(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  if (n_args != 5 || !PyLong_CheckExact(a[4])) Py_RETURN_NONE;
  int overflow = 0;
  const long pos = PyLong_AsLongAndOverflow(a[4], &overflow);
  const Tensor *x = plain(a[0]), *cos = plain(a[1]), *sin = plain(a[2]);
  if (overflow || pos < 0 || !dense(x, at::kBFloat16, 4) || !dense(cos, at::kBFloat16, 2) ||
      !dense(sin, at::kBFloat16, 2))
    Py_RETURN_NONE;
  if (cos->sizes() != sin->sizes() || cos->size(0) < x->size(1) + pos || !same_device(*x, {cos, sin}) ||
      !fits({x->size(0), x->size(1), x->size(2), x->size(3), 2 * cos->size(1), pos}))
    Py_RETURN_NONE;
  Tensor out;
  if (!output(a[3], *x, x->sizes(), at::kBFloat16, out)) Py_RETURN_NONE;
  void* st = stream_of(*x);
  const int b = i32(x->size(0)), n = i32(x->size(1)), h = i32(x->size(2)), d = i32(x->size(3)), r = i32(2 * cos->size(1));
  const int dev = x->device().index();
  const void *xp = ptr(*x), *sinp = ptr(*sin), *cosp = ptr(*cos);
  void* outp = ptr(out);
  const int rc = unlocked([&] { return hk_rotary_bnhd(xp, outp, sinp, cosp, b, n, h, d, r, i32(pos), dev, st); });
  if (rc != HK_OK) return PyLong_FromLong(rc);
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// What the norm and rotation of q and k and its gradients share; `arg` holds q, k, q_weight, k_weight, cos, sin.
struct Qkn {
  const Tensor *q, *k, *w[2], *cos, *sin, *positions;
  long long qs[3], ks[3];
  int flags = 0, pos_offset;
  float eps;
  const void *q_ptr, *k_ptr, *w_ptr[2], *cos_ptr, *sin_ptr;
  const int32_t* pos_ptr;
  int b, n, h, hkv, d, r, rows, device;
  bool take(PyObject* const* arg, PyObject* pos, PyObject* offset, PyObject* eps_arg, PyObject* interleaved) {
    q = plain(arg[0]), k = plain(arg[1]), cos = plain(arg[4]), sin = plain(arg[5]);
    if (!is(q, at::kBFloat16, 4) || !is(k, at::kBFloat16, 4) || !PyBool_Check(interleaved) || !PyFloat_CheckExact(eps_arg) ||
        !PyLong_CheckExact(offset))
      return false;
    if (k->size(0) != q->size(0) || k->size(1) != q->size(1) || k->size(3) != q->size(3) || !q->numel() || !k->numel()) return false;
    const bool q_ok = tma_strides(*q, qs), k_ok = tma_strides(*k, ks);
    if (!q_ok || !k_ok) return false;
    if (!(dense(cos, at::kBFloat16, 2) && dense(sin, at::kBFloat16, 2))) {
      if (!(dense(cos, at::kFloat, 2) && dense(sin, at::kFloat, 2))) return false;
      flags |= HK_QKN_TABLE_F32;
    }
    if (cos->sizes() != sin->sizes() || !same_device(*q, {k, cos, sin})) return false;
    bool f32 = false, b16 = false;
    for (int i = 0; i < 2; ++i) {
      w[i] = nullptr;
      if (arg[2 + i] == Py_None) continue;
      w[i] = plain(arg[2 + i]);
      if (!w[i] || w[i]->dim() != 1 || w[i]->size(0) != q->size(3) || !w[i]->is_contiguous() || w[i]->device() != q->device())
        return false;
      f32 |= w[i]->scalar_type() == at::kFloat, b16 |= w[i]->scalar_type() == at::kBFloat16;
      if (w[i]->scalar_type() != at::kFloat && w[i]->scalar_type() != at::kBFloat16) return false;
    }
    if (f32 && b16) return false;
    if (f32) flags |= HK_QKN_WEIGHT_F32;
    int overflow = 0;
    const long off = PyLong_AsLongAndOverflow(offset, &overflow);
    if (overflow || off < 0 || !fits({off, cos->size(0), 2 * cos->size(1)})) return false;
    for (int64_t v : q->sizes())
      if (!fits({v})) return false;
    positions = nullptr;
    if (pos != Py_None) {
      positions = plain(pos);
      if (!dense(positions, at::kInt, 2) || positions->size(0) != q->size(0) || positions->size(1) != q->size(1) ||
          positions->device() != q->device() || off != 0)
        return false;
    } else if (cos->size(0) < q->size(1) + off) {
      return false;
    }
    eps = static_cast<float>(PyFloat_AS_DOUBLE(eps_arg));
    if (!(eps >= 0.f)) return false;
    if (interleaved == Py_True) flags |= HK_QKN_INTERLEAVED;
    pos_offset = i32(off);
    b = i32(q->size(0)), n = i32(q->size(1)), h = i32(q->size(2)), d = i32(q->size(3)), hkv = i32(k->size(2));
    r = i32(2 * cos->size(1)), rows = i32(cos->size(0)), device = q->device().index();
    return true;
  }
  void read() {
    q_ptr = ptr(*q), k_ptr = ptr(*k), cos_ptr = ptr(*cos), sin_ptr = ptr(*sin);
    for (int i = 0; i < 2; ++i) w_ptr[i] = w[i] ? ptr(*w[i]) : nullptr;
    pos_ptr = positions ? ptr<int32_t>(*positions) : nullptr;
  }
};

// qk_norm_rotary(q, k, q_weight, k_weight, cos, sin, positions, pos_offset, eps, interleaved, q_out, k_out)
PyObject* qk_norm_rotary(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  Qkn p;
  if (n_args != 12 || !p.take(a, a[6], a[7], a[8], a[9])) Py_RETURN_NONE;
  Tensor qo, ko;
  if (!output(a[10], *p.q, p.q->sizes(), at::kBFloat16, qo) || !output(a[11], *p.q, p.k->sizes(), at::kBFloat16, ko))
    Py_RETURN_NONE;
  void* st = stream_of(*p.q);
  p.read();
  void *qop = ptr(qo), *kop = ptr(ko);
  const int rc = unlocked([&] {
    return hk_qk_norm_rotary(p.q_ptr, p.k_ptr, p.w_ptr[0], p.w_ptr[1], p.cos_ptr, p.sin_ptr, qop, kop, p.b, p.n, p.h, p.hkv,
                             p.d, p.r, p.rows, p.qs, p.ks, p.pos_ptr, p.pos_offset, p.eps, p.flags, p.device, st);
  });
  return result(rc, qo, ko);
  END_HANDLE_TH_ERRORS
}

// qk_norm_rotary_bwd(q, k, q_weight, k_weight, cos, sin, dq_out, dk_out, positions, pos_offset, eps, interleaved, weight_grads)
PyObject* qk_norm_rotary_bwd(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  Qkn p;
  if (n_args != 13 || !PyBool_Check(a[12]) || !p.take(a, a[8], a[9], a[10], a[11])) Py_RETURN_NONE;
  const Tensor* dy[2] = {plain(a[6]), plain(a[7])};
  const Tensor* x[2] = {p.q, p.k};
  Tensor dx[2], dw[2], ws;
  bool sums = false;
  for (int i = 0; i < 2; ++i) {
    if (!dense(dy[i], at::kBFloat16, 4) || dy[i]->sizes() != x[i]->sizes() || dy[i]->device() != p.q->device() ||
        !output(Py_None, *p.q, x[i]->sizes(), at::kBFloat16, dx[i]))
      Py_RETURN_NONE;
    if (a[12] == Py_True && p.w[i]) {
      if (!output(Py_None, *p.w[i], p.w[i]->sizes(), p.w[i]->scalar_type(), dw[i])) Py_RETURN_NONE;
      sums = true;
    }
  }
  const size_t need = sums ? hk_qk_norm_rotary_bwd_workspace_bytes(p.d) : 0;
  if (need && !output(Py_None, *p.q, {int64_t(need)}, at::kByte, ws)) Py_RETURN_NONE;
  void* st = stream_of(*p.q);
  p.read();
  const void *dqo = ptr(*dy[0]), *dko = ptr(*dy[1]);
  void *dq = ptr(dx[0]), *dk = ptr(dx[1]), *dqw = dw[0].defined() ? ptr(dw[0]) : nullptr,
       *dkw = dw[1].defined() ? ptr(dw[1]) : nullptr, *wsp = need ? ptr(ws) : nullptr;
  const int rc = unlocked([&] {
    return hk_qk_norm_rotary_bwd(p.q_ptr, p.k_ptr, p.w_ptr[0], p.w_ptr[1], p.cos_ptr, p.sin_ptr, dqo, dko, dq, dk, dqw, dkw,
                                 p.b, p.n, p.h, p.hkv, p.d, p.r, p.rows, p.qs, p.ks, p.pos_ptr, p.pos_offset, p.eps,
                                 p.flags, wsp, need, p.device, st);
  });
  if (rc != HK_OK) return PyLong_FromLong(rc);
  auto wrapped = [](const Tensor& t) {
    if (t.defined()) return THPVariable_Wrap(t);
    Py_INCREF(Py_None);
    return Py_None;
  };
  return Py_BuildValue("(NNNN)", THPVariable_Wrap(dx[0]), THPVariable_Wrap(dx[1]), wrapped(dw[0]), wrapped(dw[1]));
  END_HANDLE_TH_ERRORS
}

// What the paged entries share: q [S,T,H,D], pools [P,page,H_KV,D], block_table [S,max_pages], lengths [S].
struct Paged {
  const Tensor *q, *kp, *vp, *table, *lens;
  int64_t s, t, h, d, pool, page, hkv, max_pages;
  void *q_ptr, *k_pages, *v_pages;
  const int32_t *table_ptr, *lens_ptr;
  int device;
  // What the library call needs of the tensors, read before the interpreter lock is given up.
  void read() {
    q_ptr = ptr(*q), k_pages = ptr(*kp), v_pages = ptr(*vp);
    table_ptr = ptr<int32_t>(*table), lens_ptr = ptr<int32_t>(*lens);
    device = q->device().index();
  }
  bool take(PyObject* const* a) {
    q = plain(a[0]), kp = plain(a[1]), vp = plain(a[2]), table = plain(a[3]), lens = plain(a[4]);
    if (!dense(q, at::kBFloat16, 4) || !dense(kp, at::kBFloat16, 4) || !dense(vp, at::kBFloat16, 4) ||
        !dense(table, at::kInt, 2) || !dense(lens, at::kInt, 1))
      return false;
    s = q->size(0), t = q->size(1), h = q->size(2), d = q->size(3);
    pool = kp->size(0), page = kp->size(1), hkv = kp->size(2), max_pages = table->size(1);
    return kp->size(3) == d && vp->sizes() == kp->sizes() && table->size(0) == s && lens->size(0) == s &&
           same_device(*q, {kp, vp, table, lens}) && fits({s, t, h, d, pool, page, hkv, max_pages});
  }
};

// paged_decode(q, k_pages, v_pages, block_table, ctx_lens, softmax_scale, out, lse, workspace[, window, sinks])
PyObject* paged_decode(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  float scale;
  Paged p;
  int window, sinks;
  if (!window_args(a, n_args, 9, window, sinks) || !number(a[5], scale) || !p.take(a) || p.t != 1) Py_RETURN_NONE;
  const size_t need =
      window ? hk_attn_paged_decode_window_workspace_bytes(i32(p.s), i32(p.h), i32(p.d), i32(p.max_pages), i32(p.page), window, sinks)
             : hk_attn_paged_decode_workspace_bytes(i32(p.s), i32(p.h), i32(p.d), i32(p.max_pages), i32(p.page));
  Tensor out, lse, ws;
  if (need == 0 || !output(a[6], *p.q, p.q->sizes(), at::kBFloat16, out) ||
      !output(a[7], *p.q, {p.s, p.h, 1, 1}, at::kFloat, lse))
    Py_RETURN_NONE;
  if (a[8] == Py_None) {
    ws = at::empty({int64_t(need < 256 ? 256 : need)}, p.q->options().dtype(at::kByte).requires_grad(false));
    if (!ws.has_storage()) Py_RETURN_NONE;
  } else {
    const Tensor* t = plain(a[8]);
    if (!dense(t, at::kByte, 1) || t->device() != p.q->device()) Py_RETURN_NONE;
    ws = *t;
  }
  void* st = stream_of(*p.q);
  p.read();
  void *outp = ptr(out), *wsp = ptr(ws);
  float* lsep = ptr<float>(lse);
  const size_t ws_bytes = size_t(ws.numel());
  const int rc = unlocked([&] {
    if (window)
      return hk_attn_paged_decode_window(p.q_ptr, p.k_pages, p.v_pages, p.table_ptr, p.lens_ptr, outp, lsep, i32(p.s), i32(p.h),
                                         i32(p.hkv), i32(p.d), i32(p.page), i32(p.max_pages), i32(p.pool), window, sinks, scale,
                                         wsp, ws_bytes, p.device, st);
    return hk_attn_paged_decode(p.q_ptr, p.k_pages, p.v_pages, p.table_ptr, p.lens_ptr, outp, lsep, i32(p.s), i32(p.h),
                                i32(p.hkv), i32(p.d), i32(p.page), i32(p.max_pages), i32(p.pool), scale, wsp, ws_bytes,
                                p.device, st);
  });
  return result(rc, out, lse);
  END_HANDLE_TH_ERRORS
}

// attn_fwd_paged(q, k_pages, v_pages, block_table, ctx_lens, causal, softmax_scale, out, lse[, window, sinks])
PyObject* attn_fwd_paged(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  float scale;
  Paged p;
  int window, sinks;
  if (!window_args(a, n_args, 9, window, sinks) || !PyBool_Check(a[5]) || !number(a[6], scale) || !p.take(a)) Py_RETURN_NONE;
  if (window && a[5] != Py_True) Py_RETURN_NONE;
  Tensor out, lse;
  if (!output(a[7], *p.q, p.q->sizes(), at::kBFloat16, out) ||
      !output(a[8], *p.q, {p.s, p.h, 1, p.t}, at::kFloat, lse))
    Py_RETURN_NONE;
  void* st = stream_of(*p.q);
  p.read();
  const int causal = a[5] == Py_True;
  void* outp = ptr(out);
  float* lsep = ptr<float>(lse);
  const int rc = unlocked([&] {
    if (window)
      return hk_attn_fwd_paged_window(p.q_ptr, p.k_pages, p.v_pages, p.table_ptr, p.lens_ptr, outp, lsep, i32(p.s), i32(p.t),
                                      i32(p.h), i32(p.hkv), i32(p.d), i32(p.page), i32(p.max_pages), i32(p.pool), window, sinks,
                                      scale, p.device, st);
    return hk_attn_fwd_paged(p.q_ptr, p.k_pages, p.v_pages, p.table_ptr, p.lens_ptr, outp, lsep, i32(p.s), i32(p.t),
                             i32(p.h), i32(p.hkv), i32(p.d), i32(p.page), i32(p.max_pages), i32(p.pool), causal, scale,
                             p.device, st);
  });
  return result(rc, out, lse);
  END_HANDLE_TH_ERRORS
}

// paged_kv_append(k_new, v_new, k_pages, v_pages, block_table, start_pos[, cos, sin]): 0 when launched
PyObject* paged_kv_append(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  if (n_args != 6 && n_args != 8) Py_RETURN_NONE;
  const Tensor* v_new = plain(a[1]);
  PyObject* const shared[5] = {a[0], a[2], a[3], a[4], a[5]};
  Paged p;  // k_new in the place of q
  if (!p.take(shared) || !dense(v_new, at::kBFloat16, 4) || v_new->sizes() != p.q->sizes() || p.h != p.hkv ||
      v_new->device() != p.q->device())
    Py_RETURN_NONE;
  const Tensor *cos = nullptr, *sin = nullptr;
  if (n_args == 8) {
    cos = plain(a[6]), sin = plain(a[7]);
    if (!dense(cos, at::kBFloat16, 2) || !dense(sin, at::kBFloat16, 2) || cos->sizes() != sin->sizes() ||
        !same_device(*p.q, {cos, sin}) || !fits({cos->size(0), 2 * cos->size(1)}))
      Py_RETURN_NONE;
  }
  void* st = stream_of(*p.q);
  p.read();
  const void *vp = ptr(*v_new), *cosp = cos ? ptr(*cos) : nullptr, *sinp = cos ? ptr(*sin) : nullptr;
  const int rows = cos ? i32(cos->size(0)) : 0, rotary_dim = cos ? i32(2 * cos->size(1)) : 0;
  const int rc = unlocked([&] {
    if (n_args == 8)
      return hk_paged_kv_append_rotary(p.q_ptr, vp, p.k_pages, p.v_pages, p.table_ptr, p.lens_ptr, sinp, cosp, i32(p.s),
                                       i32(p.t), i32(p.h), i32(p.d), rotary_dim, rows, i32(p.page), i32(p.max_pages),
                                       i32(p.pool), p.device, st);
    return hk_paged_kv_append(p.q_ptr, vp, p.k_pages, p.v_pages, p.table_ptr, p.lens_ptr, i32(p.s), i32(p.t), i32(p.h),
                              i32(p.d), i32(p.page), i32(p.max_pages), i32(p.pool), p.device, st);
  });
  return PyLong_FromLong(rc);
  END_HANDLE_TH_ERRORS
}

// An 8-bit paged cache: k_pages, v_pages, k_scales, v_scales, block_table.
struct Fp8Cache {
  const Tensor *kp, *vp, *ks, *vs, *table;
  int64_t s, pool, page, hkv, d, max_pages;
  void *k_pages, *v_pages;
  float *k_scales, *v_scales;
  const int32_t* table_ptr;
  int device;
  bool take(PyObject* const* a) {
    kp = plain(a[0]), vp = plain(a[1]), ks = plain(a[2]), vs = plain(a[3]), table = plain(a[4]);
    if (!dense(kp, at::kFloat8_e4m3fn, 4) || !dense(vp, at::kFloat8_e4m3fn, 4) || !dense(ks, at::kFloat, 2) || !dense(vs, at::kFloat, 2) ||
        !dense(table, at::kInt, 2))
      return false;
    pool = kp->size(0), page = kp->size(1), hkv = kp->size(2), d = kp->size(3), s = table->size(0), max_pages = table->size(1);
    const std::initializer_list<int64_t> scales = {pool, hkv};
    return vp->sizes() == kp->sizes() && ks->sizes() == at::IntArrayRef(scales) && vs->sizes() == at::IntArrayRef(scales) &&
           same_device(*kp, {vp, ks, vs, table}) && fits({pool, page, hkv, d, s, max_pages}) && kp->numel() && table->numel();
  }
  void read() {
    k_pages = ptr(*kp), v_pages = ptr(*vp), k_scales = ptr<float>(*ks), v_scales = ptr<float>(*vs), table_ptr = ptr<int32_t>(*table);
    device = kp->device().index();
  }
  // int32 [n] beside it, or null for None; false: neither
  bool ints(PyObject* o, int64_t n, const Tensor*& t) const {
    t = nullptr;
    if (o == Py_None) return true;
    t = plain(o);
    return dense(t, at::kInt, 1) && t->size(0) == n && t->device() == kp->device();
  }
};

// paged_kv_append_fp8(k_new, v_new, k_pages, v_pages, k_scales, v_scales, block_table, start_pos, cos, sin, cu_seqlens): 0 when launched
PyObject* paged_kv_append_fp8(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  Fp8Cache c;
  const Tensor *start, *cu;
  if (n_args != 11 || !c.take(a + 2) || a[7] == Py_None || !c.ints(a[7], c.s, start) || !c.ints(a[10], c.s + 1, cu)) Py_RETURN_NONE;
  const int dims = cu ? 3 : 4;
  const Tensor* x[2] = {plain(a[0]), plain(a[1])};
  long long st[2][3];
  for (int i = 0; i < 2; ++i) {
    const Tensor* t = x[i];
    if (!is(t, at::kBFloat16, dims) || !t->numel() || t->size(dims - 2) != c.hkv || t->size(dims - 1) != c.d ||
        (!cu && t->size(0) != c.s) || t->device() != c.kp->device() || t->stride(dims - 1) != 1 || t->sizes() != x[0]->sizes())
      Py_RETURN_NONE;
    st[i][0] = 0;
    for (int k = cu ? 1 : 0; k < 3; ++k) {
      st[i][k] = t->stride(cu ? k - 1 : k);
      if (st[i][k] <= 0 || st[i][k] % 8 != 0) Py_RETURN_NONE;
    }
  }
  const int64_t tokens = x[0]->size(dims - 3);
  const Tensor *cos = nullptr, *sin = nullptr;
  int flags = 0;
  if (a[8] != Py_None || a[9] != Py_None) {
    cos = plain(a[8]), sin = plain(a[9]);
    if (!(dense(cos, at::kBFloat16, 2) && dense(sin, at::kBFloat16, 2))) {
      if (!(dense(cos, at::kFloat, 2) && dense(sin, at::kFloat, 2))) Py_RETURN_NONE;
      flags = HK_FP8_TABLE_F32;
    }
    if (cos->sizes() != sin->sizes() || !same_device(*c.kp, {cos, sin}) || !fits({cos->size(0), 2 * cos->size(1)})) Py_RETURN_NONE;
  }
  if (!fits({tokens})) Py_RETURN_NONE;
  void* stream = stream_of(*c.kp);
  c.read();
  const void *kn = ptr(*x[0]), *vn = ptr(*x[1]), *cosp = cos ? ptr(*cos) : nullptr, *sinp = cos ? ptr(*sin) : nullptr;
  const int rows = cos ? i32(cos->size(0)) : 0, rotary_dim = cos ? i32(2 * cos->size(1)) : 0;
  const int32_t *startp = ptr<int32_t>(*start), *cup = cu ? ptr<int32_t>(*cu) : nullptr;
  const int rc = unlocked([&] {
    return hk_paged_kv_append_fp8(kn, vn, c.k_pages, c.v_pages, c.k_scales, c.v_scales, c.table_ptr, startp, cup, sinp, cosp, i32(c.s),
                                  i32(tokens), i32(c.hkv), i32(c.d), st[0], st[1], rotary_dim, rows, flags, i32(c.page),
                                  i32(c.max_pages), i32(c.pool), c.device, stream);
  });
  return PyLong_FromLong(rc);
  END_HANDLE_TH_ERRORS
}

// paged_kv_read_fp8(k_pages, v_pages, k_scales, v_scales, block_table, rows, ctx_lens, cu_seqlens, k_out, v_out)
PyObject* paged_kv_read_fp8(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  Fp8Cache c;
  const Tensor *lens, *cu;
  if (n_args != 10 || !c.take(a) || !PyLong_CheckExact(a[5]) || !c.ints(a[6], c.s, lens) || !c.ints(a[7], c.s + 1, cu) || !lens == !cu ||
      (a[8] == Py_None) != (a[9] == Py_None))
    Py_RETURN_NONE;
  int overflow = 0;
  const long rows = PyLong_AsLongAndOverflow(a[5], &overflow);
  if (overflow || rows <= 0 || !fits({rows})) Py_RETURN_NONE;
  Tensor out[2];
  for (int i = 0; i < 2; ++i)
    if (!(cu ? output(a[8 + i], *c.kp, {rows, c.hkv, c.d}, at::kBFloat16, out[i])
             : output(a[8 + i], *c.kp, {c.s, rows, c.hkv, c.d}, at::kBFloat16, out[i])))
      Py_RETURN_NONE;
  void* stream = stream_of(*c.kp);
  c.read();
  void *ko = ptr(out[0]), *vo = ptr(out[1]);
  const int32_t *lensp = lens ? ptr<int32_t>(*lens) : nullptr, *cup = cu ? ptr<int32_t>(*cu) : nullptr;
  const int zero_rest = a[8] == Py_None;
  const int rc = unlocked([&] {
    return hk_paged_kv_read_fp8(c.k_pages, c.v_pages, c.k_scales, c.v_scales, c.table_ptr, lensp, cup, ko, vo, i32(c.s), i32(rows),
                                i32(c.hkv), i32(c.d), zero_rest, i32(c.page), i32(c.max_pages), i32(c.pool), c.device, stream);
  });
  return result(rc, out[0], out[1]);
  END_HANDLE_TH_ERRORS
}

// paged_decode_fp8(q, k_pages, v_pages, k_scales, v_scales, block_table, ctx_lens, softmax_scale, out, lse, workspace, window or 0, sinks)
PyObject* paged_decode_fp8(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  Fp8Cache c;
  float scale;
  const Tensor* lens;
  if (n_args != 13 || !c.take(a + 1) || a[6] == Py_None || !c.ints(a[6], c.s, lens) || !number(a[7], scale)) Py_RETURN_NONE;
  int window = 0, sinks = 0;
  if (!PyLong_CheckExact(a[11]) || (PyObject_IsTrue(a[11]) && !window_args(a, n_args, 11, window, sinks))) Py_RETURN_NONE;
  const Tensor* q = plain(a[0]);
  if (!dense(q, at::kBFloat16, 4) || q->size(0) != c.s || q->size(1) != 1 || q->size(3) != c.d || q->device() != c.kp->device() ||
      !fits({q->size(2)}))
    Py_RETURN_NONE;
  const int64_t h = q->size(2);
  const size_t need = hk_attn_paged_decode_fp8_workspace_bytes(i32(c.s), i32(c.hkv), i32(c.d));
  Tensor out, lse, ws;
  if (need == 0 || !output(a[8], *q, q->sizes(), at::kBFloat16, out) || !output(a[9], *q, {c.s, h, 1, 1}, at::kFloat, lse))
    Py_RETURN_NONE;
  if (a[10] == Py_None) {
    if (!output(Py_None, *q, {int64_t(need)}, at::kByte, ws)) Py_RETURN_NONE;
  } else {
    const Tensor* t = plain(a[10]);
    if (!dense(t, at::kByte, 1) || t->device() != q->device()) Py_RETURN_NONE;
    ws = *t;
  }
  void* stream = stream_of(*q);
  c.read();
  void *qp = ptr(*q), *outp = ptr(out), *wsp = ptr(ws);
  float* lsep = ptr<float>(lse);
  const int32_t* lensp = ptr<int32_t>(*lens);
  const size_t ws_bytes = size_t(ws.numel());
  const int rc = unlocked([&] {
    return hk_attn_paged_decode_fp8(qp, c.k_pages, c.v_pages, c.k_scales, c.v_scales, c.table_ptr, lensp, outp, lsep, i32(c.s), i32(h),
                                    i32(c.hkv), i32(c.d), i32(c.page), i32(c.max_pages), i32(c.pool), window, sinks, scale, wsp,
                                    ws_bytes, c.device, stream);
  });
  return result(rc, out, lse);
  END_HANDLE_TH_ERRORS
}

// A ragged batch: q, k, v, cu_seqlens_q, cu_seqlens_k or None.
struct Ragged {
  const Tensor *q, *k, *v, *cu_q, *cu_k;
  long long qs[2], ks[2], vs[2];
  int s, tq, tk, h, hkv, d, device;
  static bool strides(const Tensor& t, long long* st) {  // [rows, heads, D]
    for (int i = 0; i < 2; ++i) {
      st[i] = t.stride(i);
      if (st[i] <= 0 || st[i] % 8 != 0) return false;
    }
    return t.stride(2) == 1;
  }
  bool take(PyObject* const* a) { return take(plain(a[0]), plain(a[1]), plain(a[2]), plain(a[3]), a[4] == Py_None ? plain(a[3]) : plain(a[4])); }
  bool take(const Tensor* q_, const Tensor* k_, const Tensor* v_, const Tensor* cu_q_, const Tensor* cu_k_) {
    q = q_, k = k_, v = v_, cu_q = cu_q_, cu_k = cu_k_;
    for (const Tensor* t : {q, k, v})
      if (!is(t, at::kBFloat16, 3) || !t->numel()) return false;
    if (!dense(cu_q, at::kInt, 1) || !dense(cu_k, at::kInt, 1) || cu_q->size(0) < 2 || cu_k->size(0) != cu_q->size(0)) return false;
    if (k->sizes() != v->sizes() || k->size(2) != q->size(2) || (cu_k == cu_q && k->size(0) != q->size(0)) ||
        !same_device(*q, {k, v, cu_q, cu_k}) || !fits({q->size(0), k->size(0), q->size(1), k->size(1), cu_q->size(0)}))
      return false;
    s = i32(cu_q->size(0) - 1), tq = i32(q->size(0)), tk = i32(k->size(0)), h = i32(q->size(1)), hkv = i32(k->size(1)), d = i32(q->size(2));
    device = q->device().index();
    return strides(*q, qs) && strides(*k, ks) && strides(*v, vs);
  }
};

// attn_fwd_ragged(q, k, v, cu_seqlens_q, cu_seqlens_k, causal, softmax_scale, out, lse)
PyObject* attn_fwd_ragged(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  Ragged r;
  float scale;
  if (n_args != 9 || !PyBool_Check(a[5]) || !number(a[6], scale) || !r.take(a) || (a[7] == Py_None) != (a[8] == Py_None)) Py_RETURN_NONE;
  Tensor out, lse, ws;
  const size_t need = hk_attn_fwd_ragged_workspace_bytes(r.s, r.tq);
  if (!output(a[7], *r.q, r.q->sizes(), at::kBFloat16, out) || !output(a[8], *r.q, {r.h, r.tq}, at::kFloat, lse) ||
      !output(Py_None, *r.q, {int64_t(need)}, at::kByte, ws))
    Py_RETURN_NONE;
  void* st = stream_of(*r.q);
  const void *qp = ptr(*r.q), *kp = ptr(*r.k), *vp = ptr(*r.v);
  void *op = ptr(out), *wsp = ptr(ws);
  float* lp = ptr<float>(lse);
  const int32_t *cq = ptr<int32_t>(*r.cu_q), *ck = ptr<int32_t>(*r.cu_k);
  const int causal = a[5] == Py_True, fill = a[7] == Py_None;
  const int rc = unlocked([&] {
    return hk_attn_fwd_ragged(qp, kp, vp, op, lp, cq, ck, r.s, r.tq, r.tk, r.h, r.hkv, r.d, r.qs, r.ks, r.vs, causal, scale, fill, wsp, need,
                              r.device, st);
  });
  return result(rc, out, lse);
  END_HANDLE_TH_ERRORS
}

// attn_bwd_ragged(q, k, v, o, d_o, lse, cu_seqlens_q, cu_seqlens_k, causal, softmax_scale, dq, dk, dv)
PyObject* attn_bwd_ragged(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  Ragged r;
  float scale;
  if (n_args != 13) Py_RETURN_NONE;
  const Tensor *cu = plain(a[6]), *o = plain(a[3]), *d_o = plain(a[4]), *lse = plain(a[5]);
  if (!PyBool_Check(a[8]) || !number(a[9], scale) || !r.take(plain(a[0]), plain(a[1]), plain(a[2]), cu, a[7] == Py_None ? cu : plain(a[7])))
    Py_RETURN_NONE;
  if (!dense(o, at::kBFloat16, 3) || !dense(d_o, at::kBFloat16, 3) || !dense(lse, at::kFloat, 2) || o->sizes() != r.q->sizes() ||
      d_o->sizes() != r.q->sizes() || lse->size(0) != r.h || lse->size(1) != r.tq || !same_device(*r.q, {o, d_o, lse}))
    Py_RETURN_NONE;
  const int fill = a[10] == Py_None;
  Tensor grad[3], ws, delta;
  long long st[3][2];
  for (int i = 0; i < 3; ++i) {
    const Tensor& like = i ? *r.k : *r.q;
    if ((a[10 + i] == Py_None) != (fill != 0)) Py_RETURN_NONE;
    if (fill) {
      if (!output(Py_None, *r.q, like.sizes(), at::kBFloat16, grad[i])) Py_RETURN_NONE;
    } else {
      const Tensor* t = plain(a[10 + i]);
      if (!is(t, at::kBFloat16, 3) || t->sizes() != like.sizes() || t->device() != r.q->device()) Py_RETURN_NONE;
      grad[i] = *t;
    }
    if (!Ragged::strides(grad[i], st[i])) Py_RETURN_NONE;
  }
  const size_t need = hk_attn_bwd_ragged_workspace_bytes(r.s, r.tq, r.tk);
  if (!output(Py_None, *r.q, {int64_t(need)}, at::kByte, ws) || !output(Py_None, *r.q, lse->sizes(), at::kFloat, delta)) Py_RETURN_NONE;
  void* stream = stream_of(*r.q);
  const void *qp = ptr(*r.q), *kp = ptr(*r.k), *vp = ptr(*r.v), *op = ptr(*o), *dop = ptr(*d_o);
  const float* lp = ptr<float>(*lse);
  float* dp = ptr<float>(delta);
  void *gp[3] = {ptr(grad[0]), ptr(grad[1]), ptr(grad[2])}, *wsp = ptr(ws);
  const int32_t *cq = ptr<int32_t>(*r.cu_q), *ck = ptr<int32_t>(*r.cu_k);
  const int causal = a[8] == Py_True;
  const int rc = unlocked([&] {
    return hk_attn_bwd_ragged(qp, kp, vp, op, dop, lp, dp, gp[0], gp[1], gp[2], cq, ck, r.s, r.tq, r.tk, r.h, r.hkv, r.d, r.qs, r.ks, r.vs,
                              st[0], st[1], st[2], causal, scale, fill, wsp, need, r.device, stream);
  });
  if (rc != HK_OK) return PyLong_FromLong(rc);
  return Py_BuildValue("(NNN)", THPVariable_Wrap(grad[0]), THPVariable_Wrap(grad[1]), THPVariable_Wrap(grad[2]));
  END_HANDLE_TH_ERRORS
}

// ---- autograd. A step through the Python functions behind these spends about 55 us on them, in the caller's thread and in the
// engine's, which has to have the interpreter for its part; small steps are made of little else.

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// Thrown by a forward that the Python code behind is to look at: it makes the call again, and raises what there is to raise.
struct Refused {};

void fail(const char* what, int rc) {
  TORCH_CHECK(false, what, ": error ", rc, " (", hk_strerror(rc), ")");
}
// Waits for the device, as the Python functions do behind each direction.
void check_device(int device, const char* direction) {
  const int status = hk_last_device_status(device);
  TORCH_CHECK(status == HK_OK, "attention ", direction, " failed on the device (status ", status, ")");
}

// What a backward returns, of `arguments` of its call. Where a graph of the gradients is wanted they have none of their own, and whoever
// differentiates them again is told so.
variable_list without_a_second(variable_list grads, size_t arguments) {
  if (at::GradMode::is_enabled()) {
    for (Tensor& t : grads)
      if (t.defined()) t.requires_grad_();
    const int n = static_cast<int>(grads.size());
    grads = (*std::make_shared<torch::autograd::DelayedError>(
        "trying to differentiate twice a function that was marked with @once_differentiable", n))(std::move(grads));
  }
  grads.resize(arguments);
  return grads;
}

// The parts of a packed projection [B, S, 2 or 3, H, D], or of its gradient.
struct Parts {
  char* base;
  int64_t part;       // bytes between two of them
  long long st[3];    // element strides of batch, sequence and head
  bool good;          // as the kernels read and write them
  explicit Parts(const Tensor& t) : base(static_cast<char*>(t.data_ptr())), part(2 * t.stride(2)) {
    good = t.stride(4) == 1 && t.stride(2) % 8 == 0 && (reinterpret_cast<uintptr_t>(base) & 15) == 0;
    int i = 0;
    for (int dim : {0, 1, 3}) {
      st[i] = t.stride(dim);
      good = good && st[i] > 0 && st[i] % 8 == 0;
      ++i;
    }
  }
  void* at(int i) const { return base + i * part; }
};

// One call of the attention modules: q [B, Sq, H, D] with packed [B, Sk, 2, H_KV, D], or an undefined q and packed [B, S, 3, H, D].
struct Attention {
  bool causal;
  float scale;
  int window, sinks;
  Tensor lens;
  int b, n, nk, h, hkv, d, device;
  void shape(const Tensor& q, const Tensor& packed) {
    b = i32(packed.size(0)), nk = i32(packed.size(1)), hkv = i32(packed.size(3)), d = i32(packed.size(4));
    n = q.defined() ? i32(q.size(1)) : nk, h = q.defined() ? i32(q.size(2)) : hkv;
    device = packed.device().index();
  }
  const int32_t* lens_ptr() const { return lens.defined() ? ptr<int32_t>(lens) : nullptr; }
};

class PackedAttention : public torch::autograd::Function<PackedAttention> {
 public:
  static Tensor forward(AutogradContext* ctx, const std::optional<Tensor>& q_or_none, const Tensor& packed, const Attention& a) {
    const Tensor q = q_or_none.value_or(Tensor());
    const Tensor o = at::empty({a.b, a.n, a.h, a.d}, packed.options().requires_grad(false));
    const Tensor lse = at::empty({a.b, a.h, 1, a.n}, packed.options().dtype(at::kFloat).requires_grad(false));
    const Parts p(packed);
    long long qs[3] = {p.st[0], p.st[1], p.st[2]};
    const bool own_q = q.defined();
    if (!p.good || (own_q && !tma_strides(q, qs))) throw Refused();
    const void *qp = own_q ? ptr(q) : p.at(0), *kp = p.at(own_q ? 0 : 1), *vp = p.at(own_q ? 1 : 2);
    void *op = ptr(o), *stream = stream_of(packed);
    float* lp = ptr<float>(lse);
    const int32_t* lens = a.lens_ptr();
    int rc = HK_OK, status = HK_OK;
    unlocked([&] {
      rc = a.window ? hk_attn_fwd_window(qp, kp, vp, op, lp, a.b, a.n, a.nk, a.h, a.hkv, a.d, qs, p.st, p.st, lens, a.window, a.sinks,
                                         a.scale, a.device, stream)
                    : hk_attn_fwd_cross(qp, kp, vp, op, lp, a.b, a.n, a.nk, a.h, a.hkv, a.d, qs, p.st, p.st, lens, a.causal, a.scale,
                                        a.device, stream);
      if (rc == HK_OK) status = hk_last_device_status(a.device);
      return rc;
    });
    if (rc != HK_OK) throw Refused();
    TORCH_CHECK(status == HK_OK, "attention forward failed on the device (status ", status, ")");
    ctx->save_for_backward({q, packed, o, lse});
    ctx->saved_data["causal"] = a.causal;
    ctx->saved_data["scale"] = static_cast<double>(a.scale);
    ctx->saved_data["window"] = int64_t(a.window);
    ctx->saved_data["sinks"] = int64_t(a.sinks);
    if (a.lens.defined()) ctx->saved_data["lens"] = a.lens;
    return o;
  }

  // In a thread of the engine, without the interpreter.
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    // saved-tensor hooks may have given them back in a layout that the kernels do not read
    Tensor q = saved[0], packed = saved[1];
    const Tensor o = saved[2].contiguous(), lse = saved[3].contiguous();
    TORCH_CHECK(grads[0].defined() && grads[0].sizes() == o.sizes(), "dO shape mismatch: expected ", o.sizes());
    TORCH_CHECK(grads[0].device() == o.device(), "dO must be on correct CUDA device");
    const Tensor d_o = grads[0].to(at::kBFloat16).contiguous();
    if (!Parts(packed).good) packed = packed.contiguous();
    const Parts p(packed);
    long long qs[3] = {p.st[0], p.st[1], p.st[2]};
    if (q.defined() && !tma_strides(q, qs)) {
      q = q.contiguous();
      tma_strides(q, qs);
    }
    Attention a;
    a.shape(q, packed);
    a.causal = ctx->saved_data["causal"].toBool();
    a.scale = static_cast<float>(ctx->saved_data["scale"].toDouble());
    a.window = i32(ctx->saved_data["window"].toInt()), a.sinks = i32(ctx->saved_data["sinks"].toInt());
    if (const auto it = ctx->saved_data.find("lens"); it != ctx->saved_data.end()) a.lens = it->second.toTensor();
    const Tensor d_packed = at::empty(packed.sizes(), packed.options().requires_grad(false));
    const Tensor dq = q.defined() ? at::empty(q.sizes(), q.options().requires_grad(false)) : Tensor();
    const Tensor delta = at::empty(lse.sizes(), lse.options().requires_grad(false));
    const Parts dp(d_packed);
    const size_t need = a.window ? hk_attn_bwd_window_workspace_bytes(a.b, a.n, a.nk, a.h, a.hkv, a.d, a.window, a.sinks) : 0;
    const Tensor ws = need ? at::empty({int64_t(need)}, packed.options().dtype(at::kByte).requires_grad(false)) : Tensor();
    const bool own_q = q.defined();
    long long dqs[3] = {dp.st[0], dp.st[1], dp.st[2]};
    if (own_q) tma_strides(dq, dqs);
    const void *qp = own_q ? ptr(q) : p.at(0), *kp = p.at(own_q ? 0 : 1), *vp = p.at(own_q ? 1 : 2);
    void *dqp = own_q ? ptr(dq) : dp.at(0), *dkp = dp.at(own_q ? 0 : 1), *dvp = dp.at(own_q ? 1 : 2);
    void *stream = stream_of(packed), *wsp = need ? ptr(ws) : nullptr;
    const int rc =
        a.window ? hk_attn_bwd_window(qp, kp, vp, ptr(o), ptr(d_o), ptr<float>(lse), ptr<float>(delta), dqp, dkp, dvp, a.b, a.n, a.nk,
                                      a.h, a.hkv, a.d, qs, p.st, p.st, dqs, dp.st, dp.st, a.lens_ptr(), a.window, a.sinks, a.scale,
                                      wsp, need, a.device, stream)
                 : hk_attn_bwd_strided(qp, kp, vp, ptr(o), ptr(d_o), ptr<float>(lse), ptr<float>(delta), dqp, dkp, dvp, a.b, a.n, a.nk,
                                       a.h, a.hkv, a.d, qs, p.st, p.st, dqs, dp.st, dp.st, a.lens_ptr(), a.causal, a.scale, a.device,
                                       stream);
    if (rc != HK_OK) fail("hk_attn_bwd_strided", rc);
    check_device(a.device, "backward");
    return without_a_second({dq, d_packed}, 3);
  }
};

// packed_attention(q or None, packed, causal, softmax_scale, kv_lens, window or None, sinks): O, or None
PyObject* packed_attention(PyObject*, PyObject* const* arg, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  Attention a;
  if (n_args != 7 || !PyBool_Check(arg[2]) || !number(arg[3], a.scale)) Py_RETURN_NONE;
  a.window = a.sinks = 0;
  if (arg[5] != Py_None && !window_args(arg, n_args, 5, a.window, a.sinks)) Py_RETURN_NONE;
  a.causal = arg[2] == Py_True;
  if (a.window && !a.causal) Py_RETURN_NONE;
  const Tensor *q = nullptr, *packed = plain(arg[1]);
  if (!is(packed, at::kBFloat16, 5) || packed->size(2) != (arg[0] == Py_None ? 3 : 2)) Py_RETURN_NONE;
  for (int64_t v : packed->sizes())
    if (v == 0 || !fits({v})) Py_RETURN_NONE;
  if (arg[0] != Py_None) {
    q = plain(arg[0]);
    if (!is(q, at::kBFloat16, 4) || q->size(0) != packed->size(0) || q->size(3) != packed->size(4) ||
        q->size(2) % packed->size(3) != 0 || q->device() != packed->device() || q->numel() == 0 || !fits({q->size(1), q->size(2)}))
      Py_RETURN_NONE;
  }
  if (arg[4] != Py_None) {
    const Tensor* lens = plain(arg[4]);
    if (!dense(lens, at::kInt, 1) || lens->size(0) != packed->size(0) || lens->device() != packed->device()) Py_RETURN_NONE;
    a.lens = *lens;
  }
  const Tensor none;
  a.shape(q ? *q : none, *packed);
  try {
    return THPVariable_Wrap(PackedAttention::apply(q ? std::optional<Tensor>(*q) : std::nullopt, *packed, a));
  } catch (const Refused&) {
    Py_RETURN_NONE;
  }
  END_HANDLE_TH_ERRORS
}

// The capture that a stream is part of, 0 for none.
unsigned long long capture_of(cudaStream_t stream) {
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  unsigned long long id = 0;
  if (cudaStreamGetCaptureInfo(stream, &status, &id) == cudaSuccess) return status == cudaStreamCaptureStatusNone ? 0 : id;
  (void)cudaGetLastError();  // the legacy stream, while another one is captured that waits for it
  return 0;
}
// A gradient goes to the stream on which its tensor's node was made, and the engine makes that stream wait for the one of this backward.
// Where this backward is captured and that stream is not, as with a leaf that a graph from before the capture holds as well, the wait
// takes it into the capture. The legacy stream cannot be, nor one of another capture: the wait ends the capture and may end the process.
void check_next_streams(cudaStream_t stream) {
  const unsigned long long capture = capture_of(stream);
  if (!capture) return;
  const auto node = torch::autograd::get_current_node();
  if (!node) return;
  for (size_t i = 0; i < node->num_outputs(); ++i) {
    const auto& next = node->next_edge(i).function;
    const auto to = next && node->task_should_compute_output(i) ? next->stream() : std::nullopt;
    if (!to) continue;
    const cudaStream_t other = c10::cuda::CUDAStream(*to).stream();
    const bool legacy = other == nullptr || other == cudaStreamLegacy;
    const unsigned long long others = legacy ? 0 : capture_of(other);
    TORCH_CHECK(!legacy && (others == 0 || others == capture), "a captured backward needs tensors that no graph from before",
                " the capture holds on the default stream: delete that graph first, or capture with tensors of their own");
  }
}

// One call of the norm and rotation, as its gradients need it.
struct QknCall {
  long long qs[3], ks[3];
  int flags, pos_offset, b, n, h, hkv, d, r, rows, device;
  float eps;
};

class NormRotary : public torch::autograd::Function<NormRotary> {
 public:
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const std::optional<Tensor>& q_weight,
                               const std::optional<Tensor>& k_weight, const Tensor& cos, const Tensor& sin,
                               const std::optional<Tensor>& positions_or_none, const QknCall& c) {
    const Tensor none, wq = q_weight.value_or(none), wk = k_weight.value_or(none), positions = positions_or_none.value_or(none);
    const Tensor qo = at::empty(q.sizes(), q.options().requires_grad(false).memory_format(at::MemoryFormat::Contiguous));
    const Tensor ko = at::empty(k.sizes(), k.options().requires_grad(false).memory_format(at::MemoryFormat::Contiguous));
    const void *qp = ptr(q), *kp = ptr(k), *wqp = wq.defined() ? ptr(wq) : nullptr, *wkp = wk.defined() ? ptr(wk) : nullptr,
               *cp = ptr(cos), *sp = ptr(sin);
    const int32_t* pp = positions.defined() ? ptr<int32_t>(positions) : nullptr;
    void *qop = ptr(qo), *kop = ptr(ko), *stream = stream_of(q);
    const int rc = unlocked([&] {
      return hk_qk_norm_rotary(qp, kp, wqp, wkp, cp, sp, qop, kop, c.b, c.n, c.h, c.hkv, c.d, c.r, c.rows, c.qs, c.ks, pp,
                               c.pos_offset, c.eps, c.flags, c.device, stream);
    });
    if (rc != HK_OK) throw Refused();
    ctx->save_for_backward({q, k, wq, wk, cos, sin, positions});
    ctx->saved_data["flags"] = int64_t(c.flags);
    ctx->saved_data["offset"] = int64_t(c.pos_offset);
    ctx->saved_data["eps"] = static_cast<double>(c.eps);
    return {qo, ko};
  }

  // In a thread of the engine, without the interpreter.
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list s = ctx->get_saved_variables();
    check_next_streams(static_cast<cudaStream_t>(stream_of(s[0])));
    QknCall c;
    long long* const st[2] = {c.qs, c.ks};
    Tensor dy[2], dx[2], dw[2];
    bool weights = false;  // the tensors of the call are numbered without those that it does not have
    for (size_t i = 2, end = 2 + s[2].defined() + s[3].defined(); i < end; ++i) weights |= ctx->needs_input_grad(i);
    for (int i = 0; i < 2; ++i) {
      if (!tma_strides(s[i], st[i])) {  // saved-tensor hooks may have given it back in another layout
        s[i] = s[i].contiguous();
        tma_strides(s[i], st[i]);
      }
      dy[i] = grads[i].defined() ? grads[i].to(at::kBFloat16).contiguous()
                                 : at::zeros(s[i].sizes(), s[i].options().requires_grad(false));
      dx[i] = at::empty(s[i].sizes(), s[i].options().requires_grad(false).memory_format(at::MemoryFormat::Contiguous));
      if (weights && s[2 + i].defined()) {
        s[2 + i] = s[2 + i].contiguous();
        dw[i] = at::empty(s[2 + i].sizes(), s[2 + i].options().requires_grad(false));
      }
    }
    for (int i = 2; i < 7; ++i)
      if (s[i].defined()) s[i] = s[i].contiguous();
    const size_t need = dw[0].defined() || dw[1].defined() ? hk_qk_norm_rotary_bwd_workspace_bytes(i32(s[0].size(3))) : 0;
    const Tensor ws = need ? at::empty({int64_t(need)}, s[0].options().dtype(at::kByte).requires_grad(false)) : Tensor();
    auto opt = [](const Tensor& t) { return t.defined() ? ptr(t) : nullptr; };
    const int rc = hk_qk_norm_rotary_bwd(
        ptr(s[0]), ptr(s[1]), opt(s[2]), opt(s[3]), ptr(s[4]), ptr(s[5]), ptr(dy[0]), ptr(dy[1]), ptr(dx[0]), ptr(dx[1]), opt(dw[0]),
        opt(dw[1]), i32(s[0].size(0)), i32(s[0].size(1)), i32(s[0].size(2)), i32(s[1].size(2)), i32(s[0].size(3)),
        i32(2 * s[4].size(1)), i32(s[4].size(0)), c.qs, c.ks, static_cast<const int32_t*>(opt(s[6])),
        i32(ctx->saved_data["offset"].toInt()), static_cast<float>(ctx->saved_data["eps"].toDouble()),
        i32(ctx->saved_data["flags"].toInt()), opt(ws), need, s[0].device().index(), stream_of(s[0]));
    if (rc != HK_OK) fail("hk_qk_norm_rotary_bwd", rc);
    return without_a_second({dx[0], dx[1], dw[0], dw[1]}, 8);
  }
};

// norm_rotary(q, k, q_weight, k_weight, cos, sin, positions, pos_offset, eps, interleaved): q and k with their gradients, or None
PyObject* norm_rotary(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  Qkn p;
  if (n_args != 10 || !p.take(a, a[6], a[7], a[8], a[9]) || p.cos->requires_grad() || p.sin->requires_grad()) Py_RETURN_NONE;
  QknCall c;
  for (int i = 0; i < 3; ++i) c.qs[i] = p.qs[i], c.ks[i] = p.ks[i];
  c.flags = p.flags, c.pos_offset = p.pos_offset, c.eps = p.eps;
  c.b = p.b, c.n = p.n, c.h = p.h, c.hkv = p.hkv, c.d = p.d, c.r = p.r, c.rows = p.rows, c.device = p.device;
  auto given = [](const Tensor* t) { return t ? std::optional<Tensor>(*t) : std::nullopt; };
  try {
    const variable_list y =
        NormRotary::apply(*p.q, *p.k, given(p.w[0]), given(p.w[1]), *p.cos, *p.sin, given(p.positions), c);
    return Py_BuildValue("(NN)", THPVariable_Wrap(y[0]), THPVariable_Wrap(y[1]));
  } catch (const Refused&) {
    Py_RETURN_NONE;
  }
  END_HANDLE_TH_ERRORS
}

// Attention over a ragged batch, q [T, H, D] with a packed kv [Tk, 2, H_KV, D].
class RaggedAttention : public torch::autograd::Function<RaggedAttention> {
 public:
  // K and V of a packed projection, or of its gradient: [Tk, H_KV, D] each
  static Tensor part(const Tensor& kv, int i) { return kv.select(1, i); }

  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& kv, const Tensor& cu_q, const std::optional<Tensor>& cu_k_or_none,
                        bool causal, double scale) {
    const Tensor cu_k = cu_k_or_none.value_or(cu_q), k = part(kv, 0), v = part(kv, 1);
    Ragged r;
    if (!r.take(&q, &k, &v, &cu_q, cu_k_or_none ? &cu_k : &cu_q)) throw Refused();
    const auto options = q.options().requires_grad(false);
    const Tensor o = at::empty(q.sizes(), options.memory_format(at::MemoryFormat::Contiguous));
    const Tensor lse = at::empty({r.h, r.tq}, options.dtype(at::kFloat));
    const size_t need = hk_attn_fwd_ragged_workspace_bytes(r.s, r.tq);
    const Tensor ws = at::empty({int64_t(need)}, options.dtype(at::kByte));
    const void *qp = ptr(q), *kp = ptr(k), *vp = ptr(v);
    void *op = ptr(o), *wsp = ptr(ws), *stream = stream_of(q);
    float* lp = ptr<float>(lse);
    const int32_t *cq = ptr<int32_t>(cu_q), *ck = ptr<int32_t>(cu_k);
    const int rc = unlocked([&] {
      return hk_attn_fwd_ragged(qp, kp, vp, op, lp, cq, ck, r.s, r.tq, r.tk, r.h, r.hkv, r.d, r.qs, r.ks, r.vs, causal,
                                static_cast<float>(scale), 1, wsp, need, r.device, stream);
    });
    if (rc != HK_OK) throw Refused();
    ctx->save_for_backward({q, kv, o, lse, cu_q, cu_k_or_none.value_or(Tensor())});
    ctx->saved_data["causal"] = causal;
    ctx->saved_data["scale"] = scale;
    return o;
  }

  // In a thread of the engine, without the interpreter.
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list s = ctx->get_saved_variables();
    check_next_streams(static_cast<cudaStream_t>(stream_of(s[0])));
    // saved-tensor hooks may have given them back in a layout that the kernels do not read
    Tensor q = s[0], kv = s[1];
    const Tensor o = s[2].contiguous(), lse = s[3].contiguous(), cu_q = s[4].contiguous(),
                 cu_k = s[5].defined() ? s[5].contiguous() : cu_q;
    TORCH_CHECK(grads[0].defined() && grads[0].sizes() == o.sizes(), "dO shape mismatch: expected ", o.sizes());
    TORCH_CHECK(grads[0].device() == o.device(), "dO must be on correct CUDA device");
    const Tensor d_o = grads[0].to(at::kBFloat16).contiguous();
    long long st[2];
    if (!Ragged::strides(q, st)) q = q.contiguous();
    if (!Ragged::strides(part(kv, 0), st) || kv.stride(1) % 8 != 0) kv = kv.contiguous();
    const Tensor k = part(kv, 0), v = part(kv, 1);
    Ragged r;
    TORCH_CHECK(r.take(&q, &k, &v, &cu_q, s[5].defined() ? &cu_k : &cu_q), "ragged attention: saved tensors of another shape");
    const auto options = q.options().requires_grad(false);
    const Tensor dq = at::empty(q.sizes(), options.memory_format(at::MemoryFormat::Contiguous));
    const Tensor dkv = at::empty(kv.sizes(), options.memory_format(at::MemoryFormat::Contiguous));
    const Tensor delta = at::empty(lse.sizes(), options.dtype(at::kFloat));
    const size_t need = hk_attn_bwd_ragged_workspace_bytes(r.s, r.tq, r.tk);
    const Tensor ws = at::empty({int64_t(need)}, options.dtype(at::kByte));
    const Tensor dk = part(dkv, 0), dv = part(dkv, 1);
    const long long dqs[2] = {dq.stride(0), dq.stride(1)}, dks[2] = {dk.stride(0), dk.stride(1)};
    const int rc = hk_attn_bwd_ragged(ptr(q), ptr(k), ptr(v), ptr(o), ptr(d_o), ptr<float>(lse), ptr<float>(delta), ptr(dq), ptr(dk), ptr(dv),
                                      ptr<int32_t>(cu_q), ptr<int32_t>(cu_k), r.s, r.tq, r.tk, r.h, r.hkv, r.d, r.qs, r.ks, r.vs, dqs, dks,
                                      dks, ctx->saved_data["causal"].toBool(), static_cast<float>(ctx->saved_data["scale"].toDouble()), 1,
                                      ptr(ws), need, r.device, stream_of(q));
    if (rc != HK_OK) fail("hk_attn_bwd_ragged", rc);
    return without_a_second({dq, dkv}, 6);
  }
};

// ragged_attention(q, kv, cu_seqlens_q, cu_seqlens_k or None, causal, softmax_scale): O, or None
PyObject* ragged_attention(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  float scale;
  if (n_args != 6 || !PyBool_Check(a[4]) || !number(a[5], scale)) Py_RETURN_NONE;
  const Tensor *q = plain(a[0]), *kv = plain(a[1]), *cu_q = plain(a[2]), *cu_k = a[3] == Py_None ? nullptr : plain(a[3]);
  if (!is(q, at::kBFloat16, 3) || !is(kv, at::kBFloat16, 4) || kv->size(1) != 2 || !dense(cu_q, at::kInt, 1) ||
      (a[3] != Py_None && !dense(cu_k, at::kInt, 1)) || !q->numel() || !kv->numel())
    Py_RETURN_NONE;
  try {
    return THPVariable_Wrap(RaggedAttention::apply(*q, *kv, *cu_q, cu_k ? std::optional<Tensor>(*cu_k) : std::nullopt, a[4] == Py_True,
                                                   static_cast<double>(scale)));
  } catch (const Refused&) {
    Py_RETURN_NONE;
  }
  END_HANDLE_TH_ERRORS
}

// captured_backward(tensor): raises what the backward of `norm_rotary` does, for a Python function whose backward is running on the
// tensor's device
PyObject* captured_backward(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  const Tensor* t = n_args == 1 ? plain(a[0]) : nullptr;
  if (t) check_next_streams(static_cast<cudaStream_t>(stream_of(*t)));
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

#define HK_METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {HK_METHOD(attn_fwd),       HK_METHOD(attn_bwd_strided), HK_METHOD(rotary_bnhd),
                         HK_METHOD(paged_decode),   HK_METHOD(attn_fwd_paged),   HK_METHOD(paged_kv_append),
                         HK_METHOD(qk_norm_rotary), HK_METHOD(qk_norm_rotary_bwd),
                         HK_METHOD(paged_kv_append_fp8), HK_METHOD(paged_kv_read_fp8), HK_METHOD(paged_decode_fp8),
                         HK_METHOD(attn_fwd_ragged), HK_METHOD(attn_bwd_ragged), HK_METHOD(ragged_attention),
                         HK_METHOD(packed_attention), HK_METHOD(norm_rotary), HK_METHOD(captured_backward),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch_front", "Native tensor front ends of hipkittens_b200", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

// Looked for in the built file, before it is loaded, by whoever wants to know which torch it was compiled against.
extern "C" __attribute__((used, visibility("default"))) const char hk_torch_front_built_for[] =
    "built for torch " HK_TORCH_VERSION;

PyMODINIT_FUNC PyInit__torch_front(void) { return PyModule_Create(&module); }
