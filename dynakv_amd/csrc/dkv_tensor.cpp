// The serving operators' calls on torch tensors: module _dkv_tensor.
//
// A step of single tokens makes two calls a layer whose kernels take 4 to 6 us, and a call's checks of
// its tensors, one attribute at a time from Python, take 5 us more than its launch. Here a call that is
// as it should be and ordinary is checked, its output made and its entry point called; any other call
// (an argument to refuse, an output to write to, a copy to align) returns None, and the
// Python function, which has every check and its message, does it.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/version.h>

#include <climits>

#include "../../include/dynakv_amd.h"

namespace {

constexpr long long HEAD_DIM = 128;

const at::Tensor* tensor(PyObject* o) {
  return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr;
}

bool aligned16(const at::Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }

bool int32_on(const at::Tensor& t, c10::Device d) {
  return t.scalar_type() == at::kInt && t.device() == d && t.layout() == at::kStrided;
}

// None, or the C types of a call's integers.
bool ints(PyObject* const* args, Py_ssize_t n, long long* v) {
  for (Py_ssize_t i = 0; i < n; ++i) {
    v[i] = PyLong_AsLongLong(args[i]);
    if (v[i] == -1 && PyErr_Occurred()) {
      PyErr_Clear();
      return false;
    }
  }
  return true;
}

// What PagedBatch holds for the calls: table pointer, row stride, columns, row starts, lengths,
// requests, rows, max_new, min_new, max_len, device.
struct Batch {
  long long v[11];
  bool read(PyObject* t) {
    return PyTuple_Check(t) && PyTuple_GET_SIZE(t) == 11 &&
           ints(&PyTuple_GET_ITEM(t, 0), 11, v);
  }
  const int* table() const { return reinterpret_cast<const int*>(v[0]); }
  const int* starts() const { return reinterpret_cast<const int*>(v[3]); }
  const int* lens() const { return reinterpret_cast<const int*>(v[4]); }
  long long ld() const { return v[1]; }
  int cols() const { return (int)v[2]; }
  int requests() const { return (int)v[5]; }
  int rows() const { return (int)v[6]; }
  int max_new() const { return (int)v[7]; }
  int min_new() const { return (int)v[8]; }
  int max_len() const { return (int)v[9]; }
};

// Pages alike, of type dt on device d.
bool pages(const at::Tensor& k, const at::Tensor& v, at::ScalarType dt, c10::Device d) {
  if (k.dim() != 4 || v.dim() != 4 || k.sizes() != v.sizes() || k.strides() != v.strides())
    return false;
  if (k.scalar_type() != dt || v.scalar_type() != dt || !d.is_cuda() || k.device() != d ||
      v.device() != d)
    return false;
  const long long ps = k.size(2);
  return k.size(3) == HEAD_DIM && k.stride(3) == 1 && k.stride(2) == HEAD_DIM && ps >= 16 &&
         (ps & (ps - 1)) == 0 && k.size(0) <= INT_MAX && ps <= INT_MAX && k.size(1) > 0 &&
         k.size(1) <= 65536;
}

// The scales of 8-bit pages, alike: (pages, heads, page_size / 16).
bool scales(const at::Tensor& ks, const at::Tensor& vs, const at::Tensor& k) {
  return ks.dim() == 3 && vs.dim() == 3 && ks.sizes() == vs.sizes() && ks.strides() == vs.strides() &&
         ks.scalar_type() == at::kFloat8_e8m0fnu && vs.scalar_type() == at::kFloat8_e8m0fnu &&
         ks.device() == k.device() && vs.device() == k.device() && ks.size(0) == k.size(0) &&
         ks.size(1) == k.size(1) && ks.size(2) == k.size(2) / 16 &&
         (ks.size(2) == 1 || ks.stride(2) == 1);
}

// Pools of a call on x, whose device is the batch's: pages of x's type, or with their scales (else None,
// null here) of 8 bits.
struct Pools {
  const at::Tensor *k, *v, *ks, *vs;
  bool read(PyObject* k_pages, PyObject* v_pages, PyObject* k_scale, PyObject* v_scale,
            const at::Tensor& x, const Batch& b) {
    k = tensor(k_pages), v = tensor(v_pages), ks = vs = nullptr;
    const auto dt = x.scalar_type();
    if (!k || !v || (dt != at::kBFloat16 && dt != at::kHalf) || !x.is_cuda() ||
        x.get_device() != b.v[10])
      return false;
    if (k_scale != Py_None || v_scale != Py_None) {
      ks = tensor(k_scale), vs = tensor(v_scale);
      if (!ks || !vs) return false;
    }
    return pages(*k, *v, ks ? at::kFloat8_e4m3fn : dt, x.device()) &&
           (!ks || scales(*ks, *vs, *k)) && b.max_len() <= b.cols() * k->size(2);
  }
};

int code(const at::Tensor& t) { return t.scalar_type() == at::kBFloat16 ? DKV_BF16 : DKV_F16; }

// (page_table, q_start, lens, rows, max_new, max_len, min_new) -> the tuple above
PyObject* paged_batch(PyObject*, PyObject* const* args, Py_ssize_t n) {
  long long v[4];
  if (n != 7 || !ints(args + 3, 4, v)) Py_RETURN_NONE;
  const at::Tensor *t = tensor(args[0]), *s = tensor(args[1]), *l = tensor(args[2]);
  if (!t || !s || !l || t->dim() != 2 || s->dim() != 1 || l->dim() != 1) Py_RETURN_NONE;
  const long long B = t->size(0), cols = t->size(1), ld = t->stride(0);
  const c10::Device d = t->device();
  if (l->size(0) != B || s->size(0) != B + 1 || !int32_on(*t, d) || !int32_on(*s, d) ||
      !int32_on(*l, d) || !s->is_contiguous() || !l->is_contiguous() ||
      (cols > 1 && t->stride(1) != 1) || (B > 1 && ld < cols))
    Py_RETURN_NONE;
  if (!(0 <= v[3] && v[3] <= v[1] && v[1] <= v[0] && v[0] <= INT_MAX && 0 <= v[2] &&
        v[2] <= INT_MAX))
    Py_RETURN_NONE;
  return Py_BuildValue("(NLLNNLLLLLi)", PyLong_FromVoidPtr(t->data_ptr()), ld > cols ? ld : cols, cols,
                       PyLong_FromVoidPtr(s->data_ptr()), PyLong_FromVoidPtr(l->data_ptr()), B, v[0],
                       v[1], v[3], v[2], d.is_cuda() ? (int)t->get_device() : -1);
}

// (stream, qkv, k_pages, v_pages, batch, heads, frequencies, q_norm, k_norm, eps, k_scale, v_scale)
PyObject* paged_append(PyObject*, PyObject* const* args, Py_ssize_t n) {
  Batch b;
  long long heads, freq;
  if (n != 12 || !b.read(args[4]) || !ints(args + 5, 1, &heads) || !ints(args + 6, 1, &freq))
    Py_RETURN_NONE;
  const at::Tensor* x = tensor(args[1]);
  const double eps = PyFloat_Check(args[9]) ? PyFloat_AS_DOUBLE(args[9]) : -1.0;
  Pools pool;
  if (!x || x->dim() != 2 || !(eps >= 0.0) || heads <= 0 ||
      !pool.read(args[2], args[3], args[10], args[11], *x, b))
    Py_RETURN_NONE;
  const at::Tensor *k = pool.k, *v = pool.v;
  const long long T = x->size(0), hkv = k->size(1), ld = x->stride(0);
  if (x->stride(1) != 1 || heads > 65536 || x->size(1) < (heads + 2 * hkv) * HEAD_DIM ||
      ld < x->size(1) || b.rows() > T || !aligned16(*x))
    Py_RETURN_NONE;
  const void* norm[2];
  for (int i = 0; i < 2; ++i) {
    norm[i] = nullptr;
    if (args[7 + i] == Py_None) continue;
    const at::Tensor* w = tensor(args[7 + i]);
    if (!w || w->dim() != 1 || w->size(0) != HEAD_DIM || w->stride(0) != 1 ||
        w->scalar_type() != x->scalar_type() || w->device() != x->device())
      Py_RETURN_NONE;
    norm[i] = w->data_ptr();
  }
  at::Tensor out = at::empty({T, heads, HEAD_DIM}, x->options());
  int rc;
  void* const stream = PyLong_AsVoidPtr(args[0]);
  Py_BEGIN_ALLOW_THREADS;
  if (pool.ks)
    rc = dkv_paged_append8(
        stream, code(*x), x->data_ptr(), ld, out.data_ptr(), heads * HEAD_DIM, HEAD_DIM,
        k->data_ptr(), v->data_ptr(), k->stride(0), k->stride(1), (int)k->size(0), (int)k->size(2),
        pool.ks->data_ptr(), pool.vs->data_ptr(), pool.ks->stride(0), pool.ks->stride(1), b.table(),
        b.ld(), b.cols(), b.starts(), b.lens(), b.requests(), b.rows(), (int)heads, (int)hkv,
        (int)HEAD_DIM, norm[0], norm[1], (float)eps, reinterpret_cast<const double*>(freq));
  else
    rc = dkv_paged_append(
        stream, code(*x), x->data_ptr(), ld, out.data_ptr(), heads * HEAD_DIM, HEAD_DIM,
        k->data_ptr(), v->data_ptr(), k->stride(0), k->stride(1), (int)k->size(0), (int)k->size(2),
        b.table(), b.ld(), b.cols(), b.starts(), b.lens(), b.requests(), b.rows(), (int)heads,
        (int)hkv, (int)HEAD_DIM, norm[0], norm[1], (float)eps, reinterpret_cast<const double*>(freq));
  Py_END_ALLOW_THREADS;
  if (rc != DKV_OK) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(out));
}

// (stream, q, k_pages, v_pages, batch, scale, workspace, k_scale, v_scale): workspace(q, stream, floats)
// gives a tensor
PyObject* paged_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  Batch b;
  if (n != 9 || !b.read(args[4]) || !PyFloat_Check(args[5])) Py_RETURN_NONE;
  const at::Tensor* q = tensor(args[1]);
  Pools pool;
  if (!q || q->dim() != 3 || q->size(2) != HEAD_DIM ||
      !pool.read(args[2], args[3], args[7], args[8], *q, b))
    Py_RETURN_NONE;
  const at::Tensor *k = pool.k, *v = pool.v;
  const long long T = q->size(0), hq = q->size(1), hkv = k->size(1);
  const long long st = q->stride(0), sh = q->stride(1);
  if (hq <= 0 || hq > 65536 || hq % hkv || q->stride(2) != 1 || (st & 7) || (sh & 7) ||
      b.rows() > T || !aligned16(*q))
    Py_RETURN_NONE;
  at::Tensor out = at::empty({T, hq, HEAD_DIM}, q->options());
  const long long need =
      dkv_paged_workspace_floats_of(pool.ks ? 8 : 16, b.requests(), b.rows(), (int)hq, (int)hkv,
                                    b.max_new(), b.min_new(), b.max_len());
  float* ws = nullptr;
  long long ws_floats = 0;
  PyObject* held = nullptr;  // until the launch
  if (need > 0) {
    PyObject* floats = PyLong_FromLongLong(need);
    held = floats ? PyObject_CallFunctionObjArgs(args[6], args[1], args[0], floats, nullptr) : nullptr;
    Py_XDECREF(floats);
    const at::Tensor* t = held ? tensor(held) : nullptr;
    if (!t) {
      Py_XDECREF(held);
      PyErr_Clear();
      Py_RETURN_NONE;
    }
    ws = static_cast<float*>(t->data_ptr());
    ws_floats = t->numel();
  }
  int rc;
  const float scale = (float)PyFloat_AS_DOUBLE(args[5]);
  void* const stream = PyLong_AsVoidPtr(args[0]);
  Py_BEGIN_ALLOW_THREADS;
  if (pool.ks)
    rc = dkv_paged_attention8(
        stream, code(*q), q->data_ptr(), st, sh, k->data_ptr(), v->data_ptr(), k->stride(0),
        k->stride(1), (int)k->size(0), (int)k->size(2), pool.ks->data_ptr(), pool.vs->data_ptr(),
        pool.ks->stride(0), pool.ks->stride(1), b.table(), b.ld(), b.cols(), b.starts(), b.lens(),
        b.requests(), b.rows(), (int)hq, (int)hkv, (int)HEAD_DIM, b.max_new(), b.min_new(),
        b.max_len(), scale, ws, ws_floats, out.data_ptr(), code(*q), hq * HEAD_DIM, HEAD_DIM);
  else
    rc = dkv_paged_attention(
        stream, code(*q), q->data_ptr(), st, sh, k->data_ptr(), v->data_ptr(), k->stride(0),
        k->stride(1), (int)k->size(0), (int)k->size(2), b.table(), b.ld(), b.cols(), b.starts(),
        b.lens(), b.requests(), b.rows(), (int)hq, (int)hkv, (int)HEAD_DIM, b.max_new(), b.min_new(),
        b.max_len(), scale, ws, ws_floats, out.data_ptr(), code(*q), hq * HEAD_DIM, HEAD_DIM);
  Py_END_ALLOW_THREADS;
  Py_XDECREF(held);
  if (rc != DKV_OK) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(out));
}

// (stream, k_pages, v_pages, k_scale, v_scale, page ids, dtype code) -> (k, v)
PyObject* paged_values(PyObject*, PyObject* const* args, Py_ssize_t n) {
  long long dt;
  if (n != 7 || !ints(args + 6, 1, &dt)) Py_RETURN_NONE;
  const at::Tensor *k = tensor(args[1]), *v = tensor(args[2]), *ks = tensor(args[3]),
                   *vs = tensor(args[4]), *ids = nullptr;
  if (!k || !v || !ks || !vs || !pages(*k, *v, at::kFloat8_e4m3fn, k->device()) ||
      !scales(*ks, *vs, *k))
    Py_RETURN_NONE;
  long long count = k->size(0);
  if (args[5] != Py_None) {
    ids = tensor(args[5]);
    if (!ids || ids->dim() != 1 || !int32_on(*ids, k->device()) || !ids->is_contiguous() ||
        ids->size(0) > INT_MAX)
      Py_RETURN_NONE;
    count = ids->size(0);
  }
  const auto type = dt == DKV_BF16 ? at::kBFloat16 : dt == DKV_F16 ? at::kHalf : at::kFloat;
  at::Tensor out[2];
  for (at::Tensor& t : out)
    t = at::empty({count, k->size(1), k->size(2), HEAD_DIM}, k->options().dtype(type));
  int rc;
  void* const stream = PyLong_AsVoidPtr(args[0]);
  Py_BEGIN_ALLOW_THREADS;
  rc = dkv_paged_values(stream, (int)dt, k->data_ptr(), v->data_ptr(), k->stride(0), k->stride(1),
                        (int)k->size(0), (int)k->size(2), (int)k->size(1), (int)HEAD_DIM,
                        ks->data_ptr(), vs->data_ptr(), ks->stride(0), ks->stride(1),
                        ids ? static_cast<const int*>(ids->data_ptr()) : nullptr, (int)count,
                        out[0].data_ptr(), out[1].data_ptr());
  Py_END_ALLOW_THREADS;
  if (rc != DKV_OK) Py_RETURN_NONE;
  PyObject *a = THPVariable_Wrap(std::move(out[0])), *b = THPVariable_Wrap(std::move(out[1]));
  PyObject* both = a && b ? PyTuple_Pack(2, a, b) : nullptr;
  Py_XDECREF(a);
  Py_XDECREF(b);
  return both;
}

// A setting of the sampling: a contiguous tensor with an entry per row, or a number for all rows.
bool setting(PyObject* o, const at::Tensor& u, at::ScalarType type, const void*& rows, double& all) {
  rows = nullptr;
  all = 0.0;
  if (PyFloat_Check(o)) {
    all = PyFloat_AS_DOUBLE(o);
    return type == at::kFloat;
  }
  if (PyLong_Check(o)) {
    long long x;
    if (!ints(&o, 1, &x) || x < INT_MIN || x > INT_MAX) return false;
    all = (double)x;
    return true;
  }
  const at::Tensor* t = tensor(o);
  if (!t || t->dim() != 1 || t->size(0) != u.size(0) || t->scalar_type() != type ||
      !t->is_contiguous() || t->device() != u.device())
    return false;
  rows = t->data_ptr();
  return true;
}

// (stream, device, logits, u, temperature, top_k, top_p, min_p)
PyObject* sample_tokens(PyObject*, PyObject* const* args, Py_ssize_t n) {
  long long dev;
  if (n != 8 || !ints(args + 1, 1, &dev)) Py_RETURN_NONE;
  const at::Tensor *x = tensor(args[2]), *u = tensor(args[3]);
  if (!x || !u || x->dim() != 2 || u->dim() != 1 || !x->is_cuda() || x->get_device() != dev ||
      u->device() != x->device() || u->scalar_type() != at::kFloat || !u->is_contiguous())
    Py_RETURN_NONE;
  const long long rows = x->size(0), V = x->size(1);
  const auto dt = x->scalar_type();
  if (rows != u->size(0) || rows > INT_MAX || V < 1 || V > (1 << 19) || (V > 1 && x->stride(1) != 1) ||
      (dt != at::kBFloat16 && dt != at::kHalf && dt != at::kFloat))
    Py_RETURN_NONE;
  const void* by_row[4];
  double all[4];
  for (int i = 0; i < 4; ++i)
    if (!setting(args[4 + i], *u, i == 1 ? at::kInt : at::kFloat, by_row[i], all[i])) Py_RETURN_NONE;
  const int code = dt == at::kBFloat16 ? DKV_BF16 : dt == at::kHalf ? DKV_F16 : DKV_F32;
  at::Tensor out = at::empty({rows}, x->options().dtype(at::kLong)), ws;
  const long long need = dkv_sample_workspace_bytes(code, (int)rows, (int)V);
  if (need > 0) ws = at::empty({need}, x->options().dtype(at::kByte));
  int rc;
  void* const stream = PyLong_AsVoidPtr(args[0]);
  const int top_k = (int)(all[1] < 0.0 ? 0.0 : all[1] > (double)V ? (double)V : all[1]);
  Py_BEGIN_ALLOW_THREADS;
  rc = dkv_sample_tokens(
      stream, code, x->data_ptr(), rows > 1 ? x->stride(0) : V, (int)rows, (int)V,
      static_cast<const float*>(u->data_ptr()), static_cast<const float*>(by_row[0]), (float)all[0],
      static_cast<const int*>(by_row[1]), top_k, static_cast<const float*>(by_row[2]), (float)all[2],
      static_cast<const float*>(by_row[3]), (float)all[3], need > 0 ? ws.data_ptr() : nullptr, need,
      static_cast<long long*>(out.data_ptr()));
  Py_END_ALLOW_THREADS;
  if (rc != DKV_OK) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(out));
}

// A (rows, n) tensor of a type, on a device, with unit last stride.
const at::Tensor* matrix(PyObject* o, long long rows, c10::Device d) {
  const at::Tensor* t = tensor(o);
  return t && t->dim() == 2 && t->size(0) == rows && t->device() == d && t->size(1) <= INT_MAX &&
                 (t->size(1) <= 1 || t->stride(1) == 1)
             ? t
             : nullptr;
}

// (stream, device, logits, tokens, prompt_lens, lens, repetition, frequency, presence, bias_ids, bias,
// allowed) -> True
PyObject* adjust_logits(PyObject*, PyObject* const* args, Py_ssize_t n) {
  long long dev;
  if (n != 12 || !ints(args + 1, 1, &dev)) Py_RETURN_NONE;
  const at::Tensor* x = tensor(args[2]);
  if (!x || x->dim() != 2 || !x->is_cuda() || x->get_device() != dev) Py_RETURN_NONE;
  const long long rows = x->size(0), V = x->size(1);
  const auto dt = x->scalar_type();
  if (rows > INT_MAX || V > INT_MAX || (V > 1 && x->stride(1) != 1) ||
      (rows > 1 && x->stride(0) < V) ||
      (dt != at::kBFloat16 && dt != at::kHalf && dt != at::kFloat))
    Py_RETURN_NONE;
  const c10::Device d = x->device();
  const at::Tensor *tokens = nullptr, *ids = nullptr, *bias = nullptr, *allowed = nullptr;
  long long N = 0;
  if (args[3] != Py_None) {
    tokens = matrix(args[3], rows, d);
    if (!tokens || (tokens->scalar_type() != at::kInt && tokens->scalar_type() != at::kLong))
      Py_RETURN_NONE;
    N = tokens->size(1);
  } else if (args[4] != Py_None || args[5] != Py_None) {
    Py_RETURN_NONE;
  }
  const void* by_row[5] = {};
  double all[5] = {0.0, (double)N, 1.0, 0.0, 0.0};
  const double none[5] = {0.0, 0.0, 1.0, 0.0, 0.0};
  for (int i = 0; i < 5; ++i) {
    PyObject* o = args[4 + i];
    if (i < 2) {
      if (o == Py_None) continue;
      if (PyFloat_Check(o)) Py_RETURN_NONE;
    }
    const at::Tensor* t = tensor(o);
    if (t && (t->dim() != 1 || t->size(0) != rows || t->device() != d ||
              t->scalar_type() != (i < 2 ? at::kInt : at::kFloat) || !t->is_contiguous()))
      Py_RETURN_NONE;
    if (t) {
      by_row[i] = t->data_ptr();
      all[i] = none[i];
    } else if (PyFloat_Check(o)) {
      all[i] = PyFloat_AS_DOUBLE(o);
    } else {
      long long v;
      if (!PyLong_Check(o) || !ints(&o, 1, &v)) Py_RETURN_NONE;
      all[i] = (double)v;
    }
    if (i < 2) all[i] = all[i] < 0.0 ? 0.0 : all[i] > (double)N ? (double)N : all[i];
    if (i >= 2 && !tokens && (t || all[i] != none[i])) Py_RETURN_NONE;
  }
  if (!(all[2] > 0.0 && all[2] <= 3.4e38)) Py_RETURN_NONE;
  if (args[9] != Py_None || args[10] != Py_None) {
    ids = matrix(args[9], rows, d), bias = matrix(args[10], rows, d);
    if (!ids || !bias || ids->scalar_type() != at::kInt || bias->scalar_type() != at::kFloat ||
        ids->size(1) != bias->size(1))
      Py_RETURN_NONE;
  }
  if (args[11] != Py_None) {
    allowed = matrix(args[11], rows, d);
    if (!allowed || allowed->scalar_type() != at::kInt || allowed->size(1) * 32 < V) Py_RETURN_NONE;
  }
  const int code = dt == at::kBFloat16 ? DKV_BF16 : dt == at::kHalf ? DKV_F16 : DKV_F32;
  int rc;
  void* const stream = PyLong_AsVoidPtr(args[0]);
  auto ld = [&](const at::Tensor* t) { return t && rows > 1 ? t->stride(0) : 0; };
  Py_BEGIN_ALLOW_THREADS;
  rc = dkv_adjust_logits(
      stream, code, x->data_ptr(), rows > 1 ? x->stride(0) : V, (int)rows, (int)V,
      tokens ? tokens->data_ptr() : nullptr, tokens && tokens->scalar_type() == at::kLong ? 8 : 4,
      ld(tokens), (int)N, static_cast<const int*>(by_row[0]), (int)all[0],
      static_cast<const int*>(by_row[1]), (int)all[1], static_cast<const float*>(by_row[2]),
      (float)all[2], static_cast<const float*>(by_row[3]), (float)all[3],
      static_cast<const float*>(by_row[4]), (float)all[4],
      ids ? static_cast<const int*>(ids->data_ptr()) : nullptr, ld(ids),
      bias ? static_cast<const float*>(bias->data_ptr()) : nullptr, ld(bias),
      ids ? (int)ids->size(1) : 0,
      allowed ? static_cast<const int*>(allowed->data_ptr()) : nullptr, ld(allowed));
  Py_END_ALLOW_THREADS;
  if (rc != DKV_OK) Py_RETURN_NONE;
  Py_RETURN_TRUE;
}

// (a C++ exception, of a tensor without memory or an allocation that failed: the Python function's)
template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyObject* guarded(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  try {
    return F(self, args, n);
  } catch (const std::exception&) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
}

#define DKV_ENTRY(name) \
  {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(guarded<name>)), METH_FASTCALL, nullptr}

PyMethodDef methods[] = {DKV_ENTRY(paged_batch), DKV_ENTRY(paged_append), DKV_ENTRY(paged_attention),
                         DKV_ENTRY(paged_values), DKV_ENTRY(sample_tokens),
                         DKV_ENTRY(adjust_logits), {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_dkv_tensor", nullptr, -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__dkv_tensor(void) {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "torch_version", TORCH_VERSION) < 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
